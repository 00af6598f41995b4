"""Group normalisation with an activation, channels last, for training: the GroupNormalization + swish pairs of the bit-flip
UNet's ResBlocks (``mnist_diffusion.py:168-193``), forward and backward, in float32, bfloat16 and float16.

    y = act(xhat * gamma + beta),   xhat = (u - mean) * rstd,   u = x + shift

``x`` is (B, ..., C) with any number of axes between; ``mean`` and ``rstd = 1 / sqrt(var + eps)`` are taken over those axes and
the channels of a group.  ``shift`` (B, C), (1, C) or (C,) is the block's time vector, added to every pixel.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

ACTIVATIONS = {"none": _lib.IDM_ACT_NONE, "swish": _lib.IDM_ACT_SWISH}
DTYPES = {torch.float32: _lib.IDM_DT_F32, torch.bfloat16: _lib.IDM_DT_BF16, torch.float16: _lib.IDM_DT_F16}


def _layout(x):
    """(x, stride of a sample, stride of a pixel) with x itself where its middle axes are evenly strided, else a dense copy."""
    shape = x.shape
    if x.is_contiguous():
        c = shape[-1]
        return x, x.numel() // max(1, shape[0]), c
    stride, c = x.stride(), shape[-1]
    if x.numel() and (stride[-1] == 1 or c == 1):
        axes = [(n, s) for n, s in zip(shape[1:-1], stride[1:-1]) if n != 1]
        pixel = axes[-1][1] if axes else c
        want, even = pixel, pixel >= c
        for n, s in reversed(axes):
            even = even and s == want
            want = s * n
        if even:
            return x, stride[0] if shape[0] > 1 else 0, pixel
    x = x.contiguous()
    return x, x.numel() // max(1, shape[0]), c


def _check(x, gamma, beta, shift, groups, activation):
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        raise ValueError("x must be a tensor (B, ..., C)")
    if x.dtype not in DTYPES:
        raise ValueError("x must be float32, bfloat16 or float16")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
    b, c = x.shape[0], x.shape[-1]
    if not isinstance(groups, int) or groups <= 0 or c == 0 or c % groups:
        raise ValueError(f"groups must divide the {c} channels")
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (c,) or t.device != x.device):
            raise ValueError(f"{name} must be ({c},) float32 on the device of x")
    if shift is not None and (shift.dtype != torch.float32 or shift.device != x.device or shift.shape not in ((b, c), (1, c), (c,))):
        raise ValueError(f"shift must be ({b}, {c}), (1, {c}) or ({c},) float32 on the device of x")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dense(t):
    return None if t is None else t.contiguous()


def _desc(x, groups, activation, sample, pixel, shift, eps=0.0, dy_sample=0, dy_pixel=0):
    b, c = x.shape[0], x.shape[-1]
    per_sample = shift is not None and shift.dim() == 2 and shift.shape[0] == b and b > 1
    return _lib.GroupNormDesc(DTYPES[x.dtype], ACTIVATIONS[activation], b, x.numel() // max(1, b * c), c, groups, sample, pixel,
                              dy_sample, dy_pixel, c if per_sample else 0, eps, 0)


def _workspace(desc, backward, device):
    size = C.c_size_t()
    _lib.check(_lib.load().idm_group_norm_workspace(C.byref(desc), backward, C.byref(size)))
    return torch.empty(max(16, size.value), dtype=torch.uint8, device=device), size.value


def group_norm_forward(x, gamma, beta, groups: int = 8, *, shift=None, eps: float = 1e-3, activation: str = "swish"):
    """Returns ``(y, mean, rstd)``: y like x (dense), mean and rstd (B, groups) float32 for :func:`group_norm_backward`.
    ``gamma`` and ``beta`` (C,) float32 may be None (1 and 0).  Strided x (a slice of the channels, a cropped map) is read in
    place where its pixels are evenly spaced.  No gradients are recorded: :func:`group_norm` does that."""
    _check(x, gamma, beta, shift, groups, activation)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    dev = x.device
    x, sample, pixel = _layout(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats = torch.empty((2, x.shape[0], groups), dtype=torch.float32, device=dev)
    if x.numel() == 0:
        return y, stats[0].zero_(), stats[1].fill_(eps ** -0.5 if eps else math.inf)
    gamma, beta, shift = _dense(gamma), _dense(beta), _dense(shift)
    desc = _desc(x, groups, activation, sample, pixel, shift, eps)
    with torch.cuda.device(dev):
        ws, size = _workspace(desc, 0, dev)
        _lib.check(_lib.load().idm_group_norm_forward(dev.index, C.byref(desc), x.data_ptr(), _ptr(gamma), _ptr(beta), _ptr(shift),
                                                      y.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), ws.data_ptr(), size,
                                                      torch.cuda.current_stream(dev).cuda_stream))
    return y, stats[0], stats[1]


def group_norm_backward(dy, x, mean, rstd, gamma, beta, groups: int = 8, *, shift=None, activation: str = "swish"):
    """Gradients for ``dy`` = dL/dy: ``(dx, dgamma, dbeta, dshift)``; dgamma, dbeta and dshift are None where gamma, beta and
    shift are, dshift has the shape of shift.  The arguments after ``dy`` are those of the forward call and its statistics.
    Equal inputs give equal bits."""
    _check(x, gamma, beta, shift, groups, activation)
    b, c = x.shape[0], x.shape[-1]
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must have the shape, type and device of x")
    for t in (mean, rstd):
        if t.shape != (b, groups) or t.dtype != torch.float32 or t.device != x.device:
            raise ValueError(f"mean and rstd must be ({b}, {groups}) float32 on the device of x")
    dev = x.device
    x, sample, pixel = _layout(x)
    dy, dy_sample, dy_pixel = _layout(dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    new = lambda t: None if t is None else torch.empty(t.shape, dtype=torch.float32, device=dev)  # noqa: E731
    dgamma, dbeta, dshift = new(gamma), new(beta), new(shift)
    if x.numel() == 0:
        for t in (dgamma, dbeta, dshift):
            if t is not None:
                t.zero_()
        return dx, dgamma, dbeta, dshift
    gamma, beta, shift, mean, rstd = (_dense(t) for t in (gamma, beta, shift, mean, rstd))
    desc = _desc(x, groups, activation, sample, pixel, shift, 0.0, dy_sample, dy_pixel)
    with torch.cuda.device(dev):
        ws, size = _workspace(desc, 1, dev)
        _lib.check(_lib.load().idm_group_norm_backward(dev.index, C.byref(desc), dy.data_ptr(), x.data_ptr(), mean.data_ptr(),
                                                       rstd.data_ptr(), _ptr(gamma), _ptr(beta), _ptr(shift), dx.data_ptr(),
                                                       _ptr(dgamma), _ptr(dbeta), _ptr(dshift), ws.data_ptr(), size,
                                                       torch.cuda.current_stream(dev).cuda_stream))
    return dx, dgamma, dbeta, dshift


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, shift, groups, eps, activation):
        y, mean, rstd = group_norm_forward(x, gamma, beta, groups, shift=shift, eps=eps, activation=activation)
        ctx.save_for_backward(x, gamma, beta, shift, mean, rstd)
        ctx.how = groups, activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, gamma, beta, shift, mean, rstd = ctx.saved_tensors
        groups, activation = ctx.how
        dx, dgamma, dbeta, dshift = group_norm_backward(dy, x, mean, rstd, gamma, beta, groups, shift=shift, activation=activation)
        return dx, dgamma, dbeta, dshift, None, None, None


def group_norm(x, gamma=None, beta=None, groups: int = 8, *, shift=None, eps: float = 1e-3, activation: str = "swish"):
    """``act(GroupNorm(x + shift))`` with gradients for x, gamma, beta and shift (once differentiable).  gamma, beta and shift may
    be of any floating type here; they are computed with in float32."""
    up = lambda t: None if t is None else t.float()  # noqa: E731
    return _GroupNorm.apply(x, up(gamma), up(beta), up(shift), groups, eps, activation)

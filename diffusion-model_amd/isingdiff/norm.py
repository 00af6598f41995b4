"""Group normalisation with an activation, channels last, for training: the GroupNormalization + swish pairs of the bit-flip
UNet's ResBlocks (``mnist_diffusion.py:168-193``), forward and backward, in float32, bfloat16 and float16.

    y = act(xhat * gamma + beta),   xhat = (u - mean) * rstd,   u = x + shift

``x`` is (B, ..., C) with any number of axes between; ``mean`` and ``rstd = 1 / sqrt(var + eps)`` are taken over those axes and
the channels of a group.  ``shift`` (B, C), (1, C) or (C,) is the block's time vector, added to every pixel.
"""
from __future__ import annotations

import ctypes as C
import functools
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


def _refuse(x, gamma, beta, shift, groups, activation):
    """The reason why these arguments are refused; called once a check has failed, or for a shape that is new."""
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        return "x must be a tensor (B, ..., C)"
    if x.dtype not in DTYPES:
        return "x must be float32, bfloat16 or float16"
    if activation not in ACTIVATIONS:
        return f"activation must be one of {tuple(ACTIVATIONS)}"
    b, c = x.shape[0], x.shape[-1]
    if not isinstance(groups, int) or groups <= 0 or c == 0 or c % groups:
        return f"groups must divide the {c} channels"
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (c,) or t.device != x.device):
            return f"{name} must be ({c},) float32 on the device of x"
    if shift is not None and (shift.dtype != torch.float32 or shift.device != x.device or shift.shape not in ((b, c), (1, c), (c,))):
        return f"shift must be ({b}, {c}), (1, {c}) or ({c},) float32 on the device of x"
    if not x.is_cuda:
        return "x must be a CUDA tensor"
    return None


def _check(x, gamma, beta, shift, groups, activation):
    why = _refuse(x, gamma, beta, shift, groups, activation)
    if why:
        raise ValueError(why)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _like(x):
    """A dense tensor like x."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=256)
def _plan(shape, dtype, groups, activation, strides, per_sample, eps, aligned, backward):
    """(descriptor, bytes of workspace) of a call: a function of sizes alone."""
    b, c = shape[0], shape[-1]
    desc = _lib.GroupNormDesc(DTYPES[dtype], ACTIVATIONS[activation], b, shape.numel() // (b * c), c, groups, *strides,
                              c if per_sample else 0, eps, aligned)
    size = C.c_size_t()
    _lib.check(_lib.load().idm_group_norm_workspace(C.byref(desc), backward, C.byref(size)))
    return C.byref(desc), size.value, desc


def _call(entry, dev, plan, args):
    desc, size, _ = plan
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _lib.call(entry, dev, (desc, *args, _ptr(ws), size))


def group_norm_forward(x, gamma, beta, groups: int = 8, *, shift=None, eps: float = 1e-3, activation: str = "swish"):
    """Returns ``(y, mean, rstd)``: y like x (dense), mean and rstd (B, groups) float32 for :func:`group_norm_backward`.
    ``gamma`` and ``beta`` (C,) float32 may be None (1 and 0).  Strided x (a slice of the channels, a cropped map) is read in
    place where its pixels are evenly spaced.  No gradients are recorded: :func:`group_norm` does that."""
    _check(x, gamma, beta, shift, groups, activation)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    x, sample, pixel = _layout(x)
    shape = x.shape
    y = _like(x)
    mean = torch.empty((shape[0], groups), dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    if x.numel() == 0:
        return y, mean.zero_(), rstd.fill_(eps ** -0.5 if eps else math.inf)
    gamma, beta, shift = _dense(gamma), _dense(beta), _dense(shift)
    per_sample = shift is not None and shift.dim() == 2 and 1 < shape[0] == shift.shape[0]
    px, pg, pb, ps, py = x.data_ptr(), _ptr(gamma), _ptr(beta), _ptr(shift), y.data_ptr()
    aligned = not (px | pg | pb | ps | py) & 15
    plan = _plan(shape, x.dtype, groups, activation, (sample, pixel, 0, 0), per_sample, eps, aligned, 0)
    _call(_lib.load().idm_group_norm_forward, x.device, plan, (px, pg, pb, ps, py, mean.data_ptr(), rstd.data_ptr()))
    return y, mean, rstd


def group_norm_backward(dy, x, mean, rstd, gamma, beta, groups: int = 8, *, shift=None, activation: str = "swish"):
    """Gradients for ``dy`` = dL/dy: ``(dx, dgamma, dbeta, dshift)``; dgamma, dbeta and dshift are None where gamma, beta and
    shift are, dshift has the shape of shift.  The arguments after ``dy`` are those of the forward call and its statistics.
    Equal inputs give equal bits."""
    _check(x, gamma, beta, shift, groups, activation)
    shape = x.shape
    if dy.shape != shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must have the shape, type and device of x")
    for t in (mean, rstd):
        if t.shape != (shape[0], groups) or t.dtype != torch.float32 or t.device != x.device:
            raise ValueError(f"mean and rstd must be ({shape[0]}, {groups}) float32 on the device of x")
    x, sample, pixel = _layout(x)
    dy, dy_sample, dy_pixel = _layout(dy)
    dx = _like(x)
    new = lambda t: None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)  # noqa: E731
    dgamma, dbeta, dshift = new(gamma), new(beta), new(shift)
    if x.numel() == 0:
        for t in (dgamma, dbeta, dshift):
            if t is not None:
                t.zero_()
        return dx, dgamma, dbeta, dshift
    gamma, beta, shift, mean, rstd = _dense(gamma), _dense(beta), _dense(shift), _dense(mean), _dense(rstd)
    per_sample = shift is not None and shift.dim() == 2 and 1 < shape[0] == shift.shape[0]
    pd, px, pg, pb, ps, po = dy.data_ptr(), x.data_ptr(), _ptr(gamma), _ptr(beta), _ptr(shift), dx.data_ptr()
    aligned = not (pd | px | pg | pb | ps | po) & 15
    plan = _plan(shape, x.dtype, groups, activation, (sample, pixel, dy_sample, dy_pixel), per_sample, 0.0, aligned, 1)
    _call(_lib.load().idm_group_norm_backward, x.device, plan, (pd, px, mean.data_ptr(), rstd.data_ptr(), pg, pb, ps, po, _ptr(dgamma),
                                                                _ptr(dbeta), _ptr(dshift)))
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

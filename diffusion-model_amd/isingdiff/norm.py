"""Group normalisation with an activation, channels last, for training: the GroupNormalization + swish pairs of the bit-flip
UNet's ResBlocks (``mnist_diffusion.py:168-193``), forward and backward, in float32, bfloat16 and float16.

    y = act(xhat * gamma + beta),   xhat = (u - mean) * rstd,   u = x + shift

``x`` is (B, ..., C) with any number of axes between; ``mean`` and ``rstd = 1 / sqrt(var + eps)`` are taken over those axes and
the channels of a group.  ``shift`` (B, C), (1, C) or (C,) is the block's time vector, added to every pixel.
"""
from __future__ import annotations

import torch

from ._lib import host


def _layout(x):
    """(x, stride of a sample, stride of a pixel) with x itself where its middle axes are evenly strided, else a dense copy."""
    return host().layout(x)


def group_norm_forward(x, gamma, beta, groups: int = 8, *, shift=None, eps: float = 1e-3, activation: str = "swish"):
    """Returns ``(y, mean, rstd)``: y like x (dense), mean and rstd (B, groups) float32 for :func:`group_norm_backward`.
    ``gamma`` and ``beta`` (C,) float32 may be None (1 and 0).  Strided x (a slice of the channels, a cropped map) is read in
    place where its pixels are evenly spaced.  No gradients are recorded: :func:`group_norm` does that."""
    return host().group_norm_forward(x, gamma, beta, shift, groups, eps, activation)


def group_norm_backward(dy, x, mean, rstd, gamma, beta, groups: int = 8, *, shift=None, activation: str = "swish"):
    """Gradients for ``dy`` = dL/dy: ``(dx, dgamma, dbeta, dshift)``; dgamma, dbeta and dshift are None where gamma, beta and
    shift are, dshift has the shape of shift.  The arguments after ``dy`` are those of the forward call and its statistics.
    Equal inputs give equal bits."""
    return host().group_norm_backward(dy, x, mean, rstd, gamma, beta, shift, groups, activation)


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
    be of any floating type here; they are computed with in float32.  May be captured into a HIP graph with its backward pass, but not
    while a graph of an eager pass over the same leaves is alive."""
    if (isinstance(x, torch.Tensor) and x.is_cuda and torch.cuda.is_current_stream_capturing() and torch.is_grad_enabled()
            and host().adds_elsewhere(x, gamma, beta, shift)):
        raise ValueError("a graph of an eager pass over these leaves is alive: drop it (its loss) before a backward pass is captured")
    up = lambda t: None if t is None else t.float()  # noqa: E731
    return _GroupNorm.apply(x, up(gamma), up(beta), up(shift), groups, eps, activation)

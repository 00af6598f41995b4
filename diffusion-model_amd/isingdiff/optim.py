"""AdamW over many tensors at once, moments in 32 or in 8 bits.

    t += 1;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

Parameters and gradients are float32, bfloat16 or float16 (all parameters of a call of one type, all gradients of one type); the
arithmetic is float32 and a parameter is rounded once.  The state is a dict of flat tensors: tensor i's moments begin at the sum
of the sizes before it, each rounded up to 256 entries.

8-bit moments take 1 byte an entry and 2 bytes for each block of 256: a code is a float with three mantissa bits whose
exponent window (16 binades for m, 32 for v) follows the largest entry of its block.  What is cut off is rounded with a dither that is
equidistributed over entries and steps, so a second moment that drifts by less than a code a step still moves at its mean rate; an
entry of m or v is off by up to one code (1/8 of its binade) at any one step.
"""
from __future__ import annotations

import ctypes as C
import math
import operator
from array import array
from itertools import repeat

import torch

from . import _lib
from .norm import DTYPES

BLOCK = _lib.ADAMW_BLOCK
assert BLOCK == 1 << 8


def _room(n: int) -> int:
    return -(-n // BLOCK) * BLOCK


def adamw_state(params, moment_bits: int = 32) -> dict:
    """The state before the first step: ``step`` int64 (1,) and ``m``, ``v`` on the parameters' device, float32, or uint8 with
    ``m_base``, ``v_base`` int16 (one per block of 256) for ``moment_bits=8``."""
    params = list(params)
    if moment_bits not in (32, 8):
        raise ValueError("moment_bits must be 32 or 8")
    if not params:
        raise ValueError("no parameters")
    dev, total = params[0].device, sum(_room(p.numel()) for p in params)
    zeros = lambda n, t: torch.zeros(n, dtype=t, device=dev)  # noqa: E731
    kind = torch.float32 if moment_bits == 32 else torch.uint8
    state = {"step": zeros(1, torch.int64), "m": zeros(total, kind), "v": zeros(total, kind)}
    if moment_bits == 8:
        state.update(m_base=zeros(total // BLOCK, torch.int16), v_base=zeros(total // BLOCK, torch.int16))
    return state


def _check_state(state, total, dev):
    """Moment bits of a state that fits `total` entries (None: any whole number of blocks) on `dev`."""
    eight = state["m"].dtype == torch.uint8
    kind = torch.uint8 if eight else torch.float32
    total = state["m"].numel() if total is None else total
    for k in ("step", "m", "v", "m_base", "v_base") if eight else ("step", "m", "v"):
        t = state[k]
        want, n = (torch.int64, 1) if k == "step" else (torch.int16, total // BLOCK) if k.endswith("base") else (kind, total)
        if t.dtype != want or t.numel() != n or t.device != dev or not t.is_contiguous():
            raise ValueError(f"state[{k!r}] must be {n} dense {want} values on {dev}: make it with adamw_state for these parameters")
    return 8 if eight else 32


def adamw_step(params, grads, state, *, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01):
    """One step, in place: ``params``, and ``state`` of :func:`adamw_state`.  ``weight_decay`` is a number, or one per tensor.  A
    gradient that is None leaves its tensor and moments as they are.  Enqueued on the current stream; a captured step replays with
    the tensors, lr and decays that it was captured with, while its step count goes on."""
    # (loops over the tensors are map() of tensor methods: at 66 tensors the host is slower than the device)
    params, grads = list(params), list(grads)
    n = len(params)
    if not n or n != len(grads):
        raise ValueError("params and grads must be lists of the same length, not empty")
    given, with_grad = grads, params
    if any(map(operator.is_, grads, repeat(None))):
        with_grad = [p for p, g in zip(params, grads) if g is not None]
        given = [g for g in grads if g is not None]
    Tensor = torch.Tensor
    dev, ptype = params[0].device, params[0].dtype
    gtype = given[0].dtype if given else ptype
    if ptype not in DTYPES or gtype not in DTYPES:
        raise ValueError("parameters and gradients must be float32, bfloat16 or float16")
    where = set(map(Tensor.get_device, params)) | set(map(Tensor.get_device, given))
    if {p.dtype for p in params} != {ptype} or len(where) != 1 or not all(map(Tensor.is_contiguous, params)):
        raise ValueError("parameters must be dense, of one type and on one device")
    if given and {g.dtype for g in given} != {gtype}:
        raise ValueError("all gradients must be of one type")
    if not all(map(Tensor.is_contiguous, given)):
        given = [g.contiguous() for g in given]
    counts = list(map(Tensor.numel, params))
    sizes = array("q", counts)
    # (dense tensors of the same strides and sizes hold the same entries in the same order; shapes cost more to ask for)
    same = (list(map(Tensor.stride, given)) == list(map(Tensor.stride, with_grad))
            and list(map(Tensor.numel, given)) == (counts if with_grad is params else list(map(Tensor.numel, with_grad))))
    if not same and [g.shape for g in given] != [p.shape for p in with_grad]:
        raise ValueError("a gradient must have its parameter's shape and device")
    if isinstance(weight_decay, (int, float)):
        lowest, decay = weight_decay, array("f", (weight_decay,)) * n
    else:
        decay = array("f", weight_decay)
        if len(decay) != n:
            raise ValueError("weight_decay must be a number or one per tensor")
        lowest = min(decay)
    if not (math.isfinite(lr) and lr >= 0 and math.isfinite(eps) and eps >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1
            and lowest >= 0 and math.isfinite(sum(decay))):
        raise ValueError("lr, eps and weight_decay must be finite and not negative, betas in [0, 1)")
    bits = _check_state(state, sum([s + BLOCK - 1 >> 8 for s in counts]) * BLOCK, dev)
    if dev.type != "cuda":
        raise ValueError("parameters must be CUDA tensors")
    at = array("q", list(map(Tensor.data_ptr, params)))
    if len(given) == n:
        grad_at = array("q", list(map(Tensor.data_ptr, given)))
    else:
        it = iter(given)
        grad_at = array("q", [0 if g is None else next(it).data_ptr() for g in grads])
    cfg = _lib.AdamWCfg(DTYPES[ptype], DTYPES[gtype], bits, 0, lr, betas[0], betas[1], eps)
    base = (state["m_base"].data_ptr(), state["v_base"].data_ptr()) if bits == 8 else (None, None)
    scratch = torch.empty(2, dtype=torch.int64, device=dev)
    _lib.call(_lib.load().idm_adamw_step, dev, (C.byref(cfg), n, at.buffer_info()[0], grad_at.buffer_info()[0], sizes.buffer_info()[0],
                                            decay.buffer_info()[0], state["m"].data_ptr(), state["v"].data_ptr(), *base,
                                            state["m"].numel(), state["step"].data_ptr(), scratch.data_ptr()))
    # the kernel writes behind autograd's back: a backward pass that saved a parameter has to see that it changed
    torch.autograd.graph.increment_version(params)


def adamw_moments(state):
    """The float32 values ``(m, v)`` of a state, flat as its own tensors: those tensors themselves in 32 bits, the values that the codes
    stand for in 8."""
    dev = state["m"].device
    bits = _check_state(state, None, dev)
    if bits == 32:
        return state["m"], state["v"]
    if dev.type != "cuda":
        raise ValueError("the state must be on a CUDA device")
    n = state["m"].numel()
    m = torch.empty(n, dtype=torch.float32, device=dev)
    v = torch.empty_like(m)
    _lib.call(_lib.load().idm_adamw_moments, dev, (*(state[k].data_ptr() for k in ("m", "v", "m_base", "v_base")), m.data_ptr(), v.data_ptr(), n))
    return m, v


class AdamW:
    """``opt = AdamW(params); loss.backward(); opt.step(); opt.zero_grad()``: :func:`adamw_step` with the gradients that autograd
    left in ``p.grad``.  ``weight_decay`` may be a number or one per tensor; ``lr`` may be changed between steps."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, moment_bits: int = 32):
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.state = adamw_state(self.params, moment_bits)

    def step(self):
        with torch.no_grad():
            adamw_step(self.params, [p.grad for p in self.params], self.state, lr=self.lr, betas=self.betas, eps=self.eps,
                       weight_decay=self.weight_decay)

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    def state_dict(self) -> dict:
        return {k: v.clone() for k, v in self.state.items()}

    def load_state_dict(self, state: dict):
        if set(state) != set(self.state):
            raise ValueError("the state has other moments than this optimizer")
        for k, t in self.state.items():
            if state[k].shape != t.shape or state[k].dtype != t.dtype:
                raise ValueError(f"state[{k!r}] does not fit these parameters")
        for k, t in self.state.items():
            t.copy_(state[k])

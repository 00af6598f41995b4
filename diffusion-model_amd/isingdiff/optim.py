"""AdamW over many tensors at once, moments in 32 or in 8 bits.

    t += 1;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

Parameters and gradients are float32, bfloat16 or float16 (all parameters of a call of one type, all gradients of one type); the
arithmetic is float32 and a parameter is rounded once.  The state is a dict of flat tensors: tensor i's moments begin at the sum
of the sizes before it, each rounded up to 256 entries.  ``step`` counts the calls, for all tensors: one that gets its first gradient in a
later call has its moments corrected by that count, not by its own (with the default betas its first update is
2.5 lr at step 1 000 and 3.2 lr long after).

8-bit moments take 1 byte an entry and 2 bytes for each block of 256: a code is a float with three mantissa bits whose
exponent window (16 binades for m, 32 for v) follows the largest entry of its block.  What is cut off is rounded with a dither that is
equidistributed over entries and steps, so a second moment that drifts by less than a code a step still moves at its mean rate; an
entry of m or v is off by up to one code (1/8 of its binade) at any one step.
"""
from __future__ import annotations

import torch

from ._lib import ADAMW_BLOCK as BLOCK
from ._lib import host


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


def adamw_step(params, grads, state, *, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01):
    """One step, in place: ``params``, and ``state`` of :func:`adamw_state`.  ``weight_decay`` is a number, or one per tensor.  A
    gradient that is None leaves its tensor and moments as they are.  Enqueued on the current stream; a captured step replays with
    the tensors, lr and decays that it was captured with, while its step count goes on."""
    host().adamw_step(params, grads, state, lr, betas, eps, weight_decay)


def adamw_moments(state):
    """The float32 values ``(m, v)`` of a state, flat as its own tensors: those tensors themselves in 32 bits, the values that the codes
    stand for in 8."""
    return host().adamw_moments(state)


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
        if not 0 <= int(state["step"]) < 2 ** 53 - 1:
            raise ValueError("state['step'] must be a count of steps")
        for k, t in self.state.items():
            t.copy_(state[k])

"""Training of the bit-flip UNet: the norms, their gradients and the optimizer step together, as BitflipTrainer runs them."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from isingdiff import bitflip

pytestmark = pytest.mark.gpu


def batch(n, h, w, time_step, seed):
    r = np.random.RandomState(seed)
    x0, flips = r.rand(n, h, w) < 0.3, r.rand(n, h, w) < 0.2
    return (x0 ^ flips).astype(np.uint8), r.randint(0, time_step, n), flips.astype(np.float32)


def reference(weights, emb, X, t):
    """Logits in float64 from library operators, with gradients for a dict of weights."""
    w = {k: torch.tensor(np.asarray(v, np.float64), requires_grad=True) for k, v in weights.items()}
    conv = lambda x, k, pad: F.conv2d(x, w[k].permute(3, 2, 0, 1), padding=pad)  # noqa: E731
    temb = F.silu(torch.tensor(emb[t].astype(np.float64)) @ w["d1_w"] + w["d1_b"])
    temb = F.silu(temb @ w["d2_w"] + w["d2_b"])

    def block(i, x):
        g = lambda k: w[f"b{i}_{k}"]  # noqa: E731
        at = lambda v: v[None, :, None, None]  # noqa: E731
        h = F.silu(F.group_norm(x, 8, g("g1_g"), g("g1_b"), 1e-3))
        h = conv(h, f"b{i}_c1_w", 1) + at(g("c1_b")) + F.silu(temb @ g("t_w") + g("t_b"))[:, :, None, None]
        h = conv(F.silu(F.group_norm(h, 8, g("g2_g"), g("g2_b"), 1e-3)), f"b{i}_c2_w", 1) + at(g("c2_b"))
        return h + (conv(x, f"b{i}_s_w", 0) + at(g("s_b")) if f"b{i}_s_w" in w else x)
    grow = lambda x: F.interpolate(x, scale_factor=2, mode="nearest")  # noqa: E731
    x = conv(torch.tensor(X.astype(np.float64))[:, None], "in_w", 0) + w["in_b"][None, :, None, None]
    s1 = block(0, x)
    s2 = block(1, F.max_pool2d(s1, 2))
    mid = block(2, F.max_pool2d(s2, 2))
    d3 = block(3, torch.cat([grow(mid), s2], 1))
    d4 = block(4, torch.cat([grow(d3), s1], 1))
    return (conv(d4, "out_w", 0) + w["out_b"][None, :, None, None])[:, 0], w


def rel(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("precision,n,h,w", [("fp32", 3, 28, 28), ("fp32", 2, 12, 20), ("bf16", 4, 28, 28)])
def test_logits_and_gradients(precision, n, h, w):
    """About 30 tensors lie between a weight and the loss, each rounded once or summed over at most 9 * 192 terms: sqrt(1728) * 2^-24
    relative to its 2-norm, times 4 for the norms (values up to about three deviations from zero): 3e-4 in float32; in bfloat16 30
    roundings of 2^-9 add like a random walk, sqrt(30) * 2^-9 * 4 = 4e-2.  A weight's own gradient may be a difference of larger sums
    (an offset in front of a norm): held to 30 times that, the whole gradient to once."""
    weights = bitflip.synthetic_weights(1)
    X, t, flips = batch(n, h, w, 100, 5)
    tr = bitflip.BitflipTrainer(weights, precision=precision)
    logits = tr.logits(X, t)
    loss = F.binary_cross_entropy_with_logits(logits, torch.tensor(flips, device="cuda"))
    grads = torch.autograd.grad(loss, list(tr.params.values()))
    want, leaves = reference(weights, bitflip.sinusoidal_table(100), X, t)
    ref = torch.autograd.grad(F.binary_cross_entropy_with_logits(want, torch.tensor(flips).double()), [leaves[k] for k in tr.params])
    tol = 3e-4 if precision == "fp32" else 4e-2
    assert rel(logits.detach().cpu().double(), want.detach()) < tol
    for k, a, b in zip(tr.params, grads, ref):
        assert rel(a.cpu().double(), b) < 30 * tol, k
    flat = lambda ts: torch.cat([x.detach().cpu().double().flatten() for x in ts])  # noqa: E731
    assert rel(flat(grads), flat(ref)) < tol


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_and_the_model_they_make(bits):
    """Three steps: every weight follows the optimizer's formula from its own gradient; the sampler's model gives the trainer's
    probabilities (float32 on both sides, other orders of summation)."""
    tr = bitflip.BitflipTrainer(bitflip.synthetic_weights(2), lr=1e-3, weight_decay=0.01, moment_bits=bits)
    for k in range(3):
        X, t, flips = batch(5, 28, 28, 100, 10 + k)
        before = {n: p.detach().double().clone() for n, p in tr.params.items()}
        loss = tr.step(X, t, flips)
        assert loss.dim() == 0 and bool(torch.isfinite(loss))
        if k == 0:     # m = (1 - b1) g, v = (1 - b2) g^2: the corrected update is g / (|g| + eps)
            for n, p in tr.params.items():
                g = p.grad.double()
                want = before[n] * (1 - 1e-3 * (0.01 if n.endswith("_w") else 0)) - 1e-3 * g / (g.abs() + 1e-7)
                assert float((p.detach().double() - want).abs().max()) < 1e-3 * 2 ** -18 + 2 ** -23 * float(want.abs().max()), n
    assert int(tr.opt.state["step"]) == 3
    X, _, _ = batch(3, 28, 28, 100, 77)
    with torch.no_grad():
        mine = torch.sigmoid(tr.logits(X, np.full(3, 40)))
    theirs = tr.model("fp32")([X, np.float32(40) / np.float32(100)])[..., 0]
    assert float((mine - theirs).abs().max()) < 1e-4


def test_refusals():
    w = bitflip.synthetic_weights(0)
    with pytest.raises(ValueError):
        bitflip.BitflipTrainer(w, precision="fp16")
    with pytest.raises(ValueError):
        bitflip.BitflipTrainer({**w, "in_w": w["in_w"][..., :16]})
    tr = bitflip.BitflipTrainer(w)
    X, t, flips = batch(2, 28, 28, 100, 0)
    for args in ((X[:, :26], t, flips), (X, t[:1], flips), (X, t.astype(np.float32), flips), (X, t, flips[:1]), (X[:0], t[:0], flips[:0]),
                 (X, t * 0 + 100, flips), (X, t * 0 - 1, flips)):
        with pytest.raises(ValueError):
            tr.step(*args)


def test_a_step_is_not_captured():
    from isingdiff import bitflip
    trainer = bitflip.BitflipTrainer(bitflip.synthetic_weights(0), time_step=10)
    X, t = torch.zeros(2, 4, 4, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            trainer.step(X, t, X)
    assert bool(torch.isfinite(trainer.step(X, t, X)))

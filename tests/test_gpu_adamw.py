"""AdamW over many tensors against the formula in 64 bits (moments in 32 bits) and against the codes' definition, value for value
(moments in 8 bits).

Tolerance of a parameter after one step, e = 2^-24, u = eps / 2 of its type: one rounding of the parameter, u |p|; the update is a chain of
at most 16 float32 roundings (moment, root, product, sum, quotient, product), 16 e of its size, and 4 e |p| for p (1 - lr wd) and the
difference.  The moments are float32 sums of two products: 4 e of the sizes of the two terms.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ROT_A, ROT_B, BLOCK = 0xC13FA9A9, 0x91E10DA5, 256
SIZES = [(1,), (3, 5), (255,), (256,), (257,), (4, 1024), (4097,), (64, 129), (31,), (20000,)]


def make(sizes, ptype, gtype, seed):
    g = torch.Generator().manual_seed(seed)
    params = [(0.1 * torch.randn(s, generator=g)).to(ptype).cuda() for s in sizes]
    grads = [(10.0 ** float(torch.rand(1, generator=g) * 4 - 4) * torch.randn(s, generator=g)).to(gtype).cuda() for s in sizes]
    return params, grads


def room(n):
    return -(-n // BLOCK) * BLOCK


def flat(ts):
    """The moments' layout: each tensor from a multiple of 256 entries on."""
    return np.concatenate([np.pad(t.detach().cpu().double().numpy().ravel(), (0, room(t.numel()) - t.numel())) for t in ts])


def place(x, turn):
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.int64)
    size = bits & 0x7fffffff
    q = (size + ((turn & 0xffffffff) >> 12)) >> 20
    return np.where(size < 0x7f800000, np.minimum(q, 2039), 2047), bits >> 31


def encode(x, turn, most):
    q, sign = place(x, turn)
    top = np.where(q < 2047, q, 0).reshape(-1, BLOCK).max(1)
    base = np.maximum(top - most, 0)
    code = q - np.repeat(base, BLOCK)
    code = np.where(q > 0, np.clip(code, 1, 255), 0) if most == 255 else np.clip(code, 0, 127) + 128 * sign
    return code.astype(np.uint8), base.astype(np.int16)


def decode(code, base, most):
    c = code.astype(np.int64)
    k, b = c & most, np.repeat(base.astype(np.int64), BLOCK)
    bits = np.where(k > 0, (k + b) << 20, 0).astype(np.uint32)
    return np.where(c > most, -1, 1).astype(np.float32) * bits.view(np.float32)


def moments32(m, v, g, b1, b2):
    """One float32 rounding for each product and sum."""
    f = np.float32
    m, v, g = m.astype(f), v.astype(f), g.astype(f)
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        return m * f(b1) + g * f(1 - b1), v * f(b2) + (g * g) * f(1 - b2)


def check_params(params, before, m, v, sizes, t, lr, b1, b2, eps, decay):
    at = 0
    for k, (p, s) in enumerate(zip(params, sizes)):
        n = p.numel()
        mm, vv, p0 = m[at:at + n].astype(np.float64), v[at:at + n].astype(np.float64), before[k].double().cpu().numpy().ravel()
        up = lr / (1 - b1 ** t) * mm / (np.sqrt(vv / (1 - b2 ** t)) + eps)
        want = p0 * (1 - lr * decay[k]) - up
        u = torch.finfo(p.dtype).eps / 2
        tol = u * np.abs(want) + 16 * E * np.abs(up) + 4 * E * np.abs(p0) + (3e-8 if p.dtype == torch.float16 else 0)
        off = np.abs(p.double().cpu().numpy().ravel() - want) - tol
        assert (off <= 0).all(), (k, s, off.max())
        at += room(n)


@pytest.mark.parametrize("gtype", list(TYPES))
@pytest.mark.parametrize("ptype", list(TYPES))
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_against_the_formula(bits, ptype, gtype):
    from isingdiff import adamw_moments, adamw_state, adamw_step
    lr, b1, b2, eps = 3e-3, 0.9, 0.99, 1e-7
    params, _ = make(SIZES, TYPES[ptype], TYPES[gtype], 1)
    decay = [0.1 * (k % 3) for k in range(len(SIZES))]
    state = adamw_state(params, bits)
    m = v = np.zeros(sum(room(p.numel()) for p in params), np.float32)
    ident = np.arange(m.size, dtype=np.int64)
    inside = np.concatenate([np.arange(room(p.numel())) < p.numel() for p in params])
    for t in range(1, 6):
        _, grads = make(SIZES, TYPES[ptype], TYPES[gtype], 10 + t)
        before = [p.clone() for p in params]
        adamw_step(params, grads, state, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay)
        assert int(state["step"]) == t
        m, v = moments32(m, v, flat(grads), b1, b2)
        check_params(params, before, m, v, SIZES, t, lr, b1, b2, eps, decay)
        gm, gv = (x.cpu().numpy() for x in adamw_moments(state))
        if bits == 8:
            turns = ident * ROT_A + t * ROT_B, ident * ROT_B + t * ROT_A
            (cm, bm), (cv, bv) = encode(m, turns[0], 127), encode(v, turns[1], 255)
            assert np.array_equal(state["m"].cpu().numpy() & 127, cm & 127) and np.array_equal(state["v"].cpu().numpy(), cv)
            assert np.array_equal(state["m_base"].cpu().numpy(), bm) and np.array_equal(state["v_base"].cpu().numpy(), bv)
            m, v = decode(cm, bm, 127), decode(cv, bv, 255)
        assert np.array_equal(gm[inside], m[inside]) and np.array_equal(gv[inside], v[inside])


def test_one_to_many_tensors_and_launches():
    """130 tensors need three launches; one step equals the same tensors stepped alone."""
    from isingdiff import adamw_state, adamw_step
    sizes = [(1 + 37 * k % 1000,) for k in range(130)]
    for bits in (32, 8):
        params, grads = make(sizes, torch.float32, torch.float32, 7)
        alone = [p.clone() for p in params]
        state = adamw_state(params, bits)
        adamw_step(params, grads, state)
        for p, g, want in zip(alone, grads, params):
            adamw_step([p], [g], adamw_state([p], bits))
            assert torch.equal(p, want)


def test_missing_gradients_and_empty_tensors():
    from isingdiff import adamw_state, adamw_step
    for bits in (32, 8):
        params, grads = make([(300,), (0,), (700,), (5,)], torch.float32, torch.float32, 3)
        state = adamw_state(params, bits)
        adamw_step(params, grads, state)
        kept, before = params[2].clone(), {k: s.clone() for k, s in state.items()}
        adamw_step(params, [grads[0], None, None, grads[3]], state)
        assert torch.equal(kept, params[2])
        assert torch.equal(state["m"][512:1280], before["m"][512:1280]) and torch.equal(state["v"][512:1280], before["v"][512:1280])
        assert not torch.equal(state["v"][:300], before["v"][:300])
        adamw_step(params, [None] * 4, state)
        assert int(state["step"]) == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_and_strided_tensors(bits):
    """Views that begin at odd elements (scalar accesses), neighbours untouched; a transposed gradient."""
    from isingdiff import adamw_state, adamw_step
    for dt in TYPES.values():
        buf = torch.arange(3000, dtype=torch.float32, device="cuda").remainder(7).to(dt) / 8
        view, keep = buf[1:2050], buf.clone()
        g = torch.randn(2050, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dt)[1:]
        want = view.clone()
        state, other = adamw_state([view], bits), adamw_state([want], bits)
        adamw_step([view], [g], state)
        adamw_step([want], [g.clone()], other)
        assert torch.equal(view, want) and all(torch.equal(state[k], other[k]) for k in state)
        assert torch.equal(buf[0], keep[0]) and torch.equal(buf[2050:], keep[2050:])
    p, gt = torch.ones(30, 50, device="cuda"), torch.randn(50, 30, device="cuda").t()
    q = p.clone()
    adamw_step([p], [gt], adamw_state([p], bits))
    adamw_step([q], [gt.contiguous()], adamw_state([q], bits))
    assert torch.equal(p, q)


def test_zero_gradients_and_zero_decay_change_nothing():
    from isingdiff import adamw_state, adamw_step
    for bits in (32, 8):
        params, _ = make([(1000,)], torch.float32, torch.float32, 3)
        want = params[0].clone()
        state = adamw_state(params, bits)
        for _ in range(3):
            adamw_step(params, [torch.zeros_like(want)], state, weight_decay=0.0)
        assert torch.equal(want, params[0]) and not state["m"].any() and not state["v"].any()


def test_entries_that_are_not_finite_keep_to_themselves():
    from isingdiff import adamw_moments, adamw_state, adamw_step
    for bits in (32, 8):
        params, grads = make([(512,)], torch.float32, torch.float32, 5)
        clean = [params[0].clone()]
        state, ref = adamw_state(params, bits), adamw_state(clean, bits)
        bad = grads[0].clone()
        bad[3], bad[100], bad[300] = float("nan"), float("inf"), -float("inf")
        hurt = torch.zeros(512, dtype=torch.bool, device="cuda")
        hurt[[3, 100, 300]] = True
        small = grads[0].clone()
        small[hurt] = 0
        for _ in range(2):
            adamw_step(params, [bad], state)
            adamw_step(clean, [small], ref)
        assert torch.equal(params[0][~hurt], clean[0][~hurt]) and bool(torch.isnan(params[0][hurt]).all())
        for a, b in zip(adamw_moments(state), adamw_moments(ref)):
            assert torch.equal(a[~hurt], b[~hurt])
            assert bits == 32 or bool(torch.isfinite(a).all())


def test_extreme_sizes_of_gradients():
    """The window of a block is 16 binades of m and 32 of v; what lies below is zero in m, and the smallest code in v."""
    from isingdiff import adamw_moments, adamw_state, adamw_step
    g = torch.zeros(256, device="cuda")
    g[0], g[1], g[2], g[3], g[4] = 1.0, 2.0 ** -12, 2.0 ** -25, 1e-30, -3e38
    for top in (g.clone(), torch.where(g < 0, torch.zeros_like(g), g)):
        p = torch.zeros(256, device="cuda")
        state = adamw_state([p], 8)
        adamw_step([p], [top], state, betas=(0.0, 0.0), weight_decay=0.0)
        m, v = adamw_moments(state)
        assert bool(torch.isfinite(p).all()) and bool(torch.isfinite(m).all()) and bool(torch.isfinite(v).all())
        if not bool((top < 0).any()):
            assert abs(float(m[0]) - 1) <= 1 / 8 and abs(float(m[1]) * 2 ** 12 - 1) <= 1 / 8 and float(m[2]) == 0
            assert abs(float(v[1]) * 2 ** 24 - 1) <= 1 / 8 and float(v[2]) > 0


def test_small_drifts_of_the_second_moment_are_followed():
    """v decays by 0.1 % a step, a hundredth of a code.  Rounding to nearest would hold it; the equidistributed dither moves it at its
    mean rate: 300 steps of decay end within 10 % of 0.999^300 on average over 4096 entries beside one entry that holds the window."""
    from isingdiff import adamw_moments, adamw_state, adamw_step
    p = torch.zeros(4096, device="cuda")
    state = adamw_state([p], 8)
    g = torch.rand(4096, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) + 0.5
    hold = torch.zeros_like(g)
    hold[::256] = 4.0
    g[::256] = 4.0
    adamw_step([p], [g], state, betas=(0.9, 0.0))
    first = adamw_moments(state)[1].clone()
    for _ in range(300):
        adamw_step([p], [hold], state, betas=(0.9, 0.999))
    rest = torch.ones(4096, dtype=torch.bool, device="cuda")
    rest[::256] = False
    ratio = float((adamw_moments(state)[1][rest] / first[rest]).mean())
    assert abs(ratio / 0.999 ** 300 - 1) < 0.1, ratio


def test_captured_and_replayed_steps_go_on():
    from isingdiff import adamw_moments, adamw_state, adamw_step
    for bits in (32, 8):
        sizes = [(5000,), (31, 17), (70000,)]
        params, grads = make(sizes, torch.float32, torch.float32, 9)
        eager = [p.clone() for p in params]
        state, other = adamw_state(params, bits), adamw_state(eager, bits)
        adamw_step(params, grads, state)
        adamw_step(eager, grads, other)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            adamw_step(params, grads, state)
            seen = adamw_moments(state)
        for k in range(4):
            for g in grads:
                g.mul_(-0.7)
            graph.replay()
            adamw_step(eager, grads, other)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(params, eager)) and all(torch.equal(state[n], other[n]) for n in state), k
            assert all(torch.equal(a, b) for a, b in zip(seen, adamw_moments(other)))
        assert int(state["step"]) == 5


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_moments_that_pass_the_cache_by(kind):
    """A large step is the same, bit for bit, as steps over its parts, which stay in the cache."""
    from isingdiff import adamw_state, adamw_step
    n, part = (23 << 20) + 100, 8 << 20
    gen = torch.Generator("cuda").manual_seed(5)
    p, g = (torch.randn(n, device="cuda", generator=gen).to(TYPES[kind]) for _ in range(2))
    parts = [t.clone() for t in p.split(part)]
    state, states = adamw_state([p]), [adamw_state([t]) for t in parts]
    for k in range(3):
        adamw_step([p], [g], state)
        for t, u, s in zip(parts, g.split(part), states):
            adamw_step([t], [u], s)
        g.mul_(-0.5)
    assert torch.equal(p, torch.cat(parts)) and all(torch.equal(state[k], torch.cat([s[k] for s in states])) for k in "mv")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [256 * 4096, 256 * 4096 + 1])
def test_both_ways_to_count_a_step(n, bits):
    """256 workgroups count the step among themselves, more have it counted before: from equal states, equal steps."""
    from isingdiff import adamw_state, adamw_step
    gen = torch.Generator("cuda").manual_seed(6)
    p, g = (torch.randn(n, device="cuda", generator=gen) for _ in range(2))
    q, idle = p.clone(), torch.zeros(256 * 4096, device="cuda")      # the second tensor makes it a large step
    s, r = adamw_state([p], bits), adamw_state([q, idle], bits)
    for k in range(5):
        adamw_step([p], [g], s, lr=0.1)
        adamw_step([q, idle], [g, idle.clone()], r, lr=0.1)
        assert int(s["step"]) == int(r["step"]) == k + 1
        g.mul_(-0.8)
    m = s["m"].numel()
    assert torch.equal(p, q) and torch.equal(s["m"], r["m"][:m]) and torch.equal(s["v"], r["v"][:m])


def test_gradients_that_are_views_and_parameters_without_versions():
    from isingdiff import adamw_state, adamw_step
    with torch.inference_mode():                      # (such tensors keep no version)
        p = [torch.linspace(-1, 1, 12, device="cuda").reshape(3, 4), torch.ones(5, device="cuda")]
    q = [t.clone() for t in p]
    g = torch.randn(4, 3, device="cuda")
    s, r = adamw_state(p), adamw_state(q)
    adamw_step(p, [g.t(), torch._neg_view(q[1])], s)
    adamw_step(q, [g.t().contiguous(), -q[1]], r)
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and all(torch.equal(s[k], r[k]) for k in s)
    w, idle = torch.nn.Parameter(torch.ones(3, device="cuda")), torch.nn.Parameter(torch.ones(3, device="cuda"))
    adamw_step([w, idle], [torch.ones(3, device="cuda"), None], adamw_state([w, idle]))
    assert w._version == 1 and idle._version == 0     # only what changed


def test_optimizer_class():
    from isingdiff import AdamW
    w = torch.nn.Parameter(torch.linspace(-1, 1, 600, device="cuda"))
    b = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    opt = AdamW([w, b], lr=1e-2, weight_decay=[0.1, 0.0], moment_bits=8)
    loss = (w * w).sum() + b.sum()
    keep = (w * w).sum()          # its graph saved w
    loss.backward()
    opt.step()
    with pytest.raises(RuntimeError):
        keep.backward()           # w has changed since
    saved, at = opt.state_dict(), [w.detach().clone(), b.detach().clone()]
    w.grad = w.detach().clone()
    opt.step()
    after = [w.detach().clone(), b.detach().clone()]
    with torch.no_grad():
        w.copy_(at[0]), b.copy_(at[1])
    opt.load_state_dict(saved)
    opt.step()
    assert torch.equal(w, after[0]) and torch.equal(b, after[1])
    opt.zero_grad()
    assert w.grad is None and b.grad is None
    with pytest.raises(ValueError):
        opt.load_state_dict({k: saved[k] for k in ("step", "m", "v")})

"""Group norm with an activation, channels last, forward and backward, against the formula in 64 bits.

Tolerances, with u = eps / 2 of the tensor's type and e = 2^-24:
 * y: one rounding of the output, u |y|, and float32 arithmetic before it.  An error of the mean or of a value is relative to the
   largest |x + shift| of the group (K of them in units of the group's deviation); no chain of additions in these shapes is longer
   than 64 roundings, and the activation's slope is at most 1.1: 64 e (K + 1) (|gamma| + 1) covers it.
 * dx: the same, relative to rstd * max |dz gamma| of the sample, and xhat up to K multiplies the second mean.
 * dgamma, dbeta, dshift: float32 sums; a chain has at most 512 additions: 512 e times the sum of the terms' sizes, where a term's
   own error (64 e (K + 1)) is included by the factor (K + 1) on the smaller count.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def exact(x, gamma, beta, shift, groups, eps, act, dy=None):
    """Everything in float64 on the CPU, gradients by autograd of the formula."""
    x = x.detach().cpu().double().requires_grad_()
    b, c = x.shape[0], x.shape[-1]
    ones = lambda t, v: (torch.full((c,), v, dtype=torch.float64) if t is None else t.detach().cpu().double()).requires_grad_()  # noqa: E731
    gamma, beta = ones(gamma, 1.0), ones(beta, 0.0)
    shift = torch.zeros(b, c, dtype=torch.float64) if shift is None else shift.detach().cpu().double()
    shift = shift.expand(b, c).clone().requires_grad_()
    u = (x.reshape(b, -1, c) + shift[:, None]).reshape(b, -1, groups, c // groups)
    mean = u.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((u - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xhat = (u - mean) * rstd
    z = xhat * gamma.view(groups, -1) + beta.view(groups, -1)
    y = (z * torch.sigmoid(z) if act == "swish" else z).reshape(x.shape)
    out = {"y": y, "mean": mean.view(b, groups), "rstd": rstd.view(b, groups)}
    size = torch.maximum(u.abs(), x.reshape(u.shape).abs())
    out["k"] = float((size.amax((1, 3), keepdim=True) * rstd).detach().max())
    if dy is not None:
        dy = dy.detach().cpu().double()
        out["dx"], out["dgamma"], out["dbeta"], out["dshift"] = torch.autograd.grad(y, (x, gamma, beta, shift), dy)
        zz = z.detach().reshape(b, -1, c)
        s = torch.sigmoid(zz)
        dz = dy.reshape(zz.shape) * (s * (1 + zz * (1 - s)) if act == "swish" else 1)
        flat = xhat.detach().reshape(b, -1, c)
        out["terms"] = {"dbeta": dz.abs().sum((0, 1)), "dgamma": (dz * flat).abs().sum((0, 1))}
        r = rstd.detach().expand(u.shape).reshape(b, -1, c)
        out["scale"] = float((r * (dz * gamma.detach()).abs()).max())
        # what dshift is the difference of: rstd * (sum |dz gamma| + pixels |A| + |B| sum |xhat|)
        dg = (dz * gamma.detach()).view(b, -1, groups, c // groups)
        a, bb = dg.mean((1, 3), keepdim=True).abs(), (dg * xhat.detach()).mean((1, 3), keepdim=True).abs()
        terms = rstd.detach() * (dg.abs() + a + bb * xhat.detach().abs())
        out["terms"]["dshift"] = terms.sum(1).reshape(b, c)
    return out


def check(name, got, want, tol):
    got, want = got.detach().cpu().double(), want.detach().double()
    assert got.shape == want.shape, name
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), f"{name}: over its tolerance by {float(off.max()):.3g}, largest value {float(want.abs().max()):.3g}"


def inputs(shape, dtype, seed, groups, shift="rows", affine=True, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    b, c = shape[0], shape[-1]
    x = (torch.randn(shape, generator=g) * (0.5 + torch.rand(c, generator=g)) + offset * torch.randn(c, generator=g)).to(dtype).cuda()
    gamma = (1 + 0.2 * torch.randn(c, generator=g)).cuda() if affine else None
    beta = (0.2 * torch.randn(c, generator=g)).cuda() if affine else None
    sh = {"rows": (b, c), "one": (1, c), "flat": (c,)}.get(shift)
    sh = None if sh is None else (0.5 * torch.randn(sh, generator=g)).cuda()
    dy = torch.randn(shape, generator=g).to(dtype).cuda()
    return x, gamma, beta, sh, dy


def verify(x, gamma, beta, shift, dy, groups, act, eps=1e-3):
    from isingdiff import group_norm_backward, group_norm_forward
    y, mean, rstd = group_norm_forward(x, gamma, beta, groups, shift=shift, eps=eps, activation=act)
    dx, dgamma, dbeta, dshift = group_norm_backward(dy, x, mean, rstd, gamma, beta, groups, shift=shift, activation=act)
    w = exact(x, gamma, beta, shift, groups, eps, act, dy)
    k, u = w["k"], half_step(x.dtype)
    top = 1 + (1 if gamma is None else float(gamma.abs().max()))
    assert y.dtype == x.dtype and dx.dtype == x.dtype and y.is_contiguous() and dx.is_contiguous()
    check("mean", mean, w["mean"], 64 * E * k / w["rstd"])
    # a relative error of the variance is at most twice that of the centred values (K + 1 of e), rstd has half of it
    check("rstd", rstd, w["rstd"], 64 * E * (k + 1) * w["rstd"].abs())
    check("y", y, w["y"], u * w["y"].abs() + 64 * E * (k + 1) * top + (6e-8 if x.dtype == torch.float16 else 0))
    check("dx", dx, w["dx"], u * w["dx"].abs() + 64 * E * (k + 1) ** 2 * w["scale"] * top + (6e-8 if x.dtype == torch.float16 else 0))
    many = 512 * E * (1 + k / 8)
    if gamma is not None:
        check("dgamma", dgamma, w["dgamma"], many * (w["terms"]["dgamma"] + w["terms"]["dbeta"]))
        check("dbeta", dbeta, w["dbeta"], many * (w["terms"]["dbeta"] + w["terms"]["dgamma"]))
    else:
        assert dgamma is None and dbeta is None
    if shift is not None:
        ds, terms = w["dshift"], w["terms"]["dshift"]
        assert dshift.shape == shift.shape
        if shift.dim() == 1 or shift.shape[0] != x.shape[0]:
            ds, terms = ds.sum(0), terms.sum(0)
        check("dshift", dshift, ds.reshape(dshift.shape), many * top * terms.reshape(dshift.shape))
    else:
        assert dshift is None
    return y, dx


SHAPES = [  # shape, groups: the bit-flip UNet's maps, odd ones, one pixel, one channel a group, groups wider than a workgroup
    ((1, 28, 28, 32), 8), ((3, 14, 14, 64), 8), ((5, 7, 7, 128), 8), ((2, 14, 14, 192), 8), ((2, 28, 28, 96), 8),
    ((1, 1, 1, 8), 8), ((4, 1, 1, 32), 8), ((7, 33), 1), ((2, 1, 3, 5), 1), ((3, 5, 3, 30), 3), ((2, 9, 11, 20), 4), ((2, 6, 5, 7), 7),
    ((1, 64, 64, 64), 16), ((2, 127, 125, 16), 4), ((1, 3, 2, 2056), 1), ((2, 5, 1, 1031), 1), ((1, 2, 2, 4104), 2), ((300, 2, 3, 24), 2),
    ((2, 3, 4, 5, 16), 2), ((1, 130, 3, 512), 32),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_the_formula(shape, groups, dtype):
    n = sum(shape) + groups
    x, gamma, beta, shift, dy = inputs(shape, TYPES[dtype], n, groups, shift=["rows", "none", "one", "flat"][n % 4], affine=n % 5 > 0)
    verify(x, gamma, beta, shift, dy, groups, "swish" if n % 3 else "none")


# batches that the forms for many samples take: several samples to a block, several turns of a block, a last pack that is not full,
# groups that straddle vectors (5, 6, 12, 1 channels), one pixel, rows that are not full; the last two with backward blocks that
# take more than 64 KB of a compute unit's shared memory
MANY = [((70, 6, 6, 40), 8), ((1501, 3, 3, 16), 4), ((90, 14, 14, 192), 8), ((65, 28, 28, 96), 8), ((2051, 1, 1, 64), 8), ((777, 7, 7, 48), 8),
        ((130, 5, 13, 64), 64), ((300, 9, 9, 128), 32), ((513, 2, 1, 8), 1), ((70, 25, 41, 32), 8),
        ((11, 447, 912), 19), ((98, 11, 25, 160), 16)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,groups", MANY)
def test_many_samples(shape, groups, dtype):
    n = sum(shape) + groups
    x, gamma, beta, shift, dy = inputs(shape, TYPES[dtype], n, groups, shift=["rows", "none", "one", "none"][n % 4])
    verify(x, gamma, beta, shift, dy, groups, "swish" if n % 3 else "none")


# few samples of many channels: tiles of a part of a pixel (the last one narrower, or one group wider than a tile), chunks whose last
# rows are not full
WIDE = [((2, 40, 41, 256), 32), ((1, 33, 31, 150), 15), ((3, 700, 520), 5), ((1, 64, 65, 512), 32), ((2, 50, 43, 264), 11), ((257, 5, 7, 300), 12)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,groups", WIDE)
def test_few_samples_of_many_channels(shape, groups, dtype):
    n = sum(shape) + groups
    x, gamma, beta, shift, dy = inputs(shape, TYPES[dtype], n, groups, shift=["rows", "none", "one", "flat"][n % 4])
    verify(x, gamma, beta, shift, dy, groups, "swish" if n % 3 else "none")


@pytest.mark.parametrize("act", ["swish", "none"])
@pytest.mark.parametrize("shift", ["rows", "one", "flat", "none"])
def test_activation_and_shift(act, shift):
    x, gamma, beta, sh, dy = inputs((5, 12, 10, 48), torch.float32, 3, 8, shift=shift)
    verify(x, gamma, beta, sh, dy, 8, act)


def test_values_far_from_zero():
    """Mean a thousand deviations from zero: squares summed around zero would lose the variance altogether."""
    x, gamma, beta, _, dy = inputs((2, 40, 40, 16), torch.float32, 11, 4)
    x = x + 1000.0
    verify(x, gamma, beta, None, dy, 4, "swish")


def test_a_variance_beyond_float32():
    """Deviations of at least 2^61 (2^62 times half a unit): the squares of a group's 20 * 20 * 8 values add up to more than 3 200 * 2^122 =
    2^133, and float32 ends below 2^128.  The sum is infinite, so rstd is zero and y = act(beta); the mean is right."""
    from isingdiff import group_norm_forward
    x, gamma, beta, _, dy = inputs((3, 20, 20, 64), torch.bfloat16, 41, 8, shift="none")
    x = (x.float() * 2.0 ** 62 + 2.0 ** 66).to(torch.bfloat16)
    y, mean, rstd = group_norm_forward(x, gamma, beta, 8, eps=0.0)
    w = exact(x, gamma, beta, None, 8, 0.0, "swish")
    check("mean", mean, w["mean"], 64 * E * w["k"] / w["rstd"])
    assert not rstd.any()
    want = (beta.double() * torch.sigmoid(beta.double())).cpu().expand(y.shape)
    check("y", y, want, half_step(torch.bfloat16) * want.abs() + 16 * E)


@pytest.mark.parametrize("scale,offset", [(1.0, 100.0), (2.0 ** 40, 0.0), (2.0 ** 56, 2.0 ** 64)])
def test_bfloat16_far_from_zero_and_large(scale, offset):
    """Means of many deviations, and values whose squares leave float32 while those of the deviations do not: the short way over sums
    of squares has to give up by itself."""
    x, gamma, beta, _, dy = inputs((3, 20, 20, 64), torch.bfloat16, 41, 8, shift="none")
    verify((x.float() * scale + offset).to(torch.bfloat16), gamma, beta, None, dy, 8, "swish", eps=0.0)
    x, gamma, beta, _, dy = inputs((3, 20, 20, 32), torch.bfloat16, 42, 8, shift="none")
    verify((x.float() * scale + offset).to(torch.bfloat16), gamma, beta, None, dy, 8, "none", eps=0.0)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_inputs_are_read_in_place(dtype):
    """Channel slices, cropped maps of one row, every second sample, odd offsets (scalar loads), a transposed map (a copy)."""
    full, gamma, beta, sh, dyf = inputs((6, 9, 8, 80), TYPES[dtype], 5, 4, shift="none")
    for cut in (lambda t: t[..., 16:48], lambda t: t[::2, :, :, 3:35], lambda t: t[:, 2:3, 1:7, 8:40], lambda t: t[:, :, 2:7, 32:64],
                lambda t: t[..., 16:48].transpose(1, 2), lambda t: t[1:2, 4:5, 5:6, 1:33], lambda t: t[:, ::3, ::4, :32]):
        verify(cut(full), gamma[:32].contiguous(), beta[:32].contiguous(), None, cut(dyf), 4, "swish")
    # one sample's memory for all, one pixel's gradient for all
    x = full[:1, ..., :32].expand(4, 9, 8, 32)
    verify(x, gamma[:32].contiguous(), beta[:32].contiguous(), None, dyf[:4, :1, :1, :32].expand(4, 9, 8, 32), 4, "none")


def test_strided_vectors_of_parameters():
    from isingdiff import group_norm_forward
    x, gamma, beta, sh, _ = inputs((3, 5, 5, 32), torch.float32, 6, 8)
    wide = torch.stack([gamma, beta], 1)
    two = torch.stack([sh, sh], 2)
    a = group_norm_forward(x, gamma, beta, 8, shift=sh)[0]
    assert torch.equal(a, group_norm_forward(x, wide[:, 0], wide[:, 1], 8, shift=two[..., 1])[0])


def test_subnormal_halves():
    """Values below 2^-14, which fp16 holds with fewer bits, have a mean and a deviation like others."""
    import isingdiff as I
    x, gamma, beta, _, _ = inputs((130, 5, 8, 32), torch.float16, 22, 4)
    x = (x.float() * 2.0 ** -18).half()
    _, mean, rstd = I.group_norm_forward(x, gamma, beta, 4, eps=1e-18, activation="none")
    g = x.cpu().double().reshape(130, 40, 4, 8)
    m, v = g.mean((1, 3)), g.var((1, 3), correction=0)
    check("mean", mean, m, 64 * E * g.abs().mean((1, 3)))
    check("rstd", rstd, (v + 1e-18).rsqrt(), 64 * E * (v + 1e-18).rsqrt() * (1 + g.pow(2).mean((1, 3)) / v))


@pytest.mark.parametrize("samples", [4194304, 530000])
def test_more_samples_than_one_grid(samples):
    """Many copies of a few samples give many copies of their results."""
    import isingdiff as I
    pixels = 520 if samples == 530000 else 2
    x, gamma, beta, _, dy = inputs((1000, pixels, 8), torch.float16, 23, 2)
    n = samples // 1000
    many = lambda t: t.repeat(n, 1, 1)  # noqa: E731
    y, mean, rstd = I.group_norm_forward(many(x), gamma, beta, 2)
    for t in (y, mean, rstd):
        t = t.view(n, -1)
        assert bool((t == t[:1]).all())
    dx = I.group_norm_backward(many(dy), many(x), mean, rstd, gamma, beta, 2)[0].view(n, -1)
    assert bool((dx == dx[:1]).all()) and bool(torch.isfinite(dx).all())
    w = I.group_norm_forward(x, gamma, beta, 2)[0]
    assert float((y[:1000].float() - w.float()).abs().max()) <= 2.0 ** -10 * float(w.float().abs().max())


def test_views_that_negate():
    import isingdiff as I
    x, gamma, beta, shift, dy = inputs((2, 6, 5, 16), torch.float32, 21, 4, shift="rows")
    want = I.group_norm_forward(-x, gamma, beta, 4, shift=-shift)
    got = I.group_norm_forward(torch._neg_view(x), gamma, beta, 4, shift=torch._neg_view(shift))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = I.group_norm_backward(-dy, -x, *want[1:], -gamma, beta, 4, shift=-shift)
    got = I.group_norm_backward(torch._neg_view(dy), torch._neg_view(x), *got[1:], torch._neg_view(gamma), beta, 4, shift=torch._neg_view(shift))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_beyond_32_bits():
    """Two samples 2^31 + 64 elements apart in x and dy."""
    big = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device="cuda")
    x, gamma, beta, _, dy = inputs((2, 6, 5, 32), torch.bfloat16, 8, 8, shift="none")
    far = big.as_strided((2, 6, 5, 32), ((1 << 31) + 64, 160, 32, 1))
    far.copy_(x)
    verify(far, gamma, beta, None, dy, 8, "swish")


def test_more_than_2_31_values():
    from isingdiff import group_norm_backward, group_norm_forward
    b, hw, c = 2100, 32 * 32, 1024
    x = torch.zeros((b, hw, c), dtype=torch.bfloat16, device="cuda")
    part, gamma, beta, sh, dy = inputs((2, hw, c), torch.bfloat16, 9, 8)
    x[-1], x[0] = part[1], part[0]
    shift = torch.zeros((b, c), device="cuda")
    shift[-1], shift[0] = sh[1], sh[0]
    y, mean, rstd = group_norm_forward(x, gamma, beta, 8, shift=shift)
    w = exact(part, gamma, beta, sh, 8, 1e-3, "swish")
    tol = half_step(torch.bfloat16) * w["y"].abs() + 64 * E * (w["k"] + 1) * (1 + float(gamma.abs().max()))
    check("y", y[[0, -1]], w["y"], tol)
    dx, dgamma, _, dshift = group_norm_backward(y, x, mean, rstd, gamma, beta, 8, shift=shift)
    one, m1, r1 = group_norm_forward(x[-1:], gamma, beta, 8, shift=shift[-1:])
    ref = group_norm_backward(y[-1:], x[-1:], m1, r1, gamma, beta, 8, shift=shift[-1:])
    # the same sample alone: other chunks, so other orders of the same sums
    assert (dx[-1:].float() - ref[0].float()).abs().max() <= 2 ** -7 * ref[0].float().abs().max()
    assert bool(torch.isfinite(dgamma).all()) and (dshift[-1:] - ref[3]).abs().max() <= 1e-3 * ref[3].abs().max()


def test_nan_and_infinity_stay_in_their_group():
    from isingdiff import group_norm_backward, group_norm_forward
    x, gamma, beta, sh, dy = inputs((4, 6, 6, 32), torch.float32, 12, 8)
    y0, m0, r0 = group_norm_forward(x, gamma, beta, 8, shift=sh)
    bad = x.clone()
    bad[1, 2, 3, 5], bad[2, 0, 0, 31] = float("nan"), float("inf")
    y, m, r = group_norm_forward(bad, gamma, beta, 8, shift=sh)
    ok = torch.ones(4, 8, dtype=torch.bool, device="cuda")
    ok[1, 1] = ok[2, 7] = False
    sel = ok[:, None, None, :].expand(4, 6, 6, 8).repeat_interleave(4, 3)
    assert torch.equal(y[sel], y0[sel]) and bool(torch.isnan(y[~sel]).all())
    assert torch.equal(m[ok], m0[ok]) and torch.equal(r[ok], r0[ok])
    dx = group_norm_backward(dy, bad, m, r, gamma, beta, 8, shift=sh)[0]
    dx0 = group_norm_backward(dy, x, m0, r0, gamma, beta, 8, shift=sh)[0]
    assert torch.equal(dx[sel], dx0[sel]) and bool(torch.isnan(dx[~sel]).all())


def test_constant_groups_and_large_activations():
    """Variance zero: xhat is zero, y = act(beta).  Arguments of the activation far on both sides: no NaN from exp, whose relative error
    grows with its argument (one rounding of z log2 e), and which is infinite below z = -88.7, where |y| < 3e-37."""
    from isingdiff import group_norm_forward
    x = torch.full((2, 5, 5, 16), 7.0, device="cuda")
    beta = torch.tensor([-200.0, -90.0, 0.0, 300.0] * 4, device="cuda")
    y, mean, rstd = group_norm_forward(x, None, beta, 4)
    want = (beta.double() * torch.sigmoid(beta.double())).cpu()
    check("y", y, want.expand(2, 5, 5, 16), ((8 + 2 * beta.cpu().abs()) * E * want.abs() + 3e-37).expand(2, 5, 5, 16))
    assert torch.equal(mean, torch.full_like(mean, 7.0))


def test_empty_batches_and_maps():
    from isingdiff import group_norm, group_norm_backward, group_norm_forward
    for shape in ((0, 4, 4, 16), (3, 0, 4, 16)):
        x, gamma, beta, _, dy = inputs(shape, torch.float32, 1, 4, shift="none")
        y, mean, rstd = group_norm_forward(x, gamma, beta, 4)
        assert y.shape == shape and mean.shape == rstd.shape == (shape[0], 4)
        dx, dgamma, dbeta, _ = group_norm_backward(dy, x, mean, rstd, gamma, beta, 4)
        assert dx.shape == shape and not dgamma.any() and not dbeta.any()
    assert group_norm(torch.empty(0, 2, 2, 8, device="cuda")).shape == (0, 2, 2, 8)


def test_gradients_against_differences():
    """(L(a + h d) - L(a - h d)) / 2h of the kernel's own forward pass, L = sum w y, for a random direction d of each input.  Tolerance:
    the truncation is c h^2, a third of what halving h changes, and the rounding of y is 16 e |w y| summed, over h."""
    from isingdiff import group_norm
    x, gamma, beta, sh, w = inputs((3, 6, 7, 16), torch.float32, 21, 4)
    leaves = [t.clone().requires_grad_() for t in (x, gamma, beta, sh)]
    f = lambda a, b, c, d: (group_norm(a, b, c, 4, shift=d).double() * w.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(f(*leaves), leaves)
    gen = torch.Generator().manual_seed(4)
    noise = 16 * E * float((group_norm(x, gamma, beta, 4, shift=sh).double() * w.double()).abs().sum())
    for i, g in enumerate(grads):
        d = torch.randn(g.shape, generator=gen).cuda()
        d /= d.norm()

        def diff(h):
            at = lambda s: f(*[t + s * h * d if k == i else t for k, t in enumerate((x, gamma, beta, sh))])  # noqa: E731
            with torch.no_grad():
                return float(at(1) - at(-1)) / (2 * h)
        h = 0.05
        a, b = diff(h), diff(h / 2)
        want = float((g.double() * d.double()).sum())
        assert abs(b - want) <= abs(a - b) + 2 * noise / h, (i, a, b, want)


def test_autograd_of_all_forms():
    """Leaves of other types, a shared shift row, an expanded gradient (y.sum()), no affine terms."""
    from isingdiff import group_norm
    x, gamma, beta, sh, _ = inputs((4, 5, 6, 32), torch.bfloat16, 31, 8, shift="one")
    leaves = [x.clone().requires_grad_(), gamma.bfloat16().requires_grad_(), beta.bfloat16().requires_grad_(),
              sh.bfloat16().requires_grad_()]
    y = group_norm(leaves[0], leaves[1], leaves[2], shift=leaves[3])
    y.sum().backward()
    for t in leaves:
        assert t.grad.dtype == t.dtype and t.grad.shape == t.shape and bool(torch.isfinite(t.grad).all())
    z = x.clone().requires_grad_()
    group_norm(z, activation="none").sum().backward()
    # sum of normalised values is zero whatever x is: the gradient is nothing but rounding
    assert float(z.grad.abs().max()) < 1e-4
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(group_norm(z).float().pow(2).sum(), z, create_graph=True)
        g.sum().backward()


def test_equal_inputs_give_equal_bits():
    from isingdiff import group_norm_backward, group_norm_forward
    x, gamma, beta, sh, dy = inputs((40, 14, 14, 64), torch.bfloat16, 17, 8)
    outs = []
    for _ in range(3):
        y, m, r = group_norm_forward(x, gamma, beta, 8, shift=sh)
        outs.append((y, m, r) + group_norm_backward(dy, x, m, r, gamma, beta, 8, shift=sh))
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], o))


def test_other_stream():
    from isingdiff import group_norm_backward, group_norm_forward
    x, gamma, beta, sh, dy = inputs((64, 28, 28, 32), torch.float32, 18, 8)
    want = group_norm_forward(x, gamma, beta, 8, shift=sh)
    want += group_norm_backward(dy, x, want[1], want[2], gamma, beta, 8, shift=sh)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in side:   # two calls at once
            with torch.cuda.stream(s):
                o = group_norm_forward(x, gamma, beta, 8, shift=sh)
                got.append(o + group_norm_backward(dy, x, o[1], o[2], gamma, beta, 8, shift=sh))
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(want, o))


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed with other contents, with eager calls and synchronizations in between; a second
    graph replayed alternately."""
    from isingdiff import group_norm_backward, group_norm_forward

    def both(x, gamma, beta, sh, dy):
        o = group_norm_forward(x, gamma, beta, 8, shift=sh)
        return o + group_norm_backward(dy, x, o[1], o[2], gamma, beta, 8, shift=sh)
    graphs = []
    for shape, kind, seed in (((33, 14, 14, 64), "one", 1), ((2, 40, 40, 64), "rows", 2)):
        ins = inputs(shape, torch.bfloat16, seed, 8, shift=kind)
        both(*ins)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both(*ins)
        graphs.append((g, ins, out, shape, kind))
    for k in range(4):
        for g, ins, out, shape, kind in graphs:
            for a, b in zip(ins, inputs(shape, torch.bfloat16, 100 + k, 8, shift=kind)):
                a.copy_(b)
            g.replay()
            want = both(*ins)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_a_backward_pass_is_captured_once_eager_graphs_are_gone():
    from isingdiff import group_norm, group_norm_backward, group_norm_forward
    x, gamma, beta, shift, dy = inputs((9, 6, 5, 32), torch.float32, 31, 8)
    leaves = [t.requires_grad_() for t in (x, gamma, beta, shift)]
    eager = group_norm(x, gamma, beta, 8, shift=shift)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            group_norm(x, gamma, beta, 8, shift=shift)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = group_norm(x, gamma, beta, 8, shift=shift)
        y.backward(dy)
    for k in range(3):
        with torch.no_grad():
            for t, new in zip(leaves + [dy], inputs((9, 6, 5, 32), torch.float32, 40 + k, 8)):
                t.copy_(new)
        graph.replay()
        with torch.no_grad():
            want, mean, rstd = group_norm_forward(x, gamma, beta, 8, shift=shift)
            grads = group_norm_backward(dy, x, mean, rstd, gamma, beta, 8, shift=shift)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(t.grad, w) for t, w in zip(leaves, grads)), k


def test_half_overflow_is_infinite():
    from isingdiff import group_norm_forward
    x, _, _, _, _ = inputs((1, 4, 4, 8), torch.float16, 2, 1)
    y, _, _ = group_norm_forward(x, torch.full((8,), 1e6, device="cuda"), None, 1, activation="none")
    assert bool(torch.isinf(y).any()) and not bool(torch.isnan(y).any()) and math.isinf(float(y.float().abs().max()))

"""Group norm of groups that are constant, or constant but for one value, beside ordinary ones: there |mean| is large in units of the
deviation sqrt(var + eps), whatever the type resolves.  Both forms (one launch; chunks, for a view that is not aligned), all types.

Tolerances, per sample and group, with u = eps / 2 of the tensor's type, e = 2^-24, K = max |x + shift| or |x| of the group times its rstd:
 * Constant groups.  The values and the values with their shift have at most 11 significant bits and a group at most 2^13 values, so every
   sum of them is a whole multiple of their last bit below 2^24 of it: exact, and so is the mean.  u - mean is zero then and z = beta: y
   has its rounding and the activation's 16 float32 roundings, relative to |beta|; dgamma is a sum of zeros; dx = rstd (dz gamma - A) has
   its rounding and a sum of at most 64 roundings in line.  No K anywhere.
 * Others: the mean is off by at most d = 16 e K in units of the deviation (sum, division, the difference), the variance by d^2 of it
   besides its own 64 e, so xhat by d + |xhat| (64 e + d^2); z by gamma times that and dz by at most |dy| gamma / 2 times that.
"""
import ctypes as C

import pytest
import torch

from isingdiff import _lib, group_norm_backward, group_norm_forward

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LARGE = {"fp32": 60000.0, "bf16": 99840.0, "fp16": 60000.0}     # 11, 8 and 11 significant bits; 1 000 has 7


def case(shape, groups, dtype, seed, shifted, level):
    """Groups 0, 4, ..: ordinary; 1, 5, ..: constant; 2, 6, ..: constant, another constant in every other sample; 3, 7, ..: constant but for
    one value, one step of the type away."""
    gen = torch.Generator().manual_seed(seed)
    b, c = shape[0], shape[-1]
    gc = c // groups
    x = torch.randn(shape, generator=gen)
    v = x.view(b, -1, groups, gc)
    kind = torch.arange(groups) % 4
    v[:, :, kind == 1] = level
    v[:, :, kind == 2] = level
    v[1::2][:, :, kind == 2] = 1000.0
    v[:, :, kind == 3] = level
    v[:, -1, kind == 3, 0] = level * (1 + torch.finfo(TYPES[dtype]).eps)
    shift = None
    if shifted:     # constant groups stay constant
        shift = 0.5 * torch.randn(b, groups, gc, generator=gen)
        shift[:, kind > 0] = 512.0
        shift = shift.view(b, c).cuda()
    gamma, beta = 1 + 0.2 * torch.randn(c, generator=gen), 0.2 * torch.randn(c, generator=gen)
    return x.to(TYPES[dtype]).cuda(), gamma.cuda(), beta.cuda(), shift, torch.randn(shape, generator=gen).to(TYPES[dtype]).cuda()


def unaligned(t):
    """The same values with a pitch and an offset that allow no vectors."""
    wide = torch.zeros(t.shape[:-1] + (t.shape[-1] + 3,), dtype=t.dtype, device=t.device)
    wide[..., 1:1 + t.shape[-1]] = t
    return wide[..., 1:1 + t.shape[-1]]


def in_one_launch(x, groups):
    """Whether the aligned forward call takes the one-launch form: it then needs no workspace."""
    b, c = x.shape[0], x.shape[-1]
    n = x.numel() // (b * c)
    d = _lib.GroupNormDesc(dtype={torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype], activation=1, batch=b, pixels=n, channels=c,
                           groups=groups, x_sample=n * c, x_pixel=c, shift_sample=c, eps=1e-3, aligned=1)
    size = C.c_size_t()
    assert _lib.load().idm_group_norm_workspace(C.byref(d), 0, C.byref(size)) == 0
    return size.value == 0


def over(name, got, want, tol):
    off = (got.detach().cpu().double() - want).abs() - tol
    bad = ~(off <= 0)
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} over their tolerance, the worst by {float(off.max()):.3g}"


class Truth:
    """The formulas in 64 bits, grouped (sample, pixel, group, channel of the group), and how far xhat may be off."""

    def __init__(self, x, gamma, beta, shift, groups, act, eps):
        b, c = x.shape[0], x.shape[-1]
        self.groups, self.gc, self.u = groups, c // groups, torch.finfo(x.dtype).eps / 2
        self.tiny = 6e-8 if x.dtype == torch.float16 else 0.0        # half the spacing of fp16 below its normal numbers
        xs, self.g, self.bt = self.grouped(x), self.row(gamma), self.row(beta)
        us = xs if shift is None else xs + shift.cpu().double().view(b, 1, groups, self.gc)
        self.constant = (us == us[:, :1, :, :1]).all(3, keepdim=True).all(1, keepdim=True)
        assert bool(self.constant[:, :, torch.arange(groups) % 4 == 1].all())
        self.mean = torch.where(self.constant, us[:, :1, :, :1], us.mean((1, 3), keepdim=True))
        self.rstd = 1 / torch.sqrt((us - self.mean).square().mean((1, 3), keepdim=True) + eps)
        self.xhat = (us - self.mean) * self.rstd
        self.z = self.xhat * self.g + self.bt
        self.s = torch.sigmoid(self.z) if act == "swish" else torch.ones_like(self.z)
        self.slope = self.s * (1 + self.z * (1 - self.s)) if act == "swish" else self.s
        self.top = us.abs().amax((1, 3), keepdim=True)
        k = torch.maximum(us.abs(), xs.abs()).amax((1, 3), keepdim=True) * self.rstd
        self.d = torch.where(self.constant, 0.0, 16 * E * k)
        self.off = self.d + self.xhat.abs() * (64 * E + self.d * self.d)

    def grouped(self, t):
        return t.detach().cpu().double().reshape(t.shape[0], -1, self.groups, self.gc)

    def row(self, t):
        return t.detach().cpu().double().view(self.groups, self.gc)

    def forward(self, y, m, r):
        y, m, r = self.grouped(y), m.cpu().double().view(self.mean.shape), r.cpu().double().view(self.mean.shape)
        over("mean", m, self.mean, torch.where(self.constant, 0.0, 16 * E * self.top))
        over("rstd", r, self.rstd, (64 * E + self.d * self.d) * self.rstd)
        want = self.z * self.s
        over("y", y, want, self.u * want.abs() + 1.1 * (self.off * self.g.abs() + 16 * E * (self.z.abs() + self.bt.abs())) + self.tiny)

    def backward(self, dy, gx, gg, gb, gs):
        each, off, xhat, rstd = (1, 3), self.off, self.xhat, self.rstd
        dy = self.grouped(dy)
        dz = dy * self.slope
        dg = dz * self.g
        first, second = dg.mean(each, keepdim=True), (dg * xhat).mean(each, keepdim=True)
        dx = rstd * (dg - first - second * xhat)
        off_dz = dy.abs() * (16 * E + 0.5 * self.g.abs() * off)
        off_dg = off_dz * self.g.abs()
        off_second = dg.abs().mean(each, keepdim=True) * off.amax(each, keepdim=True) + off_dg.mean(each, keepdim=True) * xhat.abs().amax(each, keepdim=True)
        off_second = torch.where(self.constant, 0.0, off_second)
        off_dx = rstd * (64 * E * (1 + xhat.abs()) * dg.abs().amax(each, keepdim=True) + off_dg + off_dg.mean(each, keepdim=True) + off_second * xhat.abs() +
                         second.abs() * off) + self.d * self.d * dx.abs()
        over("dx", self.grouped(gx), dx, self.u * dx.abs() + off_dx + self.tiny)
        assert not bool(self.row(gg)[torch.arange(self.groups) % 4 == 1].any()), "dgamma of constant groups"
        many = 512 * E
        over("dgamma", self.row(gg), (dz * xhat).sum((0, 1)), (many * (dz * xhat).abs() + dz.abs() * off + off_dz * xhat.abs()).sum((0, 1)))
        over("dbeta", self.row(gb), dz.sum((0, 1)), (many * dz.abs() + off_dz).sum((0, 1)))
        if gs is not None:
            terms = rstd * (dg.abs() + first.abs() + second.abs() * xhat.abs())
            over("dshift", gs.cpu().double().view(-1, self.groups, self.gc), dx.sum(1), (many * terms + off_dx).sum(1))


# groups of whole vectors, of half vectors, of single values (5, 1 channels); few and many samples, several to a block; groups have at most 2^13
# values
SHAPES = [((3, 20, 20, 64), 4), ((2, 12, 11, 48), 4), ((5, 9, 7, 40), 8), ((3, 14, 13, 32), 32), ((70, 6, 6, 96), 8), ((1030, 3, 3, 64), 8), ((6, 28, 28, 32), 4)]


def cases(shape, groups, dtype, form):
    for i, (level, eps) in enumerate(((1000.0, 1e-3), (LARGE[dtype], 1e-3), (1000.0, 1e-5), (LARGE[dtype], 1e-5))):
        x, gamma, beta, shift, dy = case(shape, groups, dtype, 7 + i, i % 2 == 1, level)
        if form == "chunks":
            x, dy = unaligned(x), unaligned(dy)
        else:
            assert in_one_launch(x, groups)
        yield x, gamma, beta, shift, dy, ["swish", "none"][(i + sum(shape)) % 2], eps


@pytest.mark.parametrize("form", ["one launch", "chunks"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_constant_groups_beside_others(shape, groups, dtype, form):
    for x, gamma, beta, shift, _, act, eps in cases(shape, groups, dtype, form):
        got = group_norm_forward(x, gamma, beta, groups, shift=shift, eps=eps, activation=act)
        Truth(x, gamma, beta, shift, groups, act, eps).forward(*got)


@pytest.mark.parametrize("form", ["one launch", "chunks"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_gradients_of_constant_groups_beside_others(shape, groups, dtype, form):
    for x, gamma, beta, shift, dy, act, eps in cases(shape, groups, dtype, form):
        _, m, r = group_norm_forward(x, gamma, beta, groups, shift=shift, eps=eps, activation=act)
        got = group_norm_backward(dy, x, m, r, gamma, beta, groups, shift=shift, activation=act)
        Truth(x, gamma, beta, shift, groups, act, eps).backward(dy, *got)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_constant_group_leaves_the_others_bits(dtype):
    """What a group's neighbours (in the vector, in the wavefront, in the pack) hold does not change its result."""
    for shape, groups in SHAPES:
        x, gamma, beta, _, dy = case(shape, groups, dtype, 3, False, 1000.0)
        plain = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype]).cuda()
        keep = torch.zeros(groups, dtype=torch.bool, device="cuda")
        keep[::4] = True
        keep = keep.repeat_interleave(shape[-1] // groups)
        a, b = torch.where(keep, plain, x), plain
        ya, ma, ra = group_norm_forward(a, gamma, beta, groups)
        yb, mb, rb = group_norm_forward(b, gamma, beta, groups)
        assert torch.equal(ya[..., keep], yb[..., keep])
        da, db = group_norm_backward(dy, a, ma, ra, gamma, beta, groups), group_norm_backward(dy, b, mb, rb, gamma, beta, groups)
        assert torch.equal(da[0][..., keep], db[0][..., keep])
        assert torch.equal(da[1][keep], db[1][keep]) and torch.equal(da[2][keep], db[2][keep])


@pytest.mark.parametrize("power", [-60, -66])
def test_bfloat16_values_whose_squares_are_subnormal(power):
    """eps = 0 and deviations of 2^power: squares of 2^-120 and 2^-132, the latter below the normal float32 numbers, where they keep 17 bits:
    a relative 2^-18 of the variance, half of it in rstd."""
    gen = torch.Generator().manual_seed(9)
    x = (torch.randn(4, 12, 12, 32, generator=gen).sign() * 2.0 ** power).to(torch.bfloat16).cuda()
    _, mean, rstd = group_norm_forward(x, None, None, 4, eps=0.0, activation="none")
    g = x.cpu().double().reshape(4, 144, 4, 8)
    m, v = g.mean((1, 3)), g.var((1, 3), correction=0)
    over("mean", mean, m, 64 * E * 2.0 ** power)
    over("rstd", rstd, v.rsqrt(), (64 * E + 2.0 ** -18) * v.rsqrt())

"""CPU tests of the training operators: what they refuse, and how they read strides.  Nothing here launches a kernel: every call is
turned away by a check that comes before the first HIP call."""
import ctypes as C

import pytest
import torch

from isingdiff import (AdamW, _lib, adamw_moments, adamw_state, adamw_step, group_norm, group_norm_backward, group_norm_forward)
from isingdiff.norm import _layout


def test_norm_refuses():
    x, one = torch.zeros(2, 4, 4, 16), torch.ones(16)
    for bad in (dict(groups=3), dict(groups=0), dict(groups=-4), dict(groups=32), dict(activation="relu"), dict(shift=torch.zeros(3, 16)),
                dict(shift=torch.zeros(2, 8)), dict(shift=torch.zeros(2, 16).double()), dict(shift=torch.zeros(2, 1, 1, 16))):
        with pytest.raises(ValueError):
            group_norm_forward(x, one, one, **{"groups": 8, **bad})
    for gamma in (torch.ones(8), torch.ones(16).double(), torch.ones(1, 16)):
        with pytest.raises(ValueError):
            group_norm_forward(x, gamma, None)
    for t in (torch.zeros(16), x.double(), x.int(), torch.zeros(2, 4, 0), [1.0]):
        with pytest.raises(ValueError):
            group_norm_forward(t, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        group_norm_forward(x, one, one)
    with pytest.raises(ValueError, match="CUDA"):
        group_norm(x, one, one)
    with pytest.raises(ValueError, match="CUDA"):
        group_norm_backward(x, x, torch.zeros(2, 8), torch.zeros(2, 8), one, one)


def test_arguments_that_are_no_tensors():
    x, p = torch.zeros(2, 4, 4, 16), [torch.zeros(300)]
    s = adamw_state(p)
    for gamma, beta, shift in (([1.0] * 16, None, None), (None, 1.0, None), (None, None, "shift")):
        with pytest.raises(ValueError):
            group_norm_forward(x, gamma, beta, shift=shift)
    for groups in ("8", 8.0, None, 1 << 70):
        with pytest.raises(ValueError):
            group_norm_forward(x, None, None, groups)
    for eps in (-1e-3, float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError):
            group_norm_forward(x, None, None, eps=eps)
    with pytest.raises(TypeError):
        group_norm_forward(x, None, None, eps="small")
    for params, grads in ((p, [0.0]), ([None], [None]), ([p], [p]), (p, [torch.zeros(300).to_sparse()]), ([torch._neg_view(p[0])], p)):
        with pytest.raises(ValueError):
            adamw_step(params, grads, s)
    with pytest.raises(TypeError):
        adamw_step(p, 3, s)
    with pytest.raises(ValueError):
        adamw_step(p, p, s, betas=(0.9,))
    with pytest.raises(KeyError):
        adamw_step(p, p, {"m": s["m"], "v": s["v"]})
    for bad in ({**s, "v": None}, {**s, "v": s["m"]}):
        with pytest.raises(ValueError):
            adamw_step(p, p, bad)
    with pytest.raises(ValueError, match="CUDA"):
        adamw_step(iter(p), (q for q in p), s, weight_decay=(0.1 for _ in p))


def test_struct_layouts():
    assert C.sizeof(_lib.GroupNormDesc) == 80 and C.sizeof(_lib.AdamWCfg) == 48


def norm_desc(**over):
    f = dict(dtype=0, activation=1, batch=2, pixels=16, channels=16, groups=8, x_sample=256, x_pixel=16, dy_sample=256, dy_pixel=16,
             shift_sample=0, eps=1e-3, aligned=0)
    f.update(over)
    return _lib.GroupNormDesc(**f)


def test_norm_entry_points_refuse():
    lib, size = _lib.load(), C.c_size_t()
    assert lib.idm_group_norm_workspace(C.byref(norm_desc()), 0, C.byref(size)) == 0 and size.value > 0
    for bad in (dict(dtype=3), dict(activation=2), dict(batch=-1), dict(pixels=-1), dict(channels=0), dict(groups=0), dict(groups=5),
                dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x_pixel=15), dict(x_sample=-1), dict(shift_sample=-1),
                dict(channels=1 << 21, groups=1, x_pixel=1 << 21), dict(batch=1 << 32), dict(batch=(1 << 30) + 1)):
        d = norm_desc(**bad)
        assert lib.idm_group_norm_workspace(C.byref(d), 0, C.byref(size)) == -1, bad
        assert lib.idm_group_norm_forward(0, C.byref(d), *[16] * 8, 1 << 30, None) == -1, bad
        assert lib.idm_last_error()
    for bad in (dict(dy_pixel=15), dict(dy_sample=-1)):
        assert lib.idm_group_norm_workspace(C.byref(norm_desc(**bad)), 1, C.byref(size)) == -1
    d = norm_desc()
    for k in (0, 4, 5, 6, 7):      # x, y, mean, rstd, workspace
        args = [16] * 8
        args[k] = None
        assert lib.idm_group_norm_forward(0, C.byref(d), *args, 1 << 30, None) == -1
    for k in (0, 1, 2, 3, 7, 11):  # dy, x, mean, rstd, dx, workspace
        args = [16] * 12
        args[k] = None
        assert lib.idm_group_norm_backward(0, C.byref(d), *args, 1 << 30, None) == -1
    assert lib.idm_group_norm_forward(0, C.byref(d), *[16] * 8, 8, None) == -1 and b"workspace" in lib.idm_last_error()
    assert lib.idm_group_norm_backward(0, C.byref(d), *[16] * 12, 8, None) == -1 and b"workspace" in lib.idm_last_error()
    assert lib.idm_group_norm_forward(0, None, *[16] * 8, 1 << 30, None) == -1
    for n, entry in ((8, lib.idm_group_norm_forward), (12, lib.idm_group_norm_backward)):
        for k in range(n):             # 18: no float32's address, nor the workspace's
            args = [16] * n
            args[k] = 18
            assert entry(0, C.byref(d), *args, 1 << 30, None) == -1 and b"aligned" in lib.idm_last_error(), k
    d = norm_desc(aligned=1)
    assert lib.idm_group_norm_workspace(C.byref(d), 0, C.byref(size)) == 0 and size.value == 0
    for k in (0, 1, 2, 3, 4):      # x, gamma, beta, shift, y
        args = [16] * 8
        args[k] = 24
        assert lib.idm_group_norm_forward(0, C.byref(d), *args, 1 << 30, None) == -1 and b"aligned" in lib.idm_last_error()


def test_layout_of_strided_maps():
    t = torch.zeros(6, 9, 8, 80)
    assert _layout(t)[1:] == (9 * 8 * 80, 80)
    for cut, sample, pixel in ((t[..., 16:48], 5760, 80), (t[::2, :, :, 3:35], 11520, 80), (t[:, 2:3, 1:7, 8:40], 5760, 80),
                               (t[:, :, 2:3, :32], 5760, 640), (t[:, ::2, 0:1], 5760, 1280), (t[:, 0, 0], 5760, 80),
                               (t[:1, ..., :32].expand(4, 9, 8, 32), 0, 80)):
        got, s, p = _layout(cut)
        assert got is cut and (s, p) == (sample, pixel)
    for cut in (t[:, :, 2:7], t.transpose(1, 2), t[:, :1, :1].expand(6, 9, 8, 80), t[..., ::2], t.permute(0, 3, 1, 2),
                torch.zeros(2, 1, 1, 1).expand(2, 3, 4, 5)):
        got, s, p = _layout(cut)
        assert got.is_contiguous() and torch.equal(got, cut) and p == cut.shape[-1]
    assert _layout(torch.zeros(3, 5))[1:] == (5, 5)


def test_adamw_refuses():
    p, g = [torch.zeros(300), torch.zeros(4, 5)], [torch.zeros(300), torch.zeros(4, 5)]
    s = adamw_state(p)
    assert s["m"].shape == (768,) and s["m"].dtype == torch.float32 and set(s) == {"step", "m", "v"}
    e = adamw_state(p, 8)
    assert e["v"].dtype == torch.uint8 and e["m_base"].shape == (3,)
    for bits in (16, 4, "8"):
        with pytest.raises(ValueError):
            adamw_state(p, bits)
    with pytest.raises(ValueError):
        adamw_state([])
    for params, grads in (([], []), (p, g[:1]), (p, [g[0], torch.zeros(5, 4)]), ([p[0], p[1].half()], g), (p, [g[0], g[1].half()]),
                          ([p[0].double(), p[1].double()], g), ([p[0], torch.zeros(5, 4).t()], g)):
        with pytest.raises(ValueError):
            adamw_step(params, grads, s)
    for bad in (dict(lr=-1.0), dict(lr=float("nan")), dict(eps=-1e-8), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)),
                dict(weight_decay=[0.1]), dict(weight_decay=[0.1, -0.1]), dict(weight_decay=float("inf"))):
        with pytest.raises(ValueError):
            adamw_step(p, g, s, **bad)
    for bad in (adamw_state(p[:1]), {**s, "m": s["m"].double()}, {**s, "step": s["step"].int()}, {**e, "m_base": e["m_base"][:2]},
                {**e, "v": e["v"][::2]}):
        with pytest.raises(ValueError):
            adamw_step(p, g, bad)
    with pytest.raises(ValueError, match="CUDA"):
        adamw_step(p, g, s)
    with pytest.raises(ValueError, match="CUDA"):
        adamw_moments(e)
    assert adamw_moments(s)[0] is s["m"]
    opt = AdamW(p)
    with pytest.raises(ValueError):
        opt.load_state_dict(e)


def adamw_call(sizes=(300, 20), params=(1 << 20, 1 << 21), grads=(1 << 22, 1 << 23), decay=(0.0, 0.0), moments=768, m=4096, v=8192,
               base=(16384, 32768), step=64, scratch=128, n=None, **cfg):
    c = dict(param_dtype=0, grad_dtype=0, moment_bits=8, reserved=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    c.update(cfg)
    k = len(sizes)
    return _lib.load().idm_adamw_step(0, C.byref(_lib.AdamWCfg(**c)), k if n is None else n, (C.c_void_p * k)(*params),
                                      (C.c_void_p * k)(*grads), (C.c_int64 * k)(*sizes), (C.c_float * k)(*decay), m, v, *base, moments,
                                      step, scratch, None)


def test_adamw_entry_points_refuse():
    for bad in (dict(param_dtype=3), dict(grad_dtype=-1), dict(moment_bits=16), dict(lr=-1.0), dict(lr=float("inf")), dict(beta1=1.0),
                dict(beta2=float("nan")), dict(eps=-1.0), dict(n=-1), dict(sizes=(300, -1)), dict(sizes=(300, 1 << 41)), dict(moments=512),
                dict(moments=0), dict(params=(1 << 20, None)), dict(params=(1 << 20, (1 << 21) + 2)), dict(grads=(1 << 22, (1 << 23) + 1)),
                dict(params=(1 << 20, 1 << 20)), dict(params=(1 << 20, (1 << 20) + 1196)), dict(grads=(1 << 22, 1 << 20)), dict(grads=((1 << 20) + 4, 1 << 23)),
                dict(grads=((1 << 21) - 1196, 1 << 23)), dict(grads=(1 << 20, 1 << 23), grad_dtype=1), dict(decay=(0.0, -1.0)),
                dict(decay=(0.0, float("nan"))), dict(m=None), dict(v=8200), dict(base=(None, 32768)), dict(step=None), dict(scratch=None),
                dict(step=68), dict(scratch=132)):
        assert adamw_call(**bad) == -1, bad
        assert b"adamw" in _lib.load().idm_last_error()
    lib = _lib.load()
    assert lib.idm_adamw_moments(0, *[4096] * 6, 0, None) == 0
    for n in (-256, 100):
        assert lib.idm_adamw_moments(0, *[4096] * 6, n, None) == -1
    for k in range(6):
        args = [4096] * 6
        args[k] = None
        assert lib.idm_adamw_moments(0, *args, 256, None) == -1
    assert lib.idm_adamw_moments(0, 4096, 4104, 4096, 4096, 4096, 4096, 256, None) == -1

"""AdamW at the ends of its arguments."""
import pytest
import torch

from isingdiff import AdamW, adamw_moments, adamw_state, adamw_step

pytestmark = pytest.mark.gpu

SMALL, LARGE = 3000, 256 * 4096 + 1      # entries of a step that counts itself, and of one that is counted before


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [SMALL, 20 * 4096 + 5, LARGE])
def test_a_negative_count_stops_the_step(n, bits):
    """Nothing is written, the count included, and the same state goes on once the count is right."""
    gen = torch.Generator("cuda").manual_seed(3)
    p, g = (torch.randn(n, device="cuda", generator=gen) for _ in range(2))
    q, s = p.clone(), adamw_state([p], bits)
    r = {k: t.clone() for k, t in s.items()}
    adamw_step([p], [g], s)
    adamw_step([q], [g], r)
    for count in (-1, -2, -(2 ** 53), -(2 ** 63), -(2 ** 62) + 5):
        s["step"].fill_(count)
        keep = {k: t.clone() for k, t in s.items()}
        for _ in range(3):
            adamw_step([p], [g], s)
        assert torch.equal(p, q) and all(torch.equal(s[k], keep[k]) for k in s), count
    s["step"].fill_(1)
    adamw_step([p], [g], s)
    adamw_step([q], [g], r)
    assert torch.equal(p, q) and all(torch.equal(s[k], r[k]) for k in s) and int(s["step"]) == 2


def test_counts_that_are_none_are_not_loaded():
    opt = AdamW([torch.zeros(5, device="cuda")])
    for count in (-1, 2 ** 53, 2 ** 62):
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict({**opt.state_dict(), "step": torch.tensor([count])})
    opt.load_state_dict({**opt.state_dict(), "step": torch.tensor([2 ** 53 - 2])})
    opt.params[0].grad = torch.ones(5, device="cuda")
    opt.step()
    assert int(opt.state["step"]) == 2 ** 53 - 1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-38, 1e-42, 1e-50, 1e-300])
def test_an_eps_below_the_normal_float32_numbers(eps, bits):
    """0 / (0 + eps) is 0 for every eps above zero.  Elsewhere the root of a moment is at least 2^-75 (codes: 2^-64), where no such eps counts."""
    p = torch.linspace(-1, 1, 512, device="cuda")
    q, g = p.clone(), torch.zeros(512, device="cuda")
    g[::2] = torch.linspace(-1e-3, 1e-3, 256, device="cuda")
    g[2] = 1e-20
    s, r = adamw_state([p], bits), adamw_state([q], bits)
    for _ in range(3):
        before = p.clone()
        adamw_step([p], [g], s, eps=eps, weight_decay=0.0)
        adamw_step([q], [g], r, eps=2.0 ** -100, weight_decay=0.0)
        assert torch.equal(p[1::2], before[1::2])
    assert torch.equal(p, q) and all(torch.equal(s[k], r[k]) for k in s)


def test_more_moments_than_one_pass_of_the_grid():
    """2^30 entries are decoded in one pass, the 768 behind them in a second."""
    n = (1 << 30) + 768
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of GPU memory")
    s = {"step": torch.zeros(1, dtype=torch.int64, device="cuda")}
    for k in "mv":
        s[k] = torch.randint(0, 256, (n,), dtype=torch.uint8, device="cuda")
        s[k + "_base"] = torch.randint(0, 1500, (n // 256,), dtype=torch.int16, device="cuda")
    m, v = adamw_moments(s)
    for lo in (0, (1 << 29) - 512, (1 << 30) - 1024):     # each part by itself gives the same
        part = slice(lo, lo + 1792), slice(lo // 256, lo // 256 + 7)
        few = {k: t[part[k.endswith("base")]].clone() for k, t in s.items() if k != "step"}
        a, b = adamw_moments({**few, "step": s["step"]})
        assert torch.equal(a, m[part[0]]) and torch.equal(b, v[part[0]])
    assert int((v == 0).sum()) == int((s["v"] == 0).sum()) and int((m == 0).sum()) == int((s["m"] & 127 == 0).sum())

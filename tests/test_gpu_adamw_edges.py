"""AdamW at the ends of its arguments."""
import pytest
import torch

from isingdiff import AdamW, adamw_state, adamw_step

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

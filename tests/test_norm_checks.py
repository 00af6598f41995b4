"""CPU tests of what group norm refuses.  Nothing here launches a kernel."""
import numpy as np
import pytest
import torch

from isingdiff import group_norm, group_norm_forward


def test_an_eps_that_float32_holds_as_zero_is_refused():
    """A constant group would get an infinite rstd and NaN for 0 * rstd."""
    x = torch.zeros(2, 4, 4, 16)
    for eps in (1e-46, 1e-300, 5e-324):
        for call in (lambda: group_norm_forward(x, None, None, eps=eps), lambda: group_norm(x, eps=eps)):
            with pytest.raises(ValueError, match="eps"):
                call()
    for eps in (0.0, 1e-45, 1e-3):      # (and those get as far as the device)
        with pytest.raises(ValueError, match="CUDA"):
            group_norm_forward(x, None, None, eps=eps)


def test_any_integer_is_a_group_count():
    x = torch.zeros(2, 4, 4, 16)
    for groups in (np.int64(8), np.uint8(4), torch.tensor(2), True):
        with pytest.raises(ValueError, match="CUDA"):      # (as far as the device)
            group_norm_forward(x, None, None, groups)
    for groups in (np.float32(8), torch.tensor(2.0), np.int64(3), np.int64(-4), torch.tensor([8, 8])):
        with pytest.raises(ValueError, match="groups"):
            group_norm_forward(x, None, None, groups)

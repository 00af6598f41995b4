"""CPU tests of the AdamW step's refusals: memory that is shared, counts, sizes and numbers.  Every call is turned away by a check that comes
before the first HIP call."""
import ctypes as C

import numpy as np
import pytest
import torch

from isingdiff import _lib, adamw_state, adamw_step

PARAM, GRAD, M, V, MB, VB, STEP, SCRATCH = (k << 20 for k in range(1, 9))


def step(params=(PARAM, PARAM + 4096), grads=(GRAD, GRAD + 4096), sizes=(300, 20), m=M, v=V, bases=(MB, VB), count=STEP, scratch=SCRATCH, bits=8):
    k = len(sizes)
    cfg = _lib.AdamWCfg(param_dtype=0, grad_dtype=0, moment_bits=bits, reserved=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    rc = _lib.load().idm_adamw_step(0, C.byref(cfg), k, (C.c_void_p * k)(*params), (C.c_void_p * k)(*grads), (C.c_int64 * k)(*sizes),
                                    (C.c_float * k)(), m, v, *bases, sum(-(-n // 256) * 256 for n in sizes), count, scratch, None)
    return rc, _lib.load().idm_last_error()


# 768 entries of moments: 768 bytes of codes, 6 of bases; 3 072 bytes in 32 bits
@pytest.mark.parametrize("bits,over", [
    (8, dict(m=V)), (32, dict(m=V)),                                  # one memory for both moments
    (8, dict(v=M + 512)), (32, dict(v=M + 2048)), (32, dict(m=V + 1024)),     # shifted against each other
    (8, dict(bases=(MB, MB))), (8, dict(bases=(MB, MB + 4))), (8, dict(bases=(M + 766, VB))),
    (8, dict(m=PARAM)), (8, dict(v=PARAM + 1008)), (32, dict(m=PARAM - 1024)), (8, dict(bases=(MB, PARAM + 4096 + 78))),     # parameters
    (8, dict(m=GRAD + 1024)), (32, dict(v=GRAD - 2048)), (8, dict(bases=(GRAD + 4096, VB))),                                 # gradients
    (8, dict(count=M)), (8, dict(count=PARAM + 1192)), (8, dict(count=GRAD + 4096 + 72)), (8, dict(count=SCRATCH)), (8, dict(count=SCRATCH + 8)),
    (8, dict(scratch=V + 760)), (32, dict(scratch=M + 3064)), (8, dict(scratch=PARAM - 8)), (8, dict(scratch=GRAD + 1192)),
])
def test_state_that_shares_memory_is_refused(bits, over):
    rc, why = step(bits=bits, **over)
    assert rc == -1 and b"share" in why, (rc, why)


def test_decoding_into_its_own_input_is_refused():
    """512 entries: 512 bytes of codes, 4 of bases, 2 048 of each result."""
    args = dict(m=M, v=V, m_base=MB, v_base=VB, m_out=PARAM, v_out=GRAD)
    for over in (dict(m_out=M), dict(v_out=M + 256), dict(m_out=V - 1024), dict(v_out=VB - 16), dict(m_out=GRAD), dict(v_out=PARAM + 2032)):
        assert _lib.load().idm_adamw_moments(0, *{**args, **over}.values(), 512, None) == -1, over
        assert b"share" in _lib.load().idm_last_error()


def test_bases_that_are_not_aligned_are_refused():
    for bases in ((MB + 1, VB), (MB, VB + 3)):
        rc, why = step(bases=bases)
        assert rc == -1 and b"aligned" in why


def test_a_tensor_that_one_launch_cannot_cover_is_refused():
    """(2^24 - 1) workgroups of 256 threads and 4 096 entries: fewer than 2^32 threads."""
    most = ((1 << 24) - 1) * 4096
    at = dict(params=(1 << 45, PARAM), grads=(1 << 46, GRAD), m=1 << 47, v=1 << 48, bases=(1 << 49, 1 << 50))
    for n in (most + 1, 1 << 36, 1 << 40):
        rc, why = step(sizes=(n, 20), **at)
        assert rc == -1 and b"size" in why, (n, rc, why)
    rc, why = step(sizes=(most, 20), bases=(MB, MB), **{k: a for k, a in at.items() if k != "bases"})
    assert rc == -1 and b"share" in why, (rc, why)      # (as far as the next check)


def test_numbers_are_taken_before_the_tensors_are_looked_at():
    """A number's __float__ is anybody's code: what it does to a parameter is seen by the checks."""
    p = torch.zeros(300)

    class Decay:
        def __float__(self):
            p.data = torch.zeros(7)
            return 0.1
    state = adamw_state([p])
    with pytest.raises(ValueError, match="shape"):
        adamw_step([p], [torch.zeros(300)], state, weight_decay=[Decay()])

    class State(dict):
        def __getitem__(self, k):
            q.data = torch.zeros(7)
            return super().__getitem__(k)
    q = torch.zeros(300)
    state = State(adamw_state([q]))
    with pytest.raises(ValueError, match="shape"):
        adamw_step([q], [torch.zeros(300)], state)


@pytest.mark.parametrize("decay", [np.float32(0.1), np.float64(0.1), np.int64(0), 0, True, np.array([0.1]), torch.tensor([0.1]), (0.1 for _ in range(1))])
def test_any_number_is_a_weight_decay(decay):
    p = torch.zeros(3)
    with pytest.raises(ValueError, match="CUDA"):      # (as far as the device)
        adamw_step([p], [p.clone()], adamw_state([p]), weight_decay=decay)

"""A tensor that a step would update twice at once: the workgroups of one launch
would race on it.  Refused before anything is launched (addresses that no refused
call touches; the last case has nothing to launch)."""
import ctypes

import pytest
import torch

import spmm_amd as S
from spmm_amd import _lib as L
from spmm_amd import training as T

P = 1 << 20


def _step(tensors, dtype=S.TCA_F32, device=False):
    table = (ctypes.c_int64 * (8 * len(tensors)))()
    for k, (param, n) in enumerate(tensors):
        table[8 * k:8 * k + 8] = [param, P * 8, P * 16 * (k + 1), P * 32 * (k + 1), P * 64 * (k + 1), 0, 0, n]
    common = (ctypes.addressof(table),)
    settings = (1e-3, 0.9, 0.999, 1e-8, 0.0)
    if device:
        steps = (ctypes.c_void_p * len(tensors))(*(P + 8 * k for k in range(len(tensors))))
        return L.lib.tca_adamw_step_device(*common, ctypes.addressof(steps), len(tensors), dtype, 32, *settings, P, None)
    return L.lib.tca_adamw_step(*common, len(tensors), dtype, 32, 1, *settings, None)


@pytest.mark.parametrize("device", [False, True])
@pytest.mark.parametrize("dtype,size", [(S.TCA_F32, 4), (S.TCA_BF16, 2)])
def test_overlapping_parameters(device, dtype, size):
    for second in (P, P + size, P + 9 * size, P - 4 * size):
        assert _step([(P, 10), (P + 1000, 20), (second, 5)], dtype, device) == 1, second
        assert b"share memory" in L.lib.tca_last_error()
    far = [(P + 1000 * k, 10) for k in range(100)]
    assert _step(far + [(P + 50 * 1000, 1)], dtype, device) == 1


def test_a_parameter_given_twice():
    p = torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="more than once"):
        T.AdamW([p, torch.nn.Parameter(torch.ones(2)), p])
    opt = T.AdamW([torch.nn.Parameter(torch.ones(2))])
    with pytest.raises(ValueError, match="more than once"):
        opt.add_param_group(dict(params=[p, p]))
    assert len(opt.param_groups) == 1


def test_empty_tensors_share_nothing():
    assert _step([(P, 0), (P, 0)]) == 0

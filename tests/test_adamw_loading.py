"""What AdamW.load_state_dict takes and refuses (on the CPU: nothing is launched)."""
import copy

import pytest
import torch

from spmm_amd import training as T


def _params(dtype=torch.float32):
    return [torch.nn.Parameter(torch.arange(1.0, 1 + n).to(dtype)) for n in (5, 3)]


def _theirs(kind=torch.optim.AdamW, steps=2, dtype=torch.float32, **settings):
    ps = _params(dtype)
    opt = kind(ps, lr=0.5, **settings)
    for _ in range(steps):
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
    return opt.state_dict()


def _before(opt):
    return copy.deepcopy(opt.param_groups), len(opt.state)


def _refused(opt, saved, match):
    """A refusal leaves the optimizer as it was."""
    groups, states = _before(opt)
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(saved)
    assert len(opt.state) == states
    for g, h in zip(opt.param_groups, groups):
        assert {k: v for k, v in g.items() if k != "params"} == {k: v for k, v in h.items() if k != "params"}


@pytest.mark.parametrize("settings", [dict(maximize=True), dict(amsgrad=True), dict(maximize=True, amsgrad=True)])
@pytest.mark.parametrize("steps", [0, 2])
def test_refuses_options_it_does_not_have(settings, steps):
    _refused(T.AdamW(_params()), _theirs(steps=steps, **settings), next(iter(settings)))


def test_refuses_a_differentiable_step():
    saved = _theirs()
    saved["param_groups"][0]["differentiable"] = True
    _refused(T.AdamW(_params()), saved, "differentiable")


def test_refuses_adam_whose_decay_is_part_of_the_gradient():
    _refused(T.AdamW(_params()), _theirs(torch.optim.Adam, weight_decay=0.1), "decoupled_weight_decay")


def test_refuses_the_state_of_another_optimizer():
    _refused(T.AdamW(_params()), _theirs(torch.optim.SGD, momentum=0.9), "betas")
    _refused(T.AdamW(_params()), _theirs(torch.optim.Adamax), "exp_avg_sq")
    saved = _theirs()
    saved["state"][1]["other"] = torch.zeros(3)
    _refused(T.AdamW(_params()), saved, "other")


def test_refuses_states_of_other_bits_or_types():
    _refused(T.AdamW(_params(), state_bits=8), _theirs(), "exp_avg_rms")
    _refused(T.AdamW(_params(torch.bfloat16)), _theirs(dtype=torch.bfloat16), "master")
    saved = _theirs()
    saved["param_groups"][0]["state_bits"] = 16
    _refused(T.AdamW(_params()), saved, "state_bits")


@pytest.mark.parametrize("capturable", [False, True])
def test_takes_torchs_settings_and_keeps_its_own(capturable):
    ps = _params()
    opt = T.AdamW(ps, capturable=capturable)
    saved = _theirs(weight_decay=0.25, betas=(0.8, 0.9), eps=1e-5)
    saved["param_groups"][0]["initial_lr"] = 2.0  # a scheduler's
    opt.load_state_dict(saved)
    group, = opt.param_groups
    assert {k: v for k, v in group.items() if k != "params"} == dict(
        lr=0.5, weight_decay=0.25, betas=(0.8, 0.9), eps=1e-5, initial_lr=2.0, state_bits=32, capturable=capturable)
    for i, p in enumerate(ps):
        assert set(opt.state[p]) == {"step", "exp_avg", "exp_avg_sq"}
        assert torch.equal(opt.state[p]["exp_avg"], saved["state"][i]["exp_avg"])
        step = opt.state[p]["step"]
        assert (step.dtype == torch.int64 and int(step) == 2) if capturable else step == 2 and type(step) is int


def test_takes_its_own_with_the_settings_that_were_saved():
    first = T.AdamW(_params(), lr=0.1, state_bits=8, capturable=True)
    other = T.AdamW(_params(), lr=0.2)
    other.load_state_dict(first.state_dict())  # no step taken: settings alone
    group, = other.param_groups
    assert (group["lr"], group["state_bits"], group["capturable"]) == (0.1, 8, True) and not other.state


def test_a_wrong_number_of_parameters_is_torchs_refusal():
    saved = _theirs()
    saved["param_groups"][0]["params"] = [0]
    with pytest.raises(ValueError):
        T.AdamW(_params()).load_state_dict(saved)


@pytest.mark.parametrize("settings", [dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0),
                                      dict(state_bits=8, eps=0.0), dict(weight_decay=-0.1)])
def test_a_groups_own_settings_are_checked(settings):
    p, q = _params()
    with pytest.raises(ValueError, match="AdamW"):
        T.AdamW([dict(params=[p], **settings)])
    opt = T.AdamW([p])
    with pytest.raises(ValueError, match="AdamW"):
        opt.add_param_group(dict(params=[q], **settings))
    assert len(opt.param_groups) == 1

"""Derivatives that the training operators do not have are refused, not dropped
(on meta tensors: the refusal comes before a device is looked at)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from spmm_amd import training as T


def _x():
    return torch.randn(4, 8, device="meta")


def _target():
    return torch.zeros(4, dtype=torch.int64, device="meta")


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_layer_norm_refuses_a_tangent(which):
    given = {"x": _x(), "weight": torch.ones(8, device="meta"), "bias": torch.ones(8, device="meta")}
    with fwd.dual_level():
        given[which] = fwd.make_dual(given[which], torch.ones_like(given[which]))
        with pytest.raises(NotImplementedError, match="layer_norm.*forward-mode"):
            T.layer_norm(**given)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="layer_norm.*forward-mode"):
            T.layer_norm(**given)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_refuses_a_tangent(reduction):
    with fwd.dual_level():
        x = fwd.make_dual(_x(), _x())
        with pytest.raises(NotImplementedError, match="cross_entropy.*forward-mode"):
            T.cross_entropy(x, _target(), reduction=reduction)


def test_a_tangent_beside_a_gradient_is_refused_too():
    with fwd.dual_level():
        x = fwd.make_dual(_x(), _x())
        w = torch.ones(8, device="meta", requires_grad=True)
        with pytest.raises(NotImplementedError, match="layer_norm.*forward-mode"):
            T.layer_norm(x, w)


@pytest.mark.parametrize("f", [lambda x: T.layer_norm(x), lambda x: T.cross_entropy(x, _target())])
def test_functional_jvp_is_refused(f):
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (_x(),), (_x(),))


def test_calls_without_a_tangent_pass_within_a_dual_level():
    with fwd.dual_level():
        assert T.layer_norm(_x()).shape == (4, 8) and T.cross_entropy(_x(), _target()).shape == ()


def test_the_gradient_in_one_pass_is_a_constant_in_either_mode():
    with fwd.dual_level():
        loss, g = T.cross_entropy_grad(fwd.make_dual(_x(), _x()), _target())
        assert fwd.unpack_dual(loss).tangent is None and fwd.unpack_dual(g).tangent is None


@pytest.mark.parametrize("f", [lambda x: T.layer_norm(x).sum(), lambda x: T.cross_entropy(x, _target())])
def test_functional_grad_is_refused(f):
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(f)(_x())

"""Cross entropy of rows that lie 2^31 elements or more apart, as the last
positions of long sequences do: the same bits as for the rows side by side."""
import pytest
import torch

from spmm_amd import training as T

pytestmark = pytest.mark.gpu


def _check(x, t):
    """x against a copy whose rows lie side by side."""
    want_x = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
    x = x.detach().requires_grad_()
    for reduction in ("mean", "sum", "none"):
        a, b = T.cross_entropy(x, t, reduction=reduction), T.cross_entropy(want_x, t, reduction=reduction)
        assert torch.equal(a, b)
        up = torch.ones_like(a)
        assert torch.equal(torch.autograd.grad(a, x, up)[0], torch.autograd.grad(b, want_x, up)[0])
    for a, b in zip(T.cross_entropy_grad(x.detach(), t), T.cross_entropy_grad(want_x.detach(), t)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 3])
def test_last_positions_of_long_sequences(torch_cuda, rows):
    steps, classes = 42950, 50001  # 2.1475e9 elements a sequence, just past 2^31
    full = torch.empty(rows, steps, classes, dtype=torch.bfloat16, device="cuda:0")
    full[:, -1] = torch.randn(rows, classes, device="cuda:0").to(torch.bfloat16)
    x = full[:, -1]
    assert x.stride(0) == steps * classes > 2 ** 31 - 1
    _check(x, torch.arange(rows, device="cuda:0") * 7000)


def test_one_row_of_any_stride(torch_cuda):
    """The stride of a single row says nothing: no memory lies behind it."""
    x = torch.randn(47, device="cuda:0").as_strided((1, 47), (2 ** 33, 1))
    _check(x, torch.zeros(1, dtype=torch.int64, device="cuda:0"))

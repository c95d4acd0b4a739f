"""Layer norm of rows whose mean is far larger than their deviation: rows of one
value have a variance of 0 and give the bias, whatever the value and the width, and
a mean's error is that of its one rounding to fp32.

Tolerance of the offset rows, u = 2^-24, D = 42 additions in a sum: the first mean
is off by e <= (D + 2) u mean|x|; the mean of the distances from it corrects that to
(D + 3) u (e + mean|x - mean|), and the corrected mean is rounded once:
  e_mean = u |mean| + (D + 3) u (e + mean|x - mean|).
The variance is taken about the corrected mean, which adds the square of its error:
  r = (D + 8) u + (e_mean rstd)^2                      relative error of rstd
  e_xh = rstd (e_mean + u |x - mean|) + |xh| r."""
import numpy as np
import pytest
import torch

from spmm_amd import training as T

pytestmark = pytest.mark.gpu

U, D = 2.0 ** -24, 42
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
WIDTHS = [2, 3, 5, 6, 7, 9, 15, 47, 100, 129, 300, 384, 1000, 1025, 2049, 5000, 9001, 16383, 16384]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", WIDTHS)
def test_rows_of_one_value(torch_cuda, dtype, width):
    print(f"layer_norm {dtype} width={width}", flush=True)
    rng = np.random.default_rng(width)
    values = torch.tensor([1e4, 1e5, -1e5, 1000.1, 0.1, 3.0, -33333333.0, 1.7e-3, 6e4, 1e12, 0.0]).to(dtype)
    values = values[torch.isfinite(values)].to("cuda:0")
    x = values[:, None].expand(-1, width).contiguous().requires_grad_()
    w, b = (torch.from_numpy(rng.standard_normal(width).astype(np.float32)).to("cuda:0").requires_grad_() for _ in "wb")
    y = T.layer_norm(x, w, b)
    assert torch.equal(y, b.detach().to(dtype).expand_as(y))
    _, stats = torch.ops.spmm_amd.layer_norm_stats(x.detach(), w.detach(), b.detach(), 1e-5, None)
    assert torch.equal(stats[:, 0], values.float())
    dy = torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)).to("cuda:0").to(dtype)
    dx, dw, _ = torch.autograd.grad(y, (x, w, b), dy)
    assert bool((dw == 0).all())
    g = dy.double() * w.detach().double()
    want = 1e-5 ** -0.5 * (g - g.mean(1, keepdim=True))  # the fp32 eps is 1e-5 (1 + 2^-24) at most
    bound = 1e-5 ** -0.5 * ((D + 4) * U * g.abs().mean(1, keepdim=True) + 4 * U * g.abs()) + (D + 8) * U * want.abs()
    bound = bound + {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype] * want.abs() * (1 + 1e-3) + 2.0 ** -24
    assert bool(((dx.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("offset", [30.0, 1e3, -1e4, 1e5])
@pytest.mark.parametrize("width", [7, 47, 384, 1000, 2049, 9001])
def test_offset_rows(torch_cuda, offset, width):
    rng = np.random.default_rng(width)
    x = torch.from_numpy((rng.standard_normal((64, width)) + offset).astype(np.float32)).to("cuda:0")
    y, stats = torch.ops.spmm_amd.layer_norm_stats(x, None, None, 1e-5, None)
    d = x.double()
    mean = d.mean(1, keepdim=True)
    away = (d - mean).abs()
    rstd = (away.square().mean(1, keepdim=True) + 1e-5) ** -0.5
    e = (D + 2) * U * d.abs().mean(1, keepdim=True)
    e_mean = U * mean.abs() + (D + 3) * U * (e + away.mean(1, keepdim=True))
    r = (D + 8) * U + (e_mean * rstd) ** 2
    xh = (d - mean) * rstd
    assert bool(((stats[:, :1].double() - mean).abs() <= e_mean).all())
    assert bool(((stats[:, 1:].double() / rstd - 1).abs() <= r + 2 * U).all())
    assert bool(((y.double() - xh).abs() <= rstd * (e_mean + U * away) + xh.abs() * (r + 4 * U)).all())


def test_an_outlier_among_small_values(torch_cuda):
    """The correction is taken from the mean, not from any one entry: a first entry of
    1e8 leaves the others' places to the rounding of fp32 alone."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((4, 4096)).astype(np.float32)).to("cuda:0")
    x[0, 0] = x[1, 4095] = x[2, 77] = 1e8
    y = T.layer_norm(x)
    d = x.double() - x.double().mean(1, keepdim=True)
    want = d * (d.square().mean(1, keepdim=True) + 1e-5) ** -0.5
    # of the row's deviation, which the outlier makes: (D + 8) u of the largest distance from the mean
    assert bool(((y.double() - want).abs() <= (D + 8) * U * (want.abs() + want.abs().mean(1, keepdim=True) + 1e-3)).all())

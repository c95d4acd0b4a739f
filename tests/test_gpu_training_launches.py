"""The training operators at sizes that take every launch: several rows a turn,
several turns a chunk, several chunks, rows in flight ahead, lines streamed past the
caches, offsets past 32 bits.

Where a row is lost or taken twice among a million, no rounding bound shows it, so
the inputs here make every sum exact and outputs are compared for equality.

Cross entropy: logits of -1000 but for a 0 at a row's place a and -j (128 <= j < 256)
at its target: exp(-j) is 0 in fp32, the row's sum 1, its loss j (0 where the target
is a) and its gradient +1 at a, -1 at the target.

Layer norm with eps 0: rows of as many 1 as -1 over a power of two of columns have
mean 0 and deviation 1; weights are powers of two, output gradients small integers,
so the output and all gradients are exact.  Other widths: the bits of small calls,
row block by row block, and the exact sums of dy."""
import numpy as np
import pytest
import torch

from spmm_amd import training as T

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
IGNORE = -100


# ------------------------------------------------------------------ cross entropy
def _rows(rows, classes, share, seed):
    """Places a, targets, and j; some targets are the place itself."""
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    a, t, j = (torch.randint(lo, hi, (rows,), generator=g, device="cuda:0") for lo, hi in
               ((0, classes), (0, classes), (128, 256)))
    t[0], t[-1] = 0, classes - 1
    labelled = torch.rand((rows,), generator=g, device="cuda:0") < share
    labelled[0] = labelled[-1] = True
    return a, t, torch.where(t == a, 0, j), labelled


def _fill(x, a, t, j):
    x.fill_(-1000.0)
    x.scatter_(1, t[:, None], -j[:, None].to(x.dtype))
    x.scatter_(1, a[:, None], torch.zeros_like(a)[:, None].to(x.dtype))


def _wanted_gradient(x, a, t, j, labelled, factor):
    want = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
    moves = (labelled & (j > 0)).to(torch.float32) * factor
    want.scatter_(1, a[:, None], moves[:, None].to(x.dtype))
    at = torch.nonzero(labelled & (j > 0))[:, 0]
    want[at, t[at]] = (-moves[at]).to(x.dtype)
    return want


def _check_loss(x, a, t, j, labelled, both=True):
    _fill(x, a, t, j)
    target = torch.where(labelled, t, IGNORE)
    each = torch.where(labelled, j, 0)
    total, count = int(each.sum()), int(labelled.sum())
    leaf = x.detach().requires_grad_()
    for reduction, loss64, factor in (("sum", float(total), 1.0), ("mean", total / count, float(np.float32(1) / np.float32(count))),
                                      ("none", None, 1.0)):
        print(f"  {reduction}", flush=True)
        loss = T.cross_entropy(leaf, target, reduction=reduction)
        up = torch.ones_like(loss)
        if loss64 is None:
            assert torch.equal(loss.detach(), each.float())
        else:
            assert float(loss.detach()) == float(np.float32(loss64))
        dx, = torch.autograd.grad(loss, leaf, up)
        want = _wanted_gradient(x, a, t, j, labelled, factor)
        assert torch.equal(dx, want), reduction
        del dx
        if both and reduction != "none":
            loss, dx = T.cross_entropy_grad(x, target, reduction=reduction)
            assert float(loss) == float(np.float32(loss64)) and torch.equal(dx, want), reduction


LOSSES = [(2_200_001, 9, F32), (2_200_001, 47, F32), (600_001, 100, F16), (300_001, 300, BF16), (150_001, 500, F32),
          (40_001, 700, F32), (2_100_001, 520, F32), (20_001, 3600, F32), (17_001, 4000, BF16), (530_001, 3100, BF16),
          (14_001, 5000, F32), (2_101, 33_000, F32), (1_101, 70_003, BF16)]


@pytest.mark.parametrize("share", [1.0, 0.85, 0.2])
@pytest.mark.parametrize("rows,classes,dtype", LOSSES)
def test_losses_are_exact(torch_cuda, rows, classes, dtype, share):
    print(f"cross_entropy {rows} x {classes} {dtype} {share}", flush=True)
    x = torch.empty(rows, classes, dtype=dtype, device="cuda:0")
    _check_loss(x, *_rows(rows, classes, share, rows))


@pytest.mark.parametrize("rows,classes,pitch", [(45_000, 50_001, 50_001), (70_000, 47, 65_536)])
def test_differentiable_losses_past_32_bits(torch_cuda, rows, classes, pitch):
    print(f"cross_entropy {rows} x {classes} pitch {pitch}", flush=True)
    full = torch.empty(rows, pitch, dtype=BF16, device="cuda:0")
    _check_loss(full[:, pitch - classes:], *_rows(rows, classes, 0.5, 7))


@pytest.mark.parametrize("rows,classes,dtype", [(150_001, 47, F32), (70_001, 130, BF16), (17_001, 4000, F32), (2_201, 33_001, F32)])
def test_losses_of_random_rows(torch_cuda, rows, classes, dtype):
    """The bits of small calls, row block by row block, at large calls' launches."""
    print(f"cross_entropy {rows} x {classes} {dtype}", flush=True)
    g = torch.Generator(device="cuda:0").manual_seed(rows)
    x = (3 * torch.randn(rows, classes, generator=g, device="cuda:0")).to(dtype)
    target = torch.randint(0, classes, (rows,), generator=g, device="cuda:0")
    target[::3] = IGNORE
    leaf = x.detach().requires_grad_()
    loss = T.cross_entropy(leaf, target, reduction="none")
    dx, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    _, both = T.cross_entropy_grad(x, target, reduction="sum")
    size = max(60, rows // 100)
    for k in range(0, rows, size):
        part = x[k:k + size].clone().requires_grad_()
        each = T.cross_entropy(part, target[k:k + size], reduction="none")
        assert torch.equal(each.detach(), loss.detach()[k:k + size]), k
        assert torch.equal(torch.autograd.grad(each, part, torch.ones_like(each))[0], dx[k:k + size]), k
        assert torch.equal(T.cross_entropy_grad(part.detach(), target[k:k + size], reduction="sum")[1], both[k:k + size]), k


# --------------------------------------------------------------------- layer norm
def _signs(rows, width, seed):
    """Rows of as many 1 as -1, in an order of their own each."""
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    half = torch.rand((rows, width // 2), generator=g, device="cuda:0") < 0.5
    x = torch.where(half, 1.0, -1.0)
    return torch.cat([x, -x.flip(1)], 1), g


@pytest.mark.parametrize("rows,width,xt,yt", [
    (300_001, 128, F32, F32), (300_001, 128, F32, BF16), (600_001, 128, BF16, BF16), (530_001, 64, F32, F32),
    (1_100_001, 16, F16, F16), (70_001, 512, F32, F32), (40_001, 1024, F32, F32), (40_001, 2048, BF16, BF16),
    (9_001, 4096, F32, F16), (3_001, 16384, F32, F32), (20_001, 256, F32, F32)])
def test_norms_are_exact(torch_cuda, rows, width, xt, yt):
    print(f"layer_norm {rows} x {width} {xt} {yt}", flush=True)
    x, g = _signs(rows, width, rows)
    w = torch.tensor([0.5, 1.0, 2.0, -1.0], device="cuda:0").repeat(width)[:width]
    b = torch.randint(-3, 4, (width,), generator=g, device="cuda:0").float()
    dy = torch.randint(-2, 3, (rows, width), generator=g, device="cuda:0").float()
    leaves = [x.to(xt).requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
    y = T.layer_norm(*leaves, eps=0.0, out_dtype=yt)
    assert torch.equal(y.detach(), (x * w + b).to(yt))
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(yt))
    assert torch.equal(db, dy.sum(0, dtype=torch.float64).float())
    assert torch.equal(dw, (dy * x).sum(0, dtype=torch.float64).float())
    gw = dy * w  # means over a power of two of multiples of a half: exact in fp32
    want = gw - gw.mean(1, keepdim=True) - x * (gw * x).mean(1, keepdim=True)
    assert torch.equal(dx, want.to(xt))


@pytest.mark.parametrize("rows,width,dtype", [(300_001, 100, F32), (50_001, 704, F32), (1_000_001, 47, F16), (30_001, 2049, F16),
                                              (30_001, 1500, BF16), (3_001, 12289, F32)])
def test_norms_of_random_rows(torch_cuda, rows, width, dtype):
    """The bits of small calls, row block by row block, at large calls' launches."""
    print(f"layer_norm {rows} x {width} {dtype}", flush=True)
    g = torch.Generator(device="cuda:0").manual_seed(rows)
    x = torch.randn(rows, width, generator=g, device="cuda:0").to(dtype).requires_grad_()
    w = (1 + 0.2 * torch.randn(width, generator=g, device="cuda:0")).requires_grad_()
    b = torch.randn(width, generator=g, device="cuda:0").requires_grad_()
    dy = torch.randint(-2, 3, (rows, width), generator=g, device="cuda:0").to(dtype)
    y = T.layer_norm(x, w, b)
    dx, _, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(db, dy.sum(0, dtype=torch.float64).float())
    size = max(60, rows // 100)
    for k in range(0, rows, size):
        part = x.detach()[k:k + size].clone().requires_grad_()
        small = T.layer_norm(part, w, b)
        assert torch.equal(small.detach(), y.detach()[k:k + size]), k
        assert torch.equal(torch.autograd.grad(small, part, dy[k:k + size])[0], dx[k:k + size]), k

"""The vocabulary loss of a few rows on the CUDA cores, row by row to within f32 sums, and the target's logit of many rows on
the tensor cores row by row.

A logit on the CUDA cores is a chain of at most width / 8 fused multiply-adds in each of several lanes, and a tree. Each
addition rounds its partial sum by 2^-24 of it at most, in either direction; partial sums of products of either sign are of
the size of their root mean square times the root of their number, L = |h * w| (the norm of the row of products). The
roundings of n additions add up to about sqrt(n) 2^-24 L / 4 then; 16 2^-24 L leaves a factor of three at 4,096 columns. The
logarithm of the sum adds a few roundings of its own value."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200 import _ffi  # noqa: E402
from staleynet_b200.matmul import Storage, last_path  # noqa: E402
from test_vocabulary_loss_gpu import BF16, F32, _case, _reference, _run  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("rows,dtype", [(n, F32) for n in (1, 2, 3, 4, 5, 16)] + [(n, BF16) for n in (1, 2, 3, 4)])
def test_each_loss_of_a_few_rows(rows, dtype, storage):
    for width, classes, first in ((768, 3001, 1), (771, 2049, 0), (256, 41, 1), (5, 1, 0), (4096, 131, 3), (4095, 20011, 0)):
        hidden, weight, targets = _case(rows, width, classes, dtype, storage, seed=rows + width)
        whole = torch.full((weight.shape[0], weight.shape[1] + first), float("nan"), device="cuda", dtype=dtype)
        weight = whole[:, first:].copy_(weight)
        losses_e, lse, *_ = _reference(hidden, weight, targets, storage, 1.0)
        losses, _ = _run(hidden, weight, targets, storage)
        assert last_path() == _ffi.PATH_SIMT
        w = weight.double() if storage is Storage.TRANSPOSED else weight.double().t()
        size = (hidden.double().square() @ w.square().t()).amax(1).sqrt()
        error = (losses.double() - losses_e).abs()
        assert bool((error <= 16 * 2.0 ** -24 * (size + lse.abs() + 1)).all()), (width, classes, error.max().item())


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("width", [1024, 1003])
def test_each_loss_whose_target_is_far_from_zero(width, dtype, storage):
    """As the test of means of that name, row by row: every class's logit but the target's may lose 2^-23 of its partial sum
    at each instruction (8 or 16 products), and each counts with its share of the probability."""
    rows, classes, per = 300, 20011, 8 if dtype == F32 else 16
    g = torch.Generator(device="cuda").manual_seed(width)
    w = torch.randn(classes, width, generator=g, device="cuda") * width ** -0.5
    targets = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    hidden = (torch.randn(rows, width, generator=g, device="cuda") + 9.0 * w[targets.long()]).to(dtype)
    weight = (w if storage is Storage.TRANSPOSED else w.t().contiguous()).to(dtype)
    losses_e, lse, *_ = _reference(hidden, weight, targets, storage, 1.0)
    h, v = hidden.double(), (weight if storage is Storage.TRANSPOSED else weight.t()).double()
    z, lost = torch.zeros(rows, classes, device="cuda", dtype=torch.float64), 0.0
    for k in range(0, width, per):   # the partial sums after each instruction
        z += h[:, k:k + per] @ v[:, k:k + per].t()
        lost = lost + 2.0 ** -23 * z.abs()
    at = targets.long()[:, None]
    share = torch.exp(z - lse[:, None]).scatter_(1, at, 0.0)
    bound = (share * lost).sum(1) + 8 * 2.0 ** -24 * (lse.abs() + z.gather(1, at)[:, 0].abs())
    losses, _ = _run(hidden, weight, targets, storage)
    error = (losses.double() - losses_e).abs()
    assert bool((error <= bound).all()), (error / bound).max().item()

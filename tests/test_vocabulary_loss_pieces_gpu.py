"""The vocabulary loss where the vocabulary has to be taken in several pieces: a piece of p is bounded by 768 MB, a packed
piece of the weight by 256 MB. Each case shows by its workspace that its arrays are not held whole. Bounds as in
test_vocabulary_loss_gpu.py; the longer sums of f32 rows are added up in lengths of 256, whose own error is that of the
shorter ones there."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import Gpu, Storage, WriteMode  # noqa: E402
from test_vocabulary_loss_gpu import BF16, F32, GRAD_TOLERANCE, _case, _check, _close, _reference, _run  # noqa: E402

pytestmark = pytest.mark.gpu

STORAGES = pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())


def _need(hidden, weight, storage, gradients=True):
    grads = {"d_hidden": torch.empty_like(hidden), "d_weight": torch.empty_like(weight)} if gradients else {}
    return Gpu(0).vocabulary_cross_entropy_workspace(hidden, weight, storage=storage, **grads)


# Pieces of 2,816, 2,816 and 1,369 classes; of 3,072, 3,072 and 856, the first two with enough tiles for the weight gradient
# to be stored where the caller wants it; of 1,280, 1,280 and 441, with f32 rows of whole 16-byte pieces and without.
@STORAGES
@pytest.mark.parametrize("rows,width,classes,dtype", [(131073, 40, 7001, BF16), (131072, 1024, 7000, BF16),
                                                      (65537, 36, 3001, F32), (65537, 37, 3001, F32)])
def test_pieces_of_p(rows, width, classes, dtype, storage):
    hidden, weight, targets = _case(rows, width, classes, dtype, storage, seed=1)
    assert _need(hidden, weight, storage) < rows * classes * (2 if dtype == BF16 else 8)
    _check(hidden, weight, targets, storage)


@STORAGES
@pytest.mark.parametrize("rows,width,classes,dtype", [(40, 768, 60001, F32), (33, 1003, 140001, BF16), (130, 1003, 140001, BF16)])
def test_pieces_of_a_packed_weight(rows, width, classes, dtype, storage):
    hidden, weight, targets = _case(rows, width, classes, dtype, storage, seed=2)
    whole = classes * width * (2 if dtype == BF16 else 12)
    assert _need(hidden, weight, storage, gradients=False) < whole
    _check(hidden, weight, targets, storage)


@STORAGES
@pytest.mark.parametrize("rows,width,classes,dtype", [(131073, 40, 7001, BF16), (65537, 37, 3001, F32), (65537, 36, 3001, F32)])
def test_one_gradient_accumulation_and_order_over_pieces(rows, width, classes, dtype, storage):
    hidden, weight, targets = _case(rows, width, classes, dtype, storage, seed=3)
    *_, dh_e, dw_e = _reference(hidden, weight, targets, storage, 0.5)
    dh = torch.full_like(hidden, float("nan"))
    _run(hidden, weight, targets, storage, d_hidden=dh, grad_scale=0.5)
    _close(dh, dh_e, GRAD_TOLERANCE[dtype])
    start = torch.randn(weight.shape, device="cuda")
    dw = start.clone()
    _run(hidden, weight, targets, storage, d_weight=dw, grad_scale=0.5, write=WriteMode.ACCUMULATE)
    _close(dw - start, dw_e, GRAD_TOLERANCE[dtype] + 1e-6 * start.norm().item() / dw_e.norm().item())
    runs = []
    for _ in range(2):
        dh, dw = torch.full_like(hidden, float("nan")), torch.full_like(weight, float("nan"))
        losses, total = _run(hidden, weight, targets, storage, d_hidden=dh, d_weight=dw, grad_scale=0.5, deterministic=True)
        runs.append((dh, dw, losses, total))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    _close(runs[0][0], dh_e, GRAD_TOLERANCE[dtype])
    _close(runs[0][1], dw_e, GRAD_TOLERANCE[dtype])
    alias = hidden.clone()
    _run(alias, weight, targets, storage, d_hidden=alias, grad_scale=0.5)
    _close(alias, dh_e, GRAD_TOLERANCE[dtype])

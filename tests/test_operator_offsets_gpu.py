"""Layer norm and the vocabulary loss on tensors whose rows lie more than 2^32 bytes, and 2^31 elements, apart from the first."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import Gpu, Storage  # noqa: E402
from test_layer_norm_gpu import BF16, F32, TOLERANCE, _backward_reference, _forward_reference, _inputs, _near  # noqa: E402
from test_vocabulary_loss_gpu import GRAD_TOLERANCE, _case, _close, _reference, _run  # noqa: E402

pytestmark = pytest.mark.gpu


def _far(t, shift):
    """The rows of t 2^30 + 8 elements apart, in a buffer that ends with the last one."""
    rows, cols = t.shape
    stride = (1 << 30) + 8 + shift
    whole = torch.empty((rows - 1) * stride + cols, device="cuda", dtype=t.dtype)
    return torch.as_strided(whole, (rows, cols), (stride, 1)).copy_(t)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cols,shift", [(640, 0), (640, 3), (20000, 0)])
def test_layer_norm(cols, shift, dtype):
    x, dy, gain, bias = _inputs(4, cols, dtype, dtype)
    gpu = Gpu(0)
    xs, ys, dys = _far(x, shift), _far(x, shift), _far(dy, shift)
    mean, inv = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    gpu.layer_norm_forward(xs, gain, bias, ys, mean, inv, 1e-5)
    _near(ys, _forward_reference(x, gain, bias, 1e-5)[0], TOLERANCE[dtype])
    dg, db = torch.empty_like(gain), torch.empty_like(gain)
    workspace = torch.empty(gpu.layer_norm_workspace(4, cols), device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(dys, xs, gain, mean, inv, ys, dg, db, workspace)
    dx_e, dg_e, db_e, dg_size, db_size = _backward_reference(x, dy, gain, mean, inv)
    _near(ys, dx_e, TOLERANCE[dtype])
    assert bool(((dg.double() - dg_e).abs() <= TOLERANCE[F32] * dg_size).all())
    assert bool(((db.double() - db_e).abs() <= TOLERANCE[F32] * db_size).all())


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("far,shift", [("hidden", 0), ("hidden", 1), ("weight", 0), ("weight", 1)])
def test_vocabulary_loss(far, shift, dtype, storage):
    rows, width, classes = (5, 40, 300) if far == "hidden" else (200, 5, 4)
    if far == "weight" and storage is Storage.ROW_MAJOR:
        width, classes = 4, 5
    hidden, weight, targets = _case(rows, width, classes, dtype, storage, seed=3)
    losses_e, _, _, dh_e, dw_e = _reference(hidden, weight, targets, storage, 0.5)
    h, w = (_far(hidden, shift), weight) if far == "hidden" else (hidden, _far(weight, shift))
    dh, dw = torch.empty_like(hidden), torch.empty_like(weight)
    alone, _ = _run(h, w, targets, storage)
    losses, _ = _run(h, w, targets, storage, d_hidden=dh, d_weight=dw, grad_scale=0.5)
    _close(alone, losses_e, 1e-5)
    _close(losses, losses_e, 1e-5)
    _close(dh, dh_e, GRAD_TOLERANCE[dtype])
    _close(dw, dw_e, GRAD_TOLERANCE[dtype])

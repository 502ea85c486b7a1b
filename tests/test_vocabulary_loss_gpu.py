"""The vocabulary's softmax cross entropy (snb_vocabulary_cross_entropy) against its definition in 64 bits.

Tolerances. A logit is an f32 sum of `width` exact products on the tensor core, rounded once for each instruction's 8
(TF32) or 16 (bf16) of them: at most (width / 8 + 8) 2^-23 of the sum of the products' absolute values; the log-sum-exp
adds a few roundings of its own value (8 x 2^-23). The gradients are compared by their Frobenius norms: bf16 operands
round p and the result once each (at most 2^-8 each), f32 ones lose 2^-21 a product and the sums' roundings, which add up
to less than 2e-5 at the lengths here."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200 import _ffi  # noqa: E402
from staleynet_b200.matmul import Gpu, OperandTooSmall, SnbError, Storage, WriteMode, last_path  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
GRAD_TOLERANCE = {F32: 2e-5, BF16: 2 * 2.0 ** -8}


def _case(rows, width, classes, dtype, storage, seed=0, missing=0.2, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = (torch.randn(rows, width, generator=g, device="cuda") * scale).to(dtype)
    weight = (torch.randn(classes, width, generator=g, device="cuda") * width ** -0.5).to(dtype)
    targets = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if rows > 1:
        targets[torch.rand(rows, generator=g, device="cuda") < missing] = -1
    if storage is Storage.ROW_MAJOR:
        weight = weight.t().contiguous()
    return hidden, weight, targets


def _reference(hidden, weight, targets, storage, grad_scale):
    w = weight.double() if storage is Storage.TRANSPOSED else weight.double().t()
    h, live = hidden.double(), targets >= 0
    h = torch.where(live[:, None], h, 0.0)
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    at = targets.long().clamp(min=0)[:, None]
    losses = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    p = torch.exp(z - lse[:, None])
    p.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float64))
    p[~live] = 0.0
    dw = grad_scale * (p.t() @ h)
    size = (h.abs() @ w.abs().t()).amax(1)   # the largest sum of absolute products of the row's logits
    return losses, lse, size, grad_scale * (p @ w), dw if storage is Storage.TRANSPOSED else dw.t()


def _run(hidden, weight, targets, storage, *, d_hidden=None, d_weight=None, gpu=None, **more):
    gpu = gpu or Gpu(0)
    losses = torch.full((hidden.shape[0],), float("nan"), device="cuda")
    total = torch.full((), float("nan"), device="cuda")
    need = gpu.vocabulary_cross_entropy_workspace(hidden, weight, storage=storage, d_hidden=d_hidden, d_weight=d_weight)
    # Whatever the workspace holds must not show: NaN in every type.
    workspace = torch.full((need,), 0xFF, device="cuda", dtype=torch.uint8)
    gpu.vocabulary_cross_entropy(hidden, weight, targets, losses, total, workspace, storage=storage,
                                 d_hidden=d_hidden, d_weight=d_weight, **more)
    gpu.synchronize()
    gpu.device_status()
    return losses, total


def _close(got, expected, tolerance):
    error = (got.double() - expected).norm().item()
    assert error <= tolerance * expected.norm().item() + 1e-30, (error, expected.norm().item())


def _check(hidden, weight, targets, storage, grad_scale=0.37):
    dtype, width = hidden.dtype, hidden.shape[1]
    losses_e, lse, size, dh_e, dw_e = _reference(hidden, weight, targets, storage, grad_scale)
    dh = torch.full_like(hidden, float("nan")).contiguous()
    dw = torch.full(weight.shape, float("nan"), device="cuda", dtype=dtype)
    only, only_total = _run(hidden, weight, targets, storage)
    losses, total = _run(hidden, weight, targets, storage, d_hidden=dh, d_weight=dw, grad_scale=grad_scale)
    bound = (width / 8 + 8) * 2.0 ** -23 * 2 * size + 8 * 2.0 ** -23 * (lse.abs() + 1)
    for got, got_total in ((only, only_total), (losses, total)):
        assert bool(((got.double() - losses_e).abs() <= bound).all())
        assert abs(got_total.double() - losses_e.sum()) <= bound.sum() + 2.0 ** -23 * losses_e.sum()
    assert bool((losses[targets < 0] == 0).all())
    _close(dh, dh_e, GRAD_TOLERANCE[dtype])
    _close(dw, dw_e, GRAD_TOLERANCE[dtype])


SHAPES = [
    (1, 64, 1000), (1, 8, 1), (3, 1, 5), (2, 7, 257), (31, 768, 999), (127, 33, 128), (128, 64, 256), (129, 72, 255),
    (257, 256, 2049), (300, 99, 1003), (1000, 130, 513), (513, 512, 4096), (40, 1024, 3001), (1024, 64, 8),
]


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,width,classes", SHAPES)
def test_losses_and_gradients(rows, width, classes, dtype, storage):
    _check(*_case(rows, width, classes, dtype, storage, seed=rows + classes), storage)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,width,classes", [(300, 256, 1003), (40, 99, 513), (513, 64, 200)])
def test_the_hidden_gradient_may_replace_the_hidden_rows(rows, width, classes, dtype):
    hidden, weight, targets = _case(rows, width, classes, dtype, Storage.TRANSPOSED, seed=rows)
    hidden = hidden.contiguous()
    losses_e, _, _, dh_e, dw_e = _reference(hidden, weight, targets, Storage.TRANSPOSED, 0.5)
    dw = torch.full(weight.shape, float("nan"), device="cuda", dtype=dtype)
    losses, _ = _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=hidden, d_weight=dw, grad_scale=0.5)
    _close(losses, losses_e, 1e-5)
    _close(hidden, dh_e, GRAD_TOLERANCE[dtype])
    _close(dw, dw_e, GRAD_TOLERANCE[dtype])


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("width", [1024, 1003])
def test_a_target_far_from_zero_costs_no_accuracy(width, dtype, storage):
    """A matrix instruction (8 products of f32 operands, 16 of bf16) loses up to 2^-24 of its sum towards zero. That may show
    in the other classes' logits, weighted with their shares, but not in a target's logit, which is several times larger."""
    rows, classes = 300, 20011
    g = torch.Generator(device="cuda").manual_seed(width)
    w = torch.randn(classes, width, generator=g, device="cuda") * width ** -0.5
    targets = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    hidden = (torch.randn(rows, width, generator=g, device="cuda") + 9.0 * w[targets.long()]).to(dtype)
    weight = (w if storage is Storage.TRANSPOSED else w.t().contiguous()).to(dtype)
    losses_e, lse, *_ = _reference(hidden, weight, targets, storage, 1.0)
    z = hidden.double() @ (weight.double().t() if storage is Storage.TRANSPOSED else weight.double())
    at = targets.long()[:, None]
    share = torch.exp(z - lse[:, None]).scatter_(1, at, 0.0)
    instructions = width / (8 if dtype == F32 else 16)
    bound = instructions * 2.0 ** -24 * (share * z.abs()).sum(1) + 4 * 2.0 ** -24 * (lse.abs() + z.gather(1, at)[:, 0].abs())
    dh = torch.empty_like(hidden)
    for more in ({}, {"d_hidden": dh}):
        losses, _ = _run(hidden, weight, targets, storage, **more)
        assert (losses.double() - losses_e).abs().mean() <= bound.mean()


@pytest.mark.parametrize("offset", [0, 1, 2])
def test_f32_gradients_that_start_off_16_bytes(offset):
    hidden, weight, targets = _case(700, 100, 1003, F32, Storage.TRANSPOSED, seed=offset)
    _, _, _, dh_e, dw_e = _reference(hidden, weight, targets, Storage.TRANSPOSED, 0.5)
    whole = [torch.full((t.numel() + 8,), float("nan"), device="cuda") for t in (hidden, weight)]
    dh, dw = (w[offset:offset + t.numel()].view(t.shape) for w, t in zip(whole, (hidden, weight)))
    _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh, d_weight=dw, grad_scale=0.5)
    _close(dh, dh_e, GRAD_TOLERANCE[F32])
    _close(dw, dw_e, GRAD_TOLERANCE[F32])
    for w, t in zip(whole, (hidden, weight)):
        assert bool(w[:offset].isnan().all()) and bool(w[offset + t.numel():].isnan().all())


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 16, 17])
def test_the_loss_of_a_few_rows(rows, dtype, storage):
    """Alone, over weights that the tensor cores can read and ones that they cannot (odd row lengths, off a boundary)."""
    for width, classes, first in ((768, 3001, 0), (771, 2048, 0), (256, 40, 1), (5, 1, 0), (4096, 130, 0), (4100, 77, 3)):
        hidden, weight, targets = _case(rows, width, classes, dtype, storage, seed=rows)
        whole = torch.full((weight.shape[0], weight.shape[1] + first), float("nan"), device="cuda", dtype=dtype)
        weight = whole[:, first:].copy_(weight)
        losses_e, lse, size, *_ = _reference(hidden, weight, targets, storage, 1.0)
        losses, total = _run(hidden, weight, targets, storage)
        bound = (width / 8 + 8) * 2.0 ** -23 * 2 * size + 8 * 2.0 ** -23 * (lse.abs() + 1)
        assert bool(((losses.double() - losses_e).abs() <= bound).all())
        assert abs(total.double() - losses_e.sum()) <= bound.sum() + 2.0 ** -23 * losses_e.sum()


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("rows,width,classes,dtype", [(8192, 40, 40001, BF16), (4096, 36, 20003, F32)])
def test_a_vocabulary_of_several_pieces(rows, width, classes, dtype, storage):
    _check(*_case(rows, width, classes, dtype, storage, seed=5), storage)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_strided_and_unaligned_operands(rows, dtype):
    hidden, weight, targets = _case(rows, 96, 1000, dtype, Storage.TRANSPOSED)
    for pad, first in ((8, 0), (5, 0), (8, 1), (3, 2)):
        wide_h = torch.full((rows, 96 + pad), float("nan"), device="cuda", dtype=dtype)
        wide_w = torch.full((1000, 96 + pad), float("nan"), device="cuda", dtype=dtype)
        h, w = wide_h[:, first:first + 96], wide_w[:, first:first + 96]
        h.copy_(hidden)
        w.copy_(weight)
        _check(h, w, targets, Storage.TRANSPOSED)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rows_without_a_target_may_hold_anything(dtype):
    hidden, weight, targets = _case(200, 64, 700, dtype, Storage.TRANSPOSED)
    hidden[targets < 0] = float("nan")
    hidden[(targets < 0).nonzero()[0]] = float("inf")
    _check(hidden, weight, targets, Storage.TRANSPOSED)
    alone = torch.empty_like(hidden)
    _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=alone)
    assert bool(alone.isfinite().all()) and not alone[targets < 0].any()
    targets.fill_(-1)
    dh, dw = torch.ones_like(hidden), torch.ones_like(weight)
    losses, total = _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh, d_weight=dw)
    assert not losses.any() and total == 0 and not dh.any() and not dw.any()


def test_a_target_that_is_no_class_gives_nan_in_its_row_alone():
    hidden, weight, targets = _case(70, 64, 500, BF16, Storage.TRANSPOSED, missing=0.0)
    targets[11] = 500
    dh = torch.zeros_like(hidden)
    losses, total = _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh)
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[11] = True
    assert bool((losses.isnan() == bad).all()) and bool(total.isnan())
    assert bool((dh.isnan().all(1) == bad).all()) and bool((dh.isnan().any(1) == bad).all())


@pytest.mark.parametrize("scale", [0.0, 1e-3, 300.0])
def test_flat_and_peaked_distributions(scale):
    """Equal logits, and logits whose spread (hundreds) leaves one class with all the probability."""
    _check(*_case(150, 64, 3000, F32, Storage.TRANSPOSED, scale=scale), Storage.TRANSPOSED)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_classes_whose_logits_are_minus_infinity(dtype):
    """The first 300 classes are masked out (more than a whole tile's half), the others have very negative logits."""
    hidden, weight, targets = _case(140, 64, 900, dtype, Storage.TRANSPOSED)
    hidden[:, 0], weight[:, 0] = 16.0, -40.0
    masked = weight.clone()
    masked[:300, 0] = -3e38
    targets = torch.where(targets >= 0, 300 + targets % 600, targets)
    dw = torch.empty_like(weight)
    losses, _ = _run(hidden, masked, targets, Storage.TRANSPOSED, d_hidden=None, d_weight=dw)
    moved = torch.where(targets >= 0, targets - 300, targets)
    expected, lse, size, _, dw_e = _reference(hidden, weight[300:], moved, Storage.TRANSPOSED, 1.0)
    bound = (64 / 8 + 8) * 2.0 ** -23 * 2 * size + 8 * 2.0 ** -23 * (lse.abs() + 1)
    assert bool(((losses.double() - expected).abs() <= bound).all())
    assert not dw[:300].any()
    _close(dw[300:], dw_e, GRAD_TOLERANCE[dtype])


def test_no_rows():
    weight = torch.randn(100, 16, device="cuda")
    hidden, targets = torch.empty(0, 16, device="cuda"), torch.empty(0, device="cuda", dtype=torch.int32)
    dw = torch.ones_like(weight)
    _, total = _run(hidden, weight, targets, Storage.TRANSPOSED, d_weight=dw)
    assert total == 0 and not dw.any() and last_path() == _ffi.PATH_EMPTY


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
def test_the_weight_gradient_is_added_to_an_f32_tensor(storage, dtype):
    for classes in (700, 701):
        hidden, weight, targets = _case(333, 72, classes, dtype, storage)
        *_, dw_e = _reference(hidden, weight, targets, storage, 2.0)
        start = torch.randn(weight.shape, device="cuda")
        dw = start.clone()
        _run(hidden, weight, targets, storage, d_weight=dw, grad_scale=2.0, write=WriteMode.ACCUMULATE)
        _close(dw - start, dw_e, GRAD_TOLERANCE[dtype] + 1e-6 * start.norm().item() / dw_e.norm().item())


def test_one_gradient_alone_equals_the_same_gradient_of_both():
    hidden, weight, targets = _case(300, 128, 1500, BF16, Storage.TRANSPOSED)
    both_h, both_w = torch.empty_like(hidden), torch.empty_like(weight)
    one_h, one_w = torch.empty_like(hidden), torch.empty_like(weight)
    for dh, dw in ((both_h, both_w), (one_h, None), (None, one_w)):
        _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh, d_weight=dw, deterministic=True)
    assert torch.equal(both_h, one_h) and torch.equal(both_w, one_w)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_deterministic_gradients_are_bit_identical(dtype):
    hidden, weight, targets = _case(2048, 192, 3000, dtype, Storage.TRANSPOSED)
    *_, dh_e, dw_e = _reference(hidden, weight, targets, Storage.TRANSPOSED, 1.0)
    runs = []
    for _ in range(3):
        dh, dw = torch.empty(hidden.shape, device="cuda"), torch.empty(weight.shape, device="cuda")
        losses, total = _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh, d_weight=dw, deterministic=True)
        runs.append((dh, dw, losses, total))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    _close(runs[0][0], dh_e, GRAD_TOLERANCE[dtype])
    _close(runs[0][1], dw_e, GRAD_TOLERANCE[dtype])


def test_gradients_against_differences():
    """Along its own direction the loss changes by the gradient's norm: central differences of f32 losses (error about
    1e-6 a row) with a step of 2e-2, whose own error is of third order."""
    hidden, weight, targets = _case(37, 24, 301, F32, Storage.TRANSPOSED)
    dh, dw = torch.empty_like(hidden), torch.empty_like(weight)
    _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh, d_weight=dw)
    for grad, at in ((dh, 0), (dw, 1)):
        norm = grad.double().norm().item()
        ends = []
        for sign in (1, -1):
            moved = [hidden, weight]
            moved[at] = moved[at] + sign * 2e-2 * grad / norm
            ends.append(_run(*moved, targets, Storage.TRANSPOSED)[0].double().sum().item())
        assert abs((ends[0] - ends[1]) / 4e-2 - norm) <= 2e-3 * norm


def test_another_stream():
    hidden, weight, targets = _case(256, 64, 2000, BF16, Storage.TRANSPOSED)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    dh = torch.empty_like(hidden)
    gpu = Gpu(0, stream)
    with torch.cuda.stream(stream):
        losses, _ = _run(hidden, weight, targets, Storage.TRANSPOSED, d_hidden=dh, gpu=gpu)
    expected, *_ = _reference(hidden, weight, targets, Storage.TRANSPOSED, 1.0)
    assert (losses.double() - expected).abs().max() < 1e-4


def test_refusals():
    gpu = Gpu(0)
    hidden, weight, targets = _case(10, 32, 50, BF16, Storage.TRANSPOSED)
    losses, total = torch.zeros(10, device="cuda"), torch.zeros((), device="cuda")
    dw = torch.empty_like(weight)
    need = gpu.vocabulary_cross_entropy_workspace(hidden, weight, d_weight=dw)
    workspace = torch.empty(need, device="cuda", dtype=torch.uint8)
    call = gpu.vocabulary_cross_entropy
    with pytest.raises(SnbError, match="needs"):
        call(hidden, weight, targets, losses, total, workspace[:-1], d_weight=dw)
    with pytest.raises(SnbError, match="too few targets"):
        call(hidden, weight, targets[:9], losses, total, workspace)
    with pytest.raises(OperandTooSmall, match="losses too small"):
        call(hidden, weight, targets, losses[:9], total, workspace)
    with pytest.raises(SnbError, match="accumulating into a bf16 gradient"):
        call(hidden, weight, targets, losses, total, workspace, d_weight=dw, write=WriteMode.ACCUMULATE)
    with pytest.raises(SnbError, match="int32"):
        call(hidden, weight, targets.long(), losses, total, workspace)
    with pytest.raises(AssertionError, match="weight shape"):
        call(hidden, weight[:, :31], targets, losses, total, workspace)
    with pytest.raises(SnbError, match="rows must be contiguous"):
        call(hidden, weight.t().contiguous().t(), targets, losses, total, workspace)
    with pytest.raises(AssertionError, match="weight_grad"):
        call(hidden, weight, targets, losses, total, workspace, d_weight=dw[:49])
    with pytest.raises(SnbError, match="f32 operands have f32 gradients"):
        call(hidden.float(), weight.float(), targets, losses, total, workspace, d_weight=dw)
    with pytest.raises(SnbError, match="CUDA device memory"):
        call(hidden, weight, targets.cpu(), losses, total, workspace)

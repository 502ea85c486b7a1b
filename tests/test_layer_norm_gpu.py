"""Layer norm's forward and backward pass (snb_layer_norm_forward, snb_layer_norm_backward) against the formulas in 64
bits.

Tolerances, as relative Frobenius norms. Every value passes a handful of f32 roundings (2^-24 each) and sums whose
roundings partly cancel: f32 results are held to 4e-6 (about 64 roundings), bf16 ones to one rounding of at most 2^-8.
The sums over the rows, of terms of either sign, are held to 4e-6 of the sum of the terms' absolute values, column by
column."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200 import _ffi  # noqa: E402
from staleynet_b200.matmul import Gpu, SnbError, WriteMode, last_path  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOLERANCE = {F32: 4e-6, BF16: 2.0 ** -8}


def _inputs(rows, cols, x_type, dy_type, seed=0, mean=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * 2 + mean).to(x_type)
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(dy_type)
    gain = torch.randn(cols, generator=g, device="cuda") * 0.3 + 1
    bias = torch.randn(cols, generator=g, device="cuda")
    return x, dy, gain, bias


def _forward_reference(x, gain, bias, epsilon):
    x = x.double()
    mean = x.mean(1)
    inv = ((x - mean[:, None]).square().mean(1) + epsilon).rsqrt()
    y = (x - mean[:, None]) * inv[:, None] * gain.double()
    return y if bias is None else y + bias.double(), mean, inv


def _backward_reference(x, dy, gain, mean, inv):
    x, dy, inv = x.double(), dy.double(), inv.double()[:, None]
    n = (x - mean.double()[:, None]) * inv
    d = dy * gain.double()
    dx = inv * (d - d.mean(1, keepdim=True) - n * (d * n).mean(1, keepdim=True))
    return dx, (dy * n).sum(0), dy.sum(0), (dy * n).abs().sum(0), dy.abs().sum(0)


def _near(got, expected, tolerance, floor=0.0):
    error = (got.double() - expected).norm().item()
    assert error <= tolerance * expected.norm().item() + floor, (error, expected.norm().item())


def _check(x, dy, gain, bias, out_type, epsilon=1e-5):
    rows, cols = x.shape
    gpu = Gpu(0)
    out = torch.full((rows, cols), float("nan"), device="cuda", dtype=out_type)
    mean, inv = torch.full((rows,), float("nan"), device="cuda"), torch.full((rows,), float("nan"), device="cuda")
    gpu.layer_norm_forward(x, gain, bias, out, mean, inv, epsilon)
    dx = torch.full_like(x, float("nan"))
    dg, db = torch.full_like(gain, float("nan")), torch.full_like(gain, float("nan"))
    workspace = torch.full((gpu.layer_norm_workspace(rows, cols),), 0xFF, device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(dy, x, gain, mean, inv, dx, dg, db, workspace)
    torch.cuda.synchronize()
    y_e, mean_e, inv_e = _forward_reference(x, gain, bias, epsilon)
    size = x.double().norm().item()
    _near(mean, mean_e, TOLERANCE[F32], TOLERANCE[F32] * size / cols ** 0.5)
    _near(inv, inv_e, TOLERANCE[F32])
    _near(out, y_e, TOLERANCE[out_type])
    dx_e, dg_e, db_e, dg_size, db_size = _backward_reference(x, dy, gain, mean, inv)
    # What a row's gradient cancels (all of it in a row of one column) leaves roundings of its terms.
    _near(dx, dx_e, TOLERANCE[x.dtype], TOLERANCE[F32] * (inv.double()[:, None] * dy.double() * gain.double()).norm())
    assert bool(((dg.double() - dg_e).abs() <= TOLERANCE[F32] * dg_size + 1e-30).all())
    assert bool(((db.double() - db_e).abs() <= TOLERANCE[F32] * db_size + 1e-30).all())


TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (F32, BF16, BF16), (BF16, F32, F32)]
# One row and column up to rows past every way of holding one; odd counts leave no row on a vector boundary.
SHAPES = [(1, 1), (3, 2), (1, 768), (5, 7), (9, 32), (33, 255), (64, 256), (17, 264), (100, 513), (700, 768), (31, 1000),
          (8, 1024), (7, 1025), (21, 1032), (40, 2048), (6, 2049), (300, 4096), (5, 5003), (4, 8192), (3, 8193),
          (5, 9000), (2, 16385), (3, 32768), (2, 40001)]


@pytest.mark.parametrize("types", TYPES, ids=["f32", "bf16", "f32-bf16", "bf16-f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(rows, cols, types):
    x_type, dy_type, out_type = types
    _check(*_inputs(rows, cols, x_type, dy_type, seed=rows * 31 + cols), out_type)


@pytest.mark.parametrize("cols", [64, 768, 1500, 6000])
def test_many_rows(cols):
    """Every warp or block of the backward grid has several rows, the last ones fewer."""
    _check(*_inputs(9001 if cols < 1000 else 1201, cols, BF16, BF16), BF16)


@pytest.mark.parametrize("types", TYPES[:2], ids=["f32", "bf16"])
def test_a_mean_far_from_zero(types):
    """The deviations are 1/2000 of the mean: squares minus squared mean would leave nothing of the variance in f32. The
    mean's own rounding (2^-24 of 1000, against deviations of 0.5) is part of the operator's f32 results."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = 1000.0 + 0.5 * torch.randn(64, 640, generator=g, device="cuda")
    gain, bias = torch.ones(640, device="cuda"), torch.zeros(640, device="cuda")
    out, mean, inv = torch.empty_like(x), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    Gpu(0).layer_norm_forward(x, gain, bias, out, mean, inv, 1e-5)
    y_e, _, inv_e = _forward_reference(x, gain, bias, 1e-5)
    _near(inv, inv_e, 1e-5)
    assert (out.double() - y_e).abs().max() <= 4 * 1000 * 2.0 ** -24 / 0.5


def test_equal_values_give_the_bias():
    x = torch.full((5, 300), 7.25, device="cuda")
    bias = torch.randn(300, device="cuda")
    out, mean, inv = torch.empty_like(x), torch.empty(5, device="cuda"), torch.empty(5, device="cuda")
    Gpu(0).layer_norm_forward(x, torch.randn(300, device="cuda"), bias, out, mean, inv, 1e-5)
    assert torch.equal(out, bias.expand(5, 300)) and bool((mean == 7.25).all())
    assert torch.allclose(inv, torch.full_like(inv, 1e-5 ** -0.5), rtol=1e-6)


def test_a_row_of_nan_or_infinity_stays_in_its_row():
    x, dy, gain, bias = _inputs(40, 300, F32, F32)
    x[7, 11], x[9, 0] = float("nan"), float("inf")
    out, mean, inv = torch.empty_like(x), torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    Gpu(0).layer_norm_forward(x, gain, bias, out, mean, inv, 1e-5)
    bad = out.isnan().any(1).nonzero().flatten().tolist()
    assert bad == [7, 9]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cols", [96, 1536, 9001])
@pytest.mark.parametrize("pad,first", [(8, 0), (8, 8), (5, 3)])
def test_strided_rows(cols, pad, first, dtype):
    x, dy, gain, bias = _inputs(37, cols, dtype, dtype)
    wide = [torch.full((37, cols + 2 * pad), 9.0, device="cuda", dtype=dtype) for _ in range(4)]
    xs, dys, outs, dxs = (w[:, first:first + cols] for w in wide)
    xs.copy_(x)
    dys.copy_(dy)
    gpu = Gpu(0)
    mean, inv = torch.empty(37, device="cuda"), torch.empty(37, device="cuda")
    dense = torch.empty_like(x)
    gpu.layer_norm_forward(x, gain, bias, dense, mean, inv, 1e-5)
    gpu.layer_norm_forward(xs, gain, bias, outs, mean, inv, 1e-5)
    dg, db = torch.empty_like(gain), torch.empty_like(gain)
    workspace = torch.empty(gpu.layer_norm_workspace(37, cols), device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(dys, xs, gain, mean, inv, dxs, dg, db, workspace)
    torch.cuda.synchronize()
    _near(outs, _forward_reference(x, gain, bias, 1e-5)[0], TOLERANCE[dtype])
    _near(dxs, _backward_reference(x, dy, gain, mean, inv)[0], TOLERANCE[dtype])
    for w in wide:   # nothing outside the rows was touched
        assert bool((w[:, :first] == 9).all()) and bool((w[:, first + cols:] == 9).all())


@pytest.mark.parametrize("cols", [300, 768, 5000, 10000])
def test_in_place(cols):
    x, dy, gain, bias = _inputs(50, cols, F32, F32)
    gpu = Gpu(0)
    mean, inv = torch.empty(50, device="cuda"), torch.empty(50, device="cuda")
    y = x.clone()
    gpu.layer_norm_forward(y, gain, bias, y, mean, inv, 1e-5)
    dx, dg, db = dy.clone(), torch.empty_like(gain), torch.empty_like(gain)
    workspace = torch.empty(gpu.layer_norm_workspace(50, cols), device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(dx, x, gain, mean, inv, dx, dg, db, workspace)
    torch.cuda.synchronize()
    _near(y, _forward_reference(x, gain, bias, 1e-5)[0], TOLERANCE[F32])
    dx_e, dg_e, db_e, dg_size, db_size = _backward_reference(x, dy, gain, mean, inv)
    _near(dx, dx_e, TOLERANCE[F32])
    assert bool(((dg.double() - dg_e).abs() <= TOLERANCE[F32] * dg_size).all())
    assert bool(((db.double() - db_e).abs() <= TOLERANCE[F32] * db_size).all())


@pytest.mark.parametrize("cols", [320, 3000, 8500])
def test_accumulation_absent_bias_and_repeatability(cols):
    x, dy, gain, _ = _inputs(500, cols, F32, F32)
    gpu = Gpu(0)
    out, mean, inv = torch.empty_like(x), torch.empty(500, device="cuda"), torch.empty(500, device="cuda")
    gpu.layer_norm_forward(x, gain, None, out, mean, inv, 1e-5)
    _near(out, _forward_reference(x, gain, None, 1e-5)[0], TOLERANCE[F32])
    workspace = torch.empty(gpu.layer_norm_workspace(500, cols), device="cuda", dtype=torch.uint8)
    dx, dg = torch.empty_like(x), torch.empty_like(gain)
    gpu.layer_norm_backward(dy, x, gain, mean, inv, dx, dg, None, workspace)
    again, start = torch.empty_like(gain), torch.randn_like(gain)
    added, db = start.clone(), torch.zeros_like(gain)
    gpu.layer_norm_backward(dy, x, gain, mean, inv, dx, again, db, workspace)
    gpu.layer_norm_backward(dy, x, gain, mean, inv, dx, added, db, workspace, WriteMode.ACCUMULATE)
    torch.cuda.synchronize()
    assert torch.equal(dg, again) and torch.equal(added, start + dg)
    _near(db, 2 * dy.double().sum(0), 1e-5)


def test_no_rows():
    gpu = Gpu(0)
    x, gain = torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda")
    stats = torch.empty(0, device="cuda")
    gpu.layer_norm_forward(x, gain, gain, x, stats, stats, 1e-5)
    assert last_path() == _ffi.PATH_EMPTY
    dg, db = torch.ones_like(gain), torch.ones_like(gain)
    workspace = torch.empty(0, device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(x, x, gain, stats, stats, x, dg, db, workspace, WriteMode.ACCUMULATE)
    assert bool((dg == 1).all())
    gpu.layer_norm_backward(x, x, gain, stats, stats, x, dg, db, workspace)
    torch.cuda.synchronize()
    assert not dg.any() and not db.any()


def test_gradients_against_differences():
    """L = sum(y w) moves along each gradient by its norm: central differences in 64 bits of the f32 outputs (error about
    1e-7 a value), a step of 1e-2."""
    x, dy, gain, bias = _inputs(23, 150, F32, F32)
    gpu = Gpu(0)
    out, mean, inv = torch.empty_like(x), torch.empty(23, device="cuda"), torch.empty(23, device="cuda")

    def loss(x, gain, bias):
        gpu.layer_norm_forward(x, gain, bias, out, mean, inv, 1e-5)
        return (out.double() * dy.double()).sum().item()

    loss(x, gain, bias)
    dx, dg, db = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
    workspace = torch.empty(gpu.layer_norm_workspace(23, 150), device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(dy, x, gain, mean, inv, dx, dg, db, workspace)
    for at, grad in enumerate((dx, dg, db)):
        norm = grad.double().norm().item()
        ends = []
        for sign in (1, -1):
            moved = [x, gain, bias]
            moved[at] = moved[at] + sign * 1e-2 * grad / norm
            ends.append(loss(*moved))
        assert abs((ends[0] - ends[1]) / 2e-2 - norm) <= 1e-3 * norm


def test_another_stream():
    x, dy, gain, bias = _inputs(300, 768, BF16, BF16)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    gpu = Gpu(0, stream)
    out, mean, inv = torch.empty_like(x), torch.empty(300, device="cuda"), torch.empty(300, device="cuda")
    gpu.layer_norm_forward(x, gain, bias, out, mean, inv, 1e-5)
    stream.synchronize()
    _near(out, _forward_reference(x, gain, bias, 1e-5)[0], TOLERANCE[BF16])


def test_refusals():
    gpu = Gpu(0)
    x, dy, gain, bias = _inputs(6, 40, F32, F32)
    out, mean, inv = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    with pytest.raises(SnbError, match="params length"):
        gpu.layer_norm_forward(x, gain[:39], bias, out, mean, inv, 1e-5)
    with pytest.raises(SnbError, match="mean and inv_std too small"):
        gpu.layer_norm_forward(x, gain, bias, out, mean[:5], inv, 1e-5)
    with pytest.raises(SnbError, match="epsilon is negative"):
        gpu.layer_norm_forward(x, gain, bias, out, mean, inv, -1.0)
    with pytest.raises(AssertionError, match="output shape"):
        gpu.layer_norm_forward(x, gain, bias, out[:5], mean, inv, 1e-5)
    with pytest.raises(SnbError, match="rows must be contiguous"):
        gpu.layer_norm_forward(x.t().contiguous().t(), gain, bias, out, mean, inv, 1e-5)
    with pytest.raises(SnbError, match="float32 or bfloat16"):
        gpu.layer_norm_forward(x.half(), gain, bias, out, mean, inv, 1e-5)
    with pytest.raises(SnbError, match="CUDA device memory"):
        gpu.layer_norm_forward(x.cpu(), gain, bias, out, mean, inv, 1e-5)
    workspace = torch.empty(gpu.layer_norm_workspace(6, 40) - 1, device="cuda", dtype=torch.uint8)
    with pytest.raises(SnbError, match="workspace holds"):
        gpu.layer_norm_backward(dy, x, gain, mean, inv, out, torch.empty_like(gain), None, workspace)
    with pytest.raises(SnbError, match="must have the input's dtype"):
        gpu.layer_norm_backward(dy, x, gain, mean, inv, out.bfloat16(), torch.empty_like(gain), None, workspace)

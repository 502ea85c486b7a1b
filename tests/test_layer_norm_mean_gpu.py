"""Layer norm of bf16 rows whose mean is far from zero. Tolerances as in test_layer_norm_gpu.py."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import Gpu  # noqa: E402
from test_layer_norm_gpu import BF16, _backward_reference, _forward_reference, _near  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [640, 1003, 2816, 9001])
def test_a_bf16_mean_far_from_zero(cols):
    """Values about 1,000 with deviations of 8, of which bf16 leaves multiples of 4: the variance still comes from the
    deviations. The mean, of values of 10 bits, is off by its roundings (2^-24 of 1,000 a few times) against 8."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = (1000.0 + 8.0 * torch.randn(64, cols, generator=g, device="cuda")).to(BF16)
    dy = torch.randn(64, cols, generator=g, device="cuda").to(BF16)
    gain, bias = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    gpu = Gpu(0)
    out = torch.empty(64, cols, device="cuda")
    mean, inv = torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    gpu.layer_norm_forward(x, gain, bias, out, mean, inv, 1e-5)
    y_e, _, inv_e = _forward_reference(x, gain, bias, 1e-5)
    _near(inv, inv_e, 1e-5)
    assert (out.double() - y_e).abs().max() <= 16 * 1000 * 2.0 ** -24 / 8
    dx, dg, db = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
    workspace = torch.empty(gpu.layer_norm_workspace(64, cols), device="cuda", dtype=torch.uint8)
    gpu.layer_norm_backward(dy, x, gain, mean, inv, dx, dg, db, workspace)
    torch.cuda.synchronize()
    dx_e, dg_e, db_e, dg_size, db_size = _backward_reference(x, dy, gain, mean, inv)
    _near(dx, dx_e, 2.0 ** -8)
    assert bool(((dg.double() - dg_e).abs() <= 4e-6 * dg_size).all())
    assert bool(((db.double() - db_e).abs() <= 4e-6 * db_size).all())

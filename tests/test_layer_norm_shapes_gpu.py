"""Layer norm at the lengths where the way of holding a row changes, on and off 16-byte boundaries.
Tolerances as in test_layer_norm_gpu.py."""
import pytest

torch = pytest.importorskip("torch")

from test_layer_norm_gpu import TYPES, _check, _inputs  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", TYPES, ids=["f32", "bf16", "f32-bf16", "bf16-f32"])
@pytest.mark.parametrize("cols", [256, 257, 512, 776, 1016, 2052, 2816, 2999, 3080, 4104, 4403, 5120, 5121, 6136, 6145, 8184])
def test_rows_of_every_way_of_holding_one(cols, types):
    """700 rows: every block of the backward pass has two, some three."""
    x_type, dy_type, out_type = types
    _check(*_inputs(700, cols, x_type, dy_type, seed=cols), out_type)

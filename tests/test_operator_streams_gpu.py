"""The 8-bit AdamW plan and the output layer on a stream that is not the current one while they are made: their own tensors
are ready when the first call on that stream reads them, however busy either stream is."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.adamw8 import AdamW8, AdamW8Tensor, adamw8_state  # noqa: E402
from staleynet_b200.matmul import AdamWHyperparameters, Gpu  # noqa: E402

pytestmark = pytest.mark.gpu

BUSY = 200_000_000   # clocks, about 0.1 s


def _step(plan):
    plan.step(AdamWHyperparameters(1e-2, 0.9, 0.95, 1e-8, 0.0, 1), float("inf"), 1)


def test_adamw8_on_a_stream_of_its_own():
    parameter, gradient = torch.ones(3000, device="cuda"), torch.full((3000,), 2.0, device="cuda")
    tensors = [AdamW8Tensor(parameter, gradient, *adamw8_state(parameter))]
    gpu = Gpu(0, torch.cuda.Stream())
    _step(AdamW8(gpu, tensors))   # (a kernel's first launch may wait for the device)
    torch.cuda.synchronize()
    torch.cuda._sleep(BUSY)       # the current stream's work waits behind this
    plan = AdamW8(gpu, tensors)
    _step(plan)
    torch.cuda.synchronize()
    assert plan.gradient_square_sum.item() == 4.0 * 3000

"""The 8-bit AdamW plan and the output layer on a stream that is not the current one while they are made: their own tensors
are ready when the first call on that stream reads them, however busy either stream is."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.adamw8 import AdamW8, AdamW8Tensor, adamw8_state  # noqa: E402
from staleynet_b200.matmul import AdamWHyperparameters, Gpu  # noqa: E402
from staleynet_b200.vocabulary_head import VocabularyHead  # noqa: E402

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


@pytest.mark.parametrize("busy", ["own", "current"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_the_output_layer_on_a_stream_of_its_own(dtype, busy):
    sizes = {"rows": 256, "width": 64, "classes": 1000, "dtype": dtype}
    hidden = torch.randn(256, 64, device="cuda").to(dtype)
    targets = torch.randint(0, 1000, (256,), device="cuda", dtype=torch.int32)
    hyper = AdamWHyperparameters(1e-2, 0.9, 0.95, 1e-8, 0.0, 1)
    here = VocabularyHead(Gpu(0), **sizes)
    expected = here.step(hidden, targets, hyper)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream if busy == "own" else torch.cuda.current_stream()):
        torch.cuda._sleep(BUSY)
    there = VocabularyHead(Gpu(0, stream), **sizes)
    got = there.step(hidden, targets, hyper)
    torch.cuda.synchronize()
    # The same kernels on the same values: bf16 gradients may differ in the order of f32 sums.
    assert (got.double() - expected.double()).norm() <= 1e-3 * expected.double().norm()
    assert torch.equal(there.losses, here.losses)
    assert (there.weight.double() - here.weight.double()).norm() <= 1e-3 * here.weight.double().norm()
    if dtype == torch.bfloat16:
        assert torch.equal(there.operand, there.weight.bfloat16())

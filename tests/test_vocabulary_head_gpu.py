"""The output layer's training step (staleynet_b200/vocabulary_head.py): its gradients against torch's in 64 bits, and
that it learns."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import AdamWHyperparameters, Gpu  # noqa: E402
from staleynet_b200.vocabulary_head import VocabularyHead, main  # noqa: E402

pytestmark = pytest.mark.gpu


# f32: the chain's roundings (2e-5, as for its parts). bf16: the normalised rows, p, the gradient of the normalised rows
# and the result are rounded once each, 2^-8 at most.
@pytest.mark.parametrize("dtype,tolerance", [(torch.float32, 4e-5), (torch.bfloat16, 4 * 2.0 ** -8)],
                         ids=["f32", "bf16"])
def test_gradients_of_the_whole_layer(dtype, tolerance):
    gpu = Gpu(0)
    head = VocabularyHead(gpu, rows=300, width=96, classes=1003, dtype=dtype)
    head.gain.normal_(1.0, 0.2)
    head.bias.normal_(0.0, 0.2)
    hidden = (torch.randn(300, 96, device="cuda") * 2 + 1).to(dtype)
    targets = torch.randint(0, 1003, (300,), device="cuda", dtype=torch.int32)
    targets[::7] = -1
    d_hidden = head.backward(hidden, targets, 0.01)
    torch.cuda.synchronize()
    x, w, g, b = (t.double().detach().requires_grad_() for t in (hidden, head.operand, head.gain, head.bias))
    normal = torch.nn.functional.layer_norm(x, (96,), g, b, 1e-5)
    losses = torch.nn.functional.cross_entropy(normal @ w.t(), targets.long(), ignore_index=-1, reduction="none")
    (0.01 * losses.sum()).backward()
    assert (head.losses.double() - losses).abs().max() <= (2e-5 if dtype == torch.float32 else 0.05)
    for got, expected in ((d_hidden, x.grad), (head.d_weight, w.grad), (head.d_gain, g.grad), (head.d_bias, b.grad)):
        assert (got.double() - expected).norm() <= tolerance * expected.norm()
    assert torch.equal(head.evaluate(hidden, targets) == 0, targets < 0)


def test_training_learns_the_mapping():
    torch.manual_seed(0)
    gpu = Gpu(0)
    head = VocabularyHead(gpu, rows=512, width=64, classes=301)
    directions = torch.randn(301, 64, device="cuda")
    losses = []
    for step in range(1, 61):
        targets = torch.randint(0, 301, (512,), device="cuda", dtype=torch.int32)
        hidden = (directions[targets.long()] + 0.3 * torch.randn(512, 64, device="cuda")).bfloat16()
        head.step(hidden, targets, AdamWHyperparameters(1e-2, 0.9, 0.95, 1e-8, 0.0, step))
        losses.append(head.loss_sum.item() / 512)
    assert losses[0] > 5.0 and losses[-1] < 1.0, (losses[0], losses[-1])
    assert torch.equal(head.operand, head.weight.bfloat16())


def test_the_example_runs(capsys):
    assert main(["--rows", "256", "--width", "64", "--classes", "500", "--steps", "20"]) == 0
    assert "step 20: loss" in capsys.readouterr().out

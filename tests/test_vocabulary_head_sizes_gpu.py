"""The output layer (staleynet_b200/vocabulary_head.py) at sizes whose losses need more workspace than its gradients."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import Gpu  # noqa: E402
from staleynet_b200.vocabulary_head import VocabularyHead  # noqa: E402

pytestmark = pytest.mark.gpu


def _batch(rows, width, classes, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + classes)
    hidden = (torch.randn(rows, width, generator=g, device="cuda") * 2 + 1).to(dtype)
    targets = torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    targets[2::5] = -1
    return hidden, targets


def _losses(head, hidden, targets):
    normal = torch.nn.functional.layer_norm(hidden.double(), hidden.shape[1:], head.gain.double(), head.bias.double(), 1e-5)
    return torch.nn.functional.cross_entropy(normal @ head.operand.double().t(), targets.long(), ignore_index=-1,
                                             reduction="none")


# A weight of several packed pieces (256 MB each, three f32 values an element): f32 rows of 768 from 29,128 classes on.
# Losses of logits of about 1 over 30,000 classes: f32 sums, 2e-5; normalised rows rounded to bf16, 0.05.
@pytest.mark.parametrize("dtype,tolerance", [(torch.float32, 2e-5), (torch.bfloat16, 0.05)], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,width,classes", [(64, 768, 32768), (150, 768, 32768), (5, 771, 60001), (40, 64, 301)])
def test_a_head_evaluates_and_trains_whatever_its_pieces(rows, width, classes, dtype, tolerance):
    head = VocabularyHead(Gpu(0), rows=rows, width=width, classes=classes, dtype=dtype)
    hidden, targets = _batch(rows, width, classes, dtype)
    expected = _losses(head, hidden, targets)
    assert (head.evaluate(hidden, targets).double() - expected).abs().max() <= tolerance
    head.backward(hidden, targets, 0.01)
    torch.cuda.synchronize()
    assert (head.losses.double() - expected).abs().max() <= tolerance

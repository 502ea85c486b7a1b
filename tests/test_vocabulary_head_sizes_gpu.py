"""The output layer (staleynet_b200/vocabulary_head.py) at sizes whose losses need more workspace than its gradients,
and on batches of fewer rows than it was made for."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import AdamWHyperparameters, Gpu, SnbError  # noqa: E402
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,width,classes,fewer", [(300, 96, 1003, (299, 17, 1, 0)), (4096, 40, 100003, (3500, 4, 2049))])
def test_a_batch_may_have_fewer_rows(rows, width, classes, fewer, dtype):
    """An evaluation of one token, or the last batch of an epoch. 3,500 rows take longer pieces than 4,096, so their
    gradients need more workspace."""
    head = VocabularyHead(Gpu(0), rows=rows, width=width, classes=classes, dtype=dtype)
    hidden, targets = _batch(rows, width, classes, dtype)
    for n in fewer:
        other = VocabularyHead(head.gpu, rows=max(n, 1), width=width, classes=classes, dtype=dtype)
        h, t = hidden[:n], targets[:n]
        tolerance = 2e-5 if dtype == torch.float32 else 0.05
        losses = head.evaluate(h, t)
        assert losses.shape == (n,)
        if n > 0:
            assert (losses.double() - _losses(head, h, t)).abs().max() <= tolerance
            assert abs(head.loss_sum.item() - losses.double().sum().item()) <= 1e-6 * losses.double().sum().item() + 1e-6
        d_hidden = head.backward(h, t, 0.01)
        assert d_hidden.shape == h.shape
        if n == 0:
            assert not head.d_weight.any() and not head.d_gain.any() and not head.d_bias.any()
            continue
        expected = other.backward(h, t, 0.01)
        for got, same in ((d_hidden, expected), (head.d_weight, other.d_weight), (head.d_gain, other.d_gain),
                          (head.d_bias, other.d_bias)):
            # The same products, perhaps in other pieces: f32 sums in another order, rounded once more to bf16.
            assert (got.double() - same.double()).norm() <= (2e-5 if dtype == torch.float32 else 2.0 ** -8) * same.double().norm()
    before = head.weight.clone()
    head.step(hidden[:3], targets[:3], AdamWHyperparameters(1e-2, 0.9, 0.95, 1e-8, 0.0, 1))
    assert not torch.equal(before, head.weight)
    with pytest.raises(SnbError, match="made for at most"):
        head.evaluate(torch.zeros(rows + 1, width, device="cuda", dtype=dtype), targets)

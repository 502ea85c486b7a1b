"""Losses of the vocabulary's softmax cross entropy where one logit leads by far, to within a few f32 roundings.

The logits here are exact whatever sums them: each is one product of factors with at most 8 significant bits. A loss is
lse - z in base 2: the leading term's exponential and the logarithm of the sum are each off by 2^-22 of about 1, the sum's
own roundings by as much; the difference of the maximum and the target's logit by its rounding and that of log2 e (2^-25).
2^-20 + 2^-21 of the loss covers that with a factor of two, whatever the size of the logits."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200 import _ffi  # noqa: E402
from staleynet_b200.matmul import Gpu, Storage, last_path  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _peaked(rows, width, classes, dtype, storage):
    """z[i, v] = size_i weight_v, class 3 the leading one, a second one 2^-3 of it behind, and the rest at most half."""
    g = torch.Generator(device="cuda").manual_seed(rows + classes)
    size = (10.0 + 190.0 * torch.rand(rows, generator=g, device="cuda")).bfloat16().float()
    factor = -torch.rand(classes, generator=g, device="cuda").mul_(64).round_().div_(128)
    factor[3], factor[5] = 1.0, 0.875
    hidden, weight = torch.zeros(rows, width, device="cuda"), torch.zeros(classes, width, device="cuda")
    hidden[:, 1], weight[:, 1] = size, factor
    targets = torch.full((rows,), 3, device="cuda", dtype=torch.int32)
    targets[1::3] = 5
    targets[2::3] = torch.randint(6, classes, targets[2::3].shape, generator=g, device="cuda", dtype=torch.int32)
    z = size.double()[:, None] * factor.double()
    losses = torch.logsumexp(z, 1) - z.gather(1, targets.long()[:, None])[:, 0]
    weight = weight.to(dtype)
    return hidden.to(dtype), weight if storage is Storage.TRANSPOSED else weight.t().contiguous(), targets, losses


def _losses(hidden, weight, targets, storage, d_hidden=None):
    gpu = Gpu(0)
    losses, total = torch.empty(hidden.shape[0], device="cuda"), torch.empty((), device="cuda")
    need = gpu.vocabulary_cross_entropy_workspace(hidden, weight, storage=storage, d_hidden=d_hidden)
    gpu.vocabulary_cross_entropy(hidden, weight, targets, losses, total,
                                 torch.empty(need, device="cuda", dtype=torch.uint8), storage=storage, d_hidden=d_hidden)
    gpu.synchronize()
    gpu.device_status()
    return losses


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,width,classes,gradient", [(4, 9, 3001, False), (100, 16, 1000, False), (100, 16, 1000, True),
                                                         (300, 9, 3001, False), (700, 24, 20011, True)])
def test_the_loss_of_a_leading_class_has_no_error_of_the_logits_size(rows, width, classes, gradient, dtype, storage):
    hidden, weight, targets, expected = _peaked(rows, width, classes, dtype, storage)
    losses = _losses(hidden, weight, targets, storage, torch.empty_like(hidden) if gradient else None)
    assert last_path() == (_ffi.PATH_SIMT if rows == 4 else _ffi.PATH_TENSOR_CORE if rows == 100
                           else _ffi.PATH_TENSOR_CORE_PAIR)
    assert bool((losses >= 0).all())
    error = (losses.double() - expected).abs()
    assert bool((error <= 2.0 ** -20 + 2.0 ** -21 * expected).all()), error.max().item()

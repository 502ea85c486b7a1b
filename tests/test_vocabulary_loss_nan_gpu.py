"""NaN in the vocabulary loss's f32 operands, whatever its bits, reaches every loss and gradient that reads it."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import Gpu, Storage  # noqa: E402

pytestmark = pytest.mark.gpu


# The bits of a NaN: the usual quiet one, one of arithmetic, and two whose leading fraction bits are clear.
@pytest.mark.parametrize("bits", [0x7FC00000, 0x7FFFFFFF, 0x7F800001, -0x7FFFFF], ids=["quiet", "all", "low", "negative"])
@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("rows", [4, 200])
def test_nan_of_any_bits(rows, storage, bits):
    g = torch.Generator(device="cuda").manual_seed(rows)
    hidden = torch.randn(rows, 40, generator=g, device="cuda")
    weight = torch.randn(*((500, 40) if storage is Storage.TRANSPOSED else (40, 500)), generator=g, device="cuda")
    targets = torch.randint(0, 400, (rows,), generator=g, device="cuda", dtype=torch.int32)
    gpu = Gpu(0)

    def run(hidden, weight):
        dh, dw = torch.zeros_like(hidden), torch.zeros_like(weight)
        alone, losses, total = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros((), device="cuda")
        for out, grads in ((alone, {}), (losses, {"d_hidden": dh, "d_weight": dw})):
            need = gpu.vocabulary_cross_entropy_workspace(hidden, weight, storage=storage, **grads)
            gpu.vocabulary_cross_entropy(hidden, weight, targets, out, total, torch.empty(need, device="cuda", dtype=torch.uint8),
                                         storage=storage, **grads)
        gpu.synchronize()
        return alone, losses, total, dh, dw

    bad = weight.clone()
    (bad if storage is Storage.TRANSPOSED else bad.t()).view(torch.int32)[450, 7] = bits
    for t in run(hidden, bad):
        assert bool(t.isnan().all())
    bad = hidden.clone()
    bad.view(torch.int32)[2, 3] = bits
    alone, losses, total, dh, dw = run(bad, weight)
    row = torch.arange(rows, device="cuda") == 2
    assert torch.equal(alone.isnan(), row) and torch.equal(losses.isnan(), row) and bool(total.isnan())
    assert torch.equal(dh.isnan().all(1), row) and torch.equal(dh.isnan().any(1), row) and bool(dw.isnan().all())

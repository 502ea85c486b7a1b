"""Calls of the vocabulary loss from several threads at once, each on its own stream."""
import ctypes
import threading

import pytest

torch = pytest.importorskip("torch")

from staleynet_b200 import _ffi  # noqa: E402
from staleynet_b200.matmul import Gpu, Storage  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
def test_a_few_rows_of_several_widths_at_once(storage):
    """Each width takes another amount of shared memory. The calls go to the library directly, one after the other, so that
    the threads' launches fall between each other's steps."""
    lib = _ffi.load()
    calls, failures = [], []
    for width in (4096, 3200, 2880):
        gpu = Gpu(0, torch.cuda.Stream())
        hidden = torch.randn(4, width, device="cuda")
        weight = torch.randn(*((40, width) if storage is Storage.TRANSPOSED else (width, 40)), device="cuda") * width ** -0.5
        targets = torch.randint(0, 40, (4,), device="cuda", dtype=torch.int32)
        losses = torch.full((4,), float("nan"), device="cuda")
        a = gpu._vocabulary_loss_args(hidden, weight, storage, None, None)
        workspace = torch.empty(gpu.vocabulary_cross_entropy_workspace(hidden, weight, storage=storage), device="cuda",
                                dtype=torch.uint8)
        a.targets, a.targets_len, a.losses, a.losses_len = targets.data_ptr(), 4, losses.data_ptr(), 4
        a.workspace, a.workspace_len = workspace.data_ptr(), workspace.numel()
        calls.append((gpu, a, hidden, weight, targets, losses, workspace))
    torch.cuda.synchronize()

    def many(gpu, a):
        handle, args = gpu._stream_handle(), ctypes.byref(a)
        for _ in range(4000):
            if lib.snb_vocabulary_cross_entropy(handle, args) != _ffi.OK:
                failures.append(_ffi.last_error())
                return

    threads = [threading.Thread(target=many, args=c[:2]) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures, failures
    for _, _, hidden, weight, targets, losses, _ in calls:
        logits = hidden.double() @ (weight.double().t() if storage is Storage.TRANSPOSED else weight.double())
        expected = torch.nn.functional.cross_entropy(logits, targets.long(), reduction="none")
        # f32 sums of 4,096 products of size 1 / 64: far below 1e-5.
        assert (losses.double() - expected).abs().max() <= 1e-5

"""The Python entry points of the layer norm and the vocabulary loss refuse tensors that their kernels would write past, or
between whose elements they would write: no call reaches the library (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.matmul import Gpu, SnbError  # noqa: E402


class OnDevice(torch.Tensor):
    """A host tensor that passes for one in device memory: only its shape and strides are looked at here."""

    is_cuda = True


class NoLibrary:
    """Stands for the library: any call of it is one that should have been refused."""

    def __getattr__(self, name):
        raise RuntimeError(f"{name} was reached")


def _gpu():
    gpu = Gpu.__new__(Gpu)
    gpu.lib = NoLibrary()
    gpu._stream_handle = lambda: None
    gpu._types, gpu._f32 = {torch.float32: 0, torch.bfloat16: 1}, torch.float32
    return gpu


def _on_device(t):
    return t.as_subclass(OnDevice)


def _loss(**changes):
    t = {"hidden": torch.zeros(10, 32), "weight": torch.zeros(50, 32), "targets": torch.zeros(10, dtype=torch.int32),
         "losses": torch.zeros(10), "loss_sum": torch.zeros(()), "workspace": torch.zeros(4096, dtype=torch.uint8)}
    t.update(changes)
    _gpu().vocabulary_cross_entropy(*(_on_device(x) for x in t.values()))


def test_a_call_with_good_tensors_reaches_the_library():
    with pytest.raises(RuntimeError, match="snb_vocabulary_cross_entropy was reached"):
        _loss()


@pytest.mark.parametrize("losses", [torch.zeros(10, 4)[:, 1], torch.zeros(1).expand(10), torch.zeros(20)[::2]],
                         ids=["column", "expanded", "every_other"])
def test_the_losses_are_dense(losses):
    with pytest.raises(SnbError, match="losses must be dense float32"):
        _loss(losses=losses)


@pytest.mark.parametrize("total", [torch.zeros(0), torch.zeros(2), torch.zeros((), dtype=torch.float64)],
                         ids=["empty", "two", "f64"])
def test_the_sum_of_the_losses_is_one_f32(total):
    with pytest.raises(SnbError, match="loss_sum must be one float32"):
        _loss(loss_sum=total)


@pytest.mark.parametrize("workspace", [torch.zeros(8192, dtype=torch.uint8)[::2],
                                       torch.zeros(1, dtype=torch.uint8).expand(4096)], ids=["strided", "expanded"])
def test_the_workspace_is_dense(workspace):
    with pytest.raises(SnbError, match="vocabulary_cross_entropy: workspace must be dense"):
        _loss(workspace=workspace)
    rows, params, stats = (torch.zeros(6, 40) for _ in range(3)), (torch.zeros(40) for _ in range(3)), torch.zeros(6)
    (dy, x, dx), (gain, dg, db) = rows, params
    with pytest.raises(SnbError, match="layer_norm_backward: workspace must be dense"):
        _gpu().layer_norm_backward(*(_on_device(t) for t in (dy, x, gain, stats, stats, dx, dg, db, workspace)))

"""The layer norm, the vocabulary loss and the 8-bit AdamW step in a CUDA graph, under a budget of SMs, and resumed from a
saved state."""
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200 import _ffi  # noqa: E402
from staleynet_b200.adamw8 import AdamW8, AdamW8Tensor, adamw8_state  # noqa: E402
from staleynet_b200.matmul import AdamWHyperparameters, Gpu, Storage  # noqa: E402
from test_vocabulary_loss_gpu import BF16, F32, _case, _check  # noqa: E402

pytestmark = pytest.mark.gpu

HYPER = AdamWHyperparameters(1e-2, 0.9, 0.95, 1e-8, 0.0, 3)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 300])
def test_a_graph_repeats_the_calls_on_new_inputs(rows, dtype):
    stream, width, classes = torch.cuda.Stream(), 96, 2001
    gpu = Gpu(0, stream)
    with torch.cuda.stream(stream):
        x = torch.randn(rows, width, device="cuda").to(dtype)
        gain, bias = torch.ones(width, device="cuda"), torch.zeros(width, device="cuda")
        weight = (torch.randn(classes, width, device="cuda") * width ** -0.5).to(dtype)
        targets = torch.randint(0, classes, (rows,), device="cuda", dtype=torch.int32)
        normal, d_normal, dx = (torch.empty_like(x) for _ in range(3))
        mean, inv, losses, total = (torch.empty(s, device="cuda") for s in (rows, rows, rows, ()))
        dw, dg, db = torch.empty_like(weight), torch.empty_like(gain), torch.empty_like(bias)
        need = max(gpu.vocabulary_cross_entropy_workspace(normal, weight, d_hidden=d_normal, d_weight=dw),
                   gpu.layer_norm_workspace(rows, width))
        workspace = torch.empty(need, device="cuda", dtype=torch.uint8)
        master = weight.float()
        state = adamw8_state(master)
        plan = AdamW8(gpu, [AdamW8Tensor(master, dw, *state)])

        def step():
            gpu.layer_norm_forward(x, gain, bias, normal, mean, inv, 1e-5)
            gpu.vocabulary_cross_entropy(normal, weight, targets, losses, total, workspace, d_hidden=d_normal, d_weight=dw,
                                         deterministic=True)
            gpu.layer_norm_backward(d_normal, x, gain, mean, inv, dx, dg, db, workspace)
            plan.step(HYPER, 1.0, 7)

        outputs = (losses, total, dx, dw, dg, db, master, *state)
        start = [t.clone() for t in (master, *state)]

        def reset():
            for t, s in zip((master, *state), start):
                t.copy_(s)

        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for seed in (1, 2):
            x.copy_(torch.randn(rows, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
            reset()
            step()
            expected = [t.clone() for t in outputs]
            for t in outputs[:6]:
                t.fill_(float("nan"))
            reset()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outputs, expected))
    gpu.device_status()


@pytest.mark.parametrize("storage", list(Storage), ids=lambda s: s.name.lower())
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("budget", [1, 2, 37, 147])
def test_the_vocabulary_loss_under_a_budget_of_sms(budget, dtype, storage):
    lib = _ffi.load()
    before = lib.snb_set_sm_budget(budget)
    try:
        for rows, width, classes in ((1, 64, 1000), (300, 99, 1003), (1000, 256, 4096)):
            _check(*_case(rows, width, classes, dtype, storage, seed=budget), storage)
    finally:
        lib.snb_set_sm_budget(before)


def test_a_saved_state_resumes_bit_for_bit():
    """The parameters, codes and scales, with each step's number and seed, are all that a step depends on."""
    gpu = Gpu(0)
    parameter, gradient = torch.randn(5003, device="cuda"), torch.empty(5003, device="cuda")
    state = adamw8_state(parameter)

    def steps(parameter, state, numbers):
        plan = AdamW8(gpu, [AdamW8Tensor(parameter, gradient, *state, weight_decay=0.1)])
        for k in numbers:
            gradient.normal_(generator=torch.Generator(device="cuda").manual_seed(k))
            plan.step(AdamWHyperparameters(1e-2, 0.9, 0.95, 1e-8, 0.0, k), 1.0, 1000 + k)

    steps(parameter, state, (1, 2, 3))
    saved = [t.clone().cpu() for t in (parameter, *state)]
    steps(parameter, state, (4, 5))
    resumed = [t.cuda() for t in saved]
    steps(resumed[0], resumed[1:], (4, 5))
    assert all(torch.equal(a, b) for a, b in zip((parameter, *state), resumed))

"""AdamW with 8-bit moments (snb_adamw8_step) against the same step in 64 bits: moments decoded, updated and rounded with
the reference generator's draws, in numpy.

Tolerances. A code is decided by comparing a share (five f32 roundings, at most 3e-7 of it) with a random threshold
between levels that are 0.8 % apart or more, so f32 and 64 bits may disagree, by one code, in about one value of 10,000;
one in 1,000 is allowed. A scale is an f32 result of three roundings: 4e-7. The parameter moves by the learning rate times
a quotient of approximate root and division (2^-21 with their neighbours) and is rounded once itself."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from staleynet_b200.adamw8 import BLOCK, AdamW8, AdamW8Tensor, adamw8_state  # noqa: E402
from staleynet_b200.matmul import AdamWHyperparameters, Gpu, SnbError  # noqa: E402

pytestmark = pytest.mark.gpu

LEVELS1, LEVELS2 = (np.arange(128) / 127.0) ** 2, (np.arange(256) / 255.0) ** 4
F32, BF16 = torch.float32, torch.bfloat16


def _f(v):
    return float(np.float32(v))


def _bits(seed, first_draw, n):
    k = np.uint64(first_draw) + np.arange(1, (n + 1) // 2 + 1, dtype=np.uint64)
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + k * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    z = z ^ (z >> np.uint64(31))
    return np.stack([z & np.uint64(0xFFFFFFFF), z >> np.uint64(32)], 1).reshape(-1)[:n].astype(np.int64)


def _scales(scale, n):
    return np.repeat(scale.double().cpu().numpy(), BLOCK)[:n]


def _values(state, n):
    q1, q2 = state[0].cpu().numpy().astype(int).reshape(-1), state[2].cpu().numpy().astype(int).reshape(-1)
    return np.sign(q1) * LEVELS1[abs(q1)] * _scales(state[1], n), LEVELS2[q2] * _scales(state[3], n)


def _round(values, levels, bits):
    n = len(values)
    padded = np.pad(values, (0, -n % BLOCK)).reshape(-1, BLOCK)
    scale = padded.max(1)
    share = (padded / np.where(scale > 0, scale, 1)[:, None]).reshape(-1)[:n]
    q = np.clip(np.searchsorted(levels, share, side="right") - 1, 0, len(levels) - 2)
    chance = (share - levels[q]) / (levels[q + 1] - levels[q])
    return q + ((bits + 0.5) / 65536 < chance), scale


def _reference(parameter, gradient, state, hyper, decay, clip, seed, first_draw):
    n = parameter.numel()
    m, v = _values(state, n)
    g = gradient.double().cpu().numpy().reshape(-1) * clip
    b1, b2 = _f(hyper.beta1), _f(hyper.beta2)
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    w = parameter.double().cpu().numpy().reshape(-1)
    rate = m / (1 - b1 ** hyper.step) / (np.sqrt(v / (1 - b2 ** hyper.step)) + _f(hyper.epsilon))
    w = w - _f(hyper.learning_rate) * (rate + _f(decay) * w)
    bits = _bits(seed, first_draw, n)
    q1, s1 = _round(abs(m), LEVELS1, bits & 0xFFFF)
    q2, s2 = _round(v, LEVELS2, bits >> 16)
    return w, np.where(m < 0, -q1, q1), s1, np.where(v > 0, np.maximum(q2, 1), q2), s2, abs(rate)


def _tensor(n, gradient_type, rng, offset=0, shadow=True, filled=True):
    """A tensor's buffers, starting `offset` elements into their storage, with moments of an ongoing run."""
    def buf(values, dtype):
        whole = torch.zeros(n + offset + 8, device="cuda", dtype=dtype)
        part = whole[offset:offset + n]
        part.copy_(torch.from_numpy(values))
        return part

    spread = np.repeat(np.exp(rng.standard_normal((n + BLOCK - 1) // BLOCK)) * 1e-3, BLOCK)[:n]
    parameter = buf(rng.standard_normal(n) * 0.02, F32)
    gradient = buf(rng.standard_normal(n) * spread, gradient_type)
    state = list(adamw8_state(parameter))
    state[0], state[2] = buf(np.zeros(n), torch.int8), buf(np.zeros(n), torch.uint8)
    if filled and n:
        state[0].copy_(torch.from_numpy(rng.integers(-127, 128, n)))
        state[2].copy_(torch.from_numpy(rng.integers(1, 256, n)))
        state[1].copy_(torch.from_numpy(2.0 * spread[::BLOCK]))
        state[3].copy_(torch.from_numpy(6.0 * spread[::BLOCK] ** 2))
    return parameter, gradient, state, buf(np.zeros(n), BF16) if shadow else None


def _check_step(tensors, decays, max_norm, hyper, seed=99):
    plan = AdamW8(Gpu(0), [AdamW8Tensor(p, g, *s, weight_decay=d, shadow=sh)
                           for (p, g, s, sh), d in zip(tensors, decays)])
    squares = sum(float((g.double() ** 2).sum()) for _, g, _, _ in tensors)
    norm = squares ** 0.5
    clip = max_norm / norm if norm > max_norm else 1.0
    draw, expected = 0, []
    for (p, g, s, _), d in zip(tensors, decays):
        expected.append(_reference(p, g, s, hyper, d, clip, seed, draw))
        draw += (p.numel() + 1) // 2
    plan.step(hyper, max_norm, seed)
    torch.cuda.synchronize()
    assert abs(plan.gradient_square_sum.item() - squares) <= 1e-12 * squares
    different = count = 0
    for (p, g, s, sh), (w, q1, s1, q2, s2, rate) in zip(tensors, expected):
        if not p.numel():
            continue
        w_k = p.double().cpu().numpy()
        bound = _f(hyper.learning_rate) * 2.0 ** -20 * (rate + 1) + 2.0 ** -23 * abs(w)
        assert (abs(w_k - w) <= bound).all()
        if sh is not None:
            assert torch.equal(sh, p.bfloat16())
        for codes, scale, q, s_e in ((s[0], s[1], q1, s1), (s[2], s[3], q2, s2)):
            np.testing.assert_allclose(scale.cpu().numpy(), s_e, rtol=4e-7, atol=1e-37)
            off = abs(codes.cpu().numpy().astype(int) - q)
            assert off.max() <= 1
            different, count = different + int((off > 0).sum()), count + off.size
    assert different <= max(2, count / 1000)


HYPER = AdamWHyperparameters(3e-4, 0.9, 0.95, 1e-8, 0.0, 7)


def _levels(q, power):
    s = (q * q).float() * (1.0 / 16129.0 if power == 2 else 1.0 / 65025.0)
    return s if power == 2 else s * s


def _encode_f32(values, bits, power):
    """The codes in elementary f32 operations, each rounded by itself (torch runs one at a time)."""
    most = 127 if power == 2 else 255
    blocks = values.view(-1, BLOCK)
    scale = blocks.amax(1)
    share = (blocks * (1.0 / scale)[:, None]).view(-1)
    levels = _levels(torch.arange(most + 1, device="cuda", dtype=torch.int32), power)
    q = (torch.searchsorted(levels, share, right=True) - 1).clamp(0, most - 1)
    low, high = levels[q], levels[q + 1]
    unit = (bits.float() + 0.5) * (1.0 / 65536.0)
    threshold = low + unit * (high - low)
    return q + (threshold < share), scale


@pytest.mark.parametrize("gradient_type", [F32, BF16], ids=["f32", "bf16"])
def test_codes_and_scales_are_those_of_f32_arithmetic_to_the_bit(gradient_type):
    n, seed = BLOCK * 8000, 77
    p, g, state, _ = _tensor(n, gradient_type, np.random.default_rng(21))
    b1, b2 = _f(HYPER.beta1), _f(HYPER.beta2)
    nb1, nb2 = _f(np.float32(1) - np.float32(b1)), _f(np.float32(1) - np.float32(b2))
    q1, q2 = state[0].int(), state[2].int()
    m = (torch.sign(q1) * _levels(q1, 2)).view(-1, BLOCK) * state[1][:, None]
    v = _levels(q2, 4).view(-1, BLOCK) * state[3][:, None]
    gf = g.float()
    norm = torch.sqrt((g.double() ** 2).sum()).float()
    gf = gf * (0.5 / norm)   # clipped: the norm is above 0.5
    assert norm.item() > 0.5
    m = m.view(-1) * b1 + gf * nb1
    v = v.view(-1) * b2 + (gf * nb2) * gf
    bits = torch.from_numpy(_bits(seed, 0, n)).cuda()
    code1, scale1 = _encode_f32(m.abs(), bits & 0xFFFF, 2)
    code2, scale2 = _encode_f32(v, bits >> 16, 4)
    AdamW8(Gpu(0), [AdamW8Tensor(p, g, *state)]).step(HYPER, 0.5, seed)
    torch.cuda.synchronize()
    assert torch.equal(state[1], scale1) and torch.equal(state[3], scale2)
    assert torch.equal(state[0].long(), torch.where(m < 0, -code1, code1))
    assert torch.equal(state[2].long(), torch.where(v > 0, code2.clamp(min=1), code2))


@pytest.mark.parametrize("gradient_type", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 255, 256, 257, 1000, 8192, 8193, 300007])
def test_one_tensor(n, gradient_type):
    _check_step([_tensor(n, gradient_type, np.random.default_rng(n))], [0.1], 1e9, HYPER)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_ragged_tensors_clipped_together(offset):
    """Empty ones, odd sizes, starts off every vector boundary, both gradient types, with and without a copy."""
    rng = np.random.default_rng(offset)
    sizes = [768, 0, 1, 70001, 333, 256, 16384, 0]
    tensors = [_tensor(n, (F32, BF16)[i % 2], rng, offset, shadow=i % 3 > 0) for i, n in enumerate(sizes)]
    _check_step(tensors, [0.1, 0.0] * 4, 0.05, HYPER)


def test_more_tensors_than_one_launch_takes():
    rng = np.random.default_rng(0)
    _check_step([_tensor(1 + 7 * i % 600, F32, rng) for i in range(600)], [0.01] * 600, 0.3, HYPER)


def test_the_first_step_from_zero_moments():
    rng = np.random.default_rng(1)
    _check_step([_tensor(5000, F32, rng, filled=False)], [0.1], 1.0,
                AdamWHyperparameters(1e-3, 0.9, 0.999, 1e-8, 0.0, 1))


def test_gradients_of_zero_leave_zero_moments_and_a_v_above_zero_never_becomes_zero():
    p = torch.randn(700, device="cuda")
    before = p.clone()
    state = adamw8_state(p)
    g = torch.zeros(700, device="cuda")
    plan = AdamW8(Gpu(0), [AdamW8Tensor(p, g, *state)])
    plan.step(HYPER, 1.0, 1)
    assert torch.equal(p, before) and not any(bool(s.any()) for s in state)
    # One element dwarfs its block: the others' v is far below the lowest level above 0.
    g.fill_(1e-6)
    g[::256] = 1.0
    plan.step(HYPER, float("inf"), 2)
    assert bool((state[2] >= 1).all()) and bool((state[2][::256] == 255).all())
    # Their m may be rounded to 0 or to a level above it; the step after that stays bounded.
    g.zero_()
    moved = p.clone()
    plan.step(HYPER, float("inf"), 3)
    assert (p - moved).abs().max() < 100 * HYPER.learning_rate


def test_a_gradient_that_is_not_finite_shows_in_its_block():
    p = torch.randn(1024, device="cuda")
    g = torch.randn(1024, device="cuda")
    g[300] = float("nan")
    state = adamw8_state(p)
    plan = AdamW8(Gpu(0), [AdamW8Tensor(p, g, *state)])
    first, second = torch.empty_like(p), torch.empty_like(p)
    plan.bind_moments([(first, second)])
    plan.step(HYPER, 1.0, 5)
    plan.moments()
    torch.cuda.synchronize()
    bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
    bad[256:512] = True
    assert torch.equal(first.isnan(), bad) and torch.equal(second.isnan(), bad)
    assert p.isnan().nonzero().flatten().tolist() == [300]


@pytest.mark.parametrize("offset", [0, 1])
def test_moments_are_the_values_of_the_codes(offset):
    rng = np.random.default_rng(4)
    tensors = [_tensor(n, F32, rng, offset) for n in (1, 700, 9000)]
    plan = AdamW8(Gpu(0), [AdamW8Tensor(p, g, *s) for p, g, s, _ in tensors])
    outs = [(torch.empty(p.numel() + 4, device="cuda")[offset:offset + p.numel()], torch.empty_like(p))
            for p, *_ in tensors]
    plan.bind_moments(outs)
    plan.moments()
    torch.cuda.synchronize()
    for (p, _, s, _), (m, v) in zip(tensors, outs):
        m_e, v_e = _values(s, p.numel())
        np.testing.assert_allclose(m.cpu().numpy(), m_e, rtol=4e-7)
        np.testing.assert_allclose(v.cpu().numpy(), v_e, rtol=6e-7)


def test_the_rounding_keeps_expectations():
    """The mean of the stored moments over 400 seeds, from the same state and gradient: within six standard errors (a
    value between levels a step d apart has a deviation of at most d / 2)."""
    rng = np.random.default_rng(8)
    p, g, state, _ = _tensor(BLOCK * 4, F32, rng)
    sums = [0.0, 0.0]
    for seed in range(400):
        copy = [s.clone() for s in state]
        plan = AdamW8(Gpu(0), [AdamW8Tensor(p.clone(), g, *copy)])
        m, v = torch.empty_like(p), torch.empty_like(p)
        plan.bind_moments([(m, v)])
        plan.step(HYPER, 1e9, seed * 7919)
        plan.moments()
        sums[0], sums[1] = sums[0] + m.double(), sums[1] + v.double()
    m0, v0 = _values(state, p.numel())
    gn = g.double().cpu().numpy()
    b1, b2 = _f(0.9), _f(0.95)
    for total, exact, levels in ((sums[0], b1 * m0 + (1 - b1) * gn, LEVELS1),
                                 (sums[1], b2 * v0 + (1 - b2) * gn * gn, LEVELS2)):
        scale = np.repeat(abs(exact).reshape(-1, BLOCK).max(1), BLOCK)
        q = np.clip(np.searchsorted(levels, abs(exact) / scale, side="right") - 1, 0, len(levels) - 2)
        step = (levels[q + 1] - levels[q]) * scale
        keep = q > 0   # a v in the lowest step is raised to the first level by design
        error = abs(total.cpu().numpy() / 400 - exact)
        assert (error[keep] <= (6 * step / 2 / 20 + step / 1024 + 1e-6 * abs(exact))[keep]).all()


def test_the_same_inputs_give_the_same_bits():
    results = []
    for _ in range(2):
        rng = np.random.default_rng(12)
        tensors = [_tensor(n, F32, rng) for n in (100000, 77, 40000)]
        plan = AdamW8(Gpu(0), [AdamW8Tensor(p, g, *s) for p, g, s, _ in tensors])
        for step in range(1, 4):
            plan.step(AdamWHyperparameters(1e-3, 0.9, 0.95, 1e-8, 0.0, step), 0.5, step)
        results.append([x for p, _, s, _ in tensors for x in (p, *s)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_it_trains_like_32_bit_moments():
    """A least-squares problem, 300 steps, against snb_adamw_step on the same gradients' formula: the losses fall by the
    same factor within a fifth."""
    g = torch.Generator(device="cuda").manual_seed(0)
    a = torch.randn(512, 256, generator=g, device="cuda") * torch.logspace(-1, 0.5, 256, device="cuda")
    target = a @ torch.randn(256, 8, generator=g, device="cuda")
    gpu, losses = Gpu(0), []
    for eight in (True, False):
        w = torch.zeros(256, 8, device="cuda")
        grad = torch.empty_like(w)
        state = adamw8_state(w) if eight else (torch.zeros_like(w), torch.zeros_like(w))
        plan = AdamW8(gpu, [AdamW8Tensor(w, grad, *state)]) if eight else None
        for step in range(1, 301):
            residual = a @ w - target
            grad.copy_(a.t() @ residual / 512)
            hyper = AdamWHyperparameters(2e-2, 0.9, 0.999, 1e-8, 0.0, step)
            if eight:
                plan.step(hyper, float("inf"), step)
            else:
                gpu.adamw_step(w, grad, *state, hyper)
        losses.append(((a @ w - target) ** 2).mean().item())
    start = (target ** 2).mean().item()
    assert losses[1] < 0.2 * start and abs(np.log(losses[0] / losses[1])) < 0.2, (losses, start)


def test_refusals():
    gpu = Gpu(0)
    p, g = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    state = adamw8_state(p)
    plan = AdamW8(gpu, [AdamW8Tensor(p, g, *state)])
    with pytest.raises(SnbError, match="max_gradient_norm"):
        plan.step(HYPER, 0.0, 1)
    with pytest.raises(SnbError, match="steps count from 1"):
        plan.step(AdamWHyperparameters(1e-3, 0.9, 0.95, 1e-8, 0.0, 0), 1.0, 1)
    with pytest.raises(AssertionError, match="gradient must be 300 dense"):
        AdamW8(gpu, [AdamW8Tensor(p, g[:299], *state)])
    with pytest.raises(AssertionError, match="first_scale must be 2 dense"):
        AdamW8(gpu, [AdamW8Tensor(p, g, state[0], state[1][:1], state[2], state[3])])
    with pytest.raises(AssertionError, match="second must be"):
        AdamW8(gpu, [AdamW8Tensor(p, g, state[0], state[1], state[0], state[3])])
    with pytest.raises(SnbError, match="CUDA device memory"):
        AdamW8(gpu, [AdamW8Tensor(p.cpu(), g, *state)])
    with pytest.raises(AssertionError, match="one .first, second. pair"):
        plan.bind_moments([])
    plan._workspace = plan._workspace[:100]
    with pytest.raises(SnbError, match="workspace holds"):
        plan.step(HYPER, 1.0, 1)

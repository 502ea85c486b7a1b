"""An AdamW step over many tensors with both moments held in 8 bits (snb_adamw8_step): the optimizer of a model whose
32-bit moments would take twice the memory of its weights. A plan built once holds the tensors' argument blocks; each
step is two launches for up to 256 tensors.

    state = adamw8_state(parameter)                      # zero moments: codes and one f32 scale for each 256 elements
    plan = AdamW8(gpu, [AdamW8Tensor(parameter, gradient, *state, weight_decay=0.1, shadow=parameter_bf16)])
    plan.step(AdamWHyperparameters(3e-4, 0.9, 0.95, 1e-8, 0.0, step=1), max_gradient_norm=1.0, seed=1)

The codes and scales are the state to save; `moments` gives the values they stand for.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _ffi
from .matmul import AdamWHyperparameters, Gpu, SnbError, check

BLOCK = 256   # elements that share one scale


def adamw8_state(parameter):
    """Zero moments for `parameter`: (first codes, first scales, second codes, second scales)."""
    import torch

    blocks = (parameter.numel() + BLOCK - 1) // BLOCK
    return (torch.zeros(parameter.shape, device=parameter.device, dtype=torch.int8),
            torch.zeros(blocks, device=parameter.device),
            torch.zeros(parameter.shape, device=parameter.device, dtype=torch.uint8),
            torch.zeros(blocks, device=parameter.device))


@dataclass
class AdamW8Tensor:
    """One parameter tensor: f32 `parameter`, `gradient` (f32 or bf16), the moments' codes and scales, and optionally
    `shadow`, a bf16 copy of the parameter that the step writes (the operand of the next products). first_draw: where
    its random draws begin in the seed's stream, one for two elements; None: after those of the tensors before it."""

    parameter: object
    gradient: object
    first: object
    first_scale: object
    second: object
    second_scale: object
    weight_decay: float = 0.0
    shadow: object = None
    first_draw: int | None = None


class AdamW8:
    """The plan of one model's steps. It keeps its tensors, which must stay where they are."""

    def __init__(self, gpu: Gpu, tensors):
        import torch

        self.gpu = gpu
        self.tensors = list(tensors)
        self._args = (_ffi.AdamW8Tensor * max(1, len(self.tensors)))()
        draws = 0
        for i, t in enumerate(self.tensors):
            n = t.parameter.numel()
            blocks = (n + BLOCK - 1) // BLOCK
            wanted = [("parameter", n, (torch.float32,)), ("gradient", n, (torch.float32, torch.bfloat16)),
                      ("first", n, (torch.int8,)), ("first_scale", blocks, (torch.float32,)),
                      ("second", n, (torch.uint8,)), ("second_scale", blocks, (torch.float32,))]
            if t.shadow is not None:
                wanted.append(("shadow", n, (torch.bfloat16,)))
            for name, count, types in wanted:
                x = getattr(t, name)
                if not x.is_cuda:
                    raise SnbError(_ffi.ERR_INVALID_ARGUMENT, "tensors must live in CUDA device memory")
                if x.numel() != count or x.dtype not in types or not x.is_contiguous():
                    raise AssertionError(f"adamw8: tensor {i}: {name} must be {count} dense elements of "
                                         + " or ".join(str(d) for d in types))
            first_draw = draws if t.first_draw is None else t.first_draw
            draws = first_draw + (n + 1) // 2
            a = self._args[i]
            for name, _, _ in wanted:
                setattr(a, name, getattr(t, name).data_ptr())
            a.count, a.first_draw, a.weight_decay = n, first_draw, t.weight_decay
            a.gradient_type = _ffi.TYPE_BF16 if t.gradient.dtype == torch.bfloat16 else _ffi.TYPE_F32
        device = gpu.device
        need = gpu.lib.snb_adamw8_workspace(len(self.tensors))
        # Made on the stream that the steps run on, whichever is current: a zero written later would overwrite a step's sum.
        with torch.cuda.stream(gpu.stream):
            self.gradient_square_sum = torch.zeros((), device=device, dtype=torch.float64)
            self._workspace = torch.empty(need, device=device, dtype=torch.uint8)
        self._out = None

    def step(self, hyper: AdamWHyperparameters, max_gradient_norm: float, seed: int) -> None:
        """One step on the gradients as they are now, clipped to max_gradient_norm over all tensors (infinity: not at
        all); hyper.weight_decay is not read (each tensor has its own). Each step takes a seed of its own: the moments'
        rounding is drawn from it. The gradients' square sum is left in `gradient_square_sum` (f64, on the device)."""
        h = _ffi.AdamWHyper(hyper.learning_rate, hyper.beta1, hyper.beta2, hyper.epsilon, 0.0, hyper.step)
        check(self.gpu.lib.snb_adamw8_step(self.gpu._stream_handle(), self._args, len(self.tensors), ctypes.byref(h),
                                           max_gradient_norm, seed & 0xFFFFFFFFFFFFFFFF,
                                           self.gradient_square_sum.data_ptr(), self._workspace.data_ptr(),
                                           self._workspace.numel()))

    def bind_moments(self, outputs) -> None:
        """Names the f32 tensors that `moments` fills: one (first, second) pair for each tensor of the plan."""
        import torch

        outputs = list(outputs)
        if len(outputs) != len(self.tensors):
            raise AssertionError("adamw8: one (first, second) pair for each tensor")
        self._out = (_ffi.AdamW8Moments * max(1, len(outputs)))()
        self._outputs = outputs
        for i, (t, pair) in enumerate(zip(self.tensors, outputs)):
            for x in pair:
                if x.numel() != t.parameter.numel() or x.dtype != torch.float32 or not x.is_contiguous() or not x.is_cuda:
                    raise AssertionError(f"adamw8: tensor {i}: moments must be dense float32 of the parameter's size")
            o = self._out[i]
            o.first, o.first_scale = t.first.data_ptr(), t.first_scale.data_ptr()
            o.second, o.second_scale = t.second.data_ptr(), t.second_scale.data_ptr()
            o.first_out, o.second_out, o.count = pair[0].data_ptr(), pair[1].data_ptr(), t.parameter.numel()

    def moments(self) -> None:
        """Writes the values that the codes stand for into the tensors of bind_moments (snb_adamw8_moments)."""
        if self._out is None:
            raise AssertionError("adamw8: bind_moments first")
        check(self.gpu.lib.snb_adamw8_moments(self.gpu._stream_handle(), self._out, len(self.tensors)))

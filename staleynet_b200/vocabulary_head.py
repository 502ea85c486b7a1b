"""The output layer of a language model over a large vocabulary as one training step: layer norm of the last block's
activations, the vocabulary's softmax cross entropy with its gradients (the logits are never held), the norm's backward
pass, and AdamW with 8-bit moments on the f32 weights, which also writes the bf16 copy that the next step's products read.

    head = VocabularyHead(Gpu(0), rows=4096, width=768, classes=32000)
    d_hidden = head.step(hidden, targets, AdamWHyperparameters(3e-4, 0.9, 0.95, 1e-8, 0.0, step=1))
    loss = head.loss_sum.item() / rows

`python -m staleynet_b200.vocabulary_head` trains one on a synthetic corpus and prints its losses.
"""
from __future__ import annotations

import argparse

from . import _ffi
from .adamw8 import AdamW8, AdamW8Tensor, adamw8_state
from .matmul import AdamWHyperparameters, DeviceRandom, Gpu, SnbError, Storage


class VocabularyHead:
    """Weights, optimizer state and buffers of the layer for micro-batches of up to `rows` tokens. The weight is
    [classes, width] (a tied embedding's layout); `dtype` is the activations' and their gradients' element type."""

    def __init__(self, gpu: Gpu, rows: int, width: int, classes: int, seed: int = 1, weight_decay: float = 0.1,
                 epsilon: float = 1e-5, dtype=None):
        import torch

        self.gpu, self.rows, self.epsilon, self.seed = gpu, rows, epsilon, seed
        # On the stream that the calls run on, whichever is current: the tensors' first values are ready for them.
        with torch.cuda.stream(gpu.stream):
            self._allocate(width, classes, weight_decay, torch.bfloat16 if dtype is None else dtype)

    def _allocate(self, width, classes, weight_decay, dtype):
        import torch

        gpu, rows, seed = self.gpu, self.rows, self.seed

        def empty(*shape, dtype=torch.float32):
            return torch.empty(*shape, device=gpu.device, dtype=dtype)

        self.weight = DeviceRandom(gpu, seed).normal_(empty(classes, width), width ** -0.5)
        # The products' operand: a bf16 copy that the optimizer keeps current, or the f32 weight itself.
        bf16 = dtype == torch.bfloat16
        self.operand = self.weight.to(dtype) if bf16 else self.weight
        self.gain, self.bias = torch.ones(width, device=gpu.device), torch.zeros(width, device=gpu.device)
        self.normal, self.d_normal, self.d_hidden = (empty(rows, width, dtype=dtype) for _ in range(3))
        self.mean, self.inv_std, self.losses, self.loss_sum = empty(rows), empty(rows), empty(rows), empty(())
        self.d_weight = torch.empty_like(self.operand)
        self.d_gain, self.d_bias = torch.empty_like(self.gain), torch.empty_like(self.bias)
        # For evaluate and for backward: either may need more (the loss alone packs longer pieces of an f32 weight).
        need = max(gpu.vocabulary_cross_entropy_workspace(self.normal, self.operand),
                   gpu.vocabulary_cross_entropy_workspace(self.normal, self.operand, d_hidden=self.d_normal,
                                                          d_weight=self.d_weight),
                   gpu.layer_norm_workspace(rows, width))
        self.workspace = empty(need, dtype=torch.uint8)
        self.optimizer = AdamW8(gpu, [
            AdamW8Tensor(self.weight, self.d_weight, *adamw8_state(self.weight), weight_decay=weight_decay,
                         shadow=self.operand if bf16 else None),
            AdamW8Tensor(self.gain, self.d_gain, *adamw8_state(self.gain)),
            AdamW8Tensor(self.bias, self.d_bias, *adamw8_state(self.bias)),
        ])

    def _rows_of(self, hidden, *buffers):
        """The first rows of buffers for the rows of a batch, of which there may be fewer than the layer's."""
        n = hidden.shape[0]
        if n == self.rows:
            return buffers
        if n > self.rows:
            raise SnbError(_ffi.ERR_INVALID_ARGUMENT, f"vocabulary head: {n} rows, made for at most {self.rows}")
        return tuple(b[:n] for b in buffers)

    def _workspace_of(self, normal, **gradients):
        """A workspace for the loss of these rows. Fewer rows may need more (their pieces are longer): it grows then."""
        if normal is not self.normal:
            need = self.gpu.vocabulary_cross_entropy_workspace(normal, self.operand, **gradients)
            if need > self.workspace.numel():
                import torch

                with torch.cuda.stream(self.gpu.stream):   # (the old one goes back to the stream that may still use it)
                    self.workspace = self.workspace.new_empty(need)
        return self.workspace

    def evaluate(self, hidden, targets):
        """The rows' losses (0 where the target is -1), without gradients; `loss_sum` receives their sum. Any number of rows
        up to the layer's; the result is overwritten by the next call."""
        normal, mean, inv_std, losses = self._rows_of(hidden, self.normal, self.mean, self.inv_std, self.losses)
        self.gpu.layer_norm_forward(hidden, self.gain, self.bias, normal, mean, inv_std, self.epsilon)
        self.gpu.vocabulary_cross_entropy(normal, self.operand, targets, losses, self.loss_sum,
                                          self._workspace_of(normal), storage=Storage.TRANSPOSED)
        return losses

    def backward(self, hidden, targets, grad_scale: float):
        """Losses and gradients, times grad_scale: of hidden (returned), and of the weight, gain and bias (d_weight,
        d_gain, d_bias). Any number of rows up to the layer's."""
        gpu = self.gpu
        normal, mean, inv_std, losses, d_normal, d_hidden = self._rows_of(
            hidden, self.normal, self.mean, self.inv_std, self.losses, self.d_normal, self.d_hidden)
        workspace = self._workspace_of(normal, d_hidden=d_normal, d_weight=self.d_weight)
        gpu.layer_norm_forward(hidden, self.gain, self.bias, normal, mean, inv_std, self.epsilon)
        gpu.vocabulary_cross_entropy(normal, self.operand, targets, losses, self.loss_sum, workspace,
                                     storage=Storage.TRANSPOSED, d_hidden=d_normal, d_weight=self.d_weight,
                                     grad_scale=grad_scale)
        gpu.layer_norm_backward(d_normal, hidden, self.gain, mean, inv_std, d_hidden, self.d_gain, self.d_bias, workspace)
        return d_hidden

    def step(self, hidden, targets, hyper: AdamWHyperparameters, max_gradient_norm: float = 1.0,
             grad_scale: float | None = None):
        """One training step on hidden [rows, width] (of the layer's dtype) and targets [rows] int32; returns the
        gradient of hidden. grad_scale: 1 / rows unless given (a caller whose rows miss targets gives one over those
        that have one). A batch may have fewer rows than the layer; no rows at all leave the losses' gradients 0."""
        d_hidden = self.backward(hidden, targets, 1.0 / max(1, len(hidden)) if grad_scale is None else grad_scale)
        self.optimizer.step(hyper, max_gradient_norm, (self.seed << 32) + hyper.step)
        return d_hidden


def main(argv=None) -> int:
    import torch

    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--classes", type=int, default=10007)
    ap.add_argument("--steps", type=int, default=100)
    args = ap.parse_args(argv)
    gpu = Gpu(0)
    head = VocabularyHead(gpu, args.rows, args.width, args.classes)
    rng = DeviceRandom(gpu, 42)
    # The corpus: each class has a direction, and a token's activation is its next token's direction in noise.
    directions = rng.normal_(torch.empty(args.classes, args.width, device=gpu.device))
    targets = torch.empty(args.rows, device=gpu.device, dtype=torch.int32)
    noise = torch.empty(args.rows, args.width, device=gpu.device)
    for step in range(1, args.steps + 1):
        rng.below_(targets, args.classes)
        hidden = (directions[targets.long()] + rng.normal_(noise, 0.5)).bfloat16()
        head.step(hidden, targets, AdamWHyperparameters(3e-3, 0.9, 0.95, 1e-8, 0.0, step))
        if step == 1 or step % 20 == 0:
            print(f"step {step}: loss {head.loss_sum.item() / args.rows:.4f}")
    gpu.device_status()
    return 0


if __name__ == "__main__":
    raise SystemExit(main())

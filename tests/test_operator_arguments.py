"""The layer norm, vocabulary loss and 8-bit AdamW entry points refuse bad arguments before they touch a device (no GPU
needed), and their argument blocks have the header's layout."""
import ctypes
import re
from pathlib import Path

import pytest

from staleynet_b200 import _ffi

HEADER = (Path(__file__).resolve().parents[1] / "include" / "snb_matmul.h").read_text()
FAKE = 0x1000   # never dereferenced


@pytest.mark.parametrize("struct,name", [(_ffi.VocabularyLossArgs, "snb_vocabulary_loss_args"),
                                         (_ffi.LayerNormArgs, "snb_layer_norm_args"),
                                         (_ffi.AdamW8Tensor, "snb_adamw8_tensor"),
                                         (_ffi.AdamW8Moments, "snb_adamw8_moments_out")])
def test_argument_blocks_have_the_headers_fields(struct, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for statement in body.split(";"):
        if statement.strip():
            kind, names = re.match(r"\s*((?:const\s+)?\w+\s*\**)\s*(.*)", statement, flags=re.S).groups()
            size = 8 if "*" in kind or "64" in kind else 4
            fields += [(n.strip(" *"), 8 if "*" in n else size) for n in names.split(",")]
    assert [(n, getattr(struct, n).size) for n, _ in struct._fields_] == fields


def _loss(**changes):
    a = _ffi.VocabularyLossArgs(rows=4, width=8, classes=10, type=_ffi.TYPE_BF16, weight_transposed=1, hidden=FAKE,
                                hidden_len=32, hidden_stride=8, weight=FAKE, weight_len=80, weight_stride=8, targets=FAKE,
                                targets_len=4, losses=FAKE, losses_len=4)
    for k, v in changes.items():
        setattr(a, k, v)
    code = _ffi.load().snb_vocabulary_cross_entropy(None, ctypes.byref(a))
    return code, _ffi.last_error()


@pytest.mark.parametrize("changes,code,message", [
    (dict(width=0), _ffi.ERR_INVALID_ARGUMENT, "at least 1"),
    (dict(classes=0), _ffi.ERR_INVALID_ARGUMENT, "at least 1"),
    (dict(rows=1 << 32), _ffi.ERR_INVALID_ARGUMENT, "out of range"),
    (dict(type=3), _ffi.ERR_INVALID_ARGUMENT, "unknown element type"),
    (dict(type=_ffi.TYPE_F32, weight_grad=FAKE, weight_grad_len=80, weight_grad_type=_ffi.TYPE_BF16),
     _ffi.ERR_INVALID_ARGUMENT, "f32 operands have f32 gradients"),
    (dict(flags=2), _ffi.ERR_INVALID_ARGUMENT, "unknown flags"),
    (dict(hidden_stride=7), _ffi.ERR_INVALID_ARGUMENT, "hidden_stride"),
    (dict(weight_stride=7), _ffi.ERR_INVALID_ARGUMENT, "weight_stride"),
    (dict(weight_transposed=0), _ffi.ERR_INVALID_ARGUMENT, "weight_stride"),
    (dict(weight_grad=FAKE, weight_grad_len=80, weight_grad_type=_ffi.TYPE_BF16, accumulate=1), _ffi.ERR_UNSUPPORTED,
     "accumulating"),
    (dict(hidden_len=31), _ffi.ERR_LEFT_TOO_SMALL, "hidden too small"),
    (dict(weight_len=79), _ffi.ERR_RIGHT_TOO_SMALL, "weight too small"),
    (dict(targets_len=3), _ffi.ERR_INVALID_ARGUMENT, "too few targets"),
    (dict(losses_len=3), _ffi.ERR_OUTPUT_TOO_SMALL, "losses too small"),
    (dict(hidden_grad=FAKE, hidden_grad_len=31), _ffi.ERR_OUTPUT_TOO_SMALL, "hidden_grad too small"),
    (dict(weight_grad=FAKE, weight_grad_len=79), _ffi.ERR_OUTPUT_TOO_SMALL, "weight_grad too small"),
    (dict(hidden=None), _ffi.ERR_INVALID_ARGUMENT, "null pointer"),
    (dict(targets=FAKE + 2), _ffi.ERR_INVALID_ARGUMENT, "not aligned"),
])
def test_vocabulary_loss_refusals(changes, code, message):
    got, text = _loss(**changes)
    assert got == code and message in text


def _norm(backward=False, **changes):
    a = _ffi.LayerNormArgs(rows=4, cols=8, input=FAKE, input_len=32, input_stride=8, gain=FAKE, bias=FAKE, params_len=8,
                           mean=FAKE, inv_std=FAKE, stats_len=4, output=FAKE, output_len=32, output_stride=8,
                           output_grad=FAKE, output_grad_len=32, output_grad_stride=8, input_grad=FAKE,
                           input_grad_len=32, input_grad_stride=8, gain_grad=FAKE)
    for k, v in changes.items():
        setattr(a, k, v)
    lib = _ffi.load()
    code = (lib.snb_layer_norm_backward if backward else lib.snb_layer_norm_forward)(None, ctypes.byref(a))
    return code, _ffi.last_error()


@pytest.mark.parametrize("backward,changes,code,message", [
    (False, dict(cols=0), _ffi.ERR_INVALID_ARGUMENT, "out of range"),
    (False, dict(params_len=7), _ffi.ERR_INVALID_ARGUMENT, "params length"),
    (False, dict(stats_len=3), _ffi.ERR_INVALID_ARGUMENT, "too small"),
    (False, dict(gain=None), _ffi.ERR_INVALID_ARGUMENT, "null pointer"),
    (False, dict(mean=FAKE + 1), _ffi.ERR_INVALID_ARGUMENT, "not aligned"),
    (False, dict(input_type=9), _ffi.ERR_INVALID_ARGUMENT, "unknown type"),
    (False, dict(input_stride=7), _ffi.ERR_INVALID_ARGUMENT, "input stride"),
    (False, dict(input_len=31), _ffi.ERR_INVALID_ARGUMENT, "input too small"),
    (False, dict(epsilon=-1.0), _ffi.ERR_INVALID_ARGUMENT, "epsilon"),
    (False, dict(output_len=31), _ffi.ERR_OUTPUT_TOO_SMALL, "output too small"),
    (True, dict(output_grad_len=31), _ffi.ERR_INVALID_ARGUMENT, "output_grad too small"),
    (True, dict(input_grad_stride=6), _ffi.ERR_INVALID_ARGUMENT, "input_grad stride"),
    (True, dict(gain_grad=None), _ffi.ERR_INVALID_ARGUMENT, "null pointer"),
])
def test_layer_norm_refusals(backward, changes, code, message):
    got, text = _norm(backward, **changes)
    assert got == code and message in text


def _adamw8(hyper=None, norm=1.0, workspace=FAKE, workspace_len=1 << 20, **changes):
    t = _ffi.AdamW8Tensor(parameter=FAKE, gradient=FAKE, first=FAKE, first_scale=FAKE, second=FAKE, second_scale=FAKE,
                          count=300)
    for k, v in changes.items():
        setattr(t, k, v)
    h = hyper or _ffi.AdamWHyper(1e-3, 0.9, 0.95, 1e-8, 0.0, 1)
    code = _ffi.load().snb_adamw8_step(None, ctypes.byref(t), 1, ctypes.byref(h), norm, 1, FAKE, workspace, workspace_len)
    return code, _ffi.last_error()


@pytest.mark.parametrize("changes,message", [
    (dict(gradient_type=5), "unknown gradient type in tensor 0"),
    (dict(second=None), "null pointer in tensor 0"),
    (dict(parameter=FAKE + 2), "not aligned"),
    (dict(norm=0.0), "max_gradient_norm"),
    (dict(norm=float("nan")), "max_gradient_norm"),
    (dict(hyper=_ffi.AdamWHyper(1e-3, 0.9, 0.95, 1e-8, 0.0, 0)), "steps count from 1"),
    (dict(workspace_len=100), "workspace holds 100 bytes"),
    (dict(workspace=FAKE + 4), "8-byte boundary"),
])
def test_adamw8_refusals(changes, message):
    got, text = _adamw8(**changes)
    assert got == _ffi.ERR_INVALID_ARGUMENT and message in text

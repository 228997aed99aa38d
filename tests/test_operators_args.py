"""The C ABI of processed logits, the 8-bit head and the token table without a GPU: descriptor layouts, refusals
before any launch, workspace sizes, and the Python layer's refusals of host tensors."""

import ctypes
import json
import math
import subprocess
from pathlib import Path

import pytest
import torch

from dsv41_rocm import (Int8Head, _lib, head_logits, inthead, process, process_logits, quantize_head, token_embedding,
                        token_embedding_backward)

HEADER = Path(__file__).resolve().parents[1] / "include" / "dsv41_rocm.h"
CLASSES = {"dsv41_process_desc": _lib.ProcessDesc, "dsv41_int_head_desc": _lib.IntHeadDesc,
           "dsv41_embed_desc": _lib.EmbedDesc, "dsv41_embed_grad_desc": _lib.EmbedGradDesc}


def test_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {", 'printf("{\\"x\\":0");']
    for name, cls in CLASSES.items():
        for field, _ in cls._fields_:
            lines.append(f'printf(",\\"{name}.{field}\\": %zu", offsetof({name}, {field}));')
        lines.append(f'printf(",\\"{name}\\": %zu", sizeof({name}));')
    for bit in ("BAD_PENALTY", "BAD_BIAS", "BAD_MASK", "NO_TOKEN"):
        lines.append(f'printf(",\\"{bit}\\": %d", DSV41_STATUS_{bit});')
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ['printf("}\\n");', "return 0; }"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = json.loads(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout)
    for name, cls in CLASSES.items():
        assert ctypes.sizeof(cls) == got[name] == getattr(_lib.load(), name + "_size")()
        for field, _ in cls._fields_:
            assert getattr(cls, field).offset == got[f"{name}.{field}"], (name, field)
    for bit in ("BAD_PENALTY", "BAD_BIAS", "BAD_MASK", "NO_TOKEN"):
        assert getattr(_lib, "STATUS_" + bit) == got[bit]


def _process(**kw):
    d = _lib.ProcessDesc()
    d.struct_size = ctypes.sizeof(d)
    d.rows, d.vocab, d.logits_dtype, d.logits_row_stride, d.logits = 4, 100, 0, 100, 0x1000
    d.repetition_penalty = 1.0
    d.out, d.out_row_stride, d.grad, d.grad_row_stride = 0x9000, 100, 0x5000, 100
    for k, v in kw.items():
        setattr(d, k, v)
    return d


PROCESS = [
    (dict(struct_size=8), _lib.E_ABI, "size mismatch"),
    (dict(rows=0), _lib.E_INVALID, "shape"),
    (dict(vocab=0), _lib.E_INVALID, "shape"),
    (dict(logits=None), _lib.E_INVALID, "required"),
    (dict(logits=0x1002), _lib.E_INVALID, "aligned"),
    (dict(logits_dtype=2), _lib.E_INVALID, "fp32 or bf16"),
    (dict(logits_row_stride=99), _lib.E_INVALID, "stride"),
    (dict(vocab=(1 << 21) + 1, logits_row_stride=1 << 22, out_row_stride=1 << 22), _lib.E_UNSUPPORTED, "2^21"),
    (dict(out=None), _lib.E_INVALID, "out is required"),
    (dict(out=0x9002), _lib.E_INVALID, "aligned"),
    (dict(out_row_stride=99), _lib.E_INVALID, "out row stride"),
    (dict(repetition_penalty=0.0), _lib.E_INVALID, "repetition_penalty must be finite and positive"),
    (dict(repetition_penalty=math.inf), _lib.E_INVALID, "repetition_penalty must be finite and positive"),
    (dict(presence_penalty=math.nan), _lib.E_INVALID, "must be finite"),
    (dict(frequency_penalty=math.inf), _lib.E_INVALID, "must be finite"),
    (dict(hist_len=-1), _lib.E_INVALID, "hist_len"),
    (dict(hist_len=5), _lib.E_INVALID, "hist_len needs a history"),
    (dict(hist_len=5, history=0x1000, history_row_stride=-5), _lib.E_INVALID, "history row stride"),
    (dict(hist_len=1 << 19, history=0x1000), _lib.E_UNSUPPORTED, "524287"),
    (dict(bias_len=-1), _lib.E_INVALID, "bias_len"),
    (dict(bias_len=3, bias=0x1000), _lib.E_INVALID, "bias_len needs"),
    (dict(bias_len=3, bias_ids=0x1000), _lib.E_INVALID, "bias_len needs"),
    (dict(bias_len=3, bias_ids=0x1000, bias=0x1000, bias_row_stride=-3), _lib.E_INVALID, "bias row stride"),
    (dict(bias_len=4096, bias_ids=0x1000, bias=0x1000), _lib.E_UNSUPPORTED, "4095"),
    (dict(mask=0x1000, masks=0), _lib.E_INVALID, "mask"),
    (dict(mask=0x1000, masks=3), _lib.E_INVALID, "one per row"),
    (dict(mask=0x1000, masks=1, mask_row_stride=-4), _lib.E_INVALID, "mask row stride"),
    (dict(fill=math.nan), _lib.E_INVALID, "fill"),
    (dict(rows=1 << 22), _lib.E_UNSUPPORTED, "row slices"),
]


@pytest.mark.parametrize("kw,code,msg", PROCESS)
@pytest.mark.parametrize("name", ["process", "process_grad"])
def test_process_refusals(name, kw, code, msg):
    assert getattr(_lib.load(), f"dsv41_{name}_run")(ctypes.byref(_process(**kw)), None) == code
    assert msg in _lib.last_error()


def test_process_in_place_refusals():
    lib = _lib.load()
    assert lib.dsv41_process_run(None, None) == lib.dsv41_process_grad_run(None, None) == _lib.E_INVALID
    assert lib.dsv41_process_run(ctypes.byref(_process(out=0x1000, out_row_stride=101)), None) == _lib.E_INVALID
    assert "in place" in _lib.last_error()
    for kw in (dict(grad=None), dict(grad=0x5001), dict(grad_row_stride=99), dict(out=0x5000), dict(out=0x1000)):
        assert lib.dsv41_process_grad_run(ctypes.byref(_process(**kw)), None) == _lib.E_INVALID


def _head(**kw):
    d = _lib.IntHeadDesc()
    d.struct_size = ctypes.sizeof(d)
    d.n_tokens, d.hidden, d.vocab = 20, 200, 100
    d.x, d.x_row_stride, d.w, d.scales = 0x1000, 200, 0x2000, 0x3000
    d.out, d.out_row_stride, d.out_dtype = 0x4000, 100, 0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,code,msg", [
    (dict(struct_size=8), _lib.E_ABI, "size mismatch"),
    (dict(n_tokens=-1), _lib.E_INVALID, "hidden must be"),
    (dict(vocab=0), _lib.E_INVALID, "hidden must be"),
    (dict(hidden=0), _lib.E_INVALID, "columns"),
    (dict(hidden=133121, x_row_stride=1 << 18), _lib.E_UNSUPPORTED, "overflow"),
    (dict(x=None), _lib.E_INVALID, "required"),
    (dict(w=None), _lib.E_INVALID, "required"),
    (dict(scales=None), _lib.E_INVALID, "required"),
    (dict(out=None), _lib.E_INVALID, "required"),
    (dict(out_dtype=2), _lib.E_INVALID, "fp32 or bf16"),
    (dict(x_row_stride=199), _lib.E_INVALID, "cover"),
    (dict(out_row_stride=99), _lib.E_INVALID, "cover"),
    (dict(w=0x2008), _lib.E_INVALID, "16-byte"),
    (dict(x=0x1001), _lib.E_INVALID, "aligned"),
    (dict(scales=0x3004), _lib.E_INVALID, "aligned"),
    (dict(out=0x4002), _lib.E_INVALID, "aligned"),
    (dict(n_tokens=(1 << 22) + 1), _lib.E_UNSUPPORTED, "too large"),
    (dict(vocab=(1 << 28) + 1, out_row_stride=1 << 29), _lib.E_UNSUPPORTED, "too large"),
])
def test_head_refusals(kw, code, msg):
    lib = _lib.load()
    d = _head(**kw)
    assert lib.dsv41_int_head_run(ctypes.byref(d), 0x8000, 1 << 30, None) == code
    assert msg in _lib.last_error()
    assert lib.dsv41_int_head_workspace_bytes(ctypes.byref(d)) == 0


def test_head_workspace():
    lib = _lib.load()
    d = _head()
    size = lib.dsv41_int_head_workspace_bytes(ctypes.byref(d))
    assert size >= 32 * 256 + 20 * 4
    for ws, n in ((None, size), (0x8000, size - 1), (0x8008, size)):
        assert lib.dsv41_int_head_run(ctypes.byref(d), ws, n, None) == _lib.E_WORKSPACE
    assert lib.dsv41_int_head_run(ctypes.byref(_head(n_tokens=0)), None, 0, None) == _lib.OK
    assert lib.dsv41_int_head_run(None, None, 0, None) == _lib.E_INVALID


@pytest.mark.parametrize("args", [
    (None, 200, 3, 200, 0x1000, 0x2000), (0x1001, 200, 3, 200, 0x1000, 0x2000), (0x1000, 199, 3, 200, 0x1000, 0x2000),
    (0x1000, 200, -1, 200, 0x1000, 0x2000), (0x1000, 200, 3, 0, 0x1000, 0x2000), (0x1000, 200, 3, 200, None, 0x2000),
    (0x1000, 200, 3, 200, 0x1008, 0x2000), (0x1000, 200, 3, 200, 0x1000, None), (0x1000, 200, 3, 200, 0x1000, 0x2002),
])
def test_quantize_refusals(args):
    assert _lib.load().dsv41_quantize_rows_run(*args, None, None) == _lib.E_INVALID
    assert _lib.load().dsv41_quantize_rows_run(0x1000, 1 << 20, 1, 133121, 0x1000, 0x2000, None, None) == _lib.E_UNSUPPORTED


def _embed(**kw):
    d = _lib.EmbedDesc()
    d.struct_size = ctypes.sizeof(d)
    d.n_tokens, d.hidden, d.vocab, d.weight, d.weight_row_stride, d.ids = 5, 16, 100, 0x1000, 16, 0x2000
    d.scale, d.dtype, d.out, d.out_row_stride = 1.0, 0, 0x3000, 16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _embed_grad(**kw):
    d = _lib.EmbedGradDesc()
    d.struct_size = ctypes.sizeof(d)
    d.n_tokens, d.hidden, d.vocab, d.ids, d.grad, d.grad_row_stride = 50, 16, 100, 0x2000, 0x1000, 16
    d.scale, d.out, d.out_row_stride = 1.0, 0x3000, 16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


TABLE = [
    (dict(struct_size=8), _lib.E_ABI, "size mismatch"),
    (dict(n_tokens=-1), _lib.E_INVALID, "shape"),
    (dict(hidden=0), _lib.E_INVALID, "shape"),
    (dict(vocab=0), _lib.E_INVALID, "shape"),
    (dict(ids=None), _lib.E_INVALID, "required"),
    (dict(out=None), _lib.E_INVALID, "required"),
    (dict(out=0x3002), _lib.E_INVALID, "aligned"),
    (dict(out_row_stride=15), _lib.E_INVALID, "cover"),
]


@pytest.mark.parametrize("kw,code,msg", TABLE + [
    (dict(dtype=2), _lib.E_INVALID, "fp32 or bf16"),
    (dict(weight=None), _lib.E_INVALID, "required"),
    (dict(weight=0x1002), _lib.E_INVALID, "aligned"),
    (dict(weight_row_stride=15), _lib.E_INVALID, "cover"),
])
def test_embed_refusals(kw, code, msg):
    assert _lib.load().dsv41_embed_run(ctypes.byref(_embed(**kw)), None) == code
    assert msg in _lib.last_error()
    assert _lib.load().dsv41_embed_run(None, None) == _lib.E_INVALID
    assert _lib.load().dsv41_embed_run(ctypes.byref(_embed(n_tokens=0, ids=None, out=None)), None) == _lib.OK


def test_checked_embed_refusals():
    run = _lib.load().dsv41_embed_checked_run
    assert run(ctypes.byref(_embed()), None, None) == _lib.E_INVALID and "flags" in _lib.last_error()
    assert run(ctypes.byref(_embed(hidden=0)), 0x4000, None) == _lib.E_INVALID
    assert run(None, 0x4000, None) == _lib.E_INVALID
    assert run(ctypes.byref(_embed(n_tokens=0, ids=None, out=None)), 0x4000, None) == _lib.OK


@pytest.mark.parametrize("kw,code,msg", TABLE + [
    (dict(grad=None), _lib.E_INVALID, "required"),
    (dict(grad=0x1002), _lib.E_INVALID, "aligned"),
    (dict(grad_row_stride=15), _lib.E_INVALID, "cover"),
    (dict(grad_row_stride=-16), _lib.E_INVALID, "cover"),
    (dict(grad_dtype=2), _lib.E_INVALID, "fp32 or bf16"),
    (dict(out_dtype=2), _lib.E_INVALID, "fp32 or bf16"),
    (dict(n_tokens=0x7FFFFFFF), _lib.E_UNSUPPORTED, "too large"),
])
def test_embed_grad_refusals(kw, code, msg):
    lib = _lib.load()
    d = _embed_grad(**kw)
    assert lib.dsv41_embed_grad_run(ctypes.byref(d), 0x8000, 1 << 40, None) == code
    assert msg in _lib.last_error()
    assert lib.dsv41_embed_grad_workspace_bytes(ctypes.byref(d)) == 0


@pytest.mark.parametrize("hidden", [(1 << 24) + 1, 0x7FFFFFFF])
def test_wide_tables_are_refused(hidden):
    # 32-bit column counts would pass their range in the last step of a row
    lib = _lib.load()
    wide = dict(hidden=hidden, out_row_stride=hidden)
    assert lib.dsv41_embed_run(ctypes.byref(_embed(weight_row_stride=hidden, **wide)), None) == _lib.E_UNSUPPORTED
    grad = _embed_grad(n_tokens=1, grad_row_stride=hidden, **wide)
    assert lib.dsv41_embed_grad_run(ctypes.byref(grad), 0x8000, 1 << 60, None) == _lib.E_UNSUPPORTED
    assert "2^24" in _lib.last_error()


def test_embed_grad_workspace():
    lib = _lib.load()
    d = _embed_grad()
    size = lib.dsv41_embed_grad_workspace_bytes(ctypes.byref(d))
    assert size > 50 * 8 + 100 // 8
    for ws, n in ((None, size), (0x8000, size - 1), (0x8004, size)):
        assert lib.dsv41_embed_grad_run(ctypes.byref(d), ws, n, None) == _lib.E_WORKSPACE
    assert lib.dsv41_embed_grad_run(None, None, 0, None) == _lib.E_INVALID


def test_ids_that_are_no_tensor_are_refused():
    with pytest.raises(ValueError, match="integers"):
        token_embedding_backward(torch.zeros(2, 5), [1, 2], 5)


def test_lists_that_are_no_tensors_are_refused():
    # by name, whatever else there is to refuse
    x, ids = torch.zeros(2, 10), torch.zeros(2, 3, dtype=torch.int64)

    def arguments(**kw):
        names = ("history", "history_lens", "history_prompt_lens", "repetition_penalty", "presence_penalty", "frequency_penalty",
                 "bias_ids", "bias", "token_mask", "mask_rows", "fill")
        neutral = {"repetition_penalty": 1.0, "presence_penalty": 0.0, "frequency_penalty": 0.0, "fill": 0.0}
        return process._arguments(x, *(kw.get(n, neutral.get(n)) for n in names))

    for bad in ([[1, 2, 3], [4, 5, 6]], 7, "ids"):
        with pytest.raises(ValueError, match="history must have shape"):
            arguments(history=bad)
        with pytest.raises(ValueError, match="bias_ids and bias must have shape"):
            arguments(bias_ids=ids, bias=bad)
        with pytest.raises(ValueError, match="bias_ids and bias must have shape"):
            arguments(bias_ids=bad, bias=x[:, :3])
        with pytest.raises(ValueError, match="token_mask must be"):
            arguments(token_mask=bad)
        with pytest.raises(ValueError, match="out must have the shape"):
            process._output(bad, x)


def test_heads_and_outs_that_are_no_tensors_are_refused():
    x, ids = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for bad in ([[1]], 3, None):
        with pytest.raises(ValueError, match="weight must be int8"):
            Int8Head.from_quantized(bad, x[0])
        with pytest.raises(ValueError, match="weight must be int8"):
            Int8Head.from_quantized(x.to(torch.int8), bad)
        with pytest.raises(ValueError, match="Int8Head"):
            inthead._check_head(bad, x)
    with pytest.raises(ValueError, match="Int8Head"):
        inthead._check_head(x, x)
    for bad in ([1], 3):
        with pytest.raises(ValueError, match="out must be"):
            token_embedding_backward(x, ids, out=bad)


def test_host_tensors_are_refused():
    x, ids = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: process_logits(x), lambda: head_logits(x, Int8Head(x.to(torch.int8), x[0], 2, 10)), lambda: quantize_head(x),
                 lambda: token_embedding(ids, x), lambda: token_embedding_backward(x, ids, 5),
                 lambda: Int8Head.from_quantized(x.to(torch.int8), x[:, 0])):
        with pytest.raises(ValueError, match="on the GPU"):
            call()
    for bad in (x[0], x[:, :0], [1.0]):
        with pytest.raises(ValueError, match="shape"):
            process_logits(bad)
    with pytest.raises(ValueError, match="weight must have shape"):
        token_embedding(ids, x[0])
    with pytest.raises(ValueError, match="grad must have the shape"):
        token_embedding_backward(x, ids[:1], 5)

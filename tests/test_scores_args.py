"""The scores' and the distillation's C ABI without a GPU: descriptor layouts, refusals before any
launch, workspace sizes, and the Python layer's refusals of host tensors."""

import ctypes
import json
import math
import subprocess
from pathlib import Path

import pytest
import torch

from dsv41_rocm import _lib, distillation_loss, logit_scores

HEADER = Path(__file__).resolve().parents[1] / "include" / "dsv41_rocm.h"
CLASSES = {"dsv41_scores_desc": _lib.ScoresDesc, "dsv41_scores_grad_desc": _lib.ScoresGradDesc,
           "dsv41_distill_desc": _lib.DistillDesc, "dsv41_distill_grad_desc": _lib.DistillGradDesc}


def test_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {", 'printf("{\\"x\\":0");']
    for name, cls in CLASSES.items():
        for field, _ in cls._fields_:
            lines.append(f'printf(",\\"{name}.{field}\\": %zu", offsetof({name}, {field}));')
        lines.append(f'printf(",\\"{name}\\": %zu", sizeof({name}));')
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ['printf("}\\n");', "return 0; }"]))
    subprocess.run(["gcc", "-o", str(exe), str(src)], check=True)
    got = json.loads(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout)
    for name, cls in CLASSES.items():
        assert ctypes.sizeof(cls) == got[name] == getattr(_lib.load(), name + "_size")()
        for field, _ in cls._fields_:
            assert getattr(cls, field).offset == got[f"{name}.{field}"], (name, field)


def _desc(cls, **kw):
    d = cls()
    d.struct_size = ctypes.sizeof(cls)
    d.rows, d.vocab, d.logits_dtype, d.logits_row_stride, d.logits, d.temperature = 4, 100, 0, 100, 0x1000, 1.0
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p:
            setattr(d, name, 0x1000)
    d.top_k = 5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


ROWS = [
    (dict(struct_size=8), _lib.E_ABI, "size mismatch"),
    (dict(rows=0), _lib.E_INVALID, "shape"),
    (dict(vocab=0), _lib.E_INVALID, "shape"),
    (dict(logits=None), _lib.E_INVALID, ""),
    (dict(logits=0x1002), _lib.E_INVALID, "aligned"),
    (dict(logits=0x1001, logits_dtype=1), _lib.E_INVALID, "aligned"),
    (dict(logits_dtype=2), _lib.E_INVALID, "fp32 or bf16"),
    (dict(logits_row_stride=99), _lib.E_INVALID, "stride"),
    (dict(logits_row_stride=-100), _lib.E_INVALID, "stride"),
    (dict(temperature=0.0), _lib.E_INVALID, "temperature must be finite and positive"),
    (dict(temperature=math.nan), _lib.E_INVALID, "temperature must be finite and positive"),
    (dict(temperature=1e-31), _lib.E_INVALID, "1e-30"),
    (dict(vocab=(1 << 21) + 1, logits_row_stride=1 << 22), _lib.E_UNSUPPORTED, "2^21"),
    (dict(rows=(1 << 22) + 1), _lib.E_UNSUPPORTED, "row slices"),
    # rows that are all the same one, each in 13 slices
    (dict(rows=1 << 20, vocab=1 << 21, logits_row_stride=0), _lib.E_UNSUPPORTED, "row slices"),
]


def _scores(d, ws=None, n=0):
    return _lib.load().dsv41_scores_run(ctypes.byref(d), ws, n, None)


@pytest.mark.parametrize("kw,code,msg", ROWS + [
    (dict(top_k=-1), _lib.E_INVALID, "top_k"),
    (dict(top_k=101), _lib.E_INVALID, "top_k"),
    (dict(vocab=2000, logits_row_stride=2000, top_k=1025), _lib.E_UNSUPPORTED, "1024"),
    (dict(out_entropy=None), _lib.E_INVALID, "out_entropy"),
    (dict(out_status=None), _lib.E_INVALID, "out_status"),
    (dict(out_logprob=None), _lib.E_INVALID, "targets need"),
    (dict(out_rank=None), _lib.E_INVALID, "targets need"),
    (dict(out_top_ids=None), _lib.E_INVALID, "top_k needs"),
    (dict(out_top_logprob=None), _lib.E_INVALID, "top_k needs"),
    (dict(vocab=100000, logits_row_stride=100000), _lib.E_WORKSPACE, "workspace"),
])
def test_scores_refusals(kw, code, msg):
    assert _scores(_desc(_lib.ScoresDesc, **kw)) == code
    assert msg in _lib.last_error()


def _distill(d, ws=None, n=0):
    return _lib.load().dsv41_distill_run(ctypes.byref(d), ws, n, None)


@pytest.mark.parametrize("kw,code,msg", ROWS + [
    (dict(top_k=0), _lib.E_INVALID, "at least one entry"),
    (dict(teacher_ids=None), _lib.E_INVALID, "teacher_ids"),
    (dict(teacher_logprob=None), _lib.E_INVALID, "teacher_logprob"),
    (dict(tail=2), _lib.E_INVALID, "tail"),
    (dict(out_loss=None), _lib.E_INVALID, "out_loss"),
    (dict(out_status=None), _lib.E_INVALID, "out_status"),
    (dict(vocab=100000, logits_row_stride=100000), _lib.E_WORKSPACE, "workspace"),
])
def test_distill_refusals(kw, code, msg):
    assert _distill(_desc(_lib.DistillDesc, **kw)) == code
    assert msg in _lib.last_error()


# a gradient's rows are cut into up to 512 slices, so a batch of them is refused by its rows alone
@pytest.mark.parametrize("kw,code,msg", [r for r in ROWS if r[0].get("rows") != 1 << 20] + [
    (dict(stats=None), _lib.E_INVALID, "stats"),
    (dict(out=None), _lib.E_INVALID, "out"),
    (dict(out=0x1002), _lib.E_INVALID, "aligned"),
])
@pytest.mark.parametrize("name", ["scores", "distill"])
def test_gradient_refusals(name, kw, code, msg):
    cls = CLASSES[f"dsv41_{name}_grad_desc"]
    d = _desc(cls, **kw)
    assert getattr(_lib.load(), f"dsv41_{name}_grad_run")(ctypes.byref(d), None) == code
    assert msg in _lib.last_error()


def test_gradients_need_what_they_belong_to():
    run = _lib.load().dsv41_scores_grad_run
    assert run(ctypes.byref(_desc(_lib.ScoresGradDesc, targets=None)), None) == _lib.E_INVALID
    assert run(ctypes.byref(_desc(_lib.ScoresGradDesc, top_ids=None)), None) == _lib.E_INVALID
    assert run(ctypes.byref(_desc(_lib.ScoresGradDesc, top_k=0)), None) == _lib.E_INVALID
    assert run(None, None) == _lib.E_INVALID
    for name in ("teacher_ids", "teacher_logprob", "grad_loss"):
        d = _desc(_lib.DistillGradDesc, **{name: None})
        assert _lib.load().dsv41_distill_grad_run(ctypes.byref(d), None) == _lib.E_INVALID


def test_workspaces():
    lib = _lib.load()
    for rows, vocab, k in ((1, 100, 5), (1, 129280, 5), (8, 151936, 1024), (300, 151936, 64), (5000, 151936, 64), (1, 1 << 21, 0)):
        kw = dict(rows=rows, vocab=vocab, logits_row_stride=vocab)
        a = lib.dsv41_scores_workspace_bytes(ctypes.byref(_desc(_lib.ScoresDesc, top_k=min(k, vocab), **kw)))
        b = lib.dsv41_distill_workspace_bytes(ctypes.byref(_desc(_lib.DistillDesc, **kw)))
        assert a % (rows * (24 + 8 * k)) == 0 and b % (rows * 32) == 0
        if rows == 5000 or vocab == 100:
            assert a == b == 0
        else:
            assert a > 0 and b > 0
    # a misaligned workspace and one that is a byte short
    d = _desc(_lib.ScoresDesc, rows=1, vocab=129280, logits_row_stride=129280)
    size = lib.dsv41_scores_workspace_bytes(ctypes.byref(d))
    for ws, n in ((0x1004, size), (0x1000, size - 1), (None, size)):
        assert _scores(d, ws, n) == _lib.E_WORKSPACE
    d = _desc(_lib.DistillDesc, rows=1, vocab=129280, logits_row_stride=129280)
    size = lib.dsv41_distill_workspace_bytes(ctypes.byref(d))
    for ws, n in ((0x1004, size), (0x1000, size - 1), (None, size)):
        assert _distill(d, ws, n) == _lib.E_WORKSPACE


def test_host_tensors_are_refused():
    x = torch.zeros(2, 10)
    ids, lq = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1)
    with pytest.raises(ValueError, match="on the GPU"):
        logit_scores(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="on the GPU"):
        distillation_loss(x, ids, lq)
    for T in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature must be finite and positive"):
            logit_scores(x, temperature=T)
        with pytest.raises(ValueError, match="temperature must be finite and positive"):
            distillation_loss(x, ids, lq, temperature=T)
    for bad in (x[0], x[:, :0], [1.0]):
        with pytest.raises(ValueError, match="shape"):
            logit_scores(bad)
        with pytest.raises(ValueError, match="shape"):
            distillation_loss(bad, ids, lq)

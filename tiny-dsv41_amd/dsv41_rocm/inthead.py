"""An 8-bit scoring head on MI355X: the head's rows as integers with a scale each, and logits from it.

The reference's rollout engine and learner take their logits from ``lm_head`` in bf16
(``dsv41_train/models/dsv4/model.py:635``, ``rollout_manager/backends/qwen_kv_cache.py:112-114``).  A decoding
step is bound by reading that head; in 8 bits it is half as long, and large batches multiply at twice
the rate.  Tokens sampled from such logits have the 8-bit head's distribution, which the Token-TIS
weights of ``decoupled_token_tis_loss`` and ``selected_log_probs`` correct for.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._check import any_set
from .scores import fit_int32, launch, overlap, refuse_capture, refuse_tangents, written

LINE, GROUP = 128, 64  # columns and rows are rounded up to these
LOWEST_COLUMNS = (2 ** 31 - 1) // (127 * 128)  # of rows that hold -128: their products' sums fit 32 bits

_OUT_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


@dataclass(frozen=True)
class Int8Head:
    """A head ``[vocab, hidden]`` whose row ``v`` is ``scales[v]`` times int8 integers: ``tiles`` holds them in the
    order in which the kernels read them, ``scales`` is fp32.  :meth:`integers` gives them back as rows."""

    tiles: torch.Tensor
    scales: torch.Tensor
    vocab: int
    hidden: int

    @staticmethod
    def from_quantized(weight: torch.Tensor, scales: torch.Tensor) -> "Int8Head":
        """The head of int8 rows and their scales that a checkpoint holds, laid out for the kernels (a copy).  Rows of more
        than 132104 columns may not hold -128."""
        if not (isinstance(weight, torch.Tensor) and isinstance(scales, torch.Tensor)):
            raise ValueError("weight must be int8 [vocab, hidden], with one scale per row")
        if not (weight.is_cuda and scales.is_cuda):
            raise ValueError("weight and scales must be on the GPU (libdsv41hip has no CPU path)")
        if weight.ndim != 2 or weight.dtype != torch.int8 or 0 in weight.shape:
            raise ValueError("weight must be int8 [vocab, hidden]")
        if scales.shape != weight.shape[:1] or not scales.is_floating_point():
            raise ValueError("scales must have one value per row of weight")
        v, h = weight.shape
        if h > LOWEST_COLUMNS and int(weight.amin()) == -128:
            raise NotImplementedError(f"rows that hold -128 have at most {LOWEST_COLUMNS} columns: more overflow a 32-bit sum")
        tiles = torch.zeros(_rounded(v, GROUP), _rounded(h, LINE), dtype=torch.int8, device=weight.device)
        tiles[:v, :h] = weight
        # group, (tile, row in four) of a group, four in a tile; column tile, 16 columns of it
        tiles = tiles.view(-1, 4, 4, 4, tiles.shape[1] // 64, 4, 16).permute(0, 2, 4, 5, 1, 3, 6).contiguous()
        scales = scales.detach().to(device=weight.device, dtype=torch.float32, copy=True).contiguous()
        return Int8Head(tiles.view(-1), scales, v, h)

    def integers(self) -> torch.Tensor:
        """The int8 rows ``[vocab, hidden]`` (a copy)."""
        t = self.tiles.view(-1, 4, _rounded(self.hidden, LINE) // 64, 4, 4, 4, 16).permute(0, 4, 1, 5, 2, 3, 6)
        return t.reshape(_rounded(self.vocab, GROUP), -1)[:self.vocab, :self.hidden].contiguous()


def _rounded(n, unit):
    return (n + unit - 1) // unit * unit


def _rows(x, name):
    """Validated bf16 rows on the GPU; other dtypes are rounded to bf16."""
    if not isinstance(x, torch.Tensor) or x.ndim != 2:
        raise ValueError(f"{name} must be a matrix")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on the GPU (libdsv41hip has no CPU path)")
    if not x.is_floating_point():
        raise ValueError(f"{name} must be floating point")
    refuse_tangents(name, x)
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"the 8-bit head has no gradient: detach {name}, or call under no_grad")
    fit_int32(*x.shape)
    x = x.detach().to(torch.bfloat16)
    if x.stride(1) != 1 and x.shape[1] > 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def quantize_head(weight: torch.Tensor, *, check: bool = True) -> Int8Head:
    """The 8-bit head of a head ``weight [vocab, hidden]`` (bf16; other dtypes are rounded to it):
    ``scales[v] = max|weight[v]| / 127`` and ``rint(127 weight / max|weight|)``, ties to even.

    With ``check`` the call synchronises and raises ``ValueError`` for a row with a NaN or an infinity;
    without, such a row's scale, and so its logits, are NaN.
    """
    w = _rows(weight, "weight")
    v, h = w.shape
    if v == 0 or h == 0:
        raise ValueError("weight must be [vocab, hidden]")
    refuse_capture(check)
    tiles = torch.zeros(_rounded(v, GROUP) * _rounded(h, LINE), dtype=torch.int8, device=w.device)
    scales = torch.empty(v, dtype=torch.float32, device=w.device)
    status = torch.empty(v, dtype=torch.int32, device=w.device) if check else None
    launch(_lib.load().dsv41_quantize_rows_run, w.device, w.data_ptr(), w.stride(0) if v > 1 else h, v, h,
           tiles.data_ptr(), scales.data_ptr(), None if status is None else status.data_ptr())
    if check and any_set(status)[0]:
        raise ValueError("weight contains non-finite values")
    return Int8Head(tiles, scales, v, h)


def _check_head(head, x):
    if not isinstance(head, Int8Head):
        raise ValueError("the head must be an Int8Head: make it with quantize_head or Int8Head.from_quantized")
    v, h = head.vocab, head.hidden
    if x.shape[1] != h:
        raise ValueError("hidden must be [tokens, hidden] and the head [vocab, hidden]")
    if head.tiles.device != x.device or head.scales.device != x.device:
        raise ValueError("hidden and the head must be on the same GPU")
    if head.tiles.dtype != torch.int8 or not head.tiles.is_contiguous() or \
            head.tiles.numel() != _rounded(v, GROUP) * _rounded(h, LINE) or \
            head.scales.dtype != torch.float32 or head.scales.shape != (v,) or not head.scales.is_contiguous():
        raise ValueError("the head is not in the kernels' layout: make it with quantize_head or Int8Head.from_quantized")


def _forward(x, head, out, want_status):
    """One dsv41_int_head_run into ``out``; returns the statuses or None."""
    n, h, v = x.shape[0], head.hidden, head.vocab
    status = torch.empty(n, dtype=torch.int32, device=x.device) if want_status else None
    if n:
        d = _lib.IntHeadDesc(ctypes.sizeof(_lib.IntHeadDesc), n, h, v, x.data_ptr(), x.stride(0) if n > 1 else h,
                             head.tiles.data_ptr(), head.scales.data_ptr(), out.data_ptr(),
                             out.stride(0) if n > 1 else max(v, out.stride(0)), _OUT_DTYPES[out.dtype],
                             None if status is None else status.data_ptr())
        lib = _lib.load()
        ref = ctypes.byref(d)
        size = lib.dsv41_int_head_workspace_bytes(ref)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        launch(lib.dsv41_int_head_run, x.device, ref, ws.data_ptr(), size)
    return status


def _new_logits(n, v, dtype, device):
    """Logits whose rows begin at multiples of 64 elements."""
    return torch.empty(n, _rounded(v, 64), dtype=dtype, device=device)[:, :v]


def head_logits(
    hidden: torch.Tensor,
    head: Int8Head,
    *,
    dtype: torch.dtype = torch.float32,
    out: Optional[torch.Tensor] = None,
    check: bool = True,
) -> torch.Tensor:
    """Logits ``[tokens, vocab]`` of hidden states ``[tokens, hidden]`` (bf16; other dtypes are rounded to it)
    from an 8-bit head, fp32 or bf16.

    Each row of ``hidden`` becomes integers as the head's rows are, ``rint(127 x / max|x|)`` with the scale
    ``max|x| / 127``; their products with the head's rows are summed exactly, then multiplied by the two
    scales in fp32.  A row's logits do not depend on the batch it is in.

    The result's rows begin at multiples of 64 elements, so that of a vocabulary that is none it is a
    view; ``out`` (rows at any stride that holds them, in memory of their own) takes it instead.  There is no gradient:
    hidden states that require one are refused where it is recorded (:func:`selected_log_probs` is the learner's head).

    With ``check`` the call synchronises and raises ``ValueError`` for hidden states with a NaN or an
    infinity; without, their rows are NaN.
    """
    x = _rows(hidden, "hidden")
    _check_head(head, x)
    n, v = x.shape[0], head.vocab
    given = out
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.shape != (n, v) or out.dtype not in _OUT_DTYPES or out.device != x.device:
            raise ValueError("out must be fp32 or bf16 [tokens, vocab] on the GPU of the hidden states")
        if v > 1 and out.stride(1) != 1 or n > 1 and out.stride(0) < v:
            raise ValueError("out must have contiguous rows that do not overlap")
        if out.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("the 8-bit head has no gradient: call under no_grad")
        if overlap(out, x, head.tiles, head.scales):
            raise ValueError("out overlaps the hidden states or the head")
    elif dtype not in _OUT_DTYPES:
        raise ValueError("logits are torch.float32 or torch.bfloat16")
    else:
        out = _new_logits(n, v, dtype, x.device)
    refuse_capture(check)
    status = _forward(x, head, out, check)
    if given is not None:
        written(given)
    if check and any_set(status)[0]:
        raise ValueError("hidden states contain non-finite values")
    return out

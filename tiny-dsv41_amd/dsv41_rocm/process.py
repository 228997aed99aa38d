"""Processed rows of logits on MI355X: biases, penalties for repeated tokens and token masks, with knobs
for each row, differentiable in the logits.

Reference (paths relative to the Tiny-DSV41 tree): ``rollout_manager/backends/vllm_actor.py:178-185`` names
the penalties among an engine's SamplingParams and ``:260`` takes log-probs under the processed
distribution.  ``sample`` applies one batch's penalties inside its draw; here they, and what engines apply
beside them, come as rows of logits that ``sample``, ``logit_scores`` and ``distillation_loss`` take.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Union

import torch

from . import _lib
from ._check import any_set
from .logprob import first_order
from .scores import INTEGERS, launch, overlap, refuse_capture, refuse_tangents, row_fields, rows_of_logits, vector, written

Knob = Union[float, torch.Tensor]


def _ready(t, dtype, rows, device):
    """Whether ``t`` is a vector of one value per row as the kernels take it."""
    return t.dtype is dtype and t.shape == (rows,) and t.device == device and t.is_contiguous()


def _knob(value, name, neutral, rows, device):
    """(the scalar of all rows, a tensor of one value per row or None)"""
    if isinstance(value, torch.Tensor):
        if _ready(value, torch.float32, rows, device) and not value.requires_grad:
            refuse_tangents(name, value)
            return neutral, value
        if value.shape != (rows,):
            raise ValueError(f"{name} must be a number or have one value per row")
        if value.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"{name} has no gradient: detach it")
        refuse_tangents(name, value)
        return neutral, vector(value, torch.float32, (rows,), device)
    value = float(value)
    if not math.isfinite(value) or neutral and value <= 0:
        raise ValueError("repetition_penalty must be finite and positive" if neutral
                         else "presence_penalty and frequency_penalty must be finite")
    return value, None


def _integers(t, name, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in INTEGERS:
        raise ValueError(f"{name} must be integers")
    if t.dtype != dtype or t.device != device:
        if dtype == torch.int32 and t.dtype == torch.int64:  # (what 32 bits would wrap stays out of range)
            t = t.clamp(-(1 << 31), (1 << 31) - 1)
        t = t.to(device=device, dtype=dtype)
    return t


def _lengths(t, name, rows, device):
    if isinstance(t, torch.Tensor) and _ready(t, torch.int32, rows, device):
        return t
    t = _integers(torch.as_tensor(t), name, torch.int32, device)
    if t.shape != (rows,):
        raise ValueError(f"{name} must have one length per row")
    return t.contiguous()


def _rows_of(t):
    """A matrix whose rows are contiguous, at any row stride that is not negative."""
    return t.contiguous() if t.shape[1] > 1 and t.stride(1) != 1 else t


def _step(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _arguments(logits, history, history_lens, history_prompt_lens, repetition_penalty, presence_penalty,
               frequency_penalty, bias_ids, bias, token_mask, mask_rows, fill):
    """Validated arguments in kernel form: the numbers, and the tensors (or None) that :func:`_fields` takes."""
    rows, vocab = logits.shape
    dev = logits.device
    rp, rps = _knob(repetition_penalty, "repetition_penalty", 1.0, rows, dev)
    pres, press = _knob(presence_penalty, "presence_penalty", 0.0, rows, dev)
    freq, freqs = _knob(frequency_penalty, "frequency_penalty", 0.0, rows, dev)
    if history is not None:
        if not isinstance(history, torch.Tensor) or history.ndim != 2 or history.shape[0] != rows:
            raise ValueError("history must have shape [rows, history_length]")
        history = _rows_of(_integers(history, "history", torch.int64, dev))
        if history_lens is not None:
            history_lens = _lengths(history_lens, "history_lens", rows, dev)
        if history_prompt_lens is not None:
            history_prompt_lens = _lengths(history_prompt_lens, "history_prompt_lens", rows, dev)
    elif history_lens is not None or history_prompt_lens is not None:
        raise ValueError("history_lens and history_prompt_lens require a history")
    if bias is not None and bias_ids is not None:
        if not (isinstance(bias, torch.Tensor) and isinstance(bias_ids, torch.Tensor)):
            raise ValueError("bias_ids and bias must have shape [rows, entries] or [entries]")
        if bias.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("bias has no gradient: detach it")
        refuse_tangents("biases", bias)
        if not bias.is_floating_point() or bias.shape != bias_ids.shape or bias.ndim not in (1, 2) or \
                bias.ndim == 2 and bias.shape[0] != rows:
            raise ValueError("bias_ids and bias must have shape [rows, entries] or [entries]")
        bias_ids = _integers(bias_ids, "bias_ids", torch.int64, dev).contiguous()
        bias = vector(bias, torch.float32, bias.shape, dev)
    elif bias is not None or bias_ids is not None:
        raise ValueError("bias_ids and bias are given together")
    if token_mask is not None:
        if not isinstance(token_mask, torch.Tensor) or token_mask.dtype != torch.int32 or \
                token_mask.ndim not in (1, 2) or token_mask.shape[-1] < (vocab + 31) // 32:
            raise ValueError("token_mask must be int32 words, one bit per token: [masks, ceil(vocabulary_size / 32)]")
        if token_mask.ndim == 1:
            token_mask = token_mask[None]
        if token_mask.device != dev:
            token_mask = token_mask.to(dev)
        token_mask = _rows_of(token_mask)
        masks = token_mask.shape[0]
        if mask_rows is not None:
            if not (isinstance(mask_rows, torch.Tensor) and _ready(mask_rows, torch.int32, rows, dev)):
                mask_rows = _integers(mask_rows, "mask_rows", torch.int32, dev).contiguous()
                if mask_rows.shape != (rows,):
                    raise ValueError("mask_rows must have one mask per row")
        elif masks != 1 and masks != rows:
            raise ValueError("without mask_rows there is one token_mask, or one per row")
        if masks == 0 and rows:
            raise ValueError("token_mask holds no mask")
    elif mask_rows is not None:
        raise ValueError("mask_rows requires a token_mask")
    fill = float(fill)
    if math.isnan(fill):
        raise ValueError("fill must be a number")
    return (rp, pres, freq, fill), (rps, press, freqs, history, history_lens, history_prompt_lens, bias_ids, bias,
                                    token_mask, mask_rows)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fields(numbers, tensors):
    """The descriptor's values from history to fill.  (Formed anew in the backward: what a graph saved may have been
    moved, to the host and back, in between.)"""
    rp, pres, freq, fill = numbers
    rps, press, freqs, history, lens, prompts, ids, bias, mask, which = tensors
    return (*((None, 0, 0) if history is None else (history.data_ptr(), _step(history), history.shape[1])), _ptr(lens),
            _ptr(prompts), rp, pres, freq, _ptr(rps), _ptr(press), _ptr(freqs), _ptr(ids), _ptr(bias),
            *((0, 0) if bias is None else (bias.shape[-1] if bias.ndim == 2 else 0, bias.shape[-1])),
            *((0, None, 0) if mask is None else (mask.shape[0], mask.data_ptr(), _step(mask))), _ptr(which), fill)


def forward(logits, numbers, tensors, out, want_status):
    """One dsv41_process_run into ``out``; returns the statuses or None."""
    rows, vocab = logits.shape
    status = torch.empty(rows, dtype=torch.int32, device=logits.device) if want_status else None
    if rows:
        d = _lib.ProcessDesc(*row_fields(_lib.ProcessDesc, logits), *_fields(numbers, tensors), out.data_ptr(),
                             out.stride(0) if rows > 1 else vocab, _ptr(status), None, 0)
        launch(_lib.load().dsv41_process_run, logits.device, ctypes.byref(d))
    return status


def process_backward(logits, numbers, tensors, grad):
    """dL/dlogits of :func:`process_logits` from dL/dresult, in the logits' dtype."""
    refuse_tangents("gradients", grad)
    rows, vocab = logits.shape
    out = logits.new_empty(rows, vocab)
    if rows:
        grad = grad.to(logits.dtype)
        step, unit = grad.stride()
        if unit != 1 and vocab > 1 or rows > 1 and 0 < step < vocab:
            grad = grad.contiguous()
            step = vocab
        d = _lib.ProcessDesc(*row_fields(_lib.ProcessDesc, logits), *_fields(numbers, tensors), out.data_ptr(), vocab, None,
                             grad.data_ptr(), step if rows > 1 else vocab)
        launch(_lib.load().dsv41_process_grad_run, logits.device, ctypes.byref(d))
    return out


class _Process(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, numbers, want_status, *tensors):
        out = logits.new_empty(logits.shape)
        status = forward(logits, numbers, tensors, out, want_status)
        ctx.numbers = numbers
        ctx.save_for_backward(logits, *tensors)
        ctx.set_materialize_grads(False)
        if status is not None:
            ctx.mark_non_differentiable(status)
        return out, status

    @staticmethod
    def backward(ctx, grad, g_status):
        logits, *tensors = ctx.saved_tensors
        nothing = (None,) * (2 + len(tensors))
        if grad is None:
            return None, *nothing
        return first_order(process_backward(logits, ctx.numbers, tensors, grad), logits, grad), *nothing


def _status_error(status: torch.Tensor) -> None:
    bits = 0
    for v in status.unique().tolist():
        bits |= int(v)
    if bits & _lib.STATUS_BAD_PENALTY:
        raise ValueError("repetition penalties must be finite and positive, the other penalties finite")
    if bits & _lib.STATUS_BAD_MASK:
        raise ValueError("mask_rows names a mask that there is not")
    if bits & _lib.STATUS_BAD_HISTORY:
        raise ValueError("history token ID is outside the model vocabulary")
    if bits & _lib.STATUS_BAD_BIAS:
        raise ValueError("biased token ID is outside the model vocabulary")
    if bits & _lib.STATUS_NO_TOKEN:
        raise ValueError("token mask leaves a row without tokens")


def _output(out, logits):
    """A validated ``out``: the logits' own tensor, or one that does not touch their memory."""
    if not isinstance(out, torch.Tensor) or out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the shape, dtype and device of the logits")
    rows, vocab = out.shape
    if vocab > 1 and out.stride(1) != 1 or rows > 1 and out.stride(0) < vocab:
        raise ValueError("out must have contiguous rows that do not overlap")
    same = out is logits or out.data_ptr() == logits.data_ptr() and (rows == 1 or out.stride(0) == logits.stride(0))
    if not same and overlap(out, logits):
        raise ValueError("out overlaps the logits without being them")
    return out


def process_logits(
    logits: torch.Tensor,
    *,
    history: Optional[torch.Tensor] = None,
    history_lens: Optional[torch.Tensor] = None,
    history_prompt_lens: Optional[torch.Tensor] = None,
    repetition_penalty: Knob = 1.0,
    presence_penalty: Knob = 0.0,
    frequency_penalty: Knob = 0.0,
    bias_ids: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    token_mask: Optional[torch.Tensor] = None,
    mask_rows: Optional[torch.Tensor] = None,
    fill: float = -math.inf,
    out: Optional[torch.Tensor] = None,
    check: bool = True,
) -> torch.Tensor:
    """Rows of logits with biases added, penalties applied and masked tokens filled, in that order.

    ``logits [rows, V]`` are fp32 or bf16 on the GPU (other dtypes are converted to fp32), rows at any
    stride; arithmetic is fp32 and the result has their dtype.

    * ``bias_ids``, ``bias`` (``[rows, entries]``, or ``[entries]`` for every row): logits of these tokens
      are raised by these values; of a token named twice the last entry counts, as in a dictionary.  Up to 4095 entries.
    * ``history``, ``history_lens``, ``history_prompt_lens`` and the penalties are those of :func:`sample`,
      bit for bit, with each penalty a number or a tensor of one value per row.  A row with
      neutral penalties does not read its history.
    * ``token_mask`` (int32 words ``[masks, ceil(V / 32)]`` or one mask): token ``i`` is allowed where bit
      ``i % 32`` of word ``i // 32`` is set; others become ``fill``.  ``mask_rows [rows]`` names each row's
      mask, -1 for none; without it there is one mask, or one per row.

    Negative ids are padding.  ``logit_scores`` and ``distillation_loss`` take ``-inf`` for masked tokens;
    ``sample`` takes finite logits only, so masks for it come with a finite ``fill`` that stays finite in the logits' type
    and when divided by the temperature, and is 40 temperatures or more below the logits (-8192, say).

    ``out`` takes the result; it may be ``logits`` itself, in which case only what changes is written.  A call
    with ``out`` has no gradient.  Otherwise the result is differentiable in ``logits``, once, in backward
    mode: masked tokens get 0, tokens of the history their repetition penalty's factor.

    With ``check`` the call synchronises and raises ``ValueError`` for ids outside the vocabulary, invalid
    penalties, a mask that there is not, or one that leaves a row no token; without, such ids
    are ignored, and rows of such penalties and masks hold NaN.
    """
    logits = rows_of_logits(logits, 1.0)
    numbers, tensors = _arguments(logits, history, history_lens, history_prompt_lens, repetition_penalty, presence_penalty,
                                  frequency_penalty, bias_ids, bias, token_mask, mask_rows, fill)
    refuse_capture(check)
    tracked = torch.is_grad_enabled() and logits.requires_grad
    if out is not None:
        out = _output(out, logits)
        if tracked or torch.is_grad_enabled() and out.requires_grad:
            raise ValueError("a call with out has no gradient: leave it out, or call under no_grad")
        status = forward(logits, numbers, tensors, out, check)
        written(out)
    elif tracked:
        out, status = _Process.apply(logits, numbers, check, *tensors)
    else:
        out = logits.new_empty(logits.shape)  # (half of torch.empty's 2.2 us)
        status = forward(logits, numbers, tensors, out, check)
    if check and any_set(status)[0]:
        _status_error(status)
    return out

"""Distillation from a teacher's top tokens on MI355X: each row's divergence of the student from the
teacher's list, differentiable in the student's logits.

The reference has no distillation; this loss stands beside its policy losses (``dsv41_train/rl/
algorithm.py:169-346``, here ``grpo_loss`` and ``decoupled_token_tis_loss``).  The lists are what
``logit_scores(teacher_logits, top_k=K, temperature=T)`` returns, or what a teacher's record holds of it.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._check import any_set
from .logprob import first_order
from .scores import INTEGERS, fit_int32, launch, refuse_capture, refuse_tangents, row_fields, rows_of_logits, vector

STATS = 7  # fp64 values of a row that the backward needs of the forward
_TAILS = {"renormalize": _lib.TAIL_RENORMALIZE, "rest": _lib.TAIL_REST}


def prepare(logits, teacher_ids, teacher_log_probs, temperature, tail):
    """Validated arguments in kernel form."""
    logits = rows_of_logits(logits, temperature)
    rows = logits.shape[0]
    if tail not in _TAILS:
        raise ValueError("tail must be 'renormalize' or 'rest'")
    shape, device = teacher_ids.shape, logits.device
    for t in (teacher_ids, teacher_log_probs):
        if t.ndim != 2 or t.shape[0] != rows:
            raise ValueError("teacher_ids and teacher_log_probs must have shape [rows, entries]")
    fit_int32(*shape)
    if teacher_log_probs.shape != shape:
        raise ValueError("one teacher log probability is required per teacher ID")
    if teacher_ids.dtype not in INTEGERS:
        raise ValueError("teacher_ids must be integers")
    ids = vector(teacher_ids, torch.int64, shape, device)
    # (detached also where no gradient is required: a forward-mode tangent ends here too)
    lq = vector(teacher_log_probs.detach(), torch.float32, shape, device)
    if shape[1] == 0:  # no row has an entry
        ids, lq = ids.new_full((rows, 1), -1), lq.new_zeros(rows, 1)
    return logits, ids, lq


def forward(logits, ids, lq, temperature, tail, want_stats):
    """One dsv41_distill_run; returns (loss, statuses, stats or None)."""
    rows, dev = logits.shape[0], logits.device
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    status = torch.empty(rows, dtype=torch.int32, device=dev)
    stats = torch.empty(rows, STATS, dtype=torch.float64, device=dev) if want_stats else None
    if rows:
        d = _lib.DistillDesc(*row_fields(_lib.DistillDesc, logits), ids.data_ptr(), lq.data_ptr(), temperature, ids.shape[1],
                             _TAILS[tail], loss.data_ptr(), status.data_ptr(), None if stats is None else stats.data_ptr())
        lib = _lib.load()
        ref = ctypes.byref(d)
        size = lib.dsv41_distill_workspace_bytes(ref)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        launch(lib.dsv41_distill_run, dev, ref, None if ws is None else ws.data_ptr(), size)
    return loss, status, stats


def distillation_backward(logits, ids, lq, temperature, stats, g_loss):
    """dL/dlogits of :func:`distillation_loss`, in the logits' dtype."""
    refuse_tangents("gradients", g_loss)
    rows, vocab = logits.shape
    out = torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
    if rows:
        g_loss = vector(g_loss, torch.float32, (rows,), logits.device)
        d = _lib.DistillGradDesc(*row_fields(_lib.DistillGradDesc, logits), ids.data_ptr(), lq.data_ptr(), temperature,
                                 ids.shape[1], stats.data_ptr(), g_loss.data_ptr(), out.data_ptr())
        launch(_lib.load().dsv41_distill_grad_run, logits.device, ctypes.byref(d))
    return out


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, lq, temperature, tail):
        loss, status, stats = forward(logits, ids, lq, temperature, tail, True)
        ctx.temperature = temperature
        ctx.save_for_backward(logits, ids, lq, stats)
        ctx.mark_non_differentiable(status)
        return loss, status

    @staticmethod
    def backward(ctx, g_loss, g_status):
        logits, ids, lq, stats = ctx.saved_tensors
        grad = distillation_backward(logits, ids, lq, ctx.temperature, stats, g_loss)
        return first_order(grad, logits, g_loss), None, None, None, None


def _status_error(status: torch.Tensor) -> None:
    bits = 0
    for v in status.unique().tolist():
        bits |= int(v)
    if bits & _lib.STATUS_BAD_TARGET:
        raise ValueError("teacher token ID is outside the model vocabulary")
    if bits & _lib.STATUS_REPEATED:
        raise ValueError("a teacher's list names a token twice")
    if bits & _lib.STATUS_BAD_TEACHER:
        raise ValueError("teacher log probabilities do not form a distribution")
    if bits & _lib.STATUS_NONFINITE:
        raise ValueError("distillation loss contains non-finite values")


def distillation_loss(
    logits: torch.Tensor,
    teacher_ids: torch.Tensor,
    teacher_log_probs: torch.Tensor,
    *,
    temperature: float = 1.0,
    tail: str = "renormalize",
    check: bool = True,
) -> torch.Tensor:
    """Each row's Kullback-Leibler divergence ``sum q (log q - log p)`` of the student ``p =
    softmax(logits / temperature)`` from a teacher's list of top tokens, fp32 ``[rows]``.

    ``logits [rows, V]`` are the student's, fp32 or bf16 on the GPU (other dtypes are converted to fp32),
    rows at any stride, ``-inf`` for a masked token.  ``teacher_ids [rows, K]`` (int64) and
    ``teacher_log_probs [rows, K]`` are the teacher's, taken at the same temperature; a negative id is no
    entry, so lists may be ragged, and a row without entries has loss and gradient 0 whatever its logits.

    ``tail``: ``"renormalize"`` makes the list a distribution of its own (``q = softmax`` of its
    log-probs, so raw logits divided by the temperature do as well); ``"rest"`` takes ``q = exp`` of them
    and compares what is left of the teacher's mass, ``1 - sum q``, with the student's mass outside the
    list as one more outcome (a rest below 2^-20, which fp32 log-probs do not carry, counts as 0).  The
    student's mass there counts however small it is, and is none where its logits are all -inf or all the lowest
    value of the dtype that the kernel reads (fp32 or bf16), below the list's.

    Differentiable in ``logits``, once (no second derivatives), and not in forward mode: logits that carry a
    tangent are refused; the teacher's tensors are constants.
    The gradient is with respect to the logits before the division by ``temperature``; callers that
    keep gradients of several temperatures alike multiply the loss by its square.

    With ``check`` the call synchronises and raises ``ValueError`` for an id at or above V, a token named
    twice in a row, teacher values that form no distribution (NaN, +inf, no mass to renormalize, more than
    1.01 of it with ``"rest"``) or a loss that is not finite (a masked token that the teacher gives mass,
    NaN or +inf logits); without, such a row's loss is NaN, or inf.
    """
    logits, ids, lq = prepare(logits, teacher_ids, teacher_log_probs, temperature, tail)
    refuse_capture(check)
    if torch.is_grad_enabled() and logits.requires_grad:
        loss, status = _Distillation.apply(logits, ids, lq, temperature, tail)
    else:
        loss, status, _ = forward(logits, ids, lq, temperature, tail, False)
    if check and any_set(status)[0]:
        _status_error(status)
    return loss

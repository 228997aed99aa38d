"""Scores of rows of logits on MI355X: log-probs and ranks of given tokens, entropy and the top
alternatives, differentiable in the logits.

Reference (paths relative to the Tiny-DSV41 tree): ``dsv41_train/rl/rollout.py:144-150`` forms a step's
``log_softmax(logits.float() / T)`` and takes the token's entry; ``rollout_manager/backends/
vllm_actor.py:260`` takes a token's log-prob from an engine whose ``logprobs`` output also names the top
alternatives and the token's rank.  Here one pass over each row gives all of them, where the logits are
at hand; ``selected_log_probs`` does it from hidden states, without alternatives.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._check import any_set
from .logprob import first_order
from .sampling import validate_temperature

INTEGERS = frozenset((torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8))


@dataclass
class LogitScores:
    """Per-row outputs of :func:`logit_scores`: the targets' log-probs (fp32) and ranks (int64, 1 = the
    most likely token), both None without targets; entropies (fp32); the top alternatives' ids (int64,
    -1 past the unmasked tokens) and log-probs (fp32, -inf there), ``[rows, top_k]``."""

    log_probs: Optional[torch.Tensor]
    ranks: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_log_probs: torch.Tensor


_KERNEL_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def fit_int32(*sizes) -> None:
    """Refuses sizes that a descriptor's int32 would wrap."""
    if max(sizes) > 0x7FFFFFFF:
        raise NotImplementedError("sizes above 2^31 - 1 are not supported")


def refuse_tangents(what, *tensors) -> None:
    """The kernels would leave them out."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no level is open, so nothing carries one (1 us a tensor)
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} carry a forward-mode tangent, for which there is no rule: detach them")


def rows_of_logits(logits, temperature):
    """Validated fp32 or bf16 logits [rows, V] whose rows are contiguous."""
    validate_temperature(temperature)
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must have shape [rows, vocabulary_size]")
    refuse_tangents("logits", logits)
    if not logits.is_cuda:
        raise ValueError("logits must be on the GPU (libdsv41hip has no CPU path)")
    fit_int32(*logits.shape)
    if logits.dtype not in _KERNEL_DTYPES:
        logits = logits.float()
    # rows that overlap without being one and the same (stride 0) have no place for the kernels' row stride
    step, unit = logits.stride()
    vocab = logits.shape[1]
    if unit != 1 and vocab > 1 or 0 < step < vocab:
        logits = logits.contiguous()
    return logits


def refuse_capture(check: bool) -> None:
    if check and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a checked call waits for its answer and cannot be captured: pass check=False")


def row_fields(cls, logits) -> tuple:
    """The fields that every descriptor over rows of logits begins with."""
    rows, vocab = logits.shape
    return (ctypes.sizeof(cls), rows, vocab, _KERNEL_DTYPES[logits.dtype], logits.stride(0) if rows > 1 else vocab,
            logits.data_ptr())


def launch(call, device, *args) -> None:
    """``call(*args, stream)`` on the device's current stream, with its error raised."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = call(*args, _lib.stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _lib.stream(index))
    if rc:
        _lib.check(rc)


def written(t) -> None:
    """A kernel wrote ``t``, which was there before: autograd learns of it as of any operation in place."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _extent(t):
    """The addresses that a tensor of nonnegative strides reaches over."""
    n = t.numel()
    if n and not t.is_contiguous():
        n = 1 + sum((m - 1) * step for m, step in zip(t.shape, t.stride()))
    begin = t.data_ptr()
    return begin, begin + n * t.element_size()


def overlap(out, *others) -> bool:
    """Whether the memory that ``out`` reaches over meets that of others on its device; of matrices whose rows are as far
    apart, whether their rows do (columns side by side of one buffer do not)."""
    begin, end = _extent(out)
    for t in others:
        b, e = _extent(t)
        if begin < e and b < end and begin != end and b != e and _rows_meet(out, t, b - begin):
            return True
    return False


def _rows_meet(a, b, apart):
    """:func:`overlap` of two whose extents do; ``b`` begins ``apart`` bytes behind ``a``."""
    if not (a.ndim == b.ndim == 2 and a.stride(1) == b.stride(1) == 1):
        return True
    step = a.stride(0) * a.element_size()
    width_a, width_b = (t.shape[1] * t.element_size() for t in (a, b))
    if step != b.stride(0) * b.element_size() or step < max(width_a, width_b):
        return True
    # b's row j begins `past` bytes behind the begin of a's row j + ahead, and may reach into the next one
    ahead, past = divmod(apart, step)
    meet = lambda shift: max(0, shift) < min(a.shape[0], b.shape[0] + shift)
    return past < width_a and meet(ahead) or past + width_b > step and meet(ahead + 1)


def vector(t, dtype, shape, device):
    """A contiguous tensor of that dtype and shape on the device, ``t`` itself where it is one."""
    if t.dtype != dtype or t.device != device:
        t = t.to(device=device, dtype=dtype)
    if t.shape != shape:
        t = t.expand(shape)
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def prepare(logits, targets, top_k, temperature):
    """Validated arguments in kernel form."""
    logits = rows_of_logits(logits, temperature)
    rows, vocab = logits.shape
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= vocab:
        raise ValueError("top_k must be an integer in [0, vocabulary_size]")
    if targets is not None:
        if targets.dtype not in INTEGERS:
            raise ValueError("targets must be integers")
        if targets.numel() != rows:
            raise ValueError("one target is required per row")
        if targets.ndim != 1:
            targets = targets.reshape(rows)
        targets = vector(targets, torch.int64, targets.shape, logits.device)
    return logits, targets


def forward(logits, targets, top_k, temperature, want_stats, want_status=True):
    """One dsv41_scores_run; returns (log-probs, ranks, entropy, ids, log-probs, statuses, stats), None for
    what is not asked for.  Statuses that nobody looks at lie behind the workspace: an allocation less, 1.1 us of
    a decoding call's 21."""
    rows, dev = logits.shape[0], logits.device
    f32, i64 = torch.float32, torch.int64
    lp = rank = status = stats = ws = None
    if targets is not None:
        lp = torch.empty(rows, dtype=f32, device=dev)
        rank = torch.empty(rows, dtype=i64, device=dev)
    entropy = torch.empty(rows, dtype=f32, device=dev)
    top_ids = torch.empty(rows, top_k, dtype=i64, device=dev)
    top_lp = torch.empty(rows, top_k, dtype=f32, device=dev)
    if want_status:
        status = torch.empty(rows, dtype=torch.int32, device=dev)
    if want_stats:
        stats = torch.empty(rows, 4, dtype=torch.float64, device=dev)
    if rows:
        d = _lib.ScoresDesc(*row_fields(_lib.ScoresDesc, logits), _ptr(targets), temperature, top_k, _ptr(lp), _ptr(rank),
                            entropy.data_ptr(), top_ids.data_ptr() if top_k else None, top_lp.data_ptr() if top_k else None,
                            entropy.data_ptr() if status is None else status.data_ptr(), _ptr(stats))
        lib = _lib.load()
        ref = ctypes.byref(d)
        size = lib.dsv41_scores_workspace_bytes(ref)
        if status is None:  # (and not the entropies' place, which stood for it)
            ws = torch.empty(size + 4 * rows, dtype=torch.uint8, device=dev)
            d.out_status = ws.data_ptr() + size
        elif size:
            ws = torch.empty(size, dtype=torch.uint8, device=dev)
        launch(lib.dsv41_scores_run, dev, ref, _ptr(ws), size)
    return lp, rank, entropy, top_ids, top_lp, status, stats


def scores_backward(logits, targets, top_ids, temperature, stats, g_log_probs, g_entropy, g_top):
    """dL/dlogits of :func:`logit_scores`, in the logits' dtype; gradients that are None count as zero."""
    refuse_tangents("gradients", g_log_probs, g_entropy, g_top)
    rows, vocab = logits.shape
    dev = logits.device
    out = torch.empty(rows, vocab, dtype=logits.dtype, device=dev)
    if rows == 0:
        return out
    g_log_probs = None if g_log_probs is None or targets is None else vector(g_log_probs, torch.float32, (rows,), dev)
    g_entropy = None if g_entropy is None else vector(g_entropy, torch.float32, (rows,), dev)
    top_k = top_ids.shape[1]
    g_top = None if g_top is None or not top_k else vector(g_top, torch.float32, top_ids.shape, dev)
    d = _lib.ScoresGradDesc(*row_fields(_lib.ScoresGradDesc, logits), _ptr(targets), _ptr(top_ids) if top_k else None,
                            temperature, top_k, stats.data_ptr(), _ptr(g_log_probs), _ptr(g_entropy), _ptr(g_top),
                            out.data_ptr())
    launch(_lib.load().dsv41_scores_grad_run, dev, ctypes.byref(d))
    return out


class _LogitScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature):
        lp, rank, entropy, top_ids, top_lp, status, stats = forward(logits, targets, top_k, temperature, True)
        ctx.temperature = temperature
        ctx.save_for_backward(logits, targets, top_ids, stats)
        ctx.mark_non_differentiable(*(t for t in (rank, top_ids, status) if t is not None))
        ctx.set_materialize_grads(False)
        return lp, rank, entropy, top_ids, top_lp, status

    @staticmethod
    def backward(ctx, g_lp, g_rank, g_entropy, g_ids, g_top, g_status):
        logits, targets, top_ids, stats = ctx.saved_tensors
        if g_lp is None and g_entropy is None and g_top is None:
            return None, None, None, None
        grad = scores_backward(logits, targets, top_ids, ctx.temperature, stats, g_lp, g_entropy, g_top)
        sources = [t for t in (logits, g_lp, g_entropy, g_top) if t is not None]
        return first_order(grad, *sources), None, None, None


def _status_error(status: torch.Tensor) -> None:
    bits = 0
    for v in status.unique().tolist():
        bits |= int(v)
    if bits & _lib.STATUS_BAD_TARGET:
        raise ValueError("target token ID is outside the model vocabulary")
    if bits & _lib.STATUS_NONFINITE:
        raise ValueError("logits leave a row without a distribution (NaN, +inf or every token masked)")


def logit_scores(
    logits: torch.Tensor,
    targets: Optional[torch.Tensor] = None,
    *,
    top_k: int = 0,
    temperature: float = 1.0,
    check: bool = True,
) -> LogitScores:
    """Log-probs under ``softmax(logits / temperature)`` of one given token per row, its rank, the row's
    entropy and the ``top_k`` most likely tokens with their log-probs.

    ``logits [rows, V]`` are fp32 or bf16 on the GPU (other dtypes are converted to fp32), rows at any
    stride; ``-inf`` is a masked token, of probability 0.  ``targets [rows]`` int64.  Tokens order by
    (logit desc, index asc), with -0 equal to +0; a rank is 1 plus the number of tokens before the target.
    ``top_k`` is at most 1024 and V.

    Differentiable in ``logits``: log-probs, entropy and the alternatives' log-probs (with the
    alternatives held fixed), once (no second derivatives), and not in forward mode: logits that carry a
    tangent are refused.  A row whose upstream gradients are all zero
    gets zeros.

    With ``check`` the call synchronises and raises ``ValueError`` for a target outside the vocabulary,
    or a row with a NaN, a +inf or no unmasked token; without, such a row holds NaN (ids -1, rank 0).
    """
    logits, targets = prepare(logits, targets, top_k, temperature)
    refuse_capture(check)
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, rank, entropy, top_ids, top_lp, status = _LogitScores.apply(logits, targets, top_k, temperature)
    else:
        lp, rank, entropy, top_ids, top_lp, status, _ = forward(logits, targets, top_k, temperature, False, check)
    if check and any_set(status)[0]:
        _status_error(status)
    return LogitScores(lp, rank, entropy, top_ids, top_lp)

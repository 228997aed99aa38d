"""torch.library custom ops over libdsv41hip.so, in the reference's operator idiom
(``torch.library.custom_op(..., mutates_args=(), device_types="cuda")`` plus
``register_fake``, dsv41_train/models/dsv4/moe/kernels.py:236-281).

* ``dsv41_rocm::sample_rows`` — the row sampler; returns ``(ids, logprobs, kept, status)``.
* ``dsv41_rocm::selected_log_probs`` — the fused log-prob head; returns
  ``(logprob, entropy, ratio, lse)`` with an empty ``ratio`` when no behaviour log-probs are
  given.  Differentiable in ``hidden`` and ``weight`` through ``register_autograd`` (the
  reference registers its Triton ops' backward the same way, moe/kernels.py:283-307);
  ``ratio`` and ``lse`` carry no gradient.
* ``dsv41_rocm::logit_scores`` — scores of rows of logits; returns ``(log_probs, ranks, entropy,
  top_ids, top_log_probs, status, stats)``, the first two empty without targets.  Differentiable in
  ``logits`` through the log-probs, the entropy and the alternatives' log-probs; ``stats`` is what
  the backward needs of the forward.
* ``dsv41_rocm::distillation_loss`` — divergence from a teacher's top tokens; returns ``(loss,
  status, stats)``.  Differentiable in ``logits``.
* ``dsv41_rocm::process_logits`` — biases, penalties (numbers, or a tensor of one value per row in their place) and
  token masks; returns ``(logits, status)``.  Differentiable in ``logits``.
* ``dsv41_rocm::head_logits`` — logits of an 8-bit head's ``tiles`` and ``scales``; returns ``(logits, status)``.
* ``dsv41_rocm::token_embedding`` — rows of a token table; returns ``(rows, status)``.  Differentiable in
  ``weight``.

The ops only register a CUDA (HIP) kernel: called on CPU tensors they raise, as the library
has no CPU path.  Status bits are returned, not raised, so the ops stay traceable; the
Python wrappers in ``sampling`` and ``logprob`` raise the reference's errors.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import distill as _distill
from . import embedding as _embedding
from . import inthead as _inthead
from . import logprob as _logprob
from . import process as _process
from . import sampling as _sampling
from . import scores as _scores


@torch.library.custom_op("dsv41_rocm::sample_rows", mutates_args=(), device_types="cuda")
def sample_rows(
    logits: torch.Tensor,
    uniforms: Optional[torch.Tensor],
    history: Optional[torch.Tensor],
    history_lens: Optional[torch.Tensor],
    temperature: float,
    repetition_penalty: float,
    presence_penalty: float,
    frequency_penalty: float,
    top_k: int,
    top_p: float,
    min_p: float,
    greedy: bool,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    if not greedy and uniforms is None:
        raise ValueError("sampling requires one uniform per row")
    r = _sampling.sample(logits, temperature=temperature, uniforms=uniforms, history=history,
                         history_lens=history_lens, repetition_penalty=repetition_penalty,
                         presence_penalty=presence_penalty, frequency_penalty=frequency_penalty,
                         top_k=top_k, top_p=top_p, min_p=min_p, greedy=greedy, check=False)
    return r.ids, r.logprobs, r.kept, r.status


@sample_rows.register_fake
def _sample_rows_fake(logits, uniforms, history, history_lens, temperature, repetition_penalty,
                      presence_penalty, frequency_penalty, top_k, top_p, min_p, greedy):
    rows = logits.shape[0]
    dev = logits.device
    return (torch.empty(rows, dtype=torch.int64, device=dev),
            torch.empty(rows, dtype=torch.float32, device=dev),
            torch.empty(rows, dtype=torch.int32, device=dev),
            torch.empty(rows, dtype=torch.int32, device=dev))


@torch.library.custom_op("dsv41_rocm::selected_log_probs", mutates_args=(), device_types="cuda")
def selected_log_probs_op(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    temperature: float,
    behavior: Optional[torch.Tensor],
    is_cap: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    hidden, weight, targets = _logprob._prepare(hidden, weight, targets, temperature)
    lp, ent, ratio, lse, _ = _logprob._forward(hidden, weight, targets, temperature, behavior, is_cap)
    if ratio is None:
        ratio = lp.new_empty(0)
    return lp, ent, ratio, lse


@selected_log_probs_op.register_fake
def _selected_log_probs_fake(hidden, weight, targets, temperature, behavior, is_cap):
    n = hidden.shape[0]
    dev = hidden.device
    lp = torch.empty(n, dtype=torch.float32, device=dev)
    ent = torch.empty(n, dtype=torch.float32, device=dev)
    ratio = torch.empty(n if behavior is not None else 0, dtype=torch.float32, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    return lp, ent, ratio, lse


def _selected_log_probs_setup(ctx, inputs, output):
    hidden, weight, targets, temperature, _, _ = inputs
    _, ent, _, lse = output
    ctx.temperature = temperature
    ctx.hidden_dtype, ctx.weight_dtype = hidden.dtype, weight.dtype
    ctx.save_for_backward(hidden, weight, targets, lse, ent)


def _selected_log_probs_backward(ctx, g_lp, g_ent, g_ratio, g_lse):
    hidden, weight, targets, lse, ent = ctx.saved_tensors
    h, w, t = _logprob._prepare(hidden, weight, targets, ctx.temperature)
    dx, dw = _logprob.selected_log_probs_backward(h, w, t, ctx.temperature, lse, ent, g_lp, g_ent,
                                                  need_hidden=ctx.needs_input_grad[0],
                                                  need_weight=ctx.needs_input_grad[1])
    if dx is not None:
        dx = dx.to(ctx.hidden_dtype)
    if dw is not None:
        dw = dw.to(ctx.weight_dtype)
    sources = (hidden, weight, g_lp, g_ent)
    return _logprob.first_order(dx, *sources), _logprob.first_order(dw, *sources), None, None, None, None


selected_log_probs_op.register_autograd(_selected_log_probs_backward, setup_context=_selected_log_probs_setup)


@torch.library.custom_op("dsv41_rocm::logit_scores", mutates_args=(), device_types="cuda")
def logit_scores_op(
    logits: torch.Tensor, targets: Optional[torch.Tensor], top_k: int, temperature: float
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    logits, targets = _scores.prepare(logits, targets, top_k, temperature)
    lp, rank, entropy, top_ids, top_lp, status, stats = _scores.forward(logits, targets, top_k, temperature, True)
    if targets is None:
        lp, rank = entropy.new_empty(0), top_ids.new_empty(0)
    return lp, rank, entropy, top_ids, top_lp, status, stats


@logit_scores_op.register_fake
def _logit_scores_fake(logits, targets, top_k, temperature):
    rows, dev = logits.shape[0], logits.device
    n = 0 if targets is None else rows
    return (torch.empty(n, dtype=torch.float32, device=dev), torch.empty(n, dtype=torch.int64, device=dev),
            torch.empty(rows, dtype=torch.float32, device=dev), torch.empty(rows, top_k, dtype=torch.int64, device=dev),
            torch.empty(rows, top_k, dtype=torch.float32, device=dev), torch.empty(rows, dtype=torch.int32, device=dev),
            torch.empty(rows, 4, dtype=torch.float64, device=dev))


def _logit_scores_setup(ctx, inputs, output):
    logits, targets, top_k, temperature = inputs
    _, _, _, top_ids, _, _, stats = output
    ctx.top_k, ctx.temperature = top_k, temperature
    ctx.save_for_backward(logits, targets, top_ids, stats)


def _logit_scores_backward(ctx, g_lp, g_rank, g_entropy, g_ids, g_top, g_status, g_stats):
    logits, targets, top_ids, stats = ctx.saved_tensors
    rows, t = _scores.prepare(logits, targets, ctx.top_k, ctx.temperature)
    grad = _scores.scores_backward(rows, t, top_ids, ctx.temperature, stats, g_lp, g_entropy, g_top).to(logits.dtype)
    sources = [g for g in (logits, g_lp, g_entropy, g_top) if g is not None]
    return _logprob.first_order(grad, *sources), None, None, None


logit_scores_op.register_autograd(_logit_scores_backward, setup_context=_logit_scores_setup)


@torch.library.custom_op("dsv41_rocm::distillation_loss", mutates_args=(), device_types="cuda")
def distillation_loss_op(
    logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_log_probs: torch.Tensor, temperature: float, tail: str
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    logits, ids, lq = _distill.prepare(logits, teacher_ids, teacher_log_probs, temperature, tail)
    return _distill.forward(logits, ids, lq, temperature, tail, True)


@distillation_loss_op.register_fake
def _distillation_loss_fake(logits, teacher_ids, teacher_log_probs, temperature, tail):
    rows, dev = logits.shape[0], logits.device
    return (torch.empty(rows, dtype=torch.float32, device=dev), torch.empty(rows, dtype=torch.int32, device=dev),
            torch.empty(rows, _distill.STATS, dtype=torch.float64, device=dev))


def _distillation_loss_setup(ctx, inputs, output):
    logits, teacher_ids, teacher_log_probs, temperature, tail = inputs
    ctx.temperature, ctx.tail = temperature, tail
    ctx.save_for_backward(logits, teacher_ids, teacher_log_probs, output[2])


def _distillation_loss_backward(ctx, g_loss, g_status, g_stats):
    logits, teacher_ids, teacher_log_probs, stats = ctx.saved_tensors
    rows, ids, lq = _distill.prepare(logits, teacher_ids, teacher_log_probs, ctx.temperature, ctx.tail)
    grad = _distill.distillation_backward(rows, ids, lq, ctx.temperature, stats, g_loss).to(logits.dtype)
    return _logprob.first_order(grad, logits, g_loss), None, None, None, None


distillation_loss_op.register_autograd(_distillation_loss_backward, setup_context=_distillation_loss_setup)


@torch.library.custom_op("dsv41_rocm::process_logits", mutates_args=(), device_types="cuda")
def process_logits_op(
    logits: torch.Tensor,
    history: Optional[torch.Tensor],
    history_lens: Optional[torch.Tensor],
    history_prompt_lens: Optional[torch.Tensor],
    repetition_penalty: float,
    presence_penalty: float,
    frequency_penalty: float,
    repetition_penalties: Optional[torch.Tensor],
    presence_penalties: Optional[torch.Tensor],
    frequency_penalties: Optional[torch.Tensor],
    bias_ids: Optional[torch.Tensor],
    bias: Optional[torch.Tensor],
    token_mask: Optional[torch.Tensor],
    mask_rows: Optional[torch.Tensor],
    fill: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    rows, numbers, tensors = _process_arguments(
        logits, history, history_lens, history_prompt_lens, repetition_penalty, presence_penalty, frequency_penalty,
        repetition_penalties, presence_penalties, frequency_penalties, bias_ids, bias, token_mask, mask_rows, fill)
    out = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
    status = _process.forward(rows, numbers, tensors, out, True)
    return out, status


def _process_arguments(logits, history, history_lens, history_prompt_lens, repetition_penalty, presence_penalty,
                       frequency_penalty, repetition_penalties, presence_penalties, frequency_penalties, bias_ids, bias,
                       token_mask, mask_rows, fill):
    either = lambda number, each: number if each is None else each
    rows = _scores.rows_of_logits(logits, 1.0)
    numbers, tensors = _process._arguments(
        rows, history, history_lens, history_prompt_lens, either(repetition_penalty, repetition_penalties),
        either(presence_penalty, presence_penalties), either(frequency_penalty, frequency_penalties), bias_ids, bias,
        token_mask, mask_rows, fill)
    return rows, numbers, tensors


@process_logits_op.register_fake
def _process_logits_fake(logits, *arguments):
    dtype = logits.dtype if logits.dtype in (torch.float32, torch.bfloat16) else torch.float32
    return (torch.empty(logits.shape, dtype=dtype, device=logits.device),
            torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device))


_PROCESS_CONSTANTS = {7: "repetition_penalties", 8: "presence_penalties", 9: "frequency_penalties", 11: "bias"}


def _process_logits_setup(ctx, inputs, output):
    # (inside the op no gradient is recorded, so it cannot tell)
    for i, name in _PROCESS_CONSTANTS.items():
        if ctx.needs_input_grad[i]:
            raise NotImplementedError(f"{name} has no gradient: detach it")
    tensors = [t if isinstance(t, torch.Tensor) else None for t in inputs]
    ctx.save_for_backward(*tensors)
    ctx.numbers = [None if isinstance(t, torch.Tensor) else t for t in inputs]


def _process_logits_backward(ctx, g_out, g_status):
    inputs = [n if t is None else t for n, t in zip(ctx.numbers, ctx.saved_tensors)]
    rows, numbers, tensors = _process_arguments(*inputs)
    grad = _process.process_backward(rows, numbers, tensors, g_out).to(inputs[0].dtype)
    return (_logprob.first_order(grad, inputs[0], g_out),) + (None,) * (len(inputs) - 1)


process_logits_op.register_autograd(_process_logits_backward, setup_context=_process_logits_setup)


@torch.library.custom_op("dsv41_rocm::head_logits", mutates_args=(), device_types="cuda")
def head_logits_op(
    hidden: torch.Tensor, tiles: torch.Tensor, scales: torch.Tensor, vocab: int, dtype: torch.dtype
) -> tuple[torch.Tensor, torch.Tensor]:
    x = _inthead._rows(hidden, "hidden")
    head = _inthead.Int8Head(tiles, scales, vocab, hidden.shape[1])
    _inthead._check_head(head, x)
    if dtype not in _inthead._OUT_DTYPES:
        raise ValueError("logits are torch.float32 or torch.bfloat16")
    out = _inthead._new_logits(x.shape[0], vocab, dtype, x.device)
    return out, _inthead._forward(x, head, out, True)


@head_logits_op.register_fake
def _head_logits_fake(hidden, tiles, scales, vocab, dtype):
    n, dev = hidden.shape[0], hidden.device
    return _inthead._new_logits(n, vocab, dtype, dev), torch.empty(n, dtype=torch.int32, device=dev)


@torch.library.custom_op("dsv41_rocm::token_embedding", mutates_args=(), device_types="cuda")
def token_embedding_op(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    flat, weight, scale = _embedding.prepare(ids, weight, scale)
    status = torch.empty(flat.numel(), dtype=torch.int32, device=weight.device)
    out = _embedding.forward(flat, weight, scale, status)
    return out.view(*ids.shape, weight.shape[1]), status


@token_embedding_op.register_fake
def _token_embedding_fake(ids, weight, scale):
    return (torch.empty(*ids.shape, weight.shape[1], dtype=weight.dtype, device=weight.device),
            torch.empty(ids.numel(), dtype=torch.int32, device=weight.device))


def _token_embedding_setup(ctx, inputs, output):
    ids, weight, scale = inputs
    ctx.vocab, ctx.dtype, ctx.scale = weight.shape[0], weight.dtype, scale
    ctx.save_for_backward(ids)


def _token_embedding_backward(ctx, g_rows, g_status):
    (ids,) = ctx.saved_tensors
    with torch.no_grad():
        dw = _embedding.token_embedding_backward(g_rows, ids, ctx.vocab, scale=ctx.scale, dtype=ctx.dtype)
    return None, _logprob.first_order(dw, g_rows), None


token_embedding_op.register_autograd(_token_embedding_backward, setup_context=_token_embedding_setup)


__all__ = ["sample_rows", "selected_log_probs_op", "logit_scores_op", "distillation_loss_op", "process_logits_op",
           "head_logits_op", "token_embedding_op"]

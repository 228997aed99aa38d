"""Rows of a token table on MI355X, scaled, and the table's gradient by sorted tokens.

The reference's models begin with ``nn.Embedding`` and end with the head of the same vocabulary
(``dsv41_train/models/dsv4/model.py:635``).  Where both are one table, the embedding's gradient goes
onto the head's (``selected_log_probs_backward``): ``token_embedding_backward(..., out=)``.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._check import answer
from .logprob import first_order
from .scores import INTEGERS, fit_int32, launch, overlap, refuse_capture, refuse_tangents, written

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _ids(ids, device):
    if not isinstance(ids, torch.Tensor) or ids.dtype not in INTEGERS:
        raise ValueError("ids must be integers")
    if ids.dtype != torch.int64 or ids.device != device:
        ids = ids.to(device=device, dtype=torch.int64)
    if ids.ndim != 1:
        ids = ids.reshape(-1)
    fit_int32(ids.numel())
    return ids if ids.is_contiguous() else ids.contiguous()


def _scale(scale) -> float:
    scale = float(scale)
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError("scale must be finite")
    return scale


def _matrix(t, broadcast=False):
    """``t``, or a copy, whose rows are contiguous and do not overlap (``broadcast``: or are all the same)."""
    rows, width = t.shape
    step = t.stride(0)
    if width > 1 and t.stride(1) != 1 or rows > 1 and step < width and not (broadcast and step == 0):
        t = t.contiguous()
    return t


def _step(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def prepare(ids, weight, scale):
    """Validated arguments in kernel form."""
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2 or 0 in weight.shape:
        raise ValueError("weight must have shape [vocabulary_size, hidden]")
    if not weight.is_cuda:
        raise ValueError("weight must be on the GPU (libdsv41hip has no CPU path)")
    if weight.dtype not in _DTYPES:
        raise ValueError("weight must be fp32 or bf16")
    refuse_tangents("weight", weight)
    fit_int32(*weight.shape)
    return _ids(ids, weight.device), _matrix(weight), _scale(scale)


def forward(ids, weight, scale, status=None, check=False):
    """One dsv41_embed_run, with every id's status if asked for; with ``check`` one that raises."""
    n, (v, h) = ids.numel(), weight.shape
    out = weight.new_empty(n, h)
    if n:
        d = _lib.EmbedDesc(ctypes.sizeof(_lib.EmbedDesc), n, h, v, weight.data_ptr(), _step(weight), ids.data_ptr(), scale,
                           _DTYPES[weight.dtype], out.data_ptr(), h, None if status is None else status.data_ptr())
        if not check:
            launch(_lib.load().dsv41_embed_run, weight.device, ctypes.byref(d))
        elif answer(_lib.load().dsv41_embed_checked_run, weight.device.index, ctypes.byref(d)):
            raise ValueError("token ID is outside the model vocabulary")
    return out


def _backward(ids, grad, scale, out, accumulate):
    n, h = grad.shape
    d = _lib.EmbedGradDesc(ctypes.sizeof(_lib.EmbedGradDesc), n, h, out.shape[0], ids.data_ptr() if n else None,
                           grad.data_ptr() if n else None, _step(grad), _DTYPES[grad.dtype], scale, out.data_ptr(),
                           _step(out), _DTYPES[out.dtype], int(accumulate))
    lib = _lib.load()
    ref = ctypes.byref(d)
    size = lib.dsv41_embed_grad_workspace_bytes(ref)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=out.device)
    launch(lib.dsv41_embed_grad_run, out.device, ref, ws.data_ptr(), size)


def token_embedding_backward(
    grad: torch.Tensor,
    ids: torch.Tensor,
    vocabulary_size: Optional[int] = None,
    *,
    scale: float = 1.0,
    out: Optional[torch.Tensor] = None,
    dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """dL/dweight of :func:`token_embedding` from ``grad``, dL/d(its result), ``[*ids.shape, hidden]`` in fp32 or bf16.

    Row ``v`` is ``scale`` times the sum of the gradients of the tokens whose id is ``v``, in fp32 and in
    the order of the batch; zeros where there is none.  Ids outside the vocabulary take no part.
    The result is a new ``[vocabulary_size, hidden]`` in ``dtype`` (default: that of ``grad``).  With
    ``out`` (fp32 or bf16 ``[vocabulary_size, hidden]``) it is added to what ``out`` holds, in fp32, rounded once;
    rows of tokens that do not occur are not touched.  That is how a tied table's two gradients meet.

    Bit for bit the same for the same inputs.
    """
    if not isinstance(ids, torch.Tensor):
        raise ValueError("ids must be integers")
    if not isinstance(grad, torch.Tensor) or grad.ndim < 1 or grad.shape[-1] == 0 or grad.shape[:-1] != ids.shape:
        raise ValueError("grad must have the shape of ids and the hidden size")
    if out is not None and not isinstance(out, torch.Tensor):
        raise ValueError("out must be fp32 or bf16 [vocabulary_size, hidden] on the GPU of grad")
    if not grad.is_cuda:
        raise ValueError("grad must be on the GPU (libdsv41hip has no CPU path)")
    refuse_tangents("gradients", grad)
    if torch.is_grad_enabled() and (grad.requires_grad or out is not None and out.requires_grad):
        raise NotImplementedError("the embedding's gradient cannot be differentiated again: detach grad and out")
    h = grad.shape[-1]
    scale = _scale(scale)
    ids = _ids(ids, grad.device)
    grad = grad.reshape(-1, h)
    if grad.dtype not in _DTYPES:
        grad = grad.float()
    grad = _matrix(grad, broadcast=True)
    if out is not None:
        if out.ndim != 2 or out.shape[1] != h or out.shape[0] == 0 or out.dtype not in _DTYPES or out.device != grad.device:
            raise ValueError("out must be fp32 or bf16 [vocabulary_size, hidden] on the GPU of grad")
        if vocabulary_size is not None and vocabulary_size != out.shape[0] or dtype is not None and dtype != out.dtype:
            raise ValueError("out has another vocabulary_size or dtype")
        if h > 1 and out.stride(1) != 1 or out.shape[0] > 1 and out.stride(0) < h:
            raise ValueError("out must have contiguous rows that do not overlap")
        if overlap(out, grad):
            raise ValueError("out overlaps grad")
        fit_int32(*out.shape)
        if ids.numel():
            _backward(ids, grad, scale, out, True)
            written(out)
        return out
    if isinstance(vocabulary_size, bool) or not isinstance(vocabulary_size, int) or vocabulary_size <= 0:
        raise ValueError("vocabulary_size must be a positive integer")
    dtype = grad.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError("the gradient is torch.float32 or torch.bfloat16")
    fit_int32(vocabulary_size, h)
    out = torch.empty(vocabulary_size, h, dtype=dtype, device=grad.device)
    _backward(ids, grad, scale, out, False)
    return out


class _TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, check):
        out = forward(ids, weight, scale, check=check)
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.dtype, ctx.scale = weight.shape[0], weight.dtype, scale
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, grad):
        if grad is None:
            return None, None, None, None
        (ids,) = ctx.saved_tensors
        refuse_tangents("gradients", grad)
        dw = torch.empty(ctx.vocab, grad.shape[1], dtype=ctx.dtype, device=grad.device)
        _backward(ids, _matrix(grad, broadcast=True), ctx.scale, dw, False)
        return None, first_order(dw, grad), None, None


def token_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, check: bool = True) -> torch.Tensor:
    """``scale * weight[ids]``, ``[*ids.shape, hidden]`` in the dtype of ``weight [vocabulary_size, hidden]`` (fp32 or bf16
    on the GPU, rows at any stride); the product is formed in fp32 and rounded once.

    Negative ids are padding: rows of zeros, which take no part in the gradient.  Differentiable in
    ``weight`` (a dense gradient, see :func:`token_embedding_backward`), once, in backward mode.

    With ``check`` the call waits until the GPU has looked at the ids and raises ``ValueError`` for one at or above the
    vocabulary size; without, such a token's row is NaN.
    """
    flat, weight, scale = prepare(ids, weight, scale)
    refuse_capture(check)
    if torch.is_grad_enabled() and weight.requires_grad:
        out = _TokenEmbedding.apply(flat, weight, scale, check)
    else:
        out = forward(flat, weight, scale, check=check)
    return out if ids.ndim == 1 else out.view(*ids.shape, weight.shape[1])

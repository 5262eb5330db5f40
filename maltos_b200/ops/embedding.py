"""Token embedding with a scale, and its gradient by sorted tokens (``csrc/embedding.cu``).

``embedding(ids, weight, scale=s)`` is ``s * weight[ids]``, scaled in fp32 and rounded once; the gradient of a table row is the
sum of its tokens' output gradients in token order, in fp32, rounded once, with the same bits every time. The reference looks
tokens up with ``nn.Embedding`` (``models/llama.py``), whose gradient adds rows in the table's own type.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def embedding_reference(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    rows = nn.functional.embedding(ids, weight, padding_idx=padding_idx)
    if scale == 1.0:
        return rows
    return rows * scale if rows.dtype == torch.float64 else (rows.float() * scale).to(rows.dtype)


def _contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _lookup(ids: torch.Tensor, w: torch.Tensor, scale: float) -> torch.Tensor:
    rows, H = w.shape
    out = w.new_empty((*ids.shape, H))
    with _lib.on_device_of(w):
        _lib.check(_lib.lib().mb_embedding_fwd(ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0, w.data_ptr(), out.data_ptr(),
                                               _DTYPES[w.dtype], ids.numel(), H, rows, scale, _lib.stream_of(w)), "mb_embedding_fwd")
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return _lookup(ids, _contiguous(weight), scale)

    @staticmethod
    def backward(ctx, dout):
        _lib.refuse_second_order("embedding")
        (ids,) = ctx.saved_tensors
        H, n, dout = dout.shape[-1], ids.numel(), _contiguous(dout)
        L = _lib.lib()
        dweight = dout.new_empty((ctx.rows, H))
        with _lib.on_device_of(dout):
            scratch = ids.new_empty(L.mb_embedding_bwd_scratch_words(n, H) // (1 if ids.dtype == torch.int32 else 2) + 1)   # 4-byte words
            _lib.check(L.mb_embedding_bwd(ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0, dout.data_ptr(), dweight.data_ptr(),
                                          scratch.data_ptr(), _DTYPES[dout.dtype], n, H, ctx.rows,
                                          -1 if ctx.padding_idx is None else ctx.padding_idx, ctx.scale, _lib.stream_of(dout)),
                       "mb_embedding_bwd")
        return None, dweight, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` in the table's type: ids int32 or int64 of any shape, weight ``[rows, H]``. Tokens that are
    ``padding_idx`` are looked up like others and give their row no gradient. Differentiable (once) in ``weight``.

    On CUDA an id outside the table reads as a zero row, gets no gradient and sets the device status word (index out of
    bounds), as elsewhere in this library; on the CPU it raises an ``IndexError``."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"the embedding table is a floating-point matrix, got {tuple(weight.shape)} {weight.dtype}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"token ids are int32 or int64, got {ids.dtype}")
    if ids.device != weight.device:
        raise ValueError(f"token ids are on {ids.device}, the table on {weight.device}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale!r}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx={padding_idx} is outside the table of {weight.shape[0]} rows")
    if _lib.use_kernels(weight) and weight.dtype in _DTYPES and ids.numel() and weight.numel():
        ids = _contiguous(ids)
        if torch.is_grad_enabled() and weight.requires_grad:
            return _Embedding.apply(ids, weight, float(scale), padding_idx)
        return _lookup(ids, _contiguous(weight), float(scale))
    return embedding_reference(ids, weight, scale, padding_idx)


class ScaledEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter, same checkpoint name) whose rows come out multiplied by ``scale``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float, padding_idx: int | None = None) -> None:
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx)
        self.scale = float(scale)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding(ids, self.weight, scale=self.scale, padding_idx=self.padding_idx)

"""Sliding-window attention with first tokens that stay visible: the kernels behind
:func:`maltos_b200.ops.attention.sliding_window_attention` (``csrc/window_attn.cu`` forward, ``csrc/window_attn_bwd.cu``
backward; the rule they share is ``csrc/window.cuh``)."""
from __future__ import annotations

import math

import torch

from maltos_b200.utils.activation_checkpoint import current_checkpoint_stash

from . import _lib


def _few_queries(B: int, Hkv: int, rows: int) -> bool:
    """Whether a forward without gradients takes ``csrc/window_token.cu``: ``rows`` (queries x heads of a group) of each key/value
    head in groups of 8, K and V read once a group. Up to one group it always wins (8 rows of 2048 visible keys, 8 key/value
    heads: 20 us against 48 us in tiles of 128 rows); up to four while the groups fit the SMs (4 groups x 16 heads: 20 against
    92 us, 2 x 64: 40 against 48 us; 4 x 64 lose, 76 against 48 us)."""
    groups = -(-rows // 8)
    return groups == 1 or (groups <= 4 and B * Hkv * groups <= 148)


def _addressable(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """``[B, S, h, D]`` as the kernels address it (heads contiguous inside a token, 16-byte aligned, token and batch strides
    positive multiples of 8 elements), with the token and the batch stride; copied only where its strides do not fit."""
    B, S, H, D = t.shape
    sb, st, sh, sd = t.stride()
    if not (sd == 1 and (sh == D or H == 1) and (S == 1 or (st > 0 and st % 8 == 0)) and (B == 1 or (sb > 0 and sb % 8 == 0))
            and t.data_ptr() % 16 == 0):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        sb, st = S * H * D, H * D
    if S == 1:
        st = H * D
    return t, st, S * st if B == 1 else sb


def document_bounds(sequence_ids: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """First index and one past the last index of every token's document, int32 ``[B, S]`` each (padding: 2^31 - 1 and 0)."""
    ids = sequence_ids.contiguous()
    B, S = ids.shape
    starts, ends = torch.empty((2, B, S), dtype=torch.int32, device=ids.device)
    with _lib.on_device_of(ids):
        _lib.check(_lib.lib().mb_document_bounds(ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0, starts.data_ptr(), ends.data_ptr(),
                                                 B, S, _lib.stream_of(ids)), "mb_document_bounds")
    return starts, ends


def window_forward(q, k, v, *, window: int, sinks: int, starts, scale: float, keep: bool, want_lse: bool):
    """``(out, out_lo, lse2, lse)``: the output ``[B, Sq, hq, D]`` in bf16; for the backward (``keep``) what its rounding left and the
    log2 of the sum of the rounded weights ``[B, hq, Sq]``; the log-sum-exp of the scores where asked for."""
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    q, q_t, q_b = _addressable(q)
    k, k_t, k_b = _addressable(k)
    v, v_t, v_b = _addressable(v)
    out = q.new_empty((B, Sq, Hq, D))
    if not keep and _few_queries(B, Hkv, Sq * (Hq // Hkv)):
        lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device) if want_lse else None
        with _lib.on_device_of(q):
            _lib.check(_lib.lib().mb_window_attn_token(q.data_ptr(), q_t, q_b, k.data_ptr(), k_t, k_b, v.data_ptr(), v_t, v_b, out.data_ptr(),
                                                       _lib.address(lse), _lib.address(starts), B, Sq, Sk, Hq, Hkv, D, window, sinks, scale,
                                                       _lib.stream_of(q)), "mb_window_attn_token")
        return out, None, None, lse
    out_lo = torch.empty_like(out) if keep else None
    lse2 = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device) if keep else None
    lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device) if want_lse else None
    with _lib.on_device_of(q):
        _lib.check(_lib.lib().mb_window_attn_fwd(q.data_ptr(), q_t, q_b, k.data_ptr(), k_t, k_b, v.data_ptr(), v_t, v_b, out.data_ptr(),
                                                 _lib.address(out_lo), _lib.address(lse2), _lib.address(lse), _lib.address(starts), B, Sq, Sk,
                                                 Hq, Hkv, D, window, sinks, scale, _lib.stream_of(q)), "mb_window_attn_fwd")
    return out, out_lo, lse2, lse


def window_backward(q, k, v, out, out_lo, lse2, dout, *, window: int, sinks: int, starts, ends, scale: float):
    """``(dq, dk, dv)`` in bf16; ``out``, ``out_lo`` and ``lse2`` are the forward's."""
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    q, q_t, q_b = _addressable(q)
    k, k_t, k_b = _addressable(k)
    v, v_t, v_b = _addressable(v)
    dout, do_t, do_b = _addressable(dout)
    dq, dk, dv = q.new_empty((B, Sq, Hq, D)), q.new_empty((B, Sk, Hkv, D)), q.new_empty((B, Sk, Hkv, D))
    L = _lib.lib()
    with _lib.on_device_of(q):
        words = L.mb_window_attn_bwd_scratch_words(B, Sq, Sk, Hq, Hkv, D, window, sinks, 0 if starts is None else 1)
        scratch = lse2.new_empty(words)
        _lib.check(L.mb_window_attn_bwd(q.data_ptr(), q_t, q_b, k.data_ptr(), k_t, k_b, v.data_ptr(), v_t, v_b, out.data_ptr(),
                                        out_lo.data_ptr(), dout.data_ptr(), do_t, do_b, lse2.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                        _lib.address(starts), _lib.address(ends), scratch.data_ptr(), B, Sq, Sk, Hq, Hkv, D, window, sinks,
                                        scale, _lib.stream_of(q)), "mb_window_attn_bwd")
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, starts, ends, scale, want_lse):
        # As in dense flash attention: under activation checkpointing the recompute replays the results of the first pass.
        stash = current_checkpoint_stash()
        kept = stash.replay() if stash is not None and stash.replaying else None
        if kept is not None and len(kept) == 4 and kept[0].shape == q.shape:
            out, out_lo, lse2, lse = kept
        else:
            out, out_lo, lse2, lse = window_forward(q, k, v, window=window, sinks=sinks, starts=starts, scale=scale, keep=True, want_lse=want_lse)
            if stash is not None and not stash.replaying:
                stash.record((out, out_lo, lse2, lse))
        ctx.save_for_backward(q, k, v, out, out_lo, lse2, starts, ends)
        ctx.window, ctx.sinks, ctx.scale = window, sinks, scale
        if lse is not None:
            ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _dlse):
        _lib.refuse_second_order("sliding_window_attention")
        q, k, v, out, out_lo, lse2, starts, ends = ctx.saved_tensors
        dq, dk, dv = window_backward(q, k, v, out, out_lo, lse2, dout, window=ctx.window, sinks=ctx.sinks, starts=starts, ends=ends, scale=ctx.scale)
        return dq, dk, dv, None, None, None, None, None, None


def window_attention(q, k, v, *, window: int, sinks: int = 0, sequence_ids=None, scale: float | None = None, return_lse: bool = False):
    """The kernels' differentiable entry: bf16, head_dim 64 or 128, sizes above zero, arguments as checked by the public one."""
    Sk = k.shape[1]
    starts, ends = document_bounds(sequence_ids) if sequence_ids is not None else (None, None)
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(q.shape[3])
    window, sinks = min(window, Sk), min(sinks, Sk)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _WindowAttention.apply(q, k, v, window, sinks, starts, ends, scale, return_lse)
    else:
        out, _, _, lse = window_forward(q, k, v, window=window, sinks=sinks, starts=starts, scale=scale, keep=False, want_lse=return_lse)
    return (out, lse) if return_lse else out

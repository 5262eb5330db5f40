"""RMSNorm with an optional fused residual add (``csrc/norm_rope_act.cu``).

``rms_norm(x, w, eps)`` = ``w * x * rsqrt(mean(x^2) + eps)`` with the statistics in fp32, replacing the un-fused
eager ops of the reference (``models/llama.py:55-57``). ``add_rms_norm(x, residual, w, eps)`` returns
``(norm(x + residual), x + residual)`` from a single pass over memory; its backward also folds the gradient of
the residual stream into ``dx``. ``block_norm`` is the whole seam between two blocks (``csrc/block_norm.cu``): norm after the
block, gate, residual scale, residual add and the norm before the next block.
"""
from __future__ import annotations

import math

import torch

from . import _lib


def rms_norm_reference(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)


def _kernel_ok(x: torch.Tensor, weight: torch.Tensor) -> bool:
    return _lib.use_kernels(x) and x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and x.shape[-1] % 8 == 0


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        H = x.shape[-1]
        x2 = x.reshape(-1, H).contiguous()
        rows = x2.shape[0]
        r2 = residual.reshape(-1, H).contiguous() if residual is not None else None
        y = torch.empty_like(x2)
        h = torch.empty_like(x2) if r2 is not None else None
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
        w = weight.contiguous()
        _lib.check(_lib.lib().mb_rmsnorm_fwd(_lib.ptr(x2), _lib.ptr(r2), _lib.ptr(w), _lib.ptr(y), _lib.ptr(h), _lib.ptr(rstd),
                                             _lib.c_ll(rows), _lib.c_int(H), _lib.c_float(eps), _lib.stream_ptr()), "mb_rmsnorm_fwd")
        ctx.save_for_backward(h if h is not None else x2, w, rstd)
        ctx.shape = x.shape
        ctx.fused = r2 is not None
        if ctx.fused:
            return y.view(x.shape), h.view(x.shape)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, w, rstd = ctx.saved_tensors
        H = h.shape[-1]
        rows = h.shape[0]
        dy2 = dy.reshape(-1, H).contiguous()
        dres = dh.reshape(-1, H).contiguous() if (ctx.fused and dh is not None) else None
        L = _lib.lib()
        nblk = L.mb_rmsnorm_bwd_blocks(_lib.c_ll(rows))
        partial = torch.empty((nblk, H), device=h.device, dtype=torch.float32)
        dx = torch.empty_like(h)
        dw = torch.empty_like(w)
        _lib.check(L.mb_rmsnorm_bwd(_lib.ptr(dy2), _lib.ptr(h), _lib.ptr(w), _lib.ptr(rstd), _lib.ptr(dres), _lib.ptr(dx),
                                    _lib.ptr(partial), _lib.ptr(dw), _lib.c_void_p(0), _lib.c_int(0), _lib.c_ll(rows),
                                    _lib.c_int(H), _lib.stream_ptr()), "mb_rmsnorm_bwd")
        dx = dx.view(ctx.shape)
        if ctx.fused:
            return dx, dx, dw, None
        return dx, None, dw, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    if _kernel_ok(x, weight):
        return _RmsNorm.apply(x, None, weight, eps)
    return rms_norm_reference(x, weight, eps)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6):
    """Returns ``(rms_norm(x + residual), x + residual)``."""
    if _kernel_ok(x, weight) and residual.dtype == torch.bfloat16:
        return _RmsNorm.apply(x, residual, weight, eps)
    h = x + residual
    return rms_norm_reference(h, weight, eps), h


_BLOCK_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_BLOCK_MAX_HIDDEN = 16384


def block_norm_reference(x, residual, weight, next_weight=None, *, gate=None, scale: float = 1.0, eps: float = 1e-6):
    """Eager :func:`block_norm` in fp32 (fp64 for fp64 inputs)."""
    dt = torch.float64 if x.dtype == torch.float64 else torch.float32

    def norm(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w.to(dt)

    u = x.to(dt) if weight is None else norm(x.to(dt), weight)
    if gate is not None:
        u = u * gate.to(dt)
    h = residual.to(dt) + scale * u
    if next_weight is None:
        return h.to(x.dtype)
    return norm(h, next_weight).to(x.dtype), h.to(x.dtype)


def _dense(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous and 16-byte aligned."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _block_norm_forward(x, residual, w1, w2, g, scale, eps, keep: bool):
    """``(y or None, h, stats)`` of dense tensors; the two norms' statistics ``[2, rows]`` only where the backward will ask for them."""
    H = x.shape[-1]
    rows = x.numel() // H
    h = torch.empty_like(x)
    y = torch.empty_like(x) if w2 is not None else None
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    r1 = stats.data_ptr() if keep else None
    mode, a = 0 if g is None else 1 if g.dim() == 1 and x.dim() > 1 else 2, _lib.address
    with _lib.on_device_of(x):
        _lib.check(_lib.lib().mb_block_norm_fwd(x.data_ptr(), residual.data_ptr(), a(w1), a(w2), a(g), mode, h.data_ptr(), a(y), r1,
                                                r1 + 4 * rows if keep else None, _BLOCK_DTYPES[x.dtype], rows, H, scale, eps, _lib.stream_of(x)), "mb_block_norm_fwd")
    return y, h, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, next_weight, gate, scale, eps):
        x, w1, w2, g = _dense(x), _dense(weight), _dense(next_weight), _dense(gate)
        y, h, stats = _block_norm_forward(x, _dense(residual), w1, w2, g, scale, eps, True)
        # x is needed for its norm's and the gate's gradients, h for the next norm's
        ctx.save_for_backward(x if w1 is not None or g is not None else None, h if w2 is not None else None, w1, w2, g, stats)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return h if y is None else (y, h)

    @staticmethod
    def backward(ctx, *douts):
        _lib.refuse_second_order("block_norm")
        x, h, w1, w2, g, stats = ctx.saved_tensors
        dy, dh = douts if w2 is not None else (None, douts[0])
        if dy is None and dh is None:
            return (None,) * 7
        dy, dh = _dense(dy), _dense(dh)
        some = dy if dy is not None else dh
        H = some.shape[-1]
        rows = some.numel() // H
        mode, a = 0 if g is None else 1 if g.dim() == 1 and some.dim() > 1 else 2, _lib.address
        dx, dres = torch.empty_like(some), torch.empty_like(some)
        dw1, dw2, dg = (None if t is None else torch.empty_like(t) for t in (w1, w2, g))
        L = _lib.lib()
        with _lib.on_device_of(some):
            size = L.mb_block_norm_bwd_parts(_BLOCK_DTYPES[some.dtype], rows, H) * H
            parts = torch.empty(2 * size, dtype=torch.float32, device=some.device)
            r1, part = stats.data_ptr(), parts.data_ptr()
            _lib.check(L.mb_block_norm_bwd(a(dy), a(dh), a(x), a(h), a(w1), a(w2), a(g), mode, r1, r1 + 4 * rows, dx.data_ptr(), dres.data_ptr(),
                                           a(dw1), a(dw2), a(dg), part, part + 4 * size, _BLOCK_DTYPES[some.dtype], rows, H, ctx.scale,
                                           _lib.stream_of(some)), "mb_block_norm_bwd")
        return dx, dres, dw1, dw2, dg, None, None


def block_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None, next_weight: torch.Tensor | None = None, *,
               gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6):
    """The seam between two blocks in one pass: ``h = residual + scale * gate * norm(x, weight)`` and ``y = norm(h, next_weight)``,
    with ``norm(t, w) = w * t * rsqrt(mean(t^2) + eps)``. Returns ``(y, h)``, as :func:`add_rms_norm` does, or ``h`` alone without
    ``next_weight``. Differentiable (once) in every tensor.

    ``x`` is the block's output and ``residual`` the stream, any equal shape ``[..., H]``; ``weight=None`` leaves the norm after the
    block out; ``gate`` has one value a channel (``[H]``) or one an element (x's shape). All tensors have one type. On CUDA
    (bf16, fp16, fp32; H a multiple of 8 up to 16384) the kernels of ``csrc/block_norm.cu`` run, else :func:`block_norm_reference`."""
    H = x.shape[-1] if x.dim() else 0
    if x.shape != residual.shape or x.dim() < 1:
        raise ValueError(f"x {tuple(x.shape)} and residual {tuple(residual.shape)} need one shape [..., H]")
    dtype, device = x.dtype, x.device
    for name, t in (("residual", residual), ("weight", weight), ("next_weight", next_weight), ("gate", gate)):
        if t is None:
            continue
        if t.dtype != dtype or t.device != device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {dtype} on {device}")
        if name == "residual" or t.shape == (H,):
            continue
        if name != "gate":
            raise ValueError(f"{name} needs the shape ({H},), got {tuple(t.shape)}")
        if t.shape != x.shape:
            raise ValueError(f"gate needs the shape ({H},) or that of x, {tuple(x.shape)}, got {tuple(t.shape)}")
    if not x.is_floating_point():
        raise ValueError(f"block_norm takes floating-point tensors, got {x.dtype}")
    if not (math.isfinite(scale) and math.isfinite(eps) and eps >= 0):
        raise ValueError(f"scale and eps must be finite and eps not negative, got {scale!r}, {eps!r}")
    if _lib.use_kernels(x) and x.dtype in _BLOCK_DTYPES and x.numel() and H % 8 == 0 and H <= _BLOCK_MAX_HIDDEN:
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, next_weight, gate)):
            return _BlockNorm.apply(x, residual, weight, next_weight, gate, float(scale), float(eps))
        y, h, _ = _block_norm_forward(_dense(x), _dense(residual), _dense(weight), _dense(next_weight), _dense(gate), float(scale),
                                         float(eps), False)
        return h if y is None else (y, h)
    return block_norm_reference(x, residual, weight, next_weight, gate=gate, scale=scale, eps=eps)

"""nnop -- the NNop fused-kernel API over the B200 C-ABI library.

Python mirror of the reference's public Julia API (package ``NNop`` v0.2.0):
same function names, argument meanings, keyword defaults and error behaviour,
with the ChainRules ``rrule``s mapped to ``torch.autograd.Function``s.  Torch is
used only for device memory and streams; every computation is a kernel of
``libnnop_b200.so`` (there is no CPU fallback: CPU tensors are rejected).

Layout: a Julia array of size ``(d1, ..., dn)`` (column-major) is the torch
tensor of shape ``(dn, ..., d1)`` (row-major) over the same memory:

=============================  ===============================
Julia (reference)              torch here
=============================  ===============================
q (E, QL, QH, B)               q (B, QH, QL, E)
k, v (E, KL, KH, B)            k, v (B, KH, KL, E)
pair (QH, QL, KL, B)           pair (B, KL, QL, QH)
kpad_mask::Matrix{Bool} (KL,B) kpad_mask (B, KL) bool / uint8
x (N, cols) [online_softmax]   x (cols, N)
x (emb, n) [norms]             x (n, emb)
cos, sin (E, L, B)             cos, sin (B, L, E) float32
k_cache, v_cache (E, PS, KH, P)  k_cache, v_cache (P, KH, PS, E)
block_table (MP, B) Int32      block_table (B, MP) int32
position_ids (L, B)            position_ids (B, L) float32
=============================  ===============================
"""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from ._lib import (BF16, F16, F32, NNopError, NNopShapeError, check, lib)

__all__ = [
    "flash_attention", "_flash_attention", "grad_flash_attention",
    "flash_attention_pair_per_head", "_flash_attention_pair_per_head", "grad_flash_attention_pair_per_head",
    "flash_attention_rope", "_flash_attention_rope", "grad_flash_attention_rope",
    "online_softmax", "grad_online_softmax",
    "rms_norm", "_rms_norm", "grad_rms_norm",
    "add_rms_norm", "_add_rms_norm", "grad_add_rms_norm",
    "layer_norm", "_layer_norm", "grad_layer_norm",
    "llama_rope", "grad_llama_rope", "LlamaRotaryEmbedding",
    "paged_append", "paged_append_rope", "paged_attention", "_paged_attention", "paged_evict",
    "within_gradient", "NNopError", "NNopShapeError", "lib",
]

_DT = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _dtype_id(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise NNopError(-2, f"unsupported dtype {t.dtype} (float32, float16, bfloat16)") from None


def _dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise NNopError(-3, "nnop operates on CUDA tensors only (no CPU fallback)")
    return ts[0].device


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _contig(t):
    return None if t is None else t.contiguous()


def within_gradient(x) -> bool:
    """``within_gradient`` (src/attention_crc.jl:1-2): true while autograd is
    recording through ``x``."""
    return torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad


# =========================================================================
# flash attention   (src/attention.jl, src/attention_bwd.jl, src/attention_crc.jl)
# =========================================================================

def _mask_u8(kpad_mask):
    if kpad_mask is None:
        return None
    m = kpad_mask
    if m.dtype == torch.bool:
        m = m.view(torch.uint8) if m.is_contiguous() else m.contiguous().view(torch.uint8)
    elif m.dtype != torch.uint8:
        m = (m != 0).to(torch.uint8)
    return m.contiguous()


def _fa_dims(q, k, v, pair, kpad_mask):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise NNopShapeError(-1, "q, k, v must be 4-d (B, H, L, E)")
    B, QH, QL, QE = q.shape
    KB, KH, KL, KE = k.shape
    if QE != KE:
        raise NNopShapeError(-1, f"Embedding dim of Q `{QE}` must be the same as of K `{KE}`.")
    if tuple(k.shape) != tuple(v.shape):
        raise NNopShapeError(-1, f"Shapes of K `{tuple(k.shape)}` and V `{tuple(v.shape)}` must be the same.")
    if KB != B:
        raise NNopShapeError(-1, f"Batch of K `{KB}` must equal batch of Q `{B}`.")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise NNopError(-2, "q, k, v must share a dtype")
    if pair is not None:
        if tuple(pair.shape) != (B, KL, QL, QH):
            raise NNopShapeError(-1, f"pair must have shape (B, KL, QL, QH) = {(B, KL, QL, QH)}, got {tuple(pair.shape)}")
        if pair.dtype != q.dtype:
            raise NNopError(-2, "pair must have the dtype of q")
    if kpad_mask is not None and tuple(kpad_mask.shape) != (B, KL):
        raise NNopShapeError(-1, f"kpad_mask must have shape (B, KL) = {(B, KL)}")
    return B, QH, QL, QE, KH, KL


def _flash_attention(q, k, v, pair=None, *, causal: bool, kpad_mask=None):
    """Forward returning ``(o, lse)`` (``_flash_attention``, src/attention.jl:145-197,
    which returns ``(o, ms, ls)``; here ``lse = ms + log(ls)`` in float32)."""
    o, lse, _ = _flash_attention_ws(q, k, v, pair, causal=causal, kpad_mask=kpad_mask)
    return o, lse


def _flash_attention_ws(q, k, v, pair=None, *, causal: bool, kpad_mask=None):
    """``_flash_attention`` that also returns its workspace (None or a uint8
    tensor holding the per-head pair tiles) for ``grad_flash_attention``'s
    ``fwd_workspace``: the rrule's forward state."""
    dev = _dev(q, k, v, pair, kpad_mask)
    B, QH, QL, E, KH, KL = _fa_dims(q, k, v, pair, kpad_mask)
    q, k, v, pair = _contig(q), _contig(k), _contig(v), _contig(pair)
    m = _mask_u8(kpad_mask)
    o = torch.empty_like(q)
    lse = torch.empty((B, QH, QL), dtype=torch.float32, device=dev)
    dt = _dtype_id(q)
    ws_bytes = lib.nnop_flash_attention_fwd_workspace_size(E, QL, KL, QH, KH, B, int(pair is not None), dt)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    check(lib.nnop_flash_attention_fwd(
        _ptr(q), _ptr(k), _ptr(v), _ptr(pair), _ptr(m), _ptr(o), _ptr(lse), _ptr(ws), ws_bytes,
        E, QL, KL, QH, KH, B, int(bool(causal)), dt, _stream(dev)))
    return o, lse, ws


def grad_flash_attention(do, o, lse, q, k, v, pair=None, *, causal: bool, kpad_mask=None, fwd_workspace=None):
    """``∇flash_attention`` (src/attention_bwd.jl:213-303): returns
    ``(dq, dk, dv, dpair)``, dpair None when pair is None.  ``fwd_workspace``:
    the workspace ``_flash_attention_ws`` returned for the same inputs; its
    pair tiles are then reused instead of rebuilt."""
    dev = _dev(do, o, lse, q, k, v, pair, kpad_mask)
    B, QH, QL, E, KH, KL = _fa_dims(q, k, v, pair, kpad_mask)
    do, o, q, k, v, pair = map(_contig, (do, o, q, k, v, pair))
    if do.dtype != q.dtype:
        do = do.to(q.dtype)
    lse = lse.contiguous()
    m = _mask_u8(kpad_mask)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dpair = torch.empty_like(pair) if pair is not None else None
    dt = _dtype_id(q)
    fw_bytes = 0 if fwd_workspace is None else fwd_workspace.numel()
    ws_bytes = lib.nnop_flash_attention_bwd_workspace_size_reuse(E, QL, KL, QH, KH, B, int(pair is not None),
                                                                  fw_bytes, dt)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    check(lib.nnop_flash_attention_bwd_reuse(
        _ptr(do), _ptr(o), _ptr(lse), _ptr(q), _ptr(k), _ptr(v), _ptr(pair), _ptr(m),
        _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dpair), _ptr(fwd_workspace), fw_bytes, _ptr(ws), ws_bytes,
        E, QL, KL, QH, KH, B, int(bool(causal)), dt, _stream(dev)))
    return dq, dk, dv, dpair


class _FlashAttentionFn(torch.autograd.Function):
    """``CRC.rrule(::typeof(_flash_attention), ...)`` (src/attention_crc.jl:16-31)."""

    @staticmethod
    def forward(ctx, q, k, v, pair, kpad_mask, causal):
        o, lse, ws = _flash_attention_ws(q, k, v, pair, causal=causal, kpad_mask=kpad_mask)
        ctx.save_for_backward(o, lse, q, k, v, pair, kpad_mask, ws)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        o, lse, q, k, v, pair, kpad_mask, ws = ctx.saved_tensors
        dq, dk, dv, dpair = grad_flash_attention(do, o, lse, q, k, v, pair, causal=ctx.causal,
                                                 kpad_mask=kpad_mask, fwd_workspace=ws)
        return dq, dk, dv, dpair, None, None


def flash_attention(q, k, v, pair=None, *, causal: bool, kpad_mask=None):
    """``NNop.flash_attention(q, k, v, pair=nothing; causal, kpad_mask=nothing)``
    (src/attention_crc.jl:4-14): returns ``o``; differentiable w.r.t. q, k, v,
    pair when autograd records."""
    if any(within_gradient(t) for t in (q, k, v, pair)):
        return _FlashAttentionFn.apply(q, k, v, pair, kpad_mask, bool(causal))
    return _flash_attention(q, k, v, pair, causal=causal, kpad_mask=kpad_mask)[0]


# -------------------------------------------------------------------------
# pair bias laid out per head: Julia (QL, KL, QH, B) = torch (B, QH, KL, QL)
# -------------------------------------------------------------------------

def _per_head_dims(q, k, v, pair, kpad_mask):
    if pair is None:
        raise NNopError(-3, "the per-head entry points take a pair bias")
    if pair.dim() != 4:
        raise NNopShapeError(-1, "pair must be 4-d (B, QH, KL, QL)")
    B, QH, QL, E, KH, KL = _fa_dims(q, k, v, None, kpad_mask)
    if tuple(pair.shape) != (B, QH, KL, QL):
        raise NNopShapeError(-1, f"pair must have shape (B, QH, KL, QL) = {(B, QH, KL, QL)}, got {tuple(pair.shape)}")
    if pair.dtype != q.dtype:
        raise NNopError(-2, "pair must have the dtype of q")
    return B, QH, QL, E, KH, KL


def _flash_attention_pair_per_head(q, k, v, pair, *, causal: bool, kpad_mask=None):
    """``_flash_attention`` with the pair bias laid out per head, torch shape
    (B, QH, KL, QL) (Julia (QL, KL, QH, B)), read in place by the tensor-core
    kernel (no re-layout pass, no workspace).  bf16/f16, E = 64, QL % 8 == 0;
    −Inf bias entries only at keys ``kpad_mask`` removes.  Returns ``(o, lse)``."""
    dev = _dev(q, k, v, pair, kpad_mask)
    B, QH, QL, E, KH, KL = _per_head_dims(q, k, v, pair, kpad_mask)
    q, k, v, pair = _contig(q), _contig(k), _contig(v), _contig(pair)
    m = _mask_u8(kpad_mask)
    o = torch.empty_like(q)
    lse = torch.empty((B, QH, QL), dtype=torch.float32, device=dev)
    check(lib.nnop_flash_attention_fwd_pair_per_head(
        _ptr(q), _ptr(k), _ptr(v), _ptr(pair), _ptr(m), _ptr(o), _ptr(lse),
        E, QL, KL, QH, KH, B, int(bool(causal)), _dtype_id(q), _stream(dev)))
    return o, lse


def grad_flash_attention_pair_per_head(do, o, lse, q, k, v, pair, *, causal: bool, kpad_mask=None):
    """``∇flash_attention`` with pair and dpair laid out per head (B, QH, KL, QL):
    returns ``(dq, dk, dv, dpair)``; dS is stored straight into dpair."""
    dev = _dev(do, o, lse, q, k, v, pair, kpad_mask)
    B, QH, QL, E, KH, KL = _per_head_dims(q, k, v, pair, kpad_mask)
    do, o, q, k, v, pair = map(_contig, (do, o, q, k, v, pair))
    if do.dtype != q.dtype:
        do = do.to(q.dtype)
    lse = lse.contiguous()
    m = _mask_u8(kpad_mask)
    dq, dk, dv, dpair = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(pair)
    dt = _dtype_id(q)
    ws_bytes = lib.nnop_flash_attention_bwd_pair_per_head_workspace_size(E, QL, KL, QH, KH, B, dt)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    check(lib.nnop_flash_attention_bwd_pair_per_head(
        _ptr(do), _ptr(o), _ptr(lse), _ptr(q), _ptr(k), _ptr(v), _ptr(pair), _ptr(m),
        _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dpair), _ptr(ws), ws_bytes,
        E, QL, KL, QH, KH, B, int(bool(causal)), dt, _stream(dev)))
    return dq, dk, dv, dpair


class _FlashAttentionPerHeadFn(torch.autograd.Function):
    """The rrule of ``flash_attention_pair_per_head`` (the structure of
    src/attention_crc.jl:16-31 with the per-head pair layout)."""

    @staticmethod
    def forward(ctx, q, k, v, pair, kpad_mask, causal):
        o, lse = _flash_attention_pair_per_head(q, k, v, pair, causal=causal, kpad_mask=kpad_mask)
        ctx.save_for_backward(o, lse, q, k, v, pair, kpad_mask)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        o, lse, q, k, v, pair, kpad_mask = ctx.saved_tensors
        dq, dk, dv, dpair = grad_flash_attention_pair_per_head(do, o, lse, q, k, v, pair, causal=ctx.causal,
                                                               kpad_mask=kpad_mask)
        return dq, dk, dv, dpair, None, None


def flash_attention_pair_per_head(q, k, v, pair, *, causal: bool, kpad_mask=None):
    """``flash_attention`` with the pair bias laid out per head, torch shape
    (B, QH, KL, QL) (Julia (QL, KL, QH, B)); differentiable w.r.t. q, k, v,
    pair.  Same results as ``flash_attention(q, k, v, pair.permute(0, 2, 3, 1))``."""
    if any(within_gradient(t) for t in (q, k, v, pair)):
        return _FlashAttentionPerHeadFn.apply(q, k, v, pair, kpad_mask, bool(causal))
    return _flash_attention_pair_per_head(q, k, v, pair, causal=causal, kpad_mask=kpad_mask)[0]


# -------------------------------------------------------------------------
# Llama RoPE fused with attention: flash_attention(llama_rope(q, k)...)
# -------------------------------------------------------------------------

def _rope_tables(cos, sin, B, L, E):
    cos = cos.contiguous().to(torch.float32)
    sin = sin.contiguous().to(torch.float32)
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    if cos.shape != sin.shape or cos.shape[1] != L or cos.shape[2] != E or cos.shape[0] not in (1, B):
        raise NNopShapeError(-1, "cos/sin must have shape (B or 1, L, E)")
    return cos, sin


def _flash_attention_rope(q, k, v, *, cos, sin, causal: bool, kpad_mask=None):
    """``llama_rope`` then ``_flash_attention`` in one call: returns
    ``(o, lse, q_rot, k_rot)``; the rotated q and k are the backward's inputs.
    bf16/f16, E = 64 or 128, q and k of one length L."""
    dev = _dev(q, k, v, cos, sin, kpad_mask)
    B, QH, QL, E, KH, KL = _fa_dims(q, k, v, None, kpad_mask)
    if QL != KL:
        raise NNopShapeError(-1, "q and k must share the sequence length")
    cos, sin = _rope_tables(cos, sin, B, QL, E)
    q, k, v = _contig(q), _contig(k), _contig(v)
    m = _mask_u8(kpad_mask)
    qr, kr, o = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    lse = torch.empty((B, QH, QL), dtype=torch.float32, device=dev)
    check(lib.nnop_flash_attention_rope_fwd(
        _ptr(q), _ptr(k), _ptr(v), _ptr(cos), _ptr(sin), _ptr(m), _ptr(qr), _ptr(kr), _ptr(o), _ptr(lse),
        E, QL, QH, KH, B, cos.shape[0], int(bool(causal)), _dtype_id(q), _stream(dev)))
    return o, lse, qr, kr


def grad_flash_attention_rope(do, o, lse, q_rot, k_rot, v, *, cos, sin, causal: bool, kpad_mask=None):
    """Backward of ``_flash_attention_rope``: ``(dq, dk, dv)`` with dq, dk the
    gradients of the UN-rotated q and k (``∇llama_rope`` folded into the
    attention backward's outputs)."""
    dev = _dev(do, o, lse, q_rot, k_rot, v, cos, sin, kpad_mask)
    B, QH, L, E, KH, _ = _fa_dims(q_rot, k_rot, v, None, kpad_mask)
    cos, sin = _rope_tables(cos, sin, B, L, E)
    do, o, q_rot, k_rot, v = map(_contig, (do, o, q_rot, k_rot, v))
    if do.dtype != q_rot.dtype:
        do = do.to(q_rot.dtype)
    m = _mask_u8(kpad_mask)
    dq, dk, dv = torch.empty_like(q_rot), torch.empty_like(k_rot), torch.empty_like(v)
    dt = _dtype_id(q_rot)
    ws_bytes = lib.nnop_flash_attention_rope_bwd_workspace_size(E, L, QH, KH, B, dt)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    check(lib.nnop_flash_attention_rope_bwd(
        _ptr(do), _ptr(o), _ptr(lse.contiguous()), _ptr(q_rot), _ptr(k_rot), _ptr(v), _ptr(cos), _ptr(sin), _ptr(m),
        _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), ws_bytes, E, L, QH, KH, B, cos.shape[0], int(bool(causal)), dt,
        _stream(dev)))
    return dq, dk, dv


class _FlashAttentionRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cos, sin, kpad_mask, causal):
        o, lse, qr, kr = _flash_attention_rope(q, k, v, cos=cos, sin=sin, causal=causal, kpad_mask=kpad_mask)
        ctx.save_for_backward(o, lse, qr, kr, v, cos, sin, kpad_mask)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        o, lse, qr, kr, v, cos, sin, kpad_mask = ctx.saved_tensors
        dq, dk, dv = grad_flash_attention_rope(do, o, lse, qr, kr, v, cos=cos, sin=sin, causal=ctx.causal,
                                               kpad_mask=kpad_mask)
        return dq, dk, dv, None, None, None, None


def flash_attention_rope(q, k, v, *, cos, sin, causal: bool, kpad_mask=None):
    """``flash_attention(llama_rope(q, k; cos, sin)..., v)`` with the RoPE
    backward folded into the attention backward; differentiable w.r.t. the
    un-rotated q, k and v."""
    if any(within_gradient(t) for t in (q, k, v)):
        return _FlashAttentionRopeFn.apply(q, k, v, cos, sin, kpad_mask, bool(causal))
    return _flash_attention_rope(q, k, v, cos=cos, sin=sin, causal=causal, kpad_mask=kpad_mask)[0]


# =========================================================================
# online softmax   (src/softmax.jl)
# =========================================================================

def _softmax_fwd(x):
    dev = _dev(x)
    x = x.contiguous()
    n = x.shape[-1]
    cols = x.numel() // n if n else 0
    y = torch.empty_like(x)
    check(lib.nnop_online_softmax_fwd(_ptr(x), _ptr(y), n, cols, _dtype_id(x), _stream(dev)))
    return y


def grad_online_softmax(dy, y):
    """``∇online_softmax`` (src/softmax.jl:70-80): dy∘y − y∘Σ(dy∘y)."""
    dev = _dev(dy, y)
    y = y.contiguous()
    dy = dy.contiguous().to(y.dtype)
    n = y.shape[-1]
    dx = torch.empty_like(y)
    check(lib.nnop_online_softmax_bwd(_ptr(dy), _ptr(y), _ptr(dx), n, y.numel() // n, _dtype_id(y),
                                      _stream(dev)))
    return dx


class _SoftmaxFn(torch.autograd.Function):
    """``CRC.rrule(::typeof(online_softmax), x)`` (src/softmax.jl:82-86)."""

    @staticmethod
    def forward(ctx, x):
        y = _softmax_fwd(x)
        ctx.save_for_backward(y)
        return y

    @staticmethod
    def backward(ctx, dy):
        (y,) = ctx.saved_tensors
        return grad_online_softmax(dy, y)


def online_softmax(x):
    """``NNop.online_softmax(x)`` (src/softmax.jl:60-68): softmax over the
    contiguous axis (Julia dims=1)."""
    if within_gradient(x):
        return _SoftmaxFn.apply(x)
    return _softmax_fwd(x)


# =========================================================================
# RMSNorm   (src/rms_norm.jl)
# =========================================================================

def _norm_dims(x, w):
    emb = x.shape[-1]
    if w.numel() != emb:
        raise NNopShapeError(-1, f"weight length {w.numel()} must equal emb {emb}")
    return emb, x.numel() // emb if emb else 0


def _rms_norm(x, w, *, eps: float = 1e-6, offset: float = 0.0):
    """``_rms_norm`` (src/rms_norm.jl:117-137): returns ``(y, rstd)``."""
    dev = _dev(x, w)
    x = x.contiguous()
    w = w.contiguous().to(x.dtype)
    emb, n = _norm_dims(x, w)
    y = torch.empty_like(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    check(lib.nnop_rms_norm_fwd(_ptr(x), _ptr(w), _ptr(y), _ptr(rstd), emb, n, float(eps), float(offset),
                                _dtype_id(x), _stream(dev)))
    return y, rstd


def grad_rms_norm(dy, rstd, x, w, *, offset: float = 0.0):
    """``∇rms_norm`` (src/rms_norm.jl:139-169): returns ``(dx, dw)``, dw float32."""
    dev = _dev(dy, rstd, x, w)
    x = x.contiguous()
    w = w.contiguous().to(x.dtype)
    dy = dy.contiguous().to(x.dtype)
    emb, n = _norm_dims(x, w)
    dx = torch.empty_like(x)
    dw = torch.empty(emb, dtype=torch.float32, device=dev)
    ws_bytes = lib.nnop_rms_norm_bwd_workspace_size(emb, n)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    check(lib.nnop_rms_norm_bwd(_ptr(dy), _ptr(x), _ptr(w), _ptr(rstd.contiguous()), _ptr(dx), _ptr(dw),
                                _ptr(ws), ws_bytes, emb, n, float(offset), _dtype_id(x), _stream(dev)))
    return dx, dw


class _RmsNormFn(torch.autograd.Function):
    """``CRC.rrule(::typeof(_rms_norm), x, w)`` (src/rms_norm.jl:178-185)."""

    @staticmethod
    def forward(ctx, x, w, eps, offset):
        y, rstd = _rms_norm(x, w, eps=eps, offset=offset)
        ctx.save_for_backward(x, w, rstd)
        ctx.offset = offset
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, rstd = ctx.saved_tensors
        dx, dw = grad_rms_norm(dy, rstd, x, w, offset=ctx.offset)
        return dx, dw.to(w.dtype).reshape(w.shape), None, None


def rms_norm(x, w, *, eps: float = 1e-6, offset: float = 0.0):
    """``NNop.rms_norm(x, w; ϵ=1f-6, offset=0f0)`` (src/rms_norm.jl:171-176)."""
    if within_gradient(x) or within_gradient(w):
        return _RmsNormFn.apply(x, w, float(eps), float(offset))
    return _rms_norm(x, w, eps=eps, offset=offset)[0]


# -------------------------------------------------------------------------
# residual add fused into RMSNorm (the composition a transformer block makes
# around rms_norm; no counterpart in the reference's API)
# -------------------------------------------------------------------------

def _add_rms_norm(x, residual, w, *, eps: float = 1e-6, offset: float = 0.0):
    """``h = x + residual`` (rounded to the dtype) and ``rms_norm(h, w)`` in one
    pass: returns ``(y, h, rstd)``."""
    dev = _dev(x, residual, w)
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise NNopShapeError(-1, "residual must have the shape and dtype of x")
    x, residual = x.contiguous(), residual.contiguous()
    w = w.contiguous().to(x.dtype)
    emb, n = _norm_dims(x, w)
    h, y = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    check(lib.nnop_add_rms_norm_fwd(_ptr(x), _ptr(residual), _ptr(w), _ptr(h), _ptr(y), _ptr(rstd), emb, n,
                                    float(eps), float(offset), _dtype_id(x), _stream(dev)))
    return y, h, rstd


def grad_add_rms_norm(dy, dh, h, w, rstd, *, offset: float = 0.0):
    """Backward of ``_add_rms_norm``: ``dx = ∇rms_norm(dy, h) + dh`` (dh, the
    gradient reaching h from the residual stream, may be None) -- the gradient
    of both x and residual -- and ``dw`` (float32)."""
    dev = _dev(dy, h, w, rstd)
    h = h.contiguous()
    w = w.contiguous().to(h.dtype)
    dy = dy.contiguous().to(h.dtype)
    if dh is not None:
        dh = dh.contiguous().to(h.dtype)
    emb, n = _norm_dims(h, w)
    dx = torch.empty_like(h)
    dw = torch.empty(emb, dtype=torch.float32, device=dev)
    ws_bytes = lib.nnop_add_rms_norm_bwd_workspace_size(emb, n)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    check(lib.nnop_add_rms_norm_bwd(_ptr(dy), _ptr(dh), _ptr(h), _ptr(w), _ptr(rstd.contiguous()), _ptr(dx),
                                    _ptr(dw), _ptr(ws), ws_bytes, emb, n, float(offset), _dtype_id(h), _stream(dev)))
    return dx, dw


class _AddRmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, w, eps, offset):
        y, h, rstd = _add_rms_norm(x, residual, w, eps=eps, offset=offset)
        ctx.save_for_backward(h, w, rstd)
        ctx.offset = offset
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        h, w, rstd = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(h)
        dx, dw = grad_add_rms_norm(dy, dh, h, w, rstd, offset=ctx.offset)
        return dx, dx, dw.to(w.dtype).reshape(w.shape), None, None


def add_rms_norm(x, residual, w, *, eps: float = 1e-6, offset: float = 0.0):
    """Residual add and ``rms_norm`` fused: returns ``(y, h)`` with
    ``h = x + residual`` (the new residual stream) and ``y = rms_norm(h, w)``;
    differentiable w.r.t. x, residual and w."""
    if any(within_gradient(t) for t in (x, residual, w)):
        return _AddRmsNormFn.apply(x, residual, w, float(eps), float(offset))
    y, h, _ = _add_rms_norm(x, residual, w, eps=eps, offset=offset)
    return y, h


# =========================================================================
# LayerNorm   (src/layer_norm.jl)
# =========================================================================

def _layer_norm(x, w, b, *, eps: float = 1e-6):
    """``_layer_norm`` (src/layer_norm.jl:150-170): returns ``(y, mean, rstd)``."""
    dev = _dev(x, w, b)
    x = x.contiguous()
    w = w.contiguous().to(x.dtype)
    b = b.contiguous().to(x.dtype)
    emb, n = _norm_dims(x, w)
    if b.numel() != emb:
        raise NNopShapeError(-1, f"bias length {b.numel()} must equal emb {emb}")
    y = torch.empty_like(x)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    check(lib.nnop_layer_norm_fwd(_ptr(x), _ptr(w), _ptr(b), _ptr(y), _ptr(mean), _ptr(rstd), emb, n,
                                  float(eps), _dtype_id(x), _stream(dev)))
    return y, mean, rstd


def grad_layer_norm(dy, mean, rstd, x, w, b=None):
    """``∇layer_norm`` (src/layer_norm.jl:172-204): returns ``(dx, dw, db)`` in
    the dtype of x."""
    dev = _dev(dy, mean, rstd, x, w)
    x = x.contiguous()
    w = w.contiguous().to(x.dtype)
    dy = dy.contiguous().to(x.dtype)
    emb, n = _norm_dims(x, w)
    dx = torch.empty_like(x)
    dw = torch.empty(emb, dtype=x.dtype, device=dev)
    db = torch.empty(emb, dtype=x.dtype, device=dev)
    ws_bytes = lib.nnop_layer_norm_bwd_workspace_size(emb, n)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    check(lib.nnop_layer_norm_bwd(_ptr(dy), _ptr(x), _ptr(w), _ptr(mean.contiguous()), _ptr(rstd.contiguous()),
                                  _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), ws_bytes, emb, n, _dtype_id(x),
                                  _stream(dev)))
    return dx, dw, db


class _LayerNormFn(torch.autograd.Function):
    """``CRC.rrule(::typeof(_layer_norm), x, w, b)`` (src/layer_norm.jl:213-220)."""

    @staticmethod
    def forward(ctx, x, w, b, eps):
        y, mean, rstd = _layer_norm(x, w, b, eps=eps)
        ctx.save_for_backward(x, w, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        dx, dw, db = grad_layer_norm(dy, mean, rstd, x, w)
        return dx, dw.to(w.dtype).reshape(w.shape), db.to(w.dtype).reshape(w.shape), None


def layer_norm(x, w, b, *, eps: float = 1e-6):
    """``NNop.layer_norm(x, w, b; ϵ=1f-6)`` (src/layer_norm.jl:206-211)."""
    if any(within_gradient(t) for t in (x, w, b)):
        return _LayerNormFn.apply(x, w, b, float(eps))
    return _layer_norm(x, w, b, eps=eps)[0]


# =========================================================================
# Llama RoPE   (src/rope/llama_rope.jl)
# =========================================================================

class LlamaRotaryEmbedding:
    """``LlamaRotaryEmbedding(dim; base=10000)`` (src/rope/llama_rope.jl:1-22).

    ``emb(position_ids)`` with position_ids (B, L) float32 returns ``(cos, sin)``
    of shape (B, L, dim) float32, computed on the device."""

    def __init__(self, dim: int, *, base: int = 10000):
        if dim <= 0 or dim % 2:
            raise NNopShapeError(-1, "dim must be even and > 0")
        self.dim = int(dim)
        self.base = int(base)

    def __call__(self, position_ids):
        pos = position_ids
        if not isinstance(pos, torch.Tensor):
            pos = torch.as_tensor(pos)
        if not pos.is_cuda:
            pos = pos.cuda()
        pos = pos.to(torch.float32).contiguous()
        if pos.dim() == 1:
            pos = pos[None]
        B, L = pos.shape
        cos = torch.empty((B, L, self.dim), dtype=torch.float32, device=pos.device)
        sin = torch.empty_like(cos)
        check(lib.nnop_llama_rope_cos_sin(_ptr(pos), _ptr(cos), _ptr(sin), self.dim, L, B, self.base,
                                          _stream(pos.device)))
        return cos, sin


def _llama_rope(q, k, cos, sin, *, bwd: bool):
    dev = _dev(q, k, cos, sin)
    if q.dim() != 4 or k.dim() != 4:
        raise NNopShapeError(-1, "q, k must be 4-d (B, H, L, E)")
    B, QH, L, E = q.shape
    if k.shape[0] != B or k.shape[2] != L or k.shape[3] != E:
        raise NNopShapeError(-1, "q and k must share batch, sequence length and embedding dim")
    KH = k.shape[1]
    cos = cos.contiguous().to(torch.float32)
    sin = sin.contiguous().to(torch.float32)
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    if cos.shape != sin.shape or cos.shape[1] != L or cos.shape[2] != E:
        raise NNopShapeError(-1, "cos/sin must have shape (B or 1, L, E)")
    q, k = q.contiguous(), k.contiguous()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    check(lib.nnop_llama_rope(_ptr(q), _ptr(k), _ptr(cos), _ptr(sin), _ptr(qo), _ptr(ko), E, L, QH, KH, B,
                              cos.shape[0], -1.0 if bwd else 1.0, _dtype_id(q), _stream(dev)))
    return qo, ko


def grad_llama_rope(dq, dk, *, cos, sin):
    """``∇llama_rope`` (src/rope/llama_rope.jl:92): the rotation with sin → −sin."""
    return _llama_rope(dq, dk, cos, sin, bwd=True)


class _RopeFn(torch.autograd.Function):
    """``CRC.rrule(::typeof(llama_rope), q, k; cos, sin)`` (src/rope/llama_rope.jl:94-98)."""

    @staticmethod
    def forward(ctx, q, k, cos, sin):
        ctx.save_for_backward(cos, sin)
        return _llama_rope(q, k, cos, sin, bwd=False)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin = ctx.saved_tensors
        dq = torch.zeros_like(dq) if dq is None else dq
        dk = torch.zeros_like(dk) if dk is None else dk
        gq, gk = _llama_rope(dq, dk, cos, sin, bwd=True)
        return gq, gk, None, None


def llama_rope(q, k, *, cos, sin):
    """``NNop.llama_rope(q, k; cos, sin)`` (src/rope/llama_rope.jl:91): returns
    rotated copies ``(q, k)``."""
    if within_gradient(q) or within_gradient(k):
        return _RopeFn.apply(q, k, cos, sin)
    return _llama_rope(q, k, cos, sin, bwd=False)


# =========================================================================
# paged key-value cache (no counterpart in the reference, whose attention takes
# whole sequences: the step after it, one new token against the cached ones)
# =========================================================================

# These run once per generated token and layer, where the host's time is most of a small
# call's: plain checks in the order of a valid call, the device as its index (-1 on the
# CPU), messages made only when they are needed.

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # a torch without CUDA has none; no call gets that far there
_workspace_bytes = functools.lru_cache(maxsize=1024)(lib.nnop_paged_attention_fwd_workspace_size)


def _paged_device(name, *ts):
    """Index of the CUDA device that all of ts (None allowed) are on."""
    dev = ts[0].get_device()
    for t in ts:
        if t is not None and (dev < 0 or t.get_device() != dev):
            if not (ts[0].is_cuda and t.is_cuda):
                raise NNopError(-3, "nnop operates on CUDA tensors only (no CPU fallback)")
            raise NNopError(-3, f"{name}: all tensors must be on one device")
    return dev


def _paged_dims(name, k_cache, v_cache, block_table, lengths, write):
    """Checks of the cache arguments the paged calls share; returns the batch, KH, E
    and ``(pages, page_size, max_pages, strides...)`` as the C ABI takes them."""
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape:
        raise NNopShapeError(-1, f"{name}: k_cache and v_cache must be 4-d (P, KH, PS, E) of one shape")
    if k_cache.dtype is not v_cache.dtype:
        raise NNopError(-2, f"{name}: k_cache and v_cache must share a dtype")
    if block_table.dtype is not torch.int32 or lengths.dtype is not torch.int32:
        raise NNopError(-2, f"{name}: block_table and lengths must be int32")
    tshape, nshape = block_table.shape, lengths.shape
    if len(tshape) != 2 or len(nshape) != 1 or tshape[0] != nshape[0]:
        raise NNopShapeError(-1, f"{name}: block_table must be (B, MP) and lengths (B,)")
    P, KH, PS, E = shape
    sp, sh, sr, se = strides = k_cache.stride()
    if P <= 1 or KH <= 1 or PS <= 1 or strides != v_cache.stride():   # the stride of an axis of length 1 means nothing
        (sp, sh, sr), sv = (tuple(st if n > 1 else 0 for n, st in zip((P, KH, PS), t.stride())) for t in (k_cache, v_cache))
        if (sp, sh, sr) != sv:
            raise NNopShapeError(-1, f"{name}: k_cache and v_cache must have the same strides")
        se = se if v_cache.stride(3) == 1 else 0
    if se != 1 and E > 1:
        raise NNopShapeError(-1, f"{name}: the caches' embedding axis must be contiguous")
    if write and ((sp == 0 and P > 1) or (sh == 0 and KH > 1) or (sr == 0 and PS > 1)):
        raise NNopShapeError(-1, f"{name}: an expanded cache cannot be written")
    return nshape[0], KH, E, (P, PS, tshape[1], sp, sh, sr)


def _no_grad(name, *ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise NNopError(-3, f"{name} has no gradient: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:           # inside forward_ad.dual_level()
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NNopError(-3, f"{name} has no forward-mode derivative: call it on tensors without a tangent")


def _aligned(t):
    """Contiguous and on a 16-byte boundary (a view may start off one)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _on(dev, written, fn, *args):
    """Calls the library on device ``dev`` with its current stream last.  ``written``: the
    caller's tensors it changes in place, whose version torch is told to count up, so that
    a backward pass that saved one of them refuses to go on."""
    if dev == torch.cuda.current_device():
        status = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(dev))
    if status:
        check(status)
    if written:
        torch.autograd.graph.increment_version(written)


def _paged_append(name, q, k, v, k_cache, v_cache, block_table, lengths, cos, sin, n_new):
    dev = _paged_device(name, k_cache, v_cache, block_table, lengths, k, v, q, cos, sin, n_new)
    B, KH, E, cache = _paged_dims(name, k_cache, v_cache, block_table, lengths, True)
    _no_grad(name, q, k, v, k_cache, v_cache)
    shape, dtype = k.shape, k_cache.dtype
    if len(shape) != 4 or shape != v.shape or shape[0] != B or shape[1] != KH or shape[3] != E:
        raise NNopShapeError(-1, f"{name}: k and v must be (B, KH, T, E) = ({B}, {KH}, T, {E})")
    if k.dtype is not dtype or v.dtype is not dtype or (q is not None and q.dtype is not dtype):
        raise NNopError(-2, f"{name}: q, k and v must have the dtype of the caches")
    T = shape[2]
    QH, cb, qo = 0, 1, None
    if cos is not None:
        if cos.dim() not in (2, 3):
            raise NNopShapeError(-1, "cos/sin must have shape (B or 1, L, E)")
        cb, f32 = cos.shape[0], torch.float32
        if cos.shape == (cb, T, E) == sin.shape and cb in (1, B) and cos.dtype is f32 and sin.dtype is f32:
            cos, sin = cos.contiguous(), sin.contiguous()
        else:
            cos, sin = _rope_tables(cos, sin, B, T, E)
            cb = cos.shape[0]
    if q is not None:
        qshape = q.shape
        if len(qshape) != 4 or qshape[0] != B or qshape[2] != T or qshape[3] != E:
            raise NNopShapeError(-1, f"{name}: q must be (B, QH, T, E) = ({B}, QH, {T}, {E})")
        QH = qshape[1]
        q = _aligned(q)
        qo = torch.empty_like(q)
    if n_new is not None:
        if tuple(n_new.shape) != (B,):
            raise NNopShapeError(-1, f"{name}: n_new must be (B,) = ({B},)")
        if n_new.dtype is not torch.int32:
            raise NNopError(-2, f"{name}: n_new must be int32")
        n_new = n_new.contiguous()
    k, v, lengths, block_table = _aligned(k), _aligned(v), lengths.contiguous(), block_table.contiguous()
    new_lengths = torch.empty_like(lengths)
    _on(dev, (k_cache, v_cache), lib.nnop_paged_append, _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(cos), _ptr(sin), _ptr(n_new), _ptr(qo),
        k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), new_lengths.data_ptr(), E, T,
        QH, KH, B, cb, *cache, _dtype_id(k_cache))
    return qo, new_lengths


def paged_append(k, v, k_cache, v_cache, block_table, lengths, *, n_new=None):
    """Writes the new rows ``k``, ``v`` (B, KH, T, E) behind what each sequence
    has in the paged cache and returns the new lengths (B,) int32 (``lengths``
    itself stays).

    ``k_cache``, ``v_cache`` (P, KH, PS, E): the pools, written in place; any
    strides with E contiguous, the same for both.  ``block_table`` (B, MP) int32:
    the page of each run of PS slots; an entry outside [0, P) is no page and rows
    meant for it are dropped (their slots count as used, and are not attended to),
    as are rows past the table's MP·PS slots: the new lengths then fall short of
    ``lengths + n_new``.
    ``n_new`` (B,) int32: how many of the T rows are tokens, for a padded batch
    (default all).  A page that is written belongs to one sequence."""
    return _paged_append("paged_append", None, k, v, k_cache, v_cache, block_table, lengths, None, None, n_new)[1]


def paged_append_rope(q, k, v, k_cache, v_cache, block_table, lengths, *, cos, sin, n_new=None):
    """``llama_rope(q, k; cos, sin)`` and ``paged_append`` of the rotated k in
    one launch: returns ``(q_rot, new_lengths)``.  ``cos``, ``sin`` (B or 1, T, E)
    float32 from ``LlamaRotaryEmbedding`` at the new tokens' positions."""
    if cos is None or sin is None or q is None:
        raise NNopError(-3, "paged_append_rope takes q, cos and sin")
    return _paged_append("paged_append_rope", q, k, v, k_cache, v_cache, block_table, lengths, cos, sin, n_new)


def _paged_attention(q, k_cache, v_cache, block_table, lengths, *, weights=None):
    """``paged_attention`` returning ``(o, lse)``, lse (B, QH, 1) float32."""
    name = "paged_attention"
    dev = _paged_device(name, k_cache, v_cache, block_table, lengths, q, weights)
    B, KH, E, cache = _paged_dims(name, k_cache, v_cache, block_table, lengths, False)
    _no_grad(name, q, k_cache, v_cache, weights)
    shape = q.shape
    if len(shape) != 4 or shape[0] != B or shape[2] != 1:
        raise NNopShapeError(-1, f"{name}: q must be (B, QH, 1, E) with B = {B}")
    if shape[3] != E:
        raise NNopShapeError(-1, f"Embedding dim of Q `{shape[3]}` must be the same as of K `{E}`.")
    if q.dtype is not k_cache.dtype:
        raise NNopError(-2, f"{name}: q must have the dtype of the caches")
    QH, weigh = shape[1], weights is not None
    if weigh:
        if tuple(weights.shape) != (B, KH, cache[1] * cache[2]):
            raise NNopShapeError(-1, f"{name}: weights must have shape (B, KH, MP·PS) = {(B, KH, cache[1] * cache[2])}")
        if weights.dtype is not torch.float32 or not weights.is_contiguous():
            raise NNopError(-2, f"{name}: weights must be contiguous float32")
    q, lengths, block_table, dt = _aligned(q), lengths.contiguous(), block_table.contiguous(), _dtype_id(q)
    ws_bytes = _workspace_bytes(E, QH, KH, B, cache[1], cache[2], weigh, dt)
    o, lse = torch.empty_like(q), q.new_empty((B, QH, 1), dtype=torch.float32)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8)
    _on(dev, (weights,) if weigh else (), lib.nnop_paged_attention_fwd, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
        lengths.data_ptr(), weights.data_ptr() if weigh else None, o.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws_bytes,
        E, QH, KH, B, *cache, dt)
    return o, lse


def paged_attention(q, k_cache, v_cache, block_table, lengths, *, weights=None):
    """Attention of one new token per sequence over the paged cache:
    ``flash_attention`` of q (B, QH, 1, E) with the first ``lengths[b]`` slots of
    sequence b as its keys and values; returns o (B, QH, 1, E).

    Pools, table and lengths as in ``paged_append`` (slots without a page are
    not attended to; a sequence without a slot gets zeros).  ``weights``
    (B, KH, MP·PS) float32, contiguous: each attended slot's softmax weight,
    summed over the query heads of its kv head, is added to it in place --
    what ``paged_evict`` goes by; the call then takes a workspace of 4 bytes per
    query head and slot of the table, whatever the lengths."""
    return _paged_attention(q, k_cache, v_cache, block_table, lengths, weights=weights)[0]


def paged_evict(k_cache, v_cache, block_table, new_table, lengths, weights, *, budget: int, recent: int = 0):
    """Cuts each sequence's cache to at most ``budget`` slots per kv head: the
    last ``recent`` ones and, of the others, those with the largest accumulated
    ``weights`` (B, KH, MP·PS); equal weights: the lower slot first.  A sequence
    of at most ``budget`` slots keeps all.

    The kept rows are copied in order to the pages of ``new_table`` (B, MP')
    int32 in the same pools; those pages are distinct and none of them is read
    by this call.  The old pages are only read.  ``new_table`` has room for
    ``budget`` slots and, where it becomes the sequence's table, for what is
    appended before the next eviction: rows past its last slot are dropped.  A
    kept slot that ``block_table`` has no page for leaves its new slot's row as
    it was, so every slot in use has a page.  Returns ``(new_lengths (B,),
    new_weights (B, KH, MP'·PS), kept (B, KH, budget))``: the kept slots' weights
    (0 behind them) and their old slots, ascending (-1 behind them)."""
    name = "paged_evict"
    dev = _paged_device(name, k_cache, v_cache, block_table, lengths, new_table, weights)
    B, KH, E, cache = _paged_dims(name, k_cache, v_cache, block_table, lengths, True)
    PS = cache[1]
    _no_grad(name, k_cache, v_cache, weights)
    if new_table.dim() != 2 or new_table.shape[0] != B:
        raise NNopShapeError(-1, f"{name}: new_table must be (B, MP') with B = {B}")
    if new_table.dtype != torch.int32:
        raise NNopError(-2, f"{name}: new_table must be int32")
    if tuple(weights.shape) != (B, KH, cache[2] * PS):
        raise NNopShapeError(-1, f"{name}: weights must have shape (B, KH, MP·PS) = {(B, KH, cache[2] * PS)}")
    if weights.dtype != torch.float32:
        raise NNopError(-2, f"{name}: weights must be float32")
    budget, recent, slots = int(budget), int(recent), new_table.shape[1] * PS
    if not 0 <= recent <= budget <= slots:
        raise NNopShapeError(-1, f"{name}: 0 <= recent ({recent}) <= budget ({budget}) <= slots of new_table ({slots})")
    lengths, weights = lengths.contiguous(), weights.contiguous()
    block_table, new_table = block_table.contiguous(), new_table.contiguous()
    new_lengths = torch.empty_like(lengths)
    new_weights, kept = weights.new_empty((B, KH, slots)), lengths.new_empty((B, KH, budget))
    _on(dev, (k_cache, v_cache), lib.nnop_paged_evict, k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), new_table.data_ptr(),
        lengths.data_ptr(), weights.data_ptr(), new_lengths.data_ptr(), new_weights.data_ptr(), kept.data_ptr(), E, KH, B,
        *cache[:3], new_table.shape[1], *cache[3:], budget, recent, _dtype_id(k_cache))
    return new_lengths, new_weights, kept

"""Attention of sites to an encoder's states of another length, with a learned distance-bucket bias and dropout.

    O = dropout(softmax(scale Q K^T + table[h, bucket(i, j)])) V

next to geo_attention (stations against themselves with the fixed geo prior): queries and keys have their own lengths,
key heads may be shared by groups of query heads, keys may be absent (ragged lengths, missing stations), pairs may be
excluded (a distance cut-off), the bias per bucket is learned, and the keep mask of the dropout is recomputed in the
backward instead of stored. No [Nq, Nk] tensor per head ever reaches memory in the forward.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .counter_dropout import _dtype_code, _snapshot, _threshold

MAX_BUCKETS = 64


def _aligned(t):
    """bf16 operands and outputs go through TMA: head dim contiguous, base and other strides multiples of 16 bytes."""
    s0, s1, s2, s3 = t.stride()
    return s3 == 1 and not ((t.data_ptr() >> 1) | s0 | s1 | s2) & 7 and s0 > 0 and s1 > 0 and s2 > 0


def _padded(t):
    """Uninitialised [B, H, N, D] whose rows start on 16 bytes, heads and rows in t's order."""
    B, H, N, D = t.shape
    d8 = (D + 7) // 8 * 8
    if t.stride(1) < t.stride(2):  # heads side by side, as projections write them
        return torch.empty(B, N, H, d8, dtype=t.dtype, device=t.device).transpose(1, 2)[..., :D]
    return torch.empty(B, H, N, d8, dtype=t.dtype, device=t.device)[..., :D]


def _ready(t):
    """Operand layout of the kernels: bf16 as TMA reads it; fp32 with the head dim contiguous."""
    if t.dtype == torch.float32:
        return t if t.stride(3) == 1 else t.contiguous()
    return t if _aligned(t) else _padded(t).copy_(t)


def _like(t):
    """An output with t's layout where that keeps the head dim contiguous (split_heads views do), else contiguous; in
    bf16 with padded rows where the layout has none that start on 16 bytes (a head dim that is no multiple of 8)."""
    if t.dtype == torch.bfloat16 and t.shape[3] % 8:
        return _padded(t)
    return torch.empty_like(t) if t.stride(3) == 1 else torch.empty_like(t, memory_format=torch.contiguous_format)


def _arg(t):
    """(pointer, four strides) of an argument block."""
    s0, s1, s2, s3 = t.stride()  # of a head dim of size 1 any stride says the same
    return t.data_ptr(), s0, s1, s2, 1 if t.shape[3] == 1 else s3


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _shape(q, k, table):
    B, H, Nq, D = q.shape
    T, tdt = (0, _lib.DTYPE_FP32) if table is None else (table.shape[1], _dtype_code(table, "bias_table"))
    return B, H, k.shape[1], Nq, k.shape[2], D, _dtype_code(q, "q"), T, tdt


def _inputs(shape, q, k, v, table, ids, lens, mask, rng, thr, scale):
    return (*shape, *_arg(q), *_arg(k), *_arg(v), _ptr(ids), 0 if ids is None else ids.stride(0), _ptr(table),
            _ptr(lens), _ptr(mask), 0 if mask is None else mask.stride(0), _ptr(rng), thr, scale)


def _dense(o, q):
    """o without padded rows, in q's layout."""
    if o.dtype == torch.float32 or q.shape[3] % 8 == 0:
        return o
    return (torch.empty_like(q) if q.stride(3) == 1 else torch.empty(q.shape, dtype=q.dtype, device=q.device)).copy_(o)


def _forward(q, k, v, table, ids, lens, mask, rng, thr, scale, need_stats):
    """(o, row statistics) for operands in the kernels' layout (_ready)."""
    o = _like(q)
    if k.shape[2] == 0 or thr == 65536:  # no key, or no weight is kept
        return o.zero_(), None
    shape, dev = _shape(q, k, table), q.device
    ws = torch.empty(_lib.xattn_workspace("geoattn_xattn_fwd_workspace_bytes", *shape), dtype=torch.uint8, device=dev)
    stats = torch.empty(*q.shape[:3], 2, dtype=torch.float32, device=dev) if need_stats else None
    _lib.launch(dev, _lib.packed("geoattn_xattn_fwd"), _lib.XATTN_FWD.pack(
        *_inputs(shape, q, k, v, table, ids, lens, mask, rng, thr, scale), *_arg(o), _ptr(stats), ws.data_ptr()))
    return o, stats


def _backward(q, k, v, table, ids, lens, mask, rng, thr, scale, o, stats, do):
    dq, dk, dv = _like(q), _like(k), _like(v)
    dtable = torch.empty_like(table, memory_format=torch.contiguous_format) if table is not None else None
    if k.shape[2] == 0 or thr == 65536:
        return dq.zero_(), dk.zero_(), dv.zero_(), None if dtable is None else dtable.zero_()
    do = _ready(do)
    shape, dev = _shape(q, k, table), q.device
    ws = torch.empty(_lib.xattn_workspace("geoattn_xattn_bwd_workspace_bytes", *shape), dtype=torch.uint8, device=dev)
    _lib.launch(dev, _lib.packed("geoattn_xattn_bwd"), _lib.XATTN_BWD.pack(
        *_inputs(shape, q, k, v, table, ids, lens, mask, rng, thr, scale), *_arg(o), *_arg(do), stats.data_ptr(),
        *_arg(dq), *_arg(dk), *_arg(dv), _ptr(dtable), ws.data_ptr()))
    return dq, dk, dv, dtable


class CrossAttention(torch.autograd.Function):
    """O = dropout(softmax(scale Q K^T + table[h, ids])) V on libgeoattn (fwd + bwd)."""

    @staticmethod
    def forward(ctx, q, k, v, table, ids, lens, mask, rng, thr, scale):
        args = (_ready(q), _ready(k), _ready(v), table, ids, lens, mask, rng)
        o, stats = _forward(*args, thr, scale, True)
        ctx.save_for_backward(*args, o, stats)  # o as the kernels wrote it
        ctx.thr, ctx.scale = thr, scale
        return _dense(o, q)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        *args, o, stats = ctx.saved_tensors
        grads = _backward(*args, ctx.thr, ctx.scale, o, stats, do)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), *([None] * 6))


def cross_attention(q, k, v, *, buckets=None, bias_table=None, kv_lens=None, key_mask=None, dropout_p=0.0, rng=None,
                    scale=None):
    """Attention of q [B, H, Nq, D] to k, v [B, Hkv, Nk, D]; H is a multiple of Hkv (query head h reads key head
    h // (H // Hkv)), D <= 192, bf16 or fp32, any strides. Returns [B, H, Nq, D] in q's dtype and layout.

    buckets, bias_table: uint8 [Nq, Nk] bucket of each pair (StationGeometry.distance_buckets, or any ids) and the
        learned [H, T] or [1, T] bias, T <= 64, bf16 or fp32. Ids >= T (255 by convention) exclude their pair.
    kv_lens: int32 or int64 [B], keys of each batch entry (clamped to 0..Nk). key_mask: bool [B, Nk], True = present.
        What absent keys hold is not used (NaN included) and their gradients are zero.
    dropout_p, rng: dropout on the attention weights; rng as in `dropout`.
    scale: of the scores, positive, 1/sqrt(D) by default.
    At most 65535 batch entries and 65535 heads.
    A row with no key left gives zeros. Differentiable (once) in q, k, v and bias_table; the results do not depend on
    the order of any concurrent sums."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("q must be [B, H, Nq, D] and k, v [B, Hkv, Nk, D], got %s, %s, %s"
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1], k.shape[2]
    if (H % Hkv if Hkv else H):
        raise ValueError("query heads (%d) must be a multiple of key heads (%d)" % (H, Hkv))
    if D > 192:
        raise ValueError("head dim must be at most 192, got %d" % D)
    if q.dtype not in (torch.bfloat16, torch.float32) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k, v must all be bf16 or all be fp32")
    if (buckets is None) != (bias_table is None):
        raise ValueError("buckets and bias_table come together")
    if buckets is not None:
        if buckets.dtype != torch.uint8 or buckets.shape != (Nq, Nk):
            raise ValueError("buckets must be uint8 [%d, %d], got %s %s"
                             % (Nq, Nk, buckets.dtype, tuple(buckets.shape)))
        if bias_table.dim() != 2 or bias_table.shape[0] not in (1, H) or not 1 <= bias_table.shape[1] <= MAX_BUCKETS:
            raise ValueError("bias_table must be [%d or 1, 1..%d], got %s" % (H, MAX_BUCKETS, tuple(bias_table.shape)))
        _dtype_code(bias_table, "bias_table")
    if kv_lens is not None and (kv_lens.dtype not in (torch.int32, torch.int64) or kv_lens.shape != (B,)):
        raise ValueError("kv_lens must be int32 or int64 [%d]" % B)
    if key_mask is not None and (key_mask.dtype != torch.bool or key_mask.shape != (B, Nk)):
        raise ValueError("key_mask must be bool [%d, %d]" % (B, Nk))
    thr = _threshold(dropout_p)
    if thr and rng is None:
        raise ValueError("dropout_p > 0 needs rng")
    scale = (1.0 / math.sqrt(D) if D else 1.0) if scale is None else float(scale)
    if not 0.0 < scale < math.inf and D:
        raise ValueError("scale must be positive and finite, got %r" % (scale,))
    if not q.is_cuda:
        raise RuntimeError("cross attention runs on CUDA tensors only (no CPU path)")
    dev = q.device
    for name, t in (("k", k), ("v", v), ("buckets", buckets), ("bias_table", bias_table), ("kv_lens", kv_lens),
                    ("key_mask", key_mask)):
        if t is not None and t.device != dev:
            raise ValueError("%s lives on %s, q on %s" % (name, t.device, dev))
    key = _snapshot(rng, dev) if thr else None
    if q.numel() == 0:  # no batch, head, query or head dim: nothing to launch, and zero gradients
        o = q * 1.0
        for t in (k, v, bias_table):
            if t is not None and t.requires_grad and torch.is_grad_enabled():
                o = o + (t.flatten()[:0].sum() * 0.0).to(o.dtype)
        return o
    if bias_table is not None:
        if bias_table.shape[0] != H:
            bias_table = bias_table.expand(H, -1)
        bias_table = bias_table.contiguous()
        if buckets.stride(1) != 1 or buckets.stride(0) < Nk:
            buckets = buckets.contiguous()
    if kv_lens is not None:
        if kv_lens.dtype == torch.int64:
            kv_lens = kv_lens.clamp(0, Nk).to(torch.int32)  # clamped before it narrows
        kv_lens = kv_lens.contiguous()
    if key_mask is not None and (key_mask.stride(1) != 1 or key_mask.stride(0) < Nk):
        key_mask = key_mask.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (bias_table is not None and bias_table.requires_grad)):
        return CrossAttention.apply(q, k, v, bias_table, buckets, kv_lens, key_mask, key, thr, scale)
    o = _forward(_ready(q), _ready(k), _ready(v), bias_table, buckets, kv_lens, key_mask, key, thr, scale, False)[0]
    return _dense(o, q)

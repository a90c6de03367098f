"""Dropout from a counter-based generator: the keep mask is a function of (seed, offset, element) and is never stored.

An element is kept where its 16 bits of Philox4x32-7 are >= t = round(65536 p); kept values are scaled by
65536 / (65536 - t). The backward recomputes the same bits, so it needs only the (seed, offset) pair. ``CounterRNG``
keeps that pair on the device and moves the offset on in stream order, so a step captured as a CUDA graph draws fresh
masks at every replay (the reference's graph step: tests/test_gpu_graphs.py:34-46 there).
"""
from __future__ import annotations

import torch

from . import _lib


def _threshold(p) -> int:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability must be in [0, 1], got %r" % (p,))
    return int(p * 65536 + 0.5)


def _dtype_code(t, what):
    if t.dtype == torch.bfloat16:
        return _lib.DTYPE_BF16
    if t.dtype == torch.float32:
        return _lib.DTYPE_FP32
    raise TypeError("%s must be bf16 or fp32, got %s" % (what, t.dtype))


class CounterRNG:
    """(seed, offset) of the counter-based generator, int64[2] on one device; each `take` hands out the next offset."""

    def __init__(self, seed: int, device="cuda", offset: int = 0):
        def wrap(x):  # any integer, as the signed word with the same 64 bits
            x = int(x) & (2 ** 64 - 1)
            return x - 2 ** 64 if x >= 2 ** 63 else x
        self.state = torch.tensor([wrap(seed), wrap(offset)], dtype=torch.int64, device=device)

    def take(self) -> torch.Tensor:
        out = torch.empty_like(self.state)
        _lib.launch(self.state.device, _lib.lib().geoattn_rng_take, self.state.data_ptr(), out.data_ptr())
        return out


def _snapshot(rng, device):
    """The (seed, offset) tensor of one call: drawn from a CounterRNG, or given as int64[2]."""
    if isinstance(rng, CounterRNG):
        if rng.state.device != device:
            raise ValueError("rng lives on %s, the input on %s" % (rng.state.device, device))
        return rng.take()
    if not isinstance(rng, torch.Tensor) or rng.dtype != torch.int64 or rng.shape != (2,):
        raise TypeError("rng must be a CounterRNG or an int64 tensor (seed, offset)")
    if rng.device != device:
        raise ValueError("rng lives on %s, the input on %s" % (rng.device, device))
    return rng.contiguous()


def _run(x, residual, rng, thr):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        _lib.launch(x.device, _lib.lib().geoattn_dropout, _dtype_code(x, "x"), x.numel(), x.data_ptr(),
                    None if residual is None else residual.data_ptr(), y.data_ptr(), rng.data_ptr(), thr)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, thr):
        ctx.save_for_backward(rng)
        ctx.thr = thr
        return _run(x.contiguous(), None if residual is None else residual.contiguous(), rng, thr)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        dx = _run(dy.contiguous(), None, rng, ctx.thr) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def dropout(x, p, rng, residual=None):
    """Elements of x kept with probability 1 - p and scaled, 0 elsewhere (whatever x holds there), plus `residual`.

    x, residual: bf16 or fp32 CUDA tensors of one shape, dtype and device. rng: a CounterRNG, or an int64[2] tensor
    (seed, offset) on that device; the same pair gives the same mask. Differentiable in x and residual."""
    _dtype_code(x, "x")
    thr = _threshold(p)
    if not x.is_cuda:
        raise RuntimeError("dropout runs on CUDA tensors only (no CPU path)")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError("residual must have the shape and dtype of x")
        if residual.device != x.device:
            raise ValueError("residual lives on %s, x on %s" % (residual.device, x.device))
    if thr == 0:
        return x if residual is None else x + residual
    key = _snapshot(rng, x.device)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, key, thr)
    return _run(x.contiguous(), None if residual is None else residual.contiguous(), key, thr)

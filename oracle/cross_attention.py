"""Float64 oracle of cross attention with a bucketed bias, masks and counter-based dropout (torch on the CPU, numpy for
the generator). Gradients come from autograd on these plain operations.

TEST INFRASTRUCTURE.
"""
import math

import numpy as np
import torch

ROUNDS = 7


def philox(counter, key, rounds=ROUNDS):
    """Philox4x32 (Salmon et al., SC'11) on numpy uint64 arrays that hold 32-bit words; four words out."""
    m = np.uint64(0xFFFFFFFF)
    c = [np.asarray(x, dtype=np.uint64) & m for x in np.broadcast_arrays(*counter)]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c


def threshold(p):
    return int(p * 65536 + 0.5)


def _sixteen(words):
    w = np.stack(words, -1)
    return np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(*w.shape[:-1], 8)


def _u64(x):
    return int(x) & (2 ** 64 - 1)


def keep_attention(seed, offset, B, H, Nq, Nk, p):
    seed, offset = _u64(seed), _u64(offset)
    j8 = np.arange((Nk + 7) // 8).reshape(1, 1, -1)
    i, bh = np.arange(Nq).reshape(1, -1, 1), np.arange(B * H).reshape(-1, 1, 1)
    u = _sixteen(philox((j8, i, bh, offset % 2 ** 32), (seed % 2 ** 32, (seed >> 32) ^ (offset >> 32))))
    return torch.from_numpy((u >= threshold(p)).reshape(B, H, Nq, -1)[..., :Nk].copy())


def keep_flat(seed, offset, n, p):
    seed, offset = _u64(seed), _u64(offset)
    blk = np.arange((n + 7) // 8, dtype=np.uint64)
    u = _sixteen(philox((blk, blk >> np.uint64(32), offset % 2 ** 32, offset >> 32), (seed % 2 ** 32, seed >> 32)))
    return torch.from_numpy((u >= threshold(p)).reshape(-1)[:n].copy())


def scale_kept(p):
    t = threshold(p)
    return 0.0 if t == 65536 else 65536 / (65536 - t)


def weights(q, k, ids=None, table=None, lens=None, mask=None, scale=None, add=None):
    """softmax weights [B, H, Nq, Nk] in float64, 0 in rows with nothing left. ids: integer [Nq, Nk]. add: joins the
    scores."""
    B, H, Nq, D = q.shape
    Nk = k.shape[2]
    live = live_keys(B, Nk, lens, mask).view(B, 1, 1, Nk)
    kk = k.masked_fill(~live.view(B, 1, Nk, 1), 0.0).repeat_interleave(H // k.shape[1], dim=1)
    s = q @ kk.transpose(-1, -2) * (1 / math.sqrt(D) if scale is None else scale)
    if ids is not None:
        T = table.shape[1]
        live = live & (ids < T)
        s = s + table.expand(H, T)[:, ids.long().clamp(max=T - 1)]
    if add is not None:
        s = s + add
    s = s.masked_fill(~live, -math.inf)
    some = live.expand(B, H, Nq, Nk).any(-1, keepdim=True)
    return torch.softmax(torch.where(some, s, 0.0), -1) * some


def live_keys(B, Nk, lens=None, mask=None):
    live = torch.ones(B, Nk, dtype=torch.bool)
    if lens is not None:
        live = live & (torch.arange(Nk) < lens.view(B, 1))
    return live if mask is None else live & mask


def forward(q, k, v, ids=None, table=None, lens=None, mask=None, p=0.0, key=None, scale=None, add=None):
    """O in float64; autograd-capable in q, k, v (double) and table. What absent keys hold is not used."""
    B, H, Nq, _ = q.shape
    pr = weights(q, k, ids, table, lens, mask, scale, add)
    if p:
        pr = pr * keep_attention(*key, B, H, Nq, k.shape[2], p) * scale_kept(p)
    vv = v.masked_fill(~live_keys(B, k.shape[2], lens, mask).view(B, 1, -1, 1), 0.0)
    return pr @ vv.repeat_interleave(H // k.shape[1], dim=1)


def grads(q, k, v, do, table=None, **kw):
    """dict(o, dq, dk, dv[, dtable]) in float64 of CPU tensors of any dtype."""
    x = {n: t.double().requires_grad_(True) for n, t in (("q", q), ("k", k), ("v", v), ("table", table))
         if t is not None}
    o = forward(x["q"], x["k"], x["v"], table=x.get("table"), **kw)
    got = torch.autograd.grad(o, list(x.values()), do.double())
    return {"o": o.detach(), **{"d" + n: g for n, g in zip(x, got)}}


def table_mass(q, k, v, do, table, ids, **kw):
    """[H, T] sum of |dS| over each bucket's pairs: what a bucket's gradient would be if its terms did not cancel."""
    B, H, Nq, _ = q.shape
    add = torch.zeros(B, H, Nq, k.shape[2], dtype=torch.float64, requires_grad=True)
    o = forward(q.double(), k.double(), v.double(), ids=ids, table=table.double(), add=add, **kw)
    (ds,) = torch.autograd.grad(o, add, do.double())
    T = table.shape[1]
    out = torch.zeros(H, max(T, int(ids.max()) + 1), dtype=torch.float64)
    out.index_add_(1, ids.reshape(-1).long(), ds.abs().sum(0).reshape(H, -1))
    return out[:, :T]

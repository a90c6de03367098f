"""Cases of the cross-station attention operators: what each computes, in plain torch operations and through the package.

Three operators, measured alone and as they are used together:
  attention   O = dropout(softmax(scale Q K^T + table[h, bucket(i, j)])) V for queries and keys of different lengths
              (station embeddings against an encoder's states), with key lengths, key masks and shared key heads;
  bias        the learned bias table[h, bucket] inside it, with its gradient (buckets of the distance between stations);
  dropout     keep masks from a counter-based generator (Philox4x32 with 7 rounds), recomputed and never stored, on the
              attention weights and on hidden states with the residual they join.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls the package; False: plain torch operations

BF16, FP32 = "bf16", "fp32"
NO_PAIR = 255          # bucket id of a pair that does not attend
ELEMS_MAX = 1 << 30    # attention weights of the largest case (B * H * Nq * Nk)
FLOPS_MAX = 1.65e12    # products of the largest case


def attention(name, B, H, Hkv, Nq, Nk, D, dtype, train, lens=False, mask=False, buckets=0, cut=False, p=0.0):
    return {"name": name, "op": "attention", "B": B, "H": H, "Hkv": Hkv, "Nq": Nq, "Nk": Nk, "D": D, "dtype": dtype,
            "train": train, "lens": lens, "mask": mask, "buckets": buckets, "cut": cut, "p": p}


def hidden(name, rows, cols, dtype, train, residual, p):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "train": train,
            "residual": residual, "p": p}


def listed():
    return [
        # one new site asks one encoded issue date: a single query token, where latency counts
        attention("site_one_date", 1, 16, 16, 1, 512, 128, BF16, False),
        # a few sites against long encoded histories of different lengths, shared key heads (one history is empty)
        attention("sites_long_history", 16, 32, 8, 4, 16384, 128, BF16, False, lens=True),
        # gridded targets against the station network, some stations missing, bias by distance
        attention("targets_infer", 32, 16, 16, 700, 512, 64, BF16, False, mask=True, buckets=32),
        # a decoder layer in training over ragged encoder states
        attention("cross_train", 32, 8, 8, 384, 512, 64, BF16, True, lens=True, p=0.1),
        # the benchmark's batch (256 issue dates x 16 heads x 512 stations x 128), bias by distance, training
        attention("bias_train", 256, 16, 16, 512, 512, 128, BF16, True, buckets=32),
        # production head dim, pairs beyond the cut-off distance excluded, missing stations, dropout
        attention("bias_dropout_train", 32, 16, 16, 512, 512, 192, BF16, True, mask=True, buckets=48, cut=True, p=0.1),
        # long sequences on both sides, shared key heads
        attention("long_train", 1, 8, 2, 4096, 8192, 128, BF16, True, p=0.1),
        # fp32: odd sizes, missing stations; and the fp32 training configuration with the bias
        attention("odd_infer_fp32", 8, 8, 8, 130, 517, 48, FP32, False, mask=True, buckets=20),
        attention("bias_train_fp32", 32, 8, 8, 512, 512, 64, FP32, True, buckets=32),
        # hidden states of one issue date, of a ragged fp32 batch in training, and of the benchmark's batch
        hidden("hidden_one_date", 512, 1024, BF16, False, True, 0.1),
        hidden("hidden_train_fp32", 18907, 1000, FP32, True, True, 0.25),
        hidden("hidden_train", 131072, 2048, BF16, True, True, 0.1),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = BF16 if rng.random() < 0.75 else FP32
    if rng.random() < 0.25:
        while True:
            rows, cols = _log(rng, 1, 131072), _log(rng, 1, 4096)
            if rows * cols <= 131072 * 2048:
                break
        return {"op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "train": rng.random() < 0.6,
                "residual": rng.random() < 0.7, "p": round(rng.uniform(0.02, 0.6), 3)}
    while True:
        heads = rng.choice([1, 2, 3, 4, 5, 8])
        group = rng.choice([1, 1, 1, 2, 3, 4, 8])
        train = rng.random() < 0.6
        case = {"op": "attention", "B": _log(rng, 1, 256), "H": heads * group, "Hkv": heads,
                # a training row has several keys: with one, its score gradients are 0 and only rounding is left
                "Nq": _log(rng, 1, 4096), "Nk": _log(rng, 8 if train else 1, 16384),
                "D": rng.choice([32, 48, 64, 64, 96, 128, 128, 192, rng.randint(8, 192)]), "dtype": dtype,
                "train": train, "lens": rng.random() < 0.4, "mask": rng.random() < 0.4,
                "buckets": rng.choice([0, rng.randint(8, 64)]), "cut": rng.random() < 0.3,
                "p": rng.choice([0.0, round(rng.uniform(0.02, 0.5), 3)])}
        case["cut"] = case["cut"] and case["buckets"] > 0
        n = case["B"] * case["H"] * case["Nq"] * case["Nk"]
        if n <= ELEMS_MAX // (1 if case["p"] == 0 else 4) and 12.0 * n * case["D"] <= FLOPS_MAX:
            return case


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == BF16 else torch.float32


def _lens(case):
    """Key lengths from empty to full, half of them above three quarters: the same set for every seed."""
    B, Nk = case["B"], case["Nk"]
    share = [0.0 if (b == 0 and B > 1) else 1.0 - 0.5 * (b % 7) / 6.0 for b in range(B)]
    return [int(round(Nk * s)) if s == 0.0 else max(1, int(round(Nk * s))) for s in share]


def _key_len_sum(case):
    return sum(_lens(case)) if case["lens"] else case["B"] * case["Nk"]


def prepare(case, seed):
    dt = _dtype(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    key = torch.tensor([seed * 7919 + 12345, (seed % 1000) + 3], dtype=torch.int64, device="cuda")

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        return {"case": case, "x": normal(*shape), "res": normal(*shape) if case["residual"] else None,
                "dy": normal(*shape) if case["train"] else None, "key": key}
    B, H, Hkv, Nq, Nk, D = (case[n] for n in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    # heads side by side in a row, as a projection writes them, and split as views
    st = {"case": case, "key": key, "q": normal(B, Nq, H, D).transpose(1, 2),
          "k": normal(B, Nk, Hkv, D).transpose(1, 2), "v": normal(B, Nk, Hkv, D).transpose(1, 2),
          "do": normal(B, Nq, H, D).transpose(1, 2) if case["train"] else None,
          "lens": None, "mask": None, "ids": None, "table": None}
    if case["lens"]:
        order = torch.randperm(B, generator=g, device="cuda")
        st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[order]
    if case["mask"]:
        st["mask"] = torch.rand(B, Nk, generator=g, device="cuda") > 0.15
    if case["buckets"]:
        T = case["buckets"]
        lat = torch.rand(Nq + Nk, generator=g, device="cuda", dtype=torch.float64) * 14 + 35
        lon = torch.rand(Nq + Nk, generator=g, device="cuda", dtype=torch.float64) * 20 - 124
        a, o = torch.deg2rad(lat), torch.deg2rad(lon)
        x = torch.stack([a.cos() * o.cos(), a.cos() * o.sin(), a.sin()], 1)
        km = 6371 * torch.acos((x[:Nq] @ x[Nq:].T).clamp(-1, 1))
        edges = torch.logspace(math.log10(60.0), math.log10(1500.0), T - 1, device="cuda", dtype=torch.float64)
        ids = torch.bucketize(km, edges, right=True)
        if case["cut"]:
            ids = torch.where(km > 900.0, NO_PAIR, ids)
        st["ids"] = ids.to(torch.uint8)
        st["table"] = (torch.randn(H, T, generator=g, device="cuda") * 0.7).to(dt)
    return st


# --- the generator, and the operators in plain operations ---------------------------------------------------------
def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32 (Salmon et al. 2011) with 7 rounds on int64 tensors that hold 32-bit words."""
    M = 0xFFFFFFFF
    a0, a1, w0, w1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85

    def one(c0, c1, c2, c3, k0, k1):
        # a product of two 32-bit words may pass 2^63: its low half is right all the same, its high half is masked
        p0, p1 = c0 * a0, c2 * a1
        return ((p1 >> 32) & M) ^ c1 ^ k0, p1 & M, ((p0 >> 32) & M) ^ c3 ^ k1, p0 & M

    keys = [((k0 + r * w0) & M, (k1 + r * w1) & M) for r in range(7)]
    c = (c0, c1, c2, c3)
    c = one(*c, *keys[0])
    c = one(*c, *keys[1])
    c = one(*c, *keys[2])
    c = one(*c, *keys[3])
    c = one(*c, *keys[4])
    c = one(*c, *keys[5])
    return one(*c, *keys[6])


def _keep(words, thr):
    """[..., 8] truth values from four words: 16 bits each, the low half first."""
    u = torch.stack([words[0] & 0xFFFF, words[0] >> 16, words[1] & 0xFFFF, words[1] >> 16,
                     words[2] & 0xFFFF, words[2] >> 16, words[3] & 0xFFFF, words[3] >> 16], -1)
    return u >= thr


def _threshold(p):
    return int(p * 65536 + 0.5)


def _keep_pairs(key, B, H, Nq, Nk, thr):
    M = 0xFFFFFFFF
    dev = key.device
    j8 = torch.arange((Nk + 7) // 8, device=dev, dtype=torch.int64).view(1, 1, -1)
    i = torch.arange(Nq, device=dev, dtype=torch.int64).view(1, -1, 1)
    bh = torch.arange(B * H, device=dev, dtype=torch.int64).view(-1, 1, 1)
    seed, off = key[0], key[1]
    w = _philox(j8, i, bh, off & M, seed & M, ((seed >> 32) & M) ^ ((off >> 32) & M))
    return _keep(torch.broadcast_tensors(*w), thr).reshape(B, H, Nq, -1)[..., :Nk]


def _keep_flat(key, n, thr):
    M = 0xFFFFFFFF
    blk = torch.arange((n + 7) // 8, device=key.device, dtype=torch.int64)
    seed, off = key[0], key[1]
    w = _philox(blk & M, blk >> 32, off & M, (off >> 32) & M, seed & M, (seed >> 32) & M)
    return _keep(torch.broadcast_tensors(*w), thr).reshape(-1)[:n]


def _plain_dropout(st):
    case, x = st["case"], st["x"]
    thr = _threshold(case["p"])
    scale = 65536.0 / (65536 - thr)
    keep = _keep_flat(st["key"], x.numel(), thr).view(x.shape)
    y = torch.where(keep, x.float() * scale, 0.0)
    if st["res"] is not None:
        y = y + st["res"].float()
    out = {"y": y.to(x.dtype)}
    if case["train"]:
        out["dx"] = torch.where(keep, st["dy"].float() * scale, 0.0).to(x.dtype)
    return out


def _allowed(st, B, Nq, Nk):
    """[B, 1, Nq or 1, Nk] truth values, or None where every pair attends."""
    ok = None
    if st["lens"] is not None:
        ok = (torch.arange(Nk, device="cuda") < st["lens"].view(-1, 1)).view(B, 1, 1, Nk)
    if st["mask"] is not None:
        m = st["mask"].view(B, 1, 1, Nk)
        ok = m if ok is None else ok & m
    if st["case"]["cut"]:
        m = (st["ids"] != NO_PAIR).view(1, 1, Nq, Nk)
        ok = m if ok is None else ok & m
    return ok


def _plain_attention(st):
    case, dt = st["case"], st["q"].dtype
    B, H, Hkv, Nq, Nk, D = (case[n] for n in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    G, T, scale = H // Hkv, case["buckets"], 1.0 / math.sqrt(D)
    q = st["q"].float().reshape(B, Hkv, G * Nq, D)  # the heads that share a key head, one below the other
    k, v = st["k"].float(), st["v"].float()
    s = (q @ k.transpose(-1, -2)).view(B, H, Nq, Nk) * scale
    if T:
        flat = st["ids"].long().clamp(max=T - 1).view(-1)
        s = s + st["table"].float()[:, flat].view(1, H, Nq, Nk)
    ok = _allowed(st, B, Nq, Nk)
    if ok is not None:
        s = s.masked_fill(~ok, -math.inf)
    top = s.amax(-1, keepdim=True)
    pr = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = pr.sum(-1, keepdim=True)
    pr = pr / torch.where(total == 0, 1.0, total)
    del s
    keep, inv = None, 1.0
    a = pr
    if case["p"] > 0:
        thr = _threshold(case["p"])
        inv = 65536.0 / (65536 - thr)
        keep = _keep_pairs(st["key"], B, H, Nq, Nk, thr)
        a = torch.where(keep, pr * inv, 0.0)
    o = (a.view(B, Hkv, G * Nq, Nk) @ v).view(B, H, Nq, D)
    out = {"o": o.to(dt)}
    if not case["train"]:
        return out
    do = st["do"].float().reshape(B, Hkv, G * Nq, D)
    out["dv"] = (a.view(B, Hkv, G * Nq, Nk).transpose(-1, -2) @ do).to(dt)
    del a
    da = (do @ v.transpose(-1, -2)).view(B, H, Nq, Nk)
    if keep is not None:
        da = torch.where(keep, da * inv, 0.0)
    ds = pr * (da - (pr * da).sum(-1, keepdim=True))
    del da, pr
    if T:
        per_pair = ds.sum(0).view(H, Nq * Nk)
        at = st["ids"].long().view(1, -1).expand(H, -1)
        grad = torch.zeros(H, 256, device="cuda", dtype=torch.float64).scatter_add_(1, at, per_pair.double())
        out["dtable"] = grad[:, :T].to(dt)
    ds = ds.view(B, Hkv, G * Nq, Nk)
    out["dq"] = ((ds @ k) * scale).view(B, H, Nq, D).to(dt)
    out["dk"] = ((ds.transpose(-1, -2) @ q) * scale).to(dt)
    return out


# --- the framework's calls ----------------------------------------------------------------------------------------
def _own_dropout(st):
    from foreswe_gpu_optimization_b200 import dropout
    case = st["case"]
    if not case["train"]:
        return {"y": dropout(st["x"], case["p"], st["key"], residual=st["res"])}
    x = st["x"].detach().requires_grad_(True)
    y = dropout(x, case["p"], st["key"], residual=st["res"])
    (dx,) = torch.autograd.grad(y, (x,), st["dy"])
    return {"y": y.detach(), "dx": dx}


def _own_attention(st):
    from foreswe_gpu_optimization_b200 import cross_attention
    case = st["case"]
    kw = dict(buckets=st["ids"], kv_lens=st["lens"], key_mask=st["mask"], dropout_p=case["p"],
              rng=st["key"] if case["p"] > 0 else None)
    if not case["train"]:
        return {"o": cross_attention(st["q"], st["k"], st["v"], bias_table=st["table"], **kw)}
    names = ["q", "k", "v"] + (["table"] if case["buckets"] else [])
    x = {n: st[n].detach().requires_grad_(True) for n in names}
    o = cross_attention(x["q"], x["k"], x["v"], bias_table=x.get("table"), **kw)
    grads = torch.autograd.grad(o, [x[n] for n in names], st["do"])
    return {"o": o.detach(), **{"d" + n: d for n, d in zip(names, grads)}}


def run(state):
    if state["case"]["op"] == "dropout":
        return _own_dropout(state) if own else _plain_dropout(state)
    return _own_attention(state) if own else _plain_attention(state)


def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        arrays = 2 + int(case["residual"]) + (2 if case["train"] else 0)  # x, y, the residual; dy, dx
        return {"bytes": arrays * n * size, "flops": n * (2 if case["train"] else 1)}
    B, H, Hkv, Nq, Nk, D = (case[n] for n in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    keys = _key_len_sum(case)
    qo, kv = B * H * Nq * D, keys * Hkv * D
    small = (Nq * Nk + H * case["buckets"] * size if case["buckets"] else 0) + (B * Nk if case["mask"] else 0)
    pairs = keys * H * Nq
    if not case["train"]:
        return {"bytes": (2 * qo + 2 * kv) * size + small, "flops": 4 * pairs * D}
    # forward and backward read q, k, v and write o; the backward reads do and writes dq, dk, dv (of every key)
    return {"bytes": (4 * qo + 2 * kv + 2 * B * Nk * Hkv * D) * size + small, "flops": 12 * pairs * D}


# --- the definition in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    thr = math.floor(case["p"] * 65536 + 0.5)
    seed64, off64 = (int(x) & (2 ** 64 - 1) for x in st["key"].tolist())
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)

    def bits(c0, c1, c2, c3, k0, k1):
        """Eight 16-bit numbers for each counter (last axis): Philox4x32, 7 rounds, on numpy's unsigned words."""
        x = [np.asarray(c, dtype=np.uint64) for c in np.broadcast_arrays(c0, c1, c2, c3)]
        for r in range(7):
            kk0 = np.uint64((k0 + r * 0x9E3779B9) % 2 ** 32)
            kk1 = np.uint64((k1 + r * 0xBB67AE85) % 2 ** 32)
            m0, m1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
            x = [(m1 >> half) ^ x[1] ^ kk0, m1 & low, (m0 >> half) ^ x[3] ^ kk1, m0 & low]
        return np.stack(x, -1).astype("<u4").view("<u2")

    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        keep = np.empty((n + 7) // 8 * 8, dtype=bool)
        for at in range(0, len(keep) // 8, 1 << 18):
            blk = np.arange(at, min(at + (1 << 18), len(keep) // 8), dtype=np.uint64)
            keep[at * 8:(at + len(blk)) * 8] = bits(blk & low, blk >> half, off64 % 2 ** 32, off64 >> 32,
                                                    seed64 % 2 ** 32, seed64 >> 32).reshape(-1) >= thr
        factor = torch.from_numpy(keep[:n]).cuda().view(case["rows"], case["cols"]).double() / (1 - thr / 65536)
        y = st["x"].double() * factor
        y = y if st["res"] is None else y + st["res"].double()
        return {"y": y, "dx": st["dy"].double() * factor} if case["train"] else {"y": y}

    B, H, Hkv, Nq, Nk, D = (case[n] for n in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    if thr and B * H * Nq * Nk > 3e8:
        return None
    T, G = case["buckets"], H // Hkv
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"o": zeros(B, H, Nq, D)}
    if case["train"]:
        out.update(dq=zeros(B, H, Nq, D), dk=zeros(B, Hkv, Nk, D), dv=zeros(B, Hkv, Nk, D))
    hist = zeros(H, max(T, 1))
    member = None
    if T:
        ids = st["ids"].long()
    lens = st["lens"].tolist() if st["lens"] is not None else [Nk] * B
    for b in range(B):
        on = torch.zeros(Nk, dtype=torch.bool, device="cuda")
        on[:lens[b]] = True
        if st["mask"] is not None:
            on &= st["mask"][b]
        for h in range(H):
            kv = h // G
            logits = torch.einsum("id,jd->ij", st["q"][b, h].double(), st["k"][b, kv].double()) / D ** 0.5
            live = on.expand(Nq, Nk)
            if T:
                live = live & (ids < T)
                logits = logits + st["table"][h].double()[ids.clamp(max=T - 1)]
            logits = logits.masked_fill(~live, float("-inf"))
            w = torch.softmax(logits, -1).nan_to_num(0.0)
            f = torch.ones((), dtype=torch.float64, device="cuda")
            if thr:
                u = bits(np.arange((Nk + 7) // 8).reshape(1, -1), np.arange(Nq).reshape(-1, 1), b * H + h,
                         off64 % 2 ** 32, seed64 % 2 ** 32, (seed64 >> 32) ^ (off64 >> 32))
                f = torch.from_numpy(u.reshape(Nq, -1)[:, :Nk] >= thr).cuda().double() / (1 - thr / 65536)
            out["o"][b, h] = (w * f) @ st["v"][b, kv].double()
            if not case["train"]:
                continue
            d_o = st["do"][b, h].double()
            out["dv"][b, kv] += (w * f).T @ d_o
            dw = (d_o @ st["v"][b, kv].double().T) * f
            dl = w * (dw - (w * dw).sum(-1, keepdim=True))
            out["dq"][b, h] = dl @ st["k"][b, kv].double() / D ** 0.5
            out["dk"][b, kv] += dl.T @ st["q"][b, h].double() / D ** 0.5
            if T:
                member = ids.clamp(max=T).reshape(-1) if member is None else member
                hist[h] += torch.bincount(member, weights=dl.reshape(-1), minlength=T + 1)[:T]
    if case["train"] and T:
        out["dtable"] = hist
    return out

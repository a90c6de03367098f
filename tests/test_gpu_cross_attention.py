"""Cross attention, its bucketed bias and dropout on the GPU against float64.

Tolerances (rel-L2 over an output). bf16: one rounding is off by at most 2^-8 relative. o and dv pass two (the weights,
the result): 2 * 2^-8; dq, dk and dtable three (o inside delta, dS, the result): 3 * 2^-8. fp32: a weight is 2^t with
|t| <= 32 formed from sums of up to 192 products, an absolute error of t below 32 * 4 * 2^-24, and so a relative error
below 8e-6 of the weight with the exponential's 2^-22; the sums over keys add less: 2e-5.
"""
import math

import numpy as np
import pytest
import torch

from helpers import rel_l2, stations
from oracle import cross_attention as ox

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32
TOL = {BF: {"o": 2, "dv": 2, "dq": 3, "dk": 3, "dtable": 3}, FP: {}}


def tol(dtype, name):
    return TOL[BF][name] * 2.0 ** -8 if dtype == BF else 2e-5


def make(B, H, Hkv, Nq, Nk, D, dtype, seed=0, T=0, lens=None, mask=False, cut=False, table_heads=None):
    """CPU tensors: q, k, v as split projections ([B, N, heads * D] memory), dO, and the optional inputs."""
    g = torch.Generator().manual_seed(seed)
    x = {"q": torch.randn(B, Nq, H, D, generator=g), "k": torch.randn(B, Nk, Hkv, D, generator=g),
         "v": torch.randn(B, Nk, Hkv, D, generator=g), "do": torch.randn(B, Nq, H, D, generator=g)}
    x = {n: t.to(dtype).transpose(1, 2) for n, t in x.items()}
    kw = {}
    if T:
        ids = torch.randint(0, T, (Nq, Nk), generator=g)
        if cut:
            ids[torch.rand(Nq, Nk, generator=g) < 0.3] = 255
        kw["ids"] = ids.to(torch.uint8)
        x["table"] = torch.randn(table_heads or H, T, generator=g).to(dtype)
    if lens is not None:
        kw["lens"] = torch.tensor(lens, dtype=torch.int32)
    if mask:
        kw["mask"] = torch.rand(B, Nk, generator=g) > 0.3
    return x, kw


def run(x, kw, p=0.0, key=None, scale=None, device="cuda"):
    """The package's forward and backward; dict like the oracle's, on the CPU."""
    import foreswe_gpu_optimization_b200 as g
    y = {n: t.to(device).detach().requires_grad_(n != "do") for n, t in x.items()}
    opt = {n: t.to(device) for n, t in kw.items()}
    rng = None if key is None else torch.tensor(key, dtype=torch.int64, device=device)
    o = g.cross_attention(y["q"], y["k"], y["v"], buckets=opt.get("ids"), bias_table=y.get("table"),
                          kv_lens=opt.get("lens"), key_mask=opt.get("mask"), dropout_p=p, rng=rng, scale=scale)
    leaves = [n for n in ("q", "k", "v", "table") if n in y]
    got = torch.autograd.grad(o, [y[n] for n in leaves], y["do"])
    with torch.no_grad():
        same = g.cross_attention(y["q"], y["k"], y["v"], buckets=opt.get("ids"), bias_table=y.get("table"),
                                 kv_lens=opt.get("lens"), key_mask=opt.get("mask"), dropout_p=p, rng=rng, scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(o.detach().isnan(), same.isnan()) and torch.equal(o.detach().nan_to_num(), same.nan_to_num())
    assert o.dtype == x["q"].dtype and o.shape == x["q"].shape
    return {"o": o.detach().cpu(), **{"d" + n: t.cpu() for n, t in zip(leaves, got)}}


def delta_slack(x, kw, ref):
    """What the rounding of o leaves in the score gradients: delta_i = dO_i.o_i is off by up to e_i = 2^-8 sum |dO_id
    o_id|, so dS_ij by P_ij e_i, dq_i by scale e_i |sum_j P_ij k_j|, dk_j by scale sum_i P_ij e_i |q_i| and dtable by the
    sum of P_ij e_i over a bucket's pairs. Next to the other terms only where rows with few keys, whose dS nearly
    cancels, stand beside rows with many."""
    q, k = x["q"].double(), x["k"].double()
    B, H, Nq, D = q.shape
    G = H // k.shape[1]
    pr = ox.weights(q, k, table=x["table"].double() if "table" in x else None, **kw)
    e = 2.0 ** -8 * (x["do"].double() * ref["o"]).abs().sum(-1, keepdim=True)
    kk = k.masked_fill(~ox.live_keys(B, k.shape[2], kw.get("lens"), kw.get("mask")).view(B, 1, -1, 1), 0.0)
    out = {"dq": (e * (pr @ kk.repeat_interleave(G, dim=1)).norm(dim=-1, keepdim=True)).norm() / math.sqrt(D)}
    pe = pr * e
    out["dk"] = ((pe.transpose(-1, -2) @ q.norm(dim=-1, keepdim=True)).view(B, k.shape[1], G, -1).sum(2)).norm() / math.sqrt(D)
    if "table" in x:
        T = x["table"].shape[1]
        per = torch.zeros(H, 256, dtype=torch.float64).index_add_(1, kw["ids"].reshape(-1), pe.sum(0).reshape(H, -1))
        out["dtable"] = (per.sum(0) if x["table"].shape[0] == 1 else per)[..., :T].norm()
    return {n: t.item() for n, t in out.items()}


def check(x, kw, p=0.0, key=None, scale=None):
    got = run(x, kw, p, key, scale)
    kw = {n: t.long() if n == "ids" else t for n, t in kw.items()}
    ref = ox.grads(x["q"], x["k"], x["v"], x["do"], table=x.get("table"), p=p, key=key, scale=scale, **kw)
    slack = delta_slack(x, kw, ref) if x["q"].dtype == BF and scale is None else {}
    for name, r in ref.items():
        e = rel_l2(got[name], r)
        if r.norm() > 0:
            e -= slack.get(name, 0.0) / r.norm().item()
        if x["k"].shape[2] == 1 and name in ("dq", "dk", "dtable"):
            # one key: P = 1 and dS = dA - delta is exactly 0; both sums of D products are judged against dO
            e = (got[name].double() - r).norm().item() / x["do"].double().norm().item()
        assert torch.isfinite(got[name].float()).all(), name
        assert e <= tol(x["q"].dtype, name), (name, e)
    return got, ref


SHAPES = [  # B, H, Hkv, Nq, Nk, D
    (1, 1, 1, 1, 1, 8), (1, 2, 1, 1, 7, 16), (2, 2, 2, 5, 1, 64), (1, 3, 3, 33, 65, 48), (2, 4, 2, 128, 128, 64),
    (1, 2, 2, 129, 127, 128), (1, 2, 1, 257, 300, 128), (1, 2, 2, 130, 191, 192), (3, 6, 2, 17, 200, 96),
    (1, 1, 1, 64, 1000, 33), (2, 8, 1, 3, 640, 128), (1, 2, 2, 300, 77, 1),
]


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_plain(shape, dtype):
    check(*make(*shape, dtype, seed=1))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES[2:10], ids=lambda s: "x".join(map(str, s)))
def test_bias_masks_dropout_together(shape, dtype):
    B, H, Hkv, Nq, Nk, D = shape
    lens = [max(1, Nk - 13 * b) for b in range(B)]
    x, kw = make(*shape, dtype, seed=2, T=5, lens=lens, mask=Nk > 1, cut=Nk > 1)
    check(x, kw, p=0.25, key=[123456789012345, 2 ** 33 + 5])


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 31, 64])
@pytest.mark.parametrize("heads", [1, 4], ids=["shared", "per_head"])
def test_bias_gradient(T, heads, dtype):
    x, kw = make(3, 4, 2, 140, 150, 64, dtype, seed=T, T=T, table_heads=heads)
    if T > 1:
        check(x, kw)
        return
    # one bucket: its pairs' gradients sum to 0 in each row, so what is left is judged against their absolute values
    got = run(x, kw)
    mass = ox.table_mass(x["q"], x["k"], x["v"], x["do"], x["table"], kw["ids"])
    mass = mass.sum(0, keepdim=True) if heads == 1 else mass
    assert (got["dtable"].double().abs() <= tol(dtype, "dtable") * mass).all()


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 192])
def test_dropout_rates(D, dtype):
    for p in (0.02, 0.5, 0.97):
        check(*make(2, 2, 2, 100, 260, D, dtype, seed=4), p=p, key=[-3, 9])
    x, kw = make(1, 2, 2, 40, 90, D, dtype, seed=4)
    for name, t in run(x, kw, p=1.0, key=[1, 1]).items():             # nothing is kept
        assert (t == 0).all(), name


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(2, 3, 3, 140, 300, 64), (2, 4, 2, 1, 1500, 128), (2, 2, 1, 70, 130, 192)],
                         ids=lambda s: "x".join(map(str, s)))
def test_rows_with_nothing_left_and_garbage_in_absent_keys(shape, dtype):
    """An empty batch entry, excluded rows, and NaN or infinities in absent keys: zeros there, and the rest as if the
    absent keys were not there."""
    B, H, Hkv, Nq, Nk, D = shape
    x, kw = make(*shape, dtype, seed=6, T=3, lens=[0, Nk - 70], mask=True)
    kw["ids"][Nq // 2] = 255
    gone = torch.arange(Nk) >= kw["lens"].view(-1, 1)
    gone = (gone | ~kw["mask"]).view(B, 1, Nk, 1).expand(B, Hkv, Nk, D)
    for n, bad in (("k", math.nan), ("v", math.inf)):
        x[n] = x[n].masked_fill(gone, bad)
    got, ref = check(x, kw)
    assert (got["o"][0] == 0).all() and (got["dq"][0] == 0).all()
    assert (got["o"][:, :, Nq // 2] == 0).all() and (got["dq"][:, :, Nq // 2] == 0).all()
    for n in ("dk", "dv"):
        assert (got[n][gone] == 0).all(), n


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_infinite_bias_and_extreme_scores(dtype):
    """A bucket at -inf excludes its pairs (and takes no gradient from them); the type's lowest value does the same in
    rows that keep other pairs; scores far apart saturate without overflow."""
    for bad in (-math.inf, torch.finfo(dtype).min):
        x, kw = make(1, 2, 2, 65, 70, 64, dtype, seed=8, T=4)
        x["table"][:, 2] = bad
        kw["ids"][:, 0] = 1
        got, ref = check(x, kw)
        assert (got["dtable"][:, 2] == 0).all()
    x, kw = make(1, 2, 2, 65, 70, 64, dtype, seed=9, T=3)
    x["table"][:, 1] = torch.finfo(dtype).min
    kw["ids"][5] = 1                                                  # a row at the lowest value: all keys alike
    kw["ids"][6] = 255                                                # not the same as a row with nothing left
    got, ref = check(x, kw)
    mean = x["v"].double().mean(2)
    assert rel_l2(got["o"][:, :, 5], mean) <= tol(dtype, "o") and (got["o"][:, :, 6] == 0).all()
    x, kw = make(1, 2, 2, 65, 70, 64, dtype, seed=9)
    x["q"] = x["q"] * 64
    got = run(x, kw)
    assert all(torch.isfinite(t.float()).all() for t in got.values())
    ref = ox.forward(x["q"].double(), x["k"].double(), x["v"].double())
    # scores up to ~1000: fp32 holds them to 1000 * 2^-22, bf16 inputs' products are exact
    assert rel_l2(got["o"], ref) <= (2 * 2 ** -8 if dtype == BF else 1e-3)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_layouts(dtype):
    """Contiguous, sliced, offset, transposed and broadcast operands give the values of their contiguous copies, and
    gradients arrive in the leaves' own shapes."""
    import foreswe_gpu_optimization_b200 as g
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    B, H, Nq, Nk, D = 2, 4, 70, 90, 40
    base = r(B, Nq, H * D + 3)
    cases = {
        "sliced rows": (base[:, :, 3:].reshape(B, Nq, H, D).transpose(1, 2), r(B, H, 2 * Nk, D)[:, :, ::2],
                        r(B, H, Nk, 2 * D)[..., D:]),
        "head dim outermost": (r(D, B, H, Nq).permute(1, 2, 3, 0), r(D, B, H, Nk).permute(1, 2, 3, 0),
                               r(B, Nk, D, H).permute(0, 3, 1, 2)),
        "broadcast": (r(1, H, Nq, D).expand(B, H, Nq, D), r(B, 1, Nk, D).expand(B, H, Nk, D),
                      r(1, 1, Nk, D).expand(B, H, Nk, D)),
        "offset": (r(B * H * Nq * D + 1)[1:].view(B, H, Nq, D), r(B * H * Nk * D + 1)[1:].view(B, H, Nk, D),
                   r(B, H, Nk, D)),
    }
    wide = torch.randint(0, 3, (Nq + 1, 2 * Nk + 5), generator=gen, device="cuda").to(torch.uint8)
    mask = (torch.rand(Nk, B, generator=gen, device="cuda") > 0.3).t()
    table = r(H, 3)
    for name, ops in cases.items():
        for ids in (wide[1:, 5:5 + Nk], wide[:Nq, :2 * Nk:2], wide[:1, :Nk].expand(Nq, Nk)):
            outs = []
            for copy in (False, True):
                x = [(t.contiguous() if copy else t).detach().requires_grad_(True) for t in ops]
                t = table.detach().requires_grad_(True)
                do = torch.ones((), device="cuda", dtype=dtype).expand(B, H, Nq, D)
                o = g.cross_attention(*x, buckets=ids.contiguous() if copy else ids, bias_table=t,
                                      key_mask=mask.contiguous() if copy else mask)
                outs.append([o.detach(), *torch.autograd.grad(o, [*x, t], do)])
            for a, b in zip(*outs):
                assert torch.equal(a, b), name
    leaf = r(1, 1, Nk, D).requires_grad_(True)                        # a broadcast leaf: its copies' gradients sum
    q = r(B, H, Nq, D)
    o = g.cross_attention(q, leaf.expand(B, H, Nk, D), leaf.expand(B, H, Nk, D))
    (got,) = torch.autograd.grad(o, leaf, q)
    ref = ox.grads(q.cpu(), leaf.detach().expand(B, H, Nk, D).cpu(), leaf.detach().expand(B, H, Nk, D).cpu(), q.cpu())
    want = (ref["dk"] + ref["dv"]).sum((0, 1), keepdim=True)
    assert rel_l2(got, want) <= (4 * 2 ** -8 if dtype == BF else 2e-5)


def test_empty_inputs():
    import foreswe_gpu_optimization_b200 as g
    for B, H, Nq, Nk, D in ((0, 2, 3, 4, 8), (2, 2, 0, 4, 8), (2, 2, 3, 0, 8), (2, 0, 3, 4, 8), (2, 2, 3, 4, 0)):
        q, k = torch.randn(B, H, Nq, D, device="cuda"), torch.randn(B, H, Nk, D, device="cuda")
        x = [t.requires_grad_(True) for t in (q, k, k.clone())]
        o = g.cross_attention(*x)
        assert o.shape == q.shape and (o == 0).all()
        o.sum().backward()
        for t in x:
            assert t.grad is None or (t.grad.shape == t.shape and (t.grad == 0).all())
    assert g.dropout(torch.empty(0, 4, device="cuda"), 0.5, g.CounterRNG(1)).shape == (0, 4)


def test_empty_queries_give_zero_gradients():
    import foreswe_gpu_optimization_b200 as g
    for B, Nq in ((2, 0), (0, 3)):
        q, k = torch.randn(B, 2, Nq, 8, device="cuda"), torch.randn(B, 2, 4, 8, device="cuda")
        x = [t.requires_grad_(True) for t in (q, k, k.clone(), torch.randn(2, 5, device="cuda"))]
        o = g.cross_attention(*x[:3], buckets=torch.zeros(Nq, 4, dtype=torch.uint8, device="cuda"), bias_table=x[3])
        assert o.shape == q.shape
        for t, d in zip(x, torch.autograd.grad(o.sum(), x)):
            assert d.shape == t.shape and (d == 0).all()


def test_lengths_beyond_32_bits_are_clamped():
    import foreswe_gpu_optimization_b200 as g
    x, _ = make(3, 2, 2, 20, 70, 32, BF, seed=22)
    q, k, v = (x[n].cuda() for n in "qkv")
    got = g.cross_attention(q, k, v, kv_lens=torch.tensor([2 ** 32, -2 ** 40, 2 ** 32 + 5], device="cuda"))
    assert torch.equal(got, g.cross_attention(q, k, v, kv_lens=torch.tensor([70, 0, 70], device="cuda")))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_long_keys_with_few_rows(dtype):
    """Key ranges of one row are split over the GPU and joined: ragged lengths, one of them shorter than a range."""
    for Nq, H, Hkv, D in ((1, 4, 1, 128), (5, 2, 2, 64), (2, 3, 3, 192)):
        x, kw = make(3, H, Hkv, Nq, 5000, D, dtype, seed=D, T=4, lens=[5000, 4099, 3], mask=True)
        check(x, kw, p=0.1, key=[5, 6])


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_repeats_are_bitwise_equal(dtype):
    x, kw = make(4, 4, 2, 260, 390, 128, dtype, seed=3, T=32, mask=True)
    a, b = (run(x, kw, p=0.1, key=[1, 2]) for _ in range(2))
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_gradients_by_differences(dtype):
    """<gradient, u> against the 64-bit oracle's central difference of <o, dO> along u: step 1e-4 leaves a truncation
    error near 1e-8 relative, far below the gradients' tolerance; |<g - g', u>| <= tol |g| |u| bounds the rest."""
    x, kw = make(2, 2, 1, 40, 50, 64, dtype, seed=12, T=4, mask=True)
    got = run(x, kw, p=0.2, key=[8, 8])
    gen = torch.Generator().manual_seed(1)
    base = {n: x[n].double() for n in ("q", "k", "v", "table")}
    opt = {"ids": kw["ids"].long(), "mask": kw["mask"]}
    f = lambda y: (ox.forward(y["q"], y["k"], y["v"], table=y["table"], p=0.2, key=[8, 8], **opt)  # noqa: E731
                   * x["do"].double()).sum().item()
    for n in base:
        u = torch.randn(base[n].shape, generator=gen, dtype=torch.float64)
        d = (f({**base, n: base[n] + 1e-4 * u}) - f({**base, n: base[n] - 1e-4 * u})) / 2e-4
        grad = got["d" + n].double()
        assert abs((grad * u).sum().item() - d) <= tol(dtype, "d" + n) * grad.norm().item() * u.norm().item(), n


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 9), (512, 1024), (33, 1000)], ids=str)
def test_hidden_dropout(shape, dtype):
    """Kept elements exactly those of the generator; y = scale x + residual rounded once; dropped ones are 0 (or the
    residual) even where x is NaN."""
    import foreswe_gpu_optimization_b200 as g
    gen = torch.Generator().manual_seed(2)
    x, r, dy = (torch.randn(*shape, generator=gen).to(dtype) for _ in range(3))
    n = x.numel()
    for p, (seed, off) in ((0.1, (5, 3)), (0.6, (-9, 2 ** 40 + 1)), (1.0, (1, 0))):
        keep = ox.keep_flat(seed, off, n, p).view(shape)
        key = torch.tensor([seed, off], device="cuda")
        bad = x.clone()
        bad[~keep] = math.nan
        xd, rd = bad.cuda().requires_grad_(True), r.cuda().requires_grad_(True)
        eps = torch.finfo(dtype).eps / 2
        for res in (None, rd):
            y = g.dropout(xd, p, key, residual=res)
            want = torch.where(keep, x.double() * ox.scale_kept(p), 0.0) + (0 if res is None else r.double())
            # a rounding of the scale and of the product in fp32, and one to the type
            slack = (eps + 2 ** -22) * (want.abs() + x.double().abs() * ox.scale_kept(p) * 2 ** -22 / eps)
            assert ((y.detach().cpu().double() - want).abs() <= slack + 1e-30).all()
            grads = torch.autograd.grad(y, [xd] if res is None else [xd, rd], dy.cuda())
            want = torch.where(keep, dy.double() * ox.scale_kept(p), 0.0)
            assert ((grads[0].cpu().double() - want).abs() <= (eps + 2 ** -22) * want.abs()).all()
            if res is not None:
                assert torch.equal(grads[1].cpu(), dy)


def test_hidden_dropout_layouts():
    import foreswe_gpu_optimization_b200 as g
    key = torch.tensor([3, 4], device="cuda")
    base = torch.randn(40, 51, device="cuda")
    for x in (base.t(), base[:, 1:], base.reshape(-1)[1:], base[:1].expand(7, 51)):
        r = torch.randn(x.shape, device="cuda")
        assert torch.equal(g.dropout(x, 0.3, key, residual=r), g.dropout(x.contiguous(), 0.3, key, residual=r))
    assert g.dropout(base, 0.0, None) is base
    with pytest.raises(ValueError):
        g.dropout(base, 0.1, key, residual=base[:2])
    with pytest.raises(ValueError):
        g.dropout(base, 0.1, key.cpu())
    with pytest.raises(TypeError):
        g.dropout(base, 0.1, None)


def test_counter_rng_moves_on_and_replays_fresh():
    """Offsets are handed out in order; a captured step draws new masks at each replay, the same as eager calls."""
    import foreswe_gpu_optimization_b200 as g
    x = torch.randn(64, 256, device="cuda", dtype=BF)
    q = torch.randn(1, 2, 64, 64, device="cuda", dtype=BF, requires_grad=True)

    def step(rng):
        o = g.cross_attention(q, q, q, dropout_p=0.3, rng=rng)
        (dq,) = torch.autograd.grad(o, q, o.detach())
        return g.dropout(x, 0.4, rng), o.detach(), dq

    rng = g.CounterRNG(17)
    assert rng.take().tolist() == [17, 0] and rng.take().tolist() == [17, 1]
    eager = g.CounterRNG(17)
    want = [[t.clone() for t in step(eager)] for _ in range(3)]
    side = torch.cuda.Stream()
    rng = g.CounterRNG(17)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(rng)
    torch.cuda.current_stream().wait_stream(side)
    rng.state[1] = 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(rng)
    rng.state[1] = 0
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want[i]):
            assert torch.equal(a, b), i
    assert not torch.equal(want[0][0], want[1][0])
    del graph


def test_other_streams():
    """Two calls at once on two streams, each with its own workspace, give the results of calls one by one."""
    import foreswe_gpu_optimization_b200 as g
    sets = [make(2, 4, 2, 200, 2000, 128, BF, seed=s, T=8) for s in (1, 2)]
    dev = [({n: t.cuda() for n, t in x.items()}, kw["ids"].cuda()) for x, kw in sets]
    one = lambda x, ids: g.cross_attention(x["q"], x["k"], x["v"], buckets=ids, bias_table=x["table"])  # noqa: E731
    want = [one(*d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    for _ in range(3):
        got = []
        for s, d in zip(streams, dev):
            with torch.cuda.stream(s):
                got.append(one(*d))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_key_lengths_are_clamped(dtype):
    """Lengths below 0 and above Nk count as 0 and Nk, in either integer type and from a broadcast tensor."""
    import foreswe_gpu_optimization_b200 as g
    x, _ = make(3, 2, 2, 20, 70, 32, dtype, seed=21)
    q, k, v = (x[n].cuda() for n in "qkv")
    want = g.cross_attention(q, k, v, kv_lens=torch.tensor([0, 70, 33], device="cuda"))
    for t in (torch.int32, torch.int64):
        got = g.cross_attention(q, k, v, kv_lens=torch.tensor([-5, 1000, 33], dtype=t, device="cuda"))
        assert torch.equal(got, want)
    assert (want[0] == 0).all()
    one = g.cross_attention(q, k, v, kv_lens=torch.tensor([33], device="cuda").expand(3))
    assert torch.equal(one[2], want[2])
    row = torch.rand(1, 70, device="cuda") > 0.5
    assert torch.equal(g.cross_attention(q, k, v, key_mask=row.expand(3, 70)),
                       g.cross_attention(q, k, v, key_mask=row.repeat(3, 1)))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_scratch_in_several_launches(dtype):
    """A batch whose dS scratch passes 4 GB runs its backward in several launches: each batch entry's gradients are
    bitwise those of a call of its own, and the table's gradient (whose partial sums are grouped differently) is the
    sum of theirs to the rounding of its terms."""
    import foreswe_gpu_optimization_b200 as g
    B, H, Nq, Nk, D, T = (2, 36, 4096, 8192, 16, 6) if dtype == BF else (2, 20, 4096, 8192, 16, 6)
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    q, k, v, do = r(B, H, Nq, D), r(B, H, Nk, D), r(B, H, Nk, D), r(B, H, Nq, D)
    table = torch.randn(H, T, generator=gen, device="cuda")
    ids = torch.randint(0, T, (Nq, Nk), generator=gen, device="cuda").to(torch.uint8)

    def grads(sl):
        x = [t[sl].detach().requires_grad_(True) for t in (q, k, v)]
        t = table.detach().requires_grad_(True)
        o = g.cross_attention(*x, buckets=ids, bias_table=t)
        return torch.autograd.grad(o, [*x, t], do[sl])

    both = grads(slice(0, 2))
    ones = [grads(slice(b, b + 1)) for b in range(B)]
    for i in range(3):
        for b in range(B):
            assert torch.equal(both[i][b:b + 1], ones[b][i]), (i, b)
    # 2^12 partial sums at most, each of fp32 terms: 2^-24 * 2^12 of the sums' size bounds the regrouping
    size = sum(o[3].abs() for o in ones)
    assert ((both[3] - sum(o[3] for o in ones)).abs() <= 2.0 ** -12 * (size + size.max())).all()


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_offsets_past_32_bits(dtype):
    """Batch entries more than 2^31 elements apart in one cache."""
    import foreswe_gpu_optimization_b200 as g
    H, Nk, D = 2, 200, 64
    far = 2 ** 31 + 64
    cache = torch.zeros(far + H * Nk * D, dtype=dtype, device="cuda")
    x, _ = make(2, H, H, 30, Nk, D, dtype, seed=3)
    k = cache.as_strided((2, H, Nk, D), (far, Nk * D, D, 1))
    k.copy_(x["k"])
    outs = []
    for kk in (k, x["k"].cuda()):
        leaves = [x["q"].cuda().requires_grad_(True), kk.detach().requires_grad_(True),
                  x["v"].cuda().requires_grad_(True)]
        o = g.cross_attention(leaves[0], leaves[1], leaves[1])
        outs.append([o.detach(), *torch.autograd.grad(o, leaves[:2], x["do"].cuda())])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_query_counts_around_the_chunks():
    """1 to 200 queries: the chunk sizes of the backward and the padding of the last one."""
    for Nq in (1, 8, 9, 16, 17, 31, 63, 64, 65, 96, 127, 128, 129, 192, 193):
        for D in (64, 128, 192):
            x, kw = make(1, 2, 1, Nq, 140, D, BF, seed=Nq, T=5, mask=True)
            check(x, kw, p=0.1, key=[Nq, D])


FEW = [  # B, H, Hkv, Nq, Nk, D: few query rows per key head: every row count of a CTA, packed tiles, key ranges
    (3, 2, 2, 1, 1, 64), (2, 2, 2, 1, 63, 40), (1, 2, 2, 1, 1100, 64), (2, 4, 2, 1, 2051, 128),
    (1, 3, 1, 1, 1030, 192), (2, 6, 2, 1, 130, 100), (1, 5, 1, 1, 1500, 61), (2, 8, 1, 1, 700, 192),
    (1, 2, 2, 2, 1029, 128), (2, 4, 1, 2, 90, 64), (2, 2, 2, 7, 300, 175), (1, 2, 2, 8, 1025, 64),
    (2, 3, 3, 9, 70, 64), (1, 6, 2, 28, 1200, 192), (1, 8, 1, 32, 130, 33), (2, 2, 1, 31, 1, 128),
    (2, 16, 1, 8, 300, 64), (1, 17, 1, 3, 200, 64), (1, 32, 2, 5, 1500, 128), (2, 6, 2, 42, 130, 192),
]


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "x".join(map(str, s)))
def test_few_rows(shape, dtype):
    B, H, Hkv, Nq, Nk, D = shape
    check(*make(*shape, dtype, seed=31))
    lens = [0 if B > 1 and b == 0 else max(1, Nk - 7 * b) for b in range(B)]
    x, kw = make(*shape, dtype, seed=32, T=9, lens=lens, mask=Nk > 1, cut=Nk > 1)
    check(x, kw, p=0.2, key=[99, 7])


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Nq, G", [(1, 1), (1, 4), (3, 2)])
def test_few_rows_garbage_and_guards(Nq, G, dtype):
    """NaN in absent keys and infinity in absent values; gradients land inside their tensors and nowhere else."""
    import foreswe_gpu_optimization_b200 as g
    B, Hkv, Nk, D = 2, 2, 600, 72
    x, kw = make(B, Hkv * G, Hkv, Nq, Nk, D, dtype, seed=33, lens=[600, 517], mask=True)
    dead = ~ox.live_keys(B, Nk, kw["lens"], kw["mask"])
    clean = {n: t.clone() for n, t in x.items()}
    for n, bad in (("k", float("nan")), ("v", float("inf"))):
        clean[n] = x[n].masked_fill(dead.view(B, 1, Nk, 1), 0.0)
        x[n] = x[n].masked_fill(dead.view(B, 1, Nk, 1), bad)
    got, want = run(x, kw), run(clean, kw)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert got["dk"].masked_select(dead.view(B, 1, Nk, 1)).eq(0).all()
    # a query that is NaN gives NaN in its own row only
    y = {n: t.cuda() for n, t in clean.items()}
    y["q"][0, 0, 0, 3] = float("nan")
    o = g.cross_attention(y["q"], y["k"], y["v"], kv_lens=kw["lens"].cuda(), key_mask=kw["mask"].cuda())
    assert o[0, 0, 0].isnan().all() and o.isnan().sum() == D


def test_few_rows_repeat_bitwise_and_replay():
    """The same call twice, and captured and replayed on changed inputs, with key ranges that are joined."""
    import foreswe_gpu_optimization_b200 as g
    for dtype in (BF, FP):
        x, _ = make(1, 2, 2, 1, 5000, 64, dtype, seed=34)
        y = {n: t.cuda() for n, t in x.items()}
        for n in "qkv":
            y[n] = y[n].detach().requires_grad_()

        def step():
            o = g.cross_attention(y["q"], y["k"], y["v"])
            return (o.detach(), *torch.autograd.grad(o, [y[n] for n in "qkv"], y["do"]))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
            step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        with torch.no_grad():
            y["k"].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_many_key_tiles_per_cta():
    """More key tiles than the persistent key pass has CTAs, some of them past their batch entry's length."""
    for D, Nq in ((64, 40), (64, 130), (128, 20), (128, 300), (192, 33)):
        x, kw = make(7, 6, 6, Nq, 600, D, BF, seed=D + Nq, T=7, lens=[600, 1, 0, 129, 256, 513, 77])
        check(x, kw, p=0.2, key=[4, 4])


def test_a_thread_of_its_own():
    """Forward and backward as the first CUDA work of a thread."""
    import threading
    x, kw = make(1, 2, 2, 70, 90, 64, BF, seed=5)
    want, got = run(x, kw), {}
    t = threading.Thread(target=lambda: got.update(run(x, kw)))
    t.start()
    t.join()
    assert got and all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("nq, n, T", [(1, 1, 1), (70, 130, 20), (257, 64, 64)])
def test_distance_buckets(nq, n, T):
    import foreswe_gpu_optimization_b200 as g
    from oracle import geometry as ogeo
    a, b = stations(nq, 1), stations(n, 2)
    both = ogeo.haversine_km(np.concatenate([a[0], b[0]]), np.concatenate([a[1], b[1]]))[:nq, nq:]
    edges = np.geomspace(20.0, 1200.0, T - 1)
    want = np.searchsorted(edges, both, side="right")
    geom, query = g.StationGeometry(*b), g.StationGeometry(*a)
    assert np.array_equal(geom.distance_buckets(edges, queries=query).cpu().numpy(), want)
    want[both > 700.0] = 255
    assert np.array_equal(geom.distance_buckets(edges, queries=query, max_km=700.0).cpu().numpy(), want)
    self_ids = geom.distance_buckets(edges).cpu().numpy()
    assert self_ids.shape == (n, n) and (np.diag(self_ids) == 0).all()


def test_patched_layers_draw_from_the_generator():
    """patch_model(dropout_rng=...): the layers' dropout takes the generator's masks in training, none in evaluation."""
    import foreswe_gpu_optimization_b200 as g
    from helpers import Encoder
    torch.manual_seed(0)
    N, H, D = 96, 2, 64
    model = Encoder(H * D, H, 2).cuda()
    for layer in model.encoder_layers:
        layer.drop = torch.nn.Dropout(0.3)
        inner = layer.self_attn
        inner.register_forward_hook(lambda m, a, out, drop=layer.drop: drop(out))
    geom = g.StationGeometry(*stations(N, 3))
    rng = g.CounterRNG(11)
    g.patch_model(model, geometry=geom, dropout_rng=rng)
    x = torch.randn(2, N, H * D, device="cuda")
    y1 = model(x, None, None)
    assert rng.state.tolist() == [11, 2]
    rng.state[1] = 0
    y2 = model(x, None, None)
    assert torch.equal(y1, y2)
    y1.sum().backward()
    model.eval()
    model(x, None, None)
    assert rng.state.tolist() == [11, 2]


def test_station_step_end_to_end():
    """The operators as they are used together: stations encode themselves (geo_attention), sites attend to them with
    the learned bias by distance, missing stations and dropout, and dropout joins the residual; every gradient against
    float64 autograd of the same step."""
    import foreswe_gpu_optimization_b200 as g
    from helpers import dense_geometry
    from oracle import geo_attention as oga
    B, H, N, M, D = 2, 4, 130, 45, 64
    st, si = stations(N, 5), stations(M, 6)
    geom, sites = g.StationGeometry(*st), g.StationGeometry(*si)
    edges = np.geomspace(50.0, 900.0, 9)
    ids = geom.distance_buckets(edges, queries=sites, max_km=1100.0)
    gen = torch.Generator().manual_seed(7)
    x = {n: torch.randn(*s, generator=gen) * 0.6 for n, s in
         (("h", (B, H, N, D)), ("q", (B, H, M, D)), ("table", (H, 10)), ("res", (B, H, M, D)), ("do", (B, H, M, D)))}
    abg = [torch.rand(H, generator=gen) * 0.9 + 0.1, torch.randn(H, generator=gen) * 0.5,
           torch.randn(H, generator=gen) * 0.5]
    mask = torch.rand(B, N, generator=gen) > 0.2
    leaves = {n: t.cuda().requires_grad_(True) for n, t in x.items() if n != "do"}
    e = g.geo_attention(leaves["h"], leaves["h"], leaves["h"], geom, *(t.cuda() for t in abg))
    o = g.cross_attention(leaves["q"], e, e, buckets=ids, bias_table=leaves["table"], key_mask=mask.cuda(),
                          dropout_p=0.1, rng=torch.tensor([1, 0], device="cuda"))
    y = g.dropout(o, 0.2, torch.tensor([1, 1], device="cuda"), residual=leaves["res"])
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), x["do"].cuda())))
    dist, ang = (t.double() for t in dense_geometry(*st))
    d = {n: t.double().requires_grad_(True) for n, t in x.items()}
    er = oga.forward(d["h"], d["h"], d["h"], dist, ang, *(t.double() for t in abg))
    orf = ox.forward(d["q"], er, er, ids=ids.cpu().long(), table=d["table"], mask=mask, p=0.1, key=(1, 0))
    yr = torch.where(ox.keep_flat(1, 1, orf.numel(), 0.2).view(orf.shape), orf * ox.scale_kept(0.2), 0.0) + d["res"]
    want = dict(zip(leaves, torch.autograd.grad(yr, [d[n] for n in leaves], x["do"].double())))
    assert rel_l2(y.detach(), yr.detach()) <= 5e-4                    # the encoder runs on the TF32 path
    for n in leaves:
        # the encoder's own tolerance, 5e-4 of its output, reaches these gradients through k and v
        assert rel_l2(got[n], want[n]) <= 2e-3, n

"""Cross attention, its bucketed bias and dropout without a GPU: the oracle and the refusals."""
import math

import numpy as np
import pytest
import torch

import foreswe_gpu_optimization_b200 as g
from oracle import cross_attention as ox

BF = torch.bfloat16


def test_philox_known_answers():
    """Published test vectors of Philox4x32 with 7 rounds: all-zero and all-one counter and key."""
    zero = [int(x) for x in ox.philox((0, 0, 0, 0), (0, 0))]
    assert zero == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    f = 2 ** 32 - 1
    ones = [int(x) for x in ox.philox((f, f, f, f), (f, f))]
    assert ones == [0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662]


def test_keep_probability_of_the_generator():
    """2^20 elements at p = 0.1: the kept share is within 5 standard deviations (5 sqrt(p (1 - p) / n) = 1.5e-3)."""
    n = 1 << 20
    for seed, off in ((1, 0), (-5, 7), (2 ** 63 - 1, 2 ** 40)):
        kept = ox.keep_flat(seed, off, n, 0.1).double().mean().item()
        assert abs(kept - 0.9) < 5 * math.sqrt(0.09 / n)


def test_oracle_gradients_by_differences():
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64, requires_grad=True)  # noqa: E731
    q, k, v, table = r(2, 4, 3, 5), r(2, 2, 6, 5), r(2, 2, 6, 5), r(4, 3)
    ids = torch.randint(0, 4, (3, 6), generator=gen)
    ids[1] = 255
    kw = dict(ids=ids, lens=torch.tensor([6, 4]), mask=torch.rand(2, 6, generator=gen) > 0.2, p=0.3, key=(9, 4))
    assert torch.autograd.gradcheck(lambda q, k, v, t: ox.forward(q, k, v, table=t, **kw), (q, k, v, table))


def _qkv(B=2, H=4, Hkv=2, Nq=3, Nk=5, D=8, dtype=BF):
    return torch.zeros(B, H, Nq, D, dtype=dtype), torch.zeros(B, Hkv, Nk, D, dtype=dtype), torch.zeros(
        B, Hkv, Nk, D, dtype=dtype)


@pytest.mark.parametrize("bad, error", [
    (lambda q, k, v: dict(q=q[0]), ValueError),
    (lambda q, k, v: dict(k=k[:1], v=v[:1]), ValueError),
    (lambda q, k, v: dict(v=v[:, :, :2]), ValueError),
    (lambda q, k, v: dict(k=k[..., :4], v=v[..., :4]), ValueError),
    (lambda q, k, v: dict(q=q[:, :3]), ValueError),
    (lambda q, k, v: dict(k=k[:, :0], v=v[:, :0]), ValueError),
    (lambda q, k, v: dict(zip("qkv", _qkv(D=200))), ValueError),
    (lambda q, k, v: dict(q=q.float()), TypeError),
    (lambda q, k, v: dict(zip("qkv", _qkv(dtype=torch.float16))), TypeError),
    (lambda q, k, v: dict(buckets=torch.zeros(3, 5, dtype=torch.uint8)), ValueError),
    (lambda q, k, v: dict(bias_table=torch.zeros(4, 2)), ValueError),
    (lambda q, k, v: dict(buckets=torch.zeros(3, 5, dtype=torch.int64), bias_table=torch.zeros(4, 2)), ValueError),
    (lambda q, k, v: dict(buckets=torch.zeros(5, 3, dtype=torch.uint8), bias_table=torch.zeros(4, 2)), ValueError),
    (lambda q, k, v: dict(buckets=torch.zeros(3, 5, dtype=torch.uint8), bias_table=torch.zeros(4, 65)), ValueError),
    (lambda q, k, v: dict(buckets=torch.zeros(3, 5, dtype=torch.uint8), bias_table=torch.zeros(4, 0)), ValueError),
    (lambda q, k, v: dict(buckets=torch.zeros(3, 5, dtype=torch.uint8), bias_table=torch.zeros(2, 8)), ValueError),
    (lambda q, k, v: dict(buckets=torch.zeros(3, 5, dtype=torch.uint8), bias_table=torch.zeros(4, 8).half()),
     TypeError),
    (lambda q, k, v: dict(kv_lens=torch.ones(2)), ValueError),
    (lambda q, k, v: dict(kv_lens=torch.ones(3, dtype=torch.int32)), ValueError),
    (lambda q, k, v: dict(key_mask=torch.ones(2, 5)), ValueError),
    (lambda q, k, v: dict(key_mask=torch.ones(2, 4, dtype=torch.bool)), ValueError),
    (lambda q, k, v: dict(dropout_p=0.1), ValueError),
    (lambda q, k, v: dict(dropout_p=1.1, rng=torch.zeros(2, dtype=torch.int64)), ValueError),
    (lambda q, k, v: dict(dropout_p=float("nan"), rng=torch.zeros(2, dtype=torch.int64)), ValueError),
    (lambda q, k, v: dict(scale=math.inf), ValueError),
    (lambda q, k, v: dict(scale=math.nan), ValueError),
    (lambda q, k, v: dict(scale=0.0), ValueError),
    (lambda q, k, v: dict(scale=-1.0), ValueError),
    (lambda q, k, v: {}, RuntimeError),                              # CPU tensors
])
def test_cross_attention_refusals(bad, error):
    q, k, v = _qkv()
    kw = dict(q=q, k=k, v=v)
    kw.update(bad(q, k, v))
    with pytest.raises(error):
        g.cross_attention(kw.pop("q"), kw.pop("k"), kw.pop("v"), **kw)


def test_dropout_refusals():
    x, key = torch.zeros(4, 8, dtype=BF), torch.zeros(2, dtype=torch.int64)
    for args, kw, error in (((x, 0.5, key), {}, RuntimeError), ((x.half(), 0.5, key), {}, TypeError),
                            ((x, -0.1, key), {}, ValueError), ((x, 1.5, key), {}, ValueError)):
        with pytest.raises(error):
            g.dropout(*args, **kw)


def test_patch_model_dropout_is_checked_and_taken_away():
    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            layer = torch.nn.Module()
            layer.self_attn, layer.dropout = torch.nn.Module(), torch.nn.Dropout(0.1)
            self.encoder_layers = torch.nn.ModuleList([layer])

    m = Model()
    own = m.encoder_layers[0].dropout
    with pytest.raises(TypeError):
        g.patch_model(m, dropout_rng=torch.zeros(2, dtype=torch.int64))
    assert "forward" not in own.__dict__
    g.patch_model(m)
    assert "forward" not in own.__dict__
    g.patch_model(m, dropout_rng=g.CounterRNG(1, device="cpu"))
    assert "forward" in own.__dict__
    own.eval()
    x = torch.ones(3)
    assert own(x) is x
    g.patch_model(m, "eager")
    assert "forward" not in own.__dict__


def test_counter_rng_holds_any_seed():
    r = g.CounterRNG(2 ** 64 - 1, device="cpu", offset=3)
    assert r.state.tolist() == [-1, 3]
    assert g.CounterRNG(-7, device="cpu").state.tolist() == [-7, 0]


def test_bucket_edges_are_checked():
    geom = g.StationGeometry(np.zeros(3), np.zeros(3), np.zeros(3), device="cpu")
    for edges in ([3.0, 1.0], list(range(64)), [float("nan")]):
        with pytest.raises(ValueError):
            geom.distance_buckets(edges)
    with pytest.raises(ValueError):
        geom.distance_buckets([1.0], max_km=-1)
    with pytest.raises(TypeError):
        geom.distance_buckets([1.0], queries=torch.zeros(3))


def test_c_abi_refuses_before_any_launch():
    import ctypes

    from foreswe_gpu_optimization_b200 import _lib, build
    build.build()
    L = _lib.lib()
    assert L.geoattn_xattn_fwd(None, None) == 1 and L.geoattn_xattn_bwd(None, None) == 1
    good = dict(batch=2, heads=4, kv_heads=2, nq=3, nk=5, head_dim=8, dtype=0, buckets=0, table_dtype=1)
    size = lambda f, **kw: f(ctypes.byref(_lib.XattnShape(**{**good, **kw})))  # noqa: E731
    for f in (L.geoattn_xattn_fwd_workspace_bytes, L.geoattn_xattn_bwd_workspace_bytes):
        assert size(f) > 0
        for bad in (dict(kv_heads=3), dict(nq=0), dict(head_dim=193), dict(buckets=65), dict(dtype=2), dict(batch=-1)):
            assert size(f, **bad) == 0
    args = _lib.XattnFwdArgs()
    args.inputs.shape = _lib.XattnShape(**good)
    assert L.geoattn_xattn_fwd(ctypes.byref(args), None) == 1        # null pointers
    assert L.geoattn_dropout(0, 8, None, None, None, None, 5, None) == 1
    assert L.geoattn_dropout(7, 8, None, None, None, None, 5, None) == 1
    assert L.geoattn_rng_take(None, None, None) == 1
    assert L.geoattn_distance_buckets(3, None, None, 3, None, None, None, 0, 1.0, None, None) == 1

"""CPU tests: what ops.dot_attention, ops.embedding, ops.newton_schulz, their C entry points and their layers refuse, and the 64-bit
form that the GPU tests compare with against differences."""
import ctypes

import numpy as np
import pytest
import torch

from tests import attn_ref


def _t(*s, dtype=torch.float32):
    return torch.zeros(s, dtype=dtype)


def test_dot_attention_refuses():
    from gat_amd import ops
    q, k = _t(2, 5, 4, 8), _t(2, 7, 2, 8)
    for bad, kind in (((_t(2, 5, 8), k, k), ValueError), ((q, _t(2, 7, 3, 8), _t(2, 7, 3, 8)), ValueError), ((q, k, _t(2, 6, 2, 8)), ValueError),
                      ((q, _t(1, 7, 2, 8), _t(1, 7, 2, 8)), ValueError), ((q, k.double(), k), TypeError), ((q.half(), k.half(), k.half()), TypeError),
                      ((_t(2, 5, 4, 130), _t(2, 7, 2, 130), _t(2, 7, 2, 130)), ValueError), ((q, _t(2, 7, 0, 8), _t(2, 7, 0, 8)), ValueError),
                      ((_t(2, 5, 4, 0), _t(2, 7, 2, 0), _t(2, 7, 2, 0)), ValueError)):
        with pytest.raises(kind):
            ops.dot_attention(*bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.dot_attention(q, k, k)


def test_embedding_refuses():
    from gat_amd import ops
    with pytest.raises(TypeError):
        ops.embedding(_t(3), _t(4, 8))
    with pytest.raises(TypeError):
        ops.embedding([1, 2], _t(4, 8))
    with pytest.raises(ValueError):
        ops.embedding(_t(3, dtype=torch.int64), _t(4, 8, 2))
    with pytest.raises(ValueError):
        ops.embedding(_t(3, dtype=torch.int64), _t(4, 0))
    with pytest.raises(TypeError):
        ops.embedding(_t(3, dtype=torch.int64), _t(4, 8, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.embedding(_t(3, dtype=torch.int64), _t(4, 8))


def test_newton_schulz_refuses():
    from gat_amd import ops
    with pytest.raises(ValueError):
        ops.newton_schulz(_t(4))
    with pytest.raises(TypeError):
        ops.newton_schulz(_t(4, 4, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.newton_schulz(_t(4, 4))


def test_c_entry_points_refuse_before_any_launch():
    from gat_amd import _lib
    lib, f = _lib.lib, ctypes.c_float
    s3 = (ctypes.c_int64 * 3)(32, 16, 8)
    odd = (ctypes.c_int64 * 3)(33, 16, 8)
    P = 4096                                                       # a 16-byte aligned address that no accepted call below uses

    def fwd(B=1, Nq=2, Nk=2, H=2, G=2, D=8, dt=0, q=P, qs=s3, k=P, bias=None, br=2, out=P, scale=1.0, low=None):
        return lib.gatmi_dot_attn_fwd(B, Nq, Nk, H, G, D, dt, q, qs, k, s3, P, s3, bias, 0, br, None, None, scale, out, low, None, None, None, None, None)

    for rc, want, text in ((fwd(B=-1), -1, "B = -1"), (fwd(H=3), -1, "3 query heads"), (fwd(G=0), -1, "heads"), (fwd(D=6), -3, "head width 6"), (fwd(D=132), -3, "132"),
                           (fwd(D=12, dt=1), -3, "head width 12"), (fwd(dt=2), -1, "dtype"), (fwd(q=None), -1, "q is null"), (fwd(q=P + 4), -2, "aligned"), (fwd(qs=odd), -2, "aligned"),
                           (fwd(k=None), -1, "k is null"), (fwd(bias=P, br=1), -1, "bias row stride"), (fwd(out=None), -1, "out is null"), (fwd(low=P), -1, "out_low is for bf16"), (fwd(Nq=20, bias=P), -1, "mask words"), (fwd(Nq=2 ** 30, H=4, G=4), -4 - 1, "31 bits"), (fwd(scale=float("nan")), -1, "scale")):
        assert rc == want, (rc, want, text)
    assert fwd(B=0) == 0 and fwd(Nq=0) == 0
    rc = lib.gatmi_dot_attn_bwd(1, 2, 2, 2, 2, 8, 0, P, s3, P, s3, P, s3, P, None, P, s3, None, None, 0, 2, None, None, 1.0, None, None, P, P, P, P, None, None)
    assert rc == -1 and "null" in _lib.last_error()

    def emb(bits=64, n=4, ld=8, rows=4, w=8, dt=0, ids=P):
        return lib.gatmi_embed_fwd(ids, bits, n, P, ld, rows, w, dt, f(1.0), P, None)
    assert emb(bits=16) == -1 and emb(n=-1) == -1 and emb(ld=7) == -1 and emb(w=0) == -1 and emb(dt=5) == -1 and emb(ids=None) == -1
    assert emb(n=2 ** 31) == -5 and emb(rows=2 ** 31) == -5 and emb(w=70000) == -3 and emb(n=0) == 0
    bwd = lambda **k: lib.gatmi_embed_bwd(P, 64, k.get("n", 4), P, k.get("ld", 8), 4, 8, 0, f(1.0), k.get("out", P), k.get("ws", P), None)
    assert bwd(ld=3) == -1 and bwd(out=None) == -1 and bwd(ws=None) == -1 and bwd(ws=P + 4) == -2

    def ns(m=4, n=200, row=200, dt=0, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, x=P, ws=P):
        return lib.gatmi_newton_schulz(1, m, n, x, 16, row, dt, steps, a, b, c, eps, P, 16, row, ws, None)
    assert ns(m=-1) == -1 and ns(row=199) == -1 and ns(dt=3) == -1 and ns(steps=0) == -1 and ns(steps=33) == -1 and ns(eps=0.0) == -1 and ns(x=None) == -1 and ns(ws=P + 8) == -2
    assert ns(a=9.0) == -3 and "bounded" in _lib.last_error()
    assert ns(a=float("nan")) == -1 and ns(c=float("inf")) == -1 and ns(eps=float("nan")) == -1
    assert ns(m=2 ** 21, n=100, row=100) == -5
    assert ns(m=0) == 0


def test_layers_refuse():
    from gat_amd import layers, models
    with pytest.raises(ValueError):
        layers.DotHeads(8, 4, 8, kv_heads=3)
    with pytest.raises(ValueError):
        layers.DotHeads(8, 4, 8, storage="f16")
    m = layers.DotHeads(8, 2, 8)
    with pytest.raises(ValueError):
        m(_t(1, 3, 8), None, "elu", "mean")
    with pytest.raises(ValueError):
        m(_t(1, 3, 8), None, "elu", "sum")
    store = layers.VariableStore()
    store.next_heads(8, 2, 4, False, None)
    store.begin()
    with pytest.raises(ValueError, match="GATHeads"):
        store.next_heads(8, 2, 4, False, None, layers.DotHeads)
    w = torch.nn.Parameter(_t(4, 2, 3))
    for bad in ([w], [(w, 2)], [(torch.nn.Parameter(_t(4)), None)]):
        with pytest.raises(ValueError):
            models.Muon(bad)
    with pytest.raises(ValueError):
        models.Muon([(w, 1)], momentum=1.0)


def test_matrix_parameters_covers_every_parameter_once():
    from gat_amd import layers, models
    m = models.GAT_AE_BNF_V2(5, 12, 2, 8, [16], [2])
    mats, others = models.matrix_parameters(m)
    ids = [id(p) for p, _ in mats] + [id(p) for p in others]
    assert len(ids) == len(set(ids)) == len(list(m.parameters()))
    assert all(p.dim() == (2 if a is None else 3) for p, a in mats) and all(p.dim() <= 2 for p in others)
    assert sum(a == 1 for _, a in mats) == 10 and sum(a == 0 for _, a in mats) == 10
    mats, others = models.matrix_parameters(layers.DotHeads(8, 2, 4, residual=True))
    assert [a for _, a in mats] == [1, 1] and len(others) == 2


def test_reference_gradients_against_differences():
    rng = np.random.default_rng(0)
    B, Nq, Nk, H, G, D = 2, 5, 6, 4, 2, 3
    x = {"q": rng.normal(0, 1, (B, Nq, H, D)), "k": rng.normal(0, 1, (B, Nk, G, D)), "v": rng.normal(0, 1, (B, Nk, G, D))}
    bias = np.where(rng.random((B, Nq, Nk)) < 0.7, rng.normal(0, 1, (B, Nq, Nk)), -1e9)
    ks, qs = np.array([6, 4]), np.array([5, 3])
    dout = rng.normal(0, 1, (B, Nq, H, D))
    ref = attn_ref.attention(x["q"], x["k"], x["v"], bias, ks, qs, 0.7, dout)
    for n in ("q", "k", "v"):
        d = rng.normal(0, 1, x[n].shape)

        def f(t):
            y = dict(x)
            y[n] = x[n] + t * d
            return (attn_ref.attention(y["q"], y["k"], y["v"], bias, ks, qs, 0.7)["out"][0] * dout).sum()

        assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - (ref["d" + n][0] * d).sum()) < 1e-7

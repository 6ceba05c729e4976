"""bf16 attention without a mask on both sides of 1024 nodes, where P and dz go from two bf16 numbers each to one: widths, lengths next to the
border and to a tile, keys split and not, shared heads, padded graphs.

Bounds: the counted ones of attn_ref, and the mean: every result is a sum of terms of random signs, whose roundings (P or dz, at most 2^-8 of a
term, and the result's own, at most 2^-8 of it) add up as the terms do, so the root mean square of the error is at most 2 * 2^-8 of the results'."""
import numpy as np
import pytest
import torch

from tests import attn_ref
from tests.attn_ref import U16, within
from tests.test_dot_attention_gpu import _case, _np, _run

pytestmark = pytest.mark.gpu


def _check(c, what, mean=True):
    got = _run(c)
    ref = attn_ref.attention(_np(c["q"]), _np(c["k"]), _np(c["v"]), None, _np(c["ks"]), _np(c["qs"]), None, _np(c["dout"]), True)
    for n, (value, bound) in ref.items():
        g = _np(got[n])
        within(g, value, bound, "%s %s" % (what, n))
        if mean:
            assert np.sqrt(((g - value) ** 2).mean()) <= 2 * U16 * np.sqrt((value ** 2).mean()), (what, n)
    return got


@pytest.mark.parametrize("D", [8, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("N", [1024, 1025])
def test_widths_on_both_sides(N, D):
    _check(_case(1, N, N, 2, 1, D, "bf16", seed=D), "%d nodes, %d wide" % (N, D))


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("Nq,Nk", [(1100, 65), (1025, 64), (1025, 127), (1088, 129), (65, 1025), (65, 1600), (66, 5000), (130, 1152), (1100, 1100), (1061, 1303)])
def test_lengths(Nq, Nk, D):
    """Nq = 65 and more on many keys: split over the keys in the forward."""
    _check(_case(2, Nq, Nk, 2, 2, D, "bf16", seed=Nq + Nk), "%d x %d, %d wide" % (Nq, Nk, D))


@pytest.mark.parametrize("H,G", [(3, 1), (4, 4), (6, 2)])
def test_shared_heads(H, G):
    _check(_case(1, 1030, 1030, H, G, 64, "bf16", seed=H), "%d on %d" % (H, G))
    _check(_case(1, 40, 1500, H, G, 32, "bf16", seed=H), "few queries, %d on %d" % (H, G))


def test_keys_not_split():
    """So many graphs that each block walks all keys of one."""
    from gat_amd import _lib
    assert _lib.lib.gatmi_dot_attn_fwd_ws_floats(50, 70, 1025, 8, 8, 16) == 0 < _lib.lib.gatmi_dot_attn_fwd_ws_floats(2, 70, 1025, 8, 8, 16)
    c = _case(50, 70, 1025, 8, 8, 16, "bf16", seed=3)
    got = _run(c)
    few = {n: (None if t is None else t[:2].contiguous()) for n, t in c.items()}
    ref = attn_ref.attention(_np(few["q"]), _np(few["k"]), _np(few["v"]), None, None, None, None, _np(few["dout"]), True)
    for n, (value, bound) in ref.items():
        within(_np(got[n][:2]), value, bound, n)


@pytest.mark.parametrize("D", [20, 64, 128])
def test_padded_graphs_with_anything_behind_them(D):
    c = _case(5, 1100, 1100, 2, 1, D, "bf16", seed=D)
    sizes = [1100, 0, 1, 65, 1025]
    c["ks"] = c["qs"] = torch.tensor(sizes, dtype=torch.int32, device="cuda:0")
    want = _check(c, "%d wide" % D, mean=False)
    for n in ("q", "k", "v", "dout"):
        x = c[n].clone()
        for b, s in enumerate(sizes):
            x[b, s:] = float("nan")
        c[n] = x
    got = _run(c)
    for n in want:
        assert torch.equal(got[n], want[n]), n
        for b, s in enumerate(sizes):
            assert (got[n][b, s:] == 0).all(), n


def test_sizes_of_queries_and_keys_apart():
    c = _case(4, 1060, 700, 2, 2, 32, "bf16", seed=5)
    c["ks"] = torch.tensor([700, 1, 0, 333], dtype=torch.int32, device="cuda:0")
    c["qs"] = torch.tensor([3, 1060, 1060, 0], dtype=torch.int32, device="cuda:0")
    _check(c, "sizes apart", mean=False)


def test_scale_and_an_empty_set_of_keys():
    c = _case(1, 1030, 1030, 1, 1, 16, "bf16", seed=6)
    for scale in (-0.5, 0.0, 3.0):
        got = _run(c, scale=scale)
        ref = attn_ref.attention(_np(c["q"]), _np(c["k"]), _np(c["v"]), None, None, None, scale, _np(c["dout"]), True)
        for n, (value, bound) in ref.items():
            within(_np(got[n]), value, bound, "scale %g %s" % (scale, n))
    c["ks"] = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    for n, x in _run(c).items():
        assert (x == 0).all(), n


def test_twice_the_same_bits_on_another_stream_and_captured():
    from gat_amd import graphs, ops
    c = _case(2, 1100, 1100, 4, 2, 64, "bf16", seed=7)
    want = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(want[n], got[n]), n
    q, k, v = (c[n].clone().requires_grad_() for n in ("q", "k", "v"))

    def step():
        out = ops.dot_attention(q, k, v)
        return (out, *torch.autograd.grad(out, (q, k, v), c["dout"]))

    replay, res = graphs.capture(step, fresh_dropout=False)
    for seed in range(3):
        n = _case(2, 1100, 1100, 4, 2, 64, "bf16", seed=20 + seed)
        with torch.no_grad():
            for a, b in ((q, n["q"]), (k, n["k"]), (v, n["v"])):
                a.copy_(b)
            c["dout"].copy_(n["dout"])
        replay()
        torch.cuda.synchronize()
        for a, b in zip(res, _run(n).values()):
            assert torch.equal(a, b), seed

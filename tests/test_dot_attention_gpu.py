"""GPU parity of ops.dot_attention, forward and gradients, against its 64-bit form within counted rounding bounds: types, head
layouts, lengths from one row to long ones, masks that leave rows empty, padded graphs, strides, streams and captured graphs."""
import numpy as np
import pytest
import torch

from tests import attn_ref
from tests.attn_ref import within

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _case(B, Nq, Nk, H, G, D, dtype, density=None, shared_mask=False, sizes=False, seed=0, soft=False):
    rng = np.random.default_rng(seed)
    dev = torch.device("cuda:0")
    t = lambda *s: torch.tensor(rng.normal(0, 1, s), dtype=torch.float32).to(TYPES[dtype]).to(dev)
    c = {"q": t(B, Nq, H, D), "k": t(B, Nk, G, D), "v": t(B, Nk, G, D), "dout": t(B, Nq, H, D), "bias": None, "ks": None, "qs": None}
    if density is not None:
        bm = np.where(rng.random((1 if shared_mask else B, Nq, Nk)) < density, 0.0, -1e9)
        if soft:
            bm = np.where(bm == 0.0, rng.normal(0, 2, bm.shape), bm)
        if Nq > 2:
            bm[:, 1] = -1e9                                              # a row that the mask leaves empty
        c["bias"] = torch.tensor(bm, dtype=torch.float32, device=dev)
    if sizes:
        ks = rng.integers(0, Nk + 1, B)
        ks[0] = Nk
        if B > 2:
            ks[1], ks[2] = 0, 1
        c["ks"] = torch.tensor(ks, dtype=torch.int32, device=dev)
        c["qs"] = c["ks"] if Nq == Nk else torch.tensor(rng.integers(0, Nq + 1, B), dtype=torch.int32, device=dev)
    return c


def _np(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _run(c, grad=True, scale=None):
    from gat_amd import ops
    leaves = [c[n].detach().requires_grad_(grad) for n in ("q", "k", "v")]
    out = ops.dot_attention(*leaves, c["bias"], key_sizes=c["ks"], query_sizes=c["qs"], scale=scale)
    res = {"out": out.detach()}
    if grad:
        res.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, c["dout"])))
    return res


def _check(c, dtype, grad=True, scale=None, what=""):
    got = _run(c, grad, scale)
    ref = attn_ref.attention(_np(c["q"]), _np(c["k"]), _np(c["v"]), _np(c["bias"]), _np(c["ks"]), _np(c["qs"]), scale,
                             _np(c["dout"]) if grad else None, dtype == "bf16")
    for n, (value, bound) in ref.items():
        assert got[n].dtype == TYPES[dtype]
        within(got[n].double().cpu().numpy(), value, bound, "%s %s" % (what, n))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [8, 16, 20, 32, 64, 100, 128])
def test_every_width(D, dtype):
    _check(_case(2, 70, 70, 4, 2, D, dtype, density=0.3, seed=D), dtype, what="D=%d" % D)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 3, 7, 13])
def test_widths_that_no_vector_divides(D, dtype):
    _check(_case(2, 33, 33, 2, 2, D, dtype, density=0.5, seed=D), dtype, what="D=%d" % D)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 2), (2, 1), (1, 64), (1, 65), (15, 17), (16, 16), (17, 63), (63, 64), (64, 63), (65, 65), (127, 129),
                                   (128, 128), (129, 127), (1, 300), (300, 1), (246, 246), (264, 264)])
def test_lengths(Nq, Nk, dtype):
    _check(_case(2, Nq, Nk, 2, 2, 16, dtype, density=0.4 if Nk > 8 else None, seed=Nq + Nk), dtype, what="%dx%d" % (Nq, Nk))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (6, 6), (6, 2), (8, 2), (12, 4), (5, 5), (16, 1)])
def test_head_layouts(H, G, dtype):
    _check(_case(2, 37, 50, H, G, 32, dtype, density=0.3, seed=H), dtype, what="%d/%d" % (H, G))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shared,soft", [(False, True), (True, False), (True, True)])
def test_masks(shared, soft, dtype):
    _check(_case(3, 90, 90, 4, 4, 16, dtype, density=0.1, shared_mask=shared, soft=soft), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Nq,Nk,density", [(70, 70, None), (70, 70, 0.3), (5, 130, None), (130, 70, 0.5)])
def test_padded_graphs(Nq, Nk, density, dtype):
    _check(_case(5, Nq, Nk, 4, 2, 24, dtype, density=density, sizes=True, seed=Nk), dtype)


# masks of 512 x 512 entries and more with at most one in 16 (fp32) or 64 (bf16) attended: walked entry by entry
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Nq,Nk,H,G", [(8, 600, 600, 4, 4), (8, 4200, 90, 2, 1), (12, 513, 700, 4, 2), (16, 520, 520, 6, 2), (32, 512, 512, 2, 2), (40, 700, 512, 2, 1),
                                         (64, 600, 600, 3, 3), (100, 520, 530, 2, 1), (128, 512, 600, 2, 2)])
@pytest.mark.parametrize("density,soft,sizes,shared", [(0.004, False, False, False), (0.002, True, True, False), (0.01, True, False, True)])
def test_masks_of_few_entries(D, Nq, Nk, H, G, density, soft, sizes, shared, dtype):
    _check(_case(3 if sizes else 2, Nq, Nk, H, G, D, dtype, density=density, soft=soft, sizes=sizes, shared_mask=shared, seed=D), dtype, what="%d wide" % D)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("entries", [0, 1, 4095, 4096, 4097, 16383, 16384, 16385, 512 * 512])
def test_few_entries_or_many(entries, dtype):
    """On both sides of one entry in 64 (bf16) and in 16 (fp32), two graphs of different kinds in one batch."""
    c = _case(2, 512, 512, 2, 2, 16, dtype, seed=entries)
    rng = np.random.default_rng(entries)
    bm = np.full((2, 512 * 512), -1e9)
    bm[0, rng.permutation(512 * 512)[:entries]] = 0.0
    bm[1, rng.permutation(512 * 512)[:20000]] = 0.0
    c["bias"] = torch.tensor(bm.reshape(2, 512, 512), dtype=torch.float32, device="cuda:0")
    _check(c, dtype)
    c["q"], c["dout"] = c["q"][:, :3].contiguous(), c["dout"][:, :3].contiguous()
    c["bias"] = c["bias"][:, :3].contiguous()
    _check(c, dtype)


def test_few_entries_of_few_rows():
    """One query on 262144 keys with gradients: the mask is large though it has one row."""
    _check(_case(1, 1, 1 << 18, 2, 1, 8, "f32", density=0.001, seed=1), "f32")
    _check(_case(1, 1, 1 << 18, 2, 1, 8, "f32", density=0.001, seed=1), "f32", grad=False)


def test_few_entries_captured_twice_the_same_and_not_finite_where_masked():
    c = _case(2, 600, 600, 2, 2, 16, "f32", density=0.003, seed=2)
    never = (c["bias"] < -1e8).all(1)[0]                                 # keys that no query of the first graph attends
    want = _run(c)
    for n in ("k", "v"):
        c[n] = c[n].clone()
        c[n][0, never] = float("nan")
    again = _run(c)
    assert torch.equal(want["out"], again["out"]) and torch.equal(want["dq"], again["dq"]) and torch.equal(want["dv"][:, ~never], again["dv"][:, ~never])


# many rows of fp32 wider than 16: computed as three parts (for the gradients from 97 rows and keys on, 193 above 64 wide; alone from 257 and 769)
@pytest.mark.parametrize("D,Nq,Nk,H,G", [(20, 97, 97, 2, 2), (32, 97, 130, 2, 2), (32, 50, 200, 4, 2), (40, 129, 97, 2, 1), (64, 200, 128, 2, 2), (64, 192, 97, 3, 1),
                                         (96, 193, 193, 1, 1), (100, 97, 257, 2, 1), (128, 260, 193, 1, 1), (128, 321, 200, 2, 2)])
@pytest.mark.parametrize("density,soft,sizes", [(None, False, False), (0.1, False, False), (0.5, True, True), (0.02, False, True)])
def test_rows_in_parts(D, Nq, Nk, H, G, density, soft, sizes):
    _check(_case(3, Nq, Nk, H, G, D, "f32", density=density, soft=soft, sizes=sizes, seed=D + Nq), "f32", what="%d wide" % D)


@pytest.mark.parametrize("D,N", [(32, 256), (32, 257), (64, 300), (128, 768), (128, 769)])
@pytest.mark.parametrize("density", [None, 0.1])
def test_rows_in_parts_forward_alone(D, N, density):
    _check(_case(1, N, N, 2, 1, D, "f32", density=density, seed=N), "f32", grad=False)


def test_rows_in_parts_keys_split():
    _check(_case(1, 300, 5000, 2, 2, 64, "f32", seed=4), "f32", grad=False)
    _check(_case(2, 97, 2100, 1, 1, 32, "f32", sizes=True, seed=4), "f32")


@pytest.mark.parametrize("scale", [0.0, -0.5, 30.0])
def test_rows_in_parts_scale(scale):
    _check(_case(1, 100, 100, 2, 2, 32, "f32", density=0.3, seed=6), "f32", scale=scale)


def test_rows_in_parts_keep_a_large_range():
    c = _case(1, 100, 120, 1, 1, 32, "f32", seed=5)
    c["q"] *= 1e-12
    c["k"] *= 1e12
    c["v"] *= torch.logspace(-20, 20, 32, device="cuda:0")
    c["dout"] *= torch.logspace(20, -20, 32, device="cuda:0")
    _check(c, "f32")


def test_padding_of_rows_in_parts_is_not_used():
    c = _case(4, 130, 130, 2, 2, 32, "f32", sizes=True, seed=3)
    want = _run(c)
    for n in ("q", "k", "v", "dout"):
        x = c[n].clone()
        for b in range(4):
            x[b, int(c["ks"][b]):] = float("nan")
        c[n] = x
    got = _run(c)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_behind_the_sizes_are_not_read(dtype):
    c = _case(4, 70, 70, 2, 2, 16, dtype, sizes=True, seed=3)
    want = _run(c)
    for n in ("q", "k", "v", "dout"):
        x = c[n].clone()
        for b in range(4):
            x[b, int(c["ks"][b]):] = float("nan")
        c[n] = x
    got = _run(c)
    for n in want:
        assert torch.equal(got[n], want[n]), n
        for b in range(4):
            assert (got[n][b, int(c["ks"][b]):] == 0).all()


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e9, float("nan")])
def test_lowest_masks_and_empty_rows(low):
    c = _case(2, 40, 40, 2, 2, 8, "f32", density=0.2, seed=5)
    want = _run(c)
    c["bias"] = torch.where(c["bias"] < -1e8, torch.full_like(c["bias"], low), c["bias"])
    got = _run(c)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert (got["out"][:, 1] == 0).all() and (got["dq"][:, 1] == 0).all()


def test_nothing_attended_at_all():
    c = _case(2, 20, 30, 2, 1, 16, "f32", density=0.5)
    c["bias"].fill_(-1e9)
    for n, x in _run(c).items():
        assert (x == 0).all(), n


def test_nan_and_inf_in_an_attended_row_stay_visible():
    c = _case(1, 20, 20, 1, 1, 8, "f32")
    c["q"][0, 3] = float("nan")
    out = _run(c, grad=False)["out"]
    assert out[0, 3].isnan().all() and out[0, 4:].isfinite().all() and out[0, :3].isfinite().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,Nk,H,G,D", [(1, 1, 512, 1, 1, 64), (1, 1, 5000, 8, 2, 64), (2, 3, 3001, 4, 1, 128), (1, 40, 2000, 2, 2, 8), (3, 1, 777, 6, 3, 100),
                                           (1, 1, 70001, 4, 4, 16)])
def test_few_rows_on_many_keys(B, Nq, Nk, H, G, D, dtype):
    """Split over the keys; also with ranges that no key of a graph falls into, and gradients behind it."""
    from gat_amd import _lib
    assert Nk < 2000 or _lib.lib.gatmi_dot_attn_fwd_ws_floats(B, Nq, Nk, H, G, (D + 7) // 8 * 8) > 0
    c = _case(B, Nq, Nk, H, G, D, dtype, seed=Nk)
    _check(c, dtype, grad=Nk <= 5000)
    c["ks"] = torch.tensor([(Nk, 5, 0)[b % 3] for b in range(B)][::-1], dtype=torch.int32, device="cuda:0")
    _check(c, dtype, grad=Nk <= 5000)


@pytest.mark.parametrize("scale", [0.0, 3.0, -0.5])
def test_scale(scale):
    _check(_case(1, 50, 50, 2, 2, 16, "f32", density=0.5), "f32", scale=scale)


def test_large_logits():
    c = _case(1, 60, 60, 2, 2, 16, "f32")
    c["q"] *= 30
    _check(c, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows_equal_contiguous_ones(dtype):
    """Slices of one projection's output, a transposed layout, an offset that is not 16-byte aligned, an expanded gradient."""
    from gat_amd import ops
    dev = torch.device("cuda:0")
    B, N, H, D = 2, 45, 4, 16
    g = torch.Generator(device=dev).manual_seed(1)
    rows = torch.randn((B, N, 3 * H, D), device=dev, generator=g).to(TYPES[dtype])
    q, k, v = rows[:, :, :H], rows[:, :, H:2 * H], rows[:, :, 2 * H:]
    want = ops.dot_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(ops.dot_attention(q, k, v), want)
    turned = lambda x: x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(ops.dot_attention(turned(q), k, turned(v)), want)
    odd = torch.empty(B * N * H * D + 1, dtype=TYPES[dtype], device=dev)[1:].view(B, N, H, D)
    odd.copy_(q)
    assert odd.data_ptr() % 16 != 0
    assert torch.equal(ops.dot_attention(odd, k, v), want)
    leaf = q.contiguous().requires_grad_()
    a = torch.autograd.grad(ops.dot_attention(leaf, k, v).sum(), leaf)[0]                  # gradient: one value expanded
    b = torch.autograd.grad(ops.dot_attention(leaf, k, v), leaf, torch.ones_like(leaf))[0]
    assert torch.equal(a, b)
    wide = torch.full((B, N, 2 * N), -1e9, device=dev)
    wide[:, :, :N] = torch.where(torch.rand((B, N, N), device=dev, generator=g) < 0.3, 0.0, -1e9)
    assert torch.equal(ops.dot_attention(q, k, v, wide[:, :, :N]), ops.dot_attention(q, k, v, wide[:, :, :N].contiguous()))
    mask_t = wide[:, :, :N].transpose(1, 2)
    assert torch.equal(ops.dot_attention(q, k, v, mask_t), ops.dot_attention(q, k, v, mask_t.contiguous()))


def test_empty_shapes():
    from gat_amd import ops
    dev = torch.device("cuda:0")
    z = lambda *s: torch.zeros(s, device=dev, requires_grad=True)
    for B, Nq, Nk in ((0, 4, 4), (2, 0, 4), (2, 4, 0), (2, 0, 0)):
        q, k, v = z(B, Nq, 2, 8), z(B, Nk, 2, 8), z(B, Nk, 2, 8)
        out = ops.dot_attention(q, k, v)
        assert out.shape == q.shape and (out == 0).all()
        for x, g in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
            assert g.shape == x.shape and (g == 0).all()


def test_twice_the_same_bits_and_on_another_stream():
    c = _case(3, 100, 100, 6, 2, 64, "bf16", density=0.2)
    want = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    torch.cuda.current_stream().wait_stream(side)
    again = _run(c)
    for n in want:
        assert torch.equal(want[n], got[n]) and torch.equal(want[n], again[n]), n


def test_captured_forward_and_backward():
    """Replays with new inputs, eager work of the same sizes and synchronisations between them."""
    from gat_amd import graphs, ops
    c = _case(2, 90, 90, 4, 2, 32, "f32", density=0.2)
    q, k, v = (c[n].clone().requires_grad_() for n in ("q", "k", "v"))

    def step():
        out = ops.dot_attention(q, k, v, c["bias"])
        return (out, *torch.autograd.grad(out, (q, k, v), c["dout"]))

    replay, res = graphs.capture(step, fresh_dropout=False)
    one_query = _case(1, 1, 3000, 4, 2, 32, "f32", seed=9)                       # split over the keys: a workspace of its own
    replay_one, res_one = graphs.capture(lambda: ops.dot_attention(one_query["q"], one_query["k"], one_query["v"]), fresh_dropout=False)
    for seed in range(4):
        n = _case(2, 90, 90, 4, 2, 32, "f32", density=0.2, seed=seed)
        with torch.no_grad():
            for a, b in ((q, n["q"]), (k, n["k"]), (v, n["v"])):
                a.copy_(b)
            c["bias"].copy_(n["bias"])
            c["dout"].copy_(n["dout"])
            one_query["q"].copy_(_case(1, 1, 3000, 4, 2, 32, "f32", seed=20 + seed)["q"])
        replay()
        replay_one()
        torch.cuda.synchronize()
        want = _run(n)
        for got, name in zip(res, ("out", "dq", "dk", "dv")):
            assert torch.equal(got, want[name]), (seed, name)
        assert torch.equal(res_one, ops.dot_attention(one_query["q"], one_query["k"], one_query["v"]))


def test_captured_masks_that_change_between_replays():
    """One graph whose mask has few entries in one replay and many in the next, with fp32 rows in parts; eager work between."""
    from gat_amd import graphs, ops
    c = _case(2, 520, 520, 2, 2, 64, "f32", density=0.01)
    q, k, v = (c[n].clone().requires_grad_() for n in ("q", "k", "v"))
    e = _case(2, 520, 520, 2, 2, 64, "bf16", density=0.01)
    eq, ek, ev = (e[n].clone().requires_grad_() for n in ("q", "k", "v"))

    def step():
        out = ops.dot_attention(q, k, v, c["bias"])
        out16 = ops.dot_attention(eq, ek, ev, e["bias"])
        return (out, *torch.autograd.grad(out, (q, k, v), c["dout"]), out16, *torch.autograd.grad(out16, (eq, ek, ev), e["dout"]))

    replay, res = graphs.capture(step, fresh_dropout=False)
    for seed, density in enumerate((0.01, 0.3, 0.002, 1.0, 0.05)):
        n, m = (_case(2, 520, 520, 2, 2, 64, dt, density=density, seed=seed) for dt in ("f32", "bf16"))
        with torch.no_grad():
            for to, frm, leaves in ((c, n, (q, k, v)), (e, m, (eq, ek, ev))):
                for a, b in zip(leaves, ("q", "k", "v")):
                    a.copy_(frm[b])
                to["bias"].copy_(frm["bias"])
                to["dout"].copy_(frm["dout"])
        replay()
        torch.cuda.synchronize()
        want = [_run(n)[x] for x in ("out", "dq", "dk", "dv")] + [_run(m)[x] for x in ("out", "dq", "dk", "dv")]
        for i, (got, w) in enumerate(zip(res, want)):
            assert torch.equal(got, w), (density, i)


def test_gradient_against_differences():
    """d/dt of <out(x + t d), dout> from outputs at t = +-h: truncation is h^2 times a third derivative of order 1, rounding 1e-6 / h."""
    from gat_amd import ops
    c = _case(2, 30, 30, 4, 2, 16, "f32", density=0.4, soft=True, seed=11)
    got = _run(c)
    rng = np.random.default_rng(1)
    h = 1e-2
    for n, g in (("q", "dq"), ("k", "dk"), ("v", "dv")):
        d = torch.tensor(rng.normal(0, 1, c[n].shape), dtype=torch.float32, device="cuda:0")
        d /= d.norm()

        def f(t):
            x = {m: c[m] + t * d if m == n else c[m] for m in ("q", "k", "v")}
            return (ops.dot_attention(x["q"], x["k"], x["v"], c["bias"]).double() * c["dout"].double()).sum().item()

        slope = (f(h) - f(-h)) / (2 * h)
        assert abs(slope - (got[g].double() * d.double()).sum().item()) < 1e-3 * got[g].norm().item() + 1e-3


def test_wide_batch_and_long_rows():
    """More graphs than a grid dimension of 65535 holds; offsets that pass 2^31 elements."""
    from gat_amd import ops
    dev = torch.device("cuda:0")
    q = torch.randn((70000, 2, 1, 8), device=dev)
    out = ops.dot_attention(q, q, q)
    for b in (0, 1, 65535, 65536, 69999):
        value, bound = attn_ref.attention(*(_np(q[b:b + 1]),) * 3)["out"]
        within(_np(out[b:b + 1]), value, bound, "graph %d" % b)
    k = torch.zeros((1, 17_000_000, 1, 128), dtype=torch.bfloat16, device=dev)              # 2.2e9 elements
    k[0, -1] = 1.0
    v = torch.zeros_like(k)
    v[0, -1] = 2.0
    one = torch.full((1, 1, 1, 128), 30.0, dtype=torch.bfloat16, device=dev)                # the last key's score is 339, all others are 0
    assert (ops.dot_attention(one, k, v) == 2.0).all()


@pytest.mark.parametrize("seed", range(12))
def test_random_shapes(seed):
    rng = np.random.default_rng(1000 + seed)
    G = int(rng.choice([1, 2, 3, 4]))
    H = G * int(rng.choice([1, 1, 2, 3]))
    same = rng.random() < 0.5
    Nq = int(rng.integers(1, 300))
    Nk = Nq if same else int(rng.integers(1, 400))
    dtype = str(rng.choice(["f32", "bf16"]))
    c = _case(int(rng.integers(1, 5)), Nq, Nk, H, G, int(rng.integers(1, 129)), dtype, density=float(rng.choice([0.05, 0.5, 1.0])) if rng.random() < 0.7 else None,
              sizes=bool(rng.random() < 0.5), soft=bool(rng.random() < 0.3), seed=seed)
    _check(c, dtype, what="seed %d: %s" % (seed, [tuple(c[n].shape) for n in ("q", "k")]))

"""GPU parity of ops.newton_schulz against its 64-bit form, and of the optimizer that calls it.

Bounds.  Shorter side up to 64 and more than 128 long: formed in fp64, so the result is off by its own rounding (2^-24, bf16 2^-8, relative) and what fp64 rounding becomes after
five steps: an error in the directions of small singular values grows by a = 3.4445 a step on either side of Q, 485^2 n 2^-53 = 2e-9 of
the largest entry.  All others: a step rounds its three products and their operands to 2^-22 or better, about four such errors of the size of X, and a
later step multiplies what falls into small singular directions by a: (a^4 + a^3 + a^2 + a + 1) * 4 * 2^-22 = 2e-4 of |X|_F at the most."""
import numpy as np
import pytest
import torch

from tests import attn_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
WIDE = 2e-4


def _matrices(kind, b, m, n, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "normal":
        return rng.normal(0, 1e-3, (b, m, n))
    if kind == "low_rank":
        r = max(1, min(m, n) // 8)
        return rng.normal(0, 1, (b, m, r)) @ rng.normal(0, 1, (b, r, n)) + 1e-2 * rng.normal(0, 1, (b, m, n))
    if kind == "rank_one":
        return rng.normal(0, 1, (b, m, 1)) @ rng.normal(0, 1, (b, 1, n))
    x = np.zeros((b, m, n))
    x[:, 0, 0] = 3.0
    return x


def _check(x, dtype, steps=5, coefficients=None, what=""):
    from gat_amd import ops
    kw = {} if coefficients is None else {"coefficients": coefficients}
    xt = torch.tensor(x, dtype=torch.float32).to(TYPES[dtype]).cuda()
    got = ops.newton_schulz(xt, steps=steps, **kw)
    assert got.shape == xt.shape and got.dtype == xt.dtype
    flat, gf = xt.double().cpu().numpy().reshape(-1, *xt.shape[-2:]), got.double().cpu().numpy().reshape(-1, *xt.shape[-2:])
    last = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    for i, (a, g) in enumerate(zip(flat, gf)):
        ref = attn_ref.newton_schulz(a, steps, **kw)
        if min(a.shape) <= 64 and max(a.shape) > 128:
            attn_ref.within(g, ref, last * 1.01 * abs(ref) + 2e-9 * abs(ref).max(), "%s matrix %d" % (what, i))
        else:
            err, norm = np.linalg.norm(g - ref), np.linalg.norm(ref)
            assert err <= (WIDE + last) * norm, "%s matrix %d: off by %.3g of %.3g" % (what, i, err, norm)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 9), (9, 1), (2, 3), (15, 17), (16, 16), (17, 15), (33, 64), (64, 64), (64, 65), (64, 128), (128, 3), (31, 129), (48, 200), (1433, 8), (8, 1433), (64, 1000),
                                 (1000, 63), (5000, 31)])
def test_narrow_shapes(m, n, dtype):
    _check(_matrices("normal", 3, m, n, seed=m + n), dtype, what="%dx%d" % (m, n))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(65, 65), (65, 64 * 5), (300, 70), (100, 129), (128, 128), (129, 127), (256, 384), (384, 250), (512, 512)])
def test_wide_shapes(m, n, dtype):
    _check(_matrices("normal", 2, m, n, seed=m + n), dtype, what="%dx%d" % (m, n))


# symmetric products of a depth of 2048 and more are computed in pieces
@pytest.mark.parametrize("b,m,n,dtype", [(1, 70, 1921, "f32"), (2, 1920, 128, "f32"), (3, 66, 2048, "bf16"), (1, 2300, 200, "f32"), (2, 130, 5000, "bf16"), (1, 90, 40000, "f32"),
                                         (1, 1930, 2050, "f32")])
def test_deep_products(b, m, n, dtype):
    _check(_matrices("normal", b, m, n, seed=m + n), dtype, what="%dx%d" % (m, n))


def test_deep_products_of_many_matrices_and_of_one():
    from gat_amd import ops
    x = torch.tensor(_matrices("normal", 26, 400, 2000, seed=1), dtype=torch.float32).cuda()      # 260 tiles: a block each; alone: pieces
    many = ops.newton_schulz(x)
    for i in (0, 25):
        one = ops.newton_schulz(x[i])
        assert (many[i] - one).norm() <= 2 * (WIDE + 2.0 ** -24) * one.norm()
        assert torch.equal(one, ops.newton_schulz(x[i]))


@pytest.mark.parametrize("kind", ["low_rank", "rank_one", "one_entry"])
@pytest.mark.parametrize("m,n", [(20, 30), (64, 64), (100, 40), (50, 300), (1433, 8), (100, 150), (200, 130)])
def test_spectra(kind, m, n):
    _check(_matrices(kind, 2, m, n, seed=1), "f32", what="%s %dx%d" % (kind, m, n))


@pytest.mark.parametrize("steps,abc", [(1, None), (2, None), (8, (1.5, -0.5, 0.0)), (10, (2.0, -1.5, 0.5)), (3, (3.0, -3.2, 1.2))])
@pytest.mark.parametrize("m,n", [(30, 20), (30, 220), (70, 90)])
def test_steps_and_coefficients(m, n, steps, abc):
    _check(_matrices("normal", 2, m, n, seed=2), "f32", steps, abc)


@pytest.mark.parametrize("m,n", [(10, 12), (70, 60), (20, 200), (80, 90)])
@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-12, 1e12, 1e30])
def test_scale_of_the_input(m, n, size):
    """Zero and tiny inputs stay small (eps), large ones do not overflow: squares are summed in fp64."""
    _check(_matrices("normal", 1, m, n, seed=3) * (size * 1e3), "f32")


@pytest.mark.parametrize("m,n", [(10, 12), (20, 200), (80, 90)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_finite_input_stays_visible_and_in_its_matrix(m, n, bad):
    from gat_amd import ops
    x = torch.tensor(_matrices("normal", 3, m, n), dtype=torch.float32, device="cuda:0")
    want = ops.newton_schulz(x)
    x[1, 2, 3] = bad
    got = ops.newton_schulz(x)
    assert got[1].isnan().any() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_batches_strides_and_shapes():
    from gat_amd import ops
    dev = torch.device("cuda:0")
    w = torch.randn((40, 6, 24), device=dev)
    turned = w.permute(1, 0, 2)                                                # one 40 x 24 matrix per head of a [F, H, D] kernel
    assert torch.equal(ops.newton_schulz(turned), ops.newton_schulz(turned.contiguous()))
    assert torch.equal(ops.newton_schulz(w[:, 0]), ops.newton_schulz(turned.contiguous())[0])
    big = torch.randn((2, 3, 100, 90), device=dev)
    one = ops.newton_schulz(big)
    assert one.shape == big.shape and torch.equal(one[1, 2], ops.newton_schulz(big[1, 2]))
    cut = big[..., :80]
    assert torch.equal(ops.newton_schulz(cut), ops.newton_schulz(cut.contiguous()))
    sq = torch.randn((2, 90, 100), device=dev)
    assert torch.equal(ops.newton_schulz(sq.transpose(1, 2)), ops.newton_schulz(sq.transpose(1, 2).contiguous()))
    many = torch.randn((40000, 3, 2), device=dev)
    assert torch.equal(ops.newton_schulz(many)[[0, 32767, 32768, 39999]], ops.newton_schulz(many[[0, 32767, 32768, 39999]]))
    for shape in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        assert ops.newton_schulz(torch.empty(shape, device=dev)).shape == shape


@pytest.mark.parametrize("m,n", [(40, 24), (200, 24), (90, 130)])
def test_streams_and_captured(m, n):
    from gat_amd import graphs, ops
    x = torch.randn((2, m, n), device="cuda:0")
    want = ops.newton_schulz(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.newton_schulz(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    replay, res = graphs.capture(lambda: ops.newton_schulz(x), fresh_dropout=False)
    for _ in range(4):
        x.normal_()
        replay()
        torch.cuda.synchronize()
        assert torch.equal(res, ops.newton_schulz(x))


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_against_its_formula(nesterov):
    """Two steps on a [F, H, D] kernel, an [H, F, D] kernel and an [out, in] weight."""
    from gat_amd.models import Muon
    dev = torch.device("cuda:0")
    rng = np.random.default_rng(8)
    start = {1: rng.normal(0, 1, (30, 4, 12)), 0: rng.normal(0, 1, (3, 16, 40)), None: rng.normal(0, 1, (20, 70))}
    ps = {a: torch.nn.Parameter(torch.tensor(v, dtype=torch.float32, device=dev)) for a, v in start.items()}
    opt = Muon([(p, a) for a, p in ps.items()], lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.5)
    ref, mom = {a: v.copy() for a, v in start.items()}, {a: 0.0 for a in start}
    for _ in range(2):
        for a, p in ps.items():
            g = rng.normal(0, 1, p.shape).astype(np.float32)
            p.grad = torch.tensor(g, device=dev)
            mom[a] = 0.9 * mom[a] + g
            u = g + 0.9 * mom[a] if nesterov else mom[a]
            ref[a] = ref[a] * (1 - 0.1 * 0.5)
            if a is None:
                ref[a] -= 0.1 * max(1.0, u.shape[0] / u.shape[1]) ** 0.5 * attn_ref.newton_schulz(u)
            else:
                for h in range(u.shape[a]):
                    uh = np.take(u, h, a)
                    at = [slice(None)] * 3
                    at[a] = h
                    ref[a][tuple(at)] -= 0.1 * max(1.0, uh.shape[1] / uh.shape[0]) ** 0.5 * attn_ref.newton_schulz(uh)
        opt.step()
    for a, p in ps.items():
        np.testing.assert_allclose(p.detach().cpu().numpy(), ref[a], rtol=0, atol=2e-5)      # two steps of 0.1 with entries below 1.3, WIDE relative, fp32 sums

"""GPU tests of calls of ops.dot_attention, ops.embedding and ops.newton_schulz as documented but off the common path."""
import numpy as np
import pytest
import torch

from tests import attn_ref

pytestmark = pytest.mark.gpu


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_calls_compute_what_eager_ones_do():
    from gat_amd import ops
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    q, k, table, x = r(2, 40, 4, 13), r(2, 50, 2, 13), r(9, 24), r(3, 70, 20)
    mask = torch.where(r(2, 40, 50) > 0.5, 0.0, -1e9)
    ids = torch.randint(-1, 9, (2, 7), device=dev, generator=g)
    sizes = torch.tensor([50, 3], device=dev, dtype=torch.int32)

    def call(q, k, table, x):
        return ops.dot_attention(q, k, k, mask, key_sizes=sizes), ops.embedding(ids, table, 3.0), ops.newton_schulz(x)

    traced = torch.jit.trace(call, (q, k, table, x), check_trace=False)
    for _ in range(3):
        args = [torch.randn(t.shape, device=dev, generator=g) for t in (q, k, table, x)]
        for a, b in zip(traced(*args), call(*args)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_strides_of_dimensions_of_size_one(dtype):
    """One query of one graph out of a wider row, one head, one node: as their contiguous copies, gradients included."""
    from gat_amd import ops
    dev = torch.device("cuda:0")
    base = torch.randn(4096, device=dev).to(dtype)
    v = lambda *a: torch.as_strided(base, *a)
    k = torch.randn((1, 30, 1, 8), device=dev).to(dtype)
    cases = [(base[:9].reshape(1, 1, 9)[..., :8].unsqueeze(2), k), (v((1, 5, 1, 8), (77, 16, 3, 1)), v((1, 30, 1, 8), (3, 8, 5, 1))), (v((3, 1, 2, 8), (16, 3, 8, 1)), v((3, 20, 1, 8), (160, 8, 7, 1))),
             (v((2, 5, 1, 8), (40, 8, 5, 1), 1), v((2, 6, 1, 8), (48, 8, 1, 1)))]
    for q, k in cases:
        got, want = [], []
        for res, leaves in ((got, (q, k)), (want, (q.contiguous().clone(), k.contiguous().clone()))):
            q_, k_ = (t.detach().requires_grad_() for t in leaves)
            out = ops.dot_attention(q_, k_, k_)
            dout = torch.as_strided(base, out.shape, (out.stride(0), out.stride(1), 3 if out.shape[2] == 1 else out.stride(2), 1), 64)
            res += [ops.dot_attention(*leaves, leaves[1]), out, *torch.autograd.grad(out, (q_, k_), dout)]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [13, 16, 100])
@pytest.mark.parametrize("turned,back", [((0, 2, 1, 3), (0, 2, 1, 3)), ((0, 2, 3, 1), (0, 3, 1, 2)), ((3, 0, 1, 2), (1, 2, 3, 0)), ((0, 1, 3, 2), (0, 1, 3, 2))])
def test_rows_and_gradients_in_any_order_of_dimensions(turned, back, D, dtype):
    """Rows, and the gradient of a result that is read in another order, as their contiguous copies."""
    from gat_amd import ops
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(D)
    q, k, dout = (torch.randn((2, 45, h, D), device=dev, generator=g).to(dtype) for h in (4, 2, 4))
    got, want = [], []
    for res, other in ((got, lambda t: t.permute(*turned).contiguous().permute(*back)), (want, lambda t: t)):
        q_, k_ = (other(t).detach().requires_grad_() for t in (q, k))
        out = ops.dot_attention(q_, k_, k_)
        read = out.permute(*turned).contiguous() if res is got else out
        res += [ops.dot_attention(other(q), other(k), other(k)), out, *torch.autograd.grad(read, (q_, k_), dout.permute(*turned).contiguous() if res is got else dout)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_dot_heads_drop_their_input_in_training_only():
    from gat_amd import layers
    dev = torch.device("cuda:0")
    store, x = layers.VariableStore(), torch.randn((2, 30, 16), device=dev)

    def call(*args, **kw):
        store.begin()
        with layers.variable_scope(store):
            return layers.dot_attn_heads(x, 8, None, "elu", 2, "concat", *args, **kw)
    want = call()
    assert torch.equal(call(0.5, 0.6, False, False), want) and torch.equal(call(0.5, training=False), want)
    torch.manual_seed(1)
    a = call(0.5)
    torch.manual_seed(1)
    dropped = torch.nn.functional.dropout(x, 0.5, True)
    m = store.layers[0]
    assert not torch.equal(a, want) and torch.equal(a, m(dropped, None))
    m.eval()
    assert torch.equal(m(x, None, "elu", "concat", 0.5, 0.6), want)
    sizes = torch.tensor([30, 7], device=dev, dtype=torch.int32)
    assert torch.equal(call(sizes=sizes), m(x, None, sizes=sizes))


def test_masks_of_few_entries_captured_with_rows_that_are_not_finite_where_nothing_attends():
    """The walk over single entries does not touch rows that no query attends: replayed twice, dk compared too."""
    from gat_amd import graphs, ops
    from tests.test_dot_attention_gpu import _case, _run
    c = _case(2, 600, 600, 2, 2, 16, "f32", density=0.003, seed=2)
    never = (c["bias"] < -1e8).all(1)[0]                                 # keys of the first graph that no query attends
    assert never.any() and not never.all()
    want = _run(c)
    q, k, v = (c[n].clone().requires_grad_() for n in ("q", "k", "v"))
    with torch.no_grad():
        k[0, never], v[0, never] = float("nan"), float("inf")

    def step():
        out = ops.dot_attention(q, k, v, c["bias"])
        return (out, *torch.autograd.grad(out, (q, k, v), c["dout"]))

    replay, res = graphs.capture(step, fresh_dropout=False)
    for _ in range(2):
        for t in res:
            t.fill_(7.0)
        replay()
        torch.cuda.synchronize()
        for got, n in zip(res, ("out", "dq", "dk", "dv")):
            assert torch.equal(got, want[n]), n
        _run(c)
    assert (res[2][0, never] == 0).all() and (res[3][0, never] == 0).all()


def test_muon_on_bf16_parameters_eager_and_captured():
    """Three steps against the formula: the momentum in fp32, each step's weights rounded to bf16 twice (decay, update), 2^-8 of what they are."""
    from gat_amd import graphs
    from gat_amd.models import Muon
    dev = torch.device("cuda:0")
    rng = np.random.default_rng(3)
    bf = lambda a: torch.tensor(a, dtype=torch.float32).to(torch.bfloat16)
    start = [bf(rng.normal(0, 1, (20, 70))), bf(rng.normal(0, 1, (30, 4, 12)))]
    grads = [[bf(rng.normal(0, 1, t.shape)).to(dev) for t in start] for _ in range(3)]

    def make():
        ps = [torch.nn.Parameter(t.to(dev)) for t in start]
        return ps, Muon([(ps[0], None), (ps[1], 1)], lr=0.1, momentum=0.9, weight_decay=0.5)

    ps, opt = make()
    ref, mom, slack = [t.double().numpy() for t in start], [0.0, 0.0], [0.0, 0.0]
    for gs in grads:
        for i, (p, g) in enumerate(zip(ps, gs)):
            p.grad = g.clone()
            mom[i] = 0.9 * mom[i] + g.double().cpu().numpy()
            u = g.double().cpu().numpy() + 0.9 * mom[i]
            rate = lambda m: 0.1 * max(1.0, m.shape[0] / m.shape[1]) ** 0.5 * attn_ref.newton_schulz(m)
            before = abs(ref[i])
            ref[i] = ref[i] * 0.95 - (rate(u) if i == 0 else np.stack([rate(u[:, h].T).T for h in range(4)], 1))
            slack[i] = 0.95 * slack[i] + 2.0 ** -8 * (before + slack[i] + abs(ref[i])) * 1.01 + 1e-4
        opt.step()
    for p, r, e in zip(ps, ref, slack):
        assert p.dtype == torch.bfloat16
        attn_ref.within(p.detach().double().cpu().numpy(), r, e, "weights")
    qs, other = make()
    for q, g in zip(qs, grads[0]):
        q.grad = g.clone()
    other.step()                                                         # the state is made eagerly
    replay, _ = graphs.capture(other.step, warmup=0, fresh_dropout=False)
    for gs in grads[1:]:
        for q, g in zip(qs, gs):
            q.grad.copy_(g)
        replay()
        torch.cuda.synchronize()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)


def test_muon_captured_before_its_first_step_is_refused():
    from gat_amd.models import Muon
    p = torch.nn.Parameter(torch.randn(8, 4, device="cuda:0"))
    p.grad = torch.randn_like(p)
    opt, graph = Muon([p]), torch.cuda.CUDAGraph()
    before, x = p.detach().clone(), torch.zeros(4, device="cuda:0")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, before) and (x == 1.0).all()
    opt.step()
    assert not torch.equal(p, before)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [8, 16, 32, 64, 97, 128])
@pytest.mark.parametrize("Nq,Nk,H,G", [(1400, 190, 8, 1), (190, 1400, 8, 8)])
def test_soft_masks_of_few_entries_on_more_rows_than_run_at_once(Nq, Nk, H, G, D, dtype):
    """Biases other than 0, and so many queries, or keys, that every SIMD has several waves of the walk over single entries."""
    from tests.test_dot_attention_gpu import _case, _check
    _check(_case(2, Nq, Nk, H, G, D, dtype, density=0.01, soft=True, shared_mask=D == 32, seed=D + Nq), dtype, what="%d wide" % D)
    _check(_case(2, Nq, Nk, H, G, D, dtype, density=0.01, soft=True, seed=D + Nq), dtype, grad=False, what="%d wide, forward alone" % D)

"""CPU tests: what ops.dot_attention, ops.embedding and ops.newton_schulz do around their launches, which are replaced by a list of them."""
import inspect

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode


@pytest.fixture
def launches(monkeypatch):
    """(entry point, arguments) of every launch; nothing is computed, and tensors may lie on the CPU."""
    from gat_amd import ops
    made = []
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_launch", lambda device, name, *args: made.append((name, args)))
    return made


class Operators(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.__name__)
        return func(*args, **(kwargs or {}))


def test_a_lookup_of_a_list_of_ids_only_allocates(launches):
    """A short lookup is bound by the host: no view, no copy around its launches."""
    from gat_amd import ops
    ids, table = torch.tensor([1, 0, 2]), torch.zeros((4, 8), requires_grad=True)
    with Operators() as seen:
        ops.embedding(ids, table.detach())
    assert [n for n in seen.names if "empty" not in n and "detach" not in n] == [] and sum("empty" in n for n in seen.names) == 1
    out, dout = ops.embedding(ids, table), torch.ones((3, 8))
    with Operators() as seen:
        torch.autograd.grad(out, table, dout)
    assert [n for n in seen.names if "empty" not in n and "detach" not in n] == [] and sum("empty" in n for n in seen.names) == 2
    assert [n for n, _ in launches] == ["gatmi_embed_fwd", "gatmi_embed_fwd", "gatmi_embed_bwd"]


def _calls():
    """name -> (call of one tensor, that tensor)"""
    from gat_amd import ops
    g = torch.Generator().manual_seed(0)
    rows, ids, sizes = torch.randn((2, 3, 4, 8), generator=g), torch.tensor([[1, 0], [3, -1]]), torch.tensor([3, 1], dtype=torch.int32)
    mask = torch.zeros((1, 3, 3))
    return {"queries": (lambda x: ops.dot_attention(x, rows, rows, mask, key_sizes=sizes), rows), "keys": (lambda x: ops.dot_attention(rows, x, rows), rows),
            "values": (lambda x: ops.dot_attention(rows, rows, x, scale=2.0), rows), "odd width": (lambda x: ops.dot_attention(x, x, x), rows[..., :7]),
            "embedding": (lambda x: ops.embedding(ids, x, 0.5), rows[0, 0]), "newton_schulz": (lambda x: ops.newton_schulz(x, 3), rows),
            "newton_schulz of one": (lambda x: ops.newton_schulz(x, coefficients=(1.5, -0.5, 0.0)), rows[0, 0])}


@pytest.mark.parametrize("name", list(_calls()))
def test_tangents_are_refused(launches, name):
    import torch.autograd.forward_ad as forward_ad
    call, x = _calls()[name]
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        launches.clear()
        call(x)                                                                       # without a tangent the level changes nothing
        assert len(launches) == 1


@pytest.mark.parametrize("name", list(_calls()))
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_trace_keeps_the_launch(launches, name):
    call, x = _calls()[name]
    shape = call(x).shape
    traced = torch.jit.trace(call, x, check_trace=False)
    want = launches[0][0]
    launches.clear()
    assert traced(x + 1).shape == shape
    with torch.no_grad():
        assert traced(x + 1).shape == shape
    assert [n for n, _ in launches] == [want, want]


def test_no_gradient_saves_nothing_for_one(launches):
    """Recorded without a gradient asked, the attention takes what serving takes: no row sums, no bits of a small mask."""
    import torch.autograd.forward_ad as forward_ad
    from gat_amd import ops
    q, mask = torch.zeros((1, 2, 1, 8)), torch.zeros((1, 2, 2))
    ops.dot_attention(q, q, q, mask)
    with forward_ad.dual_level():
        ops.dot_attention(q, q, q, mask)
    (_, plain), (_, recorded) = launches
    pointers = lambda args: [a is None for a in args[7:]]
    assert pointers(plain) == pointers(recorded)


def test_newton_schulz_takes_no_gradient_recorded_or_not(launches):
    import torch.autograd.forward_ad as forward_ad
    from gat_amd import ops
    x = torch.zeros((4, 4), requires_grad=True)
    assert not ops.newton_schulz(x).requires_grad
    with forward_ad.dual_level():
        assert not ops.newton_schulz(x).requires_grad


def _odd_strides(dtype):
    """name -> [B, N, heads, 8] rows with a dimension of size 1 whose stride divides nothing"""
    base = torch.arange(2 * 5 * 3 * 9, dtype=torch.float32).to(dtype)
    v = lambda *a: torch.as_strided(base, *a)
    return {"one query of one graph": base[:9].reshape(1, 1, 9)[..., :8].unsqueeze(2), "one graph": v((1, 5, 2, 8), (77, 16, 8, 1)), "one node": v((3, 1, 2, 8), (16, 3, 8, 1)),
            "one head": v((2, 5, 1, 8), (40, 8, 5, 1)), "one head, not aligned": v((2, 5, 1, 8), (40, 8, 5, 1), 1), "one of all, not aligned": v((1, 1, 1, 8), (9, 7, 5, 1), 3),
            "one head, rows 9 apart": v((2, 5, 1, 8), (45, 9, 3, 1))}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(_odd_strides(torch.float32)))
def test_strides_of_dimensions_of_size_one_do_not_matter(name, dtype):
    from gat_amd import _lib, ops
    t = _odd_strides(dtype)[name]
    rows, strides = ops._attn_rows(t, 8)
    B, N, H, D = rows.shape
    assert torch.equal(rows, t)
    assert rows.data_ptr() % 16 == 0 and all(s * t.element_size() % 16 == 0 for s in strides)
    assert torch.equal(torch.as_strided(rows, rows.shape, (*strides, 1)), t)
    # the library takes them: it gets as far as the missing result
    rc = _lib.lib.gatmi_dot_attn_fwd(B, N, N, H, H, D, ops._FLOATS[dtype], *(rows.data_ptr(), strides) * 3, None, 0, N, None, None, 1.0, None, None, None, None, None, None, None)
    assert rc == -1 and "out is null" in _lib.last_error()


def _orders():
    """name -> (turned, order): x.permute(*turned).contiguous().permute(*order) is x with its dimensions in another order in memory"""
    return {"heads first": ((0, 2, 1, 3), (0, 2, 1, 3)), "nodes fastest": ((0, 2, 3, 1), (0, 3, 1, 2)), "graphs fastest": ((1, 2, 3, 0), (3, 0, 1, 2)), "width first": ((3, 0, 1, 2), (1, 2, 3, 0)),
            "heads fastest": ((0, 1, 3, 2), (0, 1, 3, 2))}


@pytest.mark.parametrize("D", [4, 8, 13, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("order", list(_orders()))
def test_rows_in_any_order_become_rows_of_the_kernels(order, dtype, D):
    from gat_amd import ops
    turned, back = _orders()[order]
    unit = 4 if dtype == torch.float32 else 8
    width = (D + unit - 1) // unit * unit
    x = torch.randn((2, 40, 3, D)).to(dtype)
    t = x.permute(*turned).contiguous().permute(*back)
    assert torch.equal(t, x)
    rows, strides = ops._attn_rows(t, width)
    assert rows.stride(3) == 1 and rows.data_ptr() % 16 == 0 and all(s % unit == 0 for s in strides)
    assert torch.equal(rows[..., :D], x) and (rows[..., D:] == 0).all()


def test_layers_take_the_arguments_of_their_kin_in_the_same_order():
    """A call that is moved over from the additive heads means the same by position."""
    from gat_amd import layers
    names = lambda f: [n for n, p in inspect.signature(f).parameters.items() if p.kind == p.POSITIONAL_OR_KEYWORD]
    assert names(layers.dot_attn_head) == names(layers.attn_head)
    assert names(layers.dot_attn_heads) == names(layers.attn_heads)
    assert names(layers.DotHeads.__init__) == names(layers.GATHeads.__init__)
    ours, theirs = names(layers.DotHeads.forward), names(layers.GATHeads.forward)
    assert ours[3:] == theirs[3:len(ours)] and theirs[len(ours):] == ["seed"]                  # the mask has a name of its own; no seed: torch drops the input


def test_dropout_of_the_coefficients_is_refused():
    from gat_amd import layers
    x, store = torch.zeros((1, 3, 8)), layers.VariableStore()
    with layers.variable_scope(store):
        for call in (lambda: layers.dot_attn_head(x, 8, None, layers.elu, 0.6, 0.6), lambda: layers.dot_attn_head(x, 8, None, layers.elu, coef_drop=0.6),
                     lambda: layers.dot_attn_heads(x, 8, None, "elu", 2, "concat", 0.0, 0.6), lambda: layers.DotHeads(8, 2, 8)(x, None, coef_drop=0.1)):
            store.layers = torch.nn.ModuleList()
            store.begin()
            with pytest.raises(ValueError, match="coef_drop"):
                call()
            assert not any(m.has_res for m in store.layers)
    with pytest.raises(ValueError, match="residual"):
        layers.DotHeads(8, 4, 8, 2)                                                            # not the number of shared heads


def _muon(monkeypatch, made):
    """models.Muon with its orthogonalisation replaced by the identity, whose inputs are kept."""
    from gat_amd import models, ops

    def same(x, steps=5, **kw):
        made.append(x.clone())
        return x.clone()
    monkeypatch.setattr(ops, "newton_schulz", same)
    return models.Muon


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_keeps_the_momentum_of_bf16_parameters_in_fp32(monkeypatch, nesterov):
    """A constant gradient: m_k = g (1 - 0.95^k) / 0.05.  In fp32 a step rounds twice, 2^-24 of m each, the factor itself is rounded (2^-25), and
    0.95 carries that on, 20 times in all: 50 * 2^-24 at the most, and 3 * 2^-24 more in the sum that is handed on.  (In bf16 m stays where a step
    changes it by less than half of its last place, up to some hundredths short.)"""
    made = []
    Muon = _muon(monkeypatch, made)
    p = torch.nn.Parameter(torch.zeros((3, 5), dtype=torch.bfloat16))
    opt = Muon([p], lr=0.0, nesterov=nesterov)
    g = torch.randn((3, 5), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    for _ in range(150):
        p.grad = g.clone()
        opt.step()
    m = g.double() * (1 - 0.95 ** 150) / 0.05
    want = g.double() + 0.95 * m if nesterov else m
    assert opt.state[p]["m"].dtype == torch.float32 and made[-1].dtype == torch.float32
    assert ((opt.state[p]["m"].double() - m).abs() <= 50 * 2.0 ** -24 * m.abs()).all()
    assert ((made[-1][0].double() - want).abs() <= 53 * 2.0 ** -24 * want.abs()).all()
    # saved and loaded it stays as it is
    other = Muon([torch.nn.Parameter(p.detach().clone())], lr=0.0, nesterov=nesterov)
    other.load_state_dict(opt.state_dict())
    (q,) = other.param_groups[0]["params"]
    q.grad = g.clone()
    assert torch.equal(other.state[q]["m"], opt.state[p]["m"]) and other.state[q]["m"].data_ptr() != opt.state[p]["m"].data_ptr()
    for o in (opt, other):
        o.step()
    assert torch.equal(other.state[q]["m"], opt.state[p]["m"])


def test_muon_groups_added_later_and_given_as_dicts(monkeypatch):
    made = []
    Muon = _muon(monkeypatch, made)
    t = lambda *s: torch.nn.Parameter(torch.ones(s))
    a, b, c, d = t(3, 4), t(5, 2, 3), t(2, 5), t(2, 6, 3)
    opt = Muon([a, {"params": [(b, 1)], "lr": 0.5}])
    opt.add_param_group({"params": c, "momentum": 0.0})
    opt.add_param_group({"params": [(d, 0)]})
    assert [(g["head_axis"], g["lr"], g["momentum"]) for g in opt.param_groups] == [(None, 0.02, 0.95), (1, 0.5, 0.95), (None, 0.02, 0.0), (0, 0.02, 0.95)]
    for p in (a, b, c, d):
        p.grad = torch.full_like(p, 2.0)
    opt.step()
    assert [tuple(x.shape) for x in made] == [(1, 3, 4), (1, 2, 5, 3), (1, 2, 5), (1, 2, 6, 3)]
    assert torch.allclose(c, torch.full_like(c, 1.0 - 0.02 * 2.0)) and torch.allclose(b, torch.full_like(b, 1.0 - 0.5 * 3.9))
    for bad in ({"params": [t(2, 2, 2)]}, {"params": [(t(2, 2), 0)]}, {"params": [t(4, 4)], "momentum": 1.0}, {"params": [(t(2, 2, 2), 1), t(3, 3)]}):
        with pytest.raises(ValueError):
            opt.add_param_group(bad)
    assert len(opt.param_groups) == 4
    opt.load_state_dict(opt.state_dict())
    opt.step()


def test_muon_refuses_what_its_step_cannot_do_when_it_is_made(monkeypatch):
    """Types and counts that ops.newton_schulz refuses: not in the middle of a step, when momentum and decay have been applied."""
    Muon = _muon(monkeypatch, [])
    t = lambda dtype: torch.nn.Parameter(torch.ones((3, 4), dtype=dtype))
    for dtype in (torch.float16, torch.float64):
        with pytest.raises(ValueError, match="fp32 or bf16"):
            Muon([t(dtype)])
    with pytest.raises(ValueError, match="steps"):
        Muon([t(torch.float32)], steps=33)
    from gat_amd import _lib
    P = 4096                                                       # never read: the counts are refused before any launch
    for steps, rc in ((0, -1), (33, -1)):
        assert _lib.lib.gatmi_newton_schulz(1, 4, 4, P, 16, 4, 0, steps, 3.4445, -4.775, 2.0315, 1e-7, P, 16, 4, P, None) == rc
    empty = torch.nn.Parameter(torch.ones((3, 0)))
    opt = Muon([empty, t(torch.bfloat16)], steps=32)
    for p in opt.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    opt.step()                                                     # a matrix without entries has nothing to update


def test_muon_does_not_make_its_momentum_inside_a_capture(monkeypatch):
    """The zeros it starts from would be part of the graph, and every replay would start from them."""
    Muon = _muon(monkeypatch, [])
    p = torch.nn.Parameter(torch.ones((3, 4)))
    opt = Muon([p])
    p.grad = torch.ones_like(p)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    assert not opt.state[p] and (p == 1.0).all()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    opt.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    opt.step()
    assert torch.allclose(opt.state[p]["m"], torch.full_like(p, 1.95))


def test_muon_loads_a_state_without_momentum(monkeypatch):
    """As it is saved after a step that was refused, or before the first one."""
    Muon = _muon(monkeypatch, [])
    p = torch.nn.Parameter(torch.ones((3, 4)))
    opt = Muon([p])
    opt.state[p]                                                   # an entry, but nothing in it
    other = Muon([torch.nn.Parameter(torch.ones((3, 4)))])
    other.load_state_dict(opt.state_dict())
    (q,) = other.param_groups[0]["params"]
    q.grad = torch.ones_like(q)
    other.step()
    assert torch.allclose(other.state[q]["m"], torch.ones_like(q))

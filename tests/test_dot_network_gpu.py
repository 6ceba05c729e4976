"""The operators as a network uses them: learned node rows -> dot-product heads over the dense mask -> masked cross-entropy ->
orthogonalised updates of the kernels, Adam for the rest; against the same step in float64 torch, and captured and replayed."""
import numpy as np
import pytest
import torch

from tests import attn_ref
from tests.util import assert_close

pytestmark = pytest.mark.gpu

B, N, ROWS, F, H, G, D, C = 3, 60, 40, 32, 4, 2, 16, 5


class Net(torch.nn.Module):
    def __init__(self, device, storage="f32"):
        super().__init__()
        from gat_amd import layers
        self.embed = layers.NodeEmbedding(ROWS, F, scale=F ** 0.5, device=device)
        self.first = layers.DotHeads(F, H, D, kv_heads=G, residual=True, device=device, storage=storage)
        self.last = layers.DotHeads(H * D, 2, C, device=device)

    def forward(self, ids, bias, sizes):
        x = self.first(self.embed(ids), bias, "elu", sizes=sizes)
        return self.last(x, bias, "identity", "mean", sizes=sizes)


def _data(seed=0):
    rng = np.random.default_rng(seed)
    dev = torch.device("cuda:0")
    sizes = np.array([N, 41, 7])
    ids = rng.integers(0, ROWS, (B, N))
    adj = rng.random((B, N, N)) < 0.15
    adj |= np.eye(N, dtype=bool)
    for b in range(B):
        ids[b, sizes[b]:] = -1
    labels = np.eye(C)[rng.integers(0, C, (B, N))]
    mask = (np.arange(N)[None] < sizes[:, None]) & (rng.random((B, N)) < 0.6)
    t = lambda a, dt=torch.float32: torch.tensor(a, dtype=dt, device=dev)
    return dict(ids=t(ids, torch.int64), bias=t(np.where(adj, 0.0, -1e9)), sizes=t(sizes, torch.int32), labels=t(labels), mask=t(mask.astype(np.float32)))


def _loss(net, d):
    from gat_amd.models import BaseGAttN
    logits = net(d["ids"], d["bias"], d["sizes"])
    return BaseGAttN.masked_softmax_cross_entropy(logits.reshape(B * N, C), d["labels"].reshape(B * N, C), d["mask"].reshape(-1))


def _heads_ref(m, p, x, bias, inside, act, mean):
    """A DotHeads layer in float64 torch on the CPU: p holds its parameters."""
    rows = torch.einsum("bnf,fhd->bnhd", x, p["W"])
    H_, G_, D_ = m.heads, m.kv_heads, m.width
    q, k, v = rows[:, :, :H_], rows[:, :, H_:H_ + G_], rows[:, :, H_ + G_:]
    k, v = (t.repeat_interleave(H_ // G_, dim=2) for t in (k, v))
    seen = (bias > -1e8) & inside[:, None, :] & inside[:, :, None]
    z = torch.einsum("bihd,bjhd->bhij", q, k) * D_ ** -0.5 + bias[:, None]
    z = z.masked_fill(~seen[:, None], -1e300)
    a = torch.softmax(z, -1) * seen[:, None]
    out = torch.einsum("bhij,bjhd->bihd", a, v)
    if m.has_res:
        out = out + torch.einsum("bnf,fhd->bnhd", x, p["W_res"]) + p["b_res"]
    out = out + p["bias"]
    out = torch.nn.functional.elu(out) if act == "elu" else out
    return out.mean(2) if mean else out.flatten(2)


def _reference(net, d):
    ps = {n: p.detach().double().cpu().requires_grad_() for n, p in net.named_parameters()}
    sub = lambda k: {n[len(k) + 1:]: p for n, p in ps.items() if n.startswith(k + ".")}
    ids, bias, sizes = d["ids"].cpu(), d["bias"].double().cpu(), d["sizes"].cpu()
    inside = torch.arange(N)[None] < sizes[:, None]
    ok = (ids >= 0)[..., None]
    x = torch.where(ok, ps["embed.weight"][ids.clamp(min=0)] * net.embed.scale, 0.0)
    x = _heads_ref(net.first, sub("first"), x, bias, inside, "elu", False)
    x = _heads_ref(net.last, sub("last"), x, bias, inside, "identity", True)
    y, mk = d["labels"].double().cpu(), d["mask"].double().cpu()
    ce = -(y * torch.log_softmax(x, -1)).sum(-1)
    loss = (ce * mk).sum() / mk.sum()
    loss.backward()
    return loss.item(), {n: p.grad.numpy() for n, p in ps.items()}


def _optimizers(net, capturable=False):
    from gat_amd.models import Muon, TFAdam, matrix_parameters
    mats, others = matrix_parameters(net)
    assert len(mats) == 3 and len(others) == 4
    return Muon(mats, lr=0.02), TFAdam(others, lr=0.01, capturable=capturable)


def test_one_step_against_float64():
    torch.manual_seed(0)
    net, d = Net("cuda:0"), _data()
    opts = _optimizers(net)
    before = {n: p.detach().clone() for n, p in net.named_parameters()}
    loss = _loss(net, d)
    loss.backward()
    ref_loss, ref = _reference(net, d)
    assert abs(loss.item() - ref_loss) < 1e-5 * abs(ref_loss)
    for n, p in net.named_parameters():
        assert_close(p.grad.cpu().numpy(), ref[n], rtol=1e-4, atol_scale=2e-5, what=n)       # two layers of fp32 sums: a hundred roundings of 2^-24 of the scale
    for o in opts:
        o.step()
    for n, axis, m in (("first.W", 1, net.first), ("first.W_res", 1, net.first), ("last.W", 1, net.last)):
        p, g = dict(net.named_parameters())[n], dict(net.named_parameters())[n].grad.double().cpu().numpy()
        step = (before[n] - p.detach()).double().cpu().numpy()
        for h in range(g.shape[1]):
            u = g[:, h] * 1.95                                                               # first step: m = g, u = g + 0.95 m
            np.testing.assert_allclose(step[:, h], 0.02 * max(1.0, g.shape[2] / g.shape[0]) ** 0.5 * attn_ref.newton_schulz(u), rtol=0, atol=1e-6)


def test_bf16_rows_stay_near_fp32():
    torch.manual_seed(0)
    a, d = Net("cuda:0"), _data()
    b = Net("cuda:0", storage="bf16")
    b.load_state_dict(a.state_dict())
    la, lb = (n.first(n.embed(d["ids"]), d["bias"], "elu", sizes=d["sizes"]) for n in (a, b))
    # q, k, v, P and the result are rounded by 2^-8 of values of the scale of max |la|; scores of order 10 turn into factors of e^(10 2^-7)
    assert (la - lb).abs().max() < 0.1 * la.abs().max()


def test_training_step_captured_and_replayed():
    """Replays follow the eager steps bit for bit, with eager work and synchronisations between them."""
    from gat_amd import graphs
    d = _data()

    def build():
        torch.manual_seed(1)
        net = Net("cuda:0")
        opts = _optimizers(net, capturable=True)

        def step():
            for p in net.parameters():
                p.grad = None
            loss = _loss(net, d)
            loss.backward()
            for o in opts:
                o.step()
            return loss
        return net, step

    eager, eager_step = build()
    losses = [float(eager_step().detach()) for _ in range(3 + 4)]
    net, step = build()
    replay, loss = graphs.capture(step, warmup=3, fresh_dropout=False)
    other = _data(seed=9)
    for k in range(4):
        replay()
        torch.cuda.synchronize()
        assert float(loss.detach()) == losses[3 + k]
        _loss(net, other)
    for (n, p), (_, q) in zip(net.named_parameters(), eager.named_parameters()):
        assert torch.equal(p, q), n


def test_dot_attn_head_uses_the_variable_store():
    from gat_amd import layers
    dev = torch.device("cuda:0")
    store = layers.VariableStore()
    x, d = torch.randn((B, N, F), device=dev), _data()
    with layers.variable_scope(store):
        store.begin()
        a = layers.dot_attn_head(x, 8, d["bias"], layers.elu)
        b = layers.dot_attn_heads(x, 6, d["bias"], "identity", 3, "mean", residual=True)
        store.begin()
        assert torch.equal(layers.dot_attn_head(x, 8, d["bias"], layers.elu), a)
        assert torch.equal(layers.dot_attn_heads(x, 6, d["bias"], "identity", 3, "mean", residual=True), b)
        store.begin()
        assert layers.dot_attn_head(x, 8, d["bias"], layers.elu, in_drop=0.5).shape == (B, N, 8)
    assert len(store.layers) == 2 and a.shape == (B, N, 8) and b.shape == (B, N, 6)
    m = store.layers[1]
    p = {n: q.detach().double().cpu() for n, q in m.named_parameters()}
    ref = _heads_ref(m, p, x.double().cpu(), d["bias"].double().cpu(), torch.ones((B, N), dtype=torch.bool), "identity", True)
    assert_close(b.detach().cpu().numpy(), ref.numpy(), rtol=1e-4, atol_scale=1e-5)


def test_two_streams_at_once():
    """Calls of every kind on two streams without a wait between them, each with workspaces of its own."""
    from gat_amd import ops
    g = torch.Generator(device="cuda:0").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda:0", generator=g)
    q, k, v, ids, table, x = r(2, 600, 4, 32), r(2, 600, 4, 32), r(2, 600, 4, 32), torch.randint(0, 50, (9000,), device="cuda:0", generator=g), r(50, 24), r(2, 300, 2100)
    bias = torch.where(r(2, 600, 600) > 1.0, 0.0, -1e9)

    def work():
        a = [t.detach().requires_grad_() for t in (q, k, v, table)]
        o, e = ops.dot_attention(a[0], a[1], a[2], bias), ops.embedding(ids, a[3])
        return [o.detach(), e.detach(), ops.newton_schulz(x), *torch.autograd.grad(o, a[:3], q), *torch.autograd.grad(e, a[3], e.detach())]
    want = work()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for res in got:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    from gat_amd import ops
    q = torch.randn(1, 5, 1, 8, device="cuda:0", requires_grad=True)
    (first,) = torch.autograd.grad(ops.dot_attention(q, q.detach(), q.detach()).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), q)
    table = torch.randn(4, 8, device="cuda:0", requires_grad=True)
    (first,) = torch.autograd.grad((ops.embedding(torch.tensor([1, 2], device="cuda:0"), table) ** 2).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), table)

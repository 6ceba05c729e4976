"""GPU parity of ops.embedding and its gradient by sorted ids: widths, types, repeated and padded ids, table sizes of one to four
radix passes, runs that cross chunk and block borders, strides, streams and captured graphs."""
import numpy as np
import pytest
import torch

from tests import attn_ref
from tests.attn_ref import within

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _run(ids, table, dout, scale):
    from gat_amd import ops
    leaf = table.detach().requires_grad_()
    out = ops.embedding(ids, leaf, scale=scale)
    return out.detach(), torch.autograd.grad(out, leaf, dout)[0]


def _check(ids, rows, width, dtype, scale=1.5, seed=0, id_dtype=torch.int64):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    table = torch.randn((rows, width), device=dev, generator=g).to(TYPES[dtype])
    idt = torch.as_tensor(ids).to(id_dtype).to(dev)
    dout = torch.randn((*idt.shape, width), device=dev, generator=g).to(TYPES[dtype])
    out, grad = _run(idt, table, dout, scale)
    ok = (idt >= 0) & (idt < rows)
    want = torch.zeros((*idt.shape, width), dtype=TYPES[dtype], device=dev)
    want[ok] = (table.float()[idt[ok].long()] * scale).to(TYPES[dtype])
    assert torch.equal(out, want)
    value, bound = attn_ref.embedding_grad(np.asarray(ids, dtype=np.int64), dout.double().cpu().numpy(), rows, scale, dtype == "bf16")
    within(grad.double().cpu().numpy(), value, bound, "gradient")
    return out, grad


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [1, 2, 3, 4, 7, 8, 33, 64, 100, 128, 250, 256, 500, 1000])
def test_widths(width, dtype):
    rng = np.random.default_rng(width)
    _check(rng.integers(-2, 52, 700), 50, width, dtype)


@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 127, 4095, 4096, 4097, 8192, 10000, 40000])
@pytest.mark.parametrize("rows", [1, 2, 255, 256, 257, 3000, 70000])
def test_token_and_row_counts(tokens, rows):
    rng = np.random.default_rng(tokens + rows)
    _check(rng.integers(0, rows, tokens), rows, 8, "f32", id_dtype=torch.int32 if tokens % 2 else torch.int64)


def test_four_radix_passes():
    rng = np.random.default_rng(0)
    rows = 17_000_000
    _check(np.concatenate([rng.integers(0, rows, 5000), [0, rows - 1, rows, -1, 2 ** 40, -2 ** 40]]), rows, 1, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["all_same", "two_runs", "hub", "sorted", "reversed", "all_padding", "blocks_of_64", "off_by_one"])
def test_runs(kind, dtype):
    n, rows = 20011, 300
    rng = np.random.default_rng(3)
    ids = {"all_same": np.full(n, 7), "two_runs": np.arange(n) % 2 * 299, "hub": np.where(rng.random(n) < 0.7, 11, rng.integers(0, rows, n)),
           "sorted": np.arange(n) * rows // n, "reversed": rows - 1 - np.arange(n) * rows // n, "all_padding": np.full(n, -1),
           "blocks_of_64": np.arange(n) // 64 % rows, "off_by_one": (np.arange(n) + 1) // 64 % rows}[kind]
    _check(ids, rows, 24, dtype)


def test_shapes_of_ids_and_no_tokens():
    rng = np.random.default_rng(4)
    _check(rng.integers(-1, 20, (3, 5, 7)), 20, 12, "f32")
    _check(rng.integers(0, 20, ()), 20, 12, "f32")
    out, grad = _check(np.zeros((0,), dtype=np.int64), 20, 12, "f32")
    assert out.shape == (0, 12) and (grad == 0).all()
    from gat_amd import ops
    none = ops.embedding(torch.zeros(3, dtype=torch.int64, device="cuda:0"), torch.zeros((0, 4), device="cuda:0"))
    assert none.shape == (3, 4) and (none == 0).all()


def test_ids_beyond_int32_are_padding():
    ids = np.array([2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 63 - 1, -2 ** 63, 1], dtype=np.int64)
    out, grad = _check(ids, 4, 8, "f32")
    assert (out[:5] == 0).all() and (grad[[0, 2, 3]] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype):
    from gat_amd import ops
    dev = torch.device("cuda:0")
    rng = np.random.default_rng(5)
    ids = torch.tensor(rng.integers(0, 40, (6, 50)), device=dev)
    big = torch.randn((40, 48), device=dev).to(TYPES[dtype])
    for view in (big[:, 8:40], big[:, 1:33], big[::2][:, :32], torch.randn((32, 40), device=dev).to(TYPES[dtype]).t()):
        idv = ids % view.shape[0]
        assert torch.equal(ops.embedding(idv, view, 2.0), ops.embedding(idv, view.contiguous(), 2.0))
        assert torch.equal(ops.embedding(idv.t(), view, 2.0), ops.embedding(idv, view, 2.0).transpose(0, 1))
    leaf = big[:, :32].contiguous().requires_grad_()
    wide = torch.randn((6, 50, 64), device=dev).to(TYPES[dtype])
    for d in (wide[..., :32], wide[..., 1:33], torch.ones((), device=dev, dtype=TYPES[dtype]).expand(6, 50, 32), wide[:, :, :1].expand(6, 50, 32)):
        a = torch.autograd.grad(ops.embedding(ids, leaf), leaf, d)[0]
        b = torch.autograd.grad(ops.embedding(ids, leaf), leaf, d.contiguous())[0]
        assert torch.equal(a, b)


def test_twice_the_same_bits_and_on_another_stream():
    rng = np.random.default_rng(6)
    dev = torch.device("cuda:0")
    ids = torch.tensor(rng.zipf(1.3, 50000) % 1000, device=dev)
    table, dout = torch.randn((1000, 64), device=dev), torch.randn((50000, 64), device=dev)
    want = _run(ids, table, dout, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(ids, table, dout, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(want, got, _run(ids, table, dout, 1.0)):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("tokens", [900, 9000])
def test_captured(tokens):
    from gat_amd import graphs, ops
    dev = torch.device("cuda:0")
    rng = np.random.default_rng(7)
    ids = torch.tensor(rng.integers(0, 500, tokens), device=dev)
    table = torch.randn((500, 20), device=dev, requires_grad=True)
    dout = torch.randn((tokens, 20), device=dev)

    def step():
        out = ops.embedding(ids, table, 3.0)
        return out, torch.autograd.grad(out, table, dout)[0]

    replay, res = graphs.capture(step, fresh_dropout=False)
    for seed in range(4):
        ids.copy_(torch.tensor(np.random.default_rng(seed).integers(-3, 505, tokens)))
        dout.normal_()
        replay()
        torch.cuda.synchronize()
        for a, b in zip(res, _run(ids, table, dout, 3.0)):
            assert torch.equal(a, b), seed


def test_node_embedding_layer_equals_one_hot_features():
    """scale * weight[ids] as a layer, against the one-hot product it stands for, gradient included."""
    from gat_amd.layers import NodeEmbedding
    dev = torch.device("cuda:0")
    m = NodeEmbedding(30, 16, scale=4.0, device=dev)
    ids = torch.tensor([[0, 29, -1, 5], [5, 5, 30, 2]], device=dev)
    hot = torch.zeros((2, 4, 30), device=dev)
    for i in range(2):
        for j in range(4):
            if 0 <= ids[i, j] < 30:
                hot[i, j, ids[i, j]] = 1.0
    dout = torch.randn((2, 4, 16), device=dev)
    out = m(ids)
    out.backward(dout)
    assert torch.allclose(out, 4.0 * hot @ m.weight.detach(), rtol=0, atol=1e-6)
    assert torch.allclose(m.weight.grad, 4.0 * hot.reshape(8, 30).t() @ dout.reshape(8, 16), rtol=0, atol=1e-5)

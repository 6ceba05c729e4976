"""GPU tests of calls of ops.dot_attention, ops.embedding and ops.newton_schulz as documented but off the common path."""
import pytest
import torch

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

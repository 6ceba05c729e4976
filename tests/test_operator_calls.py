"""CPU tests: what ops.dot_attention, ops.embedding and ops.newton_schulz do around their launches, which are replaced by a list of them."""
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

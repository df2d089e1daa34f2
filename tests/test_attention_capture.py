"""The rule for captured backwards without a GPU: streams and the state of capturing are made up, launches are not made."""
import contextlib

import pytest
import torch

from memarch_amd import _lib, attention


@pytest.fixture
def at(monkeypatch):
    """The present stream and whether it is being captured."""
    state = {"stream": 1, "capturing": False}
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    lib = type("L", (), {n: staticmethod(lambda *a: 0) for n in ("mce_attn_bwd_ws_bytes", "mce_pack_plan_bytes",
                                                                 "mce_pack_fwd_ws_bytes", "mce_pack_bwd_ws_bytes")})
    monkeypatch.setattr(_lib, "load_attn", lambda: lib)
    monkeypatch.setattr(_lib, "load_serve", lambda: lib)
    monkeypatch.setattr(attention, "_check_same", lambda *a: None)
    monkeypatch.setattr(attention, "_On", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(attention, "_stream", lambda dev: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    return state


def _leaves(dims):
    return [torch.zeros(*dims, dtype=torch.bfloat16).requires_grad_() for _ in range(3)]


def _packed(q, k, v):
    return attention.packed_attention(q, k, v, torch.tensor([0, 5], dtype=torch.int32), window=4)


CALLS = {"window": ((1, 5, 2, 64), lambda q, k, v: attention.window_attention(q, k, v, window=4)), "packed": ((5, 2, 64), _packed)}


@pytest.mark.parametrize("name", CALLS)
def test_a_backward_beside_an_earlier_graph_of_its_leaves(at, name):
    """Refused while a graph made on another stream lives; taken on the same stream, and once that graph is gone."""
    shape, call = CALLS[name]
    leaves = _leaves(shape)
    alive = call(*leaves)
    at.update(stream=2, capturing=True)
    out = call(*leaves)
    with pytest.raises(RuntimeError, match="graph of the same leaves"):
        torch.autograd.grad(out, leaves, torch.zeros_like(out))
    at.update(stream=1)
    out = call(*leaves)
    torch.autograd.grad(out, leaves, torch.zeros_like(out))
    at.update(stream=2)
    del alive, out
    out = call(*leaves)
    torch.autograd.grad(out, leaves, torch.zeros_like(out))


def test_eager_backwards_are_not_looked_at(at):
    leaves = _leaves((1, 5, 2, 64))
    alive = attention.window_attention(*leaves, window=4)
    at.update(stream=2)
    out = attention.window_attention(*leaves, window=4)
    torch.autograd.grad(out, leaves, torch.zeros_like(out))
    torch.autograd.grad(alive, leaves, torch.zeros_like(alive))

"""window_attention's backward captured beside an eager graph of its leaves: refused, and taken once that graph is gone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _captured(leaves, go):
    from memarch_amd.attention import window_attention
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention(*leaves, window=64, sinks=2)
        grads = torch.autograd.grad(out, leaves, go)
    return graph, (out, *grads)


def test_capture_beside_an_eager_graph_is_refused():
    from memarch_amd.attention import window_attention
    g = torch.Generator().manual_seed(9)
    q, k, v, go = (torch.randn(2, 70, h, 64, generator=g).bfloat16().cuda() for h in (2, 1, 1, 2))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    alive = window_attention(*leaves, window=64, sinks=2)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="graph of the same leaves"):
        _captured(leaves, go)
    torch.cuda.synchronize()
    ref = (alive.detach().clone(), *torch.autograd.grad(alive, leaves, go))
    del alive
    graph, got = _captured(leaves, go)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
        again = window_attention(*leaves, window=64, sinks=2)
        assert torch.equal(again, ref[0])
        del again

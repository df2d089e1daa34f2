"""packed_attention with more first tokens than most of its sequences have, on the GPU against the fp64 oracle."""
import pytest
import torch

from oracle import attn_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _step(q, k, v, go, cu, cu_k, window, sinks):
    from memarch_amd.attention import packed_attention
    q, k, v = (x.cuda().requires_grad_() for x in (q, k, v))
    out = packed_attention(q, k, v, cu.cuda(), None if cu_k is None else cu_k.cuda(), window=window, sinks=sinks)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), go.cuda()))


def _lens(n, most, g):
    x = torch.randint(0, most, (n,), generator=g)
    return torch.cat((torch.zeros(1), x.cumsum(0))).int()


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("nseq,most,hq,hkv,d,window,sinks,own_keys,first,long", [
    (40, 60, 4, 2, 64, 16, 300, False, 0, 0), (40, 60, 2, 2, 128, 16, 300, True, 5, 0), (300, 20, 2, 1, 8, 5, 2000, False, 0, 0),
    (12, 40, 4, 1, 96, 30, 1000, False, 130, 900), (9, 300, 8, 2, 80, 100, 260, True, 0, 700), (3, 1400, 4, 1, 64, 200, 4000, False, 0, 0),
    (30, 40, 1, 1, 64, 700, 2500, False, 3, 2600),
    (3, 800, 16, 4, 64, 200, 8000, False, 0, 3000)])   # (in planned order)
def test_more_first_tokens_than_sequences_hold(dt, nseq, most, hq, hkv, d, window, sinks, own_keys, first, long):
    """Short sequences with many first tokens, some with one long sequence among them, so that key blocks are shared."""
    print(f"sinks {nseq} {most} {hq} {hkv} {d} {window} {sinks} {own_keys} {first} {long} {dt}", flush=True)
    g = torch.Generator().manual_seed(nseq + most)
    cu = _lens(nseq, most, g) + first
    cu_k = _lens(nseq, most, g) + first if own_keys else None
    for c in (cu,) if cu_k is None else (cu, cu_k):
        c[nseq // 2:] += long
    n = int(cu[-1]) + 3 * first
    m = n if cu_k is None else int(cu_k[-1]) + 3 * first
    mk = lambda r, h: torch.randn(r, h, d, generator=g).to(dt)
    q, k, v, go = mk(n, hq), mk(m, hkv), mk(m, hkv), mk(n, hq)
    got = _step(q, k, v, go, cu, cu_k, window, sinks)
    ref, tol = orc.packed(q, k, v, cu.tolist(), None if cu_k is None else cu_k.tolist(), window, sinks, None, go, dt)
    for name, a, r, t in zip(("out", "dq", "dk", "dv"), got, ref, tol):
        err = (a.double().cpu() - r).abs()
        assert (err <= t).all(), (name, float((err - t).max()))
    again = _step(q, k, v, go, cu, cu_k, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_more_than_launches_hold_workgroups():
    """4096 sequences with up to 65536 first tokens each, of whom 2 have more than 100: every gradient is that of a call with as
    many first tokens as the longest has."""
    n, h, d = 65536, 16, 8
    g = torch.Generator().manual_seed(1)
    lens = torch.full((4096,), 12)
    lens[7], lens[4000] = 9000, n - 9000 - 12 * 4094
    cu = torch.cat((torch.zeros(1), lens.cumsum(0))).int()
    x = [torch.randn(n, h, d, generator=g).to(BF) for _ in range(4)]
    for sinks in (n, 10000):
        got = _step(*x, cu, None, 100, sinks)
        ref = _step(*x, cu, None, 100, 9000)
        for a, b in zip(got, ref):
            assert a.isfinite().all() and torch.equal(a, b)

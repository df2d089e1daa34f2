"""GPU parity of paged_attention against the fp64 oracle: lengths from 0, pages that end inside a tile, windows with first
tokens, bad pages, stale cache contents, strided caches, offsets past 32 bits, graphs and streams."""
import pytest
import torch

from oracle import attn_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _case(b, most, hq, hkv, d, page, dt, seed=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    pages = b * most + spare
    kc = (torch.randn(pages, page, hkv, d, generator=g) * 1.5).to(dt)
    vc = torch.randn(pages, page, hkv, d, generator=g).to(dt)
    q = (torch.randn(b, hq, d, generator=g) * 1.5).to(dt)
    table = torch.randperm(pages, generator=g)[:b * most].view(b, most).int()
    return q, kc, vc, table


def _check(q, kc, vc, table, lens, window=0, sinks=0, scale=None):
    from memarch_amd.attention import paged_attention
    ref, tol = orc.paged(q, kc, vc, table, lens, window, sinks, scale, q.dtype)
    got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(), window=window or None, sinks=sinks,
                          scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))
    return got


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d,page,most,lens", [
    (1, 1, 64, 16, 2, [1, 32, 0]), (2, 1, 8, 8, 9, [72, 71, 65]), (4, 4, 128, 16, 5, [80, 33, 31]), (8, 2, 96, 24, 4, [96, 95, 25]),
    (16, 1, 128, 64, 2, [128, 64, 63]), (40, 1, 64, 16, 3, [48, 17, 16]), (64, 2, 128, 8, 6, [48, 47, 1]),
    (4, 2, 80, 40, 20, [800, 401, 399]), (2, 2, 64, 128, 12, [1536, 1025, 513]), (6, 2, 128, 16, 200, [3200, 1111, 7])])
def test_parity(dt, hq, hkv, d, page, most, lens):
    print(f"paged {hq} {hkv} {d} {page} {lens} {dt}", flush=True)
    q, kc, vc, table = _case(3, most, hq, hkv, d, page, dt, seed=d + page)
    _check(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))


@pytest.mark.parametrize("hq,hkv,d,page,most,lens,window,sinks", [
    (4, 1, 128, 64, 700, [44800], 0, 0),                 # 175 parts
    (2, 1, 64, 16, 2500, [39999], 30000, 20),            # 118 parts of a window, the first tokens in the first of them
    (1, 1, 8, 128, 3080, [393216], 0, 0),                # 1024 parts, the most
    (2, 2, 64, 64, 700, [44800, 20000], 0, 0)])          # 175 parts a sequence at most, the second has fewer
def test_many_parts(hq, hkv, d, page, most, lens, window, sinks):
    """Few heads and long caches: more parts than the joining wave has lanes."""
    from memarch_amd import _lib
    b = len(lens)
    need = _lib.load_attn().mce_paged_ws_bytes(b, hq, hkv, d, page, most, window, sinks)
    assert need >= 65 * b * hq * (d + 2) * 4
    print(f"paged parts {hq} {hkv} {d} {lens} {window}", flush=True)
    q, kc, vc, table = _case(b, most, hq, hkv, d, page, BF, seed=most)
    _check(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32), window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 0), (32, 1), (33, 7), (100, 64), (1000, 4), (100, 1000)])
def test_windows(window, sinks):
    q, kc, vc, table = _case(4, 30, 4, 2, 64, 16, BF, seed=window)
    _check(q, kc, vc, table, torch.tensor([480, 161, 100, 3], dtype=torch.int64), window, sinks)


@pytest.mark.parametrize("split", [False, True])
def test_bad_pages_and_stale_contents(split):
    """Entries outside the cache are not seen; NaN and infinities in slots past the length, before the window and in pages
    that nobody has do not matter; lengths past the table count as its whole."""
    most = 80 if split else 6
    q, kc, vc, table = _case(5, most, 4, 2, 64, 16, BF, seed=11)
    n = most * 16
    lens = torch.tensor([n - 5, n + 1000, 37, 40, -2], dtype=torch.int32)
    table[0, 1], table[0, most - 2], table[1, 0], table[3, :3] = -1, kc.shape[0], 2 ** 31 - 1, -7
    ref = [(table.clone(), lens.clone())]
    used = set()
    for i in range(5):
        for j in range(min(max(int(lens[i]), 0), n)):
            used.add((int(table[i, j // 16]), j % 16))
    for p in range(kc.shape[0]):
        for s in range(16):
            if (p, s) not in used:
                kc[p, s], vc[p, s] = float("nan"), float("inf")
    got = _check(q, kc, vc, *ref[0])
    assert not got[3].any() and not got[4].any()
    # a window: the slots before it turn NaN as well, except for the first tokens
    for i in range(5):
        for j in range(min(max(int(lens[i]), 0), n)):
            p = int(table[i, j // 16])
            if 0 <= p < kc.shape[0] and min(int(lens[i]), n) - 1 - j >= 20 and j >= 3:
                kc[p, j % 16], vc[p, j % 16] = float("inf"), float("nan")
    got = _check(q, kc, vc, table, lens, 20, 3)
    assert torch.isfinite(got).all()


def test_strides_and_table_layouts():
    from memarch_amd.attention import paged_attention
    q, kc, vc, table = (x.cuda() for x in _case(3, 9, 4, 2, 64, 16, BF, seed=4))
    lens = torch.tensor([144, 70, 9], dtype=torch.int32, device="cuda")
    base = paged_attention(q, kc, vc, table, lens)
    both = torch.stack((kc, vc), 3).contiguous()                       # keys and values side by side
    assert torch.equal(paged_attention(q, both[:, :, :, 0], both[:, :, :, 1], table, lens), base)
    heads = kc.transpose(1, 2).contiguous().transpose(1, 2), vc.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(paged_attention(q, *heads, table, lens), base)
    qq = torch.zeros(3, 6, 128, dtype=BF, device="cuda")
    qq[:, 1:5, 32:96] = q
    assert torch.equal(paged_attention(qq[:, 1:5, 32:96], kc, vc, table, lens), base)
    assert torch.equal(paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), kc, vc, table, lens), base)
    wide = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    wide[:, :9] = table
    assert torch.equal(paged_attention(q, kc, vc, wide[:, :9], lens), base)
    assert torch.equal(paged_attention(q, kc, vc, table.T.contiguous().T, lens.long()), base)
    one = table[:1].expand(3, 9)                                       # sequences that share their pages
    assert torch.equal(paged_attention(q, kc, vc, one, lens)[1:2],
                       paged_attention(q[1:2], kc, vc, table[:1], lens[1:2]))
    for bad in (torch.cat((kc, kc), -1)[..., 4:68], torch.stack((kc, kc), -1)[..., 0]):
        with pytest.raises(ValueError, match="k_cache"):
            paged_attention(q, bad, vc, table, lens)
    assert not paged_attention(q, kc, vc, table[:, :0], lens).any()     # a table without pages
    assert not paged_attention(q, kc[:0], vc[:0], table, lens).any()    # a cache without pages
    assert paged_attention(q[:0], kc, vc, table[:0], lens[:0]).shape == (0, 4, 64)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: the last pages are read where they lie."""
    from memarch_amd.attention import paged_attention
    page, hkv, d = 64, 8, 128
    pages = (1 << 32) // (page * hkv * d * 2) + 40
    kc = torch.zeros(pages, page, hkv, d, dtype=BF, device="cuda")
    vc = torch.zeros_like(kc)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(4, page, hkv, d, generator=g).bfloat16() for _ in range(2))
    kc[-4:], vc[-4:] = k.cuda(), v.cuda()
    q = torch.randn(1, hkv, d, generator=g).bfloat16()
    lens = torch.tensor([4 * page - 3], dtype=torch.int32)
    table = torch.arange(pages - 4, pages, dtype=torch.int32)[None]
    got = paged_attention(q.cuda(), kc, vc, table.cuda(), lens.cuda())
    ref, tol = orc.paged(q, k, v, torch.arange(4)[None], lens, dtype=BF)
    assert ((got.double().cpu() - ref).abs() <= tol).all()


def test_graph_and_streams():
    from memarch_amd.attention import paged_attention
    cases = [[x.cuda() for x in _case(2, 100, 4, 2, 64, 16, BF, seed=i)] for i in range(3)]
    lens = [torch.tensor([1600 - 300 * i, 5 + 200 * i], dtype=torch.int32, device="cuda") for i in range(3)]
    x, ln = [t.clone() for t in cases[0]], lens[0].clone()
    paged_attention(*x, ln)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):               # two graphs of the same call, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(paged_attention(*x, ln))
        graphs.append(g)
    for i in (1, 2, 0):
        for a, b in zip(x, cases[i]):
            a.copy_(b)
        ln.copy_(lens[i])
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            eager = paged_attention(*cases[i], lens[i])
        torch.cuda.synchronize()
        ref = paged_attention(*cases[i], lens[i])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref) and torch.equal(eager, ref)

"""GPU parity of packed_attention against the fp64 oracle, element by element within the bounds that the oracle derives from
the roundings: sequences of no, one and many rows, queries behind earlier keys and in front of none, rows outside every
sequence, shared key blocks, strides, streams, graphs with other lengths, and against window_attention."""
import pytest
import torch

from oracle import attn_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _cu(lens, first=0):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def _inputs(n, m, hq, hkv, d, dt, seed=0, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    mk = lambda r, h, s=1.0: (torch.randn(r, h, d, generator=g) * s).to(dt)
    return mk(n, hq, gain), mk(m, hkv, gain), mk(m, hkv), mk(n, hq)


def _step(q, k, v, go, cu, cu_k, window=0, sinks=0, scale=None):
    from memarch_amd.attention import packed_attention
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = packed_attention(q, k, v, cu, cu_k, window=window or None, sinks=sinks, scale=scale)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), go))


def _check(q, k, v, go, cu, cu_k=None, window=0, sinks=0, scale=None):
    from memarch_amd.attention import packed_attention
    ref, tol = orc.packed(q, k, v, cu.tolist(), None if cu_k is None else cu_k.tolist(), window, sinks, scale, go, q.dtype)
    dev = [x.cuda() for x in (q, k, v, go)]
    cu, cu_k = cu.cuda(), None if cu_k is None else cu_k.cuda()
    got = _step(*dev, cu, cu_k, window, sinks, scale)
    assert all(x.dtype == q.dtype and x.is_contiguous() for x in got)
    for name, a, r, t in zip(("out", "dq", "dk", "dv"), got, ref, tol):
        a = a.double().cpu()
        assert a.shape == r.shape, name
        err = (a - r).abs()
        assert torch.isfinite(a).all() and (err <= t).all(), (name, float((err - t).max()), float(err.max()))
    alone = packed_attention(*dev[:3], cu, cu_k, window=window or None, sinks=sinks, scale=scale)
    assert torch.equal(alone, got[0])   # without a gradient
    return got


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("lens,hq,hkv,d,window,sinks", [
    ([1], 1, 1, 8, 0, 0), ([0], 2, 1, 64, 0, 0), ([1, 1, 1], 2, 1, 64, 0, 0), ([5, 0, 0, 31, 1], 4, 2, 64, 0, 0),
    ([128, 128], 2, 2, 128, 0, 0), ([127, 129, 1], 2, 1, 128, 0, 0), ([33, 200, 64], 3, 3, 96, 17, 0),
    ([300, 7, 258], 8, 2, 80, 40, 3), ([511, 130], 16, 1, 64, 100, 4), ([64, 63, 65], 16, 16, 128, 0, 0),
    ([260, 1, 390], 8, 8, 72, 130, 130), ([20] * 40, 2, 2, 64, 0, 0)])
def test_parity(dt, lens, hq, hkv, d, window, sinks):
    print(f"packed {lens} {hq} {hkv} {d} {window} {sinks} {dt}", flush=True)
    n = sum(lens)
    _check(*_inputs(n, n, hq, hkv, d, dt, seed=n), _cu(lens), None, window, sinks)


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("lens,keys,hq,hkv,d,window,sinks", [
    ([1], [300], 4, 2, 64, 0, 0), ([1, 1, 1], [1, 129, 0], 2, 1, 128, 0, 0), ([40, 0, 3], [41, 100, 200], 4, 1, 96, 0, 0),
    ([130, 200], [333, 200], 4, 4, 64, 50, 3), ([200, 10, 131], [100, 0, 130], 2, 1, 64, 0, 0),   # more rows than keys
    ([300], [5], 2, 2, 128, 30, 2), ([129, 7], [1, 640], 8, 2, 80, 20, 70)])
def test_queries_behind_earlier_keys(dt, lens, keys, hq, hkv, d, window, sinks):
    """A sequence's queries are its last positions; where there are more queries than keys, the first see nothing."""
    print(f"packed {lens} {keys} {hq} {hkv} {d} {window} {sinks} {dt}", flush=True)
    got = _check(*_inputs(sum(lens), sum(keys), hq, hkv, d, dt, seed=sum(keys)), _cu(lens), _cu(keys), window, sinks)
    at = 0
    for n, m in zip(lens, keys):
        blind = slice(at, at + max(0, n - m))
        assert not got[0][blind].any() and not got[1][blind].any()
        at += n


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
@pytest.mark.parametrize("own_keys", [False, True])
def test_rows_outside_every_sequence(window, sinks, own_keys):
    """Rows before the first sequence and behind the last give 0 and pass nothing on, whatever lies there."""
    lens, keys = [100, 0, 37], [140, 5, 37]
    n, m = 9 + sum(lens) + 200, (5 + sum(keys) + 133 if own_keys else 9 + sum(lens) + 200)
    q, k, v, go = _inputs(n, m, 4, 2, 64, BF, seed=3)
    cu, cu_k = _cu(lens, 9), _cu(keys, 5) if own_keys else None
    ck = cu_k if own_keys else cu
    for x, c, bad in ((q, cu, NAN), (k, ck, INF), (v, ck, NAN), (go, cu, -INF)):
        x[:int(c[0])] = bad
        x[int(c[-1]):] = bad
    got = _check(q, k, v, go, cu, cu_k, window, sinks)
    for x, c in zip(got, (cu, cu, ck, ck)):
        assert not x[:int(c[0])].any() and not x[int(c[-1]):].any()
    # int64 starts, and starts past the rows: they count as the last
    far = torch.cat((cu[:-1].long(), torch.tensor([2 ** 40])))
    if not own_keys:
        same = _step(*(x.cuda() for x in (q, k, v, go)), cu.long().cuda(), None, window, sinks)
        assert all(torch.equal(a, b) for a, b in zip(same, got))
        q, k, v, go = _inputs(n, n, 4, 2, 64, BF, seed=3)
        whole = torch.tensor([9, 109, 109, n], dtype=torch.int32)
        a = _step(*(x.cuda() for x in (q, k, v, go)), far.cuda(), None, window, sinks)
        b = _step(*(x.cuda() for x in (q, k, v, go)), whole.cuda(), None, window, sinks)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bad", ["q", "k", "v", "go"])
def test_a_nan_stays_in_its_sequence(bad):
    """A sequence full of NaN leaves its neighbours' bits alone."""
    lens = [70, 130, 64]
    x = dict(zip(("q", "k", "v", "go"), _inputs(264, 264, 4, 2, 64, BF, seed=8)))
    cu = _cu(lens).cuda()
    base = _step(*(t.cuda() for t in x.values()), cu, None, 50, 3)
    x[bad][70:200] = NAN
    got = _step(*(t.cuda() for t in x.values()), cu, None, 50, 3)
    for a, b in zip(got, base):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[200:], b[200:])
    assert got[0][70:200].isnan().any() or bad == "go"


@pytest.mark.parametrize("lens,keys,hq,hkv,d,window,sinks", [
    ([2300, 40], None, 4, 1, 64, 0, 0),          # every earlier key: a key block's rows shared by several workgroups
    ([2700, 2100, 3], None, 4, 2, 64, 300, 4),   # blocks with first tokens shared, the others not
    ([2200], None, 2, 1, 128, 700, 200),         # two blocks with first tokens
    ([600, 1500], [1900, 2100], 8, 1, 128, 0, 0)])
def test_shared_key_blocks(lens, keys, hq, hkv, d, window, sinks):
    print(f"packed shared {lens} {keys} {hq} {hkv} {d} {window} {sinks}", flush=True)
    keys = keys or lens
    x = _inputs(sum(lens), sum(keys), hq, hkv, d, BF, seed=d)
    got = _check(*x, _cu(lens), _cu(keys), window, sinks)
    again = _step(*(t.cuda() for t in x), _cu(lens).cuda(), _cu(keys).cuda(), window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, again))   # no sum depends on an order


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("lens,keys,hq,hkv,d,window,sinks,first", [
    ([1], [3001], 2, 1, 64, 0, 0, 0), ([1, 2], [4000, 1500], 4, 4, 128, 0, 0, 3), ([300], [5000], 2, 2, 64, 0, 0, 0),
    ([40, 0, 1, 129], [2000, 0, 2600, 1700], 4, 2, 96, 0, 0, 0), ([200, 7], [100, 4000], 2, 1, 128, 0, 0, 9),
    ([2900], None, 2, 1, 64, 0, 0, 0), ([17, 150], [3000, 4100], 2, 1, 128, 2000, 0, 0), ([30], [5000], 4, 1, 80, 1500, 70, 0),
    ([5, 130], [2500, 1100], 1, 1, 8, 2100, 3, 1), ([2], [13000], 1, 1, 64, 0, 0, 0),
    ([33, 100], [3000, 2700], 6, 1, 64, 0, 0, 2), ([70, 200, 31], [2500, 2500, 2500], 8, 1, 128, 0, 0, 0)])
def test_few_rows_behind_many_keys(dt, lens, keys, hq, hkv, d, window, sinks, first):
    """Blocks whose keys are shared by several workgroups, beside some that are too short for it and some that see nothing."""
    from memarch_amd import _lib
    print(f"packed few rows {lens} {keys} {hq} {hkv} {d} {window} {sinks} {dt}", flush=True)
    n, m = first + sum(lens) + 5 * first, first + sum(keys or lens) + 5 * first
    assert _lib.load_serve().mce_pack_fwd_ws_bytes(len(lens), n, m, hq, hkv, d, window, sinks) >= 2 * n * hq * (d + 2) * 4
    x = _inputs(n, m, hq, hkv, d, dt, seed=n)
    cu, cu_k = _cu(lens, first), _cu(keys or lens, first)
    got = _check(*x, cu, cu_k, window, sinks)
    again = _step(*(t.cuda() for t in x), cu.cuda(), cu_k.cuda(), window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_few_rows_large_scores_and_nan():
    """Parts whose maxima lie far apart, and one that holds a NaN."""
    q, k, v, go = _inputs(3, 4000, 2, 1, 64, BF, seed=12)
    k[1000:1100] *= 40.0                                # scores of several hundred in one part
    _check(q, k, v, go, _cu([3]), _cu([4000]))
    k[2009, 0, 3] = NAN                                 # row 0 (position 3997) sees it, rows 1 and 2 do not
    got = _step(*(t.cuda() for t in (q, k, v, go)), _cu([3]).cuda(), _cu([4000]).cuda(), 1989)
    assert got[0][0].isnan().all() and not got[0][1:].isnan().any()
    q, k, v, go = _inputs(3, 4000, 2, 1, 64, BF, seed=12)
    base = _step(*(t.cuda() for t in (q, k, v, go)), _cu([3]).cuda(), _cu([4000]).cuda(), 1500)
    k[:2400], v[:2400] = NAN, INF                       # behind the window of all rows
    got = _step(*(t.cuda() for t in (q, k, v, go)), _cu([3]).cuda(), _cu([4000]).cuda(), 1500)
    assert all(torch.equal(a, b) for a, b in zip(got, base))


def test_few_rows_graph_and_falling_starts():
    """A captured step whose blocks are shared, replayed with other lengths; starts that fall touch nothing outside."""
    q, k, v, go = (t.cuda() for t in _inputs(300, 8000, 2, 1, 64, BF, seed=6))
    from memarch_amd.attention import packed_attention
    cu, cu_k = _cu([100, 200]).cuda(), _cu([4000, 4000]).cuda()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    _step(q, k, v, go, cu, cu_k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(*leaves, cu, cu_k)
        got = (out, *torch.autograd.grad(out, leaves, go))
    for lens, keys in (([100, 200], [4000, 4000]), ([1, 299], [8000, 0]), ([0, 300], [10, 7990]), ([3, 4], [900, 7000]),
                       ([100, 200], [4000, 4000])):
        cu.copy_(_cu(lens))
        cu_k.copy_(_cu(keys))
        graph.replay()
        torch.cuda.synchronize()
        ref = _step(q, k, v, go, cu, cu_k)
        assert all(torch.equal(a, b) for a, b in zip(got, ref)), (lens, keys)
    keep = [t.detach().clone() for t in (q, k, v, go)]
    for falling in ([0, 250, 10], [300, 0, 300], [7, -3, 2]):
        for keys in ([0, 8000, 100], [8000, 0, 8000], [0, 4000, 8000]):
            _step(q, k, v, go, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (falling, keys)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(keep, (q, k, v, go)))


@pytest.mark.parametrize("lens,keys,hq,hkv,d,window,sinks,first", [
    ([3100, 0, 4200, 1, 3700], None, 8, 4, 64, 0, 0, 0), ([2100, 5000, 40, 3000], None, 8, 2, 128, 300, 4, 77),
    ([5000, 300, 2600], [5000, 3000, 2600], 8, 8, 64, 0, 0, 5), ([6000], None, 16, 1, 64, 1000, 0, 0),
    ([129, 4000, 0], [2500, 4001, 2300], 16, 4, 128, 700, 140, 0)])
def test_planned_order(lens, keys, hq, hkv, d, window, sinks, first):
    """Long sequences of many heads are taken in an order of their own: the first and the last group of heads against the
    oracle, and no result hangs on the order."""
    from memarch_amd import _lib
    print(f"packed plan {lens} {keys} {hq} {hkv} {d} {window} {sinks}", flush=True)
    n, m = first + sum(lens) + 100, first + sum(keys or lens) + 100
    assert _lib.load_serve().mce_pack_plan_bytes(len(lens), n, m, hq, hkv, d, window, sinks) > 0
    x = _inputs(n, m, hq, hkv, d, BF, seed=n)
    cu, cu_k = _cu(lens, first), _cu(keys or lens, first)
    dev = [t.cuda() for t in (*x, cu, cu_k)]
    got = _step(*dev, window, sinks)
    again = _step(*dev, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    g = hq // hkv
    for h in {0, hkv - 1}:
        of_q, of_k = slice(h * g, (h + 1) * g), slice(h, h + 1)
        q, k, v, go = x[0][:, of_q], x[1][:, of_k], x[2][:, of_k], x[3][:, of_q]
        ref, tol = orc.packed(q, k, v, cu.tolist(), cu_k.tolist(), window, sinks, None, go, BF)
        for name, a, w, t, use in zip(("out", "dq", "dk", "dv"), got, ref, tol, (of_q, of_q, of_k, of_k)):
            assert ((a[:, use].double().cpu() - w).abs() <= t).all(), (name, h)


def test_planned_graph_and_falling_starts():
    """A planned step captured, replayed with other lengths; and starts that fall, which the plan must not follow outside."""
    from memarch_amd.attention import packed_attention
    q, k, v, go = (t.cuda() for t in _inputs(6000, 6000, 16, 2, 64, BF, seed=4))
    cu = torch.tensor([0, 3000, 6000], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    _step(q, k, v, go, cu, None, 500, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(*leaves, cu, window=500, sinks=2)
        got = (out, *torch.autograd.grad(out, leaves, go))
    for mid, end in ((3000, 6000), (1, 5999), (4500, 4500), (0, 6000), (3000, 6000)):
        cu.copy_(torch.tensor([0, mid, end]))
        graph.replay()
        torch.cuda.synchronize()
        ref = _step(q, k, v, go, cu, None, 500, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, ref)), (mid, end)
    keep = [t.detach().clone() for t in (q, k, v, go)]
    for falling in ([0, 5000, 100], [6000, 0, 6000], [7, -3, 2]):
        for window in (0, 500):
            _step(q, k, v, go, torch.tensor(falling, dtype=torch.int32, device="cuda"), None, window, 2 if window else 0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(keep, (q, k, v, go)))


def test_many_sequences():
    """More sequences than one look at the starts takes (64), and than two do (4096)."""
    for nseq, dt in ((200, BF), (5000, HF)):
        g = torch.Generator().manual_seed(nseq)
        lens = torch.randint(0, 4, (nseq,), generator=g).tolist()
        lens[nseq // 2] = 150
        n = sum(lens)
        _check(*_inputs(n, n, 1, 1, 8, dt, seed=2), _cu(lens), None)
    lens = torch.randint(950, 1250, (70,), generator=g).tolist()   # in planned order
    n = sum(lens)
    _check(*_inputs(n, n, 1, 1, 8, BF, seed=3), _cu(lens), None)


def test_is_window_attention_of_each_sequence():
    """The bits of window_attention on a sequence alone, where the tiles lie alike."""
    from memarch_amd.attention import packed_attention, window_attention
    lens = [300, 128, 77]
    q, k, v, _ = (x.cuda() for x in _inputs(505, 505, 4, 2, 128, BF, seed=1))
    out = packed_attention(q, k, v, _cu(lens).cuda(), window=90, sinks=3)
    at = 0
    for n in lens:
        one = window_attention(q[None, at:at + n], k[None, at:at + n], v[None, at:at + n], window=90, sinks=3)[0]
        assert torch.equal(out[at:at + n], one)
        at += n


def test_strides_and_alignment():
    """Slices of one projection's output are read where they lie; views that cannot be are copied."""
    from memarch_amd.attention import packed_attention
    lens, cu = [90, 41], _cu([90, 41])
    n, hq, hkv, d = 131, 4, 2, 64
    q, k, v, go = _inputs(n, n, hq, hkv, d, BF, seed=4)
    ref = _check(q, k, v, go, cu)
    wide = torch.cat((q, k, v), 1).cuda()
    parts = wide[:, :hq], wide[:, hq:hq + hkv], wide[:, hq + hkv:]
    odd = [torch.empty(n * x.shape[1] * d + 3, dtype=BF, device="cuda")[3:].view(n, -1, d).copy_(x.cuda()) for x in (q, k, v)]
    turned = [x.cuda().transpose(0, 2).contiguous().transpose(0, 2) for x in (q, k, v)]
    for x in (parts, odd, turned):
        got = _step(*x, go.cuda(), cu.cuda(), None)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    every = go.cuda()[:, :1].expand(n, hq, d)   # a broadcast upstream gradient
    a = _step(*parts, every, cu.cuda(), None)
    b = _step(*parts, every.contiguous(), cu.cuda(), None)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    cut = torch.stack((cu, cu), 1).cuda()[:, 0]   # starts that do not lie side by side
    assert torch.equal(packed_attention(*parts, cut), ref[0])


def test_no_rows_no_keys():
    from memarch_amd.attention import packed_attention
    q, k, v, go = (x.cuda() for x in _inputs(5, 7, 2, 1, 64, BF))
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = _step(q, k, v, go, none, none)          # no sequence at all
    assert all(not x.any() for x in got)
    two = torch.tensor([0, 5], device="cuda")
    got = _step(q, k[:0], v[:0], go, two, torch.zeros_like(two))
    assert not got[0].any() and not got[1].any() and got[2].shape == (0, 1, 64)
    got = _step(q[:0], k, v, go[:0], torch.zeros_like(two), torch.tensor([0, 7], device="cuda"))
    assert got[0].shape == (0, 2, 64) and not got[2].any() and not got[3].any()
    assert packed_attention(q[:0], k[:0], v[:0], none).shape == (0, 2, 64)


def test_falling_starts_touch_nothing_outside():
    """Starts that fall are the caller's mistake: results are not defined, but nothing outside the results is written (host
    arithmetic keeps every address inside; guards around the outputs cannot be placed here, so the neighbours' tensors are
    looked at)."""
    q, k, v, go = (x.cuda() for x in _inputs(300, 300, 2, 1, 64, BF))
    keep = [x.clone() for x in (q, k, v, go)]
    for cu in ([0, 200, 50, 300], [300, 0], [5, -7, 4000, 2, 299]):
        _step(q, k, v, go, torch.tensor(cu, dtype=torch.int32, device="cuda"), None)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(keep, (q, k, v, go)))


def test_streams_and_another_current_stream():
    x = [t.cuda() for t in _inputs(400, 400, 4, 2, 64, BF, seed=6)]
    cu = _cu([150, 250]).cuda()
    ref = _step(*x, cu, None)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(_step(*x, cu, None))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, ref))


def _captured(leaves, go, cu):
    from memarch_amd.attention import packed_attention
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(*leaves, cu, window=64, sinks=2)
        grads = torch.autograd.grad(out, leaves, go)
    return graph, (out, *grads)


def test_graph_replayed_with_other_lengths():
    """A captured step replayed with other lengths and inputs, eager work and synchronisations between the replays; and two
    captured steps at a time, each with buffers of its own."""
    q, k, v, go = (t.cuda() for t in _inputs(300, 300, 4, 2, 64, BF, seed=9))
    cu = _cu([100, 200]).cuda()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    _step(q, k, v, go, cu, None, 64, 2)
    torch.cuda.synchronize()
    first, got = _captured(leaves, go, cu)
    second, more = _captured(leaves, go, cu)
    for i, lens in enumerate(([100, 200], [0, 300], [299, 1], [30, 40], [100, 200])):
        with torch.no_grad():
            for t in (q, k, v, go):
                t.mul_(1.0 if i == 0 else -0.75)
        cu.copy_(_cu(lens))
        first.replay()
        second.replay()
        torch.cuda.synchronize()
        ref = _step(q, k, v, go, cu, None, 64, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, ref)), lens
        assert all(torch.equal(a, b) for a, b in zip(more, ref)), lens


def test_capture_beside_an_eager_graph_is_refused():
    """A backward of leaves whose earlier graph is alive is refused under capture; once that graph is gone it is captured."""
    from memarch_amd.attention import packed_attention
    q, k, v, go = (t.cuda() for t in _inputs(70, 70, 2, 1, 64, BF, seed=9))
    cu = _cu([30, 40]).cuda()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    alive = packed_attention(*leaves, cu, window=64, sinks=2)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="graph of the same leaves"):
        _captured(leaves, go, cu)
    torch.cuda.synchronize()
    ref = (alive.detach().clone(), *torch.autograd.grad(alive, leaves, go))
    del alive
    graph, got = _captured(leaves, go, cu)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_autocast_and_modes():
    from memarch_amd.attention import packed_attention
    q, k, v, go = (t.cuda() for t in _inputs(90, 90, 4, 2, 64, BF, seed=2))
    cu = _cu([50, 40]).cuda()
    ref = packed_attention(q, k, v, cu)
    with torch.autocast("cuda", dtype=BF):
        assert torch.equal(packed_attention(q.float(), k.float(), v, cu), ref)
    with torch.inference_mode():
        assert torch.equal(packed_attention(q, k, v, cu), ref)
    leaf = q.float().requires_grad_()
    with torch.autocast("cuda", dtype=BF):
        out = packed_attention(leaf, k, v, cu)
    out.backward(go)
    assert leaf.grad.dtype == torch.float32
    assert torch.equal(leaf.grad, _step(q, k, v, go, cu, None)[1].float())
    x = q.clone().requires_grad_()
    out = packed_attention(x, k, v, cu)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(go)


def test_gradients_against_differences():
    """The loss's difference between two points along each gradient, from the operator's outputs, against the gradient. They may
    differ by the outputs' bounds at both points, by the gradient's, and by what the difference itself is off by (the
    oracle's in 64 bits from its own derivative)."""
    from memarch_amd.attention import packed_attention
    cu = _cu([7, 5])
    x = _inputs(12, 12, 2, 1, 16, HF, seed=12, gain=1.0)
    go = x[3].double()
    grads = _step(*(t.cuda() for t in x), cu.cuda(), None)[1:]
    ref, tol = orc.packed(*x[:3], cu.tolist(), None, 0, 0, None, x[3], HF)
    for i in range(3):
        d = ref[1 + i] / ref[1 + i].square().mean().sqrt()
        out, exact, off, at = [], [], 0.0, []
        for sign in (1, -1):
            y = list(x[:3])
            y[i] = (y[i].double() + sign * 0.0625 * d).half()
            at.append(y[i].double())
            r, t = orc.packed(*y, cu.tolist(), None, 0, 0, None, x[3], HF)
            out.append(float((packed_attention(*(z.cuda() for z in y), cu.cuda()).double().cpu() * go).sum()))
            exact.append(float((r[0] * go).sum()))
            off += float((t[0] * go.abs()).sum())
        move = at[0] - at[1]
        off += abs(exact[0] - exact[1] - float((move * ref[1 + i]).sum())) + float((move.abs() * tol[1 + i]).sum())
        want = float((move * grads[i].double().cpu()).sum())
        assert off < 0.15 * abs(want), (i, off, want)   # the comparison says something
        assert abs(out[0] - out[1] - want) <= off, (i, out, want, off)


def test_calls_from_several_threads():
    """Steps of different kinds from several threads, each on a stream of its own, have the bits of those made alone."""
    import threading
    cases = [([300], [300], 4, 2, 64, 50), ([3], [4000], 4, 1, 64, 0), ([6000, 4000], [6000, 4000], 8, 2, 64, 0),
             ([20, 30], [2500, 2700], 2, 2, 128, 0)]
    made = []
    for lens, keys, hq, hkv, d, window in cases:
        x = [t.cuda() for t in _inputs(sum(lens), sum(keys), hq, hkv, d, BF, seed=d)] + [_cu(lens).cuda(), _cu(keys).cuda()]
        made.append((x, window, _step(*x, window)))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        x, window, ref = made[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = _step(*x, window)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, ref)):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

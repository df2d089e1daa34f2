"""GPU parity of the attention operators against the fp64 oracle (oracle/attn_oracle.py), element by element within the
bounds that the oracle derives from the roundings; their strides, lengths, streams, threads and graphs; and a run of them
together, as a block's training step and as decoding."""
import threading

import pytest
import torch

from oracle import attn_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _inputs(b, t, hq, hkv, d, dt, seed=0, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h, s=1.0: (torch.randn(b, t, h, d, generator=g) * s).to(dt)
    return mk(hq, gain), mk(hkv, gain), mk(hkv), mk(hq)


def _step(q, k, v, go, window, sinks, lengths=None, scale=None):
    from memarch_amd.attention import window_attention
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = window_attention(q, k, v, window=window or None, sinks=sinks, lengths=lengths, scale=scale)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), go))


def _inside(got, ref, tol, names=("out", "dq", "dk", "dv")):
    for n, a, r, t in zip(names, got, ref, tol):
        a = a.double().cpu()
        assert a.shape == r.shape, n
        err = (a - r).abs()
        assert torch.isfinite(a).all() and (err <= t).all(), (n, float((err - t).max()), float(err.max()))


def _check(q, k, v, go, window, sinks, lengths=None, scale=None):
    ref, tol = orc.attention(q, k, v, window, sinks, lengths, scale, go, q.dtype)
    dev = [x.cuda() for x in (q, k, v, go)]
    got = _step(*dev, window, sinks, None if lengths is None else lengths.cuda(), scale)
    assert all(x.dtype == q.dtype and x.is_contiguous() for x in got)
    _inside(got, ref, tol)
    return got


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("b,t,hq,hkv,d,window,sinks", [
    (2, 1, 2, 1, 64, 0, 0), (1, 2, 1, 1, 8, 1, 0), (2, 31, 2, 2, 64, 5, 0), (1, 33, 4, 2, 64, 0, 0),
    (1, 64, 1, 1, 128, 64, 0), (1, 65, 2, 1, 128, 64, 3), (1, 129, 3, 3, 96, 0, 0), (1, 200, 2, 1, 80, 17, 1),
    (1, 257, 2, 2, 128, 100, 70), (2, 300, 2, 1, 64, 33, 5), (1, 300, 8, 1, 72, 40, 0), (1, 511, 1, 1, 128, 130, 130),
    (1, 640, 2, 1, 64, 600, 4), (3, 97, 4, 4, 40, 96, 1)])
def test_parity(dt, b, t, hq, hkv, d, window, sinks):
    print(f"attn {b} {t} {hq} {hkv} {d} {window} {sinks} {dt}", flush=True)
    _check(*_inputs(b, t, hq, hkv, d, dt, seed=t), window, sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,hq,hkv,window,sinks", [
    (4, 300, 4, 2, 0, 0), (8, 190, 1, 1, 50, 3), (2, 333, 16, 8, 100, 130),   # whole heads per XCD: B Hkv = 8, 8, 16
    (1, 520, 8, 8, 0, 0), (1, 260, 16, 8, 20, 0),
    (2, 310, 8, 2, 0, 0), (1, 400, 8, 1, 70, 2), (3, 200, 8, 1, 0, 0)])       # B Hq = 16, 8, 24, B Hkv no multiple of 8
def test_heads_placed_by_xcd(d, b, t, hq, hkv, window, sinks):
    """Batches whose heads are a multiple of the 8 XCDs, with several blocks of rows and keys: every workgroup finds its
    own."""
    print(f"attn xcd {b} {t} {hq} {hkv} {d} {window} {sinks}", flush=True)
    lens = None if b == 1 else torch.tensor([t - 37 * i for i in range(b)]).clamp(min=0)
    _check(*_inputs(b, t, hq, hkv, d, BF, seed=t + d), window, sinks, lens)


@pytest.mark.parametrize("lens", [[0, 0, 0], [1, 0, 150], [150, 64, 65], [127, 128, 129], [200, -3, 3]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
def test_padded_batches(lens, window, sinks):
    """Rows at or past a sequence's length give 0 and pass no gradient on, whatever lies there: NaN and infinities."""
    q, k, v, go = _inputs(3, 150, 4, 2, 64, BF, seed=5)
    for i, n in enumerate(lens):
        for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (go, float("-inf"))):
            x[i, max(n, 0):] = bad
    for dt in (torch.int32, torch.int64):
        got = _check(q, k, v, go, window, sinks, torch.tensor(lens, dtype=dt))
    for i, n in enumerate(lens):
        assert all(not x[i, max(n, 0):].any() for x in got)


@pytest.mark.parametrize("t,n,hq,hkv,d,window,sinks", [(150, 70, 4, 2, 64, 0, 0), (150, 97, 2, 1, 128, 20, 3),
                                                       (2300, 2100, 4, 1, 64, 0, 0)])
@pytest.mark.parametrize("bad", ["q", "k", "v", "go"])
def test_padded_rows_stay_zero_beside_a_nan(bad, t, n, hq, hkv, d, window, sinks):
    """What lies in a sequence's last rows, NaN among it, does not reach the rows behind its length: outputs and gradients
    there are 0. (The third shape shares its key blocks among workgroups, so parts are joined.)"""
    x = dict(zip(("q", "k", "v", "go"), _inputs(1, t, hq, hkv, d, BF, seed=n)))
    x[bad][0, n - 3, 0], x[bad][0, n - 1, 0, 1] = float("nan"), float("inf")
    got = _step(*(x[i].cuda() for i in ("q", "k", "v", "go")), window, sinks, torch.tensor([n], device="cuda"))
    for name, y in zip(("out", "dq", "dk", "dv"), got):
        assert not y[0, n:].any(), name
    assert torch.isfinite(got[0][0, :n - 64]).all()


@pytest.mark.parametrize("window,sinks,at", [(40, 3, 5), (40, 3, 63), (100, 70, 80), (64, 1, 33), (130, 0, 20)])
@pytest.mark.parametrize("d", [64, 128])
def test_a_nan_stays_near_the_rows_that_see_it(d, window, sinks, at):
    """A NaN key and value, beside the first tokens and in the same tile as they, reach no row more than 95 positions behind
    the last that sees them: outputs and dq there have the bits that finite values give."""
    t = 600
    q, k, v, go = (x.cuda() for x in _inputs(1, t, 2, 1, d, BF, seed=at))
    base = _step(q, k, v, go, window, sinks)
    k[0, at], v[0, at] = float("nan"), float("inf")
    got = _step(q, k, v, go, window, sinks)
    far = at + window + 95
    assert got[0][0, at].isnan().all()
    assert all(torch.equal(a[0, far:], b[0, far:]) for a, b in zip(got[:2], base[:2]))


@pytest.mark.parametrize("b,t,hq,hkv,d,window,sinks", [
    (1, 2300, 4, 1, 64, 0, 0),         # every earlier key: rows of a key block shared by several workgroups
    (1, 2300, 4, 1, 128, 1000, 4),     # a window long enough for that, and the block with the first tokens apart
    (1, 2100, 2, 2, 64, 70, 200),      # two blocks with first tokens, each shared
    (2, 1300, 8, 1, 96, 300, 130)])
def test_shared_key_blocks(b, t, hq, hkv, d, window, sinks):
    print(f"attn shared {b} {t} {window} {sinks}", flush=True)
    lens = None if b == 1 else torch.tensor([t, 700])
    _check(*_inputs(b, t, hq, hkv, d, BF, seed=t + d), window, sinks, lens)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t,hq,hkv,window,sinks", [(8, 1100, 4, 1, 0, 0), (4, 1200, 4, 2, 60, 140)])
def test_shared_key_blocks_placed_by_xcd(d, b, t, hq, hkv, window, sinks):
    """B Hkv = 8 and key blocks with several workgroups each (the first tokens', or all without a window)."""
    from memarch_amd import _lib
    need = _lib.load_attn().mce_attn_bwd_ws_bytes(b, t, hq, hkv, d, window, sinks)
    assert need > b * hq * t * 8 + 4 * 128 * d * 4                            # parts there are
    print(f"attn xcd shared {b} {t} {d} {window} {sinks}", flush=True)
    lens = torch.tensor([t - 100 * i for i in range(b)])
    _check(*_inputs(b, t, hq, hkv, d, HF, seed=t + d), window, sinks, lens)


def test_window_as_long_as_the_text_and_longer():
    """A window that holds the whole text is no window; sinks change nothing then."""
    x = [t.cuda() for t in _inputs(2, 200, 4, 2, 64, HF, seed=12)]
    base = _step(*x, 0, 0)
    for window, sinks in ((200, 0), (200, 7), (201, 3), (2 ** 40, 2 ** 40)):
        assert all(torch.equal(a, b) for a, b in zip(_step(*x, window, sinks), base)), window


@pytest.mark.parametrize("scale", [1e-4, 1.0, 3.0])
def test_scales(scale):
    _check(*_inputs(1, 100, 2, 1, 64, BF, seed=6), 30, 0, None, scale)


def test_peaked_scores():
    """Scores up to several hundred apart: rows that are nearly one-hot, maxima that grow along the row."""
    q, k, v, go = _inputs(1, 260, 2, 2, 64, BF, seed=7, gain=4.0)
    k = (k.float() * torch.linspace(0.1, 3.0, 260)[None, :, None, None]).bfloat16()
    _check(q, k, v, go, 0, 0, None, 1.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt,power,scale", [(BF, 0, 2e4), (BF, 10, None), (BF, 0, 1e9), (BF, 14, 1.0), (BF, 58, None),
                                            (HF, 13, None), (HF, 15, None), (HF, 0, 1e12)])
def test_scores_of_any_finite_size(dt, power, scale, d):
    """Scores from 1e6 to 1e36: q and k hold -1, 0 and 1 times a power of two, so that scores are exact and either equal or
    too far apart to share a softmax: a row's output is the mean of v over its highest scores. Exponentials are 1 and 0 then,
    so what rounds is fp32 sums (2^-24 a term) and the result (u). The same from pages for the last row."""
    from memarch_amd.attention import paged_attention, window_attention
    t, n, window, sinks = 200, 183, 70, 3
    g = torch.Generator().manual_seed(power + d)
    q, k = (torch.randint(-1, 2, (2, t, 2, d), generator=g).to(dt) * 2.0 ** power for _ in range(2))
    v = torch.randn(2, t, 2, d, generator=g).to(dt)
    assert torch.isfinite(q).all() and q.dtype == dt
    lens = torch.tensor([t, n])
    see = torch.stack([orc.visible(t, int(i), window, sinks) for i in lens])[:, None]
    s = (q.double().transpose(1, 2) @ k.double().transpose(1, 2).mT).masked_fill(~see, -torch.inf)
    top = (s == s.amax(-1, keepdim=True)) & see
    p = top / top.sum(-1, keepdim=True).clamp(min=1).double()
    vd = v.double().transpose(1, 2)
    ref, mag = p @ vd, p @ vd.abs()
    tol = (torch.finfo(dt).eps / 2 * ref.abs() + (t + 2) * 2.0 ** -24 * mag).transpose(1, 2) * 1.01
    got = window_attention(q.cuda(), k.cuda(), v.cuda(), window=window, sinks=sinks, lengths=lens.cuda(), scale=scale)
    err = (got.double().cpu() - ref.transpose(1, 2)).abs()
    assert (err <= tol).all(), float((err - tol).max())          # (NaN fails it too)
    pad = torch.zeros(2, 8, 2, d, dtype=dt)
    kc, vc = (torch.cat((x, pad), 1).view(26, 16, 2, d).cuda() for x in (k, v))
    last = torch.stack((q[0, t - 1], q[1, n - 1])).cuda()
    out = paged_attention(last, kc, vc, torch.arange(26, device="cuda", dtype=torch.int32).view(2, 13), lens.cuda(),
                          window=window, sinks=sinks, scale=scale)
    for i, r in ((0, t - 1), (1, n - 1)):
        assert ((out[i].double().cpu() - ref[i, :, r]).abs() <= tol[i, r]).all(), i


def test_strided_operands():
    """Slices of one packed projection, head-first layouts, a broadcast batch and head, an unaligned base, a strided last
    dimension; upstream gradients expanded from one value and transposed."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 70, 4 + 2 + 2, 64, generator=g).bfloat16().cuda()
    q, k, v = x[:, :, :4], x[:, :, 4:6], x[:, :, 6:]
    go = torch.randn(2, 70, 4, 64, generator=g).bfloat16().cuda()
    base = _step(q.contiguous(), k.contiguous(), v.contiguous(), go, 20, 2)
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, base))
    assert same(_step(q, k, v, go, 20, 2))
    heads = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    assert same(_step(heads(q), heads(k), heads(v), heads(go), 20, 2))
    last = lambda t: torch.stack((t, t), -1)[..., 0]
    assert same(_step(last(q), last(k), last(v), last(go), 20, 2))

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        return buf.view(t.shape).copy_(t)
    assert same(_step(off(q), off(k), off(v), off(go), 20, 2))
    wide = torch.zeros(2, 70, 8, 100, dtype=BF, device="cuda")       # rows 100 elements apart: not multiples of 8
    wide[..., :64] = x
    assert same(_step(wide[:, :, :4, :64], wide[:, :, 4:6, :64], wide[:, :, 6:, :64], go, 20, 2))
    # one sequence and one head shared by all: gradients summed by autograd over the expanded dimensions
    from memarch_amd.attention import window_attention
    k1 = k[:1, :, :1].contiguous().requires_grad_()
    out = window_attention(q, k1.expand(2, 70, 2, 64), v, window=20)
    (dk1,) = torch.autograd.grad(out.sum(), (k1,))                   # an upstream gradient of stride 0
    full = _step(q, k1.expand(2, 70, 2, 64).contiguous(), v, torch.ones_like(go), 20, 0)[2]
    assert torch.allclose(dk1.float(), full.float().sum((0, 2), keepdim=True), rtol=2 ** -6, atol=2 ** -6)


def test_one_token_strides():
    """A size of 1 may have any stride."""
    q, k, v, go = (x.cuda() for x in _inputs(3, 1, 2, 1, 64, BF, seed=3))
    odd = lambda t: torch.as_strided(t, t.shape, (t.stride(0), 3, t.stride(2) if t.shape[2] > 1 else 5, 1))
    base = _step(q, k, v, go, 4, 0)
    got = _step(odd(q), odd(k), odd(v), odd(go), 4, 0)
    assert all(torch.equal(a, b) for a, b in zip(got, base))
    assert torch.equal(base[0], v.expand(3, 1, 2, 64))


def test_empty():
    from memarch_amd.attention import window_attention
    for shape in ((0, 5), (3, 0)):
        q = torch.zeros(*shape, 4, 64, dtype=BF, device="cuda", requires_grad=True)
        k = torch.zeros(*shape, 2, 64, dtype=BF, device="cuda", requires_grad=True)
        out = window_attention(q, k, k, window=3)
        assert out.shape == q.shape
        out.sum().backward()
        assert q.grad.shape == q.shape and k.grad.shape == k.shape


def test_no_grad_matches_and_only_wanted_gradients():
    from memarch_amd.attention import window_attention
    q, k, v, go = (x.cuda() for x in _inputs(2, 90, 4, 2, 64, HF, seed=4))
    base = _step(q, k, v, go, 30, 1)
    assert torch.equal(window_attention(q, k, v, window=30, sinks=1), base[0])
    with torch.no_grad():
        assert torch.equal(window_attention(q.requires_grad_(), k, v, window=30, sinks=1), base[0])
    vl = v.detach().clone().requires_grad_()
    (dv,) = torch.autograd.grad(window_attention(q.detach(), k, vl, window=30, sinks=1), vl, go)
    assert torch.equal(dv, base[3])
    out = window_attention(q, k, v, window=30)
    with pytest.raises(RuntimeError):     # differentiable once
        (gq,) = torch.autograd.grad(out, q, go, create_graph=True)
        gq.sum().backward()


def test_autocast_and_compile():
    from memarch_amd.attention import window_attention
    q, k, v, go = (x.float().cuda() for x in _inputs(1, 50, 2, 1, 64, BF, seed=2))
    ref = _step(q.bfloat16(), k.bfloat16(), v.bfloat16(), go.bfloat16(), 20, 0)
    ql, kl, vl = (x.clone().requires_grad_() for x in (q, k, v))
    with torch.autocast("cuda", dtype=BF):
        out = window_attention(ql, kl, vl, window=20)
    assert out.dtype == BF and torch.equal(out, ref[0])
    grads = torch.autograd.grad(out, (ql, kl, vl), go.bfloat16())
    assert all(g.dtype == torch.float32 and torch.equal(g, r.float()) for g, r in zip(grads, ref[1:]))
    with pytest.raises(ValueError, match="bfloat16"):
        window_attention(q, k, v)
    f = torch.compile(lambda q, k, v: window_attention(q * 1.0, k, v, window=20) * 2, backend="aot_eager")
    assert torch.equal(f(q.bfloat16(), k.bfloat16(), v.bfloat16()), 2 * ref[0])


def test_no_host_sync():
    q, k, v, go = (x.cuda() for x in _inputs(2, 300, 4, 2, 64, BF))
    lens = torch.tensor([300, 100], device="cuda")
    _step(q, k, v, go, 50, 4, lens)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        _step(q, k, v, go, 50, 4, lens)
    finally:
        torch.cuda.set_sync_debug_mode(0)


@pytest.mark.parametrize("t,window,sinks,ragged", [(200, 0, 0, False), (700, 40, 4, True)])
def test_graph_replays_match_eager(t, window, sinks, ragged):
    print(f"attn graph {t} {window}", flush=True)
    vals = [[x.cuda() for x in _inputs(2, t, 4, 2, 64, BF, seed=i)] for i in range(4)]
    lens = [torch.tensor([t - 7 * i, t // (i + 2)], dtype=torch.int32, device="cuda") for i in range(4)]
    x = [v.clone() for v in vals[0]]
    ln = lens[0].clone() if ragged else None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(*x, window, sinks, ln)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(*x, window, sinks, ln)
    for i in (1, 2, 3, 0):
        for a, b in zip(x, vals[i]):
            a.copy_(b)
        if ragged:
            ln.copy_(lens[i])
        graph.replay()
        torch.cuda.synchronize()
        ref = _step(*vals[i], window, sinks, lens[i] if ragged else None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref)), i


def test_threads_and_streams_match_sequential():
    cases = [[x.cuda() for x in _inputs(1, 400 + 33 * i, 4, 2, 64, BF, seed=i)] for i in range(4)]
    seq = [_step(*c, 50, 4) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(3):
                    got[i] = _step(*cases[i], 50, 4)
            st.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(timeout=100)
    assert not errors and not any(th.is_alive() for th in threads), errors
    for a, b in zip(seq, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_long_text_rows():
    """8192 tokens with a window and first tokens, grouped heads: sampled rows of out and dq, and the gradients of the
    first keys (which every row sees) and of sampled ones, against dense fp64 rows on the GPU's host."""
    t, w, s, hq, hkv, d = 8192, 200, 3, 2, 1, 64
    q, k, v, go = _inputs(1, t, hq, hkv, d, BF, seed=31)
    out, dq, dk, dv = (x.double().cpu() for x in _step(*(x.cuda() for x in (q, k, v, go)), w, s))
    qd, kd, vd, gd = (x[0].double() for x in (q, k, v, go))
    u, scale = 2.0 ** -8, d ** -0.5
    j = torch.arange(t)
    rdk = torch.zeros(t, d, dtype=torch.float64)
    rdv, adk, adv = torch.zeros_like(rdk), torch.zeros_like(rdk), torch.zeros_like(rdk)
    for h in range(hq):
        for i0 in range(0, t, 1024):
            i = torch.arange(i0, i0 + 1024)[:, None]
            see = (j <= i) & ((i - j < w) | (j < s))
            p = torch.softmax((qd[i0:i0 + 1024, h] @ kd[:, 0].T * scale).masked_fill(~see, -torch.inf), -1)
            o = p @ vd[:, 0]
            g = gd[i0:i0 + 1024, h]
            ds = p * (g @ vd[:, 0].T - (g * o).sum(-1, keepdim=True))
            # bounds: P and its error u, dS likewise and the error of d (u sum |go| P|v|); 2^-12 covers the fp32 sums
            ao = p @ vd[:, 0].abs()
            eds = (u + 2 ** -12) * ds.abs() + p * ((u + 2 ** -12) * (g.abs() * ao).sum(-1, keepdim=True))
            rows = slice(i0, i0 + 1024)
            assert ((out[0, rows, h] - o).abs() <= 1.05 * (u * o.abs() + (u + 2 ** -12) * ao)).all()
            ref = scale * ds @ kd[:, 0]
            assert ((dq[0, rows, h] - ref).abs() <= 1.05 * (u * ref.abs() + scale * eds @ kd[:, 0].abs())).all()
            rdk += scale * ds.T @ qd[rows, h]
            rdv += p.T @ g
            adk += scale * eds.T @ qd[rows, h].abs()
            adv += (u + 2 ** -12) * p.T @ g.abs()
    assert ((dk[0, :, 0] - rdk).abs() <= 1.05 * (u * rdk.abs() + adk)).all()
    assert ((dv[0, :, 0] - rdv).abs() <= 1.05 * (u * rdv.abs() + adv)).all()


# ------------------------------------------------------------------------------------------------------- a run of them


def test_a_block_training_step():
    """One packed projection, norms with rotation, window attention, an output projection, the SwiGLU gate and the
    cross-entropy: gradients of every parameter against fp64 autograd of the same formulas (relative Frobenius norm; 16-bit
    activations of six operators in a row, each within 2^-8, amplified by the norms' gains)."""
    from memarch_amd.attention import window_attention
    from memarch_amd.fused_ops import linear_ce, swiglu
    from memarch_amd.rotary import qk_norm_rope, rope_table
    g = torch.Generator().manual_seed(77)
    b, t, hq, hkv, d, vocab = 2, 150, 4, 2, 64, 500
    dm = hq * d
    mk = lambda *s: torch.randn(*s, generator=g) / s[-1] ** 0.5
    par = dict(wqkv=mk((hq + 2 * hkv) * d, dm), wo=mk(dm, dm), wu=mk(2 * dm, dm), wv=mk(vocab, dm),
               qw=1 + 0.1 * torch.randn(d, generator=g), kw=1 + 0.1 * torch.randn(d, generator=g))
    x = torch.randn(b, t, dm, generator=g).bfloat16()
    y = torch.randint(0, vocab, (b, t), generator=g)
    cos, sin = rope_table(t, d)
    p = {n: w.cuda().requires_grad_() for n, w in par.items()}
    xg = x.cuda()
    qkv = (xg @ p["wqkv"].bfloat16().T).view(b, t, hq + 2 * hkv, d)
    q, k = qk_norm_rope(qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], cos.cuda(), sin.cuda(), p["qw"], p["kw"])
    o = window_attention(q, k, qkv[:, :, hq + hkv:], window=40, sinks=2).reshape(b, t, dm)
    h = xg + o @ p["wo"].bfloat16().T
    h = h + swiglu(h @ p["wu"].bfloat16().T)
    loss = linear_ce(h.reshape(-1, dm), p["wv"], y.cuda().reshape(-1)) / (b * t)
    loss.backward()

    r = {n: w.double().requires_grad_() for n, w in par.items()}
    xd = x.double()
    qkv = (xd @ r["wqkv"].T).view(b, t, hq + 2 * hkv, d)
    q = orc.rope(qkv[:, :, :hq], cos, sin, r["qw"])
    k = orc.rope(qkv[:, :, hq:hq + hkv], cos, sin, r["kw"])
    see = orc.visible(t, t, 40, 2)
    kk, vv = (a.repeat_interleave(2, 2).transpose(1, 2) for a in (k, qkv[:, :, hq + hkv:]))
    s = (q.transpose(1, 2) @ kk.mT * d ** -0.5).masked_fill(~see, -torch.inf)
    o = (torch.softmax(s, -1) @ vv).transpose(1, 2).reshape(b, t, dm)
    h = xd + o @ r["wo"].T
    gu = h @ r["wu"].T
    h = h + torch.nn.functional.silu(gu[..., :dm]) * gu[..., dm:]
    ref = torch.nn.functional.cross_entropy((h @ r["wv"].T).reshape(-1, vocab), y.reshape(-1))
    ref.backward()
    assert abs(float(loss) - float(ref)) <= 1e-2 * float(ref)
    for n in par:
        got, want = p[n].grad.double().cpu(), r[n].grad
        assert float((got - want).norm() / want.norm()) <= 3e-2, n


def test_decoding_follows_the_prompt():
    """A prompt through window_attention, then token after token through qk_norm_rope at its position, the cache's page
    and paged_attention: each token's output is the row that window_attention gives for the whole text."""
    from memarch_amd.attention import paged_attention, window_attention
    from memarch_amd.rotary import qk_norm_rope, rope_table
    g = torch.Generator().manual_seed(21)
    b, t, hq, hkv, d, page = 3, 75, 4, 2, 64, 16
    prompt = [60, 41, 1]
    x = torch.randn(b, t, hq + 2 * hkv, d, generator=g).bfloat16().cuda()
    cos, sin = rope_table(t, d, device="cuda")
    q, k = qk_norm_rope(x[:, :, :hq], x[:, :, hq:hq + hkv], cos, sin)
    v = x[:, :, hq + hkv:]
    for window, sinks in ((None, 0), (20, 3)):
        full = window_attention(q, k, v, window=window, sinks=sinks)
        kc = torch.full((20, page, hkv, d), float("nan"), dtype=BF, device="cuda")   # what was never written
        vc = kc.clone()
        table = torch.randperm(20, generator=g)[:15].view(3, 5).int().cuda()
        lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
        for i in range(b):
            for j in range(prompt[i]):
                kc[table[i, j // page].long(), j % page], vc[table[i, j // page].long(), j % page] = k[i, j], v[i, j]
        for _ in range(14):
            pos = lens.long()
            rows = torch.arange(b, device="cuda")
            qn, kn = qk_norm_rope(x[rows, pos, :hq][:, None], x[rows, pos, hq:hq + hkv][:, None], cos, sin,
                                  positions=pos[:, None])
            pg = table[rows, pos // page].long()
            kc[pg, pos % page], vc[pg, pos % page] = kn[:, 0], v[rows, pos]
            lens += 1
            got = paged_attention(qn[:, 0], kc, vc, table, lens, window=window, sinks=sinks)
            want = full[rows, pos].float()
            # both are within (u + u) of the same sum: u |out| each, and u P|v| <= u max|v| each
            tol = 2 * 1.05 * 2.0 ** -8 * (want.abs() + float(v.abs().max()))
            assert torch.isfinite(got).all() and ((got.float() - want).abs() <= tol).all()


def test_backward_twice_inference_and_changed_inputs():
    """A kept graph gives the same gradients again, inference mode the same values, and an input changed between forward
    and backward an error."""
    from memarch_amd.attention import window_attention
    from memarch_amd.rotary import qk_norm_rope, rope_table
    q, k, v, go = (x.cuda() for x in _inputs(2, 150, 4, 2, 64, BF, seed=21))
    cos, sin = rope_table(150, 64, device="cuda")
    w = torch.ones(64, device="cuda")

    def run(q, k, v, n):
        a, b = qk_norm_rope(q, k, cos, sin, w, w)
        return window_attention(a, b, v, window=40, sinks=2, lengths=n)
    n = torch.tensor([150, 77], dtype=torch.int32, device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = run(*leaves, n)
    first = torch.autograd.grad(out, leaves, go, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, leaves, go)))
    with torch.inference_mode():
        assert torch.equal(run(q, k, v, n), out)
    for change in (lambda: n.add_(1), lambda: mid.add_(1)):
        mid = leaves[2] * 1
        out = run(leaves[0], leaves[1], mid, n)
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, leaves, go)

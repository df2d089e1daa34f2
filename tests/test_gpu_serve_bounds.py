"""What the serving operators write where starts fall (the caller's mistake: results are not defined) and lengths are of any size:
nothing outside their own buffers. The C entries get buffers that lie between guards, which have to be as they were afterwards."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
GUARD, FILL = 1 << 16, 0xA5


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class Guarded:
    """Buffers between guards of 64 KiB."""

    def __init__(self):
        self.held = []

    def buf(self, nbytes, fill=FILL):
        room = -(-nbytes // 256) * 256
        whole = torch.full((GUARD + room + GUARD,), FILL, dtype=torch.uint8, device="cuda")
        assert whole.data_ptr() % 256 == 0
        whole[GUARD:GUARD + nbytes] = fill
        self.held.append((whole, nbytes))
        return whole[GUARD:GUARD + nbytes]

    def check(self, what):
        torch.cuda.synchronize()
        for i, (whole, nbytes) in enumerate(self.held):
            assert (whole[:GUARD] == FILL).all() and (whole[GUARD + nbytes:] == FILL).all(), (what, i)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _falling(n, nseq):
    """Starts that fall, of nseq sequences over n rows."""
    g = torch.Generator().manual_seed(nseq)
    yield torch.randint(-n // 4, 2 * n, (nseq + 1,), generator=g)
    yield torch.arange(nseq, -1, -1) * (n // nseq)
    yield torch.where(torch.arange(nseq + 1) % 2 == 0, 0, n)
    yield torch.where(torch.arange(nseq + 1) % 2 == 0, n, 0)
    even = torch.arange(nseq + 1) * (n // nseq)
    even[nseq // 2] = n + 7
    yield even


@pytest.mark.parametrize("nseq,n,m,hq,hkv,d,window,sinks,has", [
    (3, 300, 300, 2, 1, 64, 0, 0, ""), (5, 500, 700, 8, 2, 80, 60, 200, "parts"), (3, 6000, 6000, 16, 4, 64, 500, 3, "plan parts"),
    (3, 6000, 6000, 16, 4, 64, 0, 0, "plan"), (2, 30, 6000, 4, 1, 128, 0, 0, "split"), (70, 70, 2000, 2, 2, 64, 0, 0, ""),
    (40, 1500, 1500, 2, 1, 64, 20, 900, "parts"), (3, 4000, 4000, 16, 4, 64, 200, 8000, "plan parts")])
def test_packed_attention(nseq, n, m, hq, hkv, d, window, sinks, has):
    from memarch_amd import _lib
    print(f"bounds packed {nseq} {n} {m} {hq} {hkv} {d} {window} {sinks}", flush=True)
    lib, size = _lib.load_serve(), (nseq, n, m, hq, hkv, d, window, sinks)
    plan_bytes, fwd_bytes = lib.mce_pack_plan_bytes(*size), lib.mce_pack_fwd_ws_bytes(*size)
    bwd_bytes = lib.mce_pack_bwd_ws_bytes(*size)
    stat = -(-n * hq * 8 // 256) * 256
    assert (plan_bytes > 0) == ("plan" in has) and (fwd_bytes > 0) == ("split" in has)
    assert bwd_bytes > stat if "parts" in has or "split" in has else bwd_bytes >= stat
    g = torch.Generator(device="cuda").manual_seed(0)
    mk = lambda r, h: torch.randn(r, h, d, generator=g, device="cuda").to(BF)
    q, k, v, go = mk(n, hq), mk(m, hkv), mk(m, hkv), mk(n, hq)
    rows = lambda t: (t.data_ptr(), t.shape[1] * d, d)
    stream = torch.cuda.current_stream().cuda_stream
    for i, (cu, cu_k) in enumerate(zip(_falling(n, nseq), _falling(m, nseq))):
        for own_keys in (True,) if n != m else (True, False):
            print(f"  starts {i} {own_keys}", flush=True)
            a, b = _ints(cu.tolist()), _ints(cu_k.tolist())
            at = Guarded()
            out, res, dq = (at.buf(n * hq * d * 2) for _ in range(3))
            dk, dv = (at.buf(m * hkv * d * 2) for _ in range(2))
            lse = at.buf(n * hq * 4, 0)
            plan, ws, wb = at.buf(plan_bytes), at.buf(fwd_bytes, 0), at.buf(bwd_bytes, 0)
            keys = b.data_ptr() if own_keys else None
            _lib.call("mce_pack_fwd", *rows(q), *rows(k), *rows(v), a.data_ptr(), keys, *size, d ** -0.5, 1, out.data_ptr(),
                      res.data_ptr(), lse.data_ptr(), plan.data_ptr(), plan_bytes, ws.data_ptr(), fwd_bytes, stream)
            at.check(("forward", i, own_keys))
            _lib.call("mce_pack_bwd", *rows(q), *rows(k), *rows(v), *rows(go), a.data_ptr(), keys, *size, d ** -0.5, 1,
                      out.data_ptr(), res.data_ptr(), lse.data_ptr(), plan.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                      dv.data_ptr(), wb.data_ptr(), bwd_bytes, stream)
            at.check(("backward", i, own_keys))


def _cache(at, pages, page, block, h, d):
    codes = [at.buf(pages * page * h * d, 0x11).view(F8).view(pages, page, h, d) for _ in range(2)]
    scales = [at.buf(pages * (page // block) * h * 4).view(torch.float32).view(pages, page // block, h) for _ in range(2)]
    for s in scales:
        s.fill_(0.5)
    return codes, scales


@pytest.mark.parametrize("nseq,rows,h,d,page,block", [(3, 130, 2, 64, 16, 8), (70, 900, 3, 96, 32, 32), (2, 3000, 9, 48, 128, 128)])
def test_cache_read(nseq, rows, h, d, page, block):
    from memarch_amd import _lib
    print(f"bounds read {nseq} {rows} {h} {d}", flush=True)
    stream = torch.cuda.current_stream().cuda_stream
    most = -(-rows // page) // 2 + 1
    for i, cu in enumerate(_falling(rows, nseq)):
        at = Guarded()
        (kc, vc), (ks, vs) = _cache(at, nseq * most, page, block, h, d)
        out = [at.buf(rows * h * d * 2) for _ in range(2)]
        table, cu = torch.arange(nseq * most, device="cuda").int(), _ints(cu.tolist())
        strides = (page * h * d, h * d, d)
        _lib.call("mce_cache_read", kc.data_ptr(), *strides, vc.data_ptr(), *strides, ks.data_ptr(), vs.data_ptr(), table.data_ptr(),
                  most, cu.data_ptr(), nseq, rows, h, d, nseq * most, page, block, most, 1, *(x.data_ptr() for x in out), stream)
        at.check(i)
        assert all((x.view(torch.uint8) == 0x11).all() for x in (kc, vc)) and all((s == 0.5).all() for s in (ks, vs))


@pytest.mark.parametrize("nseq,rows,h,d,page,block", [(3, 130, 2, 64, 16, 8), (70, 900, 3, 96, 32, 32), (2, 3000, 9, 48, 128, 128)])
def test_cache_write(nseq, rows, h, d, page, block):
    """Of the cache itself: pages that no table row holds, and slots behind the sequences' ends, are as they were."""
    from memarch_amd import _lib
    print(f"bounds write {nseq} {rows} {h} {d}", flush=True)
    stream = torch.cuda.current_stream().cuda_stream
    most = -(-rows // page) // 2 + 1
    pages = 2 * nseq * most
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(rows, h, d, generator=g, device="cuda").to(BF) for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:nseq * most].view(nseq, most)
    lens = torch.randint(0, most * page + 9, (nseq,), generator=torch.Generator().manual_seed(2))
    mine = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(nseq):
        for j in range(min(int(lens[b]), most * page)):
            mine[table[b, j // page], j % page] = True
    mine = mine.cuda()
    held = mine.view(pages, -1, block).any(2)
    gtable, glens = table.int().cuda(), lens.int().cuda()
    for i, cu in enumerate(_falling(rows, nseq)):
        at = Guarded()
        (kc, vc), (ks, vs) = _cache(at, pages, page, block, h, d)
        cu = _ints(cu.tolist())
        strides = (page * h * d, h * d, d)
        _lib.call("mce_cache_write", k.data_ptr(), h * d, d, v.data_ptr(), h * d, d, kc.data_ptr(), *strides, vc.data_ptr(), *strides,
                  ks.data_ptr(), vs.data_ptr(), gtable.data_ptr(), most, glens.data_ptr(), cu.data_ptr(), nseq, rows, h, d, pages,
                  page, block, most, 1, stream)
        at.check(i)
        for x, s in ((kc, ks), (vc, vs)):
            assert (x.view(torch.uint8)[~mine] == 0x11).all() and (s[~held] == 0.5).all(), i


@pytest.mark.parametrize("b,most,hq,hkv,d,page,window,sinks", [
    (5, 6, 4, 2, 64, 16, 0, 0), (3, 400, 40, 1, 128, 16, 0, 0), (70, 300, 64, 64, 16, 8, 0, 0), (2, 800, 17, 1, 96, 32, 9000, 40)])
def test_cache_attention(b, most, hq, hkv, d, page, window, sinks):
    """Lengths of any number, pages of any number: the output and the workspace only."""
    from memarch_amd import _lib
    print(f"bounds attention {b} {most} {hq} {hkv} {d} {page}", flush=True)
    stream, block = torch.cuda.current_stream().cuda_stream, 8
    need = _lib.load_serve().mce_cache_attn_ws_bytes(b, hq, hkv, d, page, most, window, sinks)
    assert (need > 0) == (most > 6)
    g = torch.Generator().manual_seed(0)
    pages = 50
    q = torch.randn(b, hq, d, generator=g).to(BF).cuda()
    table = torch.randint(-5, pages + 5, (b, most), generator=g).int().cuda()
    for i, lens in enumerate((torch.randint(-9, most * page + 99, (b,), generator=g), torch.full((b,), 2 ** 31 - 1), torch.full((b,), -2 ** 31),
                              torch.arange(b) * (most * page // b))):
        at = Guarded()
        (kc, vc), (ks, vs) = _cache(at, pages, page, block, hkv, d)
        out, ws = at.buf(b * hq * d * 2), at.buf(need, 0)
        lens, strides = _ints(lens.tolist()), (page * hkv * d, hkv * d, d)
        _lib.call("mce_cache_attn", q.data_ptr(), hq * d, d, kc.data_ptr(), *strides, vc.data_ptr(), *strides, ks.data_ptr(),
                  vs.data_ptr(), table.data_ptr(), most, lens.data_ptr(), b, hq, hkv, d, pages, page, block, most, window, sinks,
                  d ** -0.5, 1, out.data_ptr(), ws.data_ptr(), need, stream)
        at.check(i)
        assert all((x.view(torch.uint8) == 0x11).all() for x in (kc, vc)) and all((s == 0.5).all() for s in (ks, vs))
        assert out.view(BF).isfinite().all()

"""The 8-bit cache on the GPU: codes, scales and values bit for bit against the fp64 oracle, the attention within its bounds;
tokens one by one and at once, pages that are not the cache's, values that are not finite, strides, offsets past 32 bits,
streams and graphs; and a run of the serving operators together."""
import pytest
import torch

from oracle import attn_oracle, cache_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class Cache:
    """A cache full of earlier codes on the CPU, and its copy on the GPU."""

    def __init__(self, b, most, hkv, d, page, block, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        pages = b * most + spare
        code = lambda: torch.randint(0, 256, (pages, page, hkv, d), generator=g).to(torch.uint8)
        self.codes = [torch.where(c & 0x7F == 0x7F, c - 1, c).view(F8) for c in (code(), code())]
        self.scales = [torch.exp2(torch.randint(-8, 1, (pages, page // block, hkv), generator=g).float()) for _ in range(2)]
        self.table = torch.randperm(pages, generator=g)[:b * most].view(b, most).int()
        self.upload()

    def upload(self):
        self.dev = [x.cuda() for x in (*self.codes, *self.scales)]
        self.gtable = self.table.cuda()

    @property
    def args(self):
        return (*self.dev, self.gtable)

    def exact(self, i):
        return self.codes[i].float().double(), self.scales[i].double()

    def after(self, x, lengths, cu=None):
        """What the oracle has in the cache after x = (k, v) was written."""
        return [orc.write(x[i], *self.exact(i), self.table, lengths, cu) for i in (0, 1)]

    def same(self, want):
        """Whether the GPU's codes and scales are these; NaN codes alike."""
        for i, (codes, scale) in enumerate(want):
            got = self.dev[i].cpu().float().double()
            assert torch.equal(self.dev[2 + i].cpu().double(), scale), ("scales", i)
            assert torch.equal(got.isnan(), codes.isnan()), ("NaN codes", i)
            assert torch.equal(got.nan_to_num(0.0), codes.nan_to_num(0.0)), ("codes", i)


def _rows(n, h, d, dt, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, n, h, d, generator=g) * torch.exp2(torch.randn(2, n, 1, 1, generator=g) * spread)
    return [t.to(dt) for t in x]


def _cu(lens, first=0):
    return torch.tensor([first] + list(lens)).cumsum(0).int()


# ------------------------------------------------------------------------------------------------------------- write


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hkv,d,page,block,new,lens", [
    (1, 16, 8, 8, [1, 8, 0], [1, 8, 0]), (2, 64, 16, 16, [5, 17, 1], [5, 17, 40]), (3, 128, 16, 8, [33, 1, 30], [48, 41, 30]),
    (4, 96, 32, 32, [31, 33, 2], [70, 96, 96]), (2, 80, 48, 24, [47, 1, 100], [60, 48, 143]), (1, 112, 64, 64, [64, 65, 3], [128, 66, 190]),
    (2, 128, 128, 128, [127, 129, 200], [255, 129, 384]), (5, 48, 128, 16, [7, 0, 300], [300, 100, 384])])
def test_write(dt, hkv, d, page, block, new, lens):
    from memarch_amd.kv_cache import cache_write
    print(f"write {hkv} {d} {page} {block} {new} {lens} {dt}", flush=True)
    c = Cache(3, -(-max(lens) // page), hkv, d, page, block, seed=d + page)
    k, v = _rows(sum(new), hkv, d, dt, seed=d)
    want = c.after((k, v), lens, _cu(new))
    assert cache_write(k.cuda(), v.cuda(), *c.args, torch.tensor(lens).cuda(), _cu(new).cuda()) is None
    c.same(want)
    # the same again changes nothing: the scales cover these tokens already
    cache_write(k.cuda(), v.cuda(), *c.args, torch.tensor(lens).int().cuda(), _cu(new).long().cuda())
    c.same(want)


@pytest.mark.parametrize("d,block", [(64, 8), (128, 16), (96, 128)])
def test_tokens_one_by_one(d, block):
    """A sequence's tokens step by step, each step as the oracle has it, scales growing on the way; what lies behind the last
    token is left as it was."""
    from memarch_amd.kv_cache import cache_write
    c = Cache(2, 2, 2, d, 128, block, seed=block)
    for t in range(1, 20):
        x = _rows(2, 2, d, BF, seed=t, spread=4.0)
        lens = torch.tensor([t, t + 120])
        want = c.after(x, lens)
        c.codes, c.scales = [w[0].float().to(F8) for w in want], [w[1].float() for w in want]
        cache_write(x[0].cuda(), x[1].cuda(), *c.args, lens.cuda())
        c.same(want)


def test_scales_at_their_borders():
    """The largest magnitude on, just below and just above 448 times a power of two, zeros, the smallest and largest
    numbers."""
    from memarch_amd.kv_cache import cache_write
    tops = [448.0, 450.0, 446.0, 1.0, 1.75, 1.7578125, 0.0, 2.0 ** -133, 2.0 ** -92, 1.5 * 2.0 ** -92, 3.3895e38, 7 * 2.0 ** -20]
    c = Cache(len(tops), 1, 1, 16, 8, 8)
    k = torch.zeros(len(tops), 1, 16)
    for i, t in enumerate(tops):
        k[i, 0] = torch.linspace(-1, 1, 16) * t
        k[i, 0, 3] = t
    k = k.to(BF)
    lens = torch.ones(len(tops), dtype=torch.int32)
    want = c.after((k, -k), lens)
    cache_write(k.cuda(), -k.cuda(), *c.args, lens.cuda())
    c.same(want)


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
def test_every_rounding(dt):
    """All finite numbers of the type below a block's largest, at the scale 1: to nearest, ties to even, subnormal codes."""
    from memarch_amd.kv_cache import cache_write
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
    x = torch.zeros(65536 // 16 + 8, 16)
    ok = bits.float().abs() <= 448
    x.view(-1)[:65536] = torch.where(ok, bits.float(), torch.zeros(()))
    n = x.shape[0] // 8 * 8
    x = x[:n].view(n // 8, 8, 16)
    x[:, 0, 0] = 448.0
    b = n // 8
    c = Cache(b, 1, 1, 16, 8, 8)
    k = x.view(n, 1, 16).to(dt)
    lens = torch.full((b,), 8)
    cu = _cu([8] * b)
    cache_write(k.cuda(), k.cuda(), *c.args, lens.cuda(), cu.cuda())
    got = c.dev[0].cpu().float()[c.table[:, 0].long()].view(n, 1, 16)
    assert torch.equal(c.dev[2].cpu()[c.table[:, 0].long()], torch.ones(b, 1, 1))
    assert torch.equal(got.double(), orc.nearest8(k.double()))


def test_values_that_are_not_finite():
    """They become NaN codes, and the others' scale is that of the finite ones."""
    from memarch_amd.kv_cache import cache_write
    for dt in (BF, HF):
        c = Cache(2, 2, 2, 64, 16, 16)
        k, v = _rows(20, 2, 64, dt, spread=1.0)
        k[3, 0, 5], k[4, 1, 60], v[11, 0, 0], k[12] = NAN, INF, -INF, INF
        want = c.after((k, v), [9, 30], _cu([9, 11]))
        cache_write(k.cuda(), v.cuda(), *c.args, torch.tensor([9, 30]).cuda(), _cu([9, 11]).cuda())
        c.same(want)


def test_pages_that_are_not_the_caches():
    """Tokens in pages of -1, past the cache or past the table, more new tokens than a length, rows outside every sequence:
    left out; everything else is written, and nothing more."""
    from memarch_amd.kv_cache import cache_read, cache_write
    c = Cache(4, 3, 2, 64, 16, 8)
    c.table[0, 1], c.table[1, 0], c.table[2, 2] = -1, c.codes[0].shape[0], 2 ** 31 - 1
    c.upload()
    new, lens = [40, 20, 48, 10], [48, 36, 70, 4]      # sequence 2 past its table, sequence 3 shorter than its rows
    cu = _cu(new, 5)
    k, v = _rows(5 + sum(new) + 9, 2, 64, BF)
    want = c.after((k, v), lens, cu)
    cache_write(k.cuda(), v.cuda(), *c.args, torch.tensor(lens).cuda(), cu.cuda())
    c.same(want)
    back = _cu([48, 60, 3, 0], 2)
    got = cache_read(*c.args, back.cuda(), 130)
    for i in (0, 1):
        assert torch.equal(got[i].double().cpu(), orc.read(orc.values(*want[i]), c.table, back, 130).to(BF).double())


@pytest.mark.parametrize("d,page,block", [(128, 64, 16), (64, 128, 128)])
def test_large_batches(d, page, block):
    """64 MiB of rows and more are read, and of results written, past the caches: the same codes, scales and values as in
    pieces that are not."""
    from memarch_amd.kv_cache import cache_read, cache_write
    n, hkv = 2 ** 17, 256 // d                       # 128 MiB of keys and values
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(n, hkv, d, generator=g, device="cuda").to(BF) for _ in range(2))
    table = torch.randperm(n // page, generator=torch.Generator().manual_seed(1)).int().cuda()[None]
    new = lambda: [torch.zeros(n // page, page, hkv, d, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)] + \
        [torch.zeros(n // page, page // block, hkv, device="cuda") for _ in range(2)]
    once, parts = new(), new()
    cu = lambda m: torch.tensor([0, m], device="cuda")
    cache_write(k, v, *once, table, torch.tensor([n]).cuda(), cu(n))
    for i in range(0, n, n // 8):
        cache_write(k[i:i + n // 8], v[i:i + n // 8], *parts, table, torch.tensor([i + n // 8]).cuda(), cu(n // 8))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(once[:2], parts[:2]))
    assert all(torch.equal(a, b) and a.min() > 0 for a, b in zip(once[2:], parts[2:]))
    got = cache_read(*once, table, cu(n), n)
    for x, c, s, src in zip(got, once[:2], once[2:], (k, v)):
        want = (c.float() * s.repeat_interleave(block, 1)[..., None])[table[0].long()].flatten(0, 1).to(BF)
        assert torch.equal(x, want)
        assert ((x.float() - src.float()).abs() <= src.float().abs() * 2.0 ** -4 + 2.0 ** -10 * s.max()).all()
    few = cache_read(*once, table, cu(n // 8), n // 8)
    assert torch.equal(few[0], got[0][:n // 8]) and torch.equal(few[1], got[1][:n // 8])


def test_nothing_to_write():
    from memarch_amd.kv_cache import cache_attention, cache_read, cache_write
    c = Cache(2, 1, 2, 64, 16, 16)
    none = [x.double() for x in (c.codes[0].float(), c.scales[0], c.codes[1].float(), c.scales[1])]
    k, v = (x.cuda() for x in _rows(6, 2, 64, BF))
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    lens = torch.tensor([0, -5]).cuda()
    cache_write(k[:0], v[:0], *c.args, lens, zero)
    cache_write(k, v, *c.args, lens, zero)
    cache_write(k[:2], v[:2], *c.args, lens)
    cache_write(k[:0], v[:0], *c.dev, c.gtable[:0], lens[:0])
    cache_write(k[:2], v[:2], *c.dev, c.gtable[:, :0], lens + 9)
    empty = [x[:0] for x in c.dev]
    cache_write(k[:2], v[:2], *empty, c.gtable, lens + 9)
    c.same([(none[0], none[1]), (none[2], none[3])])
    assert not any(x.any() for x in cache_read(*empty, c.gtable, torch.tensor([0, 3, 5]).cuda(), 6))
    assert not any(x.any() for x in cache_read(*c.args, zero, 7))
    assert cache_read(*c.args, zero, 0)[0].shape == (0, 2, 64)
    assert not cache_attention(k[:2], *empty, c.gtable, lens + 9).any()
    assert not cache_attention(k[:2], *c.dev, c.gtable[:, :0], lens + 9).any()
    assert not cache_attention(k[:2], *c.args, lens).any()
    assert cache_attention(k[:0], *c.dev, c.gtable[:0], lens[:0]).shape == (0, 2, 64)


# -------------------------------------------------------------------------------------------------------------- read


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hkv,d,page,block,lens", [
    (1, 16, 8, 8, [1, 16, 0]), (2, 64, 16, 16, [5, 48, 7]), (3, 128, 24, 8, [70, 1, 23]), (16, 96, 32, 16, [64, 33, 31]),
    (9, 48, 16, 8, [3, 2, 1]), (5, 112, 128, 128, [129, 380, 100])])
def test_read(dt, hkv, d, page, block, lens):
    from memarch_amd.kv_cache import cache_read
    print(f"read {hkv} {d} {page} {block} {lens} {dt}", flush=True)
    c = Cache(3, -(-max(lens) // page), hkv, d, page, block, seed=d)
    for first, more in ((0, 0), (3, 11)):
        cu = _cu(lens, first)
        rows = first + sum(lens) + more
        got = cache_read(*c.args, cu.cuda(), rows, dtype=dt)
        for i in (0, 1):
            assert got[i].dtype == dt and got[i].is_contiguous()
            want = orc.read(orc.values(*c.exact(i)), c.table, cu, rows)
            assert torch.equal(got[i].cpu(), want.to(dt)), i
    falling = torch.tensor([0, 50, 10, rows + 70])     # not defined, but inside the results
    cache_read(*c.args, falling.cuda(), rows, dtype=dt)
    torch.cuda.synchronize()


def test_read_past_the_types_range():
    """Beyond fp16's largest value: that value, with its sign; NaN codes stay NaN."""
    from memarch_amd.kv_cache import cache_read
    c = Cache(1, 1, 1, 16, 8, 8)
    c.scales[0][:] = 2.0 ** 9
    c.codes[0][:, 1] = torch.full((16,), NAN).to(F8)
    c.upload()
    got = cache_read(*c.args, torch.tensor([0, 8]).cuda(), 8, dtype=HF)[0].cpu().float()
    want = orc.values(*c.exact(0))[int(c.table[0, 0])].clamp(-65504, 65504).float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


# --------------------------------------------------------------------------------------------------------- attention


def _attend(c, q, lens, window=0, sinks=0, scale=None):
    from memarch_amd.kv_cache import cache_attention
    (kc, ks), (vc, vs) = c.exact(0), c.exact(1)
    ref, tol = orc.attention(q, kc, ks, vc, vs, c.table, lens, window, sinks, scale, q.dtype)
    got = cache_attention(q.cuda(), *c.args, lens.cuda(), window=window or None, sinks=sinks, scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))
    return got


def _filled(b, most, hkv, d, page, block, seed=0, spread=1.0, spare=3):
    """A cache of ordinary keys and values (the codes of random bits give scores that leave one key)."""
    c = Cache(b, most, hkv, d, page, block, seed, spare)
    g = torch.Generator().manual_seed(seed + 1)
    for i in (0, 1):
        x = torch.randn(c.codes[i].shape, generator=g)
        x *= torch.exp2(spread * torch.randn(*x.shape[:2], 1, 1, generator=g)) if i else 1.0
        s = x.abs().view(x.shape[0], -1, block, hkv, d).amax((2, 4))
        c.scales[i] = torch.exp2(torch.ceil(torch.log2(s / 448)))
        c.codes[i] = (x / c.scales[i].repeat_interleave(block, 1)[..., None]).to(F8)
    c.upload()
    return c


def _q(b, hq, d, dt, seed=0):
    return (1.5 * torch.randn(b, hq, d, generator=torch.Generator().manual_seed(seed))).to(dt)


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d,page,block,most,lens", [
    (1, 1, 64, 16, 16, 2, [1, 32, 0]), (2, 1, 16, 8, 8, 9, [72, 71, 65]), (4, 4, 128, 16, 8, 5, [80, 33, 31]),
    (8, 2, 96, 24, 24, 4, [96, 95, 25]), (16, 1, 128, 64, 32, 2, [128, 64, 63]), (40, 1, 64, 16, 16, 3, [48, 17, 16]),
    (64, 2, 128, 8, 8, 6, [48, 47, 1]), (17, 1, 128, 32, 16, 20, [640, 333, 2]), (4, 2, 80, 40, 40, 20, [800, 401, 399]),
    (2, 2, 64, 128, 128, 12, [1536, 1025, 513]), (6, 2, 128, 16, 16, 200, [3200, 1111, 7]), (3, 3, 48, 64, 64, 4, [250, 8, 129])])
def test_attention(dt, hq, hkv, d, page, block, most, lens):
    print(f"attention {hq} {hkv} {d} {page} {block} {lens} {dt}", flush=True)
    _attend(_filled(3, most, hkv, d, page, block, seed=d + page), _q(3, hq, d, dt), torch.tensor(lens, dtype=torch.int32))


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (32, 0), (33, 4), (100, 40), (500, 3), (5000, 7)])
@pytest.mark.parametrize("hq,hkv,d,dt", [(4, 2, 64, BF), (16, 1, 128, HF), (20, 1, 96, BF)])
def test_windows(window, sinks, hq, hkv, d, dt):
    c = _filled(4, 60, hkv, d, 16, 8, seed=window)
    _attend(c, _q(4, hq, d, dt), torch.tensor([960, 517, 33, 1]), window, sinks)


@pytest.mark.parametrize("hq,hkv,d,page,block,most,lens,window,sinks", [
    (4, 1, 128, 64, 64, 700, [44800], 0, 0), (2, 1, 64, 16, 8, 2500, [39999], 30000, 20), (1, 1, 16, 128, 32, 3080, [393216], 0, 0),
    (2, 2, 64, 64, 16, 700, [44800, 20000], 0, 0)])
def test_many_parts(hq, hkv, d, page, block, most, lens, window, sinks):
    from memarch_amd import _lib
    b = len(lens)
    need = _lib.load_serve().mce_cache_attn_ws_bytes(b, hq, hkv, d, page, most, window, sinks)
    assert need >= 20 * b * hq * d * 4                 # parts by the dozen, or more than the joining wave has lanes
    c = _filled(b, most, hkv, d, page, block, seed=9)
    first = _attend(c, _q(b, hq, d, BF), torch.tensor(lens), window, sinks)
    assert torch.equal(first, _attend(c, _q(b, hq, d, BF), torch.tensor(lens), window, sinks))


@pytest.mark.parametrize("hq,hkv,d,most,lens,w", [
    (64, 64, 16, 104, [0, 1, 1664, 0, 700, 33, 32, 31, 64, 2, 0, 0, 1664, 1500, 3, 256, 5, 90, 0, 1024], 16),
    (128, 64, 16, 104, [1664] * 3 + [0] * 16 + [40], 16), (1024, 1024, 16, 62, [992, 500], 1)])
def test_more_sequences_than_workgroups(hq, hkv, d, most, lens, w):
    """A workgroup takes several sequences, and those that go on past its end are found from the ends."""
    from memarch_amd import _lib
    b = len(lens)
    assert _lib.load_serve().mce_cache_attn_ws_bytes(b, hq, hkv, d, 16, most, 0, 0) == 2 * w * hq * (d * 4 + 8) and b > w
    c = _filled(b, most, hkv, d, 16, 16, seed=3)
    first = _attend(c, _q(b, hq, d, BF), torch.tensor(lens))
    assert torch.equal(first, _attend(c, _q(b, hq, d, BF), torch.tensor(lens)))


def test_scales_far_apart():
    """Blocks whose scales differ by up to 2^40 in the keys and the values: nothing overflows, and in fp16 what the bound
    allows for."""
    for dt in (BF, HF):
        c = _filled(2, 8, 2, 64, 16, 8, seed=4)
        g = torch.Generator().manual_seed(1)
        c.scales[0] *= torch.exp2(torch.randint(-20, 2, c.scales[0].shape, generator=g).float())
        c.scales[1] *= torch.exp2(torch.randint(-20, 21, c.scales[1].shape, generator=g).float() // (1 if dt is BF else 8))
        c.upload()
        _attend(c, _q(2, 4, 64, dt), torch.tensor([128, 77]))
    c = _filled(2, 8, 2, 64, 16, 8, seed=4)
    c.scales = [s * f for s, f in zip(c.scales, (1.3, 0.7))]   # scales that are no powers of two
    c.upload()
    _attend(c, _q(2, 4, 64, BF), torch.tensor([128, 77]))


def test_large_scores():
    """Scores of thousands: one key is left, whose value comes out to its own rounding."""
    c = _filled(3, 20, 2, 128, 16, 16, seed=2)
    _attend(c, _q(3, 8, 128, BF), torch.tensor([320, 200, 31]), scale=40.0)


@pytest.mark.parametrize("hq", [4, 40])
def test_what_is_not_seen_does_not_matter(hq):
    """NaN codes and scales of any kind behind a sequence's end, before its window and in pages that no table holds, pages
    outside the cache in the middle of a sequence, and a sequence none of whose pages is the cache's."""
    d, page, block = 64, 16, 8
    c = _filled(4, 12, 2, d, page, block, seed=3)
    lens = torch.tensor([100, 37, 192, 64])
    c.table[2, 4], c.table[2, 5], c.table[0, 0] = -1, 10 ** 6, -7
    c.table[3] = -1
    c.upload()
    q = _q(4, hq, d, BF)
    for window, sinks in ((0, 0), (20, 3)):
        ref = _attend(c, q, lens, window, sinks)
        assert not ref[3].any()
        dirty = Cache(4, 12, 2, d, page, block, seed=3)
        dirty.table = c.table
        seen = torch.zeros(c.codes[0].shape[:2], dtype=torch.bool)
        for b, n in enumerate(lens.tolist()):
            for j in range(n):
                pg = int(c.table[b, j // page])
                if 0 <= pg < seen.shape[0] and (not window or n - 1 - j < window or j < sinks):
                    seen[pg, j % page] = True
        used = seen.view(seen.shape[0], -1, block).any(2)
        for i in (0, 1):
            bits = torch.where(seen[..., None, None], c.codes[i].view(torch.uint8), torch.tensor(0x7F, dtype=torch.uint8))
            dirty.codes[i] = bits.view(F8)
            for bad in (NAN, INF, 0.0):
                dirty.scales[i] = torch.where(used[..., None], c.scales[i], torch.tensor(bad))
        for bad in (NAN, INF, 0.0, -1.0):
            for i in (0, 1):
                dirty.scales[i] = torch.where(used[..., None], c.scales[i], torch.tensor(bad))
            dirty.upload()
            from memarch_amd.kv_cache import cache_attention
            got = cache_attention(q.cuda(), *dirty.args, lens.cuda(), window=window or None, sinks=sinks)
            assert torch.equal(got, ref), (window, bad)


def test_a_nan_that_is_seen_comes_out():
    from memarch_amd.kv_cache import cache_attention
    c = _filled(2, 4, 2, 64, 16, 16)
    c.codes[0][int(c.table[0, 1]), 3, 0, 7] = torch.tensor(NAN).to(F8)
    c.codes[1][int(c.table[1, 0]), 2, 1, 9] = torch.tensor(NAN).to(F8)
    c.upload()
    out = cache_attention(_q(2, 4, 64, BF).cuda(), *c.args, torch.tensor([40, 40]).cuda()).cpu()
    assert out[0, :2].isnan().all() and out[0, 2:].isfinite().all()
    assert out[1, 2:, 9].isnan().all() and out[1, :2].isfinite().all() and out[1, 2:, :9].isfinite().all()


# ----------------------------------------------------------------------------------------------- where things lie


def test_strided_caches_and_rows():
    """Keys and values side by side in one tensor, heads outside slots, slices of a projection, a table inside a wider one;
    and caches that cannot be read where they lie are refused."""
    from memarch_amd.kv_cache import cache_attention, cache_read, cache_write
    b, most, hkv, d, page, block = 2, 3, 2, 64, 16, 8
    c = _filled(b, most, hkv, d, page, block)
    pages = c.codes[0].shape[0]
    both = torch.zeros(pages, 2, page, hkv, d, dtype=torch.uint8, device="cuda")
    turned = torch.zeros(2, pages, hkv, page, d, dtype=torch.uint8, device="cuda")
    for i in (0, 1):
        both[:, i] = c.dev[i].view(torch.uint8)
        turned[i] = c.dev[i].view(torch.uint8).transpose(1, 2)
    wide = torch.full((b, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:5] = c.gtable
    x = torch.stack(_rows(2 * 5, hkv, d, BF, seed=1), 1).cuda()   # [n, k or v, h, d]
    new, lens, cu = [5, 5], torch.tensor([20, 41]), _cu([5, 5])
    want = c.after((x[:, 0].cpu(), x[:, 1].cpu()), lens, cu)
    cache_write(x[:, 0], x[:, 1], *c.args, lens.cuda(), cu.cuda())
    c.same(want)
    q = _q(b, 4, d, BF).cuda()
    cur = _cu([20, 41]).cuda()
    ref, back = cache_attention(q, *c.args, lens.cuda()), cache_read(*c.args, cur, 61)
    for kc, vc in ((both[:, 0].view(F8), both[:, 1].view(F8)),
                   (turned[0].view(F8).transpose(1, 2), turned[1].view(F8).transpose(1, 2))):
        scales = [s.cuda() for s in c.scales]
        cache_write(x[:, 0].contiguous(), x[:, 1].transpose(0, 2).contiguous().transpose(0, 2), kc, vc, *scales, wide[:, 2:5],
                    lens.cuda(), cu.cuda())
        assert all(torch.equal(a.float(), e.float()) for a, e in zip((kc, vc), c.dev[:2]))
        assert torch.equal(cache_attention(q, kc, vc, *scales, wide[:, 2:5], lens.cuda()), ref)
        odd = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view_as(q).copy_(q)
        assert torch.equal(cache_attention(odd, kc, vc, *scales, c.gtable.t().contiguous().t(), lens.cuda()), ref)
        assert all(torch.equal(a, e) for a, e in zip(cache_read(kc, vc, *scales, wide[:, 2:5], cur, 61), back))
    for bad in (torch.zeros(pages * page * hkv * d + 8, dtype=torch.uint8, device="cuda")[8:].view(F8).view_as(c.dev[0]),
                c.dev[0].view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(F8)):
        with pytest.raises(ValueError, match="contiguous last dimension"):
            cache_attention(q, bad, c.dev[1], *c.args[2:], lens.cuda())
    with pytest.raises(ValueError, match="scales must be contiguous"):
        cache_read(*c.dev[:2], c.dev[2].transpose(0, 1).contiguous().transpose(0, 1), c.dev[3], c.gtable, cur, 61)


def test_offsets_past_32_bits():
    """Pages 4 GiB apart: written, read and attended."""
    from memarch_amd.kv_cache import cache_attention, cache_read, cache_write
    page, hkv, d = 128, 16, 128
    pages = 20000                                       # 5.2 GB a cache
    kc = torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device="cuda").view(F8)
    vc = torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device="cuda").view(F8)
    ks = torch.ones(pages, 2, hkv, device="cuda")
    vs = torch.ones_like(ks)
    table = torch.tensor([[pages - 1, 3], [17000, 18000]], dtype=torch.int32)
    k, v = _rows(300, hkv, d, BF, spread=1.0)
    cu, lens = _cu([140, 160]), torch.tensor([140, 160])
    cache_write(k.cuda(), v.cuda(), kc, vc, ks, vs, table.cuda(), lens.cuda(), cu.cuda())
    small = Cache(2, 2, hkv, d, page, 64, spare=0)
    small.table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    small.upload()
    cache_write(k.cuda(), v.cuda(), *small.args, lens.cuda(), cu.cuda())
    a, b = cache_read(kc, vc, ks, vs, table.cuda(), cu.cuda(), 300), cache_read(*small.args, cu.cuda(), 300)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[0][:, 3].any()
    q = _q(2, 16, d, BF).cuda()
    assert torch.equal(cache_attention(q, kc, vc, ks, vs, table.cuda(), lens.cuda()), cache_attention(q, *small.args, lens.cuda()))
    assert int((kc.view(torch.uint8).view(pages, -1) != 0).any(1).sum()) == 4


def test_streams_and_graphs():
    """A decoding step (write, then attend) on side streams and captured: replayed with other lengths and rows, two graphs
    with buffers of their own, eager work between the replays."""
    from memarch_amd.kv_cache import cache_attention, cache_write
    b, hq, hkv, d = 3, 8, 2, 128
    c = _filled(b, 40, hkv, d, 16, 16, seed=5)
    keep = [x.clone() for x in c.dev]
    lens = torch.tensor([500, 1, 640], dtype=torch.int32).cuda()
    k, v = (x.cuda() for x in _rows(b, hkv, d, BF, spread=2.0))
    q = _q(b, hq, d, BF).cuda()

    def step(dev):
        cache_write(k, v, *dev, c.gtable, lens)
        return cache_attention(q, *dev, c.gtable, lens)

    ref = step([x.clone() for x in keep])
    torch.cuda.synchronize()
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = step([x.clone() for x in keep])
        torch.cuda.synchronize()
        assert torch.equal(got, ref)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        dev = [x.clone() for x in keep]
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = step(dev)
        graphs.append((g, dev, out))
    for i in range(4):
        lens.copy_(torch.tensor([500 + i, 1 + 200 * i, 640 - 7 * i]))
        for t in (k, v, q):
            t.mul_(-1.5)
        want = [x.clone() for x in keep]
        expect = step(want)
        for g, dev, out in graphs:
            for x, y in zip(dev, keep):
                x.copy_(y)
            g.replay()
        torch.cuda.synchronize()
        for g, dev, out in graphs:
            assert torch.equal(out, expect), i
            assert all(torch.equal(x.float(), y.float()) for x, y in zip(dev, want)), i


def test_inference_mode_and_versions():
    from memarch_amd.kv_cache import cache_attention, cache_read, cache_write
    c = _filled(2, 2, 2, 64, 16, 16)
    k, v = (x.cuda() for x in _rows(2, 2, 64, BF))
    lens = torch.tensor([5, 9]).cuda()
    before = [x._version for x in c.dev]
    cache_write(k.requires_grad_(), v, *c.args, lens)
    assert all(x._version > y for x, y in zip(c.dev, before))
    q = _q(2, 4, 64, BF).cuda().requires_grad_()
    out = cache_attention(q, *c.args, lens)
    assert not out.requires_grad
    with torch.inference_mode():
        dev = [x.clone() for x in c.dev]
        cache_write(k, v, *dev, c.gtable, lens)
        assert torch.equal(cache_attention(q, *dev, c.gtable, lens), out)
        assert cache_read(*dev, c.gtable, _cu([5, 9]).cuda(), 14)[0].shape == (14, 2, 64)


# ------------------------------------------------------------------------------------------------------ as they are used


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 4)])
def test_serving_run(window, sinks):
    """Prompts in pieces of different lengths, then tokens one by one: rotation, writing, reading back, attention of the
    pieces over what is in the cache, attention of each new token; every output against the fp64 oracle of what the cache
    holds."""
    from memarch_amd.attention import packed_attention
    from memarch_amd.kv_cache import cache_attention, cache_read, cache_write
    from memarch_amd.rotary import qk_norm_rope, rope_table
    b, hq, hkv, d, page, block = 3, 4, 2, 64, 16, 8
    c = Cache(b, 8, hkv, d, page, block, seed=7)
    cos, sin = (t.cuda() for t in rope_table(256, d))
    lens = torch.zeros(b, dtype=torch.int64)
    g = torch.Generator().manual_seed(0)
    for piece in ([17, 40, 1], [30, 0, 25], [1, 1, 1], [1, 1, 1], [9, 3, 20], [1, 1, 1]):
        n = sum(piece)
        x = torch.randn(1, n, hq + 2 * hkv, d, generator=g).to(BF).cuda()
        pos = torch.cat([torch.arange(int(a), int(a) + m) for a, m in zip(lens, piece)])[None].cuda()
        q, k = qk_norm_rope(x[:, :, :hq], x[:, :, hq:hq + hkv], cos, sin, positions=pos)
        q, k, v = q[0], k[0], x[0, :, hq + hkv:]
        lens = lens + torch.tensor(piece)
        cu = _cu(piece)
        want = c.after((k.cpu(), v.cpu()), lens, cu)
        cache_write(k, v, *c.args, lens.cuda(), None if piece == [1, 1, 1] else cu.cuda())
        c.same(want)
        c.codes, c.scales = [w[0].float().to(F8) for w in want], [w[1].float() for w in want]
        if piece == [1, 1, 1]:
            _attend(c, q.cpu(), lens, window, sinks)
            continue
        cu_k = _cu(lens.tolist())
        kk, vv = cache_read(*c.args, cu_k.cuda(), int(lens.sum()))
        for got, w in zip((kk, vv), want):
            assert torch.equal(got.double().cpu(), orc.read(orc.values(*w), c.table, cu_k, int(lens.sum())))
        out = packed_attention(q, kk, vv, cu.cuda(), cu_k.cuda(), window=window or None, sinks=sinks)
        (ref,), (tol,) = attn_oracle.packed(q.cpu(), kk.cpu(), vv.cpu(), cu.tolist(), cu_k.tolist(), window, sinks, None, None, BF)
        assert ((out.double().cpu() - ref).abs() <= tol).all()

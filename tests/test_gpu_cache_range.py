"""cache_attention at the ends of its range: scales as far apart as cache_write makes them, scores of any finite size."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
PAGE, BLOCK = 16, 8


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _cached(k, v, kscale, vscale):
    """The arguments of a call over k and v [b, n, h, d] (fp64), which their codes hold exactly at the scales [b, n / BLOCK, h];
    pages in another order than the tokens."""
    b, n, h, d = k.shape
    most = n // PAGE
    order = torch.randperm(b * most, generator=torch.Generator().manual_seed(n))
    dev = []
    for x, s in ((k, kscale), (v, vscale)):
        codes = (x.view(b, -1, BLOCK, h, d) / s[:, :, None, :, None]).view(b * most, PAGE, h, d)
        assert torch.equal(codes.to(F8).double(), codes)
        pages = torch.zeros(b * most, PAGE, h, d, dtype=torch.uint8)
        pages[order] = codes.to(F8).view(torch.uint8)
        dev.append(pages.view(F8).cuda())
    for s in (kscale, vscale):
        pages = torch.zeros(b * most, PAGE // BLOCK, h)
        pages[order] = s.float().view(b * most, PAGE // BLOCK, h)
        dev.append(pages.cuda())
    return (*dev, order.view(b, most).int().cuda())


def _bound(p, v, vscale, dt, mag, d):
    """How far an output may be off, p [b, hq, n] and v [b, hq, n, d] in fp64: half a step of the type for the result and for
    each operand exp(score) scale; twice the relative error of those and of the denominator's terms (the score's d + 14
    roundings of 2^-24 of mag, 2^-24 of the scale's logarithm of at most 128, for an element and its maximum; 2^-19 for
    exponentials and division; 2^-24 per key summed); operands below the type's range, which are 2^-125 (in fp16 2^-25) of the
    largest one; and results there, whose steps no longer shrink with them: fp16 has steps of 2^-14 2^-10 below 2^-14, bf16 of
    2^-126 2^-7 below 2^-126, so a result is off by half of that however small it is."""
    u, step = torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    e = 2 * ((d + 14) * 2.0 ** -24 * mag + 2.0 ** -24 * (mag + 128)) + 2.0 ** -19 + p.shape[-1] * 2.0 ** -24
    lost = 2.0 ** -125 + (2.0 ** -25 if dt is HF else 0.0)
    codes = (v.abs() / vscale[..., None]).sum(2)
    top = (p * vscale).amax(-1, keepdim=True)
    o = (p[:, :, None] @ v)[:, :, 0]
    return o, 1.05 * (u * o.abs() + (u + 2 * e) * (p[:, :, None] @ v.abs())[:, :, 0] + lost * top * codes) + step / 2


# where the large values stand among n tokens: within a tile of 32 keys, in two tiles of a wave, in those of different waves, and
# in parts of a sequence that several workgroups share
PLACES = [(32, 0, 8), (32, 24, 32), (64, 8, 16), (128, 32, 64), (128, 96, 128), (256, 0, 32), (256, 128, 160), (304, 120, 303),
          (20000, 0, 700), (20000, 19296, 20000), (20000, 9000, 9008)]


@pytest.mark.parametrize("n,first,last", PLACES)
@pytest.mark.parametrize("dt,up,down", [(BF, 30, -100), (BF, 110, -100), (BF, -20, -100), (BF, 60, -30), (HF, 6, -100)])
@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 64), (40, 2, 128)])
def test_scales_far_apart(hq, hkv, d, dt, up, down, n, first, last):
    """A few large values beside small ones or zeros (whose scale is 2^-100): every token counts in the denominator."""
    from memarch_amd import _lib
    from memarch_amd.kv_cache import cache_attention
    print(f"far apart {hq} {hkv} {d} {dt} {up} {down} {n} {first} {last}", flush=True)
    g = torch.Generator().manual_seed(n + first)
    full = -(-n // PAGE) * PAGE
    k = torch.randn(1, full, hkv, d, generator=g).mul(16).round().clamp(-15, 15).double()
    kscale = torch.full((1, full // BLOCK, hkv), 2.0 ** -4, dtype=torch.float64)
    k = k * 2.0 ** -4
    big = torch.zeros(full // BLOCK, dtype=torch.bool)
    big[first // BLOCK:-(-last // BLOCK)] = True
    vscale = torch.where(big, 2.0 ** up, 2.0 ** down).double()[None, :, None].expand(1, -1, hkv).contiguous()
    v = torch.randint(-15, 16, (1, full, hkv, d), generator=g).double()
    if down == -100:
        v *= big.repeat_interleave(BLOCK)[None, :, None, None]
    v = v * vscale.repeat_interleave(BLOCK, 1)[..., None]
    cache = _cached(k, v, kscale, vscale)
    if n == 20000:
        assert _lib.load_serve().mce_cache_attn_ws_bytes(1, hq, hkv, d, PAGE, full // PAGE, 0, 0) > 0
    wide = lambda t: t[:, :n].repeat_interleave(hq // hkv, 2).transpose(1, 2)
    vs = wide(vscale.repeat_interleave(BLOCK, 1)[..., None])[..., 0]
    for gain in (0.0, 1.0, 8.0):
        q = (gain * torch.randn(1, hq, d, generator=g)).to(dt)
        s = (q.double()[:, :, None] @ wide(k).mT)[:, :, 0] * d ** -0.5
        mag = float((q.double().abs()[:, :, None] @ wide(k).abs().mT).max()) * d ** -0.5
        ref, tol = _bound(torch.softmax(s, -1), wide(v), vs, dt, mag, d)
        out = cache_attention(q.cuda(), *cache, torch.tensor([n]).cuda())
        err = (out.double().cpu() - ref).abs()
        assert (err <= tol).all(), (gain, float((err / tol.clamp(min=1e-300)).max()))


def test_zeros_that_were_written():
    """The same as cache_write leaves it: texts that begin or end with values of 0, read over what it wrote."""
    from memarch_amd.kv_cache import cache_attention, cache_read, cache_write
    lens, d = torch.tensor([70, 70, 33]), 64
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(173, 2, d, generator=g) for _ in range(2))
    v *= 2.0 ** 39
    v[:35], v[100:140], v[141:] = 0, 0, 0
    table = torch.arange(15, dtype=torch.int32).view(3, 5).cuda()
    cache = [torch.zeros(15, PAGE, 2, d, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
    cache += [torch.zeros(15, PAGE // BLOCK, 2, device="cuda") for _ in range(2)]
    cu = torch.tensor([0, 70, 140, 173]).cuda()
    cache_write(k.to(BF).cuda(), v.to(BF).cuda(), *cache, table, lens.cuda(), cu)
    assert float(cache[3][cache[3] > 0].min()) == 2.0 ** -100 and float(cache[3].max()) >= 2.0 ** 30
    kk, vv = (x.double().cpu() for x in cache_read(*cache, table, cu, 173))
    q = torch.randn(3, 4, d, generator=g).to(BF)
    out = cache_attention(q.cuda(), *cache, table, lens.cuda()).double().cpu()
    scales = cache[3].double().cpu()
    for i in range(3):
        rows = slice(int(cu[i]), int(cu[i + 1]))
        w = lambda t: t[rows].repeat_interleave(2, 1).transpose(0, 1)[None]
        at = torch.arange(int(lens[i]))
        vs = scales[i * 5 + at // PAGE, at % PAGE // BLOCK].repeat_interleave(2, 1).t()[None]
        s = (q[i].double()[None, :, None] @ w(kk).mT)[:, :, 0] * d ** -0.5
        mag = float((q[i].double().abs()[None, :, None] @ w(kk).abs().mT).max()) * d ** -0.5
        ref, tol = _bound(torch.softmax(s, -1), w(vv), vs, BF, mag, d)
        assert ((out[i] - ref[0]).abs() <= tol[0]).all(), i


@pytest.mark.parametrize("dt,move", [(BF, 40), (BF, -60), (HF, 12)])
def test_scales_of_keys_far_from_one(dt, move):
    """Keys by a power of two larger and queries by as much smaller: the same scores."""
    from memarch_amd.kv_cache import cache_attention
    n, h, d = 304, 2, 64
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randint(-15, 16, (1, n, h, d), generator=g).double() * 2.0 ** -4 for _ in range(2))
    s = torch.full((1, n // BLOCK, h), 2.0 ** -4, dtype=torch.float64)
    q = torch.randn(1, 4, d, generator=g).to(dt)
    far = (q.double() * 2.0 ** -move).to(dt)
    q = (far.double() * 2.0 ** move).to(dt)            # (what is left of it in fp16)
    w = lambda t: t.repeat_interleave(2, 2).transpose(1, 2)
    scores = (q.double()[:, :, None] @ w(k).mT)[:, :, 0] * d ** -0.5
    mag = float((q.double().abs()[:, :, None] @ w(k).abs().mT).max()) * d ** -0.5
    ref, tol = _bound(torch.softmax(scores, -1), w(v), torch.full((1, 4, n), 2.0 ** -4).double(), dt, mag, d)
    lens = torch.tensor([n]).cuda()
    for x, f in ((q, 0), (far, move)):
        out = cache_attention(x.cuda(), *_cached(k * 2.0 ** f, v, s * 2.0 ** f, s), lens).double().cpu()
        assert ((out - ref).abs() <= tol).all(), f


def _blocks_of(values, power, g):
    """Scales [b, n / BLOCK, h] of 2^power over 1, 2 or 4: `values`, multiples of 2^power, have codes of different sizes then."""
    b, n, h, _ = values.shape
    return 2.0 ** power / 2.0 ** torch.randint(0, 3, (b, n // BLOCK, h), generator=g).double()


def _spread_values(b, n, h, d, g):
    vscale = torch.exp2(torch.randint(-4, 4, (b, n // BLOCK, h), generator=g).double())
    return torch.randint(-15, 16, (b, n, h, d), generator=g).double() * vscale.repeat_interleave(BLOCK, 1)[..., None], vscale


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt,power,scale", [(BF, 0, 2e4), (BF, 10, None), (BF, 0, 1e9), (BF, 4, 1.0), (BF, 14, 1.0), (BF, 58, None),
                                            (HF, 13, None), (HF, 15, None), (HF, 0, 1e12)])
def test_scores_of_any_finite_size(dt, power, scale, d, window, sinks):
    """Scores from 1e4 to 1e36: q and k hold -1, 0 and 1 times a power of two, so that scores are exact and either equal or too
    far apart to share a softmax: the output is the mean of v over the highest scores, whatever their blocks' scales. Exponentials
    are powers of two then, so what rounds is the result (u), fp32 sums (2^-24 a key) and the division (2^-20)."""
    from memarch_amd.kv_cache import cache_attention
    g = torch.Generator().manual_seed(power + d)
    for lens in ([200, 183, 1], [20000]):
        b, n = len(lens), -(-max(lens) // PAGE) * PAGE
        k = torch.randint(-1, 2, (b, n, 2, d), generator=g).double() * 2.0 ** power
        v, vscale = _spread_values(b, n, 2, d, g)
        q = torch.randint(-1, 2, (b, 4, d), generator=g).to(dt) * 2.0 ** power
        assert torch.isfinite(q).all() and q.dtype == dt
        out = cache_attention(q.cuda(), *_cached(k, v, _blocks_of(k, power, g), vscale), torch.tensor(lens).cuda(),
                              window=window or None, sinks=sinks, scale=scale).double().cpu()
        for i, m in enumerate(lens):
            j = torch.arange(m)
            j = j[(m - 1 - j < window) | (j < sinks)] if window else j
            kk, vv = (x[i, j].repeat_interleave(2, 1).transpose(0, 1) for x in (k, v))
            s = (q[i].double()[:, None] @ kk.mT)[:, 0]
            p = (s == s.amax(-1, keepdim=True)).double()
            p = (p / p.sum(-1, keepdim=True))[:, None]
            ref, mag = (p @ vv)[:, 0], (p @ vv.abs())[:, 0]
            tol = (torch.finfo(dt).eps / 2 * ref.abs() + (m * 2.0 ** -24 + 2.0 ** -20) * mag) * 1.01
            assert ((out[i] - ref).abs() <= tol).all(), (i, float((out[i] - ref).abs().max()))   # (NaN fails it too)


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 16, 2.0 ** 20, 2.0 ** 24, 2.0 ** 28, 2.0 ** 31, 2.0 ** 32, 2.0 ** 60])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
def test_equal_keys_of_large_scores(dt, sign, size):
    """One key row everywhere, of any score (both signs): the mean of v; and a sequence of one token: its value. The scores are equal
    to the last bit (codes and scales differ by powers of two), so the bound is that of the test above."""
    from memarch_amd.kv_cache import cache_attention
    g = torch.Generator().manual_seed(9)
    lens, d = [1, 64, 333, 20000], 64
    n = 20000
    row = torch.randint(1, 4, (4, 1, 2, d), generator=g).double()
    k = row.expand(4, n, 2, d).contiguous()
    v, vscale = _spread_values(4, n, 2, d, g)
    q = (sign * torch.rand(4, 4, d, generator=g)).to(dt)
    most = float((q.double().abs() * row[:, 0].repeat_interleave(2, 1)).sum(-1).max())
    out = cache_attention(q.cuda(), *_cached(k, v, _blocks_of(k, 0, g), vscale), torch.tensor(lens).cuda(),
                          scale=size / most).double().cpu()
    for i, m in enumerate(lens):
        vv = v[i, :m].repeat_interleave(2, 1)
        ref, mag = vv.mean(0), vv.abs().mean(0)
        tol = (torch.finfo(dt).eps / 2 * ref.abs() + (m * 2.0 ** -24 + 2.0 ** -20) * mag) * 1.01
        assert ((out[i] - ref).abs() <= tol).all(), (m, float((out[i] - ref).abs().max()))


@pytest.mark.parametrize("sign", [1, -1])
def test_scores_next_to_the_largest_number(sign):
    """Scores of 3.2e38, which fp32 holds and their product with log2 e does not: the mean of v, as above."""
    from memarch_amd.kv_cache import cache_attention
    g = torch.Generator().manual_seed(10)
    lens, d, n = [1, 64, 333, 20000], 64, 20000
    row = torch.randint(1, 4, (4, 1, 2, d), generator=g).double() * 2.0 ** 60
    v, vscale = _spread_values(4, n, 2, d, g)
    q = (sign * 2.0 ** 60 * torch.rand(4, 4, d, generator=g)).to(BF)
    most = float((q.double().abs() * row[:, 0].repeat_interleave(2, 1)).sum(-1).max())
    k = row.expand(4, n, 2, d).contiguous()
    out = cache_attention(q.cuda(), *_cached(k, v, _blocks_of(k, 60, g), vscale), torch.tensor(lens).cuda(),
                          scale=3.2e38 / most).double().cpu()
    for i, m in enumerate(lens):
        vv = v[i, :m].repeat_interleave(2, 1)
        ref, mag = vv.mean(0), vv.abs().mean(0)
        tol = (torch.finfo(BF).eps / 2 * ref.abs() + (m * 2.0 ** -24 + 2.0 ** -20) * mag) * 1.01
        assert ((out[i] - ref).abs() <= tol).all(), (m, float((out[i] - ref).abs().max()))

"""The 8-bit cache without a GPU: the oracle against torch's own float8 and dense attention, what the entry points refuse, and
the C ABI's checks."""
import contextlib
import ctypes
import inspect
import math
import os

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from memarch_amd import _lib, attention, kv_cache
from oracle import attn_oracle, cache_oracle as orc

F8 = torch.float8_e4m3fn


def test_oracle_rounds_as_float8_does():
    x = torch.cat((torch.randn(4000, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.arange(4000) % 20 - 12.0),
                   torch.arange(-900, 901) / 2.0 ** 10, torch.tensor([448.0, -448.0, 432.0, 0.0, 2.0 ** -10, 3 * 2.0 ** -10])))
    x = x[x.abs() <= 448]
    assert torch.equal(orc.nearest8(x.double()), x.to(F8).double())
    for a, s in ((448.0, 1.0), (448.0001, 2.0), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7), (0.0, 2.0 ** -100), (1e-38, 2.0 ** -100),
                 (3.38e38, 2.0 ** 120)):
        assert orc.scale_for(a) == s, a


def test_oracle_writes_one_by_one_as_at_once():
    """Up to what a second rounding takes from codes below 2^-6: half a step of 2^-9 of the block's scale."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(30, 2, 16, generator=g) * torch.exp2(torch.randn(30, 1, 1, generator=g))
    codes, scale = torch.zeros(4, 16, 2, 16, dtype=torch.float64), torch.zeros(4, 2, 2, dtype=torch.float64)
    table = torch.tensor([[2, 0]])
    once = orc.write(x, codes, scale, table, [30], [0, 30])
    step = (codes, scale)
    for t in range(30):
        step = orc.write(x[t:t + 1], *step, table, [t + 1])
    assert torch.equal(once[1], step[1])
    a, b = (orc.read(orc.values(*c), table, [0, 30], 30) for c in (once, step))
    s = once[1][table[0].long()].repeat_interleave(8, 1).flatten(0, 1)[:30, :, None]
    assert ((a - b).abs() <= s * 2.0 ** -9).all()
    assert ((a - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, s * 2.0 ** -10)).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (7, 2)])
def test_oracle_attention_is_that_of_the_values(window, sinks):
    g = torch.Generator().manual_seed(1)
    codes = [orc.nearest8(torch.randn(5, 16, 2, 16, generator=g, dtype=torch.float64)) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-3, 4, (5, 2, 2), generator=g).double()) for _ in range(2)]
    table, lens = torch.tensor([[3, 1], [0, -1]], dtype=torch.int32), torch.tensor([29, 20])
    q = torch.randn(2, 4, 16, generator=g)
    got = orc.attention(q, codes[0], scales[0], codes[1], scales[1], table, lens, window, sinks)
    want = attn_oracle.paged(q, orc.values(codes[0], scales[0]), orc.values(codes[1], scales[1]), table, lens, window, sinks)
    assert (got - want).abs().max() < 1e-12


def _meta(*shape, dtype=torch.bfloat16, device="meta"):
    return torch.zeros(*shape, dtype=dtype, device=device)


def _cache(pages=10, page=16, h=2, d=64, per=2, device="meta"):
    c = lambda: _meta(pages, page, h, d, dtype=F8, device=device)
    s = lambda: _meta(pages, per, h, dtype=torch.float32, device=device)
    return [c(), c(), s(), s(), _meta(3, 5, dtype=torch.int32, device=device)]


def test_surfaces():
    names = lambda f: list(inspect.signature(f).parameters)
    cache = ["k_cache", "v_cache", "k_scale", "v_scale", "block_table"]
    assert names(kv_cache.cache_write) == ["k", "v", *cache, "lengths", "cu_seqlens"]
    assert names(kv_cache.cache_read) == [*cache, "cu_seqlens", "rows", "dtype"]
    assert names(kv_cache.cache_attention) == ["q", *cache, "lengths", "window", "sinks", "scale"]


def test_refusals():
    k, q, lens = _meta(3, 2, 64), _meta(3, 4, 64), _meta(3, dtype=torch.int32)
    cu = _meta(4, dtype=torch.int32)
    calls = {"write": lambda c, k=k, v=None, lens=lens, cu=None: kv_cache.cache_write(k, k if v is None else v, *c, lens, cu),
             "read": lambda c, cu=cu, rows=9, dtype=torch.float16: kv_cache.cache_read(*c, cu, rows, dtype),
             "attend": lambda c, q=q, lens=lens, **kw: kv_cache.cache_attention(q, *c, lens, **kw)}
    bad = [(0, _meta(10, 16, 2, 64), "float8_e4m3fn"), (0, _meta(10, 16, 2, 64, dtype=torch.float8_e5m2), "float8_e4m3fn"),
           (0, _meta(16, 2, 64, dtype=F8), "float8_e4m3fn"), (1, _meta(9, 16, 2, 64, dtype=F8), "one shape"),
           (2, _meta(10, 2, 2), "float32"), (2, _meta(10, 2, 3, dtype=torch.float32), "k_scale"),
           (2, _meta(9, 2, 2, dtype=torch.float32), "k_scale"), (2, _meta(10, 0, 2, dtype=torch.float32), "k_scale"),
           (2, _meta(10, 3, 2, dtype=torch.float32), "k_scale"), (3, _meta(10, 1, 2, dtype=torch.float32), "v_scale"),
           (4, _meta(3, 5, dtype=torch.int64), "block_table"), (4, _meta(3, dtype=torch.int32), "block_table"),
           (4, _meta(3, (1 << 26) + 1, dtype=torch.int32), "per sequence")]
    for call in calls.values():
        for i, x, match in bad:
            c = _cache()
            c[i] = x
            with pytest.raises(ValueError, match=match):
                call(c)
        for kw, match in ((dict(page=12, per=1), "pages of 12"), (dict(page=4, per=1), "pages of 4"), (dict(per=4), "blocks of 4"),
                          (dict(page=256, per=1), "blocks of 256"), (dict(page=65544, per=1), "pages of 65544"),
                          (dict(page=24, per=2), "blocks of 12"), (dict(d=72), "multiple of 16"), (dict(d=144), "multiple of 16"),
                          (dict(d=8), "multiple of 16"), (dict(h=0), "multiple of 16")):
            with pytest.raises(ValueError, match=match):
                call(_cache(**kw))
    for args, match in ((dict(k=k[0]), "must both be"), (dict(v=k[:2]), "must both be"), (dict(k=k.float()), "bfloat16"),
                        (dict(v=k.half()), "bfloat16"), (dict(k=_meta(3, 2, 32)), "does not fit"), (dict(k=_meta(3, 1, 64)), "does not fit"),
                        (dict(k=_meta(4, 2, 64)), "cu_seqlens"), (dict(lens=None), "lengths"), (dict(lens=lens[:2]), "lengths"),
                        (dict(lens=lens.float()), "lengths"), (dict(cu=cu[:3]), "cu_seqlens"), (dict(cu=cu.float()), "cu_seqlens"),
                        (dict(lens=torch.zeros(3, dtype=torch.int32)), "lengths is on cpu")):
        with pytest.raises(ValueError, match=match):
            calls["write"](_cache(), **args)
    for args, match in ((dict(cu=cu[:3]), "cu_seqlens"), (dict(cu=cu.double()), "cu_seqlens"), (dict(rows=-1), "rows"),
                        (dict(rows=2 ** 27 + 1), "rows"), (dict(dtype=torch.float32), "dtype"),
                        (dict(cu=torch.zeros(4, dtype=torch.int32)), "cu_seqlens is on cpu")):
        with pytest.raises(ValueError, match=match):
            calls["read"](_cache(), **args)
    for args, match in ((dict(q=q[0]), "must be"), (dict(q=_meta(3, 3, 64)), "must be"), (dict(q=_meta(3, 4, 32)), "must be"),
                        (dict(q=_meta(3, 0, 64)), "must be"), (dict(q=q.float()), "bfloat16"), (dict(q=_meta(2, 4, 64)), "block_table"),
                        (dict(lens=None), "lengths"), (dict(lens=lens[:2]), "lengths"), (dict(window=0, sinks=1), "window"),
                        (dict(window=3, sinks=-1), "sinks"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
                        (dict(lens=torch.zeros(3, dtype=torch.int32)), "lengths is on cpu")):
        with pytest.raises(ValueError, match=match):
            calls["attend"](_cache(), **args)
    host = _cache(device="cpu")
    for call in (lambda: kv_cache.cache_write(k.new_zeros(3, 2, 64, device="cpu"), k.new_zeros(3, 2, 64, device="cpu"), *host, torch.zeros(3, dtype=torch.int32)),
                 lambda: kv_cache.cache_read(*host, torch.zeros(4, dtype=torch.int32), 5),
                 lambda: kv_cache.cache_attention(q.new_zeros(3, 4, 64, device="cpu"), *host, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="GPU only"):
            call()


def test_forward_mode_derivatives_are_refused(monkeypatch):
    launched = []
    monkeypatch.setattr(_lib, "call", lambda *a: launched.append(a[0]))
    for mod in (attention, kv_cache):
        monkeypatch.setattr(mod, "_check_same", lambda *a: None)
        monkeypatch.setattr(mod, "_On", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(kv_cache, "_stream", lambda dev: 0)
    monkeypatch.setattr(_lib, "load_serve", lambda: type("L", (), {"mce_cache_attn_ws_bytes": staticmethod(lambda *a: 0)}))
    x, lens, host = _meta(3, 2, 64, device="cpu"), torch.zeros(3, dtype=torch.int32), _cache(device="cpu")
    kv_cache.cache_write(x, x, *host, lens)
    kv_cache.cache_attention(x, *host, lens)
    assert launched == ["mce_cache_write", "mce_cache_attn"]
    with fwAD.dual_level():
        dual = fwAD.make_dual(x.clone(), torch.ones_like(x))
        scale = fwAD.make_dual(host[2].clone(), torch.ones_like(host[2]))
        for call in (lambda: kv_cache.cache_write(dual, x, *host, lens), lambda: kv_cache.cache_write(x, dual, *host, lens),
                     lambda: kv_cache.cache_attention(dual, *host, lens),
                     lambda: kv_cache.cache_attention(x, *host[:2], scale, *host[3:], lens),
                     lambda: kv_cache.cache_read(*host[:2], scale, *host[3:], torch.zeros(4, dtype=torch.int32), 2)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    assert len(launched) == 2


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.SERVE_LIB_PATH):
        pytest.skip("libmce_serve.so not built")
    return _lib.load_serve()


def test_c_abi_checks_need_no_gpu(lib):
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    sizes = dict(kc=p, st=128, sp=2048, ks=p, table=p, B=2, Hkv=2, D=64, pages=4, page=16, block=8, most=2, dtype=1)

    def write(k=p, k_st=128, lens=p, cu=p, N=9, **kw):
        s = {**sizes, **kw}
        return lib.mce_cache_write(k, k_st, 64, p, 128, 64, s["kc"], s["sp"], s["st"], 64, p, 2048, 128, 64, s["ks"], p,
                                   s["table"], 2, lens, cu, s["B"], N, s["Hkv"], s["D"], s["pages"], s["page"], s["block"],
                                   s["most"], s["dtype"], None)

    def read(cu=p, rows=9, k=p, v=p, **kw):
        s = {**sizes, **kw}
        return lib.mce_cache_read(s["kc"], s["sp"], s["st"], 64, p, 2048, 128, 64, s["ks"], p, s["table"], 2, cu, s["B"], rows,
                                  s["Hkv"], s["D"], s["pages"], s["page"], s["block"], s["most"], s["dtype"], k, v, None)

    def attend(q=p, sh=64, Hq=4, lens=p, window=0, sinks=0, scale=0.1, out=p, ws=None, nb=0, **kw):
        s = {**sizes, **kw}
        return lib.mce_cache_attn(q, 256, sh, s["kc"], s["sp"], s["st"], 64, p, 2048, 128, 64, s["ks"], p, s["table"], 2, lens,
                                  s["B"], Hq, s["Hkv"], s["D"], s["pages"], s["page"], s["block"], s["most"], window, sinks,
                                  scale, s["dtype"], out, ws, nb, None)

    for call in (write, read, attend):
        for kw in (dict(B=-1), dict(Hkv=0), dict(D=72), dict(D=8), dict(D=144), dict(page=12), dict(page=4, block=4),
                   dict(block=0), dict(block=12), dict(block=32), dict(page=256, block=256), dict(pages=-1), dict(pages=1 << 31),
                   dict(most=-1), dict(most=1 << 40), dict(page=65536, most=1 << 14), dict(dtype=0), dict(dtype=3), dict(kc=None),
                   dict(ks=None), dict(table=None), dict(st=48), dict(st=1 << 22), dict(sp=-16)):
            assert call(**kw) == 1, (call.__name__, kw)
        for kw in (dict(kc=p + 8), dict(st=136), dict(sp=2056), dict(ks=p + 2)):
            assert call(**kw) == 2, (call.__name__, kw)
    for kw in (dict(k=None), dict(lens=None), dict(N=-1), dict(N=(1 << 27) + 1), dict(cu=None), dict(k_st=56), dict(B=1 << 24),
               dict(B=1 << 22, Hkv=16)):
        assert write(**kw) == 1, kw
    assert write(k=p + 2) == 2 and write(k_st=132) == 2
    assert write(B=0, N=0, k=None, lens=None) == 0 and write(N=0, k=None) == 0 and write(pages=0, kc=None, ks=None) == 0
    for kw in (dict(cu=None), dict(rows=-1), dict(rows=(1 << 27) + 1), dict(k=None), dict(v=None), dict(B=1 << 24),
               dict(rows=1 << 27, B=(1 << 24) - 1)):
        assert read(**kw) == 1, kw
    assert read(k=p + 2) == 2 and read(rows=0, cu=None, k=None) == 0
    for kw in (dict(q=None), dict(lens=None), dict(out=None), dict(Hq=5), dict(Hq=0), dict(window=-1), dict(sinks=-1),
               dict(scale=0.0), dict(scale=math.inf), dict(sh=32), dict(B=1 << 22, Hq=8)):
        assert attend(**kw) == 1, kw
    assert attend(q=p + 2) == 2 and attend(out=p + 8) == 2 and attend(B=0, q=None, out=None, lens=None) == 0
    need = lib.mce_cache_attn_ws_bytes(2, 4, 2, 64, 16, 4096, 0, 0)
    assert need > 0 and lib.mce_cache_attn_ws_bytes(2, 5, 2, 64, 16, 4096, 0, 0) == 0
    assert lib.mce_cache_attn_ws_bytes(2, 4, 2, 64, 16, 2, 0, 0) == 0                 # short caches are not split
    assert attend(most=4096) == 3 and attend(most=4096, ws=p, nb=need - 1) == 3 and attend(most=4096, ws=p + 16, nb=need) == 3

"""The attention operators without a GPU: the oracle pinned (oracle/attn_oracle.py), argument checks of the Python
surface and the C ABI, the library's exports and what its kernels must not hold."""
import contextlib
import ctypes
import inspect
import os
import re
import shutil
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from memarch_amd import _lib, attention, rotary
from oracle import attn_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = [os.path.join(ROOT, "include", h) for h in ("mce_attn.h", "mce_paged.h", "mce_rope.h")]
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def _leaves(b, t, hq, hkv, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h: torch.randn(b, t, h, d, generator=g, dtype=torch.float64)
    return mk(hq), mk(hkv), mk(hkv), mk(hq)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 0), (3, 2), (100, 1)])
@pytest.mark.parametrize("lens", [None, [7, 0, 3]])
def test_oracle_matches_autograd(window, sinks, lens):
    """The closed forms against autograd through torch.softmax with an explicit mask."""
    q, k, v, go = _leaves(3, 7, 4, 2, 8)
    lengths = None if lens is None else torch.tensor(lens)
    got = orc.attention(q, k, v, window, sinks, lengths, 0.3, go)
    ql, kl, vl = (x.clone().requires_grad_() for x in (q, k, v))
    out = torch.zeros_like(q)
    rows = []
    for b in range(3):
        n = 7 if lens is None else lens[b]
        for h in range(4):
            for i in range(n):
                js = [j for j in range(i + 1) if not window or i - j < window or j < sinks]
                s = torch.stack([(ql[b, i, h] * kl[b, j, h // 2]).sum() * 0.3 for j in js])
                o = (torch.softmax(s, 0)[:, None] * torch.stack([vl[b, j, h // 2] for j in js])).sum(0)
                out[b, i, h] = o.detach()
                rows.append((o * go[b, i, h]).sum())
    grads = torch.autograd.grad(sum(rows), (ql, kl, vl))
    for a, r in zip(got, (out, *grads)):
        assert torch.allclose(a, r, rtol=1e-12, atol=1e-13)


def test_oracle_gradients_against_differences():
    q, k, v, go = _leaves(1, 6, 2, 1, 8, seed=3)
    _, dq, dk, dv = orc.attention(q, k, v, 3, 1, None, None, go)
    f = lambda q, k, v: float((orc.attention(q, k, v, 3, 1) * go).sum())
    g = torch.Generator().manual_seed(5)
    for x, dx, place in ((q, dq, 0), (k, dk, 1), (v, dv, 2)):
        for _ in range(6):
            i = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in x.shape)
            args = [q, k, v]
            vals = []
            for s in (1e-5, -1e-5):
                y = x.clone()
                y[i] += s
                args[place] = y
                vals.append(f(*args))
            assert abs((vals[0] - vals[1]) / 2e-5 - float(dx[i])) < 1e-8


def test_oracle_bounds_catch_planted_mistakes():
    """Implementations with one mistake each fall outside the bounds that a 16-bit implementation has to keep."""
    q, k, v, go = (x.bfloat16() for x in _leaves(2, 40, 2, 1, 16, seed=8))
    (out, dq, dk, dv), tol = orc.attention(q, k, v, 9, 2, None, None, go, torch.bfloat16)
    for args in ((10, 2), (8, 2), (9, 1), (9, 3), (0, 0)):   # window and sinks off by one, no window
        o2 = orc.attention(q, k, v, *args)
        assert ((o2 - out).abs() > tol[0]).any(), args
    o2 = orc.attention(q, k, v, 9, 2, None, 0.26)            # scale
    assert ((o2 - out).abs() > tol[0]).any()
    wrong = orc.attention(q.flip(1), k, v, 9, 2, None, None, go)   # rows in another order
    for i in range(4):
        assert ((wrong[i] - (out, dq, dk, dv)[i]).abs() > tol[i]).any(), i
    # a softmax backward without its row sum
    p, *_ = orc.probs(q, k, 9, 2, torch.full((2,), 40), 0.25)
    dp = go.double().transpose(1, 2) @ v.double().transpose(1, 2).repeat_interleave(2, 1).mT
    bad = (0.25 * (p * dp) @ k.double().transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2)
    assert ((bad - dq).abs() > tol[1]).any()
    # and rounding the exact results stays inside
    for r, t in zip((out, dq, dk, dv), tol):
        assert ((r.bfloat16().double() - r).abs() <= t).all()


def test_oracle_paged_is_the_last_row():
    q, k, v, _ = _leaves(3, 21, 4, 2, 8, seed=2)
    lens = torch.tensor([21, 0, 9])
    table = torch.tensor([[4, 0, 7], [1, 2, 3], [5, 8, 6]])
    kc, vc = torch.full((9, 8, 2, 8), 9.0, dtype=torch.float64), torch.full((9, 8, 2, 8), 9.0, dtype=torch.float64)
    for b in range(3):
        for j in range(21):
            kc[table[b, j // 8], j % 8], vc[table[b, j // 8], j % 8] = k[b, j], v[b, j]
    for window, sinks in ((0, 0), (5, 0), (5, 2)):
        full = orc.attention(q, k, v, window, sinks, lens)
        last = torch.stack([q[b, max(int(lens[b]) - 1, 0)] for b in range(3)])
        got = orc.paged(last, kc, vc, table, lens, window, sinks)
        for b in range(3):
            ref = full[b, int(lens[b]) - 1] if lens[b] else torch.zeros_like(got[b])
            assert torch.allclose(got[b], ref, atol=1e-13)
    # a page outside the cache is not seen: the first 8 tokens of sequence 0 gone
    table[0, 0] = -1
    got = orc.paged(q[:, 20], kc, vc, table, torch.tensor([21, 0, 0]))
    ref = orc.attention(q[:1, 8:], k[:1, 8:], v[:1, 8:])[0, 12]
    assert torch.allclose(got[0], ref, atol=1e-13) and not got[1:].any()


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rope(interleaved):
    """Against sines and cosines written out; norms of rotated pairs kept; position 0 changes nothing."""
    cos, sin = rotary.rope_table(11, 6, theta=50.0, scale=2.0)
    for i in range(3):
        for p in range(11):
            ang = p / 2.0 * 50.0 ** (-2 * i / 6)
            assert abs(float(cos[p, i]) - torch.cos(torch.tensor(ang, dtype=torch.float64))) < 1e-7
            assert abs(float(sin[p, i]) - torch.sin(torch.tensor(ang, dtype=torch.float64))) < 1e-7
    x = torch.randn(2, 5, 3, 10, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    w = torch.rand(10, dtype=torch.float64) + 0.5
    y = orc.rope(x, cos, sin, w, True, 1e-3, torch.tensor([0, 7, 2, 10, 1]), interleaved)
    n = x / (x.pow(2).mean(-1, keepdim=True) + 1e-3).sqrt() * w
    for t, p in enumerate([0, 7, 2, 10, 1]):
        for i in range(3):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 3)
            c, s = float(cos[p, i]), float(sin[p, i])
            assert torch.allclose(y[:, t, :, a], n[:, t, :, a] * c - n[:, t, :, b] * s)
            assert torch.allclose(y[:, t, :, b], n[:, t, :, b] * c + n[:, t, :, a] * s)
    assert torch.equal(y[..., 6:], n[..., 6:]) and torch.allclose(y[:, 0], n[:, 0])


# --------------------------------------------------------------------------------------------------- refusals


def test_surfaces():
    assert list(inspect.signature(attention.window_attention).parameters) == \
        ["q", "k", "v", "window", "sinks", "lengths", "scale"]
    assert list(inspect.signature(attention.paged_attention).parameters) == \
        ["q", "k_cache", "v_cache", "block_table", "lengths", "window", "sinks", "scale"]
    assert list(inspect.signature(rotary.qk_norm_rope).parameters) == \
        ["q", "k", "cos", "sin", "q_weight", "k_weight", "norm", "eps", "positions", "interleaved"]


def _bf(*shape, device="meta"):
    return torch.zeros(*shape, dtype=torch.bfloat16, device=device)


def test_window_attention_refusals():
    wa = attention.window_attention
    q, k = _bf(2, 5, 4, 64), _bf(2, 5, 2, 64)
    with pytest.raises(ValueError, match="GPU only"):
        wa(_bf(2, 5, 4, 64, device="cpu"), _bf(2, 5, 2, 64, device="cpu"), _bf(2, 5, 2, 64, device="cpu"))
    for bad in ((q[0], k, k), (q, k[:, :4], k[:, :4]), (q, k, k[..., :32]), (q, k[:, :, :1], k), (q, _bf(2, 5, 3, 64), _bf(2, 5, 3, 64)),
                (_bf(2, 5, 4, 136), _bf(2, 5, 2, 136), _bf(2, 5, 2, 136)), (_bf(2, 5, 4, 60), _bf(2, 5, 2, 60), _bf(2, 5, 2, 60)),
                (q.float(), k.float(), k.float()), (q, k.half(), k), (q, _bf(2, 5, 0, 64), _bf(2, 5, 0, 64))):
        with pytest.raises(ValueError):
            wa(*bad)
    for kw, match in ((dict(window=0, sinks=3), "window"), (dict(window=-2), "window"), (dict(window=4, sinks=-1), "sinks"),
                      (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=1e-31), "scale"),
                      (dict(scale=float("nan")), "scale"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
                      (dict(lengths=torch.zeros(2)), "lengths"), (dict(lengths=torch.zeros(2, 1, dtype=torch.int32)), "lengths"),
                      (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths is on cpu")):
        with pytest.raises(ValueError, match=match):
            wa(q, k, k, **kw)


def test_paged_attention_refusals():
    pa = attention.paged_attention
    q, kc = _bf(3, 4, 64), _bf(10, 16, 2, 64)
    i32 = dict(dtype=torch.int32, device="meta")
    table, lens = torch.zeros(3, 5, **i32), torch.zeros(3, **i32)
    with pytest.raises(ValueError, match="GPU only"):
        pa(_bf(3, 4, 64, device="cpu"), _bf(10, 16, 2, 64, device="cpu"), _bf(10, 16, 2, 64, device="cpu"),
           torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    for args, match in (((q[0], kc, kc, table, lens), "q"), ((q, kc, kc[:9], table, lens), "one shape"),
                        ((q, _bf(10, 12, 2, 64), _bf(10, 12, 2, 64), table, lens), "pages of 12"),
                        ((q, _bf(10, 4, 2, 64), _bf(10, 4, 2, 64), table, lens), "pages of 4"),
                        ((q, kc, kc, table[:2], lens), "block_table"), ((q, kc, kc, table.long(), lens), "block_table"),
                        ((q, kc, kc, table, lens[:2]), "lengths"), ((q, kc, kc, table, None), "lengths"),
                        ((q.half(), kc, kc, table, lens), "bfloat16"), ((q, kc.float(), kc.float(), table, lens), "bfloat16"),
                        ((_bf(3, 3, 64), kc, kc, table, lens), "share")):
        with pytest.raises(ValueError, match=match):
            pa(*args)
    with pytest.raises(ValueError, match="sinks"):
        pa(q, kc, kc, table, lens, window=3, sinks=-1)
    with pytest.raises(ValueError, match="per sequence"):
        pa(q, kc, kc, torch.zeros(3, (1 << 26) + 1, **i32), lens)
    big = _bf(2, 65536, 2, 64)
    with pytest.raises(ValueError, match="per sequence"):
        pa(q, big, big, torch.zeros(3, 65, **i32), lens)
    with pytest.raises(ValueError, match="lengths is on cpu"):
        pa(q, kc, kc, table, torch.zeros(3, dtype=torch.int32))


def test_qk_norm_rope_refusals():
    f = rotary.qk_norm_rope
    q, k = _bf(2, 5, 4, 64), _bf(2, 5, 2, 64)
    cos = torch.zeros(8, 16, device="meta")
    w = torch.zeros(64, device="meta")
    with pytest.raises(ValueError, match="GPU only"):
        f(torch.zeros(2, 5, 4, 64), torch.zeros(2, 5, 2, 64), torch.zeros(8, 16), torch.zeros(8, 16))
    for args, kw, match in (((q, k[:, :4], cos, cos), {}, "must be"), ((q, k[..., :32], cos, cos), {}, "must be"),
                            ((q, k.half(), cos, cos), {}, "float32"), ((q.double(), k.double(), cos, cos), {}, "float32"),
                            ((q, k, cos, cos[:7]), {}, "cos"), ((q, k, cos.half(), cos.half()), {}, "cos"),
                            ((q, k, torch.zeros(8, 33, device="meta"), torch.zeros(8, 33, device="meta")), {}, "cos"),
                            ((q, k, cos[:4], cos[:4]), {}, "table"), ((q, k, cos, cos, w, w), dict(norm=False), "norm"),
                            ((q, k, cos, cos, w), {}, "together"), ((q, k, cos, cos, w[:3], w), {}, "q_weight"),
                            ((q, k, cos, cos), dict(eps=-1.0), "eps"), ((q, k, cos, cos), dict(eps=float("nan")), "eps"),
                            ((q, k, cos, cos), dict(positions=torch.zeros(4, dtype=torch.int64)), "positions"),
                            ((q, k, cos, cos), dict(positions=torch.zeros(3, 5, dtype=torch.int64)), "positions"),
                            ((q, k, cos, cos), dict(positions=torch.zeros(5)), "positions"),
                            ((_bf(2, 5, 4, 264), _bf(2, 5, 2, 264), cos, cos), {}, "head dimension"),
                            ((_bf(2, 5, 0, 64), k, cos, cos), {}, "heads"),
                            ((q, k, torch.zeros(8, 16), torch.zeros(8, 16)), {}, "cos is on cpu")):
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)
    for args in ((-1, 4), (4, 3), (4, 0)):
        with pytest.raises(ValueError):
            rotary.rope_table(*args)
    with pytest.raises(ValueError):
        rotary.rope_table(4, 4, theta=0.0)
    assert rotary.rope_table(0, 4)[0].shape == (0, 2)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor among the inputs raises, whether or not one requires a gradient: no output loses a tangent. (The
    launches are stubbed; outside a dual level the calls go through.)"""
    launched = []
    monkeypatch.setattr(_lib, "call", lambda *a: launched.append(a[0]))
    for mod in (attention, rotary):
        monkeypatch.setattr(mod, "_check_same", lambda *a: None)
        monkeypatch.setattr(mod, "_stream", lambda dev: 0)
        monkeypatch.setattr(mod, "_On", lambda dev: contextlib.nullcontext())
    q, w, cos = _bf(1, 3, 2, 64, device="cpu"), torch.ones(64), torch.zeros(3, 32)
    kc, table, lens = _bf(2, 8, 2, 64, device="cpu"), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    calls = [(attention.window_attention, (q, q, q), 3), (rotary.qk_norm_rope, (q, q, cos, cos, w, w), 6),
             (attention.paged_attention, (q[0], kc, kc, table, lens), 3)]
    for fn, args, n in calls:
        fn(*args)
        with fwAD.dual_level():
            fn(*args)
            count = len(launched)
            for i in range(n):
                for needs in (False, True):
                    x = args[i].clone().requires_grad_(needs)
                    dual = fwAD.make_dual(x, torch.ones_like(x))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        fn(*args[:i], dual, *args[i + 1:])
                    with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                        fn(*args[:i], dual, *args[i + 1:])
            assert len(launched) == count


# ------------------------------------------------------------------------------------------------------ the library


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.ATTN_LIB_PATH):
        pytest.skip("libmce_attn.so not built")
    return _lib.load_attn()


def test_exports_every_declared_symbol(lib):
    src = "".join(open(h).read() for h in HEADERS)
    names = re.findall(r"MCE_(?:ATTN|ROPE)_API\s+[\w\s\*]+?\b(mce_\w+)\s*\(", src)
    assert len(names) == len(set(names)) >= 8
    for n in names:
        assert hasattr(lib, n), n
    assert set(names) == set(_lib.ATTN_SIGNATURES) and not set(names) & set(_lib.SIGNATURES)
    for code in range(6):
        assert lib.mce_attn_error_string(code)


def _kernels(tmp_path):
    """{kernel: its instructions} of the built library."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    shutil.copy(_lib.ATTN_LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    out, name = {}, None
    for f in sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950")):
        for line in subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], cwd=tmp_path, check=True, capture_output=True,
                                   text=True).stdout.splitlines():
            m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
            if m:
                name = m[1]
                out[name] = []
            elif name and line.startswith("\t"):
                out[name].append(line.split("//")[0].strip())
    return out


def test_loads_into_lds_wait_for_their_scalar_operands(lib, tmp_path):
    """Each load into LDS stands behind five wait states of its own (a scalar register that a vector instruction has just
    written may not be read earlier), and behind a write of M0 that the compiler knows of."""
    loads = 0
    for name, ins in _kernels(tmp_path).items():
        for i, x in enumerate(ins):
            if x.startswith("buffer_load") and x.endswith(" lds"):
                loads += 1
                m = re.fullmatch(r"s_nop (\d+)", ins[i - 1])
                assert m and int(m[1]) >= 4, (name, ins[i - 2:i + 1])
                back = next(y for y in ins[i - 1::-1] if re.match(r"\w+ m0,|s_c?branch|buffer_load.* lds$", y))
                assert " m0," in back, (name, back)
    assert loads > 100


@pytest.mark.parametrize("kernel,most", [("k_paged", {"Li64": {8}, "Li128": {16}}),
                                         ("k_attn_dkv", {"Li64": {3, 6}, "Li128": {5, 10}})])
def test_loops_wait_for_their_own_tile_only(lib, tmp_path, kernel, most):
    """Loads return in order, so a wait for an operand from before the loop, put among the loop's products, would be a wait
    for every tile under way. Behind the first load into LDS only the kernel's own waits are left: for the tile at hand (so
    many later loads stay under way) and for all, where no product follows."""
    found = 0
    for name, ins in _kernels(tmp_path).items():
        if kernel + "I" not in name:
            continue
        found += 1
        first = next(i for i, x in enumerate(ins) if x.endswith(" lds"))
        allowed = {0} | next(v for k, v in most.items() if k + "E" in name)
        for i, x in enumerate(ins[first:], first):
            m = re.match(r"s_waitcnt vmcnt\((\d+)\)", x)
            if m:
                assert int(m[1]) in allowed and not ins[i + 1].startswith("v_mfma"), (name, ins[i - 1:i + 2])
    assert found == 4


def test_kernels_hold_no_l2_writeback_and_no_packed_fp32(lib, tmp_path):
    """No device-scope release (buffer_wbl2), no scratch memory spills in the attention kernels' inner loops to speak of,
    and none of the packed fp32 operations that the build switches off."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    shutil.copy(_lib.ATTN_LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    objs = sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950"))
    assert len(objs) == 3, objs   # attn, paged, rope
    text = "".join(subprocess.run([OBJDUMP, "-d", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
                   for f in objs)
    assert "v_mfma_f32_32x32x16_bf16" in text and "v_mfma_f32_32x32x16_f16" in text
    for bad in ("buffer_wbl2", "v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32", "scratch_store"):
        assert bad not in text, bad


def test_attn_c_abi_checks_need_no_gpu(lib):
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256

    def fwd(q=p, st=64, sh=64, B=2, T=4, Hq=2, Hkv=1, D=64, window=0, sinks=0, scale=0.1, dtype=1, out=p, res=None):
        return lib.mce_attn_fwd(q, 1024, st, sh, p, 1024, 64, 64, p, 1024, 64, 64, None, B, T, Hq, Hkv, D, window, sinks,
                                scale, dtype, out, res, None, None)

    for kw in (dict(B=-1), dict(T=-1), dict(Hq=3, Hkv=2), dict(Hkv=0), dict(D=60), dict(D=136), dict(D=0),
               dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(scale=1e-31), dict(dtype=0), dict(q=None), dict(out=None), dict(st=56), dict(st=1 << 22), dict(T=(1 << 27) + 1),
               dict(B=1 << 40)):
        assert fwd(**kw) == 1, kw
    for kw in (dict(q=p + 2), dict(out=p + 8), dict(res=p + 4), dict(st=68), dict(sh=4)):
        assert fwd(**kw) == 2, kw
    assert fwd(B=0, q=None, out=None) == 0 and fwd(T=0, q=None, out=None) == 0

    def bwd(ws=p, nb=1 << 20, go=p, lse=p, dq=p, st=64):
        return lib.mce_attn_bwd(p, 1024, 64, 64, p, 1024, 64, 64, p, 1024, 64, 64, go, 1024, st, 64, None, 2, 4, 2, 1, 64,
                                0, 0, 0.1, 1, p, p, lse, dq, p, p, ws, nb, None)

    need = lib.mce_attn_bwd_ws_bytes(2, 4, 2, 1, 64, 0, 0)
    assert need >= 2 * 2 * 4 * 4 and lib.mce_attn_bwd_ws_bytes(2, 4, 3, 2, 64, 0, 0) == 0
    assert bwd(ws=None) == 3 and bwd(nb=need - 1) == 3 and bwd(ws=p + 16) == 3
    assert bwd(go=None) == 1 and bwd(lse=None) == 1 and bwd(dq=None) == 1 and bwd(dq=p + 2) == 2 and bwd(st=8) == 1


def test_paged_c_abi_checks_need_no_gpu(lib):
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256

    def call(q=p, sh=64, k=p, k_st=128, B=2, Hq=4, Hkv=2, D=64, pages=4, page=16, most=2, window=0, sinks=0, scale=0.1,
             dtype=1, out=p, ws=None, nb=0, lens=p, table=p):
        return lib.mce_paged(q, 256, sh, k, 2048, k_st, 64, p, 2048, 128, 64, table, most, lens, B, Hq, Hkv, D, pages, page,
                             most, window, sinks, scale, dtype, out, ws, nb, None)

    for kw in (dict(B=-1), dict(Hq=5), dict(Hkv=0), dict(D=12), dict(D=136), dict(page=12), dict(page=0), dict(page=4),
               dict(most=-1), dict(pages=-1), dict(window=-1), dict(sinks=-1), dict(scale=-1.0), dict(dtype=0),
               dict(out=None), dict(lens=None), dict(table=None), dict(k=None), dict(q=None), dict(sh=32), dict(k_st=32),
               dict(page=64, most=1 << 40), dict(page=65536, most=1 << 14)):
        assert call(**kw) == 1, kw
    for kw in (dict(q=p + 2), dict(k=p + 8), dict(out=p + 2), dict(k_st=132)):
        assert call(**kw) == 2, kw
    assert call(B=0, q=None, out=None, lens=None) == 0
    need = lib.mce_paged_ws_bytes(2, 4, 2, 64, 16, 4096, 0, 0)
    assert need > 0 and lib.mce_paged_ws_bytes(2, 5, 2, 64, 16, 4096, 0, 0) == 0
    assert lib.mce_paged_ws_bytes(2, 4, 2, 64, 16, 2, 0, 0) == 0                 # short caches are not split
    assert call(most=4096) == 3 and call(most=4096, ws=p, nb=need - 1) == 3 and call(most=4096, ws=p + 16, nb=need) == 3


def test_sizes_that_no_launch_can_hold_are_refused(lib):
    """2^24 workgroups of 256 threads are 2^32 threads, one more than a launch takes: refused as arguments, not found out by
    the launch. (Calls below that pass the checks: without a workspace or a sound address they end there.)"""
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    x = lambda q: (q, 64, 64, 64)

    def fwd(B, T, Hq):
        return lib.mce_attn_fwd(*x(p + 2), *x(p), *x(p), None, B, T, Hq, 1, 64, 0, 0, 0.1, 1, p, None, None, None)

    def bwd(B, T, Hq):
        return lib.mce_attn_bwd(*x(p), *x(p), *x(p), *x(p), None, B, T, Hq, 1, 64, 0, 0, 0.1, 1, p, p, p, p, p, p, None, 0,
                                None)

    for b, t, h in ((1 << 24, 1, 1), (1 << 20, 1, 16), (1 << 16, 129, 128), (1 << 27, 1, 1), (1 << 23, 129, 1)):
        assert fwd(b, t, h) == 1 and bwd(b, t, h) == 1 and lib.mce_attn_bwd_ws_bytes(b, t, h, 1, 64, 0, 0) == 0, (b, t, h)
    for b, t, h in (((1 << 24) - 1, 1, 1), ((1 << 24) - 1, 128, 1), ((1 << 20) - 1, 128, 16), ((1 << 16) - 1, 129, 128)):
        assert fwd(b, t, h) == 2 and bwd(b, t, h) == 3, (b, t, h)

    def paged(B, Hq, Hkv):
        return lib.mce_paged(p + 2, 64, 64, p, 4096, 64, 64, p, 4096, 64, 64, p, 1, p, B, Hq, Hkv, 64, 1, 16, 1, 0, 0, 0.1,
                             1, p, None, 0, None)

    for b, hq, hkv in ((1 << 24, 1, 1), (1 << 20, 16, 16), (1 << 8, 65536, 65536)):
        assert paged(b, hq, hkv) == 1 and lib.mce_paged_ws_bytes(b, hq, hkv, 64, 16, 1, 0, 0) == 0, (b, hq, hkv)
    for b, hq, hkv in (((1 << 24) - 1, 1, 1), (1 << 20, 16, 8), (1 << 8, 65536, 16)):
        assert paged(b, hq, hkv) == 2, (b, hq, hkv)


def test_rope_c_abi_checks_need_no_gpu(lib):
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256

    def fwd(q=p, P=8, pos=None, qw=None, kw=None, B=2, T=4, Hq=2, Hkv=1, D=64, R=32, norm=1, eps=1e-6, dtype=1, yq=p,
            cos=p):
        return lib.mce_rope_fwd(q, 512, 128, 64, p, 256, 64, 64, cos, p, P, pos, 1, 0, 0, qw, kw, B, T, Hq, Hkv, D, R, norm,
                                eps, 0, dtype, yq, p, None)

    for kw in (dict(q=None), dict(yq=None), dict(cos=None), dict(P=3), dict(P=-1), dict(R=3), dict(R=0), dict(R=66),
               dict(D=258, R=2), dict(Hq=0), dict(dtype=3), dict(eps=-1.0), dict(eps=float("nan")), dict(qw=p),
               dict(B=-1), dict(B=1 << 30, T=1 << 30)):
        assert fwd(**kw) == 1, kw
    assert fwd(B=0, q=None, yq=None) == 0
    need = lib.mce_rope_bwd_ws_bytes(2, 4, 2, 1, 64, 1)
    assert need > 0 and lib.mce_rope_bwd_ws_bytes(2, 4, 2, 1, 64, 0) == 0

    def bwd(ws=p, nb=need, gq=p, dqw=p, dkw=p):
        return lib.mce_rope_bwd(p, 512, 128, 64, p, 256, 64, 64, gq, 512, 128, 64, p, 256, 64, 64, p, p, 8, None, 1, 0, 0, p,
                                p, 2, 4, 2, 1, 64, 32, 1, 1e-6, 0, 1, p, p, dqw, dkw, ws, nb, None)

    assert bwd(ws=None) == 3 and bwd(nb=need - 1) == 3 and bwd(ws=p + 4) == 3
    assert bwd(gq=None) == 1 and bwd(dqw=None) == 1 and bwd(dkw=None) == 1

"""Attention over packed sequences without a GPU: the oracle against autograd, what the entry point refuses, the C ABI of
libmce_serve.so and what its kernels must not hold."""
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

from memarch_amd import _lib, attention
from oracle import attn_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = [os.path.join(ROOT, "include", h) for h in ("mce_pack.h", "mce_cache.h")]
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.mark.parametrize("window,sinks", [(0, 0), (4, 0), (3, 2)])
@pytest.mark.parametrize("lens,keys", [([5, 0, 9, 1], None), ([3, 4, 2], [7, 4, 0]), ([6], [4]), ([0, 2], [3, 9])])
def test_oracle_matches_autograd(lens, keys, window, sinks):
    g = torch.Generator().manual_seed(0)
    n, m = sum(lens) + 3, sum(keys or lens) + 3
    q, k, v, go = (torch.randn(r, h, 8, generator=g, dtype=torch.float64) for r, h in ((n, 4), (m, 2), (m, 2), (n, 4)))
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    out = torch.zeros(n, 4, 8, dtype=torch.float64)
    a = b = 2
    for x, y in zip(lens, keys or lens):
        i, j = torch.arange(x)[:, None] + y - x, torch.arange(y)[None]
        see = (j <= i) & ((i - j < (window or 10 ** 9)) | (j < sinks))
        for h in range(4):
            s = (q[a:a + x, h] @ k[b:b + y, h // 2].T) * 8 ** -0.5
            p = torch.nan_to_num(torch.softmax(s.masked_fill(~see, -1e300), -1) * see)
            out[a:a + x, h] = p @ v[b:b + y, h // 2]
        a, b = a + x, b + y
    ref = (out, *torch.autograd.grad(out, (q, k, v), go, allow_unused=True))
    cu = lambda l: torch.tensor([2] + l).cumsum(0).tolist()
    got = orc.packed(q.detach(), k.detach(), v.detach(), cu(lens), cu(keys) if keys else None, window, sinks, None, go)
    for x, y in zip(got, ref):
        assert (x - (0 if y is None else y)).abs().max() < 1e-12


def _bf(*shape, device="meta"):
    return torch.zeros(*shape, dtype=torch.bfloat16, device=device)


def test_packed_attention_refusals():
    pa = attention.packed_attention
    assert list(inspect.signature(pa).parameters) == \
        ["q", "k", "v", "cu_seqlens", "cu_seqlens_k", "window", "sinks", "scale"]
    q, k, cu = _bf(5, 4, 64), _bf(5, 2, 64), torch.zeros(3, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="GPU only"):
        pa(*(torch.zeros(5, 2, 64, dtype=torch.bfloat16) for _ in range(3)), torch.zeros(2, dtype=torch.int32))
    for args, match in (((q[0], k, k, cu), "must be"), ((q[None], k[None], k[None], cu), "must be"),
                        ((q, k, k[:4], cu), "one shape"), ((q, k[:4], k[:4], cu), "cu_seqlens_k"),
                        ((q, _bf(5, 3, 64), _bf(5, 3, 64), cu), "share"), ((q, _bf(5, 0, 64), _bf(5, 0, 64), cu), "share"),
                        ((_bf(5, 4, 60), _bf(5, 2, 60), _bf(5, 2, 60), cu), "head dimension"),
                        ((_bf(5, 4, 136), _bf(5, 2, 136), _bf(5, 2, 136), cu), "head dimension"),
                        ((q.float(), k.float(), k.float(), cu), "bfloat16"), ((q, k.half(), k.half(), cu), "bfloat16"),
                        ((q, k, k, cu.float()), "cu_seqlens"), ((q, k, k, cu[:0]), "cu_seqlens"),
                        ((q, k, k, cu[None]), "cu_seqlens"), ((q, k, k, cu, cu[:2]), "one shape"),
                        ((q, k, k, cu, cu.double()), "cu_seqlens_k"),
                        ((q, k, k, torch.zeros(3, dtype=torch.int32)), "cu_seqlens is on cpu")):
        with pytest.raises(ValueError, match=match):
            pa(*args)
    for kw, match in ((dict(window=0, sinks=3), "window"), (dict(window=-2), "window"), (dict(window=4, sinks=-1), "sinks"),
                      (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")):
        with pytest.raises(ValueError, match=match):
            pa(q, k, k, cu, **kw)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    launched = []
    monkeypatch.setattr(_lib, "call", lambda *a: launched.append(a[0]))
    monkeypatch.setattr(attention, "_check_same", lambda *a: None)
    monkeypatch.setattr(attention, "_stream", lambda dev: 0)
    monkeypatch.setattr(attention, "_On", lambda dev: contextlib.nullcontext())
    q, cu = _bf(3, 2, 64, device="cpu"), torch.tensor([0, 3], dtype=torch.int32)
    attention.packed_attention(q, q, q, cu)
    assert launched == ["mce_pack_fwd"]
    with fwAD.dual_level():
        for i in range(3):
            args = [q, q, q]
            args[i] = fwAD.make_dual(q.clone(), torch.ones_like(q))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                attention.packed_attention(*args, cu)
    assert len(launched) == 1


# ------------------------------------------------------------------------------------------------------ the library


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.SERVE_LIB_PATH):
        pytest.skip("libmce_serve.so not built")
    return _lib.load_serve()


def test_exports_every_declared_symbol(lib):
    src = "".join(open(h).read() for h in HEADERS if os.path.exists(h))
    names = re.findall(r"MCE_SERVE_API\s+[\w\s\*]+?\b(mce_\w+)\s*\(", src)
    assert len(names) == len(set(names)) >= 5
    for n in names:
        assert hasattr(lib, n), n
    assert set(names) == set(_lib.SERVE_SIGNATURES)
    assert not set(names) & (set(_lib.SIGNATURES) | set(_lib.ATTN_SIGNATURES))
    for code in range(6):
        assert lib.mce_serve_error_string(code)


@pytest.fixture(scope="module")
def kernels(lib, tmp_path_factory):
    """{kernel: its instructions} of the built library."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    d = tmp_path_factory.mktemp("isa")
    shutil.copy(_lib.SERVE_LIB_PATH, d / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=d, check=True, capture_output=True)
    out, name = {}, None
    for f in sorted(f for f in os.listdir(d) if f.endswith("gfx950")):
        for line in subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], cwd=d, check=True, capture_output=True,
                                   text=True).stdout.splitlines():
            m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
            if m:
                name = m[1]
                out[name] = []
            elif name and line.startswith("\t"):
                out[name].append(line.split("//")[0].strip())
    return out


def test_kernels_hold_no_l2_writeback_no_spills_and_no_packed_fp32(kernels):
    text = "\n".join(x for ins in kernels.values() for x in ins)
    assert "v_mfma_f32_32x32x16_bf16" in text and "v_mfma_f32_32x32x16_f16" in text
    for bad in ("buffer_wbl2", "v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32", "scratch_store"):
        assert bad not in text, bad


def test_loads_into_lds_wait_for_their_scalar_operands(kernels):
    """Each load into LDS stands behind five wait states of its own and behind a write of M0 that the compiler knows of."""
    loads = 0
    for name, ins in kernels.items():
        for i, x in enumerate(ins):
            if x.startswith("buffer_load") and x.endswith(" lds"):
                loads += 1
                m = re.fullmatch(r"s_nop (\d+)", ins[i - 1])
                assert m and int(m[1]) >= 4, (name, ins[i - 2:i + 1])
                back = next(y for y in ins[i - 1::-1] if re.match(r"\w+ m0,|s_c?branch|buffer_load.* lds$", y))
                assert " m0," in back, (name, back)
    assert loads > 50


def test_loops_wait_for_their_own_tile_only(kernels):
    """Behind the first load into LDS k_attn_dkv holds its own waits only: for the tile at hand and for all."""
    found = 0
    for name, ins in kernels.items():
        if "k_attn_dkvI" not in name:
            continue
        found += 1
        first = next(i for i, x in enumerate(ins) if x.endswith(" lds"))
        allowed = {0, 3, 6} if "Li64E" in name else {0, 5, 10}
        for i, x in enumerate(ins[first:], first):
            m = re.match(r"s_waitcnt vmcnt\((\d+)\)", x)
            if m:
                assert int(m[1]) in allowed and not ins[i + 1].startswith("v_mfma"), (name, ins[i - 1:i + 2])
    assert found == 4


def test_pack_c_abi_checks_need_no_gpu(lib):
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256

    def fwd(q=p, st=64, sh=64, k=p, cu=p, cu_k=p, nseq=2, N=8, M=9, Hq=2, Hkv=1, D=64, window=0, sinks=0, scale=0.1, dtype=1,
            out=p, res=None, plan=None, nb=0, ws=None, wb=0):
        return lib.mce_pack_fwd(q, st, sh, k, 64, 64, p, 64, 64, cu, cu_k, nseq, N, M, Hq, Hkv, D, window, sinks, scale,
                                dtype, out, res, None, plan, nb, ws, wb, None)

    for kw in (dict(N=-1), dict(M=-1), dict(nseq=-1), dict(Hq=3, Hkv=2), dict(Hkv=0), dict(D=60), dict(D=136), dict(D=0),
               dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(dtype=0), dict(q=None),
               dict(k=None), dict(out=None), dict(cu=None), dict(cu_k=None), dict(st=56), dict(st=1 << 22),
               dict(N=(1 << 27) + 1), dict(M=(1 << 27) + 1), dict(nseq=1 << 24), dict(nseq=1 << 23, Hq=4),
               dict(nseq=1 << 22, window=5, sinks=1 << 20, M=1 << 20)):
        assert fwd(**kw) == 1, kw
    for kw in (dict(q=p + 2), dict(out=p + 8), dict(res=p + 4), dict(st=68), dict(sh=4)):
        assert fwd(**kw) == 2, kw
    assert fwd(N=0, q=None, out=None, cu=None) == 0
    plan = lib.mce_pack_plan_bytes(2, 8000, 9000, 64, 1, 64, 0, 0)
    assert plan > 0 and lib.mce_pack_plan_bytes(2, 8, 9, 2, 1, 64, 0, 0) == 0
    big = dict(N=8000, M=9000, Hq=64)
    assert fwd(**big) == 3 and fwd(**big, plan=p, nb=plan - 1) == 3 and fwd(**big, plan=p + 16, nb=plan) == 3

    few = lib.mce_pack_fwd_ws_bytes(2, 8, 9000, 2, 1, 64, 0, 0)
    assert few >= 2 * 8 * 2 * 66 * 4 and lib.mce_pack_fwd_ws_bytes(2, 8, 9, 2, 1, 64, 0, 0) == 0
    assert lib.mce_pack_plan_bytes(2, 8, 9000, 2, 1, 64, 0, 0) == 0
    assert lib.mce_pack_bwd_ws_bytes(2, 8, 9000, 2, 1, 64, 0, 0) >= few + 2 * 2 * 8 * 4
    row = dict(N=8, M=9000)
    assert fwd(**row) == 3 and fwd(**row, ws=p, wb=few - 1) == 3 and fwd(**row, ws=p + 16, wb=few) == 3

    need = lib.mce_pack_bwd_ws_bytes(2, 8, 9, 2, 1, 64, 0, 0)
    assert need >= 2 * 2 * 8 * 4 and lib.mce_pack_bwd_ws_bytes(2, 8, 9, 3, 2, 64, 0, 0) == 0

    def bwd(ws=p, nb=need, go=p, lse=p, dq=p, dk=p, st=64, N=8, M=9, Hq=2, plan=None):
        return lib.mce_pack_bwd(p, 64, 64, p, 64, 64, p, 64, 64, go, st, 64, p, p, 2, N, M, Hq, 1, 64, 0, 0, 0.1, 1, p, p, lse,
                                plan, dq, dk, p, ws, nb, None)

    assert bwd(**big) == 3 and bwd(**big, plan=p + 16) == 3   # the forward's plan is missing

    assert bwd(ws=None) == 3 and bwd(nb=need - 1) == 3 and bwd(ws=p + 16) == 3
    assert bwd(go=None) == 1 and bwd(lse=None) == 1 and bwd(dq=None) == 1 and bwd(dk=None) == 1 and bwd(st=8) == 1
    assert bwd(dq=p + 2) == 2 and bwd(dk=p + 2) == 2 and bwd(N=0, M=0, go=None, dq=None, dk=None, ws=None) == 0

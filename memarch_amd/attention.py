"""Causal attention over a sliding window with first tokens that stay visible, over a padded batch or packed sequences, and
its form for one new token per sequence over a paged cache, on MI355X (libmce_attn.so, libmce_serve.so).

`window_attention(q, k, v, window, sinks, lengths)` stands where memarch's blocks call scaled_dot_product_attention or
their block-window helpers (lm.py:448-554, full2.py:154-181): one kernel forward, two backward, no scores in memory.
Position i of a sequence sees position j <= i when i - j < window or j < sinks. Products take bf16 or fp16 operands and
sum in fp32; softmax statistics are fp32 (include/mce_attn.h, include/mce_paged.h). `paged_attention` is the last row of
the same attention for each sequence, its keys and values lying in the pages of a cache. All device work runs on
torch's current stream; a tensor that is not on a GPU raises, and there is no other code path.
"""
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .fused_ops import _ptr, _stream

# element-type codes of include/mce_attn.h
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
MAX_HEAD_DIM = 128
_MAX_INT = 2 ** 31 - 1   # more than any position
_MAX_STRIDE = 1 << 21   # elements between two tokens (the library's limit)


def _check_same(ref, *named):
    """All tensors on ref's GPU."""
    for name, t in named:
        if t is not None and t.device != ref.device:
            raise ValueError(f"{name} is on {t.device}, expected {ref.device}")
    if not ref.is_cuda:
        raise ValueError("memarch_amd.attention runs on the GPU only; got a tensor on " + str(ref.device))


def _check_tangents(*tensors):
    """Refuses dual tensors: the kernels have no forward-mode derivative, and their fresh outputs would carry no tangent,
    which forward mode takes for zero. Outside a dual level (the usual case) no tensor is looked at."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise NotImplementedError("the attention operators have no forward-mode derivative; got a dual tensor")


class _On:
    """Makes the tensors' GPU current around a launch if it is not (a launch goes to the current device)."""

    def __init__(self, dev):
        self.dev = dev
        self.prev = -1

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.dev.index:
            self.prev = cur
            torch.cuda.set_device(self.dev)

    def __exit__(self, *exc):
        if self.prev >= 0:
            torch.cuda.set_device(self.prev)


def _strided(t):
    """(tensor, (pointer, batch, token, head strides)) of a [B, T, H, D] operand: the tensor itself when the library
    can read it where it lies (contiguous last dimension, 16-byte alignment, tokens at least D apart), else a
    contiguous copy."""
    t = t.detach()
    b, n, h, d = t.shape
    sb, st, sh, sd = t.stride()
    sb, st, sh = sb if b > 1 else 0, st if n > 1 else d, sh if h > 1 else 0
    if sd != 1 or (sb | st | sh) & 7 or not d <= st <= _MAX_STRIDE or t.data_ptr() & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        sb, st, sh = n * h * d, h * d, d
    return t, (t.data_ptr(), sb, st, sh)


def _lengths(lengths, b, most):
    """[B] int32 device lengths (None: all of them whole); values outside 0 .. most count as the nearest of the two."""
    if lengths is None:
        return None
    if lengths.dim() != 1 or lengths.shape[0] != b or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"lengths must be [B={b}] int32 or int64, got {tuple(lengths.shape)} {lengths.dtype}")
    if lengths.dtype is torch.int64:
        lengths = lengths.clamp(0, most).int()
    return lengths.contiguous()


def _mask_args(window, sinks):
    window = 0 if window is None else int(window)
    if window < 0 or (window == 0 and sinks):
        raise ValueError("window must be at least 1 (None: every earlier position is seen, without sinks)")
    if sinks < 0:
        raise ValueError(f"sinks={sinks} must not be negative")
    return min(window, _MAX_INT), min(int(sinks), _MAX_INT)


def _scale(scale, d):
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"scale={scale} must be positive and between 1e-30 and 1e30")
    return scale


def _check_heads(q, k, v, what):
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    if q.shape[-1] != k.shape[-1] or q.shape[-1] % 8 or not 8 <= q.shape[-1] <= MAX_HEAD_DIM:
        raise ValueError(f"the head dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, alike for all, got "
                         f"{q.shape[-1]} and {k.shape[-1]}")
    if k.shape[-2] < 1 or q.shape[-2] < 1 or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"{q.shape[-2]} query heads cannot share {k.shape[-2]} key/value heads")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what} must all be bfloat16 or all float16, got {q.dtype}, {k.dtype} and {v.dtype}")


def _forward(q, k, v, lengths, window, sinks, scale, train):
    B, T, Hq, D = q.shape
    (q, qs), (k, ks), (v, vs) = _strided(q), _strided(k), _strided(v)
    out = torch.empty(B, T, Hq, D, dtype=q.dtype, device=q.device)
    res = torch.empty_like(out) if train else None
    lse = torch.empty(B, Hq, T, dtype=torch.float32, device=q.device) if train else None
    with _On(q.device):
        _lib.call("mce_attn_fwd", *qs, *ks, *vs, _ptr(lengths), B, T, Hq, k.shape[2], D, window, sinks, scale,
                  _DTYPES[q.dtype], out.data_ptr(), _ptr(res), _ptr(lse), _stream(q.device))
    return q, k, v, out, res, lse


def _mark_leaves(out, dev):
    """Leaves the current stream's number on the gradient accumulators of the call's leaves, which live as long as a graph
    that uses them."""
    here = _stream(dev)
    for node, _ in out.grad_fn.next_functions:
        if node is not None and type(node).__name__ == "AccumulateGrad":
            node.metadata.setdefault("memarch_stream", here)


def _check_capture(ctx, dev):
    """Refuses to capture a backward whose leaves an earlier graph still holds: autograd makes their accumulators wait on
    the stream where that graph was made, which draws the stream into the capture and ends the process."""
    if not torch.cuda.is_current_stream_capturing():
        return
    here = _stream(dev)
    for node, _ in ctx.next_functions:
        if node is not None and type(node).__name__ == "AccumulateGrad" and \
                node.metadata.get("memarch_stream", here) != here:
            raise RuntimeError("a backward cannot be captured while a graph of the same leaves that was made on another "
                               "stream is alive: delete its outputs first, or capture with detached leaves")


class _WindowAttention(torch.autograd.Function):
    """forward(ctx, q, k, v, lengths, window, sinks, scale) -> out; backward -> dq, dk, dv."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, window, sinks, scale):
        q, k, v, out, res, lse = _forward(q, k, v, lengths, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, out, res, lse, lengths)
        ctx.mask = (window, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, out, res, lse, lengths = ctx.saved_tensors
        _check_capture(ctx, q.device)
        window, sinks, scale = ctx.mask
        B, T, Hq, D = q.shape
        Hkv = k.shape[2]
        (q, qs), (k, ks), (v, vs), (go, gs) = _strided(q), _strided(k), _strided(v), _strided(go)
        dq = torch.empty(B, T, Hq, D, dtype=q.dtype, device=q.device)
        dk = torch.empty(B, T, Hkv, D, dtype=q.dtype, device=q.device)
        dv = torch.empty_like(dk)
        n = _lib.load_attn().mce_attn_bwd_ws_bytes(B, T, Hq, Hkv, D, window, sinks)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        with _On(q.device):
            _lib.call("mce_attn_bwd", *qs, *ks, *vs, *gs, _ptr(lengths), B, T, Hq, Hkv, D, window, sinks, scale,
                      _DTYPES[q.dtype], out.data_ptr(), res.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                      ws.data_ptr(), n, _stream(q.device))
        return dq, dk, dv, None, None, None, None


@torch.compiler.disable
def window_attention(q, k, v, window=None, sinks=0, lengths=None, scale=None):
    """Causal attention of q [B, T, Hq, D] over k, v [B, T, Hkv, D] (bf16 or fp16, Hq a multiple of Hkv, D a multiple of
    8 up to 128, any strides) -> [B, T, Hq, D]. Position i sees j <= i with i - j < window or j < sinks (window None:
    every j <= i). lengths [B] marks a padded batch: positions at or past a sequence's length see nothing and are seen
    by none, their output and gradients are 0 and what lies in their rows is not read (inside a length, a NaN or an
    infinity may reach rows near it that do not see it, as 0 * NaN does in a dense form). scale defaults to D^-0.5.
    Under torch.autocast fp32 tensors are cast to its type, as for scaled_dot_product_attention. Differentiable once
    in q, k and v, in reverse mode: a tensor with a forward-mode tangent raises. Capturing a backward raises while an earlier
    graph of leaves that are q, k or v themselves, made here or by packed_attention on another stream, is alive (as for any
    operator, one of leaves farther up must not be)."""
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = (t.to(dt) if t.dtype is torch.float32 else t for t in (q, k, v))
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or q.shape[:2] != k.shape[:2]:
        raise ValueError(f"q {tuple(q.shape)} must be [B, T, Hq, D], k {tuple(k.shape)} and v {tuple(v.shape)} "
                         "[B, T, Hkv, D]")
    _check_heads(q, k, v, "q, k and v")
    window, sinks = _mask_args(window, sinks)
    scale = _scale(scale, q.shape[3])
    lengths = _lengths(lengths, q.shape[0], q.shape[1])
    _check_same(q, ("k", k), ("v", v), ("lengths", lengths))
    _check_tangents(q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _WindowAttention.apply(q, k, v, lengths, window, sinks, scale)
        _mark_leaves(out, q.device)
        return out
    return _forward(q, k, v, lengths, window, sinks, scale, False)[3]


def _packed_forward(q, k, v, cu, cu_k, window, sinks, scale, train):
    N, Hq, D = q.shape
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    out = torch.empty(N, Hq, D, dtype=q.dtype, device=q.device)
    res = torch.empty_like(out) if train else None
    lse = torch.empty(Hq, N, dtype=torch.float32, device=q.device) if train else None
    lib, sizes = _lib.load_serve(), (cu.shape[0] - 1, N, k.shape[0], Hq, k.shape[1], D, window, sinks)
    n, w = lib.mce_pack_plan_bytes(*sizes), lib.mce_pack_fwd_ws_bytes(*sizes)
    plan = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    ws = torch.empty(w, dtype=torch.uint8, device=q.device) if w else None
    with _On(q.device):
        _lib.call("mce_pack_fwd", *qs, *ks, *vs, cu.data_ptr(), _ptr(cu_k), *sizes, scale, _DTYPES[q.dtype], out.data_ptr(),
                  _ptr(res), _ptr(lse), _ptr(plan), n, _ptr(ws), w, _stream(q.device))
    return q, k, v, out, res, lse, plan


class _PackedAttention(torch.autograd.Function):
    """forward(ctx, q, k, v, cu, cu_k, window, sinks, scale) -> out; backward -> dq, dk, dv."""

    @staticmethod
    def forward(ctx, q, k, v, cu, cu_k, window, sinks, scale):
        q, k, v, out, res, lse, plan = _packed_forward(q, k, v, cu, cu_k, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, out, res, lse, plan, cu, cu_k)
        ctx.mask = (window, sinks, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, out, res, lse, plan, cu, cu_k = ctx.saved_tensors
        _check_capture(ctx, q.device)
        window, sinks, scale = ctx.mask
        (N, Hq, D), (M, Hkv, _) = q.shape, k.shape
        nseq = cu.shape[0] - 1
        (q, qs), (k, ks), (v, vs), (go, gs) = _rows(q), _rows(k), _rows(v), _rows(go)
        dq = torch.empty(N, Hq, D, dtype=q.dtype, device=q.device)
        dk = torch.empty(M, Hkv, D, dtype=q.dtype, device=q.device)
        dv = torch.empty_like(dk)
        n = _lib.load_serve().mce_pack_bwd_ws_bytes(nseq, N, M, Hq, Hkv, D, window, sinks)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        with _On(q.device):
            _lib.call("mce_pack_bwd", *qs, *ks, *vs, *gs, cu.data_ptr(), _ptr(cu_k), nseq, N, M, Hq, Hkv, D, window, sinks,
                      scale, _DTYPES[q.dtype], out.data_ptr(), res.data_ptr(), lse.data_ptr(), _ptr(plan), dq.data_ptr(),
                      dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n, _stream(q.device))
        return dq, dk, dv, None, None, None, None, None


def _rows(t):
    """_strided of a packed [N, H, D] operand: (tensor, (pointer, token, head strides))."""
    n, h, d = t.shape
    st, sh, sd = t.stride()
    if n < 2:
        st = d
    if h < 2:
        sh = 0
    at = t.data_ptr()
    if sd != 1 or (st | sh) & 7 or not d <= st <= _MAX_STRIDE or at & 15:
        t = t.detach().contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        at, st, sh = t.data_ptr(), h * d, d
    return t, (at, st, sh)


def _starts(t, name):
    """[nseq + 1] int32 device starts of packed sequences."""
    if t.dim() != 1 or t.shape[0] < 1 or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be [sequences + 1] int32 or int64, got {tuple(t.shape)} {t.dtype}")
    if t.dtype is torch.int64:
        t = t.clamp(0, _MAX_INT).int()
    return t.contiguous()


@torch.compiler.disable
def packed_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, window=None, sinks=0, scale=None):
    """Causal attention over packed sequences of different lengths, q [N, Hq, D] over k, v [M, Hkv, D] -> [N, Hq, D]: the
    types, heads, mask, scale, autocast and derivatives of window_attention without its padding. Sequence b holds rows
    cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (int32 or int64 [sequences + 1], not falling). With cu_seqlens_k, k and v have
    rows of their own for each sequence, and a sequence's queries are the last of its positions (the next piece of a text
    whose earlier keys are at hand): row i of n is position i + m - n of m. Rows that see nothing (m < n, or outside every
    sequence) and the gradients of rows that nothing sees are 0. The numbers stay on the device: they are not checked, a
    call does not wait for them, and a captured call may be replayed with others. Capturing a backward raises where that of
    window_attention does."""
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = (t.to(dt) if t.dtype is torch.float32 else t for t in (q, k, v))
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"q {tuple(q.shape)} must be [N, Hq, D], k {tuple(k.shape)} and v {tuple(v.shape)} [M, Hkv, D]")
    _check_heads(q, k, v, "q, k and v")
    if cu_seqlens_k is None and k.shape[0] != q.shape[0]:
        raise ValueError(f"{q.shape[0]} rows of q and {k.shape[0]} of k ask for cu_seqlens_k")
    if cu_seqlens_k is not None and cu_seqlens_k.shape != cu_seqlens.shape:
        raise ValueError(f"cu_seqlens {tuple(cu_seqlens.shape)} and cu_seqlens_k {tuple(cu_seqlens_k.shape)} must have one "
                         "shape")
    window, sinks = _mask_args(window, sinks)
    scale = _scale(scale, q.shape[2])
    cu = _starts(cu_seqlens, "cu_seqlens")
    cu_k = None if cu_seqlens_k is None else _starts(cu_seqlens_k, "cu_seqlens_k")
    _check_same(q, ("k", k), ("v", v), ("cu_seqlens", cu), ("cu_seqlens_k", cu_k))
    _check_tangents(q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _PackedAttention.apply(q, k, v, cu, cu_k, window, sinks, scale)
        _mark_leaves(out, q.device)
        return out
    return _packed_forward(q, k, v, cu, cu_k, window, sinks, scale, False)[3]


def _cache(t, name):
    """Element strides (page, slot, head) of a cache, which is never copied: the library reads it where it lies."""
    _, page, h, d = t.shape
    sp, st, sh, sd = t.stride()
    sh = sh if h > 1 else 0
    if sd != 1 or (sp | st | sh) & 7 or not d <= st <= _MAX_STRIDE or t.data_ptr() & 15:
        raise ValueError(f"{name} must have a contiguous last dimension, a 16-byte aligned base, strides that are "
                         f"multiples of 8 and slots at least {d} elements apart, got strides {t.stride()}")
    return t.data_ptr(), sp, st, sh


@torch.compiler.disable
@torch.no_grad()
def paged_attention(q, k_cache, v_cache, block_table, lengths, window=None, sinks=0, scale=None):
    """Attention of one new token per sequence, q [B, Hq, D], over the pages of a cache, k_cache and v_cache [pages,
    page, Hkv, D] (bf16 or fp16; page and D multiples of 8, D up to 128) -> [B, Hq, D]. Token j of sequence b lies in
    page block_table[b, j // page] (int32 [B, max_pages]) at slot j % page; lengths [B] (int32 or int64) counts a
    sequence's cached tokens with the new one, whose keys and values are in the cache already. The mask is that of
    window_attention's last row. A sequence of length 0 gives 0; tokens in pages outside the cache (entries of -1, say)
    and past max_pages are not seen. The caches are read where they lie, 16 bytes at a time. No gradient; a tensor with a
    forward-mode tangent raises."""
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError(f"q {tuple(q.shape)} must be [B, Hq, D], k_cache {tuple(k_cache.shape)} and v_cache "
                         f"{tuple(v_cache.shape)} [pages, page, Hkv, D]")
    _check_heads(q, k_cache, v_cache, "q and the caches")
    B, Hq, D = q.shape
    pages, page, Hkv, _ = k_cache.shape
    if page < 8 or page % 8 or page > 65536:
        raise ValueError(f"pages of {page} tokens are not supported (a multiple of 8 up to 65536 is)")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype is not torch.int32:
        raise ValueError(f"block_table must be int32 [B={B}, max_pages], got {tuple(block_table.shape)} "
                         f"{block_table.dtype}")
    if block_table.shape[1] * page > min(2 ** 30, 2 ** 38 // page):
        raise ValueError(f"{block_table.shape[1]} pages of {page} tokens per sequence are not supported (2^30 tokens, "
                         "2^38 / page)")
    window, sinks = _mask_args(window, sinks)
    scale = _scale(scale, D)
    if lengths is None:
        raise ValueError("lengths must be given")
    lengths = _lengths(lengths, B, _MAX_INT)
    _check_same(q, ("k_cache", k_cache), ("v_cache", v_cache), ("block_table", block_table), ("lengths", lengths))
    _check_tangents(q, k_cache, v_cache)
    max_pages = block_table.shape[1]
    if max_pages > 1 and block_table.stride(1) != 1 or B > 1 and block_table.stride(0) < max_pages:
        block_table = block_table.contiguous()
    sb, sh, sd = q.stride()
    sb, sh = sb if B > 1 else 0, sh if Hq > 1 else D
    if sd != 1 or (sb | sh) & 7 or not D <= sh <= _MAX_STRIDE or q.data_ptr() & 15:
        q = q.contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
        sb, sh = Hq * D, D
    kc, vc = _cache(k_cache, "k_cache"), _cache(v_cache, "v_cache")
    out = torch.empty(B, Hq, D, dtype=q.dtype, device=q.device)
    n = _lib.load_attn().mce_paged_ws_bytes(B, Hq, Hkv, D, page, max_pages, window, sinks)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    with _On(q.device):
        _lib.call("mce_paged", q.data_ptr(), sb, sh, *kc, *vc, block_table.data_ptr(),
                  block_table.stride(0) if B > 1 else 0, lengths.data_ptr(), B, Hq, Hkv, D, pages, page, max_pages,
                  window, sinks, scale, _DTYPES[q.dtype], out.data_ptr(), _ptr(ws), n, _stream(q.device))
    return out

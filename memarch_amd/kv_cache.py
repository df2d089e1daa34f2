"""A paged key/value cache held in 8 bits on MI355X (libmce_serve.so): `cache_write` quantises new tokens' keys and values
into it, `cache_read` gives them back, `cache_attention` is one new token's attention over it, as paged_attention is over a
cache of 16-bit elements.

k_cache and v_cache are float8_e4m3fn [pages, page, Hkv, D], k_scale and v_scale float32 [pages, page // block, Hkv]: `block`
neighbouring slots of a page and a head share a scale, a value is its code times its scale. Token j of sequence b lies in
page block_table[b, j // page] (int32 [B, max_pages]) at slot j % page. The rules of the scales, which are powers of two,
are in include/mce_cache.h. All device work runs on torch's current stream; a tensor that is not on a GPU raises, and there
is no other code path. None of the three has a gradient; a tensor with a forward-mode tangent raises.
"""
import torch

from . import _lib
from .attention import (_DTYPES, _MAX_INT, _MAX_STRIDE, MAX_HEAD_DIM, _check_tangents, _lengths, _mask_args, _On, _rows,
                        _scale, _starts)
from .fused_ops import _ptr, _stream

MAX_BLOCK = 128   # slots that share a scale


_F8, _F32, _I32 = torch.float8_e4m3fn, torch.float32, torch.int32


def _check_same(ref, *named):
    """All tensors on ref's GPU."""
    dev = ref.device
    for name, t in named:
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if dev.type != "cuda":
        raise ValueError("memarch_amd.kv_cache runs on the GPU only; got a tensor on " + str(dev))


def _codes(cache, scale, shape, name):
    """(pointer, byte strides of page, slot and head, scale's pointer) of a cache, which is read and written where it lies."""
    sp, st, sh, sd = cache.stride()
    if shape[0] < 2:
        sp = 0
    if shape[2] < 2:
        sh = 0
    at = cache.data_ptr()
    if (sd != 1 or (sp | st | sh | at) & 15 or not shape[3] <= st <= _MAX_STRIDE) and shape[0]:
        raise ValueError(f"{name} must have a contiguous last dimension, a 16-byte aligned base, strides that are multiples "
                         f"of 16 and slots at least {shape[3]} elements apart, got strides {cache.stride()}")
    if not scale.is_contiguous():
        raise ValueError(f"{name}'s scales must be contiguous")
    return at, sp, st, sh, scale.data_ptr()


def _check_written(k_cache, v_cache, k_scale, v_scale):
    """Refuses a cache two of whose elements share memory (expanded heads, one buffer for both): several waves would write it."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        span = 1   # of the dimensions with smaller strides
        for stride, n in () if t.is_contiguous() else sorted(zip(t.stride(), t.shape)):
            if n > 1:
                if stride < span:
                    raise ValueError(f"{name}, which is written, has elements that share memory: {tuple(t.shape)}, strides "
                                     f"{t.stride()}")
                span += stride * (n - 1)
    if k_cache.data_ptr() == v_cache.data_ptr() != 0 or k_scale.data_ptr() == v_scale.data_ptr() != 0:
        raise ValueError("the keys and values, or their scales, are written to the same memory")


def _check_cache(k_cache, v_cache, k_scale, v_scale, block_table):
    """The cache's shape [pages, page, Hkv, D], its block and the table's max_pages."""
    shape = k_cache.shape
    if k_cache.dtype is not _F8 or v_cache.dtype is not _F8 or len(shape) != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache and v_cache must be float8_e4m3fn [pages, page, Hkv, D], got "
                         f"{tuple(shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}")
    if v_cache.shape != shape:
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(v_cache.shape)} must have one shape")
    pages, page, h, d = shape
    if h < 1 or d % 16 or not 16 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"the head dimension must be a multiple of 16 up to {MAX_HEAD_DIM}, got {h} heads of {d}")
    if page < 8 or page % 8 or page > 65536:
        raise ValueError(f"pages of {page} tokens are not supported (a multiple of 8 up to 65536 is)")
    per = k_scale.shape[1] if k_scale.dim() == 3 else 0
    want = (pages, per, h)
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype is not _F32 or t.shape != want or per < 1 or page % per:
            raise ValueError(f"{name} must be float32 [pages={pages}, page / block, Hkv={h}], alike for both, got "
                             f"{tuple(t.shape)} {t.dtype}")
    block = page // per
    if block < 8 or block % 8 or block > MAX_BLOCK:
        raise ValueError(f"blocks of {block} tokens are not supported (a multiple of 8 up to {MAX_BLOCK} is)")
    if block_table.dim() != 2 or block_table.dtype is not _I32:
        raise ValueError(f"block_table must be int32 [B, max_pages], got {tuple(block_table.shape)} {block_table.dtype}")
    most = block_table.shape[1]
    if most * page > min(2 ** 30, 2 ** 38 // page):
        raise ValueError(f"{most} pages of {page} tokens per sequence are not supported (2^30 tokens, 2^38 / page)")
    return shape, block, most


def _table(t):
    """(tensor, row stride) of a block table whose rows the library can read."""
    b, most = t.shape
    if most > 1 and t.stride(1) != 1 or b > 1 and t.stride(0) < most:
        t = t.contiguous()
    return t, t.stride(0) if b > 1 else 0


@torch.compiler.disable
def cache_write(k, v, k_cache, v_cache, k_scale, v_scale, block_table, lengths, cu_seqlens=None):
    """Writes the keys and values of new tokens, k and v [N, Hkv, D] (bf16 or fp16, any strides), into the cache in place.
    cu_seqlens [B + 1] (int32 or int64): rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 are the last tokens of sequence b, which
    has lengths[b] with them (int32 or int64 [B], the argument that cache_attention takes afterwards); without it row b is
    sequence b's one new token. A block of slots that gets tokens keeps those in front of them; its scale grows with what is
    written, never shrinks while it holds older tokens, and starts anew with its first slot. Tokens whose page is outside
    the cache (entries of -1, say) are left out. A page that gets tokens must belong to one sequence. A cache whose elements
    share memory raises."""
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must both be [N, Hkv, D]")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise ValueError(f"k and v must both be bfloat16 or both float16, got {k.dtype} and {v.dtype}")
    shape, block, most = _check_cache(k_cache, v_cache, k_scale, v_scale, block_table)
    _check_written(k_cache, v_cache, k_scale, v_scale)
    pages, page, h, d = shape
    if k.shape[1:] != (h, d):
        raise ValueError(f"k {tuple(k.shape)} does not fit a cache of {h} heads of {d}")
    B, N = block_table.shape[0], k.shape[0]
    if lengths is None:
        raise ValueError("lengths must be given")
    if cu_seqlens is None and N != B:
        raise ValueError(f"{N} rows for {B} sequences ask for cu_seqlens")
    if cu_seqlens is not None and cu_seqlens.shape != (B + 1,):
        raise ValueError(f"cu_seqlens must be [B + 1 = {B + 1}], got {tuple(cu_seqlens.shape)}")
    lengths = _lengths(lengths, B, _MAX_INT)
    cu = None if cu_seqlens is None else _starts(cu_seqlens, "cu_seqlens")
    _check_same(k, ("v", v), ("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale),
                ("block_table", block_table), ("lengths", lengths), ("cu_seqlens", cu))
    _check_tangents(k, v, k_cache, v_cache, k_scale, v_scale)
    kc, vc = _codes(k_cache, k_scale, shape, "k_cache"), _codes(v_cache, v_scale, shape, "v_cache")
    (k, ks), (v, vs) = _rows(k), _rows(v)
    block_table, bt = _table(block_table)
    with _On(k.device):
        _lib.call("mce_cache_write", *ks, *vs, *kc[:4], *vc[:4], kc[4], vc[4], block_table.data_ptr(), bt,
                  lengths.data_ptr(), _ptr(cu), B, N, h, d, pages, page, block, most, _DTYPES[k.dtype], _stream(k.device))
    # they were changed, as by an operation in place
    torch.autograd.graph.increment_version([t for t in (k_cache, v_cache, k_scale, v_scale) if not t.is_inference()])


@torch.compiler.disable
def cache_read(k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, rows, dtype=torch.bfloat16):
    """The first tokens of each sequence out of the cache, (k, v) [rows, Hkv, D] of bf16 or fp16: token j of sequence b in
    row cu_seqlens[b] + j, up to cu_seqlens[b + 1] - 1 (int32 or int64 [B + 1]). packed_attention takes them with
    cu_seqlens_k = cu_seqlens. Rows outside every sequence, and tokens whose page is outside the cache, are 0."""
    shape, block, most = _check_cache(k_cache, v_cache, k_scale, v_scale, block_table)
    pages, page, h, d = shape
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
    rows = int(rows)
    if not 0 <= rows <= 2 ** 27:
        raise ValueError(f"rows={rows} must be between 0 and 2^27")
    B = block_table.shape[0]
    if cu_seqlens.shape != (B + 1,):
        raise ValueError(f"cu_seqlens must be [B + 1 = {B + 1}], got {tuple(cu_seqlens.shape)}")
    cu = _starts(cu_seqlens, "cu_seqlens")
    _check_same(k_cache, ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale), ("block_table", block_table),
                ("cu_seqlens", cu))
    _check_tangents(k_cache, v_cache, k_scale, v_scale)
    kc, vc = _codes(k_cache, k_scale, shape, "k_cache"), _codes(v_cache, v_scale, shape, "v_cache")
    block_table, bt = _table(block_table)
    k = torch.empty(rows, h, d, dtype=dtype, device=k_cache.device)
    v = torch.empty_like(k)
    with _On(k.device):
        _lib.call("mce_cache_read", *kc[:4], *vc[:4], kc[4], vc[4], block_table.data_ptr(), bt, cu.data_ptr(), B, rows, h, d,
                  pages, page, block, most, _DTYPES[dtype], k.data_ptr(), v.data_ptr(), _stream(k.device))
    return k, v


@torch.compiler.disable
def cache_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, window=None, sinks=0, scale=None):
    """paged_attention over the 8-bit cache: attention of one new token per sequence, q [B, Hq, D] (bf16 or fp16, Hq a
    multiple of Hkv) -> [B, Hq, D]. lengths [B] (int32 or int64) counts a sequence's tokens with the new one, which
    cache_write has put there. The mask is that of window_attention's last row. A sequence of length 0 gives 0; tokens in
    pages outside the cache (entries of -1, say) and past max_pages are not seen. The same call gives the same bits; the last
    bits of a sequence may differ between batches whose other lengths differ, as those decide where its sums are cut."""
    shape, block, most = _check_cache(k_cache, v_cache, k_scale, v_scale, block_table)
    pages, page, h, d = shape
    if q.dim() != 3 or q.shape[2] != d or q.shape[1] < 1 or q.shape[1] % h:
        raise ValueError(f"q {tuple(q.shape)} must be [B, Hq, {d}], Hq a multiple of {h}")
    if q.dtype not in _DTYPES:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    B, Hq, _ = q.shape
    if block_table.shape[0] != B:
        raise ValueError(f"block_table {tuple(block_table.shape)} must have {B} rows")
    window, sinks = _mask_args(window, sinks)
    scale = _scale(scale, d)
    if lengths is None:
        raise ValueError("lengths must be given")
    lengths = _lengths(lengths, B, _MAX_INT)
    _check_same(q, ("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale),
                ("block_table", block_table), ("lengths", lengths))
    _check_tangents(q, k_cache, v_cache, k_scale, v_scale)
    kc, vc = _codes(k_cache, k_scale, shape, "k_cache"), _codes(v_cache, v_scale, shape, "v_cache")
    block_table, bt = _table(block_table)
    sb, sh, sd = q.stride()
    sb, sh = sb if B > 1 else 0, sh if Hq > 1 else d
    if sd != 1 or (sb | sh) & 7 or not d <= sh <= _MAX_STRIDE or q.data_ptr() & 15:
        q = q.detach().contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
        sb, sh = Hq * d, d
    out = torch.empty(B, Hq, d, dtype=q.dtype, device=q.device)
    n = _lib.load_serve().mce_cache_attn_ws_bytes(B, Hq, h, d, page, most, window, sinks)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    with _On(q.device):
        _lib.call("mce_cache_attn", q.data_ptr(), sb, sh, *kc[:4], *vc[:4], kc[4], vc[4], block_table.data_ptr(), bt,
                  lengths.data_ptr(), B, Hq, h, d, pages, page, block, most, window, sinks, scale, _DTYPES[q.dtype],
                  out.data_ptr(), _ptr(ws), n, _stream(q.device))
    return out

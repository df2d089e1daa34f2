"""Norms of queries and keys for each head and their position rotation in one pass, on MI355X (libmce_attn.so).

`qk_norm_rope(q, k, cos, sin, q_weight, k_weight)` stands where memarch's blocks norm and rotate with torch operations
(baseline.py:35-53): one kernel forward and, with the weights' gradients, two backward. With norm=False it is the
rotation alone. `rope_table` makes the cosines and sines it reads. All arithmetic is fp32 (include/mce_rope.h); device
work runs on torch's current stream, a tensor that is not on a GPU raises, and there is no other code path.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import _check_same, _check_tangents, _On
from .fused_ops import _ptr, _stream

# element-type codes of include/mce_rope.h
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_HEAD_DIM = 256


def rope_table(n, rot_dim, theta=10000.0, scale=1.0, device=None):
    """cos, sin [n, rot_dim / 2] fp32 of the angles (position / scale) * theta^(-2i / rot_dim), formed in fp64 (at
    position 2^17 an fp32 angle is off by 4e-3). scale > 1 stretches the positions a model was trained on over longer
    texts."""
    if n < 0 or rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"n={n} must not be negative, rot_dim={rot_dim} must be even and at least 2")
    if not (theta > 0 and scale > 0):
        raise ValueError(f"theta={theta} and scale={scale} must be positive")
    freq = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    ang = torch.arange(n, dtype=torch.float64, device=device)[:, None] / scale * freq
    return ang.cos().float(), ang.sin().float()


def _operand(t):
    """(tensor, (pointer, batch, token, head strides)) of [B, T, H, D], copied only if its last dimension is strided."""
    t = t.detach()
    if t.stride(3) != 1 and t.shape[3] > 1:
        t = t.contiguous()
    (b, n, h, _), (sb, st, sh, _) = t.shape, t.stride()
    return t, (t.data_ptr(), sb if b > 1 else 0, st if n > 1 else 0, sh if h > 1 else 0)


def _table_args(cos, sin, positions):
    pos = (None, 0, 0, 0) if positions is None else (
        positions.data_ptr(), int(positions.dtype is torch.int64), *positions.stride())
    return cos.data_ptr(), sin.data_ptr(), cos.shape[0], *pos


def _forward(q, k, cos, sin, positions, qw, kw, norm, eps, interleaved):
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    (q, qs), (k, ks) = _operand(q), _operand(k)
    yq = torch.empty(B, T, Hq, D, dtype=q.dtype, device=q.device)
    yk = torch.empty(B, T, Hkv, D, dtype=q.dtype, device=q.device)
    with _On(q.device):
        _lib.call("mce_rope_fwd", *qs, *ks, *_table_args(cos, sin, positions), _ptr(qw), _ptr(kw), B, T, Hq, Hkv, D,
                  2 * cos.shape[1], norm, eps, interleaved, _DTYPES[q.dtype], yq.data_ptr(), yk.data_ptr(),
                  _stream(q.device))
    return q, k, yq, yk


class _QKNormRope(torch.autograd.Function):
    """forward(ctx, q, k, cos, sin, positions, qw, kw, norm, eps, interleaved) -> rotated q and k; backward -> the
    gradients of q, k, qw and kw."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, qw, kw, norm, eps, interleaved):
        q, k, yq, yk = _forward(q, k, cos, sin, positions, qw, kw, norm, eps, interleaved)
        ctx.save_for_backward(q, k, cos, sin, positions, qw, kw)
        ctx.args = (norm, eps, interleaved)
        return yq, yk

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, cos, sin, positions, qw, kw = ctx.saved_tensors
        norm, eps, interleaved = ctx.args
        B, T, Hq, D = q.shape
        Hkv = k.shape[2]
        (q, qs), (k, ks), (gq, gqs), (gk, gks) = _operand(q), _operand(k), _operand(gq), _operand(gk)
        dq = torch.empty(B, T, Hq, D, dtype=q.dtype, device=q.device)
        dk = torch.empty(B, T, Hkv, D, dtype=q.dtype, device=q.device)
        dw = ws = None
        n = 0
        if norm and (ctx.needs_input_grad[5] or ctx.needs_input_grad[6]):
            dw = torch.empty(2, D, dtype=torch.float32, device=q.device)
            n = _lib.load_attn().mce_rope_bwd_ws_bytes(B, T, Hq, Hkv, D, norm)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        dqw, dkw = (None, None) if dw is None else (dw[0], dw[1])
        with _On(q.device):
            _lib.call("mce_rope_bwd", *qs, *ks, *gqs, *gks, *_table_args(cos, sin, positions), _ptr(qw), _ptr(kw),
                      B, T, Hq, Hkv, D, 2 * cos.shape[1], norm, eps, interleaved, _DTYPES[q.dtype], dq.data_ptr(),
                      dk.data_ptr(), _ptr(dqw), _ptr(dkw), _ptr(ws), n, _stream(q.device))
        return dq, dk, None, None, None, dqw, dkw, None, None, None


@torch.compiler.disable
def qk_norm_rope(q, k, cos, sin, q_weight=None, k_weight=None, *, norm=True, eps=1e-6, positions=None,
                 interleaved=False):
    """Each head vector of q [B, T, Hq, D] and k [B, T, Hkv, D] (fp32, bf16 or fp16, any strides) divided by its root
    mean square and multiplied by q_weight / k_weight [D] (None: 1; norm=False: neither), then its first R elements
    rotated by the angles whose cosines and sines are the rows of cos, sin [P, R/2] (fp32, rope_table): pairs
    (i, i + R/2), or (2i, 2i + 1) with interleaved=True. Returns q and k, contiguous. The tables take no gradient. A
    token's row is its index in the text, or positions [T] or [B, T] (int32 or int64); a position outside the table gives
    NaN (in the weights' gradients as a whole). Differentiable once in q, k and the weights, in reverse mode: a tensor with
    a forward-mode tangent raises."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must be [B, T, Hq, D] and [B, T, Hkv, D]")
    B, T, Hq, D = q.shape
    if not 2 <= D <= MAX_HEAD_DIM or Hq < 1 or k.shape[2] < 1:
        raise ValueError(f"the head dimension must be 2 to {MAX_HEAD_DIM} and there must be heads, got q "
                         f"{tuple(q.shape)} and k {tuple(k.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise ValueError(f"q and k must both be float32, bfloat16 or float16, got {q.dtype} and {k.dtype}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 \
            or not 2 <= 2 * cos.shape[1] <= D:
        raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be float32 [P, R/2] with R <= D={D}")
    if not norm and (q_weight is not None or k_weight is not None):
        raise ValueError("weights belong to the norm (norm=False was given)")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight must be given together")
    if norm and not float(eps) >= 0:
        raise ValueError(f"eps={eps} must not be negative")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (D,) or not w.is_floating_point()):
            raise ValueError(f"{name} must be floating-point [D={D}], got {tuple(w.shape)} {w.dtype}")
    if positions is None:
        if T > cos.shape[0]:
            raise ValueError(f"texts of {T} tokens need a table of as many rows, got {cos.shape[0]}")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.dim() not in (1, 2) or positions.shape[-1] != T or positions.dim() == 2 and \
                positions.shape[0] not in (1, B):
            raise ValueError(f"positions {tuple(positions.shape)} must be [T] or [B, T] with B={B}, T={T}")
    _check_same(q, ("k", k), ("cos", cos), ("sin", sin), ("q_weight", q_weight), ("k_weight", k_weight),
                ("positions", positions))
    _check_tangents(q, k, cos, sin, q_weight, k_weight)
    if positions is not None:
        positions = positions.expand(B, T)
    cos, sin = cos.detach().contiguous(), sin.detach().contiguous()
    if q_weight is not None:
        q_weight, k_weight = (w.to(torch.float32).contiguous() for w in (q_weight, k_weight))
    norm, eps, interleaved = int(bool(norm)), float(eps), int(bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QKNormRope.apply(q, k, cos, sin, positions, q_weight, k_weight, norm, eps, interleaved)
    qw, kw = (None, None) if q_weight is None else (q_weight.detach(), k_weight.detach())
    return _forward(q, k, cos, sin, positions, qw, kw, norm, eps, interleaved)[2:]

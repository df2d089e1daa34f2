"""CPU oracle for the attention operators (memarch_amd.attention, memarch_amd.rotary).

TEST INFRASTRUCTURE ONLY. Only tests/ may import this module, as the checker; the product path never calls it.

torch on the CPU in fp64, closed forms with dense scores:
    see_ij = j <= i and (window = 0 or i - j < window or j < sinks) and i < n
    P = softmax of scale q k^T over see; out = P v; rows that see nothing: 0
    d = go . out; dS = P (go v^T - d); dq = scale dS k; dk = scale dS^T q; dv = P^T go (summed over a group's heads)
and for the rotation the pairs (u, v) of x / sqrt(mean x^2 + eps) * w become (u cos - v sin, v cos + u sin).

`bounds` carries the roundings of a 16-bit implementation with fp32 sums through the same formulas, element by element;
every term is an upper bound:
    u        half a step of the element type (P, dS and the results are rounded to it once)
    e        relative error of an fp32 P: twice the error of its scores (D + 8 roundings of 2^-24 on sum |q||k| scale,
             exponent and row maximum alike) + 2^-20 for exp2, the logarithm and the division + 2^-24 per key summed
    range    2^-125 (1 + |go v| + |d|) per P or dS entry: an fp32 or bf16 value below 2^-126 may become 0 (the exponential
             of a score 88 below its row's maximum, and its product with go v - d)
    fp16     2^-25 per P or dS entry: half the spacing of its subnormals (P is at most 2^8 when rounded, and then divided by
             a denominator of at least 1; dS is rounded as it is)
Second-order terms are covered by a factor 1.05.

Pinning (tests/test_attention.py): torch autograd in fp64, central differences, hand-made masks, planted mistakes.
"""
import math

import torch


def visible(t, n, window, sinks):
    """[t, t] bool: whether row i sees column j in a sequence of n tokens."""
    i = torch.arange(t)[:, None]
    j = torch.arange(t)[None]
    see = (j <= i) & (i < n) & (j < n)
    if window:
        see &= (i - j < window) | (j < sinks)
    return see


def _heads(q, k):
    return q.shape[2] // k.shape[2]


def probs(q, k, window, sinks, lengths, scale):
    """P [B, Hq, T, T] of q [B, T, Hq, D], k [B, T, Hkv, D], and the scores' magnitude sum |q||k| scale."""
    b, t, hq, d = q.shape
    g = _heads(q, k)
    qd = q.double().transpose(1, 2)
    kd = k.double().transpose(1, 2).repeat_interleave(g, 1)
    see = torch.stack([visible(t, int(n), window, sinks) for n in lengths])[:, None]
    # what lies in masked rows must not matter, NaN among it
    live = (torch.arange(t)[None] < lengths[:, None])[:, None, :, None]
    qd, kd = (torch.where(live, x, torch.zeros((), dtype=x.dtype)) for x in (qd, kd))
    s = (qd @ kd.mT * scale).masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e300)
    p = (s - m).exp()
    z = p.sum(-1, keepdim=True)
    p = torch.where(z > 0, p / z.clamp(min=1e-300), torch.zeros_like(p))
    return p, (qd.abs() @ kd.abs().mT * scale), qd, kd, live


def attention(q, k, v, window=0, sinks=0, lengths=None, scale=None, go=None, dtype=None):
    """out, or (out, dq, dk, dv) with go; with dtype also their bounds, as a second tuple. Layouts as the operator's."""
    b, t, hq, d = q.shape
    g = _heads(q, k)
    hkv = k.shape[2]
    lengths = torch.full((b,), t) if lengths is None else lengths.long().clamp(0, t).cpu()
    scale = d ** -0.5 if scale is None else scale
    p, mag, qd, kd, live = probs(q, k, window, sinks, lengths, scale)
    vd = torch.where(live, v.double().transpose(1, 2).repeat_interleave(g, 1), torch.zeros((), dtype=torch.float64))
    out = p @ vd
    back = lambda x: x.transpose(1, 2).contiguous()
    fold = lambda x: back(x.reshape(b, hkv, g, t, d).sum(2))
    res = [back(out)]
    if go is not None:
        gd = torch.where(live, go.double().transpose(1, 2), torch.zeros((), dtype=torch.float64))
        dp = gd @ vd.mT
        delta = (gd * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        res += [back(scale * ds @ kd), fold(scale * ds.mT @ qd), fold(p.mT @ gd)]
    if dtype is None:
        return res[0] if go is None else tuple(res)
    u = torch.finfo(dtype).eps / 2
    sub = 2.0 ** -125 + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    e = 2 * (d + 8) * 2.0 ** -24 * mag.amax(-1, keepdim=True) + 2.0 ** -20 + t * 2.0 ** -24
    see = torch.stack([visible(t, int(n), window, sinks) for n in lengths])[:, None].double()
    a = p @ vd.abs()
    eo = (u + 2 * e) * a + sub * see @ vd.abs()      # before the result's rounding
    tol = [back(1.05 * (u * out.abs() + eo) + tiny)]
    if go is not None:
        edp = (d + 2) * 2.0 ** -24 * (gd.abs() @ vd.abs().mT)
        ed = (gd.abs() * (eo + (u * u + (d + 2) * 2.0 ** -24) * (out.abs() + eo))).sum(-1, keepdim=True)
        eds = (u + 2 * e) * ds.abs() + p * (edp + ed) + see * (sub + 2.0 ** -125 * (dp.abs() + delta.abs()))
        tol += [back(1.05 * (u * scale * (ds @ kd).abs() + scale * (eds + t * 2.0 ** -24 * ds.abs()) @ kd.abs()) + tiny),
                1.05 * (u * res[2].abs() + fold(scale * (eds + g * t * 2.0 ** -24 * ds.abs()).mT @ qd.abs())) + tiny,
                1.05 * (u * res[3].abs() + fold(((u + 2 * e + g * t * 2.0 ** -24) * p + sub * see).mT @ gd.abs())) + tiny]
    return tuple(res), tuple(tol)


def paged(q, k_cache, v_cache, table, lengths, window=0, sinks=0, scale=None, dtype=None):
    """out [B, Hq, D] of q [B, Hq, D] over the pages of the caches; with dtype also its bound."""
    b, hq, d = q.shape
    pages, page, hkv, _ = k_cache.shape
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), table.shape[1] * page)
        js = [j for j in range(n) if (not window or n - 1 - j < window or j < sinks)
              and 0 <= int(table[i, j // page]) < pages]
        if not js:
            continue
        pg = torch.tensor([int(table[i, j // page]) for j in js])
        sl = torch.tensor([j % page for j in js])
        k = k_cache[pg, sl].double().repeat_interleave(g, 1).transpose(0, 1)   # [hq, n, d]
        v = v_cache[pg, sl].double().repeat_interleave(g, 1).transpose(0, 1)
        qd = q[i].double()[:, None]
        s = (qd @ k.mT * scale)
        p = torch.softmax(s, -1)
        o = p @ v
        out[i] = o[:, 0]
        if dtype is not None:
            u = torch.finfo(dtype).eps / 2
            sub = 2.0 ** -125 + (2.0 ** -25 if dtype is torch.float16 else 0.0)
            e = 2 * (d + 8) * 2.0 ** -24 * (qd.abs() @ k.abs().mT * scale).amax(-1, keepdim=True) + 2.0 ** -20 \
                + len(js) * 2.0 ** -24
            tol[i] = (1.05 * (u * o.abs() + (u + 2 * e) * (p @ v.abs()) + sub * v.abs().sum(1, keepdim=True)))[:, 0] \
                + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return out if dtype is None else (out, tol)


def rope(x, cos, sin, w=None, norm=True, eps=1e-6, positions=None, interleaved=False):
    """The normed and rotated heads of x [B, T, H, D] in fp64 (differentiable: pass fp64 leaves)."""
    b, t = x.shape[:2]
    pos = torch.arange(t)[None].expand(b, t) if positions is None else positions.long().expand(b, t)
    rot = 2 * cos.shape[1]
    c, s = (t.double()[pos][:, :, None] for t in (cos, sin))
    y = x.double()
    if norm:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
        if w is not None:
            y = y * w.double()
    head = y[..., :rot]
    pair = head.unflatten(-1, (rot // 2, 2)) if interleaved else head.unflatten(-1, (2, rot // 2)).mT
    u, v = pair[..., 0], pair[..., 1]
    z = torch.stack((u * c - v * s, v * c + u * s), -1)
    z = z.flatten(-2) if interleaved else z.mT.flatten(-2)
    return torch.cat((z, y[..., rot:]), -1)

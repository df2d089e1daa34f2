"""CPU oracle for the 8-bit key/value cache (memarch_amd.kv_cache).

TEST INFRASTRUCTURE ONLY. Only tests/ may import this module, as the oracle; the product path never calls it.

torch on the CPU in fp64, one block after the other. Codes are kept as the e4m3 values that they stand for:
    nearest8(x)  to nearest, ties to even, 3 bits behind the leading one, steps of 2^-9 at least, up to 448
    scale        max(2^e, the block's old scale if it holds earlier tokens), 2^e >= 2^-100 the smallest with amax <= 448 2^e
Everything here is exact (values are fp32 numbers times powers of two), so results are compared bit for bit.
"""
import math

import torch


def nearest8(x):
    """x in fp64 rounded to e4m3 values."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def scale_for(amax):
    """The smallest power of two s >= 2^-100 with amax <= 448 s."""
    m, e = math.frexp(amax / 448)
    return 2.0 ** max(-100, e - 1 if m == 0.5 else e) if amax > 0 else 2.0 ** -100


def write(x, codes, scale, table, lengths, cu=None):
    """The codes [pages, page, h, d] and scales [pages, page / block, h] (fp64, new tensors) after x [n, h, d] was written."""
    codes, scale = codes.clone(), scale.clone()
    pages, page, heads, _ = codes.shape
    block = page // scale.shape[1]
    x = x.double()
    cu = list(range(len(lengths) + 1)) if cu is None else [min(max(int(c), 0), x.shape[0]) for c in cu]
    for b in range(len(lengths)):
        n = int(lengths[b])
        fresh = cu[b + 1] - cu[b]
        at = max(n - fresh, 0)
        while at < n:
            stop = min(n, at // block * block + block)
            rows = x[cu[b + 1] - (n - at):cu[b + 1] - (n - stop)]
            pi, slot = at // page, at % page
            pg = int(table[b, pi]) if pi < table.shape[1] else -1
            if 0 <= pg < pages:
                had, blk = slot % block, slot // block
                for h in range(heads):
                    r = rows[:, h]
                    s = scale_for(float(torch.where(r.isfinite(), r.abs(), torch.zeros_like(r)).max()))
                    if had:
                        old = float(scale[pg, blk, h])
                        s = max(s, old)
                        codes[pg, slot - had:slot, h] = nearest8(codes[pg, slot - had:slot, h] * (old / s))
                    q = nearest8(torch.where(r.isfinite(), r, torch.zeros_like(r)) / s)
                    codes[pg, slot:slot + stop - at, h] = torch.where(r.isfinite(), q, torch.full_like(q, math.nan))
                    scale[pg, blk, h] = s
            at = stop
    return codes, scale


def values(codes, scale):
    return codes * scale.repeat_interleave(codes.shape[1] // scale.shape[1], 1)[..., None]


def read(vals, table, cu, rows):
    """[rows, h, d] out of a cache's values."""
    pages, page, h, d = vals.shape
    out = torch.zeros(rows, h, d, dtype=torch.float64)
    cu = [min(max(int(c), 0), rows) for c in cu]
    for b in range(len(cu) - 1):
        for j in range(cu[b + 1] - cu[b]):
            pg = int(table[b, j // page]) if j // page < table.shape[1] else -1
            if 0 <= pg < pages:
                out[cu[b] + j] = vals[pg, j % page]
    return out


def attention(q, kc, ks, vc, vs, table, lengths, window=0, sinks=0, scale=None, dtype=None):
    """out [B, Hq, D]; with dtype also its bound, from the roundings of a 16-bit implementation with fp32 sums:
    u      half a step of the element type, for exp(score) scale_v as an operand and for the result
    e      relative error of an fp32 exp(score) scale_v and of the denominator's terms: the score's (D + 8 roundings of 2^-24
           on sum |q||k| scale), the sum of score and log2 scale_v in fp32 (2^-24 of both, times ln 2), each for the element
           and for the maximum, 2^-19 for exp2, logarithm, reciprocal and division, 2^-24 per key summed
    range  operands below the type's normal range: 2^-125 each, in fp16 2^-25, on codes whose scale may be smaller than that
           of the largest exp(score) scale_v, which is at least 1
    Second-order terms are covered by a factor 1.05."""
    b, hq, d = q.shape
    pages, page, hkv, _ = kc.shape
    g, per = hq // hkv, page // ks.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), table.shape[1] * page)
        j = torch.arange(n)
        pg = table[i].long()[j // page] if n else j
        ok = (pg >= 0) & (pg < pages)
        if window:
            ok &= (n - 1 - j < window) | (j < sinks)
        pg, sl = pg[ok], (j % page)[ok]
        if not len(pg):
            continue
        sk, sv = ks[pg, sl // per].double(), vs[pg, sl // per].double()
        k = (kc[pg, sl] * sk[..., None]).repeat_interleave(g, 1).transpose(0, 1)   # [hq, n, d]
        v = (vc[pg, sl] * sv[..., None]).repeat_interleave(g, 1).transpose(0, 1)
        qd = q[i].double()[:, None]
        p = torch.softmax(qd @ k.mT * scale, -1)
        o = p @ v
        out[i] = o[:, 0]
        if dtype is not None:
            u = torch.finfo(dtype).eps / 2
            sub = 2.0 ** -125 + (2.0 ** -25 if dtype is torch.float16 else 0.0)
            mag = (qd.abs() @ k.abs().mT * scale).amax(-1, keepdim=True)
            log = sv.log2().abs().amax().item()
            spread = (sv.amax(0) / sv.amin(0)).repeat_interleave(g)[:, None, None]
            e = 2 * ((d + 10) * 2.0 ** -24 * mag + 2.0 ** -24 * (mag + log)) + 2.0 ** -19 + len(pg) * 2.0 ** -24
            tol[i] = (1.05 * (u * o.abs() + (u + 2 * e) * (p @ v.abs()) + sub * spread * v.abs().sum(1, keepdim=True)))[:, 0] \
                + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return out if dtype is None else (out, tol)

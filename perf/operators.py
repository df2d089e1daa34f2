"""The attention operators' calls whose speed is measured: norms and rotation of queries and keys, attention over a
sliding window with first tokens that stay visible, and one new token's attention over a paged cache.

`listed()` gives the named cases, `draw(rng)` one more of the same ranges; `prepare` makes what a training or serving
program holds before the call, `run` is one pass (the framework's entry points where `own` is true, elementary torch
operations in fp32 otherwise), `exact` the same results in 64 bits, `work` the bytes and operations a pass needs.

Values: activations are N(0, 1) before the norms; queries and keys of the attention cases are RMS-normalised head
vectors with a gain of 1.5 (scores with a standard deviation of about 2) that share a direction per head, so that some
keys draw many queries; upstream gradients are N(0, 1).
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
_DEV = "cuda"
_EPS = 1e-6


def listed():
    return [
        # the queries and keys of one decoding step of 64 sequences: latency counts
        dict(name="rope_decode_64", op="rope", b=64, t=1, hq=16, hkv=2, d=128, rot=128, norm=True, interleaved=False,
             dtype="bf16", train=False, table=8192, packed=True),
        # a training step of 32 texts of 1024 tokens at d = 2048, norms with weights, whole heads rotated
        dict(name="rope_32x1024", op="rope", b=32, t=1024, hq=16, hkv=16, d=128, rot=128, norm=True,
             interleaved=False, dtype="bf16", train=True, table=1024, packed=True),
        # long texts of odd length in fp32 without norms: pairs side by side, half of each head rotated
        dict(name="rope_long_fp32", op="rope", b=3, t=16001, hq=12, hkv=4, d=64, rot=32, norm=False,
             interleaved=True, dtype="fp32", train=True, table=16384, packed=False),
        # a small model's step, as unit runs make it: launches and host time count
        dict(name="attn_tiny", op="attn", b=2, t=250, hq=4, hkv=4, d=64, window=64, sinks=4, ragged=False,
             dtype="bf16", train=True),
        # the training step of 32 texts of 1024 tokens at d = 2048
        dict(name="attn_32x1024", op="attn", b=32, t=1024, hq=16, hkv=16, d=128, window=512, sinks=4, ragged=False,
             dtype="bf16", train=True),
        # a padded batch of texts of different lengths in fp16, no window
        dict(name="attn_ragged_fp16", op="attn", b=8, t=2999, hq=12, hkv=12, d=64, window=0, sinks=0, ragged=True,
             dtype="fp16", train=True),
        # long texts with grouped heads
        dict(name="attn_4x16384", op="attn", b=4, t=16384, hq=16, hkv=4, d=128, window=1024, sinks=4, ragged=False,
             dtype="bf16", train=True),
        # a long prompt read once, every earlier token visible
        dict(name="attn_prompt_32k", op="attn", b=1, t=32768, hq=16, hkv=2, d=128, window=0, sinks=0, ragged=False,
             dtype="bf16", train=False),
        # one sequence's next token after a short text
        dict(name="paged_1x1000", op="paged", b=1, len=1000, hq=16, hkv=16, d=128, page=16, window=0, sinks=0,
             dtype="bf16"),
        # a batch of sequences of different lengths
        dict(name="paged_64x8192", op="paged", b=64, len=8192, hq=16, hkv=4, d=128, page=64, window=0, sinks=0,
             dtype="bf16"),
        # the same model with its window: few keys are read out of long caches
        dict(name="paged_window", op="paged", b=96, len=16384, hq=16, hkv=8, d=64, page=16, window=1024, sinks=4,
             dtype="fp16"),
        # a few very long sequences: work has to be split over the cache's length
        dict(name="paged_8x131072", op="paged", b=8, len=131072, hq=16, hkv=4, d=128, page=64, window=0, sinks=0,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "paged"])
    hkv = rng.choice([1, 2, 4, 8, 12, 16])
    hq = hkv * rng.choice([g for g in (1, 1, 2, 4, 8, 16) if hkv * g <= 16])
    if op == "rope":
        train = rng.random() < 0.7
        d = rng.choice([64, 128, 128, 80, 96])
        rot = rng.choice([d, d, d // 2, d // 4])
        t = _log(rng, 1, 16384) if train or rng.random() < 0.3 else 1
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        room = (1 << (26 if dtype == "fp32" else 27)) // ((hq + hkv) * d)   # tokens of the largest listed case
        t = min(t, room)
        b = _log(rng, 1, max(1, min(256, room // t)))
        return dict(op=op, b=b, t=t, hq=hq, hkv=hkv, d=d, rot=rot, norm=rng.random() < 0.7,
                    interleaved=rng.random() < 0.4, dtype=dtype, train=train,
                    table=_log(rng, t, 32768), packed=rng.random() < 0.5)
    d = rng.choice([64, 128, 128, 80, 96])
    if op == "attn":
        window = 0 if rng.random() < 0.3 else _log(rng, 16, 2048)
        t = _log(rng, 1, 16384 if window else 8192)
        # pairs and elements of the largest listed training case
        b = _log(rng, 1, max(1, min(64, (5 << 25) // (t * (hq + hkv) * d), (1 << 26) // _pairs(t, window, 0))))
        return dict(op=op, b=b, t=t, hq=hq, hkv=hkv, d=d, window=window, sinks=rng.choice([0, 1, 4, 16]) if window
                    else 0, ragged=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    train=rng.random() < 0.75)
    n = _log(rng, 1, 131072)
    b = _log(rng, 1, max(1, min(256, int(3 * (1 << 27) / (n * max(hkv, hq / 4) * d)))))
    window = 0 if rng.random() < 0.6 else _log(rng, 16, 4096)
    return dict(op=op, b=b, len=n, hq=hq, hkv=hkv, d=d, page=rng.choice([16, 16, 32, 64, 128]), window=window,
                sinks=rng.choice([0, 1, 4, 16]) if window else 0, dtype=rng.choice(["bf16", "bf16", "fp16"]))


# ------------------------------------------------------------------------------------------------------ inputs


def _heads(g, b, t, h, d, dt, gain=1.5):
    """RMS-normalised head vectors [b, t, h, d] with a gain, sharing a direction per head."""
    x = torch.randn(b, t, h, d, generator=g, device=_DEV)
    x += 0.3 * torch.randn(1, 1, h, d, generator=g, device=_DEV)
    x *= gain * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + _EPS)
    return x.to(dt)


def _lens(case, g):
    """Lengths of a batch's sequences: a third to the whole of the largest, one of them the largest."""
    n = case["len"] if case["op"] == "paged" else case["t"]
    x = (n * (1 / 3 + 2 / 3 * torch.rand(case["b"], generator=g, device=_DEV))).long().clamp_(1, n)
    x[0] = n
    return x.int()


def _table(case):
    """cos, sin [table, rot/2] fp32 of a rotation scaled by 4 for positions past 8192, as a model keeps them."""
    half = case["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=_DEV) / half)
    pos = torch.arange(case["table"], dtype=torch.float64, device=_DEV) / (4.0 if case["table"] > 8192 else 1.0)
    ang = pos[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    st = dict(case=case)
    if op == "rope":
        t = case["t"]
        if case["packed"]:   # slices of one projection's output
            x = torch.randn(b, t, hq + 2 * hkv, d, generator=g, device=_DEV).to(dt)
            st["q"], st["k"] = x[:, :, :hq], x[:, :, hq:hq + hkv]
        else:
            st["q"] = torch.randn(b, t, hq, d, generator=g, device=_DEV).to(dt)
            st["k"] = torch.randn(b, t, hkv, d, generator=g, device=_DEV).to(dt)
        st["cos"], st["sin"] = _table(case)
        # a decoding step's tokens stand anywhere in their sequences, a text's tokens at 0, 1, ...
        st["pos"] = torch.randint(0, case["table"], (b, 1), generator=g, device=_DEV) if t == 1 else None
        st["qw"] = st["kw"] = None
        if case["norm"]:
            st["qw"] = 1 + 0.2 * torch.randn(d, generator=g, device=_DEV)
            st["kw"] = 1 + 0.2 * torch.randn(d, generator=g, device=_DEV)
        if case["train"]:
            st["gq"] = torch.randn(b, t, hq, d, generator=g, device=_DEV).to(dt)
            st["gk"] = torch.randn(b, t, hkv, d, generator=g, device=_DEV).to(dt)
            for n in ("q", "k", "qw", "kw"):
                if st[n] is not None:
                    st[n] = st[n].detach().requires_grad_()
        return st
    if op == "attn":
        t = case["t"]
        st["q"] = _heads(g, b, t, hq, d, dt)
        st["k"] = _heads(g, b, t, hkv, d, dt)
        st["v"] = torch.randn(b, t, hkv, d, generator=g, device=_DEV).to(dt)
        st["lens"] = _lens(case, g) if case["ragged"] else None
        if case["train"]:
            st["go"] = torch.randn(b, t, hq, d, generator=g, device=_DEV).to(dt)
            for n in ("q", "k", "v"):
                st[n].requires_grad_()
        return st
    page = case["page"]
    lens = _lens(case, g)
    per = -(-case["len"] // page)
    pages = b * per
    st["kc"] = _heads(g, pages, page, hkv, d, dt)
    st["vc"] = torch.randn(pages, page, hkv, d, generator=g, device=_DEV).to(dt)
    st["q"] = _heads(g, b, 1, hq, d, dt)[:, 0]
    st["table"] = torch.randperm(pages, generator=g, device=_DEV).view(b, per).int()
    st["lens"] = lens
    st["host_lens"] = lens.tolist()   # for the plain form's loops
    return st


# ------------------------------------------------------------------------------------------- the framework's calls


def _own(st):
    from memarch_amd import attention, rotary
    case = st["case"]
    if case["op"] == "rope":
        q, k = rotary.qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], st["qw"], st["kw"], norm=case["norm"],
                                   eps=_EPS, positions=st["pos"], interleaved=case["interleaved"])
        if not case["train"]:
            return q, k
        leaves = [st[n] for n in ("q", "k", "qw", "kw") if st[n] is not None]
        return (q, k, *torch.autograd.grad((q, k), leaves, (st["gq"], st["gk"])))
    window = case["window"] or None
    if case["op"] == "attn":
        out = attention.window_attention(st["q"], st["k"], st["v"], window=window, sinks=case["sinks"],
                                         lengths=st["lens"])
        if not case["train"]:
            return (out,)
        return (out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["go"]))
    return (attention.paged_attention(st["q"], st["kc"], st["vc"], st["table"], st["lens"], window=window,
                                      sinks=case["sinks"]),)


# --------------------------------------------------------------------------------------------------- plain forms


def _turn(x, cos, sin, rot, interleaved):
    """The rotation of the first `rot` elements of each head vector by the angles of cos, sin [..., rot/2]."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_rope_one(x, w, cos, sin, go, case):
    dt = x.dtype
    x = x.detach().float()
    n = x
    if case["norm"]:
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        xn = x * r
        n = xn * w.detach()
    y = _turn(n, cos, sin, case["rot"], case["interleaved"]).to(dt)
    if go is None:
        return y, None, None
    dn = _turn(go.float(), cos, -sin, case["rot"], case["interleaved"])
    if not case["norm"]:
        return y, dn.to(dt), None
    dw = (dn * xn).double().sum((0, 1, 2)).float()
    dn = dn * w.detach()
    return y, (r * (dn - xn * (dn * xn).mean(-1, keepdim=True))).to(dt), dw


def _plain_rope(st):
    case = st["case"]
    t = case["t"]
    rows = st["pos"] if st["pos"] is not None else torch.arange(t, device=_DEV)[None]
    cos, sin = st["cos"][rows][:, :, None], st["sin"][rows][:, :, None]
    q, dq, dqw = _plain_rope_one(st["q"], st["qw"], cos, sin, st.get("gq"), case)
    k, dk, dkw = _plain_rope_one(st["k"], st["kw"], cos, sin, st.get("gk"), case)
    if not case["train"]:
        return q, k
    return (q, k, dq, dk, dqw, dkw) if case["norm"] else (q, k, dq, dk)


_ROWS = 1024   # query rows of one block of scores


def _plain_attn(st):
    """Block after block of query rows against the keys that any of them sees; the first tokens before the window
    are put in front of them."""
    case = st["case"]
    b, t, hq, hkv, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    window, sinks, train = case["window"] or t, case["sinks"], case["train"]
    dt, grp, scale = st["q"].dtype, hq // hkv, 1 / math.sqrt(d)
    q = st["q"].detach().float().transpose(1, 2).reshape(b, hkv, grp, t, d)
    k, v = (st[n].detach().float().transpose(1, 2)[:, :, None] for n in ("k", "v"))
    out = torch.zeros_like(q)
    if train:
        go = st["go"].float().transpose(1, 2).reshape(b, hkv, grp, t, d)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    pos = torch.arange(t, device=_DEV)
    lens = st["lens"] if st["lens"] is not None else torch.full((b,), t, device=_DEV)
    step = max(1, min(b, (1 << 28) // (_ROWS * hq * min(t, window + _ROWS + sinks))))
    for b0 in range(0, b, step):
        bs = slice(b0, b0 + step)
        for i0 in range(0, t, _ROWS):
            rows = slice(i0, min(t, i0 + _ROWS))
            lo = max(0, i0 - window + 1)
            cols = torch.cat((pos[:min(sinks, lo)], pos[lo:rows.stop]))
            first = min(sinks, lo)
            i, j = pos[rows, None], cols[None]
            see = (j <= i) & ((i - j < window) | (j < sinks))
            see = see & (i < lens[bs, None, None]) & (j < lens[bs, None, None])
            see = see[:, None, None]
            qb = q[bs, :, :, rows]
            kb = torch.cat((k[bs, :, :, :first], k[bs, :, :, lo:rows.stop]), 3)
            vb = torch.cat((v[bs, :, :, :first], v[bs, :, :, lo:rows.stop]), 3)
            s = torch.matmul(qb, kb.transpose(-1, -2).contiguous()) * scale
            s = s.masked_fill(~see, -math.inf)
            m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
            p = s.sub_(m).exp_()
            p = p / p.sum(-1, keepdim=True).clamp_(min=1e-30)
            ob = torch.matmul(p, vb)
            out[bs, :, :, rows] = ob
            if train:
                gb = go[bs, :, :, rows]
                dvb = torch.matmul(p.transpose(-1, -2).contiguous(), gb).sum(2, keepdim=True)
                ds = torch.matmul(gb, vb.transpose(-1, -2).contiguous())
                ds = p * (ds - (gb * ob).sum(-1, keepdim=True)) * scale
                dq[bs, :, :, rows] = torch.matmul(ds, kb)
                dkb = torch.matmul(ds.transpose(-1, -2).contiguous(), qb).sum(2, keepdim=True)
                for acc, part in ((dk, dkb), (dv, dvb)):
                    acc[bs, :, :, :first] += part[:, :, :, :first]
                    acc[bs, :, :, lo:rows.stop] += part[:, :, :, first:]

    def back(x):
        return x.reshape(b, -1, t, d).transpose(1, 2).to(dt).contiguous()
    return (back(out), back(dq), back(dk), back(dv)) if train else (back(out),)


def _seen(n, window, sinks):
    """The positions that the last token of a sequence of n tokens sees."""
    lo = max(0, n - window) if window else 0
    return torch.cat((torch.arange(min(sinks, lo), device=_DEV), torch.arange(lo, n, device=_DEV)))


def _plain_paged(st):
    case = st["case"]
    grp, d, page = case["hq"] // case["hkv"], case["d"], case["page"]
    out = torch.zeros_like(st["q"])
    for i, n in enumerate(st["host_lens"]):
        j = _seen(n, case["window"], case["sinks"])
        blk = st["table"][i, j // page].long()
        k, v = st["kc"][blk, j % page].float(), st["vc"][blk, j % page].float()
        q = st["q"][i].float().view(-1, grp, d) / math.sqrt(d)
        s = torch.matmul(q, k.permute(1, 2, 0).contiguous())
        p = (s - s.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
        out[i] = torch.matmul(p, v.transpose(0, 1).contiguous()).reshape(-1, d).to(out.dtype)
    return (out,)


_PLAIN = {"rope": _plain_rope, "attn": _plain_attn, "paged": _plain_paged}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------ 64 bits


def _exact_rope(case, st):
    """Each pair as a complex number times e^(i angle); gradients by autograd."""
    pos = st["pos"] if st["pos"] is not None else torch.arange(case["t"], device=_DEV)[None]
    turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, :, None]
    rot, outs, leaves, gos = case["rot"], [], [], []
    for n, w in (("q", "qw"), ("k", "kw")):
        x = st[n].detach().double().requires_grad_(case["train"])
        leaves.append(x)
        y = x
        if case["norm"]:
            wt = st[w].detach().double().requires_grad_(case["train"])
            leaves.append(wt)
            y = x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * wt
        head = y[..., :rot]
        pair = head.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, rot // 2)).mT
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.mT.flatten(-2)
        outs.append(torch.cat((z, y[..., rot:]), -1))
        gos.append(st.get("g" + n))
    if not case["train"]:
        return tuple(outs)
    grads = torch.autograd.grad(outs, leaves, [g.double() for g in gos])
    order = (0, 2, 1, 3) if case["norm"] else (0, 1)
    return tuple(o.detach() for o in outs) + tuple(grads[i] for i in order)


def _exact_attn(case, st):
    """One sequence and one group of query heads at a time, dense scores of a band of rows, gradients by autograd."""
    b, t, hq, hkv, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    grp = hq // hkv
    lens = st["lens"].tolist() if st["lens"] is not None else [t] * b
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device=_DEV)
    grads = [torch.zeros(b, t, h, d, dtype=torch.float64, device=_DEV) for h in (hq, hkv, hkv)]
    for i in range(b):
        n = lens[i]
        band = max(1, min(n, (1 << 27) // n))
        for h in range(hq):
            for r0 in range(0, n, band):
                r1 = min(n, r0 + band)
                q = st["q"][i, r0:r1, h].detach().double().requires_grad_(case["train"])
                k = st["k"][i, :r1, h // grp].detach().double().requires_grad_(case["train"])
                v = st["v"][i, :r1, h // grp].detach().double().requires_grad_(case["train"])
                dist = torch.arange(r0, r1, device=_DEV)[:, None] - torch.arange(r1, device=_DEV)[None]
                hide = dist < 0
                if case["window"]:
                    far = dist >= case["window"]
                    far[:, :case["sinks"]] = False
                    hide = hide | far
                s = (q @ k.T / d ** 0.5).masked_fill(hide, float("-inf"))
                o = torch.softmax(s, -1) @ v
                out[i, r0:r1, h] = o.detach()
                if case["train"]:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), st["go"][i, r0:r1, h].double())
                    grads[0][i, r0:r1, h] = dq
                    grads[1][i, :r1, h // grp] += dk
                    grads[2][i, :r1, h // grp] += dv
    return (out, *grads) if case["train"] else (out,)


def _exact_paged(case, st):
    """The cache of one sequence laid out in order, one head after the other."""
    grp = case["hq"] // case["hkv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEV)
    for i, n in enumerate(st["host_lens"]):
        blocks = st["table"][i].long()
        k = st["kc"][blocks].flatten(0, 1)[:n]
        v = st["vc"][blocks].flatten(0, 1)[:n]
        back = n - 1 - torch.arange(n, device=_DEV)
        for h in range(case["hq"]):
            s = k[:, h // grp].double() @ st["q"][i, h].double() / case["d"] ** 0.5
            if case["window"]:
                hide = back >= case["window"]
                hide[:case["sinks"]] = False
                s[hide] = float("-inf")
            out[i, h] = torch.softmax(s, 0) @ v[:, h // grp].double()
    return (out,)


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "paged": _exact_paged}[case["op"]](case, st)


# --------------------------------------------------------------------------------------------------------- work


def _pairs(n, window, sinks):
    """Visible (query, key) pairs of a sequence of n tokens."""
    if not window or window >= n:
        return n * (n + 1) // 2
    pairs = window * (window + 1) // 2 + (n - window) * window
    return pairs + sum(max(0, min(n, n - window - j)) for j in range(sinks))


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    if case["op"] == "rope":
        n = b * case["t"] * (hq + hkv) * d
        table = min(case["table"], b if case["t"] == 1 else case["t"]) * case["rot"] * 4
        return {"bytes": n * e * (5 if case["train"] else 2) + table, "flops": n * (20 if case["train"] else 6)}
    if case["op"] == "attn":
        t = case["t"]
        share = 2 / 3 if case["ragged"] and b > 1 else 1.0   # mean length, and of pairs about 13/27
        pairs = b * _pairs(t, case["window"], case["sinks"]) * (13 / 27 if share < 1 and not case["window"] else share)
        io = b * t * d * e * ((4 * hq + 4 * hkv) if case["train"] else (2 * hq + 2 * hkv))
        return {"bytes": int(io * share), "flops": int(pairs * hq * d * (14 if case["train"] else 4))}
    n = case["len"] * (2 / 3 if b > 1 else 1)
    keys = min(n, case["window"] + case["sinks"]) if case["window"] else n
    return {"bytes": int(b * (2 * keys * hkv * d * e + 2 * hq * d * e)), "flops": int(b * keys * hq * d * 4)}

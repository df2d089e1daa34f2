"""GPU parity of qk_norm_rope against the fp64 oracle and its autograd.

Bars, element by element. Forward: u |y| (the result's rounding, u half a step of its type) plus 2^-20 (|n_a| + |n_b|):
fewer than 16 fp32 roundings on the two normed values of a pair. Backward: u |dx| + 2^-19 r (S + |x| r mean(S |x| r)),
S = |g_a w| + |g_b w| of the pair: the same terms in absolute value. dw: (n / 2^24 + 2^-19) of the sum of absolute terms,
n the terms summed."""
import pytest
import torch

from oracle import attn_oracle as orc

pytestmark = pytest.mark.gpu

DTS = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _pair_sum(x, rot, il):
    """|x_a| + |x_b| on both elements of each pair."""
    a = x.abs()
    head = a[..., :rot]
    if il:
        s = head.unflatten(-1, (rot // 2, 2)).sum(-1, keepdim=True).expand(*head.shape[:-1], rot // 2, 2).flatten(-2)
    else:
        s = head.unflatten(-1, (2, rot // 2)).sum(-2, keepdim=True).expand(*head.shape[:-1], 2, rot // 2).flatten(-2)
    return torch.cat((s, a[..., rot:]), -1)


def _check(q, k, cos, sin, qw, kw, gq, gk, norm=True, eps=1e-6, positions=None, il=False, dev=None):
    from memarch_amd.rotary import qk_norm_rope
    dt, rot = q.dtype, 2 * cos.shape[1]
    u = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    leaves = [None if t is None else t.detach().cuda().requires_grad_() for t in (q, k, qw, kw)]
    qg, kg = leaves[:2] if dev is None else [d.detach().requires_grad_() for d in dev]
    leaves[:2] = qg, kg
    yq, yk = qk_norm_rope(qg, kg, cos.cuda(), sin.cuda(), leaves[2], leaves[3], norm=norm, eps=eps,
                          positions=None if positions is None else positions.cuda(), interleaved=il)
    grads = torch.autograd.grad((yq, yk), [t for t in leaves if t is not None], (gq.cuda(), gk.cuda()))
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == yk.dtype == dt
    for i, (x, w, g, y) in enumerate(((q, qw, gq, yq), (k, kw, gk, yk))):
        xd = x.double().requires_grad_()
        wd = None if w is None else w.double().requires_grad_()
        ref = orc.rope(xd, cos, sin, wd, norm, eps, positions, il)
        n = xd.detach()
        r = torch.ones_like(n[..., :1])
        if norm:
            r = (n.square().mean(-1, keepdim=True) + eps).rsqrt()
            n = n * r * (1.0 if w is None else w.double())
        tol = u * ref.detach().abs() + 2.0 ** -20 * _pair_sum(n, rot, il) + tiny
        assert ((y.detach().double().cpu() - ref.detach()).abs() <= tol).all(), ("y", i)
        want = torch.autograd.grad(ref, [t for t in (xd, wd) if t is not None], g.double())
        s = _pair_sum(g.double(), rot, il)
        xr = xd.detach().abs() * r
        sw = s * (1.0 if w is None else w.double().abs())
        mag = r * (sw + xr * (sw * xr).mean(-1, keepdim=True)) if norm else s
        got = grads[i].double().cpu()
        assert grads[i].dtype == dt and ((got - want[0]).abs() <= u * want[0].abs() + 2.0 ** -19 * mag + tiny).all(), ("dx", i)
        if w is not None:
            terms = x.shape[0] * x.shape[1] * x.shape[2]
            bar = (terms * 2.0 ** -24 + 2.0 ** -19) * (s * xr).sum((0, 1, 2))
            assert ((grads[2 + i].double().cpu() - want[1]).abs() <= bar + u * want[1].abs()).all(), ("dw", i)
    return (yq.detach(), yk.detach(), *grads)


def _inputs(b, t, hq, hkv, d, rot, dt, seed=0, weights=True, rows=None):
    from memarch_amd.rotary import rope_table
    g = torch.Generator().manual_seed(seed)
    mk = lambda h: torch.randn(b, t, h, d, generator=g).to(dt)
    w = [1 + 0.3 * torch.randn(d, generator=g) if weights else None for _ in range(2)]
    return (mk(hq), mk(hkv), *rope_table(rows or t, rot), *w, mk(hq), mk(hkv))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("il", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("b,t,hq,hkv,d,rot", [
    (1, 1, 1, 1, 64, 64), (2, 7, 4, 2, 128, 128), (3, 5, 3, 1, 128, 64), (1, 9, 6, 2, 96, 96), (2, 3, 5, 5, 80, 80),
    (1, 4, 2, 1, 80, 16), (2, 2, 2, 2, 256, 256), (1, 3, 1, 2, 256, 16), (1, 5, 2, 1, 8, 8), (1, 6, 2, 1, 6, 4), (2, 3, 3, 2, 33, 10),
    (1, 2, 1, 1, 2, 2), (1, 130, 9, 3, 40, 20), (1, 3, 2, 2, 24, 16)])
def test_parity(dt, il, b, t, hq, hkv, d, rot):
    print(f"rope {b} {t} {hq} {hkv} {d} {rot} {dt} {il}", flush=True)
    x = _inputs(b, t, hq, hkv, d, rot, DTS[dt], seed=d + t)
    _check(*x, il=il)
    _check(x[0], x[1], x[2], x[3], None, None, x[6], x[7], il=il)               # norms without weights
    _check(x[0], x[1], x[2], x[3], None, None, x[6], x[7], norm=False, il=il)   # the rotation alone


def test_many_tokens():
    """More tokens than the backward's workgroups take in one round: parts of the weights' gradients over many units."""
    _check(*_inputs(3, 1500, 6, 2, 64, 32, torch.bfloat16, seed=3))
    _check(*_inputs(2, 900, 3, 1, 33, 32, torch.float32, seed=4))


@pytest.mark.parametrize("pdt", [torch.int32, torch.int64])
def test_positions(pdt):
    x = _inputs(3, 6, 4, 2, 64, 64, torch.bfloat16, seed=5, rows=5000)
    g = torch.Generator().manual_seed(2)
    pos = torch.randint(0, 5000, (3, 6), generator=g).to(pdt)
    pos[0, 0], pos[2, 5] = 4999, 0
    _check(*x, positions=pos)
    _check(*x, positions=pos[0])          # one row of positions for all sequences
    _check(*x, positions=pos[:1])
    _check(*x, positions=pos.T.contiguous().T)


def test_positions_outside_the_table_give_nan():
    from memarch_amd.rotary import qk_norm_rope
    for d, rot in ((64, 64), (66, 10)):
        q, k, cos, sin, qw, kw, gq, gk = (t.cuda() for t in _inputs(1, 4, 2, 1, d, rot, torch.float32, rows=9))
        pos = torch.tensor([[3, 9, -1, 8]], device="cuda")
        ql = q.clone().requires_grad_()
        yq, yk = qk_norm_rope(ql, k, cos, sin, qw, kw, positions=pos)
        good = qk_norm_rope(q, k, cos, sin, qw, kw, positions=pos.clamp(0, 8))
        for y, r in ((yq.detach(), good[0]), (yk, good[1])):
            assert torch.equal(y[:, [0, 3]], r[:, [0, 3]]) and y[:, [1, 2]].isnan().all()
        (dq,) = torch.autograd.grad(yq, ql, gq)
        assert torch.isfinite(dq[:, [0, 3]]).all() and dq[:, [1, 2]].isnan().all()


@pytest.mark.parametrize("il", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 32), (66, 10)])
def test_positions_outside_the_table_give_nan_weight_gradients(d, rot, il):
    """One such token, and no column of the weights' gradients passes for a finite one; the other tokens' are as ever."""
    from memarch_amd.rotary import qk_norm_rope
    q, k, cos, sin, qw, kw, gq, gk = (t.cuda() for t in _inputs(1, 40, 2, 1, d, rot, torch.float32, rows=40))
    pos = torch.arange(40, device="cuda")
    pos[17] = 40
    ls = [t.requires_grad_() for t in (q, k, qw, kw)]
    grads = torch.autograd.grad(qk_norm_rope(q, k, cos, sin, qw, kw, positions=pos, interleaved=il), ls, (gq, gk))
    assert grads[2].isnan().all() and grads[3].isnan().all()
    good = torch.autograd.grad(qk_norm_rope(q, k, cos, sin, qw, kw, interleaved=il), ls, (gq, gk))
    rest = pos < 40
    assert all(torch.equal(a[:, rest], b[:, rest]) for a, b in zip(grads[:2], good[:2]))


def test_strided_operands():
    """Slices of one packed projection, head-first layouts, strided last dimensions, unaligned bases, broadcast heads and
    expanded upstream gradients."""
    from memarch_amd.rotary import qk_norm_rope
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 9, 8, 64, generator=g).bfloat16()
    q, k = x[:, :, :4], x[:, :, 4:6]
    _, _, cos, sin, qw, kw, gq, gk = _inputs(2, 9, 4, 2, 64, 64, torch.bfloat16, seed=1)
    run = lambda a, b, ga=gq, gb=gk: _check(q, k, cos, sin, qw, kw, ga, gb, dev=(a, b))
    xg = x.cuda()
    base = run(xg[:, :, :4], xg[:, :, 4:6])
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, base))
    heads = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    assert same(run(heads(xg[:, :, :4]), heads(xg[:, :, 4:6])))
    last = lambda t: torch.stack((t, t), -1)[..., 0]
    assert same(run(last(xg[:, :, :4]), last(xg[:, :, 4:6])))
    assert same(run(xg[:, :, :4], xg[:, :, 4:6], heads(gq), last(gk)))
    buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(xg)
    run(buf[:, :, :4], buf[:, :, 4:6])                      # element by element: other sums, the same bars
    one = x[:, :, :1].expand(2, 9, 4, 64)
    _check(one, k, cos, sin, qw, kw, gq[:1, :1, :1, :1].expand_as(gq), gk, dev=(xg[:, :, :1].expand(2, 9, 4, 64), xg[:, :, 4:6]))
    # weights of another type: gradients come back in it
    wl = [w.cuda().bfloat16().requires_grad_() for w in (qw, kw)]
    yq, yk = qk_norm_rope(xg[:, :, :4], xg[:, :, 4:6], cos.cuda(), sin.cuda(), *wl)
    grads = torch.autograd.grad((yq, yk), wl, (gq.cuda(), gk.cuda()))
    assert all(t.dtype == torch.bfloat16 for t in grads)


def test_zero_heads_and_eps():
    """A head of zeros with eps gives zeros and finite gradients."""
    q, k, cos, sin, qw, kw, gq, gk = _inputs(1, 4, 2, 1, 64, 64, torch.float32, seed=2)
    q[:, 1], k[:, 2] = 0, 0
    got = _check(q, k, cos, sin, qw, kw, gq, gk, eps=1e-5)
    assert all(torch.isfinite(t).all() for t in got) and not got[0][:, 1].any()


def test_empty_and_one_output():
    from memarch_amd.rotary import qk_norm_rope, rope_table
    cos, sin = rope_table(4, 64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    for shape in ((0, 3), (2, 0)):
        q = torch.zeros(*shape, 2, 64, device="cuda", requires_grad=True)
        yq, yk = qk_norm_rope(q, q[:, :, :1], cos, sin, w, w)
        gq, gw = torch.autograd.grad(yq.sum() + yk.sum(), (q, w))
        assert gq.shape == q.shape and not gw.any()
    q, k, *_ = (t.cuda() for t in _inputs(1, 4, 2, 1, 64, 64, torch.float32)[:2])
    ql = q.clone().requires_grad_()
    yq, _ = qk_norm_rope(ql, k, cos, sin)       # only the queries are used further
    (dq,) = torch.autograd.grad(yq.sum(), ql)
    assert torch.isfinite(dq).all()
    kl = k.clone().requires_grad_()
    _, yk = qk_norm_rope(q, kl, cos, sin, norm=False)
    (dk,) = torch.autograd.grad(yk.sum(), kl)
    assert torch.isfinite(dk).all()


def test_graph_sync_and_repeats():
    from memarch_amd.rotary import qk_norm_rope
    vals = [[t.cuda() for t in _inputs(2, 300, 4, 2, 128, 128, torch.bfloat16, seed=i)] for i in range(3)]

    def step(q, k, cos, sin, qw, kw, gq, gk):
        ls = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
        y = qk_norm_rope(ls[0], ls[1], cos, sin, ls[2], ls[3])
        return (*(t.detach() for t in y), *torch.autograd.grad(y, ls, (gq, gk)))

    x = [t.clone() for t in vals[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        step(*x)
    finally:
        torch.cuda.set_sync_debug_mode(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*x)
    for i in (1, 2, 0):
        for a, b in zip(x, vals[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        ref, again = step(*vals[i]), step(*vals[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(b, c) for a, b, c in zip(got, ref, again)), i


def test_more_heads_than_one_launch_has_waves():
    """2^26 head vectors element by element: one wave each would be more threads than a launch can hold. Each part of the
    text alone gives the same bits."""
    from memarch_amd.rotary import qk_norm_rope, rope_table
    t, hq, parts = 1 << 22, 16, 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k = (torch.randn(1, t, h, 2, generator=gen, device="cuda").bfloat16() for h in (hq, 1))
    cos, sin = rope_table(1000, 2, device="cuda")
    pos = torch.arange(t, device="cuda") % 1000
    got = qk_norm_rope(q, k, cos, sin, positions=pos)
    for i in range(parts):
        s = slice(i * t // parts, (i + 1) * t // parts)
        for a, b in zip(got, qk_norm_rope(q[:, s], k[:, s], cos, sin, positions=pos[s])):
            assert torch.equal(a[:, s], b), i

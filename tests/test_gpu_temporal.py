"""
Temporal operators (srvp_amd.temporal) against their definitions in 64 bits.

Tolerances count roundings: a rounding to type t is off by at most eps_t / 2 relative to the value it rounds (bf16 2^-8, fp32 2^-24).  For sums the bound
is that of the sum of the terms' magnitudes, which the references below return beside the value ("size").
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, FP = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -24}


def rnd(g, *s, dtype=FP, scale=1.0):
    return (scale * torch.randn(*s, generator=g)).to(dtype).to(DEV)


def scan(a, b, c, ld, scale, rev, carry=None, off=0, lengths=None):
    """out_i = scale * sum over j before and at i (after, if rev) of decay^|i-j| (a_i . b_j) c_j + decay^(distance + off) a_i carry, token pairs in 64 bits;
    returns (out, size) with size the same sum over the magnitudes of all products."""
    T, B, H, _ = a.shape
    out = torch.zeros(T, B, H, c.shape[3], dtype=torch.float64, device=a.device)
    size = torch.zeros_like(out)
    for s in range(B):
        n = T if lengths is None else min(max(int(lengths[s]), 0), T)
        i = torch.arange(n, dtype=torch.float64, device=a.device)
        gap = (i[None] - i[:, None]) if rev else (i[:, None] - i[None])
        for h in range(H):
            l = ld[h].double()
            w = torch.where(gap >= 0, torch.where(gap == 0, torch.ones_like(gap), torch.exp(l * gap.clamp(min=1))), torch.zeros_like(gap))
            A, Bm, Cm = (x[:n, s, h].double() for x in (a, b, c))
            out[:n, s, h] = scale * ((A @ Bm.t()) * w) @ Cm
            size[:n, s, h] = abs(scale) * ((A.abs() @ Bm.abs().t()) * w) @ Cm.abs()
            if carry is not None:
                d = (n - 1 - i if rev else i) + off
                p = torch.where(d == 0, torch.ones_like(d), torch.exp(l * d.clamp(min=1)))[:, None]
                out[:n, s, h] += (p * A) @ carry[s, h].double()
                size[:n, s, h] += (p * A.abs()) @ carry[s, h].double().abs()
    return out, size


def state_sum(k, v, ld, lengths, s0, scale=1.0, from_end=True, off=0):
    """sum_j decay^(n-1-j or j, + off) k_j v_j^T * scale + decay^n s0, and its size."""
    T, B, H, Dk = k.shape
    out = torch.zeros(B, H, Dk, v.shape[3], dtype=torch.float64, device=k.device)
    size = torch.zeros_like(out)
    for s in range(B):
        n = T if lengths is None else min(max(int(lengths[s]), 0), T)
        i = torch.arange(n, dtype=torch.float64, device=k.device)
        d = (n - 1 - i if from_end else i) + off
        for h in range(H):
            l = ld[h].double()
            p = torch.where(d == 0, torch.ones_like(d), torch.exp(l * d.clamp(min=1)))[:, None]
            K, V = k[:n, s, h].double(), v[:n, s, h].double()
            out[s, h] = scale * (p * K).t() @ V
            size[s, h] = abs(scale) * (p * K.abs()).t() @ V.abs()
            if s0 is not None:
                keep = torch.exp(l * n) if n else 1.0
                out[s, h] += keep * s0[s, h].double()
                size[s, h] += keep * s0[s, h].double().abs()
    return out, size


def within(got, ref, size, dtype, inner, what):
    """got (type dtype) is within one rounding of ref plus `inner` relative to size."""
    tol = HALF[dtype] * ref.abs() + inner * size * (1 + HALF[dtype]) + 1e-30
    bad = (got.double() - ref).abs() / tol
    assert torch.isfinite(got.float()).all(), what
    assert got.dtype == dtype and bad.max().item() <= 1.0, (what, bad.max().item())


def inner_of(dtype, T, D):
    """fp32 sums of D products and of T terms, decays formed by an exponential of 2 ulp and multiplied up (a few roundings a chunk); bf16: the score or the
    state, whichever a term passes through, is rounded once."""
    n = D + min(T, 4096) + 64
    return n * 2.0 ** -24 + (2.0 ** -8 if dtype is BF else 0.0)


ATTN = [
    # T, B, H, Dk, Dv, dtype, state, lengths
    (12, 3, 4, 64, 64, FP, False, None), (1, 1, 1, 1, 1, FP, True, None), (1, 2, 3, 64, 64, BF, True, None), (7, 2, 2, 33, 17, FP, True, [7, 0]),
    (33, 3, 2, 40, 72, BF, True, [33, 1, 32]), (64, 2, 2, 128, 128, BF, False, None), (65, 2, 2, 128, 64, BF, True, [65, 64]),
    (129, 2, 3, 64, 128, FP, True, [100, 129]), (300, 1, 2, 128, 128, BF, True, None), (300, 1, 2, 128, 128, FP, True, None),
    (1000, 2, 1, 96, 80, BF, True, [999, 513]), (1000, 2, 1, 17, 250, FP, True, [0, 1000]), (515, 1, 2, 256, 256, BF, True, None),
    (515, 1, 1, 200, 256, FP, False, None), (2500, 1, 1, 128, 16, BF, False, None), (90, 40, 8, 32, 32, BF, True, list(range(40))),
    (40, 130, 2, 64, 8, FP, False, list(range(0, 130))),
]


def decays(H, kind=0):
    if kind == 1:
        return torch.tensor([float('-inf'), 0.0, -1e-3, -30.0][:H] + [-0.1] * max(0, H - 4), device=DEV)
    return torch.log1p(-torch.logspace(-0.9, -2.7, H, dtype=torch.float64)).float().to(DEV)


@pytest.mark.parametrize('case', range(len(ATTN)))
def test_linear_attention_forward_backward(case):
    from srvp_amd import temporal as t
    T, B, H, Dk, Dv, dt, has_state, lengths = ATTN[case]
    g = torch.Generator().manual_seed(100 + case)
    q, k, v, do = rnd(g, T, B, H, Dk, dtype=dt), rnd(g, T, B, H, Dk, dtype=dt), rnd(g, T, B, H, Dv, dtype=dt), rnd(g, T, B, H, Dv, dtype=dt)
    s0 = rnd(g, B, H, Dk, Dv) if has_state else None
    dn = rnd(g, B, H, Dk, Dv)
    n = None if lengths is None else torch.tensor(lengths, device=DEV)
    if n is not None:
        for b, m in enumerate(lengths):              # what lies behind a sequence is not read
            for x in (q, k, v, do):
                x[m:, b] = float('nan')
    ld = decays(H, kind=case % 2)
    sc = Dk ** -0.5
    leaves = [x.clone().requires_grad_() for x in (q, k, v)] + ([s0.clone().requires_grad_()] if has_state else [])
    o, new = t.linear_attention(*leaves[:3], ld, state=leaves[3] if has_state else None, lengths=n, return_state=True)
    clean = lambda x: torch.nan_to_num(x) if n is not None else x
    qc, kc, vc, gc = clean(q), clean(k), clean(v), clean(do)
    inn = inner_of(dt, T, max(Dk, Dv))
    ref, size = scan(qc, kc, vc, ld, sc, False, None if s0 is None else sc * s0, off=1, lengths=lengths)
    within(o.detach(), ref, size, dt, inn, 'o')
    sref, ssize = state_sum(kc, vc, ld, lengths, s0)
    within(new.detach(), sref, ssize, FP, inner_of(FP, T, 0), 'state')
    plain = t.linear_attention(q, k, v, ld, state=s0, lengths=n)
    assert torch.equal(plain, o.detach())
    grads = torch.autograd.grad([o, new], leaves, [do, dn])
    r, z = scan(gc, vc, kc, ld, sc, False, None if s0 is None else sc * s0.transpose(2, 3), off=1, lengths=lengths)
    within(grads[0], r, z, dt, inn, 'dq')
    r, z = scan(vc, gc, qc, ld, sc, True, dn.transpose(2, 3), lengths=lengths)
    within(grads[1], r, z, dt, inn, 'dk')
    r, z = scan(kc, qc, gc, ld, sc, True, dn, lengths=lengths)
    within(grads[2], r, z, dt, inn, 'dv')
    if has_state:
        r, z = state_sum(qc, gc, ld, lengths, dn, scale=sc, from_end=False, off=1)
        within(grads[3], r, z, FP, inner_of(FP, T, 0) * 2, 'dstate')
    again = t.linear_attention_backward(do, q, k, v, ld, state=s0, lengths=n, d_state=dn)
    for a, b in zip(again, grads):
        assert torch.equal(a, b)


def test_linear_attention_gradients_against_differences():
    """<o, do> is linear in q, in k, in v and in the state: central differences are exact, whatever the step."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(4)
    T, B, H, Dk, Dv = 70, 2, 2, 24, 40
    ins = [rnd(g, T, B, H, Dk), rnd(g, T, B, H, Dk), rnd(g, T, B, H, Dv), rnd(g, B, H, Dk, Dv)]
    do, ld = rnd(g, T, B, H, Dv), decays(H)
    f = lambda x: t.linear_attention(x[0], x[1], x[2], ld, state=x[3]).double()
    grads = t.linear_attention_backward(do, *ins[:3], ld, state=ins[3])
    for i in range(4):
        d = rnd(g, *ins[i].shape)
        hi, lo = list(ins), list(ins)
        hi[i], lo[i] = ins[i] + d, ins[i] - d
        oh, ol = f(hi), f(lo)
        diff = ((oh - ol) * do.double()).sum().item() / 2
        dot = (grads[i].double() * d.double()).sum().item()
        # both sides: outputs of fp32 sums over up to T + Dk terms, off by 2^-24 times that many of their own size at most
        size = ((oh.abs() + ol.abs()) * do.double().abs()).sum().item() / 2 + (grads[i].double() * d.double()).abs().sum().item()
        assert abs(diff - dot) <= 2.0 ** -24 * (T + Dk + 64) * size, (i, diff, dot)


@pytest.mark.parametrize('dt', [FP, BF])
def test_linear_attention_layouts(dt):
    """Batch-major views, shared (expanded) heads, sliced features at odd offsets: the same results as the packed copy."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(8)
    T, B, H, D = 75, 3, 4, 48
    ld = decays(H)
    q = rnd(g, B, T, H, D, dtype=dt).transpose(0, 1)
    k = rnd(g, T, B, 1, D, dtype=dt).expand(T, B, H, D)
    wide = rnd(g, T, B, H, D + 3, dtype=dt)
    v = wide[..., 3:]
    copy = t.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), ld)
    assert torch.equal(t.linear_attention(q, k, v, ld), copy)
    # the gradient of a shared head is the sum over its copies
    k1 = rnd(g, T, B, 1, D, dtype=dt).requires_grad_()
    do = rnd(g, T, B, H, D, dtype=dt)
    (dk,) = torch.autograd.grad(t.linear_attention(q, k1.expand(T, B, H, D), v, ld), k1, do)
    full = t.linear_attention_backward(do, q, k1.detach().expand(T, B, H, D), v, ld)[1]
    assert torch.equal(dk, full.sum(2, keepdim=True))
    # features not contiguous: copied
    vt = rnd(g, T, B, D, H, dtype=dt).transpose(2, 3)
    assert torch.equal(t.linear_attention(q, k, vt, ld), t.linear_attention(q, k, vt.contiguous(), ld))


def test_linear_attention_pieces_and_steps_continue_each_other():
    """A prompt in one call, in two calls with the state handed on, and token by token through the recurrent form: the same within their roundings."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(11)
    T, B, H, Dk, Dv = 130, 3, 4, 64, 32
    q, k, v = rnd(g, T, B, H, Dk), rnd(g, T, B, H, Dk), rnd(g, T, B, H, Dv)
    ld = decays(H)
    o, s = t.linear_attention(q, k, v, ld, return_state=True)
    ref, size = scan(q, k, v, ld, Dk ** -0.5, False)
    sref, ssize = state_sum(k, v, ld, None, None)
    oa, sa = t.linear_attention(q[:77], k[:77], v[:77], ld, return_state=True)
    ob, sb = t.linear_attention(q[77:], k[77:], v[77:], ld, state=sa, return_state=True)
    within(torch.cat([oa, ob]), ref, size, FP, inner_of(FP, T, Dk), 'two calls')
    within(sb, sref, ssize, FP, inner_of(FP, T, 0), 'state of two calls')
    pool = torch.zeros(B + 2, H, Dk, Dv, device=DEV)
    slots = torch.tensor([4, 0, 2], device=DEV)
    outs = [t.linear_attention_step(q[i], k[i], v[i], ld, pool, slots=slots) for i in range(T)]
    within(torch.stack(outs), ref, size, FP, inner_of(FP, T, Dk), 'steps')
    within(pool[slots], sref, ssize, FP, inner_of(FP, T, 0), 'state of steps')
    assert not pool[[1, 3]].any()


STEP = [(1, 1, 4, 64, 64, FP), (5, 9, 3, 33, 17, FP), (5, 5, 2, 128, 128, BF), (3, 4, 2, 256, 250, BF), (70, 300, 1, 1, 256, FP), (2, 2, 1, 256, 3, BF), (300, 301, 2, 16, 36, FP)]


@pytest.mark.parametrize('B,N,H,Dk,Dv,dt', STEP)
def test_linear_attention_step(B, N, H, Dk, Dv, dt):
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(B + Dk)
    q, k, v = rnd(g, B, H, Dk, dtype=dt), rnd(g, B, H, Dk, dtype=dt), rnd(g, B, H, Dv, dtype=dt)
    ld, pool = decays(H), rnd(g, N, H, Dk, Dv)
    before = pool.clone()
    slots = torch.randperm(N, generator=g)[:B]
    if B > 2:
        slots[1], slots[2] = -1, N                    # padded rows
    on = (slots >= 0) & (slots < N)
    o = t.linear_attention_step(q, k, v, ld, pool, slots=slots.to(DEV))
    a = torch.exp(ld.double()).view(1, H, 1, 1)
    s = before[slots[on].to(DEV)].double()
    kv = k[on.to(DEV)].double().unsqueeze(3) * v[on.to(DEV)].double().unsqueeze(2)
    new = a * s + kv
    got = pool[slots[on].to(DEV)]
    within(got, new, a * s.abs() + kv.abs(), FP, 8 * 2.0 ** -24, 'state')
    ref = Dk ** -0.5 * (q[on.to(DEV)].double().unsqueeze(3) * new).sum(2)
    size = Dk ** -0.5 * (q[on.to(DEV)].double().abs().unsqueeze(3) * (a * s.abs() + kv.abs())).sum(2)
    within(o[on.to(DEV)], ref, size, dt, (Dk + 16) * 2.0 ** -24, 'o')
    assert not o[~on.to(DEV)].any()
    untouched = torch.ones(N, dtype=torch.bool)
    untouched[slots[on]] = False
    assert torch.equal(pool[untouched.to(DEV)], before[untouched.to(DEV)])


def test_linear_attention_step_same_slot_twice():
    """Rows of one slot are successive tokens: the same as one call a token."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(2)
    B, H, D = 9, 2, 40
    q, k, v, ld = rnd(g, B, H, D), rnd(g, B, H, D), rnd(g, B, H, D), decays(2)
    slots = torch.tensor([3, 1, 3, 3, 0, 1, -1, 3, 2], device=DEV)
    a, b = rnd(g, 4, H, D, D), None
    b = a.clone()
    o = t.linear_attention_step(q, k, v, ld, a, slots=slots)
    for i in range(B):
        one = t.linear_attention_step(q[i:i + 1], k[i:i + 1], v[i:i + 1], ld, b, slots=slots[i:i + 1])
        assert torch.equal(one[0], o[i]), i
    assert torch.equal(a, b)


def turned(x, pos, w, inter, mag, back=False):
    T, B = x.shape[:2]
    p = pos.view(T, -1).expand(T, B).double()
    ang = (p.unsqueeze(-1) * w).unsqueeze(2) * (-1 if back else 1)
    n = w.numel()
    x = x.double()
    u, v = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if inter else (x[..., :n], x[..., n:2 * n])
    a, b = mag * (u * torch.cos(ang) - v * torch.sin(ang)), mag * (u * torch.sin(ang) + v * torch.cos(ang))
    r = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    z = mag * (u.abs() + v.abs())
    z = torch.stack([z, z], -1).flatten(-2) if inter else torch.cat([z, z], -1)
    return torch.cat([r, x[..., 2 * n:]], -1), torch.cat([z, torch.zeros_like(x[..., 2 * n:])], -1)


ROT = [(1, 1, 1, 1, 2, 2, FP, False, 0), (5, 3, 4, 2, 64, 64, BF, False, 0), (5, 3, 4, 0, 64, 32, BF, True, 10 ** 6), (33, 2, 3, 1, 81, 30, FP, True, 9 * 10 ** 8),
       (33, 2, 3, 1, 81, 30, BF, False, 77), (40, 7, 2, 5, 128, 128, FP, False, 10 ** 7), (3, 300, 1, 1, 16, 0, BF, False, 3), (9, 2, 2, 2, 512, 512, FP, True, 5),
       (2, 2, 16, 16, 24, 16, BF, False, 1), (2, 2, 16, 16, 24, 8, BF, True, 1)]


@pytest.mark.parametrize('T,B,Hq,Hk,D,rot,dt,inter,far', ROT)
def test_rotary(T, B, Hq, Hk, D, rot, dt, inter, far):
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(T + D)
    q, k = rnd(g, T, B, Hq, D, dtype=dt), (rnd(g, T, B, Hk, D, dtype=dt) if Hk else None)
    pos = (torch.randint(0, far + 1, (1, B), generator=g) + torch.arange(T).view(T, 1)).to(DEV)
    if T % 2:
        pos = pos[:, 0].contiguous() - 2              # one position for the whole batch, negative ones among them
    w = t.rotary_frequencies(rot, method=('none', 'linear', 'base', 'parts')[T % 4], factor=8.0, device=DEV)
    mag = 1.0 if T % 3 else 1.25
    leaves = [x.clone().requires_grad_() for x in ((q, k) if Hk else (q,))]
    out = t.rotary(leaves[0], leaves[1] if Hk else None, pos, w, interleaved=inter, magnitude=mag)
    out = out if Hk else (out,)
    inner = 12 * 2.0 ** -24                           # the reduced angle (half a turn, fp32), sine, cosine, magnitude, two products and their sum
    do = [rnd(g, *x.shape, dtype=dt) for x in leaves]
    grads = torch.autograd.grad(out, leaves, do)
    for x, y, gy, gx in zip(leaves, out, do, grads):
        ref, size = turned(x.detach(), pos, w, inter, mag)
        within(y.detach(), ref, size, dt, inner, 'turned')
        ref, size = turned(gy, pos, w, inter, mag, back=True)
        within(gx, ref, size, dt, inner, 'gradient')
        assert torch.equal(y.detach()[..., rot:], x.detach()[..., rot:])
    # one of the outputs alone
    if Hk:
        out = t.rotary(leaves[0], leaves[1], pos, w, interleaved=inter, magnitude=mag)
        (gk,) = torch.autograd.grad(out[1], leaves[1], do[1])
        assert torch.equal(gk, grads[1])
    strided = torch.cat([q, q], 3)[..., :D]
    a = t.rotary(strided, None, pos, w, interleaved=inter, magnitude=mag)
    assert torch.equal(a, (t.rotary(q, None, pos, w, interleaved=inter, magnitude=mag)))


NORM = [(1, 1, FP), (3, 7, BF), (5, 64, FP), (2304, 256, FP), (17, 513, BF), (9, 1000, FP), (9, 1024, BF), (6, 2048, BF), (600, 1030, BF), (3, 4096, FP), (5, 8192, BF),
        (2, 10001, FP), (2, 16384, BF), (2, 16384, FP), (1300, 40, BF)]


@pytest.mark.parametrize('M,N,dt', NORM)
@pytest.mark.parametrize('joint', [False, True])
def test_rms_norm(M, N, dt, joint):
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(M + N)
    x, w = rnd(g, M, N, dtype=dt), rnd(g, N)
    r = rnd(g, M, N, dtype=dt) if joint else None
    if M > 2:
        x[1] = 0
        if joint:
            r[1] = 0
    dy, ds = rnd(g, M, N, dtype=dt), (rnd(g, M, N, dtype=dt) if joint else None)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()] + ([r.clone().requires_grad_()] if joint else [])
    out = t.rms_norm(leaves[0], leaves[1], residual=leaves[2] if joint else None, eps=1e-5)
    y = out[0] if joint else out
    h = x.double() + (r.double() if joint else 0)
    rs = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
    u = 2.0 ** -24
    within(y.detach(), h * rs * w.double(), (h * rs * w.double()).abs(), dt, (math.log2(N) + 24) * u, 'y')
    if joint:
        within(out[1].detach(), h, h.abs(), dt, u, 'sum')
    grads = torch.autograd.grad(list(out) if joint else [y], leaves, [dy, ds] if joint else [dy])
    n = h * rs
    dn = dy.double() * w.double()
    dx = rs * (dn - n * (dn * n).mean(1, keepdim=True)) + (ds.double() if joint else 0)
    size = rs * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True)) + (ds.double().abs() if joint else 0)
    within(grads[0], dx, size, dt, (N / 256 + 40) * u, 'dx')
    within(grads[1], (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0), FP, (M / 512 + 60) * u, 'dw')
    if joint:
        assert torch.equal(grads[2], grads[0])
    again = t.rms_norm_backward(dy, x, w, residual=r, d_sum=ds, eps=1e-5)
    assert torch.equal(again[0], grads[0]) and torch.equal(again[1], grads[1])


def test_rms_norm_gradients_against_differences():
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(6)
    M, N, e = 4, 48, 2.0 ** -6
    x, w, dy = rnd(g, M, N), rnd(g, N), rnd(g, M, N)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    gx, gw = torch.autograd.grad(t.rms_norm(*leaves), leaves, dy)
    f = lambda a, b: (t.rms_norm(a, b).double() * dy.double()).sum().item()
    with torch.no_grad():
        d = rnd(g, M, N)
        size = (t.rms_norm(x, w).double() * dy.double()).abs().sum().item()
        diff = (f(x + e * d, w) - f(x - e * d, w)) / (2 * e)
        # rounding: 2^-24 * ~30 of the size over the step; truncation: the third derivative of h / |h| along d is a few |d|^3 / |h|^3 ~ a few, times e^2 / 6
        assert abs(diff - (gx.double() * d.double()).sum().item()) <= 30 * 2.0 ** -24 * size / e + 6 * e * e * size
        d = rnd(g, N)
        diff = (f(x, w + e * d) - f(x, w - e * d)) / (2 * e)
        assert abs(diff - (gw.double() * d.double()).sum().item()) <= 30 * 2.0 ** -24 * size / e


def rows8(h, w, eps):
    """The 8-bit rows of a norm (w given) or of h itself, in 64 bits.  The factor 127 / max is one rounded quotient, as documented: a number over a tensor
    would be the number times the reciprocal in torch, two roundings, which decide the exact ties that bfloat16 rows have (x * 127 / max = k + 1/2)."""
    z = h * w if w is not None else h
    top = z.abs().amax(-1, keepdim=True)
    to = torch.full_like(top, 127.0) / torch.where(top > 0, top, torch.ones_like(top))
    q = torch.where(top > 0, torch.round(z * to), torch.zeros_like(z))
    s = top / 127 * (1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) if w is not None else 1)
    return q, s.squeeze(-1)


@pytest.mark.parametrize('M,N,dt', NORM)
def test_rms_norm_int8(M, N, dt):
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(M * 3 + N)
    x, r, w = rnd(g, M, N, dtype=dt), rnd(g, M, N, dtype=dt), rnd(g, N)
    if M > 2:
        x[1], r[1] = 0, 0
        x[2, N // 2] = float('inf')
    bad = torch.zeros(M, dtype=torch.bool, device=DEV)
    if M > 2:
        bad[2] = True
    h = x.double() + r.double()
    q, s, total = t.rms_norm_int8(x, w, residual=r)
    rq, rs = rows8(h[~bad], w.double(), 1e-6)
    assert torch.equal(q[~bad].double(), rq)
    within(s[~bad], rs, rs, FP, (math.log2(N) + 24) * 2.0 ** -24, 'scale')
    assert torch.isnan(s[bad]).all() and not q[bad].any()
    assert torch.equal(total[~bad], (x.float() + r.float()).to(dt)[~bad])
    q, s = t.quantize_int8(x)
    rq, rs = rows8(x[~bad].double(), None, 0)
    assert torch.equal(q[~bad].double(), rq) and torch.isnan(s[bad]).all()
    within(s[~bad], rs, rs, FP, 2.0 ** -24, 'plain scale')


GEMM8 = [(1, 1, 1), (1, 16, 4), (3, 17, 5), (7, 4096, 4096), (16, 64, 128), (33, 65, 129), (128, 128, 128), (130, 1001, 77), (257, 192, 260), (512, 512, 512), (1000, 333, 300), (5, 20000, 40),
         (40, 1000, 500), (64, 1040, 90), (17, 80, 33), (2000, 144, 2100), (1500, 48, 1500), (4000, 208, 4100), (3000, 65, 3100)]


@pytest.mark.parametrize('M,K,N', GEMM8)
@pytest.mark.parametrize('dt', [FP, BF])
def test_linear_int8(M, K, N, dt):
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(M + K + N)
    x, w = (torch.randint(-128, 128, s, generator=g, dtype=torch.int8).to(DEV) for s in ((M, K), (N, K)))
    xs, ws, bias = rnd(g, M).abs(), rnd(g, N), rnd(g, N)
    acc = x.double() @ w.double().t()
    prod = acc * xs.double().view(-1, 1) * ws.double()
    got = t.linear_int8(x, xs, w, ws, bias=bias, out_dtype=dt)
    within(got, prod + bias.double(), prod.abs() + bias.double().abs(), dt, 4 * 2.0 ** -24, 'y')
    within(t.linear_int8(x, xs, w, ws, out_dtype=dt), prod, prod.abs(), dt, 4 * 2.0 ** -24, 'y without bias')
    # rows at other strides and any byte offset
    wide, wide_w = torch.zeros(M, K + 37, dtype=torch.int8, device=DEV), torch.zeros(N, K + 16, dtype=torch.int8, device=DEV)
    wide += 99
    wide_w += 77
    wide[:, 5:5 + K], wide_w[:, 3:3 + K] = x, w
    assert torch.equal(t.linear_int8(wide[:, 5:5 + K], xs, wide_w[:, 3:3 + K], ws, bias=bias, out_dtype=dt), got)


def test_linear_int8_extremes():
    from srvp_amd import temporal as t
    K = 131071
    x, w = torch.full((2, K), -128, dtype=torch.int8, device=DEV), torch.full((3, K), -128, dtype=torch.int8, device=DEV)
    one = lambda n: torch.ones(n, device=DEV)
    assert torch.equal(t.linear_int8(x, one(2), w, one(3)), torch.full((2, 3), float(K * 16384), device=DEV))
    y = t.linear_int8(x[:, :0], one(2), w[:, :0], one(3), bias=2 * one(3))
    assert torch.equal(y, torch.full((2, 3), 2.0, device=DEV))
    assert t.linear_int8(x[:0], one(0), w, one(3)).shape == (0, 3)


def test_empty_sizes():
    from srvp_amd import temporal as t
    z = lambda *s: torch.zeros(*s, device=DEV)
    ld = decays(2)
    s = rnd(torch.Generator().manual_seed(0), 3, 2, 4, 5)
    o, n = t.linear_attention(z(0, 3, 2, 4), z(0, 3, 2, 4), z(0, 3, 2, 5), ld, state=s, return_state=True)
    assert o.shape == (0, 3, 2, 5) and torch.equal(n, s)
    assert t.linear_attention(z(4, 0, 2, 4), z(4, 0, 2, 4), z(4, 0, 2, 5), ld).shape == (4, 0, 2, 5)
    d = t.linear_attention_backward(z(0, 3, 2, 5), z(0, 3, 2, 4), z(0, 3, 2, 4), z(0, 3, 2, 5), ld, state=s, d_state=s)
    assert (d[3] - s).abs().max() <= 2.0 ** -23 * s.abs().max()       # (multiplied by 1 / scale and by scale)
    assert t.linear_attention_step(z(0, 2, 4), z(0, 2, 4), z(0, 2, 5), ld, s).shape == (0, 2, 5)
    assert t.rotary(z(0, 3, 2, 4), None, torch.zeros(0, dtype=torch.int64, device=DEV), t.rotary_frequencies(4, device=DEV)).shape == (0, 3, 2, 4)
    x = z(0, 8).requires_grad_()
    w = torch.ones(8, device=DEV, requires_grad=True)
    gx, gw = torch.autograd.grad(t.rms_norm(x, w), [x, w], z(0, 8))
    assert gx.shape == (0, 8) and not gw.any()
    assert t.rms_norm_int8(z(0, 8), w.detach())[0].shape == (0, 8)


def test_other_stream_and_capture():
    """Launches go to the current stream; captured calls replay on new inputs, two graphs side by side, with eager work in between."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(21)
    T, B, H, D = 600, 1, 2, 64                             # cut into segments: the call has a workspace
    ld, w = decays(H), t.rotary_frequencies(D, device=DEV)
    pos = torch.arange(T, device=DEV)
    wt = rnd(g, H * D)

    def block(x):
        q, k = t.rotary(x, x, pos, w)
        o = t.linear_attention(q, k, x, ld)
        y, h = t.rms_norm(o.view(T, B, H * D), wt, residual=x.view(T, B, H * D))
        return (y, h) + t.linear_attention_backward(o, q, k, x, ld)[:3]
    xs = [rnd(g, T, B, H, D) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = block(xs[0])
    side.synchronize()
    for a, b in zip(there, block(xs[0])):
        assert torch.equal(a, b)
    graphs = []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = block(x)
        graphs.append((gr, x, out))
    for turn in range(3):
        for i, (gr, x, out) in enumerate(graphs):
            x.copy_(rnd(g, T, B, H, D))
        for gr, x, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, x, out in graphs:
            for a, b in zip(out, block(x)):
                assert torch.equal(a, b), turn
    # recording inside a capture is refused
    x = xs[0].clone().requires_grad_()
    gr = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(gr):
        y = xs[1] + 1
        try:
            t.linear_attention(x, x, x, ld)
        except RuntimeError as e:
            refused = 'capture' in str(e)
    assert refused

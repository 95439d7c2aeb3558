"""
Temporal operators at their edges: values that are not finite, offsets past 32 bits, rows of the largest values, calls from two threads, refusals.
"""
import math
import threading

import pytest
import torch

from test_gpu_temporal import BF, DEV, FP, decays, inner_of, rnd, rows8, scan, turned, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize('T,Dk,Dv,dt', [(50, 64, 64, FP), (50, 33, 17, FP), (150, 128, 128, BF), (150, 40, 72, BF), (150, 21, 35, BF), (90, 256, 200, BF)])
def test_linear_attention_is_causal_for_what_is_not_finite(T, Dk, Dv, dt, bad):
    """A NaN or infinity of token p changes nothing in front of p (gradients that run backwards in time: behind it), nor other columns of v."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(T + Dk)
    H, p, c = 2, T // 2 + 3, Dv - 2
    ld, sc = decays(H), Dk ** -0.5
    q, k, v, do = rnd(g, T, 1, H, Dk, dtype=dt), rnd(g, T, 1, H, Dk, dtype=dt), rnd(g, T, 1, H, Dv, dtype=dt), rnd(g, T, 1, H, Dv, dtype=dt)
    inn = inner_of(dt, T, max(Dk, Dv))

    def spoil(x, col):
        y = x.clone()
        y[p, :, 0, col] = bad
        return y
    others = [i for i in range(Dv) if i != c]
    fwd = lambda x: t.linear_attention(*x, ld)
    full, size = scan(q, k, v, ld, sc, False)
    o = fwd((q, k, spoil(v, c)))
    within(o[:p], full[:p], size[:p], dt, inn, 'o in front of a spoilt v')
    within(o[..., others], full[..., others], size[..., others], dt, inn, 'o beside a spoilt v')
    assert torch.equal(o[:, :, 1], fwd((q, k, v))[:, :, 1]) and not torch.isfinite(o[p, 0, 0, c])
    o = fwd((q, spoil(k, 0), v))
    within(o[:p], full[:p], size[:p], dt, inn, 'o in front of a spoilt k')
    o = fwd((spoil(q, 0), k, v))
    keep = [i for i in range(T) if i != p]
    within(o[keep], full[keep], size[keep], dt, inn, 'o beside a spoilt q')

    def back(*x):
        return t.linear_attention_backward(*x, ld)[:3]
    (rq, zq), (rk, zk), (rv, zv) = scan(do, v, k, ld, sc, False), scan(v, do, q, ld, sc, True), scan(k, q, do, ld, sc, True)
    after = slice(p + 1, T)
    dq, dk, dv = back(spoil(do, c), q, k, v)
    within(dq[keep], rq[keep], zq[keep], dt, inn, 'dq beside a spoilt do')
    within(dk[after], rk[after], zk[after], dt, inn, 'dk behind a spoilt do')
    within(dv[after], rv[after], zv[after], dt, inn, 'dv behind a spoilt do')
    within(dv[..., others], rv[..., others], zv[..., others], dt, inn, 'dv beside a spoilt do')
    dq, dk, dv = back(do, spoil(q, 0), k, v)
    within(dq, rq, zq, dt, inn, 'dq of a spoilt q')
    within(dk[after], rk[after], zk[after], dt, inn, 'dk behind a spoilt q')
    within(dv[after], rv[after], zv[after], dt, inn, 'dv behind a spoilt q')
    dq, dk, dv = back(do, q, spoil(k, 0), v)
    within(dq[:p], rq[:p], zq[:p], dt, inn, 'dq in front of a spoilt k')
    within(dk, rk, zk, dt, inn, 'dk of a spoilt k')
    within(dv[keep], rv[keep], zv[keep], dt, inn, 'dv beside a spoilt k')
    dq, dk, dv = back(do, q, k, spoil(v, c))
    within(dq[:p], rq[:p], zq[:p], dt, inn, 'dq in front of a spoilt v')
    within(dk[keep], rk[keep], zk[keep], dt, inn, 'dk beside a spoilt v')
    within(dv, rv, zv, dt, inn, 'dv of a spoilt v')


def test_linear_attention_padding_without_lengths():
    """Right-padded rows full of NaN leave the tokens in front of them alone, also where a sequence is cut into segments."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(7)
    T, H, D = 900, 2, 64
    q, k, v = (rnd(g, T, 2, H, D, dtype=BF) for _ in range(3))
    ref, size = scan(q, k, v, decays(H), D ** -0.5, False)
    for x in (q, k, v):
        x[517:, 0] = float('nan')
    o = t.linear_attention(q, k, v, decays(H))
    within(o[:517], ref[:517], size[:517], BF, inner_of(BF, T, D), 'in front of the padding')
    within(o[:, 1], ref[:, 1], size[:, 1], BF, inner_of(BF, T, D), 'the other sequence')


@pytest.mark.parametrize('dt', [FP, BF])
def test_int8_rows_of_the_largest_values(dt):
    """Rows whose squares pass 32 bits, and rows of the smallest values: as exact as any other."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(3)
    x = rnd(g, 6, 300)
    for i, e in enumerate((1e20, 3e37, 1e-30, 1e-38, 1.0, 0.0)):
        x[i] *= e
    x, w = x.to(dt), rnd(g, 300)
    q, s = t.quantize_int8(x)
    rq, rs = rows8(x.double(), None, 0)
    assert torch.equal(q.double(), rq)
    # half a step, and 2^-150 where the scale is subnormal
    assert ((s.double() - rs).abs() <= 2.0 ** -24 * rs + 2.0 ** -150).all()
    q, s = t.rms_norm_int8(x, w)
    rq, rs = rows8(x.double(), w.double(), 1e-6)
    assert torch.equal(q.double(), rq)
    assert ((s.double() - rs).abs() <= (2.0 ** -24 + 1e-12) * rs + 2.0 ** -150).all()


def test_offsets_past_32_bits():
    """Strides and slots whose products pass 2^31 elements: the results of the packed copies."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(5)
    big = torch.empty(5 * 2 ** 30, dtype=torch.uint8, device=DEV)

    def apart(x, stride):
        """x with its rows `stride` elements apart."""
        inner = x[0].numel()
        y = big.view(x.dtype).as_strided(x.shape, (stride,) + x[0].contiguous().stride())
        assert (x.shape[0] - 1) * stride + inner <= big.numel() // x.element_size() and (x.shape[0] - 1) * stride >= 2 ** 31 // (1 if x.element_size() < 4 else 2)
        return y.copy_(x)
    H, D = 2, 64
    ld = decays(H)
    # by 16-byte loads (a step under 2^23 elements) and one by one
    for T, stride in ((300, 2 ** 23 - 8), (36, 2 ** 26 + 8)):
        q, k, v = (rnd(g, T, 1, H, D, dtype=BF) for _ in range(3))
        ref = t.linear_attention(q, k, v, ld)
        assert torch.equal(t.linear_attention(apart(q, stride), k, v, ld), ref)
        assert torch.equal(t.linear_attention(q, apart(k, stride), v, ld), ref)
        assert torch.equal(t.linear_attention(q, k, apart(v, stride), ld), ref)
        ref = t.linear_attention_backward(v, q, k, v, ld)
        for a, b in zip(t.linear_attention_backward(apart(v, stride), q, k, v, ld)[:3], ref):
            assert torch.equal(a, b)
    pos, w = torch.arange(36, device=DEV), t.rotary_frequencies(D, device=DEV)
    assert torch.equal(t.rotary(apart(q, stride), None, pos, w), t.rotary(q, None, pos, w))
    x, wt = q.reshape(36, -1), rnd(g, H * D)
    wide = apart(x, stride)
    for a, b in zip(t.rms_norm(wide, wt, residual=x) + t.rms_norm_int8(x, wt, residual=wide) + t.rms_norm_backward(wide, x, wt),
                    t.rms_norm(x, wt, residual=x) + t.rms_norm_int8(x, wt, residual=x) + t.rms_norm_backward(x, x, wt)):
        assert torch.equal(a, b)
    for M, K in ((40, 128), (70, 128), (70, 51)):
        a, b = (torch.randint(-128, 128, s, generator=g, dtype=torch.int8).to(DEV) for s in ((M, K), (70, K)))
        sa, sb = rnd(g, M), rnd(g, 70)
        ref = t.linear_int8(a, sa, b, sb)
        assert torch.equal(t.linear_int8(apart(a, 2 ** 26), sa, b, sb), ref)
        assert torch.equal(t.linear_int8(a, sa, apart(b, 2 ** 26), sb), ref)
    # a pool of states of more than 2^31 bytes and elements: 140000 slots of 8192 values
    pool = big.view(FP)[:140000 * 8192].view(140000, H, D, D)
    slots = torch.tensor([139999, 7, 70001], device=DEV)
    few = rnd(g, 3, H, D, D)
    pool[slots] = few
    q, k, v = (rnd(g, 3, H, D) for _ in range(3))
    assert torch.equal(t.linear_attention_step(q, k, v, ld, pool, slots=slots), t.linear_attention_step(q, k, v, ld, few))
    assert torch.equal(pool[slots], few)


def test_two_threads():
    """Calls from two threads on their own streams: each thread's own results."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(6)
    ld = decays(2)
    ins = [tuple(rnd(g, 700, 1, 2, 64, dtype=BF) for _ in range(3)) for _ in range(2)]
    ref = [t.linear_attention(*x, ld) for x in ins]
    torch.cuda.synchronize()
    out = [None, None]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            out[i] = [t.linear_attention(*ins[i], ld) for _ in range(20)]
        s.synchronize()
    both = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in both:
        x.start()
    for x in both:
        x.join()
    for i in range(2):
        assert all(torch.equal(o, ref[i]) for o in out[i])


def test_inference_mode_and_versions():
    """States that are advanced in place are seen as changed; inference mode takes the same calls."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(9)
    q, k, v, ld = rnd(g, 2, 2, 16), rnd(g, 2, 2, 16), rnd(g, 2, 2, 16), decays(2)
    s = torch.zeros(2, 2, 16, 16, device=DEV)
    n = s._version
    o = t.linear_attention_step(q, k, v, ld, s)
    assert s._version == n + 1
    x = rnd(g, 5, 2, 2, 16).requires_grad_()
    y = t.linear_attention(x, x, x, ld, state=s)
    t.linear_attention_step(q, k, v, ld, s)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    with torch.inference_mode():
        z = torch.zeros(2, 2, 16, 16, device=DEV)
        assert torch.equal(t.linear_attention_step(q, k, v, ld, z), o)
        assert torch.equal(t.linear_attention(x, x, x, ld, state=s), t.linear_attention(x.detach(), x.detach(), x.detach(), ld, state=s))


def test_refusals():
    from srvp_amd import temporal as t
    from srvp_amd._lib import SrvpHipError
    z = lambda *s, dt=FP: torch.zeros(*s, dtype=dt, device=DEV)
    x, ld, w = z(4, 2, 3, 8), decays(3), t.rotary_frequencies(8, device=DEV)
    st, pos, i8 = z(2, 3, 8, 8), torch.arange(4, device=DEV), lambda *s: z(*s, dt=torch.int8)
    la, step, rot, norm, lin = t.linear_attention, t.linear_attention_step, t.rotary, t.rms_norm, t.linear_int8
    grad = lambda *s: z(*s).requires_grad_()
    cases = [
        (ValueError, lambda: la(x[0], x[0], x[0], ld)), (ValueError, lambda: la(x, z(4, 2, 3, 9), x, ld)), (ValueError, lambda: la(x, x, z(4, 2, 2, 8), ld)),
        (TypeError, lambda: la(x.half(), x.half(), x.half(), ld)), (TypeError, lambda: la(x, x.to(BF), x, ld)), (ValueError, lambda: la(x, x, x, ld.double())),
        (ValueError, lambda: la(x, x, x, ld[:2])), (ValueError, lambda: la(x, x, x, ld.clone().requires_grad_())), (ValueError, lambda: la(x, x, x, ld.cpu())),
        (ValueError, lambda: la(x, x, x, ld, state=st[:1])), (ValueError, lambda: la(x, x, x, ld, state=st.to(BF))), (ValueError, lambda: la(x, x, x, ld, lengths=pos)),
        (TypeError, lambda: la(x, x, x, ld, lengths=z(2))), (ValueError, lambda: la(x, x, x, ld, scale=0.0)), (ValueError, lambda: la(x, x, x, ld, scale=1e-35)),
        (ValueError, lambda: la(x, x, x, ld, scale=float('nan'))), (ValueError, lambda: la(z(1, 1, 1, 257), z(1, 1, 1, 257), z(1, 1, 1, 4), ld[:1])),
        (ValueError, lambda: la(z(1, 1, 1, 8).expand(2, 2 ** 20, 1, 8), z(1, 1, 1, 8).expand(2, 2 ** 20, 1, 8), z(1, 1, 1, 8).expand(2, 2 ** 20, 1, 8), ld[:1])),
        (ValueError, lambda: t.linear_attention_backward(x[:3], x, x, x, ld)), (ValueError, lambda: t.linear_attention_backward(x, x, x, x, ld, d_state=st[:1])),
        (ValueError, lambda: t.linear_attention_backward(x, grad(4, 2, 3, 8), x, x, ld)), (SrvpHipError, lambda: la(x.cpu(), x.cpu(), x.cpu(), ld.cpu())),
        (ValueError, lambda: step(x, x, x, ld, st)), (ValueError, lambda: step(x[:, 0], x[:, 0], x[:, 0], ld, st)), (ValueError, lambda: step(x[0], x[0], x[0], ld, st.transpose(2, 3))),
        (ValueError, lambda: step(x[0], x[0], x[0], ld, st.to(BF))), (TypeError, lambda: step(x[0], x[0], x[0], ld, st, slots=z(2))), (ValueError, lambda: step(x[0], x[0], x[0], ld, st, slots=pos)),
        (ValueError, lambda: step(grad(2, 3, 8), x[0], x[0], ld, st)), (ValueError, lambda: step(x[0], x[0], x[0], ld, z(2 * 3 * 64 + 1)[1:].view(2, 3, 8, 8))),
        (ValueError, lambda: rot(x, z(4, 2, 3, 6), pos, w)), (ValueError, lambda: rot(x, None, pos[:3], w)), (TypeError, lambda: rot(x, None, z(4), w)),
        (ValueError, lambda: rot(x, None, pos, w.float())), (ValueError, lambda: rot(x, None, pos, t.rotary_frequencies(10, device=DEV))), (ValueError, lambda: rot(x, None, pos.cpu(), w)),
        (ValueError, lambda: rot(x, None, pos, w, magnitude=float('inf'))), (ValueError, lambda: rot(z(1, 1, 1, 8).expand(2 ** 20, 2 ** 11, 1, 8), None, pos, w)),
        (ValueError, lambda: rot(z(1, 1, 1, 2).expand(1, 1, 2 ** 20, 2), None, pos[:1], w[:1])),
        (ValueError, lambda: norm(x, z(7))), (ValueError, lambda: norm(x, z(8, dt=BF))), (ValueError, lambda: norm(x, z(8), residual=x[:2])), (TypeError, lambda: norm(x, z(8), residual=x.to(BF))),
        (TypeError, lambda: norm(x.double(), z(8))), (ValueError, lambda: norm(z(2, 16385), z(16385))), (ValueError, lambda: norm(x, torch.zeros(8))), (ValueError, lambda: norm(z(2, 0), z(0))),
        (ValueError, lambda: t.rms_norm_backward(x[:2], x, z(8))), (ValueError, lambda: t.rms_norm_int8(grad(2, 8), z(8))), (ValueError, lambda: t.quantize_int8(grad(2, 8))),
        (TypeError, lambda: lin(x, z(4, 2, 3), i8(5, 8), z(5))), (ValueError, lambda: lin(i8(4, 9), z(4), i8(5, 8), z(5))), (ValueError, lambda: lin(i8(4, 8), z(4, 1), i8(5, 8), z(5))),
        (ValueError, lambda: lin(i8(4, 8), z(4), i8(5, 8), z(4))), (ValueError, lambda: lin(i8(4, 8), z(4), i8(5, 8), z(5), bias=z(4))), (TypeError, lambda: lin(i8(4, 8), z(4), i8(5, 8), z(5), out_dtype=torch.float16)),
        (ValueError, lambda: lin(i8(1, 131072), z(1), i8(1, 131072), z(1))), (ValueError, lambda: lin(i8(4, 8), z(4), i8(5, 8).cpu(), z(5))), (ValueError, lambda: lin(i8(4, 8), z(4), i8(5, 8), grad(5))),
    ]
    for i, (kind, f) in enumerate(cases):
        try:
            f()
        except kind:
            continue
        except Exception as e:
            raise AssertionError(f'case {i}: {type(e).__name__}: {e}')
        raise AssertionError(f'case {i}: not refused')
    # differentiable once
    q = rnd(torch.Generator().manual_seed(1), 4, 2, 3, 8).requires_grad_()
    for y in (la(q, q, q, ld), rot(q, None, pos, w), norm(q, torch.ones(8, device=DEV))):
        with pytest.raises(RuntimeError, match='create_graph'):
            torch.autograd.grad(y.sum(), q, create_graph=True)
    # an output that cannot be allocated is torch's own error, and the next call works
    far = z(1, 1, 1, 256).expand(2 ** 29, 4, 1, 256)
    with pytest.raises(torch.OutOfMemoryError):
        la(far, far, far, ld[:1])
    assert la(x, x, x, ld).shape == x.shape


def inside(g, T, B, H, D, dt, off, pad):
    """Rows of D features that begin `off` elements into rows of D + pad; what lies around them is NaN."""
    wide = torch.full((T, B, H, D + pad), float('nan'), dtype=dt, device=DEV)
    wide[..., off:off + D] = rnd(g, T, B, H, D, dtype=dt)
    return wide[..., off:off + D]


@pytest.mark.parametrize('T,Dk,Dv,off,pad,lengths', [
    (1, 8, 9, 1, 2, None), (33, 7, 9, 3, 3, [33, 0]), (70, 9, 15, 1, 1, [70, 1]), (129, 83, 32, 1, 8, None), (150, 63, 60, 2, 5, [65, 150]),
    (200, 127, 129, 7, 7, None), (66, 64, 128, 1, 8, [66, 64]), (300, 249, 250, 5, 6, [299, 2]), (900, 65, 11, 0, 3, None), (90, 4, 5, 1, 2, None),
])
@pytest.mark.parametrize('dt', [BF, FP])
def test_linear_attention_of_rows_at_odd_places(T, Dk, Dv, off, pad, lengths, dt):
    """Feature counts and addresses that no wide access divides, inside rows whose other elements are NaN."""
    from srvp_amd import temporal as t
    B, H = 2, 3
    g = torch.Generator().manual_seed(T + Dk)
    q, k, v, do = (inside(g, T, B, H, D, dt, off, pad) for D in (Dk, Dk, Dv, Dv))
    ld, sc = decays(H), Dk ** -0.5
    n = None if lengths is None else torch.tensor(lengths, device=DEV)
    for b, m in enumerate(lengths or []):
        for x in (q, k, v, do):
            x[m:, b] = float('nan')
    inn = inner_of(dt, T, max(Dk, Dv))
    qc, kc, vc, gc = (torch.nan_to_num(x) for x in (q, k, v, do))
    o = t.linear_attention(q, k, v, ld, lengths=n)
    within(o, *scan(qc, kc, vc, ld, sc, False, lengths=lengths), dt, inn, 'o')
    dq, dk, dv = t.linear_attention_backward(do, q, k, v, ld, lengths=n)[:3]
    within(dq, *scan(gc, vc, kc, ld, sc, False, lengths=lengths), dt, inn, 'dq')
    within(dk, *scan(vc, gc, qc, ld, sc, True, lengths=lengths), dt, inn, 'dk')
    within(dv, *scan(kc, qc, gc, ld, sc, True, lengths=lengths), dt, inn, 'dv')


@pytest.mark.parametrize('N,off,pad', [(1, 1, 2), (3, 1, 1), (4, 1, 2), (5, 3, 4), (7, 1, 3), (8, 1, 1), (9, 7, 8), (77, 2, 2), (513, 1, 5), (1001, 3, 3), (1024, 1, 8), (2050, 5, 6),
                                       (4095, 1, 2), (4096, 3, 8), (8191, 1, 1), (10001, 5, 7), (16384, 1, 1)])
@pytest.mark.parametrize('dt', [BF, FP])
def test_rms_norm_of_rows_at_odd_places(N, off, pad, dt):
    """Rows that begin at any element, inside rows whose other elements are NaN; rows of whole vectors give what the same rows give at wide borders."""
    from srvp_amd import temporal as t
    M = 11
    g = torch.Generator().manual_seed(N)
    x, r, dy, ds = (inside(g, M, 1, 1, N, dt, off, pad)[:, 0, 0] for _ in range(4))
    w = inside(g, 1, 1, 1, N, FP, off, pad)[0, 0, 0]
    u, h, wd = 2.0 ** -24, x.double() + r.double(), w.double()
    rs = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)
    y, total = t.rms_norm(x, w, residual=r)
    within(y, h * rs * wd, (h * rs * wd).abs(), dt, (math.log2(N) + 24) * u, 'y')
    within(total, h, h.abs(), dt, u, 'sum')
    dx, dw = t.rms_norm_backward(dy, x, w, residual=r, d_sum=ds)[:2]
    n, dn = h * rs, dy.double() * wd
    size = rs * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True)) + ds.double().abs()
    within(dx, rs * (dn - n * (dn * n).mean(1, keepdim=True)) + ds.double(), size, dt, (N / 256 + 40) * u, 'dx')
    within(dw, (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0), FP, (M / 512 + 60) * u, 'dw')
    q, s, again = t.rms_norm_int8(x, w, residual=r)
    rq, rscale = rows8(h, wd, 1e-6)
    assert torch.equal(q.double(), rq) and torch.equal(again, total)
    within(s, rscale, rscale, FP, (math.log2(N) + 24) * u, 'scale')
    if N % (16 // x.element_size()) == 0:
        xa, ra, dya, dsa, wa = (a.contiguous().clone() for a in (x, r, dy, ds, w))
        assert torch.equal(t.rms_norm(xa, wa, residual=ra)[0], y)
        for a, b in zip(t.rms_norm_backward(dya, xa, wa, residual=ra, d_sum=dsa), (dx, dw)):
            assert torch.equal(a, b)


@pytest.mark.parametrize('D,rot', [(1, 0), (2, 2), (5, 4), (7, 6), (8, 8), (9, 8), (16, 0), (17, 16), (21, 18), (33, 16), (63, 62), (65, 32), (84, 84), (126, 126), (127, 126), (127, 34),
                                   (128, 128), (250, 200), (515, 514)])
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('dt', [BF, FP])
def test_rotary_of_heads_at_odd_places(D, rot, inter, dt):
    """Heads that begin at any element and turn any number of pairs, inside rows whose other elements are NaN; the rest of a head is copied as it is."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(D + rot)
    T, B = 19, 3
    q, k = inside(g, T, B, 5, D, dt, 1, 2), inside(g, T, B, 2, D, dt, 3, 4)
    pos = torch.randint(0, 10 ** 6, (T, B), generator=g).to(DEV)
    w = t.rotary_frequencies(rot, device=DEV)
    back = D % 2 == 1
    for x, o in zip((q, k), t.rotary(q, k, pos, w, interleaved=inter, back=back)):
        ref, size = turned(x, pos, w, inter, 1.0, back)
        within(o, ref, size, dt, 12 * 2.0 ** -24, 'rotary')
        assert torch.equal(o[..., rot:], x[..., rot:])
        assert torch.equal(o, t.rotary(x.contiguous(), None, pos, w, interleaved=inter, back=back))


@pytest.mark.parametrize('M,N', [(3, 7), (9, 300), (5, 1024), (3, 4095), (4, 9000), (2, 16384)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize('dt', [BF, FP])
def test_int8_rows_of_a_weight_that_is_not_finite(M, N, bad, dt):
    """One weight that is NaN or infinite leaves no row of the norm finite, rows of zeros among them (0 * infinity): scale NaN, and NaN behind the product."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(N)
    x, r, w = rnd(g, M, N, dtype=dt), rnd(g, M, N, dtype=dt), rnd(g, N)
    x[1], r[1] = 0, 0
    for col in {0, N // 2, N - 1}:
        spoilt = w.clone()
        spoilt[col] = bad
        q, s, total = t.rms_norm_int8(x, spoilt, residual=r)
        assert torch.isnan(s).all() and not q.any()
        assert torch.equal(total, (x.float() + r.float()).to(dt))
        assert not torch.isfinite(t.rms_norm(x, spoilt, residual=r)[0][:, col]).any()
    y = t.linear_int8(q, s, torch.ones(3, N, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV))
    assert torch.isnan(y).all()


def test_forward_mode_is_refused():
    """A tangent on any input of any operator, with gradients enabled or not: an error, never an output without its tangent."""
    import torch.autograd.forward_ad as fwd
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(13)
    x, st, ld = rnd(g, 4, 2, 3, 8), rnd(g, 2, 3, 8, 8), decays(3)
    w, pos, freq = rnd(g, 8), torch.arange(4, device=DEV), t.rotary_frequencies(8, device=DEV)
    i8, one = torch.ones(4, 8, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    calls = [
        (lambda q, k, v, l, s: t.linear_attention(q, k, v, l, state=s), (x, x, x, ld, st)),
        (lambda d, q, k, v, l, s, n: t.linear_attention_backward(d, q, k, v, l, state=s, d_state=n), (x, x, x, x, ld, st, st)),
        (lambda q, k, v, l, s: t.linear_attention_step(q, k, v, l, s), (x[0], x[0], x[0], ld, st)),
        (lambda q, k, f: t.rotary(q, k, pos, f), (x, x, freq)),
        (lambda a, b, r: t.rms_norm(a, b, residual=r), (x, w, x)),
        (lambda d, a, b, r, s: t.rms_norm_backward(d, a, b, residual=r, d_sum=s), (x, x, w, x, x)),
        (lambda a, b, r: t.rms_norm_int8(a, b, residual=r), (x, w, x)),
        (lambda a: t.quantize_int8(a), (x,)),
        (lambda a, b, c: t.linear_int8(i8, a, i8, b, bias=c), (one, one, one)),
    ]
    for f, args in calls:
        f(*args)
        before = [a.clone() for a in args]
        for i in range(len(args)):
            for enabled in (True, False):
                with fwd.dual_level(), torch.set_grad_enabled(enabled):
                    duals = list(args)
                    duals[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(RuntimeError, match='forward-mode'):
                        f(*duals)
        for a, b in zip(args, before):
            assert torch.equal(a, b)


def test_frequencies_take_no_gradient():
    """Frequencies that ask for a gradient would be left without one: refused, as decays are; without recording they are taken as they are."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(14)
    x, pos, w = rnd(g, 4, 2, 3, 8), torch.arange(4, device=DEV), t.rotary_frequencies(8, device=DEV)
    learnt = w.clone().requires_grad_()
    for q in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match='frequencies'):
            t.rotary(q, None, pos, learnt)
    with torch.no_grad():
        assert torch.equal(t.rotary(x, None, pos, learnt), t.rotary(x, None, pos, w))


def test_learnt_decays_without_recording():
    """Decays that ask for a gradient are refused where one would be recorded, and taken as they are elsewhere."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(15)
    x, s, ld = rnd(g, 4, 2, 3, 8), rnd(g, 2, 3, 8, 8), decays(3)
    learnt = ld.clone().requires_grad_()
    for f in (lambda l: t.linear_attention(x, x, x, l), lambda l: t.linear_attention_backward(x, x, x, x, l)[0], lambda l: t.linear_attention_step(x[0], x[0], x[0], l, s.clone())):
        with pytest.raises(ValueError, match='constants'):
            f(learnt)
        with torch.no_grad():
            assert torch.equal(f(learnt), f(ld))


def test_step_of_many_rows():
    """Thousands of rows, slots in any order, padded ones and slots that come several times: one call is as many calls of rows of different slots."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(16)
    B, H, D, N = 6000, 1, 16, 7000
    q, k, v, ld = rnd(g, B, H, D), rnd(g, B, H, D), rnd(g, B, H, D), decays(H)
    slots = torch.randperm(N, generator=g)[:B]
    slots[5::7] = -1
    slots[4000:4020] = slots[0:20]                        # a second token for some
    pool = rnd(g, N, H, D, D)
    again = pool.clone()
    slots = slots.to(DEV)
    o = t.linear_attention_step(q, k, v, ld, pool, slots=slots)
    for a, b in ((0, 4000), (4000, B)):
        assert torch.equal(o[a:b], t.linear_attention_step(q[a:b], k[a:b], v[a:b], ld, again, slots=slots[a:b]))
    assert torch.equal(pool, again)
    on = (slots >= 0)[:4000]
    assert not o[:4000][~on].any() and o[:4000][on].any(-1).all()


def test_rows_with_slots_have_a_bound():
    from srvp_amd import temporal as t
    x, st, slots = torch.zeros(65537, 1, 1, device=DEV), torch.zeros(65537, 1, 1, 1, device=DEV), torch.arange(65537, device=DEV)
    with pytest.raises(ValueError, match='65536 rows'):
        t.linear_attention_step(x, x, x, decays(1), st, slots=slots)
    assert t.linear_attention_step(x, x, x, decays(1), st).shape == x.shape          # (without a search)
    assert t.linear_attention_step(x[1:], x[1:], x[1:], decays(1), st, slots=slots[1:]).shape == (65536, 1, 1)


@pytest.mark.parametrize('T,B,lengths', [(0, 2, None), (1, 2, None), (90, 2, [0, 90]), (700, 1, None), (700, 1, [0]), (700, 1, [300])])
@pytest.mark.parametrize('dt', [BF, FP])
def test_state_gradients_at_the_ends_of_sequences(T, B, lengths, dt):
    """No tokens, one, none in a sequence of several, segments behind the last token; with and without a gradient of the new state; eager, and captured and replayed."""
    from srvp_amd import temporal as t
    from test_gpu_temporal import state_sum
    g = torch.Generator().manual_seed(T + B)
    H, Dk, Dv = 2, 64, 40
    q, k, v, do = rnd(g, T, B, H, Dk, dtype=dt), rnd(g, T, B, H, Dk, dtype=dt), rnd(g, T, B, H, Dv, dtype=dt), rnd(g, T, B, H, Dv, dtype=dt)
    s0, dn, ld, sc = rnd(g, B, H, Dk, Dv), rnd(g, B, H, Dk, Dv), decays(H), Dk ** -0.5
    n = None if lengths is None else torch.tensor(lengths, device=DEV)
    for d in (dn, None):
        call = lambda: t.linear_attention_backward(do, q, k, v, ld, state=s0, lengths=n, d_state=d)
        eager = call()
        ref, size = state_sum(q, do, ld, lengths, d, scale=sc, from_end=False, off=1)
        within(eager[3], ref, size, FP, (T + 64) * 2.0 ** -24, 'dstate')
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for i in range(3):
            for x in (q, do) if T else ():
                x.copy_(rnd(g, *x.shape, dtype=dt))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, call()):
                assert torch.equal(a, b), i

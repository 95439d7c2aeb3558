"""
What the bfloat16 attention may round: its outputs to their own type, and nothing else to as few bits.  Short sequences behind a state, so that the bound counts a handful of
roundings and not the length of the sums.
"""
import math
from decimal import Context, Decimal, localcontext

import pytest
import torch

from test_gpu_temporal import BF, DEV, decays, rnd, scan, state_sum, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('T,H,Dk,Dv', [(1, 2, 64, 64), (3, 2, 128, 128), (5, 3, 40, 72), (17, 2, 128, 64), (70, 2, 64, 128), (9, 2, 83, 35), (4, 2, 256, 256)])
def test_bf16_attention_rounds_its_outputs_only(T, H, Dk, Dv):
    """The state where it multiplies q (and the gradients' carries) and the scores are two bfloat16 terms, each off by 2^-8 of what it stands for: 2^-16; decay x value at least two as
    well; a sum of n products in fp32 2^-24 n.  A state rounded once (2^-8 of it) is 2^6 of these bounds a product, and 2^3 after sums of 64 products of either sign."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(T + Dk)
    B = 2
    q, k, v, do = rnd(g, T, B, H, Dk, dtype=BF), rnd(g, T, B, H, Dk, dtype=BF), rnd(g, T, B, H, Dv, dtype=BF), rnd(g, T, B, H, Dv, dtype=BF)
    s0, dn, ld, sc = rnd(g, B, H, Dk, Dv, scale=3.0), rnd(g, B, H, Dk, Dv, scale=3.0), decays(H), Dk ** -0.5
    inner = 2 * 2.0 ** -16 + (max(Dk, Dv) + T + 64) * 2.0 ** -24
    within(t.linear_attention(q, k, v, ld, state=s0), *scan(q, k, v, ld, sc, False, sc * s0, off=1), BF, inner, 'o')
    dq, dk, dv, _ = t.linear_attention_backward(do, q, k, v, ld, state=s0, d_state=dn)
    within(dq, *scan(do, v, k, ld, sc, False, sc * s0.transpose(2, 3), off=1), BF, inner, 'dq')
    within(dk, *scan(v, do, q, ld, sc, True, dn.transpose(2, 3)), BF, inner, 'dk')
    within(dv, *scan(k, q, do, ld, sc, True, dn), BF, inner, 'dv')


@pytest.mark.parametrize('T,B,H,Dk,Dv', [(200, 3, 8, 128, 128), (900, 1, 2, 64, 64), (130, 2, 3, 83, 35), (70, 2, 2, 200, 96)])
@pytest.mark.parametrize('dt', [BF, torch.float32])
def test_results_do_not_depend_on_what_else_was_asked_for(T, B, H, Dk, Dv, dt):
    """dq, dk, dv with the state's gradient and without it, o with the new state and without it: the same bits."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(T)
    q, k, v, do = rnd(g, T, B, H, Dk, dtype=dt), rnd(g, T, B, H, Dk, dtype=dt), rnd(g, T, B, H, Dv, dtype=dt), rnd(g, T, B, H, Dv, dtype=dt)
    ld = decays(H)
    with_state = t.linear_attention_backward(do, q, k, v, ld, state=torch.zeros(B, H, Dk, Dv, device=DEV))
    for a, b in zip(t.linear_attention_backward(do, q, k, v, ld)[:3], with_state):
        assert torch.equal(a, b)
    s0 = rnd(g, B, H, Dk, Dv)
    outs = []
    for wanted in (False, True):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        s = s0.clone().requires_grad_(wanted)
        o = t.linear_attention(*leaves, ld, state=s, return_state=wanted)
        o = o[0] if wanted else o
        outs.append((o.detach(),) + torch.autograd.grad(o, leaves + ([s] if wanted else []), do)[:3])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


DIGITS = Context(prec=70)


def exact_pi():
    """pi = 16 arctan(1/5) - 4 arctan(1/239), by the series."""
    def arctan_of_inverse(n):
        term = total = Decimal(1) / n
        k = 1
        while abs(term) > Decimal(10) ** -68:
            term, k = -term / (n * n), k + 2
            total += term / k
        return total
    with localcontext(DIGITS):
        return 16 * arctan_of_inverse(5) - 4 * arctan_of_inverse(239)


PI = exact_pi()


def exact_angle(position, frequency):
    """position * frequency without its whole turns, to about 1e-30 (the double nearest to it)."""
    with localcontext(DIGITS):
        a = Decimal(position) * Decimal(frequency)
        return float(a - (a / (2 * PI)).to_integral_value() * 2 * PI)


@pytest.mark.parametrize('far', [10 ** 3, 10 ** 8, 2 ** 33 + 5, 10 ** 12, 2 ** 45 + 1, 2 ** 53 - 9])
@pytest.mark.parametrize('inter', [False, True])
def test_rotary_at_any_position(far, inter):
    """Angles against exact arithmetic, negative positions among them: the sine's and cosine's own rounding wherever the position lies (an angle formed in 64 bits
    alone would be off by 1e-4 radians at 10^12 and by whole turns at 2^53)."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(far % 1000)
    T, D = 8, 16
    x = rnd(g, T, 1, 2, D)
    pos = [far - i if i % 2 else i - far for i in range(T)]
    w = t.rotary_frequencies(D, base=500.0)
    angles = torch.tensor([[exact_angle(p, f) for f in w.tolist()] for p in pos], dtype=torch.float64, device=DEV).view(T, 1, 1, D // 2)
    c, s = torch.cos(angles), torch.sin(angles)
    at = (slice(0, D, 2), slice(1, D, 2)) if inter else (slice(0, D // 2), slice(D // 2, D))
    u, v = x.double()[..., at[0]], x.double()[..., at[1]]
    ref, size = torch.empty(T, 1, 2, D, dtype=torch.float64, device=DEV), torch.empty(T, 1, 2, D, dtype=torch.float64, device=DEV)
    ref[..., at[0]], ref[..., at[1]] = u * c - v * s, u * s + v * c
    size[..., at[0]] = size[..., at[1]] = u.abs() + v.abs()
    out = t.rotary(x, None, torch.tensor(pos, device=DEV), w.to(DEV), interleaved=inter)
    # the fraction of a turn in fp32, half a turn at most: pi 2^-24 radians; sine and cosine 2 units each, two products and a sum
    within(out, ref, size, torch.float32, 8 * 2.0 ** -24, 'turned')


@pytest.mark.parametrize('far', [0, 5 * 10 ** 6])
def test_sines_and_cosines_are_exact_to_their_own_rounding(far):
    """Unit vectors show the table itself.  Relative to each sine and cosine, also where it is close to zero: two units of the function's own (2^-22), a sum's rounding;
    the fraction of a turn in fp32 alone would put 10^-7 radians on it, all of a cosine of that size."""
    from srvp_amd import temporal as t
    T, D = 256, 128
    x = torch.zeros(T, 1, 1, D, device=DEV)
    x[..., :D // 2] = 1
    w, pos = t.rotary_frequencies(D), far + torch.arange(T)
    out = t.rotary(x, None, pos.to(DEV), w.to(DEV)).double().cpu().view(T, D)
    angles = [[exact_angle(p, f) for f in w.tolist()] for p in pos.tolist()]
    ref = torch.tensor([[math.cos(a) for a in row] + [math.sin(a) for a in row] for row in angles], dtype=torch.float64)
    assert ref.abs()[ref != 0].min() < 1e-4
    bad = (out - ref).abs() / (6 * 2.0 ** -24 * ref.abs() + 2.0 ** -44)
    assert bad.max().item() <= 1.0, bad.max().item()


SHORT = [(2, 2, 64, 64), (3, 3, 128, 128), (5, 2, 40, 72), (8, 2, 256, 96), (6, 2, 83, 35)]


@pytest.mark.parametrize('T,H,Dk,Dv', SHORT)
def test_bf16_state_and_its_gradient_have_fp32_accuracy(T, H, Dk, Dv):
    """A few tokens, decays well below one, no state in front: every term is decay x value as three bfloat16 values (2^-24 of it), a product and a sum in fp32; the decays'
    exponents are off by 2^-23 of themselves, at most half of a term for what still weighs.  (Two values, 2^-17, are four to six times over this bound.)"""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(T)
    B = 3
    q, k, v, do = rnd(g, T, B, H, Dk, dtype=BF), rnd(g, T, B, H, Dk, dtype=BF), rnd(g, T, B, H, Dv, dtype=BF), rnd(g, T, B, H, Dv, dtype=BF)
    ld, sc = torch.linspace(-0.15, -0.8, H, device=DEV), Dk ** -0.5
    new = t.linear_attention(q, k, v, ld, return_state=True)[1]
    within(new, *state_sum(k, v, ld, None, None), torch.float32, (T + 16) * 2.0 ** -24, 'state')
    ds = t.linear_attention_backward(do, q, k, v, ld, state=torch.zeros(B, H, Dk, Dv, device=DEV))[3]
    within(ds, *state_sum(q, do, ld, None, None, scale=sc, from_end=False, off=1), torch.float32, (T + 18) * 2.0 ** -24, 'dstate')


def test_norm_weight_gradient_sums_in_pairs():
    """2048 equal rows: 2048 times the gradient of one, but for the sum of four rows a workgroup holds (two roundings); everything behind it adds equal numbers in pairs,
    which is exact.  One behind the other the workgroups' sums are several times over this."""
    from srvp_amd import temporal as t
    g = torch.Generator().manual_seed(17)
    M, N = 2048, 256
    x, w, dy = rnd(g, 1, N), rnd(g, N), rnd(g, 1, N)
    one = t.rms_norm_backward(dy, x, w)[1].double()
    many = t.rms_norm_backward(dy.expand(M, N), x.expand(M, N), w)[1].double()
    assert ((many - M * one).abs() / (M * one.abs())).max().item() <= 2.25 * 2.0 ** -24

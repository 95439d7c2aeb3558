"""
What the bfloat16 attention may round: its outputs to their own type, and nothing else to as few bits.  Short sequences behind a state, so that the bound counts a handful of
roundings and not the length of the sums.
"""
import pytest
import torch

from test_gpu_temporal import BF, DEV, decays, rnd, scan, within

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

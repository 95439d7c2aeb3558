"""Temporal operators, what needs no GPU: descriptor layouts, frequency tables, refusals."""
import ctypes as C
import math
import os
import subprocess
import tempfile

import pytest
import torch

from srvp_amd import _lib as L
from srvp_amd import temporal as t

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {'srvp_linear_attention_desc': L.LinearAttentionDesc, 'srvp_linear_attention_bwd_desc': L.LinearAttentionBwdDesc,
           'srvp_linear_attention_step_desc': L.LinearAttentionStepDesc, 'srvp_rotary_desc': L.RotaryDesc, 'srvp_rms_norm_desc': L.RmsNormDesc,
           'srvp_rms_norm_bwd_desc': L.RmsNormBwdDesc, 'srvp_linear_int8_desc': L.LinearInt8Desc}


def test_descriptors_match_the_header():
    """Size and the offset of every field."""
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "srvp_hip.h"\nint main(void){'
    mine = []
    for name, s in STRUCTS.items():
        src += f'printf("%zu ", sizeof({name}));' + ''.join(f'printf("%zu ", offsetof({name}, {f}));' for f, _ in s._fields_)
        mine += [C.sizeof(s)] + [getattr(s, f).offset for f, _ in s._fields_]
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, 'a.c'), 'w').write(src + 'return 0;}')
        subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), os.path.join(d, 'a.c'), '-o', os.path.join(d, 'a')])
        theirs = [int(x) for x in subprocess.check_output([os.path.join(d, 'a')]).split()]
    assert theirs == mine


def attention(T=8192, B=2, H=16, Dk=128, Dv=128, p=0, **kw):
    d = L.LinearAttentionDesc(T=T, B=B, H=H, Dk=Dk, Dv=Dv, q=p, k=p, v=p, o=p, log_decay=p)
    for k, v in dict(dict(scale=1.0), **kw).items():
        setattr(d, k, v)
    return d


def test_workspace_sizes():
    """Long sequences of few heads are cut into segments (a state each); many heads and short sequences are not."""
    ws = lambda T, B, H, backward, **kw: L.load().srvp_linear_attention_ws_bytes(C.byref(attention(T, B, H, **kw)), backward)
    assert ws(12, 192, 4, 0) == 0 and ws(12, 192, 4, 1) == 0 and ws(64, 1, 1, 0) == 0 and ws(0, 1, 1, 0) == 0 and ws(4096, 0, 2, 0) == 0 and ws(4096, 2, 0, 1) == 0
    assert ws(8192, 2, 16, 0) % (2 * 16 * 128 * 128 * 4) == 0 and ws(8192, 2, 16, 0) > 0
    assert ws(8192, 2, 16, 1) % (2 * 2 * 16 * 128 * 128 * 4) == 0 and ws(8192, 2, 16, 1) > 0
    assert ws(8192, 2, 16, 0, Dk=300) == -1 and b'256' in L.load().srvp_last_error()
    assert ws(8192, 2, 16, 0, scale=0.0) == -1 and ws(8192, 2, 16, 0, scale=math.inf) == -1 and ws(-1, 2, 16, 0) == -1


def test_c_entries_refuse_before_any_launch():
    """Null pointers, sizes and workspaces are turned into errors on the host."""
    lib, r = L.load(), C.byref
    assert lib.srvp_linear_attention_fwd(r(attention()), None) == 1
    assert lib.srvp_linear_attention_fwd(r(attention(p=16)), None) == 1 and b'workspace' in lib.srvp_last_error()
    assert lib.srvp_linear_attention_bwd(r(L.LinearAttentionBwdDesc(f=attention(p=16))), None) == 1
    for f in (lib.srvp_linear_attention_fwd, lib.srvp_linear_attention_bwd, lib.srvp_linear_attention_step, lib.srvp_rotary, lib.srvp_rms_norm,
              lib.srvp_rms_norm_bwd, lib.srvp_linear_int8):
        assert f(None, None) == 1
    two_rows = dict(q=16, k=16, v=16, o=16, log_decay=16, state=16, B=2, H=1, Dk=8, Dv=8, nslots=1, scale=1.0)
    assert lib.srvp_linear_attention_step(r(L.LinearAttentionStepDesc(**two_rows)), None) == 1 and b'2 rows for 1' in lib.srvp_last_error()
    five_pairs = dict(q=16, oq=16, positions=16, freq=16, T=1, B=1, Hq=1, D=8, pairs=5, magnitude=1.0)
    assert lib.srvp_rotary(r(L.RotaryDesc(**five_pairs)), None) == 1
    assert lib.srvp_rms_norm(r(L.RmsNormDesc(x=16, w=16, y=16, M=4, N=20000)), None) == 1
    assert lib.srvp_rms_norm_bwd(r(L.RmsNormBwdDesc(x=16, d_y=16, w=16, dx=16, dw=16, ws=16, M=4, N=64)), None) == 1 and b'workspace' in lib.srvp_last_error()
    wide = dict(x=16, w=16, x_scale=16, w_scale=16, y=16, M=1, N=1)
    assert lib.srvp_linear_int8(r(L.LinearInt8Desc(K=200000, **wide)), None) == 1 and lib.srvp_linear_int8(r(L.LinearInt8Desc(K=0, **wide)), None) == 1
    # more workgroups than a launch takes
    assert lib.srvp_linear_int8(r(L.LinearInt8Desc(K=16, **dict(wide, M=1, N=2 ** 30))), None) == 1 and b'too many' in lib.srvp_last_error()
    assert lib.srvp_linear_int8(r(L.LinearInt8Desc(K=16, **dict(wide, M=2 ** 20, N=2 ** 20))), None) == 1 and b'too many' in lib.srvp_last_error()
    assert lib.srvp_linear_int8(r(L.LinearInt8Desc(K=16, **dict(wide, M=2 ** 31 - 1, N=1))), None) == 1 and b'too many' in lib.srvp_last_error()
    assert lib.srvp_linear_attention_step(r(L.LinearAttentionStepDesc(**dict(two_rows, B=2 ** 20, H=16, nslots=2 ** 20))), None) == 1
    many = dict(q=16, oq=16, positions=16, freq=16, T=2 ** 26, B=1, Hq=1, D=4096, pairs=2048, magnitude=1.0)
    assert lib.srvp_rotary(r(L.RotaryDesc(**many)), None) == 1 and b'too many' in lib.srvp_last_error()
    assert lib.srvp_linear_attention_fwd(r(attention(scale=1e-35, p=16)), None) == 1 and b'scale' in lib.srvp_last_error()


def test_no_cpu_path():
    x = torch.zeros(2, 1, 1, 4)
    for f in (lambda: t.linear_attention(x, x, x, torch.zeros(1)), lambda: t.linear_attention_step(x[0], x[0], x[0], torch.zeros(1), torch.zeros(1, 1, 4, 4)),
              lambda: t.rotary(x, None, torch.arange(2), t.rotary_frequencies(4)), lambda: t.rms_norm(x, torch.ones(4)),
              lambda: t.rms_norm_int8(x, torch.ones(4)), lambda: t.quantize_int8(x),
              lambda: t.linear_int8(x.to(torch.int8), torch.ones(2, 1, 1), torch.zeros(3, 4, dtype=torch.int8), torch.ones(3))):
        with pytest.raises(L.SrvpHipError):
            f()


def test_rotary_frequencies():
    w = t.rotary_frequencies(8)
    assert w.dtype == torch.float64 and torch.allclose(w, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(t.rotary_frequencies(8, method='linear', factor=4.0), w / 4)
    b = t.rotary_frequencies(8, method='base', factor=4.0)
    assert abs(b[0] - 1) < 1e-15 and abs(b[3] / w[3] - 0.25) < 1e-12
    p = t.rotary_frequencies(8, method='parts', factor=4.0, trained=4096)          # turns in 4096 positions: 652, 65, 6.5, 0.65
    assert torch.equal(p[:2], w[:2]) and p[3] == w[3] / 4 and w[2] / 4 < p[2] < w[2]
    assert t.rotary_frequencies(0).numel() == 0
    for bad in (dict(features=7), dict(features=8, method='other'), dict(features=8, factor=0.0), dict(features=8, method='parts', fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            t.rotary_frequencies(**bad)


def test_decay_rates():
    d = t.decay_rates(4, 8, 512)
    assert d.shape == (4,) and torch.allclose(torch.exp(d.double()), 1 - 1 / torch.tensor([8.0, 32, 128, 512], dtype=torch.float64), atol=1e-7)
    assert t.decay_rates(1, 4, 16).exp().item() == pytest.approx(1 - 1 / 8, abs=1e-6)
    with pytest.raises(ValueError):
        t.decay_rates(2, 1.0, 5.0)


def test_posterior_option():
    """The attention posterior is asked for by name; without it the model, its state and its options are the reference's."""
    import srvp_amd
    from srvp_amd import args
    ctor = (64, 1, 4, 8, 3, 3, False, 2, 24, 3, 16, 4, 'dcgan')
    m = srvp_amd.StochasticLatentResidualVideoPredictor(*ctor, posterior='attention', posterior_heads=3)
    assert [k for k in m.state_dict() if k.startswith('inf_z.')] == ['inf_z.inp.weight', 'inf_z.inp.bias', 'inf_z.norm.weight', 'inf_z.qkv.weight',
                                                                     'inf_z.out_norm.weight', 'inf_z.out.weight', 'inf_z.last_norm.weight']
    assert m.inf_z.heads == 3 and m.inf_z.width == 8 and 'inf_z.weight_hh_l0' in srvp_amd.StochasticLatentResidualVideoPredictor(*ctor).state_dict()
    for bad in (dict(posterior='other'), dict(posterior='attention', posterior_heads=5), dict(posterior='attention', posterior_heads=0), dict(posterior_heads=3)):
        with pytest.raises(ValueError):
            srvp_amd.StochasticLatentResidualVideoPredictor(*ctor, **bad)
    req = ['--save_path', 'x', '--ny', '2', '--nz', '2', '--nt_inf', '2', '--dataset', 'smmnist', '--data_dir', 'd', '--seq_len', '5', '--nc', '1', '--nt_cond', '2']
    p = args.create_args()
    assert 'posterior' not in vars(p.parse_args(req))
    o = vars(p.parse_args(req + ['--posterior', 'attention', '--posterior_heads', '4']))
    assert o['posterior'] == 'attention' and o['posterior_heads'] == 4
    with pytest.raises(SystemExit):
        p.parse_args(req + ['--posterior', 'other'])


def test_rotary_in_place_is_refused():
    """Threads share features at the end of a head: an output over its input would turn them twice."""
    one = dict(q=16, oq=32, positions=16, freq=16, T=1, B=1, Hq=1, D=8, pairs=4, magnitude=1.0)
    for same in (dict(oq=16), dict(k=64, ok=64, Hk=1)):
        assert L.load().srvp_rotary(C.byref(L.RotaryDesc(**dict(one, **same))), None) == 1 and b'in the place' in L.load().srvp_last_error()


def test_posterior_weights_of_another_number_of_heads_are_refused(tmp_path):
    """No parameter's shape tells the heads apart: the decays do, through every way a state dict travels; weights saved before they were in it come with a warning."""
    import warnings
    import srvp_amd
    from srvp_amd.posterior import AttentionPosterior
    torch.manual_seed(0)
    three, two = AttentionPosterior(8, 24, 3), AttentionPosterior(8, 24, 2)
    with pytest.raises(RuntimeError, match='size mismatch for log_decay'):
        two.load_state_dict(three.state_dict())
    ctor = (64, 1, 4, 8, 3, 3, False, 2, 24, 3, 16, 4, 'dcgan')
    make = lambda heads: srvp_amd.StochasticLatentResidualVideoPredictor(*ctor, posterior='attention', posterior_heads=heads)
    a = make(3)
    a.inf_z.log_decay[1] = -0.25                       # (decays travel as values)
    path = tmp_path / 'model.pt'
    torch.save(dict(model=a.state_dict()), path)
    ways = {'itself': a.state_dict(), 'plain': {k: v.clone() for k, v in a.state_dict().items()}, 'file': torch.load(path, weights_only=True)['model']}
    for way, sd in ways.items():
        with pytest.raises(RuntimeError, match='size mismatch for inf_z.log_decay'):
            make(2).load_state_dict(sd)
        b = make(3)
        assert str(b.load_state_dict(sd)) == '<All keys matched successfully>', way
        for (k, x), (l, y) in zip(a.state_dict().items(), b.state_dict().items()):
            assert k == l and torch.equal(x, y)
        assert b.inf_z.log_decay[1] == -0.25
    inside = torch.nn.Sequential(a)
    assert '0.posterior_log_decay' in inside.state_dict()
    torch.nn.Sequential(make(3)).load_state_dict(inside.state_dict())
    with pytest.raises(RuntimeError, match='size mismatch'):
        torch.nn.Sequential(make(2)).load_state_dict(inside.state_dict())
    missing = {k: v for k, v in a.state_dict().items() if k != 'posterior_log_decay'}
    with pytest.raises(RuntimeError, match='Missing key'):
        make(3).load_state_dict(missing)
    # the form without the decays
    old = a.state_dict()
    del old['posterior_log_decay']
    old._metadata['inf_z']['version'] = 1
    c = make(3)
    with pytest.warns(UserWarning, match='number of heads'):
        c.load_state_dict(old)
    assert torch.equal(c.inf_z.qkv.weight, a.inf_z.qkv.weight) and torch.equal(c.inf_z.log_decay, t.decay_rates(3))
    # the LSTM's state dict is the reference's
    lstm = srvp_amd.StochasticLatentResidualVideoPredictor(*ctor)
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        lstm.load_state_dict(lstm.state_dict())
    assert not any('decay' in k for k in lstm.state_dict())


def test_posterior_constants_keep_their_types():
    """Casts of the model, one after another, leave the decays and frequencies as they are."""
    from srvp_amd.posterior import AttentionPosterior
    net = torch.nn.Sequential(AttentionPosterior(8, 24, 3))
    ld, fr = t.decay_rates(3), t.rotary_frequencies(8)
    for cast in (lambda: net.half(), lambda: net.float(), lambda: net.bfloat16(), lambda: net.double(), lambda: net.to(torch.float32), lambda: net.float().double().float()):
        cast()
        a, b = net[0]._constants()
        assert a.dtype is torch.float32 and b.dtype is torch.float64 and torch.equal(a, ld) and torch.equal(b, fr)
    net[0].log_decay.fill_(-0.5)
    net.half().float()
    assert (net[0].log_decay == -0.5).all()
    with torch.device('meta'):
        far = AttentionPosterior(8, 24, 3)
    far.to_empty(device='cpu')
    assert torch.equal(far.log_decay, ld) and torch.equal(far.frequencies, fr)


def test_step_refuses_rows_without_bound():
    """The search through the slots grows with the square of the rows: where it would hold the GPU for minutes the call is refused, on the host."""
    one = dict(q=16, k=16, v=16, o=16, log_decay=16, state=16, slots=16, H=1, Dk=8, Dv=8, nslots=2 ** 24, scale=1.0)
    for B in (65537, 2 ** 23):
        assert L.load().srvp_linear_attention_step(C.byref(L.LinearAttentionStepDesc(**dict(one, B=B))), None) == 1 and b'65536 rows' in L.load().srvp_last_error()

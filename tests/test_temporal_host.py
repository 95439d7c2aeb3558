"""Temporal operators, what needs no GPU: descriptor layouts, frequency tables, refusals."""
import ctypes as C
import math
import os
import re
import subprocess
import tempfile

import pytest
import torch

from srvp_amd import _lib as L
from srvp_amd import temporal as t

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {'srvp_linear_attention_desc': t.ATTENTION, 'srvp_linear_attention_bwd_desc': t.ATTENTION_BWD, 'srvp_linear_attention_step_desc': t.STEP,
           'srvp_rotary_desc': t.ROTARY, 'srvp_rms_norm_desc': t.NORM, 'srvp_rms_norm_bwd_desc': t.NORM_BWD, 'srvp_linear_int8_desc': t.INT8}


def test_packed_descriptors_match_the_header():
    """Sizes, and that no padding lies between the fields (a packed string has none)."""
    names = list(STRUCTS)
    src = '#include <stdio.h>\n#include "srvp_hip.h"\nint main(void){' + ''.join(f'printf("%zu\\n", sizeof({n}));' for n in names) + 'return 0;}'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, 'a.c'), 'w').write(src)
        subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), os.path.join(d, 'a.c'), '-o', os.path.join(d, 'a')])
        sizes = [int(x) for x in subprocess.check_output([os.path.join(d, 'a')]).split()]
    assert sizes == [STRUCTS[n].size for n in names]
    for s in STRUCTS.values():
        assert s.size == sum(C.sizeof({'Q': C.c_uint64, 'q': C.c_int64, 'i': C.c_int32, 'f': C.c_float}[c]) * int(n or 1)
                             for n, c in re.findall(r'(\d*)([Qqif])', s.format))


def test_workspace_sizes():
    """Long sequences of few heads are cut into segments (a state each); many heads and short sequences are not."""
    def ws(T, B, H, backward, Dk=128, Dv=128, f32=0, scale=1.0):
        return L.load().srvp_linear_attention_ws_bytes(t.ATTENTION.pack(*([0] * 20), 0, 0, T, B, H, Dk, Dv, scale, f32, 0), backward)
    assert ws(12, 192, 4, 0) == 0 and ws(12, 192, 4, 1) == 0 and ws(64, 1, 1, 0) == 0 and ws(0, 1, 1, 0) == 0 and ws(4096, 0, 2, 0) == 0 and ws(4096, 2, 0, 1) == 0
    assert ws(8192, 2, 16, 0) % (2 * 16 * 128 * 128 * 4) == 0 and ws(8192, 2, 16, 0) > 0
    assert ws(8192, 2, 16, 1) % (2 * 2 * 16 * 128 * 128 * 4) == 0 and ws(8192, 2, 16, 1) > 0
    assert ws(8192, 2, 16, 0, Dk=300) == -1 and b'256' in L.load().srvp_last_error()
    assert ws(8192, 2, 16, 0, scale=0.0) == -1 and ws(8192, 2, 16, 0, scale=math.inf) == -1 and ws(-1, 2, 16, 0) == -1


def test_c_entries_refuse_before_any_launch():
    """Null pointers, sizes and workspaces are turned into errors on the host."""
    lib = L.load()
    att = lambda ws=0, T=8192, D=128, p=0: t.ATTENTION.pack(*([p] * 4), *([0] * 12), p, 0, 0, 0, 0, ws, T, 1, 1, D, D, 1.0, 0, 0)
    assert lib.srvp_linear_attention_fwd(att(), None) == 1
    assert lib.srvp_linear_attention_fwd(att(p=16), None) == 1 and b'workspace' in lib.srvp_last_error()
    assert lib.srvp_linear_attention_bwd(att(p=16) + bytes(t.ATTENTION_BWD.size - t.ATTENTION.size), None) == 1
    assert lib.srvp_linear_attention_fwd(None, None) == 1 and lib.srvp_linear_attention_bwd(None, None) == 1 and lib.srvp_linear_attention_step(None, None) == 1
    assert lib.srvp_linear_attention_step(t.STEP.pack(*([16] * 4), *([0] * 8), 16, 16, 0, 2, 1, 8, 8, 1, 1.0, 0, 0), None) == 1      # 2 rows, 1 state
    assert lib.srvp_rotary(None, None) == 1 and lib.srvp_rms_norm(None, None) == 1 and lib.srvp_rms_norm_bwd(None, None) == 1 and lib.srvp_linear_int8(None, None) == 1
    assert lib.srvp_rotary(t.ROTARY.pack(*([16] * 4), *([0] * 12), 16, 0, 0, 16, 1, 1, 1, 1, 8, 5, 0, 0, 1.0, 0), None) == 1           # 5 pairs of 8 features
    assert lib.srvp_rms_norm(t.NORM.pack(*([16] * 7), *([0] * 5), 4, 20000, 0.0, 0, 0), None) == 1
    assert lib.srvp_rms_norm_bwd(t.NORM_BWD.pack(*([16] * 8), *([0] * 5), 4, 0, 64, 0.0, 0, 0), None) == 1 and b'workspace' in lib.srvp_last_error()
    assert lib.srvp_linear_int8(t.INT8.pack(*([16] * 6), 0, 0, 0, 1, 1, 200000, 1), None) == 1


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

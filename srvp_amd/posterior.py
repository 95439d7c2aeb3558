"""
The posterior network over frame encodings as one causal attention block, the alternative to the LSTM of reference module/srvp.py:130,366
(`StochasticLatentResidualVideoPredictor(..., posterior='attention')`): every frame of a sequence is processed at once instead of one after another, and
a single new frame costs one update of a state (`PosteriorStream`).

    u = W_in hx + b      n = norm(u)      (q, k, v) = W_qkv n, q and k turned by their frame's position
    o = linear attention with a decay for each head       z = W_out norm(o)       hz = norm(u + z)

fp32 like the rest of the latent path; for inference the two inner products can run on 8-bit integers (`quantize`).
"""
import warnings

import torch
import torch.nn as nn

from . import _lib as L
from . import temporal


def default_heads(nh):
    """Heads of 64 features where they divide the width, one head otherwise."""
    return nh // 64 if nh % 64 == 0 else 1


def _empty(like, *shape):
    """fp32, which is what the launches write, whatever torch's default type is."""
    return torch.empty(*shape, dtype=torch.float32, device=like.device)


def _taken(x):
    """x, if the products can take it: float32, one row behind the other."""
    if x.dtype is not torch.float32 or not x.is_contiguous():
        raise TypeError(f'posterior attention: contiguous float32 encodings and weights, got {x.dtype} {tuple(x.shape)} with strides {x.stride()}')
    return x


class _Scale(nn.Module):
    """Parameter container of a row norm."""

    def __init__(self, n):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(n))


class AttentionPosterior(nn.Module):
    """Parameter container (like every module of the model, its forward is never called): decays and frequencies are constants.  The decays, one a head, are part of the
    state dict: no parameter's shape tells the number of heads, and weights of another number are refused by their length."""

    _version = 2                                       # 1: without the decays

    def __init__(self, nhx, nh, heads=None):
        super().__init__()
        heads = default_heads(nh) if heads is None else int(heads)
        if heads < 1 or nh % heads or nh // heads > 256:
            raise ValueError(f'posterior attention: {nh} features in {heads} heads (heads of at most 256 features)')
        self.heads, self.width = heads, nh // heads
        self.inp = nn.Linear(nhx, nh)
        self.norm = _Scale(nh)
        self.qkv = nn.Linear(nh, 3 * nh, bias=False)
        self.out_norm = _Scale(nh)
        self.out = nn.Linear(nh, nh, bias=False)
        self.last_norm = _Scale(nh)
        self.register_buffer('log_decay', temporal.decay_rates(heads))
        self.register_buffer('frequencies', temporal.rotary_frequencies(self.width // 2 * 2), persistent=False)
        self._eight_bits = False

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, *args):
        if prefix + 'log_decay' not in state_dict and local_metadata.get('version') == 1:
            warnings.warn(f'srvp_amd: weights of an attention posterior that were saved without its number of heads: taken for {self.heads}')
            state_dict[prefix + 'log_decay'] = self.log_decay
        super()._load_from_state_dict(state_dict, prefix, local_metadata, *args)

    def _apply(self, fn, *args, **kw):
        # the constants follow the model to its device and keep their types and values: .half() or .float() would round them for good
        ld, fr = self.log_decay, self.frequencies
        r = super()._apply(fn, *args, **kw)
        dev = self.log_decay.device
        if ld.is_meta and dev.type != 'meta':
            ld, fr = temporal.decay_rates(self.heads), temporal.rotary_frequencies(self.width // 2 * 2)
        self.log_decay, self.frequencies = ld.to(dev), fr.to(dev)
        return r

    def _constants(self):
        return self.log_decay, self.frequencies

    # ---- 8-bit inference
    def quantize(self):
        """The two inner products on 8-bit integers, for the inference calls from here on (dropped by the next training pass)."""
        self._eight_bits = True

    def drop_quantized(self):
        self._eight_bits = False

    @torch.no_grad()
    def quantized(self):
        """None, or the two inner weights in 8 bits as they are now (w, scales of its rows), and the weights these stand for.  Formed anew for every call (one launch a
        weight): the fused optimizer and writes through .data leave nothing by which a kept copy would know that it is old."""
        if not self._eight_bits:
            return None
        w = self.qkv.weight, self.out.weight
        return temporal.quantize_int8(w[0]), temporal.quantize_int8(w[1]), w

    # ---- the block
    def _project(self, x, weight, out):
        from .latent import linear_fwd
        return linear_fwd(L.stream(), x, _taken(weight), None, out)

    def _inputs(self, hx, q8):
        """hx (rows, nhx), contiguous -> u, norm(u) (None in 8 bits), (rows, 3 nh)."""
        from .latent import linear_fwd
        inp = self.inp
        w = _taken(inp.weight)
        if hx.shape[-1] != w.shape[1] or hx.device != w.device:
            raise ValueError(f'posterior attention: encodings of {w.shape[1]} features on {w.device}, got {tuple(hx.shape)} on {hx.device}')
        u = _empty(hx, hx.shape[0], self.heads * self.width)
        linear_fwd(L.stream(), _taken(hx), w, inp.bias, u)
        if q8 is not None:
            return u, None, temporal.linear_int8(*temporal.rms_norm_int8(u, self.norm.weight), *q8[0])
        n = temporal.rms_norm(u, self.norm.weight)
        return u, n, self._project(n, self.qkv.weight, _empty(hx, hx.shape[0], 3 * u.shape[1]))

    def _outputs(self, o, u, q8):
        """Attention's output (rows, nh) and u -> norm(o) (None in 8 bits), z, hz."""
        if q8 is not None:
            m, z = None, temporal.linear_int8(*temporal.rms_norm_int8(o, self.out_norm.weight), *q8[1])
        else:
            m = temporal.rms_norm(o, self.out_norm.weight)
            z = self._project(m, self.out.weight, torch.empty_like(o))
        return m, z, temporal.rms_norm(z, self.last_norm.weight, residual=u)[0]

    @torch.no_grad()
    def run(self, hx, training):
        """hx (T, B, nhx) float32 -> hz (T * B, nh) and, in training, what `backward` needs."""
        T, B = hx.shape[0], hx.shape[1]
        if training:
            self.drop_quantized()
        q8 = None if training else self.quantized()
        ld, fr = self._constants()
        u, n, qkv = self._inputs(hx.reshape(T * B, -1).contiguous(), q8)      # (rows of a slice may lie apart: the products take whole ones)
        q, k, v = qkv.view(T, B, 3, self.heads, self.width).unbind(2)
        pos = torch.arange(T, device=hx.device)
        q, k = temporal.rotary(q, k, pos, fr)
        o = temporal.linear_attention(q, k, v, ld).view(T * B, -1)
        m, z, hz = self._outputs(o, u, q8)
        return hz, ((u, n, q, k, v, pos, o, m, z) if training else None)

    @torch.no_grad()
    def backward(self, hx, d_hz, saved, grads, prefix, d_hx, defer=None):
        """Gradients of `run` for d_hz (T * B, nh): parameters' into `grads` (names under `prefix`), the input's added to d_hx.  Returns what the deferred
        weight-gradient launches still read (to be kept until they are done)."""
        from .latent import axpby, linear_bwd
        st = L.stream()
        u, n, q, k, v, pos, o, m, z = saved
        ld, fr = self._constants()
        R = u.shape[0]

        def add(name, g):
            axpby(st, grads[f'{prefix}.{name}.weight'], 1.0, grads[f'{prefix}.{name}.weight'], 1.0, g)
        d_zu, dw = temporal.rms_norm_backward(d_hz, z, self.last_norm.weight, residual=u)       # the gradient of z, and u's share of it
        add('last_norm', dw)
        d_m = torch.empty_like(m)
        linear_bwd(st, m, self.out.weight, d_zu, grads[f'{prefix}.out.weight'], None, dx=d_m, defer=defer)
        d_o, dw = temporal.rms_norm_backward(d_m, o, self.out_norm.weight)
        add('out_norm', dw)
        d_q, d_k, d_v, _ = temporal.linear_attention_backward(d_o.view(v.shape), q, k, v, ld)
        d_q, d_k = temporal.rotary(d_q, d_k, pos, fr, back=True)
        d_qkv = torch.stack([d_q, d_k, d_v], 2).view(R, -1)
        d_n = torch.empty_like(n)
        linear_bwd(st, n, self.qkv.weight, d_qkv, grads[f'{prefix}.qkv.weight'], None, dx=d_n, defer=defer)
        d_u, dw = temporal.rms_norm_backward(d_n, u, self.norm.weight, d_sum=d_zu)
        add('norm', dw)
        x = hx.reshape(R, -1).contiguous()
        linear_bwd(st, x, self.inp.weight, d_u, grads[f'{prefix}.inp.weight'], grads[f'{prefix}.inp.bias'], dx=d_hx, dx_acc=1, defer=defer)
        return x, d_zu, d_qkv, d_u, saved


class PosteriorStream:
    """The posterior of `rows` live videos, one frame at a time: what `model.encode` gives for a new frame -> (hz, q_z parameters), the same values as those
    of the whole sequence at that frame.  Keeps one state (heads, width, width) a row."""

    def __init__(self, net, q_z, rows, device):
        self.net, self.q_z = net, q_z
        self.state = torch.zeros(rows, net.heads, net.width, net.width, dtype=torch.float32, device=device)
        self.position = torch.zeros(1, rows, dtype=torch.int64, device=device)

    def reset(self, rows=None):
        """Starts the given rows (indices; None: all) over."""
        if rows is None:
            rows = slice(None)
        self.state[rows] = 0
        self.position[0, rows] = 0

    @torch.no_grad()
    def step(self, hx):
        from .latent import linear_fwd
        net, B = self.net, hx.shape[0]
        if hx.dim() != 2 or B != self.state.shape[0]:
            raise ValueError(f'PosteriorStream.step: the encodings of one frame of all {self.state.shape[0]} rows, got {tuple(hx.shape)}')
        ld, fr = net._constants()
        q8 = net.quantized()
        u, _, qkv = net._inputs(hx.contiguous().float(), q8)
        q, k, v = qkv.view(1, B, 3, net.heads, net.width).unbind(2)
        q, k = temporal.rotary(q, k, self.position, fr)
        o = temporal.linear_attention_step(q[0], k[0], v[0], ld, self.state).view(B, -1)
        self.position += 1
        hz = net._outputs(o, u, q8)[2]
        p = _empty(hz, B, self.q_z.weight.shape[0])
        linear_fwd(L.stream(), hz, self.q_z.weight, self.q_z.bias, p)
        return hz, p

"""
Operators over the time axis, the parallel counterpart of the posterior LSTM (reference module/srvp.py:130,366): linear attention with a decay for
each head (chunked form for whole sequences, recurrent form for single frames), rotary positions, the root-mean-square norm with the residual's
addition, and products on 8-bit integers for inference.  `posterior.AttentionPosterior` is the network built of them.

Tensors are time-major, (T, B, heads, features), float32 or bfloat16; any strides are taken as they are (features contiguous, otherwise the tensor is
copied first), so a batch-major tensor is passed as a transposed view and shared heads as an expanded one.  Every sum, state and norm is held in 32
bits or more.  Launches go to torch's current stream on the tensors' device; workspaces are ordinary tensors of the call.

Gradients: `linear_attention`, `rotary` and `rms_norm` are autograd nodes.  Inside a stream capture they record none (a captured backward pass cannot be
told apart from the eager one of the same leaves) and raise: call `linear_attention_backward`, `rotary(..., back=True)`, `rms_norm_backward` there.
"""
import math
import struct

import torch

from . import _lib as L

F32, BF16 = torch.float32, torch.bfloat16

# The descriptors of include/srvp_hip.h, packed in one call each (a ctypes structure of 30 fields costs more host time than the smallest kernels take).
ATTENTION = struct.Struct('4Q12q4QQq5if2i')
ATTENTION_BWD = struct.Struct('4Q12q4QQq5if2i' + '4Q12q2Q')
STEP = struct.Struct('4Q8q3Q5if2i')
ROTARY = struct.Struct('4Q12qQ2qQ8ifi')
NORM = struct.Struct('7Q6qifii')
NORM_BWD = struct.Struct('8Q7qifii')
INT8 = struct.Struct('6Q3q4i')


# ------------------------------------------------------------------------------------------------------------------------- checks
def _device(x, what):
    i = x.get_device()
    if i < 0:
        raise L.SrvpHipError(f'{what}: srvp_amd runs on an MI355X only: move the tensors to the GPU; there is no CPU compute path')
    return i


def _launch(i, name, packed):
    """`name` on torch's current stream of device i."""
    if i == L._get_dev():
        L.call(name, packed, L._raw_stream(i))
    else:
        with torch.cuda.device(i):
            L.call(name, packed, L._raw_stream(i))


def _floats(what, *ts):
    d = ts[0].dtype
    if d is not F32 and d is not BF16:
        raise TypeError(f'{what}: float32 or bfloat16 tensors, got {d}')
    for t in ts[1:]:
        if t.dtype is not d:
            raise TypeError(f'{what}: tensors of one type, got {d} and {t.dtype}')


def _same_device(what, i, *ts):
    for t in ts:
        if t is not None and t.get_device() != i:
            raise ValueError(f'{what}: all tensors on one device')


def _inner(x):
    """x with contiguous features."""
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _decay(what, log_decay, H):
    if log_decay.dtype is not F32 or log_decay.shape != (H,):
        raise ValueError(f'{what}: log_decay is a float32 tensor of one value a head ({H}), got {tuple(log_decay.shape)} {log_decay.dtype}')
    if log_decay.requires_grad:
        raise ValueError(f'{what}: the decays are constants: log_decay must not require a gradient')
    return log_decay.contiguous()


def _state(what, state, shape):
    if state.dtype is not F32 or tuple(state.shape) != shape:
        raise ValueError(f'{what}: state is a float32 tensor {shape}, got {tuple(state.shape)} {state.dtype}')
    return state.contiguous()


def _whole(what, x, name):
    if x.dtype is torch.int64:
        return x
    if x.dtype is torch.int32:
        return x.long()
    raise TypeError(f'{what}: {name} is an int64 or int32 tensor, got {x.dtype}')


def _records(what, *ts):
    """Whether the call is to be recorded for autograd."""
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in ts):
        return False
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f'{what}: no gradient is recorded inside a stream capture; detach the inputs and call the backward function itself')
    return True


def _no_gradient(what, *ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError(f'{what}: an inference operator: call it under torch.no_grad() or with detached tensors')


# --------------------------------------------------------------------------------------------------------------- linear attention
def decay_rates(heads, shortest=8.0, longest=512.0, device=None):
    """log_decay (heads,) float32 of memories that are `shortest` to `longest` frames long, spread evenly in their logarithm: decay 1 - 1/length."""
    if not 1.0 < shortest <= longest:
        raise ValueError('decay_rates: 1 < shortest <= longest')
    n = torch.linspace(math.log(shortest), math.log(longest), heads, dtype=torch.float64) if heads > 1 else torch.tensor([0.5 * math.log(shortest * longest)], dtype=torch.float64)
    return torch.log1p(-torch.exp(-n)).to(torch.float32).to(device)


def _attention_args(what, q, k, v, log_decay, state, lengths, scale):
    i = _device(q, what)
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:3] != q.shape[:3]:
        raise ValueError(f'{what}: q, k (T, B, H, Dk) and v (T, B, H, Dv), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    _floats(what, q, k, v)
    T, B, H, Dk = q.shape
    Dv = v.shape[3]
    if not (1 <= Dk <= 256 and 1 <= Dv <= 256):
        raise ValueError(f'{what}: heads of 1 to 256 features, got {Dk} and {Dv}')
    log_decay = _decay(what, log_decay, H)
    if state is not None:
        state = _state(what, state, (B, H, Dk, Dv))
    if lengths is not None:
        if lengths.shape != (B,):
            raise ValueError(f'{what}: one length a sequence ({B}), got {tuple(lengths.shape)}')
        lengths = _whole(what, lengths, 'lengths').contiguous()
    _same_device(what, i, k, v, log_decay, state, lengths)
    scale = Dk ** -0.5 if scale is None else float(scale)
    if scale == 0.0 or not math.isfinite(scale):
        raise ValueError(f'{what}: scale must be finite and not zero')
    return i, _inner(q), _inner(k), _inner(v), log_decay, state, lengths, scale


def _pack_attention(q, k, v, o, log_decay, state, new_state, lengths, ws, nws, scale):
    T, B, H, Dk = q.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    os_ = (0, 0, 0) if o is None else o.stride()
    return (q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if o is None else o.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
            os_[0], os_[1], os_[2], log_decay.data_ptr(), 0 if state is None else state.data_ptr(), 0 if new_state is None else new_state.data_ptr(),
            0 if lengths is None else lengths.data_ptr(), 0 if ws is None else ws.data_ptr(), nws, T, B, H, Dk, v.shape[3], scale,
            1 if q.dtype is F32 else 0, 0)


def _workspace(args, backward, device):
    n = L.load().srvp_linear_attention_ws_bytes(ATTENTION.pack(*args), backward)
    if n < 0:
        L.check(1, 'srvp_linear_attention_ws_bytes')
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


def _attention_fwd(i, q, k, v, log_decay, state, lengths, scale, want_state):
    T, B, H, Dk = q.shape
    o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    new = torch.empty(B, H, Dk, v.shape[3], dtype=F32, device=v.device) if want_state else None
    args = _pack_attention(q, k, v, o, log_decay, state, new, lengths, None, 0, scale)
    ws, n = _workspace(args, 0, v.device)
    if n:
        args = args[:20] + (ws.data_ptr(), n) + args[22:]
    _launch(i, 'srvp_linear_attention_fwd', ATTENTION.pack(*args))
    return o, new


def _attention_bwd(i, d_out, q, k, v, log_decay, state, lengths, scale, d_new, want_state):
    dev = q.device
    d_out = _inner(d_out)
    dq, dk = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(q.shape, dtype=q.dtype, device=dev)
    dv = torch.empty(v.shape, dtype=v.dtype, device=dev)
    ds = torch.empty(q.shape[1], q.shape[2], q.shape[3], v.shape[3], dtype=F32, device=dev) if want_state else None
    args = _pack_attention(q, k, v, None, log_decay, state, None, lengths, None, 0, scale)
    ws, n = _workspace(args, 1, dev)
    if n:
        args = args[:20] + (ws.data_ptr(), n) + args[22:]
    gs, a, b = d_out.stride(), dq.stride(), dv.stride()
    _launch(i, 'srvp_linear_attention_bwd', ATTENTION_BWD.pack(
        *args, d_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), gs[0], gs[1], gs[2], a[0], a[1], a[2], a[0], a[1], a[2], b[0], b[1], b[2],
        0 if d_new is None else d_new.data_ptr(), 0 if ds is None else ds.data_ptr()))
    return dq, dk, dv, ds


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, i, q, k, v, log_decay, state, lengths, scale, want_state):
        o, new = _attention_fwd(i, q, k, v, log_decay, state, lengths, scale, want_state)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.i, ctx.scale = i, scale
        ctx.set_materialize_grads(False)
        return (o, new) if want_state else o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_new=None):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        if d_out is None:
            d_out = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        dq, dk, dv, ds = _attention_bwd(ctx.i, d_out, q, k, v, log_decay, state, lengths, ctx.scale, None if d_new is None else d_new.contiguous(),
                                        state is not None and ctx.needs_input_grad[5])
        return None, dq, dk, dv, None, ds, None, None, None


def linear_attention(q, k, v, log_decay, *, state=None, lengths=None, scale=None, return_state=False):
    """S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,  o_t = scale * q_t S_t, causal over the first axis.

    q, k (T, B, H, Dk), v (T, B, H, Dv), heads of 1 to 256 features; log_decay (H,) float32, normally <= 0 (-inf: no memory); state (B, H, Dk, Dv)
    float32: S in front of the first token (None: zero; it is not changed); lengths (B,): tokens of each sequence (outputs behind them are zero, values
    there are not read); scale: default Dk ** -0.5.  Returns o (T, B, H, Dv), or (o, new state) with return_state.  Gradients: q, k, v, state.
    A NaN or infinity in v or k reaches the outputs of the chunk (64 tokens, float32: 32) that its token lies in, and those behind it."""
    a = _attention_args('linear_attention', q, k, v, log_decay, state, lengths, scale)
    if _records('linear_attention', q, k, v, state):
        return _LinearAttention.apply(*a, return_state)
    o, new = _attention_fwd(*a, return_state)
    return (o, new) if return_state else o


def linear_attention_backward(d_out, q, k, v, log_decay, *, state=None, lengths=None, scale=None, d_state=None):
    """(dq, dk, dv, d_state_in) of linear_attention for the gradients d_out of o and d_state of the new state (None: not used); d_state_in is None
    without a state.  The explicit form of what autograd calls."""
    i, q, k, v, log_decay, state, lengths, scale = _attention_args('linear_attention_backward', q, k, v, log_decay, state, lengths, scale)
    _no_gradient('linear_attention_backward', d_out, q, k, v, state, d_state)
    if d_out.shape != v.shape:
        raise ValueError(f'linear_attention_backward: d_out {tuple(v.shape)}, got {tuple(d_out.shape)}')
    _floats('linear_attention_backward', q, d_out)
    if d_state is not None:
        d_state = _state('linear_attention_backward', d_state, (q.shape[1], q.shape[2], q.shape[3], v.shape[3]))
    _same_device('linear_attention_backward', i, d_out, d_state)
    return _attention_bwd(i, d_out, q, k, v, log_decay, state, lengths, scale, d_state, state is not None)


def linear_attention_step(q, k, v, log_decay, state, *, slots=None, scale=None):
    """One token of each of B sequences: q, k (B, H, Dk), v (B, H, Dv) -> o (B, H, Dv); state (slots, H, Dk, Dv) float32, contiguous, is advanced in place.
    slots (B,): where each row's state lies (None: row b has state b).  A slot outside the pool marks a padded row: its output is zero, no state is
    touched.  Rows that name the same slot are successive tokens of one sequence, in row order."""
    what = 'linear_attention_step'
    i = _device(q, what)
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f'{what}: q, k (B, H, Dk) and v (B, H, Dv), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    _floats(what, q, k, v)
    _no_gradient(what, q, k, v, state)
    B, H, Dk = q.shape
    Dv = v.shape[2]
    if not (1 <= Dk <= 256 and 1 <= Dv <= 256):
        raise ValueError(f'{what}: heads of 1 to 256 features, got {Dk} and {Dv}')
    log_decay = _decay(what, log_decay, H)
    if state.dtype is not F32 or state.dim() != 4 or state.shape[1:] != (H, Dk, Dv) or not state.is_contiguous():
        raise ValueError(f'{what}: state is a contiguous float32 tensor (slots, {H}, {Dk}, {Dv}), got {tuple(state.shape)} {state.dtype}')
    if slots is None:
        if B > state.shape[0]:
            raise ValueError(f'{what}: {B} rows for {state.shape[0]} states')
    else:
        if slots.shape != (B,):
            raise ValueError(f'{what}: one slot a row ({B}), got {tuple(slots.shape)}')
        slots = _whole(what, slots, 'slots').contiguous()
    _same_device(what, i, k, v, log_decay, state, slots)
    scale = Dk ** -0.5 if scale is None else float(scale)
    q, k, v = _inner(q), _inner(k), _inner(v)
    o = torch.empty(B, H, Dv, dtype=v.dtype, device=v.device)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    _launch(i, 'srvp_linear_attention_step', STEP.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], H * Dv, Dv, log_decay.data_ptr(),
        state.data_ptr(), 0 if slots is None else slots.data_ptr(), B, H, Dk, Dv, state.shape[0], scale, 1 if q.dtype is F32 else 0, 0))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)      # (changed behind autograd's back)
    return o


# ------------------------------------------------------------------------------------------------------------------------- rotary
def rotary_frequencies(features, base=10000.0, *, method='none', factor=1.0, trained=4096, fast=32.0, slow=1.0, device=None):
    """Radians a position of the features / 2 pairs, float64: base ** (-2p / features), and its forms for contexts `factor` times longer than those
    trained on: 'linear' divides every frequency by factor; 'base' raises the base so that the slowest pair turns factor times slower; 'parts' keeps the
    pairs that turn `fast` times or more within `trained` positions, divides those that turn `slow` times or less, and blends in between."""
    if features < 0 or features % 2:
        raise ValueError(f'rotary_frequencies: an even number of features, got {features}')
    if method not in ('none', 'linear', 'base', 'parts') or not factor > 0 or not base > 0:
        raise ValueError("rotary_frequencies: method 'none', 'linear', 'base' or 'parts', positive base and factor")
    if method == 'base' and features > 2:
        base = base * factor ** (features / (features - 2))
    w = base ** (-torch.arange(0, features, 2, dtype=torch.float64) / max(features, 1))
    if method == 'linear':
        w = w / factor
    if method == 'parts':
        if not fast > slow:
            raise ValueError('rotary_frequencies: fast > slow')
        keep = ((trained * w / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        w = w * keep + w / factor * (1 - keep)
    return w.to(device)


def _rotary(i, q, k, positions, frequencies, interleaved, back, magnitude):
    q = _inner(q)
    T, B, Hq, D = q.shape
    oq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    qs, oqs = q.stride(), oq.stride()
    if k is None:
        ok, Hk, kp, okp, ks, oks = None, 0, 0, 0, (0, 0, 0), (0, 0, 0)
    else:
        k = _inner(k)
        ok = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        Hk, kp, okp, ks, oks = k.shape[2], k.data_ptr(), ok.data_ptr(), k.stride(), ok.stride()
    _launch(i, 'srvp_rotary', ROTARY.pack(
        q.data_ptr(), kp, oq.data_ptr(), okp, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], oqs[0], oqs[1], oqs[2], oks[0], oks[1], oks[2],
        positions.data_ptr(), positions.stride(0), positions.stride(1) if positions.dim() == 2 else 0, frequencies.data_ptr(), T, B, Hq, Hk, D,
        frequencies.numel(), 1 if interleaved else 0, 1 if back else 0, magnitude, 1 if q.dtype is F32 else 0))
    return oq, ok


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, i, q, k, positions, frequencies, interleaved, back, magnitude):
        ctx.save_for_backward(positions, frequencies)
        ctx.rest, ctx.shapes = (i, interleaved, back, magnitude), (q.shape, None if k is None else k.shape, q.dtype)
        oq, ok = _rotary(i, q, k, positions, frequencies, interleaved, back, magnitude)
        ctx.set_materialize_grads(False)
        return oq if k is None else (oq, ok)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        positions, frequencies = ctx.saved_tensors
        i, interleaved, back, magnitude = ctx.rest
        none = (None,) * 8
        if dq is None and dk is None:
            return none
        if dq is None or dk is None:
            one, _ = _rotary(i, dq if dk is None else dk, None, positions, frequencies, interleaved, not back, magnitude)
            return (None, one, None) + none[3:] if dk is None else (None, None, one) + none[3:]
        gq, gk = _rotary(i, dq, dk, positions, frequencies, interleaved, not back, magnitude)
        return (None, gq, gk) + none[3:]


def rotary(q, k, positions, frequencies, *, interleaved=False, back=False, magnitude=1.0):
    """Turns the pairs of features of q (T, B, Hq, D) and, in the same launch, of k (T, B, Hk, D; None: q alone) by positions * frequencies radians.

    positions (T,) or (T, B), whole numbers of any size (angles are formed in 64 bits); frequencies float64 (pairs,) on the device, 2 * pairs <= D
    (rotary_frequencies): features behind the first 2 * pairs are passed on unchanged.  interleaved: pair p is features (2p, 2p + 1), otherwise
    (p, pairs + p).  magnitude multiplies the turned features.  back: the negative angle, which is the gradient's.  Returns q', or (q', k')."""
    what = 'rotary'
    i = _device(q, what)
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError(f'{what}: q (T, B, Hq, D) and k (T, B, Hk, D), got {tuple(q.shape)}' + ('' if k is None else f', {tuple(k.shape)}'))
    _floats(what, *((q,) if k is None else (q, k)))
    T, B, _, D = q.shape
    if D < 1:
        raise ValueError(f'{what}: heads of at least one feature')
    if positions.shape != (T,) and positions.shape != (T, B):
        raise ValueError(f'{what}: positions ({T},) or ({T}, {B}), got {tuple(positions.shape)}')
    positions = _whole(what, positions, 'positions')
    if frequencies.dtype is not torch.float64 or frequencies.dim() != 1 or 2 * frequencies.numel() > D or not frequencies.is_contiguous():
        raise ValueError(f'{what}: frequencies is a contiguous float64 tensor of at most {D // 2} pairs, got {tuple(frequencies.shape)} {frequencies.dtype}')
    _same_device(what, i, k, positions, frequencies)
    if _records(what, q, k):
        return _Rotary.apply(i, q, k, positions, frequencies, interleaved, back, float(magnitude))
    oq, ok = _rotary(i, q, k, positions, frequencies, interleaved, back, float(magnitude))
    return oq if k is None else (oq, ok)


# --------------------------------------------------------------------------------------------------------------------------- norm
def _norm_args(what, x, weight, residual):
    i = _device(x, what)
    _floats(what, *((x,) if residual is None else (x, residual)))
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise ValueError(f'{what}: rows of 1 to 16384 features, got {tuple(x.shape)}')
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f'{what}: residual {tuple(residual.shape)} for x {tuple(x.shape)}')
    if weight is not None and (weight.dtype is not F32 or weight.shape != x.shape[-1:]):
        raise ValueError(f'{what}: weight is a float32 tensor ({x.shape[-1]},), got {tuple(weight.shape)} {weight.dtype}')
    _same_device(what, i, weight, residual)
    return i


def _matrix(x):
    """(rows, features) with contiguous features."""
    return _inner(x.reshape(-1, x.shape[-1]))


def _norm_fwd(i, x, weight, residual, eps):
    N = x.shape[-1]
    x2, r2, w = _matrix(x), None if residual is None else _matrix(residual), weight.contiguous()
    M = x2.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch(i, 'srvp_rms_norm', NORM.pack(
        x2.data_ptr(), 0 if r2 is None else r2.data_ptr(), w.data_ptr(), y.data_ptr(), 0 if total is None else total.data_ptr(),
        0, 0, x2.stride(0), 0 if r2 is None else r2.stride(0), N, N, 0, M, N, eps, 1 if x.dtype is F32 else 0, 0))
    return y, total


def _norm_bwd(i, d_y, d_sum, x, weight, residual, eps):
    N = x.shape[-1]
    x2, y2, w = _matrix(x), _matrix(d_y), weight.contiguous()
    r2, t2 = None if residual is None else _matrix(residual), None if d_sum is None else _matrix(d_sum)
    M, f32 = x2.shape[0], 1 if x.dtype is F32 else 0
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if M == 0:
        return dx, torch.zeros(N, dtype=F32, device=x.device)
    dw = torch.empty(N, dtype=F32, device=x.device)
    n = L.load().srvp_rms_norm_bwd_ws_bytes(M, N, f32)
    ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    _launch(i, 'srvp_rms_norm_bwd', NORM_BWD.pack(
        x2.data_ptr(), 0 if r2 is None else r2.data_ptr(), y2.data_ptr(), 0 if t2 is None else t2.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(),
        ws.data_ptr(), x2.stride(0), 0 if r2 is None else r2.stride(0), y2.stride(0), 0 if t2 is None else t2.stride(0), N, M, n, N, eps, f32, 0))
    return dx, dw


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, i, x, weight, residual, eps):
        y, total = _norm_fwd(i, x, weight, residual, eps)
        ctx.i, ctx.eps = i, eps
        ctx.save_for_backward(x, weight, residual)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_sum=None):
        x, weight, residual = ctx.saved_tensors
        if d_y is None:
            return None, d_sum, None, None if residual is None else d_sum, None
        dx, dw = _norm_bwd(ctx.i, d_y, d_sum, x, weight, residual, ctx.eps)
        return None, dx, dw, None if residual is None else dx, None


def rms_norm(x, weight, *, residual=None, eps=1e-6):
    """y = h * weight / sqrt(mean(h^2) + eps) over the last axis, h = x + residual.  x, residual (..., N), N <= 16384; weight (N,) float32.  Returns y, or
    (y, h) with a residual (h rounded to x's type; y and the gradients are those of the unrounded sum).  Gradients: x, residual, weight."""
    i = _norm_args('rms_norm', x, weight, residual)
    if _records('rms_norm', x, weight, residual):
        return _RmsNorm.apply(i, x, weight, residual, float(eps))
    y, total = _norm_fwd(i, x, weight, residual, float(eps))
    return y if residual is None else (y, total)


def rms_norm_backward(d_y, x, weight, *, residual=None, d_sum=None, eps=1e-6):
    """(dh, dweight) of rms_norm for the gradients d_y of y and d_sum of the sum (None: not used); dh is the gradient of x and of the residual.  The explicit
    form of what autograd calls."""
    what = 'rms_norm_backward'
    i = _norm_args(what, x, weight, residual)
    _norm_args(what, x, weight, d_y)
    if d_sum is not None:
        _norm_args(what, x, weight, d_sum)
    _no_gradient(what, d_y, x, weight, residual, d_sum)
    return _norm_bwd(i, d_y, d_sum, x, weight, residual, float(eps))


# -------------------------------------------------------------------------------------------------------------------------- 8 bits
def _rows8(i, x, weight, residual, eps):
    N = x.shape[-1]
    x2, r2 = _matrix(x), None if residual is None else _matrix(residual)
    w = None if weight is None else weight.contiguous()
    M, P = x2.shape[0], (N + 15) // 16 * 16                 # rows start at 16-byte borders, for the product's loads
    q = torch.empty(x.shape[:-1] + (P,), dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=F32, device=x.device)
    total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch(i, 'srvp_rms_norm', NORM.pack(
        x2.data_ptr(), 0 if r2 is None else r2.data_ptr(), 0 if w is None else w.data_ptr(), 0, 0 if total is None else total.data_ptr(),
        q.data_ptr(), scale.data_ptr(), x2.stride(0), 0 if r2 is None else r2.stride(0), 0, N, P, M, N, eps, 1 if x.dtype is F32 else 0, 0))
    return q if P == N else q[..., :N], scale, total


def rms_norm_int8(x, weight, *, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: (q int8 (..., N), scale float32 (...)[, h]) with y ~ q * scale, scale = max|y| / 127 a row and q =
    round(h weight * (127 / max|h weight|)), half to even, in 64 bits (it does not depend on the order of a sum).  A row of zeros has scale 0, a row with an infinity or NaN scale NaN."""
    i = _norm_args('rms_norm_int8', x, weight, residual)
    _no_gradient('rms_norm_int8', x, weight, residual)
    q, scale, total = _rows8(i, x, weight, residual, float(eps))
    return (q, scale) if residual is None else (q, scale, total)


def quantize_int8(x):
    """(q int8 (..., N), scale float32 (...)) with x ~ q * scale for each row: activations without a norm, and a weight (out, in) by output channel."""
    i = _norm_args('quantize_int8', x, None, None)
    _no_gradient('quantize_int8', x)
    q, scale, _ = _rows8(i, x, None, None, 0.0)
    return q, scale


def linear_int8(x, x_scale, w, w_scale, *, bias=None, out_dtype=F32):
    """y[..., n] = (sum_k x[..., k] w[n, k]) * x_scale[...] * w_scale[n] + bias[n]: x (..., K) and w (N, K) int8 (K <= 131071: the sum is exact in 32 bits),
    scales and bias float32, y float32 or bfloat16."""
    what = 'linear_int8'
    i = _device(x, what)
    if x.dtype is not torch.int8 or w.dtype is not torch.int8:
        raise TypeError(f'{what}: x and w are int8 tensors, got {x.dtype} and {w.dtype}')
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f'{what}: x (..., K) and w (N, K), got {tuple(x.shape)} and {tuple(w.shape)}')
    N, K = w.shape
    if K > 131071:
        raise ValueError(f'{what}: the sum of {K} products could pass 32 bits (at most 131071)')
    for t, s, name in ((x_scale, x.shape[:-1], 'x_scale'), (w_scale, (N,), 'w_scale')) + (((bias, (N,), 'bias'),) if bias is not None else ()):
        if t.dtype is not F32 or t.shape != s:
            raise ValueError(f'{what}: {name} is a float32 tensor {tuple(s)}, got {tuple(t.shape)} {t.dtype}')
    if out_dtype is not F32 and out_dtype is not BF16:
        raise TypeError(f'{what}: float32 or bfloat16 output, got {out_dtype}')
    _same_device(what, i, x_scale, w, w_scale, bias)
    _no_gradient(what, x_scale, w_scale, bias)
    y = torch.empty(x.shape[:-1] + (N,), dtype=out_dtype, device=x.device)
    if K == 0:
        return y.zero_() if bias is None else y.copy_(bias.expand_as(y))
    x2, w = _matrix(x), _inner(w)
    x_scale, w_scale = x_scale.contiguous(), w_scale.contiguous()
    b = 0
    if bias is not None:
        bias = bias.contiguous()
        b = bias.data_ptr()
    _launch(i, 'srvp_linear_int8', INT8.pack(x2.data_ptr(), w.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(), b, y.data_ptr(), x2.stride(0), w.stride(0),
                                             N, x2.shape[0], N, K, 1 if out_dtype is F32 else 0))
    return y

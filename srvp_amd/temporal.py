"""
Operators over the time axis, the parallel counterpart of the posterior LSTM (reference module/srvp.py:130,366): linear attention with a decay for
each head (chunked form for whole sequences, recurrent form for single frames), rotary positions, the root-mean-square norm with the residual's
addition, and products on 8-bit integers for inference.

Tensors are time-major, (T, B, heads, features), float32 or bfloat16; any strides are taken as they are (features contiguous, otherwise the tensor is
copied first), so a batch-major tensor is passed as a transposed view and shared heads as an expanded one.  Every sum, state and norm is held in 32
bits or more.  Launches go to torch's current stream on the tensors' device; workspaces are ordinary tensors of the call.

Gradients: `linear_attention`, `rotary` and `rms_norm` are autograd nodes, differentiable once, in reverse mode (tensors with a forward-mode tangent are refused).  Inside a stream capture they record none (a captured backward
pass cannot be told apart from the eager one of the same leaves) and raise: call `linear_attention_backward`, `rotary(..., back=True)`, `rms_norm_backward`
there.

Checks, allocation and autograd nodes are csrc/temporal_ext.cpp (built beside libsrvp_hip.so), the kernels csrc/linear_attention.hip, rows.hip and int8.hip.
"""
import ctypes as C
import math

import torch

from . import _lib as L

_ENTRIES = ('srvp_last_error', 'srvp_stream_is_capturing', 'srvp_linear_attention_ws_bytes', 'srvp_linear_attention_fwd', 'srvp_linear_attention_bwd',
            'srvp_linear_attention_step', 'srvp_rotary', 'srvp_rms_norm', 'srvp_rms_norm_bwd_ws_bytes', 'srvp_rms_norm_bwd', 'srvp_linear_int8')
_ext = None


def load():
    """The extension, bound to the kernel library (once).  Raises if either has not been built."""
    global _ext
    if _ext is None:
        lib = L.load()
        try:
            from . import _temporal as ext
        except ImportError as e:
            raise L.SrvpHipError(f'srvp_amd/_temporal.so: {e}.  Build it with `make -C srvp_amd/csrc` (or `python -c "import __graft_entry__ as g; '
                                 'g.build()"`).') from e
        ext.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in _ENTRIES}, L.SrvpHipError, torch.OutOfMemoryError)
        _ext = ext
    return _ext


def decay_rates(heads, shortest=8.0, longest=512.0, device=None):
    """log_decay (heads,) float32 of memories that are `shortest` to `longest` frames long, spread evenly in their logarithm: decay 1 - 1/length."""
    if not 1.0 < shortest <= longest:
        raise ValueError('decay_rates: 1 < shortest <= longest')
    n = torch.linspace(math.log(shortest), math.log(longest), heads, dtype=torch.float64) if heads > 1 else torch.tensor([0.5 * math.log(shortest * longest)], dtype=torch.float64)
    return torch.log1p(-torch.exp(-n)).to(torch.float32).to(device)


def linear_attention(q, k, v, log_decay, *, state=None, lengths=None, scale=None, return_state=False):
    """S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,  o_t = scale * q_t S_t, causal over the first axis.

    q, k (T, B, H, Dk), v (T, B, H, Dv), heads of 1 to 256 features; log_decay (H,) float32, normally <= 0 (-inf: no memory); state (B, H, Dk, Dv)
    float32: S in front of the first token (None: zero; it is not changed); lengths (B,): tokens of each sequence (outputs behind them are zero, values
    there are not read); scale: default Dk ** -0.5.  Returns o (T, B, H, Dv), or (o, new state) with return_state.  Gradients: q, k, v, state.
    A NaN or infinity reaches the outputs of its own token and of those behind it, as an infinity or as NaN (which
    of the two is not kept apart: an infinity in v mostly comes out as NaN, in its column).
    The decays are constants: no gradient."""
    return (_ext or load()).linear_attention(q, k, v, log_decay, state, lengths, scale, return_state)


def linear_attention_backward(d_out, q, k, v, log_decay, *, state=None, lengths=None, scale=None, d_state=None):
    """(dq, dk, dv, d_state_in) of linear_attention for the gradients d_out of o and d_state of the new state (None: not used); d_state_in is None
    without a state.  The explicit form of what autograd calls."""
    return (_ext or load()).linear_attention_backward(d_out, q, k, v, log_decay, state, lengths, scale, d_state)


def linear_attention_step(q, k, v, log_decay, state, *, slots=None, scale=None):
    """One token of each of B sequences: q, k (B, H, Dk), v (B, H, Dv) -> o (B, H, Dv); state (slots, H, Dk, Dv) float32, contiguous, is advanced in place.
    slots (B,): where each row's state lies (None: row b has state b), for at most 65536 rows.  A slot outside the pool marks a padded row: its output is zero, no state is
    touched.  Rows that name the same slot are successive tokens of one sequence, in row order."""
    return (_ext or load()).linear_attention_step(q, k, v, log_decay, state, slots, scale)


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


def rotary(q, k, positions, frequencies, *, interleaved=False, back=False, magnitude=1.0):
    """Turns the pairs of features of q (T, B, Hq, D) and, in the same launch, of k (T, B, Hk, D; None: q alone) by positions * frequencies radians.

    positions (T,) or (T, B), whole numbers up to 2^53 (angles are formed to 2^-52 of a turn); frequencies float64 (pairs,) on the device, 2 * pairs <= D
    (rotary_frequencies; constants, no gradient): features behind the first 2 * pairs are passed on unchanged.  interleaved: pair p is features (2p, 2p + 1), otherwise
    (p, pairs + p).  magnitude multiplies the turned features.  back: the negative angle, which is the gradient's.  Returns q', or (q', k')."""
    return (_ext or load()).rotary(q, k, positions, frequencies, interleaved, back, magnitude)


def rms_norm(x, weight, *, residual=None, eps=1e-6):
    """y = h * weight / sqrt(mean(h^2) + eps) over the last axis, h = x + residual.  x, residual (..., N), N <= 16384; weight (N,) float32.  Returns y, or
    (y, h) with a residual (h rounded to x's type; y and the gradients are those of the unrounded sum).  Squares are summed in float32: rows above 1.8e19
    come out as zero.  Gradients: x, residual, weight."""
    return (_ext or load()).rms_norm(x, weight, residual, eps)


def rms_norm_backward(d_y, x, weight, *, residual=None, d_sum=None, eps=1e-6):
    """(dh, dweight) of rms_norm for the gradients d_y of y and d_sum of the sum (None: not used); dh is the gradient of x and of the residual.  The explicit
    form of what autograd calls."""
    return (_ext or load()).rms_norm_backward(d_y, x, weight, residual, d_sum, eps)


def rms_norm_int8(x, weight, *, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: (q int8 (..., N), scale float32 (...)[, h]) with y ~ q * scale, scale = max|y| / 127 a row and q =
    round(h weight * (127 / max|h weight|)), half to even, in 64 bits (it does not depend on the order of a sum).  A row of zeros has scale 0, a row of y with
    an infinity or NaN, its own or the weight's, scale NaN."""
    return (_ext or load()).rms_norm_int8(x, weight, residual, eps)


def quantize_int8(x):
    """(q int8 (..., N), scale float32 (...)) with x ~ q * scale for each row: activations without a norm, and a weight (out, in) by output channel."""
    return (_ext or load()).quantize_int8(x)


def linear_int8(x, x_scale, w, w_scale, *, bias=None, out_dtype=torch.float32):
    """y[..., n] = (sum_k x[..., k] w[n, k]) * x_scale[...] * w_scale[n] + bias[n]: x (..., K) and w (N, K) int8 (K <= 131071: the sum is exact in 32 bits),
    scales and bias float32, y float32 or bfloat16."""
    return (_ext or load()).linear_int8(x, x_scale, w, w_scale, bias, out_dtype)

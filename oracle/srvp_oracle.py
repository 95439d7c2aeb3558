"""
CPU oracle for the SRVP training / rollout hot path  --  TEST INFRASTRUCTURE ONLY.

This file is a from-scratch *functional restatement* (plain torch CPU ops, explicit noise tape,
state-dict in / tensors out) of the algorithm implemented by the reference's
``module/conv.py``, ``module/mlp.py``, ``module/utils.py``, ``module/srvp.py`` and ``train.py:train``.
It is the checker the HIP path is compared against; it is NOT part of the product:

  * only ``tests/``, ``__graft_entry__.smoke()`` and ``bench.py``'s ``cpu_baseline`` leg may import it;
  * nothing under ``srvp_amd/`` imports it, and the product raises if the HIP library is missing.

Pinning: the reference ships no tests / golden vectors, so the oracle is pinned by the
fixtures under ``tests/golden/`` which ``tests/make_golden.py`` generated by importing the real reference
from ``/root/reference`` in the build container (forward outputs, ELBO terms, every parameter gradient,
post-Adam parameters and BN running statistics).  ``tests/test_oracle_golden.py`` checks this file against
those fixtures.

Every function cites the reference lines it restates.  Key layout facts:
  x is time-major ``(T, B, C, H, W)`` float in [0, 1]; conv weights OIHW, ConvTranspose weights IOHW;
  LSTM gate order i, f, g, o.
"""
import math
from typing import Dict, List, Optional, Tuple

import torch
import torch.nn.functional as F

Tensor = torch.Tensor
SD = Dict[str, Tensor]

BN_EPS = 1e-5        # torch.nn.BatchNorm2d default used by conv.py:104
BN_MOMENTUM = 0.1
LRELU_SLOPE = 0.2    # utils.py:41
HALF_LOG_2PI = 0.5 * math.log(2 * math.pi)


# ----------------------------------------------------------------------------------------------------
# Architecture tables (conv.py:157-224, 278-355).  Each entry describes one conv block.
#   kind: 'conv' | 'convT';  k/s/p;  bn;  act;  pre: None|'pool' (MaxPool2 before, conv.py:204..222)
#   post_up: nearest x2 after the block (conv.py:331,338,344,349);  cat: skip concat before the block (conv.py:270)
#   skip_out: the block output (after act) is the stage output collected as a skip (conv.py:148-150)
# ----------------------------------------------------------------------------------------------------
def encoder_spec(archi: str, nc: int, nh: int, nf: int) -> List[dict]:
    L = []
    if archi == 'dcgan':  # conv.py:173-179
        chans = [nc, nf, nf * 2, nf * 4, nf * 8]
        for i in range(4):
            L.append(dict(kind='conv', key=f'encoder.conv.{i}.0', bnkey=(f'encoder.conv.{i}.1' if i > 0 else None),
                          cin=chans[i], cout=chans[i + 1], k=4, s=2, p=1, act='leaky_relu', pre=None,
                          skip_out=True))
        L.append(dict(kind='conv', key='encoder.last_conv.0', bnkey='encoder.last_conv.1', cin=nf * 8, cout=nh,
                      k=4, s=1, p=0, act='tanh', pre=None, skip_out=False))
    elif archi == 'vgg':  # conv.py:198-224
        stages = [[(nc, nf), (nf, nf)],
                  [(nf, nf * 2), (nf * 2, nf * 2)],
                  [(nf * 2, nf * 4), (nf * 4, nf * 4), (nf * 4, nf * 4)],
                  [(nf * 4, nf * 8), (nf * 8, nf * 8), (nf * 8, nf * 8)]]
        for si, st in enumerate(stages):
            off = 0 if si == 0 else 1  # index 0 of stages >0 is the MaxPool module
            for li, (ci, co) in enumerate(st):
                L.append(dict(kind='conv', key=f'encoder.conv.{si}.{li + off}.0', bnkey=f'encoder.conv.{si}.{li + off}.1',
                              cin=ci, cout=co, k=3, s=1, p=1, act='leaky_relu',
                              pre=('pool' if (si > 0 and li == 0) else None), skip_out=(li == len(st) - 1)))
        L.append(dict(kind='conv', key='encoder.last_conv.1.0', bnkey='encoder.last_conv.1.1', cin=nf * 8, cout=nh,
                      k=4, s=1, p=0, act='tanh', pre='pool', skip_out=False))
    else:
        raise ValueError(f"No encoder named '{archi}'")  # conv.py:49
    L[0]['role'] = 'in'          # image-side layer: fp32 frames in (numerics model only)
    L[-1]['f32_out'] = True      # hx is handed to the fp32 latent path unrounded
    return L


def decoder_spec(archi: str, nc: int, ny: int, nf: int, skip: bool) -> List[dict]:
    c = 2 if skip else 1
    L = []
    if archi == 'dcgan':  # conv.py:298-305
        L.append(dict(kind='convT', key='decoder.first_upconv.0', bnkey='decoder.first_upconv.1', cin=ny, cout=nf * 8,
                      k=4, s=1, p=0, act='leaky_relu', cat=None, post_up=False))
        chans = [nf * 8, nf * 4, nf * 2, nf]
        for i in range(3):
            L.append(dict(kind='convT', key=f'decoder.conv.{i}.0', bnkey=f'decoder.conv.{i}.1', cin=chans[i] * c,
                          cout=chans[i + 1], k=4, s=2, p=1, act='leaky_relu', cat=(i if skip else None), post_up=False))
        L.append(dict(kind='convT', key='decoder.conv.3', bnkey=None, cin=nf * c, cout=nc, k=4, s=2, p=1, act='none',
                      cat=(3 if skip else None), post_up=False))
    elif archi == 'vgg':  # conv.py:329-355
        L.append(dict(kind='convT', key='decoder.first_upconv.0.0', bnkey='decoder.first_upconv.0.1', cin=ny,
                      cout=nf * 8, k=4, s=1, p=0, act='leaky_relu', cat=None, post_up=True))
        stages = [[(nf * 8 * c, nf * 8), (nf * 8, nf * 8), (nf * 8, nf * 4)],
                  [(nf * 4 * c, nf * 4), (nf * 4, nf * 4), (nf * 4, nf * 2)],
                  [(nf * 2 * c, nf * 2), (nf * 2, nf)],
                  [(nf * c, nf)]]
        for si, st in enumerate(stages):
            for li, (ci, co) in enumerate(st):
                L.append(dict(kind='conv', key=f'decoder.conv.{si}.{li}.0', bnkey=f'decoder.conv.{si}.{li}.1', cin=ci,
                              cout=co, k=3, s=1, p=1, act='leaky_relu', cat=(si if (skip and li == 0) else None),
                              post_up=(si < 3 and li == len(st) - 1)))
        L.append(dict(kind='convT', key='decoder.conv.3.1', bnkey=None, cin=nf, cout=nc, k=3, s=1, p=1, act='none',
                      cat=None, post_up=False))
    else:
        raise ValueError(f"No decoder named '{archi}'")  # conv.py:78
    L[-1]['role'] = 'out'        # image-side layer: fp32 frames out (numerics model only)
    return L


# ----------------------------------------------------------------------------------------------------
# Blocks
# ----------------------------------------------------------------------------------------------------
def activation(h: Tensor, name: str) -> Tensor:
    """utils.py:23-48 (out-of-place; the reference's in-place variants are value-identical)."""
    if name == 'relu':
        return F.relu(h)
    if name == 'leaky_relu':
        return F.leaky_relu(h, LRELU_SLOPE)
    if name == 'tanh':
        return torch.tanh(h)
    if name == 'sigmoid':
        return torch.sigmoid(h)
    if name == 'none':
        return h
    raise ValueError(name)


# SyncBatchNorm hook for the multi-rank tests (reference train.py:278-283 converts every BatchNorm2d with
# nn.SyncBatchNorm.convert_sync_batchnorm): a callable (sum, sumsq, count) -> the same three summed over all ranks,
# differentiable (torch.distributed.nn.functional.all_reduce).  None = single process.
BN_SYNC = None


def batch_norm(h: Tensor, sd: SD, key: str, training: bool, bn_stats: Optional[dict] = None) -> Tensor:
    """
    nn.BatchNorm2d as placed by conv.py:103-104 (BN *before* the activation).  Training: batch statistics over
    (N, H, W) -- N = T*B since time is flattened into batch (srvp.py:176, 215) -- biased variance for normalisation,
    unbiased for running_var, momentum 0.1.  ``bn_stats`` (optional) maps key -> (mean, var, count) of the *global* batch;
    with ``BN_SYNC`` set the statistics are the global ones obtained through that hook (SyncBatchNorm, train.py:283).
    """
    w, b = sd[key + '.weight'], sd[key + '.bias']
    rm, rv = sd[key + '.running_mean'], sd[key + '.running_var']
    if training:
        if bn_stats is not None and key in bn_stats:
            mean, var, count = bn_stats[key]
        elif BN_SYNC is not None:
            hd = h.double()
            s1, s2, count = BN_SYNC(hd.sum(dim=(0, 2, 3)), (hd * hd).sum(dim=(0, 2, 3)), h.numel() // h.shape[1])
            mean64 = s1 / count
            mean, var = mean64.to(h.dtype), (s2 / count - mean64 * mean64).to(h.dtype)
        else:
            mean = h.mean(dim=(0, 2, 3))
            var = h.var(dim=(0, 2, 3), unbiased=False)
            count = h.numel() // h.shape[1]
        with torch.no_grad():
            rm.mul_(1 - BN_MOMENTUM).add_(BN_MOMENTUM * mean.detach())
            rv.mul_(1 - BN_MOMENTUM).add_(BN_MOMENTUM * var.detach() * (count / max(count - 1, 1)))
            if key + '.num_batches_tracked' in sd:
                sd[key + '.num_batches_tracked'] += 1
    else:
        mean, var = rm, rv
    inv = torch.rsqrt(var + BN_EPS)
    return (h - mean[None, :, None, None]) * (inv * w)[None, :, None, None] + b[None, :, None, None]


# ----------------------------------------------------------------------------------------------------
# Numerics model of the HIP path (test infrastructure).  PRECISION = 'fp32' is the reference's arithmetic.
# PRECISION = 'bf16' inserts the product's documented rounding points (DESIGN.md "precision") into the SAME
# algorithm -- bf16 operands for the MFMA layers (fp32 accumulate), raw conv outputs and activations stored as
# bf16, BatchNorm statistics taken from the fp32 accumulators, the two image-side layers and the whole latent
# path in fp32 -- with straight-through gradients.  It lets the tests separate "the kernels implement the
# algorithm" (tight, vs this model) from "bf16 storage perturbs an ill-conditioned small-batch network"
# (loose, vs the fp32 fixtures).
# ----------------------------------------------------------------------------------------------------
PRECISION = 'fp32'


class _RoundBF16(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.to(torch.bfloat16).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g


def _bf(x: Tensor) -> Tensor:
    return _RoundBF16.apply(x)


def _conv_block_bf16(h: Tensor, sd: SD, spec: dict, training: bool) -> Tensor:
    w = sd[spec['key'] + '.weight']
    role = spec.get('role', 'mfma')
    if role in ('mfma', 'out'):          # 'out': MFMA layer too, but fp32 (unrounded) frames out
        h, w = _bf(h), _bf(w)
    r = F.conv2d(h, w, None, spec['s'], spec['p']) if spec['kind'] == 'conv' else F.conv_transpose2d(h, w, None, spec['s'], spec['p'])
    if role == 'out':
        return activation(r, spec['act'])
    if spec['bnkey'] is not None:
        key = spec['bnkey']
        gam, bet, rm, rv = sd[key + '.weight'], sd[key + '.bias'], sd[key + '.running_mean'], sd[key + '.running_var']
        if training:
            mean, var = r.mean(dim=(0, 2, 3)), r.var(dim=(0, 2, 3), unbiased=False)      # from the fp32 accumulators
            count = r.numel() // r.shape[1]
            with torch.no_grad():
                rm.mul_(1 - BN_MOMENTUM).add_(BN_MOMENTUM * mean.detach())
                rv.mul_(1 - BN_MOMENTUM).add_(BN_MOMENTUM * var.detach() * (count / max(count - 1, 1)))
                if key + '.num_batches_tracked' in sd:
                    sd[key + '.num_batches_tracked'] += 1
        else:
            mean, var = rm, rv
        scale = gam * torch.rsqrt(var + BN_EPS)
        shift = bet - mean * scale
        r = _bf(r) * scale[None, :, None, None] + shift[None, :, None, None]
    else:
        r = _bf(r)
    a = activation(r, spec['act'])
    return a if spec.get('f32_out') else _bf(a)


def conv_block(h: Tensor, sd: SD, spec: dict, training: bool) -> Tensor:
    """conv.py:81-107: conv (bias=False) -> [BatchNorm2d] -> [activation]."""
    if PRECISION == 'bf16':
        return _conv_block_bf16(h, sd, spec, training)
    w = sd[spec['key'] + '.weight']
    if spec['kind'] == 'conv':
        h = F.conv2d(h, w, None, spec['s'], spec['p'])
    else:
        h = F.conv_transpose2d(h, w, None, spec['s'], spec['p'])
    if spec['bnkey'] is not None:
        h = batch_norm(h, sd, spec['bnkey'], training)
    return activation(h, spec['act'])


def encoder_forward(sd: SD, cfg: dict, x_flat: Tensor, training: bool) -> Tuple[Tensor, List[Tensor]]:
    """conv.py:129-154: run the blocks, collect stage outputs deepest-first, flatten last_conv output to (N, nh)."""
    skips = []
    h = x_flat
    for spec in encoder_spec(cfg['archi'], cfg['nc'], cfg['nhx'], cfg['nf']):
        if spec['pre'] == 'pool':
            h = F.max_pool2d(h, 2, 2, 0)
        h = conv_block(h, sd, spec, training)
        if spec['skip_out']:
            skips.append(h)
    return h.reshape(-1, cfg['nhx']), skips[::-1]


def decoder_forward(sd: SD, cfg: dict, z: Tensor, skip: Optional[List[Tensor]], training: bool,
                    sigmoid: bool = True) -> Tensor:
    """conv.py:249-275: first_upconv on (N, Cz, 1, 1); per stage cat([h, skip[i]], 1) then the stage; sigmoid."""
    assert (skip is None) == (not cfg['skipco'])
    h = z.reshape(z.shape[0], z.shape[1], 1, 1)
    if PRECISION == 'bf16':
        h = _bf(h)
    for spec in decoder_spec(cfg['archi'], cfg['nc'], cfg['nh_inf'] + cfg['ny'], cfg['nf'], cfg['skipco']):
        if spec['cat'] is not None:
            h = torch.cat([h, skip[spec['cat']]], 1)
        h = conv_block(h, sd, spec, training)
        if spec['post_up']:
            h = F.interpolate(h, scale_factor=2, mode='nearest')
    return torch.sigmoid(h) if sigmoid else h


def linear(sd: SD, key: str, h: Tensor) -> Tensor:
    return F.linear(h, sd[key + '.weight'], sd[key + '.bias'])


def mlp(sd: SD, prefix: str, n_layers: int, h: Tensor) -> Tensor:
    """mlp.py:47-90: Linear, then (ReLU -> Linear) x (n_layers-1); keys '<prefix>.module.0.0', '.1.1', '.2.1', ..."""
    for il in range(n_layers):
        if il > 0:
            h = F.relu(h)
        h = linear(sd, f'{prefix}.module.{il}.{0 if il == 0 else 1}', h)
    return h


def lstm(sd: SD, prefix: str, x: Tensor) -> Tensor:
    """nn.LSTM(nhx, nh_inf, 1) with zero initial state (srvp.py:132,366); gate order i, f, g, o."""
    w_ih, w_hh = sd[prefix + '.weight_ih_l0'], sd[prefix + '.weight_hh_l0']
    b = sd[prefix + '.bias_ih_l0'] + sd[prefix + '.bias_hh_l0']
    nh = w_hh.shape[1]
    h = x.new_zeros(x.shape[1], nh)
    c = x.new_zeros(x.shape[1], nh)
    out = []
    for t in range(x.shape[0]):
        g = F.linear(x[t], w_ih) + F.linear(h, w_hh) + b
        i, f, gg, o = g.chunk(4, 1)
        c = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(gg)
        h = torch.sigmoid(o) * torch.tanh(c)
        out.append(h)
    return torch.stack(out)


def normal_params(raw: Tensor) -> Tuple[Tensor, Tensor]:
    """utils.py:88-112: loc, scale = chunk(raw, 2, -1); scale = softplus(scale) + 1e-8."""
    loc, raw_scale = torch.chunk(raw, 2, -1)
    return loc, F.softplus(raw_scale) + 1e-8


def rsample(raw: Tensor, eps: Tensor) -> Tensor:
    """utils.py:115-134 with the N(0,1) draw made explicit: loc + eps * scale."""
    loc, scale = normal_params(raw)
    return loc + eps * scale


def kl_normal(q_raw: Tensor, p_raw: Optional[Tensor]) -> Tensor:
    """torch.distributions.kl_divergence(Normal, Normal) as called by train.py:95,98 (p=None -> N(0,1))."""
    ql, qs = normal_params(q_raw)
    if p_raw is None:
        pl, ps = torch.zeros_like(ql), torch.ones_like(qs)
    else:
        pl, ps = normal_params(p_raw)
    var_ratio = (qs / ps) ** 2
    t1 = ((ql - pl) / ps) ** 2
    return 0.5 * (var_ratio + t1 - 1 - var_ratio.log())


def neg_logprob(loc: Tensor, data: Tensor, scale: float) -> Tensor:
    """utils.py:137-159: -Normal(loc, scale).log_prob(data) with a scalar scale."""
    return (data - loc) ** 2 / (2 * scale * scale) + math.log(scale) + HALF_LOG_2PI


# ----------------------------------------------------------------------------------------------------
# Euler schedule (srvp.py:370-405).  The reference walks np.linspace(dt, nt-1, n*(nt-1)) and uses ceil /
# is_integer on floats; for n_euler in {1,2,4,...} that is exactly: step i -> frame i//n + 1, new frame iff
# i % n == 0, keep the state iff (i+1) % n == 0.  (For other n the float grid mis-detects integers -- SURVEY §7;
# the oracle and the product use the integer schedule and document the divergence.)
# ----------------------------------------------------------------------------------------------------
def euler_schedule(nt: int, n_euler: int) -> List[Tuple[int, bool, bool]]:
    return [(i // n_euler + 1, i % n_euler == 0, (i + 1) % n_euler == 0) for i in range(n_euler * (nt - 1))]


# ----------------------------------------------------------------------------------------------------
# Model-level functions (srvp.py)
# ----------------------------------------------------------------------------------------------------
def make_cfg(nx, nc, nf, nhx, ny, nz, skipco, nt_inf, nh_inf, nlayers_inf, nh_res, nlayers_res, archi) -> dict:
    """Same positional order as the reference constructor (srvp.py:76)."""
    return dict(nx=nx, nc=nc, nf=nf, nhx=nhx, ny=ny, nz=nz, skipco=skipco, nt_inf=nt_inf, nh_inf=nh_inf,
                nlayers_inf=nlayers_inf, nh_res=nh_res, nlayers_res=nlayers_res, archi=archi)


def encode(sd: SD, cfg: dict, x: Tensor, training: bool, t_skip: Optional[Tensor]):
    """srvp.py:156-193.  ``t_skip`` (B,) is the recorded torch.randint draw of srvp.py:185 (train + skipco only)."""
    nt, bsz = x.shape[0], x.shape[1]
    hx_flat, skips = encoder_forward(sd, cfg, x.reshape(nt * bsz, *x.shape[2:]), training)
    hx = hx_flat.view(nt, bsz, cfg['nhx'])
    if cfg['skipco']:
        if training:
            idx = torch.arange(bsz)
            skips = [s.view(nt, bsz, *s.shape[1:])[t_skip, idx] for s in skips]
        else:
            skips = [s.view(nt, bsz, *s.shape[1:])[-1] for s in skips]
    else:
        skips = None
    return hx, skips


def infer_w(sd: SD, cfg: dict, hx: Tensor, training: bool, t_w: Optional[Tensor]) -> Tensor:
    """srvp.py:229-256.  ``t_w`` (nt_inf, B): stacked randperm(nt)[:nt_inf] draws of srvp.py:246."""
    bsz = hx.shape[1]
    if training:
        idx = torch.arange(bsz).repeat(cfg['nt_inf'], 1)
        h = hx[t_w.reshape(-1), idx.reshape(-1)].view(cfg['nt_inf'], bsz, cfg['nhx'])
    else:
        h = hx[-cfg['nt_inf']:]
    h = F.relu(linear(sd, 'w_proj.0', h)).sum(0)
    return torch.tanh(linear(sd, 'w_inf.0', h))


def infer_y(sd: SD, cfg: dict, hx: Tensor, eps_y0: Tensor) -> Tuple[Tensor, Tensor]:
    """srvp.py:258-278."""
    q = mlp(sd, 'q_y', cfg['nlayers_inf'], hx.permute(1, 0, 2).reshape(hx.shape[1], cfg['nt_inf'] * cfg['nhx']))
    return rsample(q, eps_y0), q


def residual_step(sd: SD, cfg: dict, y: Tensor, z: Tensor, dt: float) -> Tuple[Tensor, Tensor]:
    """srvp.py:300-323."""
    res = dt * mlp(sd, 'dynamics', cfg['nlayers_res'], torch.cat([y, z], 1))
    return y + res, res


def generate(sd: SD, cfg: dict, y_0: Tensor, hx, nt: int, n_euler: int, eps_z: Tensor, training: bool, remove_intermediate: bool = True):
    """
    srvp.py:325-413 (remove_intermediate, srvp.py:402: False keeps the state after every Euler sub-step).  ``eps_z`` (nt-1, B, nz): one N(0,1) draw per frame in order,
    used for the posterior sample while data lasts (srvp.py:387) and for the prior sample afterwards (srvp.py:392).
    """
    dt = 1.0 / n_euler
    n_data = len(hx)
    hx_z = lstm(sd, 'inf_z', hx) if n_data > 0 else []
    y, z, qz, pz, res = [y_0], [], [], [], []
    y_prev = y_0
    for frame, new_frame, keep in euler_schedule(nt, n_euler):
        if new_frame:
            p = mlp(sd, 'p_z', cfg['nlayers_res'], y_prev)
            pz.append(p)
            if frame < n_data:
                q = linear(sd, 'q_z', hx_z[frame])
                qz.append(q)
                z.append(rsample(q, eps_z[frame - 1]))
            else:
                assert not training  # srvp.py:391
                z.append(rsample(p, eps_z[frame - 1]))
        y_prev, r = residual_step(sd, cfg, y_prev, z[-1], dt)
        if keep or not remove_intermediate:
            y.append(y_prev)
        res.append(r)
    st = lambda l: torch.stack(l) if len(l) > 0 else None
    return torch.stack(y), st(z), st(qz), st(pz), torch.stack(res)


def decode(sd: SD, cfg: dict, w: Tensor, y: Tensor, skip, training: bool) -> Tensor:
    """srvp.py:195-227: rows ordered t*B + b, w tiled over t, skips expanded over t."""
    nt, bsz = y.shape[0], y.shape[1]
    dec_inp = torch.cat([w.repeat(nt, 1, 1).view(nt * bsz, cfg['nh_inf']), y.reshape(nt * bsz, cfg['ny'])], 1)
    if skip is not None:
        skip = [s.expand(nt, *s.shape).reshape(nt * bsz, *s.shape[1:]) for s in skip]
    x_flat = decoder_forward(sd, cfg, dec_inp, skip, training)
    return x_flat.view(nt, bsz, *x_flat.shape[1:])


def forward(sd: SD, cfg: dict, x: Tensor, nt: int, n_euler: int, tape: dict, training: bool, remove_intermediate: bool = True):
    """srvp.py:415-470.  tape: t_skip (B,), t_w (nt_inf,B), eps_y0 (B,ny), eps_z (nt-1,B,nz)."""
    hx, skips = encode(sd, cfg, x, training, tape.get('t_skip'))
    w = infer_w(sd, cfg, hx, training, tape.get('t_w'))
    y_0, q_y0 = infer_y(sd, cfg, hx[:cfg['nt_inf']], tape['eps_y0'])
    y, z, qz, pz, res = generate(sd, cfg, y_0, hx, nt, n_euler, tape['eps_z'], training, remove_intermediate)
    x_ = decode(sd, cfg, w, y, skips, training)
    return x_, y, z, w, q_y0, qz, pz, res


def elbo(x: Tensor, outs, obs_scale: float, beta_y: float, beta_z: float, l2_res: float) -> dict:
    """train.py:90-106 (loss /= local batch)."""
    x_, y, z, w, q_y0, qz, pz, res = outs
    n = x.shape[1]
    nll = neg_logprob(x_, x, obs_scale).sum()
    kl_y0 = kl_normal(q_y0, None).sum()
    kl_z = kl_normal(qz, pz).sum()
    loss = nll + beta_y * kl_y0 + beta_z * kl_z
    l2 = torch.norm(res, p=2, dim=2).sum()
    if l2_res > 0:
        loss = loss + l2_res * l2
    return dict(loss=loss / n, nll=nll, kl_y0=kl_y0, kl_z=kl_z, l2_res=l2)


def split_state(sd: SD) -> Tuple[List[str], List[str]]:
    """Parameter keys (in module registration order = state-dict order) and buffer keys."""
    buf = ('running_mean', 'running_var', 'num_batches_tracked', 'log_decay')
    p = [k for k in sd if not k.endswith(buf)]
    b = [k for k in sd if k.endswith(buf)]
    return p, b


def adam_step(sd: SD, grads: Dict[str, Tensor], state: dict, lr: float, betas=(0.9, 0.999), eps=1e-8) -> None:
    """torch.optim.Adam defaults as constructed by train.py:289 (no weight decay, no amsgrad)."""
    state['step'] = state.get('step', 0) + 1
    t = state['step']
    b1, b2 = betas
    with torch.no_grad():
        for k, g in grads.items():
            m = state.setdefault('m.' + k, torch.zeros_like(g))
            v = state.setdefault('v.' + k, torch.zeros_like(g))
            m.mul_(b1).add_(g, alpha=1 - b1)
            v.mul_(b2).addcmul_(g, g, value=1 - b2)
            denom = (v.sqrt() / math.sqrt(1 - b2 ** t)).add_(eps)
            sd[k].addcdiv_(m, denom, value=-lr / (1 - b1 ** t))


def train_step(sd: SD, cfg: dict, x: Tensor, n_euler: int, tape: dict, hp: dict, adam_state: Optional[dict] = None,
               lr: Optional[float] = None):
    """
    train.py:49-129 as one function: forward (training mode), ELBO, backward, optional Adam step.
    ``sd`` is modified in place (BN running stats; parameters if ``adam_state`` is given).
    Returns (terms dict of python floats incl. the 4 logged scalars, outs, grads dict).
    """
    pkeys, _ = split_state(sd)
    leaves = {k: sd[k].detach().clone().requires_grad_(True) for k in pkeys}
    work = dict(sd)
    work.update(leaves)
    outs = forward(work, cfg, x, x.shape[0], n_euler, tape, training=True)
    for k in sd:  # BN buffers were updated through `work` (same tensor objects)
        pass
    terms = elbo(x, outs, hp['obs_scale'], hp['beta_y'], hp['beta_z'], hp['l2_res'])
    grads_list = torch.autograd.grad(terms['loss'], [leaves[k] for k in pkeys])
    grads = {k: g for k, g in zip(pkeys, grads_list)}
    if adam_state is not None:
        adam_step(sd, grads, adam_state, lr)
    n = x.shape[1]
    scal = dict(loss=terms['loss'].item(), nll=terms['nll'].item() / n, kl_y_0=terms['kl_y0'].item() / n,
                kl_z=terms['kl_z'].item() / n, l2_res=terms['l2_res'].item())
    return scal, [o.detach() if o is not None else None for o in outs], grads


def lr_lambda(i: int, n_iter: int) -> float:
    """train.py:292-293."""
    return max(0, (n_iter - i) / n_iter)


# ----------------------------------------------------------------------------------------------------
# Evaluation metrics: restated in float64 with explicit window sums (no conv call).
def gaussian_window(size: int = 11, sigma: float = 1.5) -> Tensor:
    """metrics/ssim.py:81-90: softmax over the grid of -(dx^2 + dy^2) / (2 sigma^2) = normalised 2-D gaussian (size, size)."""
    c = torch.arange(size, dtype=torch.float64) - (size - 1) / 2
    e = -(c ** 2) / (2 * sigma ** 2)
    w = torch.exp(e.view(1, -1) + e.view(-1, 1))
    return w / w.sum()


def _window_mean(img: Tensor, win: Tensor) -> Tensor:
    """'valid' cross-correlation of every (H, W) plane with the window (conv2d(..., groups=channel), ssim.py:97-105)."""
    f = win.shape[0]
    patches = img.unfold(-2, f, 1).unfold(-2, f, 1)              # (..., H-f+1, W-f+1, f, f)
    return (patches * win).sum(dim=(-1, -2))


def ssim_map(inp: Tensor, target: Tensor, max_val: float = 1.0, filter_size: int = 11, k1: float = 0.01, k2: float = 0.03,
             sigma: float = 1.5) -> Tensor:
    """metrics/ssim.py:93-110 (`_ssim`, first return value), any leading dims, float64."""
    x, y = inp.double(), target.double()
    win = gaussian_window(filter_size, sigma)
    c1, c2 = (k1 * max_val) ** 2, (k2 * max_val) ** 2
    mu1, mu2 = _window_mean(x, win), _window_mean(y, win)
    s1 = _window_mean(x * x, win) - mu1 ** 2
    s2 = _window_mean(y * y, win) - mu2 ** 2
    s12 = _window_mean(x * y, win) - mu1 * mu2
    v1, v2 = 2 * s12 + c2, s1 + s2 + c2
    return ((2 * mu1 * mu2 + c1) * v1) / ((mu1 ** 2 + mu2 ** 2 + c1) * v2)


def video_ssim(sample: Tensor, gt: Tensor) -> Tensor:
    """test.py:36-57 (`_ssim_wrapper`): pixel-averaged SSIM, (length, batch, channels)."""
    return ssim_map(sample, gt, max_val=1.0).mean(dim=(-1, -2))


def video_mse(sample: Tensor, gt: Tensor) -> Tensor:
    """test.py:249: torch.mean((x_pred - x_target) ** 2, dim=[3, 4])."""
    return ((sample.double() - gt.double()) ** 2).mean(dim=(3, 4))


def video_psnr(sample: Tensor, gt: Tensor) -> Tensor:
    """test.py:251 / train.py:175-176: 10 log10(1 / mse) per (frame, video, channel)."""
    return 10 * torch.log10(1 / video_mse(sample, gt))


# ----------------------------------------------------------------------------------------------------
# Stochastic Moving-MNIST frame assembly, numpy restatement of data/mmnist.py:116-124.
def mmnist_render(digits, idx, pos, nx: int):
    """digits (n, h, w) uint8, idx (B, nd), pos (B, nd, T, 2) -> uint8 videos (B, T, nx, nx): float32 slice-adds of the
    digits at their (row, col) offsets, clamp at 255, cast (mmnist.py:113-124)."""
    import numpy as np
    B, nd, T, _ = pos.shape
    h, w = digits.shape[1:]
    out = np.zeros((B, T, nx, nx), np.float32)
    for b in range(B):
        for n in range(nd):
            img = digits[idx[b, n]]
            for t in range(T):
                r, c = pos[b, n, t]
                out[b, t, r:r + h, c:c + w] += img
    out[out > 255] = 255
    return out.astype(np.uint8)

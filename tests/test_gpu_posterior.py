"""
The attention posterior (srvp_amd.posterior) in the model: the block and its gradients against plain float64 autograd, the latent path and a whole training
step against the CPU oracle with its LSTM exchanged for the plain block, single frames against sequences, 8-bit inference against its definition.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain_block(sd, x, heads, prefix='inf_z'):
    """u = W x + b, norm, q k v, rotary, decayed linear attention token pair by token pair, norm, product, norm of the residual sum: (T, B, nhx) -> (T, B, nh)."""
    from srvp_amd import temporal
    p = lambda k: sd[f'{prefix}.{k}.weight']
    norm = lambda h, w: h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w
    T, B = x.shape[:2]
    u = x @ p('inp').t() + sd[f'{prefix}.inp.bias']
    nh = u.shape[-1]
    D = nh // heads
    q, k, v = (norm(u, p('norm')) @ p('qkv').t()).view(T, B, 3, heads, D).unbind(2)
    n = D // 2
    a = torch.arange(T, dtype=torch.float64).view(T, 1, 1, 1) * temporal.rotary_frequencies(2 * n)
    c, s = torch.cos(a).to(x), torch.sin(a).to(x)
    turn = lambda h: torch.cat([h[..., :n] * c - h[..., n:2 * n] * s, h[..., :n] * s + h[..., n:2 * n] * c, h[..., 2 * n:]], -1)
    q, k = turn(q), turn(k)
    gap = torch.arange(T).view(T, 1) - torch.arange(T).view(1, T)
    w = torch.exp(temporal.decay_rates(heads).double().view(-1, 1, 1) * gap.clamp(min=0)).to(x) * (gap >= 0)
    score = (q.permute(1, 2, 0, 3) @ k.permute(1, 2, 3, 0)) * w * D ** -0.5
    o = (score @ v.permute(1, 2, 0, 3)).permute(2, 0, 1, 3).reshape(T, B, nh)
    z = norm(o, p('out_norm')) @ p('out').t()
    return norm(u + z, p('last_norm'))


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return ((a - b).norm() / (b.norm() + 1e-30)).item()


CASES = [(1, 2, 8, 24, 1), (4, 3, 16, 24, 3), (12, 20, 128, 256, None), (50, 3, 32, 48, 3), (7, 5, 16, 15, 3)]


@pytest.mark.parametrize('T,B,nhx,nh,heads', CASES)
def test_block_forward_backward(T, B, nhx, nh, heads):
    from srvp_amd.posterior import AttentionPosterior
    torch.manual_seed(T + nh)
    net = AttentionPosterior(nhx, nh, heads)
    for m in (net.norm, net.out_norm, net.last_norm):
        m.weight.data += 0.3 * torch.randn(nh)
    g = torch.Generator().manual_seed(3)
    hx, d = torch.randn(T, B, nhx, generator=g), torch.randn(T * B, nh, generator=g)
    names = [k for k, _ in net.named_parameters()]
    leaves = {f'inf_z.{k}': p.detach().double().requires_grad_() for k, p in net.named_parameters()}
    x = hx.double().requires_grad_()
    ref = plain_block(leaves, x, net.heads).view(T * B, nh)
    gref = torch.autograd.grad(ref, [x] + list(leaves.values()), d.double())
    net = net.cuda()
    hz, saved = net.run(hx.cuda(), True)
    assert rel(hz, ref.detach()) < 2e-6, rel(hz, ref.detach())
    grads = {f'inf_z.{k}': torch.zeros_like(p) for k, p in net.named_parameters()}
    d_hx = torch.full((T * B, nhx), 0.5, device='cuda')
    keep = net.backward(hx.cuda(), d.cuda(), saved, grads, 'inf_z', d_hx)
    # fp32 sums of up to a few hundred terms in each of nine operators behind each other, conditioned by three norms
    assert rel(d_hx - 0.5, gref[0].view(T * B, nhx)) < 2e-5
    for k, r in zip(names, gref[1:]):
        assert rel(grads[f'inf_z.{k}'], r) < 2e-5 or r.norm() < 1e-6, (k, rel(grads[f'inf_z.{k}'], r))
    del keep
    assert net.run(hx.cuda(), False)[1] is None and torch.equal(net.run(hx.cuda(), False)[0], hz)


def small_model(heads=2, archi='vgg'):
    import srvp_amd
    ctor = (64, 3, 8, 16, 5, 7, True, 2, 24, 3, 40, 4, archi)
    torch.manual_seed(1)
    model = srvp_amd.StochasticLatentResidualVideoPredictor(*ctor, posterior='attention', posterior_heads=heads)
    model.init(res_gain=1.2)
    return ctor, model


def test_training_step_against_oracle(monkeypatch):
    """Forward, ELBO and every gradient of a whole step: the oracle with its LSTM exchanged for the plain block."""
    import srvp_amd
    from oracle import srvp_oracle as O
    from srvp_amd import train as T_
    ctor, model = small_model()
    assert not any('lstm' in k.lower() or 'weight_hh' in k for k in model.state_dict())
    monkeypatch.setattr(O, 'lstm', lambda sd, prefix, x: plain_block(sd, x, 2, prefix))
    sd = {k: v.detach().clone() for k, v in model.state_dict().items()}
    T, B, ne = 5, 3, 2
    g = torch.Generator().manual_seed(123)
    x = torch.rand(T, B, 3, 64, 64, generator=g)
    tape = dict(t_skip=torch.randint(T, (B,), generator=g), t_w=torch.stack([torch.randperm(T, generator=g)[:2] for _ in range(B)], 1),
                eps_y0=torch.randn(B, 5, generator=g), eps_z=torch.randn(T - 1, B, 7, generator=g))
    hp = dict(obs_scale=0.2, beta_y=1.0, beta_z=1.0, l2_res=1.0)
    ref, _, gref = O.train_step(sd, O.make_cfg(*ctor), x, ne, tape, hp)
    model = model.to('cuda:0').train().set_precision('fp32')
    opt = srvp_amd.DotDict(dict(n_euler_steps=ne, **hp))
    optim = srvp_amd.FusedAdam(model, lr=3e-4)
    for _ in range(2):                                   # (the second pass: buffers and streams in their steady state)
        optim.zero_grad()
        acc = T_.fused_step(model, x.to('cuda:0'), opt, tape=tape)
        torch.cuda.synchronize()
        loss = sum(acc.cpu().tolist()) / B
        assert abs(loss - ref['loss']) / abs(ref['loss']) < 1e-5
        for k, p in model.named_parameters():
            # the tolerance of the fp32 mode's gradients (two fp32 summation orders of this ill-conditioned network differ by up to 1e-2 on its encoder)
            if k.startswith(('inf_z', 'q_z')):
                assert rel(p.grad, gref[k]) < 2e-3, (k, rel(p.grad, gref[k]))
    before = model.inf_z.qkv.weight.detach().clone()
    optim.step()
    assert not torch.equal(before, model.inf_z.qkv.weight)
    out = T_.train(model, optim, None, x, torch.device('cuda:0'), opt)
    assert all(v == v for v in out)


def test_single_frames_equal_the_sequence():
    ctor, model = small_model(heads=3)
    model = model.cuda().eval()
    g = torch.Generator().manual_seed(7)
    T, B = 9, 4
    hx = torch.randn(T, B, 16, generator=g).cuda()
    hz, _ = model.inf_z.run(hx, False)
    stream = model.posterior_stream(B)
    for again in range(2):
        for t in range(T):
            h, p = stream.step(hx[t])
            assert rel(h, hz.view(T, B, -1)[t]) < 2e-6
            assert rel(p, h.double() @ model.q_z.weight.double().t() + model.q_z.bias.double()) < 2e-6
        stream.reset()
    # one row starts over, the others go on
    for t in range(3):
        stream.step(hx[t])
    stream.reset([1])
    mixed = hx[3].clone()
    mixed[1] = hx[0, 1]
    h, _ = stream.step(mixed)
    want = hz.view(T, B, -1)[3].clone()
    want[1] = hz.view(T, B, -1)[0, 1]
    assert rel(h, want) < 2e-6
    with pytest.raises(ValueError):
        stream.step(hx[0, :2])
    with pytest.raises(ValueError):
        stream.step(hx[0].cpu())


def test_quantized_inference():
    from srvp_amd import temporal
    ctor, model = small_model()
    model = model.cuda().eval()
    g = torch.Generator().manual_seed(8)
    hx = torch.randn(6, 5, 16, generator=g).cuda()
    net = model.inf_z
    exact, _ = net.run(hx, False)
    model.quantize_posterior()
    (wq, ws), _, _ = net.quantized()
    with torch.no_grad():
        u, n, qkv = net._inputs(hx.view(30, 16), net.quantized())
        xq, xs = temporal.rms_norm_int8(u, net.norm.weight)
    assert n is None
    want = (xq.double() @ wq.double().t()) * xs.double().view(-1, 1) * ws.double()
    assert rel(qkv, want) < 1e-6
    got, _ = net.run(hx, False)
    # rows and weights in steps of max / 127: each product's operands are off by at most half a step, 1 / 254 of the largest of a row or of a channel; a
    # row's largest is at most sqrt(24) times its root mean square, so two such products in a row move a unit-norm block by less than a few percent
    assert 0 < rel(got, exact) < 0.1
    stream = model.posterior_stream(5)
    for t in range(6):
        h, _ = stream.step(hx[t])
        assert rel(h, got.view(6, 5, -1)[t]) < 0.02              # (a value next to a border may fall on its other side)
    # new weights are quantised again, a training pass drops them
    with torch.no_grad():
        net.qkv.weight.mul_(1.5)
    assert torch.equal(net.quantized()[0][0], temporal.quantize_int8(net.qkv.weight.detach())[0])
    net.run(hx, True)
    assert net.quantized() is None
    model.quantize_posterior()
    model.quantize_posterior(False)
    assert torch.equal(net.run(hx, False)[0], net.run(hx, True)[0])


def test_evaluation_paths():
    """forward, sample and encode / generate of a model in eval mode, fp32 and 8-bit posterior."""
    ctor, model = small_model(archi='dcgan')
    model = model.cuda().eval()
    g = torch.Generator().manual_seed(5)
    x = torch.rand(3, 2, 3, 64, 64, generator=g).cuda()
    for q in (False, True):
        model.quantize_posterior(q)
        x_, y, z, w, qy0, qz, pz, res = model(x, 6, dt=0.5)
        assert x_.shape == (6, 2, 3, 64, 64) and torch.isfinite(x_).all() and qz.shape == (2, 2, 14)
        assert torch.isfinite(model.sample(x, 5, 3, dt=0.5)).all()
        hx, _ = model.encode(x)
        y0, _ = model.infer_y(hx[:2])
        assert torch.isfinite(model.generate(y0, hx, 4, 1.0)[0]).all()


def test_lstm_model_refuses():
    import srvp_amd
    ctor = (64, 3, 8, 16, 5, 7, True, 2, 24, 3, 40, 4, 'vgg')
    model = srvp_amd.StochasticLatentResidualVideoPredictor(*ctor).cuda()
    for f in (model.quantize_posterior, lambda: model.posterior_stream(2)):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize('change', ['out.data', 'qkv.data in place', 'out.data in place', 'optimizer', 'state dict', 'parameter'])
def test_quantized_inference_uses_the_weights_of_the_call(change):
    """Whatever changes a weight after quantize_posterior: the next sequence, and the next frame of a stream, run on 8-bit copies of the new one."""
    import srvp_amd
    from srvp_amd.posterior import AttentionPosterior, PosteriorStream
    ctor, model = small_model()
    model = model.cuda().eval()
    net = model.inf_z
    optim = srvp_amd.FusedAdam(model, lr=1e-2)
    optim.zero_grad()
    g = torch.Generator().manual_seed(9)
    hx = torch.randn(6, 5, 16, generator=g).cuda()
    model.quantize_posterior()
    before = net.run(hx, False)[0].clone()
    stream = model.posterior_stream(5)
    first = stream.step(hx[0])[0].clone()
    other = (0.3 * torch.randn(24, 24, generator=g)).cuda()
    if change == 'out.data':
        net.out.weight.data = other
    elif change == 'qkv.data in place':
        net.qkv.weight.data.mul_(-1.5)
    elif change == 'out.data in place':
        net.out.weight.data.copy_(other)
    elif change == 'optimizer':
        model._flat[1].normal_()
        optim.step()
    elif change == 'state dict':
        net.load_state_dict({**net.state_dict(), 'out.weight': other})
    else:
        net.out.weight = torch.nn.Parameter(other)
    fresh = AttentionPosterior(16, 24, 2).cuda()
    fresh.load_state_dict({k: v.clone() for k, v in net.state_dict().items()})
    fresh.quantize()
    want = fresh.run(hx, False)[0]
    got = net.run(hx, False)[0]
    assert torch.equal(got, want) and not torch.equal(got, before)
    stream.reset()
    again = PosteriorStream(fresh, model.q_z, 5, 'cuda')
    frame = stream.step(hx[0])[0]
    assert torch.equal(frame, again.step(hx[0])[0]) and not torch.equal(frame, first)


@pytest.mark.parametrize('default', [torch.float64, torch.bfloat16])
def test_default_type_does_not_matter(default):
    """The block's buffers are float32 whatever torch's default type is (a smaller one would be written past its end)."""
    from srvp_amd.posterior import AttentionPosterior, PosteriorStream
    torch.manual_seed(2)
    net, qz = AttentionPosterior(16, 24, 2).cuda(), torch.nn.Linear(24, 14).cuda()
    g = torch.Generator().manual_seed(4)
    hx, d = torch.randn(7, 3, 16, generator=g).cuda(), torch.randn(21, 24, generator=g).cuda()

    def everything():
        out = []
        net.drop_quantized()
        hz, saved = net.run(hx, True)
        grads = {f'inf_z.{k}': torch.zeros_like(p) for k, p in net.named_parameters()}
        d_hx = torch.zeros(21, 16, dtype=torch.float32, device='cuda')
        keep = net.backward(hx, d, saved, grads, 'inf_z', d_hx)
        for bits in (False, True):
            if bits:
                net.quantize()
            out.append(net.run(hx, False)[0])
            stream = PosteriorStream(net, qz, 3, 'cuda')
            for t in range(3):
                out += stream.step(hx[t])
        torch.cuda.synchronize()
        del keep
        return [hz, d_hx] + list(grads.values()) + out
    want = everything()
    torch.set_default_dtype(default)
    try:
        got = everything()
    finally:
        torch.set_default_dtype(torch.float32)
    for a, b in zip(got, want):
        # (weight gradients are sums over parts of the rows in any order)
        assert a.dtype is torch.float32 and rel(a, b) < 1e-5


def test_encodings_of_any_strides():
    """Slices and transposed views of encodings: the results of their copies; other types than float32 are refused."""
    from srvp_amd.posterior import AttentionPosterior
    torch.manual_seed(2)
    net = AttentionPosterior(16, 24, 2).cuda()
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(7, 3, 40, generator=g).cuda()
    for hx in (wide[..., 5:21], wide[:, :, :16], torch.randn(3, 7, 16, generator=g).cuda().transpose(0, 1)):
        copy = hx.clone(memory_format=torch.contiguous_format)
        d = torch.randn(24, 21, generator=g).cuda().t()
        results = []
        for x, dy in ((hx, d), (copy, d.contiguous())):
            hz, saved = net.run(x, True)
            grads = {f'inf_z.{k}': torch.zeros_like(p) for k, p in net.named_parameters()}
            d_hx = torch.zeros(21, 16, device='cuda')
            later = []
            keep = net.backward(x, dy, saved, grads, 'inf_z', d_hx, defer=later)
            assert any(torch.is_tensor(a) and a.shape == (21, 16) and torch.equal(a, copy.view(21, 16)) for a in keep)      # (a slice's copy lives until the deferred launches end)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for f in later:
                    f(side.cuda_stream)
            del later
            torch.cuda.synchronize()
            results.append([hz, d_hx] + list(grads.values()))
            del keep
        assert torch.equal(results[0][0], results[1][0])
        for a, b in zip(*results):
            assert rel(a, b) < 1e-5
    for bad in (wide[..., :16].double(), wide[..., :16].bfloat16()):
        with pytest.raises(TypeError):
            net.run(bad, False)
    with pytest.raises(TypeError):
        AttentionPosterior(16, 24, 2).cuda().double().run(wide[..., :16], False)
    for name in ('inp', 'qkv', 'out'):
        net = AttentionPosterior(16, 24, 2).cuda()
        w = getattr(net, name).weight
        w.data = w.data.t().contiguous().t()              # (another order in memory)
        with pytest.raises(TypeError):
            net.run(wide[..., :16], False)

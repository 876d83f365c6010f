"""Units that keep their activations in 8 bits between the passes (set_saved_activations): outputs unchanged, gradients exactly those of the
plain engine on the kept values, half the bytes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _off():
    import keypoints_amd as ka
    yield
    ka.set_saved_activations(None)
    ka.runtime.set_keep_saved_activations(False)


def unit(kind, cfg, cin, cout, precision):
    import torch.nn as nn
    from keypoints_amd.models import knn, vgg
    torch.manual_seed(5)
    table = vgg.vgg_cfg if kind == 'encoder' else vgg.decoder_cfg
    layers = vgg.make_layers(table[cfg], nonlinearity=nn.LeakyReLU, nonlinearity_kwargs={'inplace': True}) if kind == 'encoder' else vgg.make_layers(table[cfg])
    u = knn.Unit(cin, cout, layers).cuda()
    u.precision = precision
    return u


CASES = [('encoder', 'VGG_PONG', 1, 16, (4, 1, 32, 32)), ('encoder', 'VGG_PONG_LAYERNECK', 1, 4, (3, 1, 84, 84)), ('decoder', 'VGG_PONG', 16, 1, (2, 16, 16, 16)),
         ('encoder', 'F', 3, 64, (2, 3, 64, 64)), ('decoder', 'F', 64, 3, (2, 64, 16, 16)), ('encoder', 'VGG_PACMAN', 3, 5, (2, 3, 18, 22))]


def tensors(ctx):
    """Every saved activation of a Unit's forward as (owner, key): inputs and conv outputs, each once."""
    seen, out = set(), []
    for sv in ctx.saved:
        for key in ('a', 'y'):
            t = sv[key]
            if t is not None and id(t) not in seen:
                seen.add(id(t))
                out.append((sv, key))
    if not isinstance(ctx.head_in, dict):
        out.append((ctx, 'head_in'))
    return out


def run(u, x, gout, change=None):
    for p in u.parameters():
        p.grad = None
    x = x.clone().requires_grad_()
    out = u(x)
    ctx = out.grad_fn
    if change is not None:
        change(ctx)
    kept = [sv[k] if isinstance(sv, dict) else getattr(sv, k) for sv, k in tensors(ctx)]
    out.backward(gout)
    return out.detach(), [x.grad.clone()] + [p.grad.clone() for p in u.parameters()], kept


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('precision', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('kind,cfg,cin,cout,shape', CASES)
def test_gradients_are_those_of_the_kept_values(kind, cfg, cin, cout, shape, precision, fmt):
    import keypoints_amd as ka
    from keypoints_amd import lowp
    from keypoints_amd.unit_engine import _Kept
    u = unit(kind, cfg, cin, cout, precision)
    state = {k: v.clone() for k, v in u.state_dict().items()}
    x = torch.randn(*shape, device='cuda')
    gout = torch.randn_like(u(x)) * 1e-2
    u.load_state_dict(state)

    def swap(ctx):   # the plain engine, every saved activation replaced by its 8-bit values
        news = {}
        for sv, key in tensors(ctx):
            t = sv[key] if isinstance(sv, dict) else getattr(sv, key)
            if sv is not ctx and sv.get('first_fused'):
                continue
            news[id(t)] = new = lowp.checkpoint8(t, fmt).unpack()
            if isinstance(sv, dict):
                sv[key] = new
            else:
                setattr(ctx, key, new)
        for f in [sv['fin'] for sv in ctx.saved] + [ctx.head_in]:
            if isinstance(f, dict):
                f['y'] = news[id(f['y'])]

    plain_out, want, _ = run(u, x, gout, swap)
    stats = {k: v.clone() for k, v in u.state_dict().items()}
    u.load_state_dict(state)
    ka.set_saved_activations(fmt)
    out, got, kept = run(u, x, gout)
    assert torch.equal(out, plain_out)
    assert all(torch.equal(v, stats[k]) for k, v in u.state_dict().items())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    packed = [k for k in kept if isinstance(k, _Kept)]
    assert len(packed) >= len(kept) - 1   # (the image in front of a recomputed first layer stays as it is)
    size = {'fp32': 4, 'bf16': 2, 'fp16': 2}[precision]
    for k in packed:
        assert k.tensor is None and k.packed.nbytes <= k.packed.values.numel() * (1 + 1 / 128) + 1 and k.packed.dtype.itemsize == size


def test_second_backward_with_kept_activations():
    import keypoints_amd as ka
    ka.set_saved_activations('e4m3')
    ka.runtime.set_keep_saved_activations(True)
    u = unit('encoder', 'VGG_PONG', 1, 16, 'bf16')
    x = torch.randn(2, 1, 32, 32, device='cuda', requires_grad=True)
    out = u(x)
    g = torch.randn_like(out)
    first = torch.autograd.grad(out, x, g, retain_graph=True)[0]
    second = torch.autograd.grad(out, x, g)[0]
    assert torch.equal(first, second)


@pytest.mark.parametrize('model,args,size', [('VGG_PONG_LAYERNECK', (1, 16, 3), 32), ('F', (3, 64, 4), 64)])
def test_train_step_and_its_graph(model, args, size):
    """A whole Transporter step in this mode, eager and replayed from one graph several times: the same losses, bit for bit."""
    import keypoints_amd as ka
    from keypoints_amd.models import transporter
    ka.set_saved_activations('e4m3')
    x, x_ = torch.rand(2, 2, args[0], size, size, device='cuda').unbind(0)

    def losses(graphed):
        torch.manual_seed(3)
        net = transporter.make(model, *args).cuda().set_precision('bf16')
        opt = ka.FusedAdam(net.parameters(), lr=1e-4).bind(net)
        if graphed:
            step = ka.graph.GraphedTrainStep(net, opt, None, (x, x_))
            return [step(x, x_).item() for _ in range(4)]
        opt.scaler = ka.amp.LossScaler(x.device, init_scale=1.0, growth_factor=1.0, backoff_factor=1.0, growth_interval=1 << 30, max_scale=1.0)
        opt.scaler.unit = True   # (the graph's optimizer kernels: step count and bias corrections on the device)
        out = []
        for _ in range(7):
            opt.zero_grad()
            loss = ka.l2_reconstruction_loss(net(x, x_)[0], x_)
            with ka.amp.scale_loss(loss, opt) as scaled:
                scaled.backward()
            opt.step()
            out.append(loss.item())
        return out

    eager, graphed = losses(False), losses(True)   # (three warm-up steps before the capture)
    assert eager[3:] == graphed, (eager, graphed)

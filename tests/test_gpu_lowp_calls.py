"""lowp and norm on what the framework itself returns and on layers as programs hold them; Units that a program checkpoints."""
import pytest
import torch

from test_gpu_t_interchange import _pong_net

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('op', ['norm', 'kept', 'linear'])
def test_a_returned_blend_passes_its_gradient_on(op):
    """TransporterNet.forward's second output as it is handed out (made on first use), against the tensor behind it: the same gradients in the
    feature encoder, and some at all."""
    from keypoints_amd import lowp, norm
    from keypoints_amd.models import functional as MF
    g = torch.Generator().manual_seed(31)
    xs, xt = torch.rand(4, 1, 84, 84, generator=g).cuda(), torch.rand(4, 1, 84, 84, generator=g).cuda()
    w = torch.randn(50, 84, generator=g).cuda()
    grads = []
    for lazy in (True, False):
        net = _pong_net('bf16')
        phi = net(xs, xt)[1]
        assert type(phi) is MF.LazyNCHW
        phi = phi if lazy else phi.materialize()
        leaf = w.clone().requires_grad_()
        y = lowp.linear8(phi, leaf) if op == 'linear' else norm.layer_norm(phi, leaf[0], keep='e4m3' if op == 'kept' else None)
        (y * y).mean().backward()
        gr = [leaf.grad] + [p.grad.detach().clone() for p in net.feature.parameters() if p.grad is not None]
        assert len(gr) > 1 and any(float(t.abs().max()) > 0 for t in gr[1:])
        grads.append(gr)
    assert len(grads[0]) == len(grads[1]) and all(torch.equal(a, b) for a, b in zip(*grads))


def test_a_layer_with_and_without_gradients():
    from keypoints_amd import lowp
    g = torch.Generator().manual_seed(5)
    for rows, K, N in ((300, 200, 130), (1, 77, 5), (2100, 640, 700)):
        x = torch.randn(rows, K, generator=g).bfloat16().cuda()
        w, b = torch.nn.Parameter(torch.randn(N, K, generator=g).cuda()), torch.nn.Parameter(torch.randn(N, generator=g).cuda())
        y = lowp.linear8(x, w, b)
        with torch.no_grad():
            assert torch.equal(lowp.linear8(x, w, b), y) and torch.equal(lowp.linear8(x.clone().requires_grad_(), w, b), y)


def test_many_rows_without_gradients():
    """More rows than one sum takes, with a Parameter as weight."""
    from keypoints_amd import lowp
    rows = lowp.MOST + 200
    x = torch.randn(rows, 8, device='cuda', dtype=torch.bfloat16)
    w = torch.nn.Parameter(torch.randn(16, 8, device='cuda'))
    with torch.no_grad():
        y = lowp.linear8(x, w)
        assert torch.equal(y[-300:], lowp.linear8(x[-300:].contiguous(), w)) and torch.equal(y[:300], lowp.linear8(x[:300].contiguous(), w))


@pytest.mark.parametrize('wtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('most', [256, 1024, 1920])
def test_a_batch_in_parts_is_the_whole_batch(monkeypatch, most, wtype):
    """Whole numbers, whose sums are exact in any grouping: a step that packs its batch in parts gives what one part gives, bit for bit."""
    from keypoints_amd import lowp
    g = torch.Generator().manual_seed(8)
    numbers = lambda *s: torch.randint(-7, 8, s, generator=g).float()
    wide = numbers(2049, 150).bfloat16().cuda()
    for x in (wide[:, 3:133], wide[:2048, :130].contiguous().view(2, 1024, 130)):
        leaves = [x.detach().clone().requires_grad_() if x.dim() == 3 else x.detach().requires_grad_(), numbers(70, 130).to(wtype).cuda().requires_grad_(),
                  numbers(70).cuda().requires_grad_()]
        dy = numbers(x.numel() // 130, 70).bfloat16().cuda().view(*x.shape[:-1], 70)
        got = []
        for n in (lowp.MOST, most):
            monkeypatch.setattr(lowp, 'MOST', n)
            y = lowp.linear8(*leaves)
            got.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
            for i in range(3):   # ... and each gradient by itself
                alone = [t.detach().requires_grad_(i == k) for k, t in enumerate(leaves)]
                one, = torch.autograd.grad(lowp.linear8(*alone), alone[i], dy)
                assert torch.equal(one, got[-1][1 + i])
            for t in leaves:
                t.requires_grad_()
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert torch.equal(got[1][2], (dy.reshape(-1, 70).double().t().contiguous() @ x.reshape(-1, 130).double()).float().to(wtype))
        monkeypatch.undo()


@pytest.mark.parametrize('N,K', [(16, 8), (300, 260)])
def test_a_training_step_of_more_rows_than_one_sum_takes(N, K):
    """128 frames of 256 x 256 and some more, as rows of -1, 0 and 1: sums stay far below 2^24 and are exact."""
    from keypoints_amd import lowp
    rows = 128 * 256 * 256 + 77
    g = torch.Generator(device='cuda').manual_seed(9)
    few = lambda *s: torch.randint(-1, 2, s, generator=g, device='cuda', dtype=torch.int8)
    x, w, b, dy = few(rows, K).bfloat16().requires_grad_(), few(N, K).float().requires_grad_(), few(N).float().requires_grad_(), few(rows, N).bfloat16()
    y = lowp.linear8(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = torch.zeros(N, K, device='cuda', dtype=torch.float64)
    sums = torch.zeros(N, device='cuda', dtype=torch.float64)
    with torch.no_grad():
        for at in range(0, rows, 1 << 20):
            part = slice(at, at + (1 << 20))
            xd, dyd = x[part].double(), dy[part].double()
            want += torch.mm(dyd.t().contiguous(), xd)
            sums += dyd.sum(0)
            assert torch.equal(y[part], (torch.mm(xd, w.double().t().contiguous()) + b.double()).bfloat16())
            assert torch.equal(dx[part], torch.mm(dyd, w.double()).bfloat16())
    assert want.abs().max() < 1 << 20 and torch.equal(dw, want.float()) and torch.equal(db, sums.float())


def test_saved_forms_given_back_strided():
    """Hooks that give the 8-bit copy and the statistics back as parts of wider tensors."""
    from keypoints_amd import lowp, norm
    g = torch.Generator().manual_seed(6)
    x, w, weight = torch.randn(37, 300, generator=g).bfloat16().cuda(), torch.randn(300, generator=g).cuda(), torch.randn(70, 300, generator=g).cuda()
    dy = torch.randn(37, 70, generator=g).bfloat16().cuda()

    def step():
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_(), weight.clone().requires_grad_()]
        return leaves, lowp.linear8(norm.layer_norm(leaves[0], leaves[1], keep='e4m3'), leaves[2])

    leaves, y = step()
    want = torch.autograd.grad(y, leaves, dy)
    for back in (lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]], lambda t: torch.stack([t, t], 1).flatten(0, 1)[::2]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), back):
            leaves, y = step()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


@pytest.mark.parametrize('reentrant', [True, False])
def test_a_checkpointed_keypoint_encoder(reentrant):
    """The encoder that runs in a side block, wrapped by torch.utils.checkpoint: the gradients of the unwrapped one, read by the optimizer's
    stream right after the backward."""
    from torch.utils.checkpoint import checkpoint

    class Again(torch.nn.Module):
        def __init__(self, unit, on):
            super().__init__()
            self.unit, self.on = unit, on

        def forward(self, x):
            return checkpoint(self.unit, x, use_reentrant=reentrant) if self.on and torch.is_grad_enabled() else self.unit(x)

        @property
        def out_block(self):
            return self.unit.out_block

    g = torch.Generator().manual_seed(7)
    xs, xt = torch.rand(4, 1, 84, 84, generator=g).cuda(), torch.rand(4, 1, 84, 84, generator=g).cuda()
    grads = []
    for on in (False, True):
        net = _pong_net('fp32')
        net.keypoint = Again(net.keypoint, on)
        x = xt.clone().requires_grad_()
        out = net(xs, x)[0]
        (out * out).mean().backward()
        grads.append([x.grad.clone()] + [p.grad.detach().clone() for p in net.parameters() if p.grad is not None])
    assert len(grads[0]) == len(grads[1]) > 1 and all(torch.equal(a, b) for a, b in zip(*grads))

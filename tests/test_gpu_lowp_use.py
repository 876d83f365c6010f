"""lowp and norm as programs use them: strides, empty batches, partial gradients, streams, graphs, not-a-numbers, long tensors, and a run of
them together."""
import pytest
import torch

from blocks8 import quantise, same

pytestmark = pytest.mark.gpu


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def views(seed, rows, width, dtype=torch.bfloat16):
    """Tensors of `rows` x `width` numbers that lie in memory in different ways."""
    base = rnd(rows, width, seed=seed, dtype=dtype)
    wide = torch.zeros(rows, width + 13, dtype=dtype, device='cuda')
    wide[:, 5:5 + width] = base
    odd = torch.zeros(rows * width + 3, dtype=dtype, device='cuda')
    odd[3:] = base.flatten()
    every = torch.zeros(2 * rows, width, dtype=dtype, device='cuda')
    every[::2] = base
    return base, [wide[:, 5:5 + width], odd[3:].view(rows, width), base.t().contiguous().t(), every[::2], base.view(1, rows, 1, width),
                  base.view(rows, 1, width).expand(rows, 1, width)]


@pytest.mark.parametrize('width', [64, 129, 1000])
def test_strides(width):
    from keypoints_amd import lowp, norm
    w, b = rnd(width, seed=1, dtype=torch.float32), rnd(width, seed=2, dtype=torch.float32)
    weight = rnd(70, width, seed=3, dtype=torch.float32)
    dense, xs = views(4, 37, width)
    dyd, dys = views(5, 37, width)
    gyd, gys = views(6, 37, 70)

    def results(x, dy, gy):
        x = x.detach().requires_grad_()
        leaves = [t.clone().requires_grad_() for t in (w, b, weight)]
        y = norm.layer_norm(x, leaves[0], leaves[1])
        z = lowp.linear8(x, leaves[2])
        out = [y, z, *torch.autograd.grad(y, (x, *leaves[:2]), dy.view(y.shape) if dy.dim() != y.dim() else dy),
               *torch.autograd.grad(z, (x, leaves[2]), gy.view(z.shape) if gy.dim() != z.dim() else gy),
               lowp.pack8(x).unpack(), lowp.linear8(x.detach(), lowp.pack8(weight), None)]
        return [t.detach().reshape(-1) for t in out]

    want = results(dense, dyd, gyd)
    for x in xs:
        assert all(torch.equal(a, c) for a, c in zip(results(x, dyd, gyd), want))
    for dy, gy in zip(dys, gys):
        if dy.dim() == 2:
            assert all(torch.equal(a, c) for a, c in zip(results(dense, dy, gy), want))
    wt = weight.t().contiguous().t()
    assert torch.equal(lowp.linear8(dense, wt), lowp.linear8(dense, weight))


def test_empty_and_impossible_shapes():
    from keypoints_amd import lowp, norm
    w = rnd(8, dtype=torch.float32).requires_grad_()
    x = torch.zeros(0, 8, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    y = norm.layer_norm(x, w, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 8) and torch.equal(dw, torch.zeros_like(w))
    weight = rnd(5, 8, dtype=torch.float32).requires_grad_()
    bias = rnd(5, dtype=torch.float32).requires_grad_()
    y = lowp.linear8(x, weight, bias)
    grads = torch.autograd.grad(y, (x, weight, bias), torch.zeros_like(y))
    assert y.shape == (0, 5) and grads[0].shape == (0, 8) and not grads[1].any() and not grads[2].any()
    none = torch.zeros(0, 8, device='cuda')
    x2 = rnd(3, 8).requires_grad_()
    y = lowp.linear8(x2, none.requires_grad_())
    assert y.shape == (3, 0) and not torch.autograd.grad(y, x2, torch.zeros_like(y))[0].any()
    assert lowp.linear8(x.detach(), lowp.pack8(weight)).shape == (0, 5) and lowp.linear8(x2.detach(), lowp.pack8(none)).shape == (3, 0)
    assert lowp.matmul8(lowp.pack8(x), lowp.pack8(weight)).shape == (0, 5)
    kept = lowp.checkpoint8(x)
    assert kept.unpack().shape == (0, 8) and kept.nbytes == 0
    flat = torch.zeros(3, 0, device='cuda')
    for call in (lambda: norm.layer_norm(flat), lambda: lowp.pack8(flat), lambda: lowp.linear8(flat, torch.zeros(2, 0, device='cuda')),
                 lambda: norm.layer_norm(torch.zeros((), device='cuda'))):
        with pytest.raises(ValueError):
            call()


def test_refusals_on_the_device():
    from keypoints_amd import lowp, norm
    x, weight = rnd(4, 8), rnd(6, 8, dtype=torch.float32)
    cases = [(ValueError, lambda: norm.layer_norm(x, torch.ones(7, device='cuda'))), (ValueError, lambda: norm.layer_norm(x, None, torch.ones(8, 1, device='cuda'))),
             (ValueError, lambda: norm.layer_norm(x, torch.ones(8, device='cuda', dtype=torch.long))), (ValueError, lambda: norm.layer_norm(x, eps=-1.0)),
             (ValueError, lambda: norm.layer_norm(x, eps=float('nan'))), (ValueError, lambda: norm.layer_norm(x, keep='fp8')),
             (TypeError, lambda: norm.layer_norm(x.double())), (RuntimeError, lambda: norm.layer_norm(x, torch.ones(8))),
             (ValueError, lambda: lowp.linear8(x, weight[:, :7])), (ValueError, lambda: lowp.linear8(x, weight, torch.ones(5, device='cuda'))),
             (TypeError, lambda: lowp.linear8(x.long(), weight)), (TypeError, lambda: lowp.linear8(x, weight.double())),
             (RuntimeError, lambda: lowp.linear8(x, weight.cpu())), (ValueError, lambda: lowp.linear8(x, weight, fmt='e4m2')),
             (ValueError, lambda: lowp.linear8(x, weight, grad_fmt='')), (TypeError, lambda: lowp.linear8(x, lowp.checkpoint8(weight))),
             (RuntimeError, lambda: lowp.linear8(x.clone().requires_grad_(), lowp.pack8(weight))),
             (TypeError, lambda: lowp.matmul8(lowp.checkpoint8(x), lowp.pack8(weight)))]
    for kind, call in cases:
        with pytest.raises(kind):
            call()
    with torch.no_grad():
        assert torch.equal(lowp.linear8(x.clone().requires_grad_(), lowp.pack8(weight)), lowp.linear8(x, lowp.pack8(weight)))
    # a first-order gradient with a graph is fine, a second one is not
    leaf = x.float().requires_grad_()
    first, = torch.autograd.grad(norm.layer_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


@pytest.mark.parametrize('which', range(1, 8))
def test_only_the_gradients_asked_for(which):
    from keypoints_amd import lowp, norm
    full = {}
    for mask in (7, which):
        x, w, b = rnd(300, 96, seed=1), rnd(96, seed=2, dtype=torch.float32), rnd(96, seed=3, dtype=torch.float32)
        W, B = rnd(140, 96, seed=4, dtype=torch.float32), rnd(140, seed=5, dtype=torch.float32)
        for f, (args, gy) in dict(norm=((x, w, b), rnd(300, 96, seed=6)), kept=((x, w, b), rnd(300, 96, seed=6)), linear=((x, W, B), rnd(300, 140, seed=7))).items():
            args = [a.clone().requires_grad_(bool(mask >> i & 1)) for i, a in enumerate(args)]
            y = lowp.linear8(*args) if f == 'linear' else norm.layer_norm(*args, keep='e4m3' if f == 'kept' else None)
            got = torch.autograd.grad(y, [a for a in args if a.requires_grad], gy)
            full.setdefault(f, {})[mask] = [y.detach(), dict(zip([i for i in range(3) if mask >> i & 1], got))]
    for f, by in full.items():
        assert torch.equal(by[7][0], by[which][0])
        for i, g in by[which][1].items():
            assert torch.equal(g, by[7][1][i]), (f, i)


def test_norm_gradient_against_differences():
    """Directional derivatives of sum(c * layer_norm) in fp32, central differences with h = 2^-7.  With z = |v| h of the order of 2^-7 the
    third derivative adds h^2 / 6 * |f'''| (rows of unit variance: |f'''| <= 20 |c| |v|^3), rounding 2^-23 * |f| / h; both bounded by the sums
    of magnitudes below."""
    from keypoints_amd import norm
    for rows, width in ((3, 40), (5, 300)):
        x, w, b, c = rnd(rows, width, dtype=torch.float32), 1 + 0.1 * rnd(width, seed=1, dtype=torch.float32), rnd(width, seed=2, dtype=torch.float32), rnd(rows, width, seed=3, dtype=torch.float32)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(norm.layer_norm(*leaves), leaves, c)
        f = lambda *a: (norm.layer_norm(*[t.detach() for t in a]).double() * c.double()).sum().item()
        h = 2.0 ** -7
        for i, g in enumerate(grads):
            v = rnd(*leaves[i].shape, seed=9 + i, dtype=torch.float32)
            args = [[t.detach() + s * h * v if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1)]
            want = (f(*args[0]) - f(*args[1])) / (2 * h)
            size = (c.abs() * (1 + v.abs().amax()) ** 3).sum().item()
            assert abs((g.double() * v.double()).sum().item() - want) <= size * (20 * h * h / 6 + 2.0 ** -20 / h)


def test_not_a_numbers_stay_in_their_rows():
    from keypoints_amd import lowp, norm
    x = rnd(40, 200, seed=1)
    x[3, 7], x[11, 150], x[20, 0] = float('nan'), float('inf'), -float('inf')
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 11, 20]] = True
    w = rnd(30, 200, seed=2, dtype=torch.float32)
    clean = x.clone()
    clean[bad.cuda()] = 0
    for y, z in ((norm.layer_norm(x), norm.layer_norm(clean)), (lowp.linear8(x, w), lowp.linear8(clean, w)),
                 (lowp.linear8(x[:16], lowp.pack8(w)), lowp.linear8(clean[:16], lowp.pack8(w)))):
        n = y.shape[0]
        assert bool(y.cpu()[bad[:n]].isnan().any(1).all()) and torch.equal(y.cpu()[~bad[:n]], z.cpu()[~bad[:n]])
    # a batch that holds one: the weight's gradient says so (the loss scaler's check sees it)
    leaf = w.clone().requires_grad_()
    dw, = torch.autograd.grad(lowp.linear8(x, leaf), leaf, rnd(40, 30, seed=3))
    assert bool(dw[:, 7].isnan().all()) and bool(dw[:, 8].isfinite().all())


@pytest.mark.parametrize('keep', [None, 'e4m3'])
def test_an_overflow_stays_in_its_column(keep):
    """Row 0's element 0 is further from the mean than fp32 reaches: its normalised value is no number, every other one of the row is 0."""
    from keypoints_amd import norm
    x = rnd(3, 16, seed=1, dtype=torch.float32)
    x[0] = -4e37
    x[0, 0] = 3.4e38
    w = rnd(16, seed=2, dtype=torch.float32)
    dy = rnd(3, 16, seed=3, dtype=torch.float32)

    def grads(rows):
        leaves = [x[rows].clone().requires_grad_(), w.clone().requires_grad_(), w.clone().requires_grad_()]
        return torch.autograd.grad(norm.layer_norm(*leaves, keep=keep), leaves, dy[rows])
    dx, dw, db = grads(slice(0, 3))
    _, want, _ = grads(slice(1, 3))
    assert not dw[0].isfinite() and torch.equal(dw[1:], want[1:]) and bool(db.isfinite().all()) and bool(dx[1:].isfinite().all())


def test_equal_calls_give_equal_bits_on_any_stream():
    from keypoints_amd import lowp, norm
    x, w, b = rnd(5000, 384, seed=1), rnd(384, seed=2, dtype=torch.float32), rnd(384, seed=3, dtype=torch.float32)
    W, dy = rnd(200, 384, seed=4, dtype=torch.float32), rnd(5000, 200, seed=5)

    def work():
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, W)]
        y = lowp.linear8(norm.layer_norm(*leaves[:3], keep='e4m3'), leaves[3])
        return [y.detach(), lowp.checkpoint8(y).unpack(), *torch.autograd.grad(y, leaves, dy)]

    want = work()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:   # all three in flight at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, c) for a, c in zip(g, want))


def test_two_captured_steps_replayed_in_turn():
    """A training step of norm and projection, captured twice on one stream over different data; replays alternate with eager work on the same
    stream, and every one gives the eager result for what then lies in its inputs."""
    from keypoints_amd import lowp, norm
    w, b, W, B = rnd(256, seed=1, dtype=torch.float32), rnd(256, seed=2, dtype=torch.float32), rnd(160, 256, seed=3, dtype=torch.float32), rnd(160, seed=4, dtype=torch.float32)

    def step(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, W, B)]
        y = lowp.linear8(norm.layer_norm(*leaves[:3], keep='e5m2'), leaves[3], leaves[4], grad_fmt='e5m2')
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    s = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(s):
        for i in range(2):
            ins = [rnd(700, 256, seed=10 + i), rnd(700, 160, seed=20 + i)]
            step(*ins)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                out = step(*ins)
            graphs.append((g, ins, out))
        for r in range(4):
            for i, (g, ins, out) in enumerate(graphs):
                ins[0].copy_(rnd(700, 256, seed=30 + 2 * r + i))
                ins[1].copy_(rnd(700, 160, seed=50 + 2 * r + i))
                g.replay()
                other = step(rnd(700, 256, seed=90 + r), rnd(700, 160, seed=91 + r))   # eager work behind it on the stream
                want = step(*[t.clone() for t in ins])
                torch.cuda.synchronize()
                assert all(torch.equal(a, c) for a, c in zip(out, want)), (r, i)
                del other


def test_a_block_of_them_trains_as_its_parts():
    """norm -> expand -> LeakyReLU -> project back, on channels-last maps with FusedAdam: the gradients of the chain are those of its stages
    called one by one, and a step moves every parameter."""
    import keypoints_amd as ka
    from keypoints_amd import lowp, norm
    B, H, W, C = 2, 12, 10, 64
    maps = rnd(B, C, H, W, seed=1).contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)   # [B, H, W, C]
    params = [torch.nn.Parameter(t) for t in (1 + 0.1 * rnd(C, seed=2, dtype=torch.float32), 0.1 * rnd(C, seed=3, dtype=torch.float32),
                                              rnd(4 * C, C, seed=4, dtype=torch.float32) / 8, torch.zeros(4 * C, device='cuda'),
                                              rnd(C, 4 * C, seed=5, dtype=torch.float32) / 16, torch.zeros(C, device='cuda'))]
    act = lambda t: torch.nn.functional.leaky_relu(t, 0.01)
    x = maps.detach().requires_grad_()
    h = norm.layer_norm(x, params[0], params[1], keep='e4m3')
    u = lowp.linear8(h, params[2], params[3])
    v = act(u)
    y = lowp.linear8(v, params[4], params[5])
    gy = rnd(B, H, W, C, seed=6)
    got = torch.autograd.grad(y, [x, *params], gy, retain_graph=True)

    vd = v.detach().requires_grad_()
    dv, dw2, db2 = torch.autograd.grad(lowp.linear8(vd, params[4], params[5]), (vd, params[4], params[5]), gy)
    ud = u.detach().requires_grad_()
    du, = torch.autograd.grad(act(ud), ud, dv)
    hd = h.detach().requires_grad_()
    dh, dw1, db1 = torch.autograd.grad(lowp.linear8(hd, params[2], params[3]), (hd, params[2], params[3]), du)
    dx, dw, db = torch.autograd.grad(norm.layer_norm(x, params[0], params[1], keep='e4m3'), (x, params[0], params[1]), dh)
    assert all(torch.equal(a, c) for a, c in zip(got, (dx, dw, db, dw1, db1, dw2, db2)))

    opt = ka.FusedAdam(params, lr=1e-3)
    before = [p.detach().clone() for p in params]
    loss = ka.l2_reconstruction_loss(y.permute(0, 3, 1, 2).float(), maps.permute(0, 3, 1, 2).float())
    loss.backward()
    opt.step()
    assert all(bool((p != q).any()) and bool(p.isfinite().all()) for p, q in zip(params, before))


def test_tensors_past_two_to_the_thirty_one():
    from keypoints_amd import lowp, norm
    n = (1 << 31) + 64 * 37
    x = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
    tail = rnd(64 * 40, seed=1)
    x[-tail.numel():] = tail
    kept = lowp.checkpoint8(x)
    want, _ = quantise(torch.cat([torch.zeros((n - tail.numel()) % 128, dtype=torch.bfloat16), tail.cpu()]), 'e4m3')   # from the block the tail begins in
    assert same(kept.unpack()[-tail.numel():], want[-tail.numel():].to(torch.bfloat16))
    del kept
    rows = x.view(-1, 64)
    w, b = (1 + rnd(64, seed=2, dtype=torch.float32)).requires_grad_(), rnd(64, seed=3, dtype=torch.float32)
    y = norm.layer_norm(rows, w, b, keep='e4m3')
    small = norm.layer_norm(rows[-40:], w, b, keep='e4m3')
    assert torch.equal(y[-40:].detach(), small.detach())
    dy = torch.zeros_like(y)
    dy[-40:] = rnd(40, 64, seed=4)
    big, = torch.autograd.grad(y, w, dy)
    little, = torch.autograd.grad(small, w, dy[-40:].contiguous())
    assert torch.allclose(big, little, rtol=2.0 ** -18, atol=2.0 ** -18 * float(little.abs().max()))   # (40 products, added in another order)
    del x, y, dy, rows


def test_products_past_two_to_the_thirty_one():
    from keypoints_amd import lowp
    a, b = rnd(40001, 130, seed=1), rnd(56003, 130, seed=2)
    y = lowp.matmul8(lowp.pack8(a), lowp.pack8(b))
    for r, c in ((slice(0, 70), slice(0, 70)), (slice(-70, None), slice(-70, None)), (slice(-70, None), slice(0, 70)), (slice(20000, 20070), slice(30000, 30070))):
        part = lowp.matmul8(lowp.pack8(a[r]), lowp.pack8(b[c]))
        assert torch.allclose(y[r, c].float(), part.float(), rtol=2.0 ** -7, atol=1e-2)   # (another tile: one rounding apart)


@pytest.mark.parametrize('keep', [None, 'e4m3'])
def test_saved_tensors_that_come_back_with_other_strides(keep):
    """Saved-tensor hooks (offloading to the host, say) give a strided x back dense."""
    from keypoints_amd import lowp, norm
    wide = rnd(37, 400, seed=1)
    w, weight, dy = rnd(100, seed=2, dtype=torch.float32), rnd(100, 100, seed=3, dtype=torch.float32), rnd(37, 100, seed=4)

    def step():
        leaves = [wide.clone().requires_grad_(), w.clone().requires_grad_(), weight.clone().requires_grad_()]
        y = lowp.linear8(norm.layer_norm(leaves[0][:, 200:300], leaves[1], keep=keep), leaves[2])
        return leaves, y

    leaves, y = step()
    want = torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.cuda()):
        leaves, y = step()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))

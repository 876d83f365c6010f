"""keypoints_amd.norm on the GPU against the formulas in 64 bits."""
import pytest
import torch

from blocks8 import quantise

pytestmark = pytest.mark.gpu

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def oracle(x, w, b, dy, eps, kept):
    """y, dx, dw, db and a bound for each of what fp32 arithmetic may add: a sum's chain is at most 100 additions a row (32 elements in
    a thread, 10 lane and 16 wave steps, and the few operations around them), rows + 100 over the batch."""
    u = 2.0 ** -24
    x, w, b, dy = (t.detach().cpu().double() for t in (x, w, b, dy))
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    dxh = 100 * u * (xh.abs() + rstd * x.abs().amax(-1, keepdim=True))   # of xh: its own roundings, the mean's error, the deviation's
    y, by = xh * w + b, dxh * w.abs() + 4 * u * ((xh * w).abs() + b.abs())
    if kept:
        xh = (quantise(x, kept)[0] - mean) * rstd
        dxh = 100 * u * (xh.abs() + rstd * x.abs().amax(-1, keepdim=True))
    g = dy * w
    a, c = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - a - xh * c)
    da = 100 * u * g.abs().mean(-1, keepdim=True)
    dc = 100 * u * (g * xh).abs().mean(-1, keepdim=True) + (g.abs() * dxh).mean(-1, keepdim=True)
    bx = rstd * (100 * u * (g.abs() + a.abs() + (xh * c).abs()) + da + xh.abs() * dc + dxh * (c.abs() + dc))
    n = x.shape[0] + 100
    dw, bw = (dy * xh).sum(0), n * u * (dy * xh).abs().sum(0) + (dy.abs() * dxh).sum(0)
    db, bb = dy.sum(0), n * u * dy.abs().sum(0)
    return (y, by), (dx, bx), (dw, bw), (db, bb)


def close(got, want, dtype):
    want, bound = want
    got = got.detach().cpu().double()
    info = torch.finfo(TYPES[dtype])
    tol = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    assert got.shape == want.shape
    worst = ((got - want).abs() - tol).max().item()
    assert worst <= 0.0, f'off by {worst} beyond the bound'


def data(rows, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(torch.randn(width, generator=g))
    x = torch.randn(rows, width, generator=g) * spread + 0.5 * torch.randn(width, generator=g)
    return (x.to(TYPES[dtype]).cuda(), (1 + 0.3 * torch.randn(width, generator=g)).cuda(), (0.3 * torch.randn(width, generator=g)).cuda(),
            (1e-2 * torch.randn(rows, width, generator=g)).to(TYPES[dtype]).cuda())


@pytest.mark.parametrize('keep', [None, 'e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 2), (5, 7), (1, 8), (257, 16), (65, 31), (1030, 64), (33, 65), (70, 128), (9, 200), (40, 256), (300, 333),
                                        (50, 512), (7, 513), (21, 1000), (16, 1024), (4, 1025), (9, 2048), (5, 2050), (6, 4096), (3, 4100),
                                        (2, 8192), (3, 10000), (2, 16384), (2, 16385), (70, 20000)])
def test_layer_norm(rows, width, dtype, keep):
    from keypoints_amd.norm import layer_norm
    x, w, b, dy = data(rows, width, dtype)
    y, dx, dw, db = oracle(x, w, b, dy, 1e-5, keep)
    close(layer_norm(x, w, b), y, dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    out = layer_norm(x, w, b, keep=keep)
    close(out, y, dtype)
    grads = torch.autograd.grad(out, leaves, dy)
    close(grads[0], dx, dtype)
    close(grads[1], dw, 'fp32')
    close(grads[2], db, 'fp32')

"""Layer norm where a workgroup meets several rows one after another (the row ahead in registers, sums in alternating slots, the weight's
gradient over all of them, a last turn that is not full), and its gradient against differences of the formula."""
import pytest
import torch

from test_gpu_norm import close, data, oracle

pytestmark = pytest.mark.gpu


# the largest grids take 65536 rows of 64, 8192 of 513 .. 1024, 2048 of 1025 .. 2048, 1024 of up to 4096 and 512 of up to 16384 at once in the
# forward, half of that and less in the backward; 1024 rows past 16384
@pytest.mark.parametrize('keep', [None, 'e4m3', 'e5m2'])
@pytest.mark.parametrize('rows,width,dtype', [(70000, 64, 'bf16'), (70000, 33, 'fp16'), (150000, 7, 'fp32'), (20000, 256, 'bf16'), (17000, 500, 'fp32'),
                                              (8500, 513, 'bf16'), (9000, 1024, 'fp16'), (4200, 1025, 'fp32'), (4133, 1536, 'bf16'), (2100, 2048, 'bf16'),
                                              (2100, 2050, 'fp16'), (1100, 4096, 'fp32'), (1100, 4100, 'bf16'), (600, 8192, 'fp16'), (1100, 10000, 'bf16'),
                                              (1100, 10001, 'bf16'), (600, 16384, 'bf16'), (1030, 16392, 'bf16')])
def test_several_rows_a_workgroup(rows, width, dtype, keep):
    from keypoints_amd.norm import layer_norm
    x, w, b, dy = data(rows, width, dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    out = layer_norm(x, w, b, keep=keep)
    grads = torch.autograd.grad(out, leaves, dy)
    wants = oracle(x, w, b, dy, 1e-5, keep)
    for got, want, kind in zip((out, *grads), wants, (dtype, dtype, 'fp32', 'fp32')):
        close(got, want, kind)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), out)


def formula(x, w, b, eps=1e-5):
    m = x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt((x - m).square().mean(-1, keepdim=True) + eps) * w + b


@pytest.mark.parametrize('rows,width', [(3, 40), (5, 300), (4, 2100)])
def test_gradient_against_differences_of_the_formula(rows, width):
    """Directional derivatives of sum(c * y): fp32 gradients against central differences of the formula in fp64, h = 2^-17: the third derivative
    adds less than 2^-34 * 20 of the sum of magnitudes, rounding 2^-52 / h; both are far below what fp32 may add (`oracle`'s bounds and the
    gradient's own rounding).  c has a part along each of the two terms that the mean and the variance bring, so that a gradient without
    either, or without its bias, is off by 100 times the tolerance and more."""
    from keypoints_amd.norm import layer_norm
    g = torch.Generator().manual_seed(rows)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float().double()   # (numbers that fp32 holds)
    x, w, b = rnd(rows, width), (1 + 0.1 * rnd(width)).float().double(), rnd(width)
    hat = formula(x, torch.ones(width), 0.0)
    c = (((0.5 + hat) / w + 0.3 * rnd(rows, width))).float().double()   # c w: a mean of 0.5 and a correlation of 1 with the normalised row
    h = 2.0 ** -17
    leaves = [t.float().cuda().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, c.float().cuda())
    _, (dx, bx), (dw, bw), (db, bb) = oracle(x, w, b, c, 1e-5, None)
    v = [0.5 + hat + dx / dx.std(), dw / dw.std(), db / db.std()]       # directions along both terms and along the gradients
    want, tol = [], []
    for i, bound, full in ((0, bx, dx), (1, bw, dw), (2, bb, db)):
        ends = [(formula(*[t + s * h * v[j] if j == i else t for j, t in enumerate((x, w, b))]) * c).sum().item() for s in (1, -1)]
        size = (c.abs() * (1 + v[i].abs().amax()) ** 3 * (1 + w.abs())).sum().item()
        want.append((ends[0] - ends[1]) / (2 * h))
        tol.append(((bound + full.abs() * 2.0 ** -24) * v[i].abs()).sum().item() + size * (20 * h * h / 6 + 2.0 ** -52 / h))
        assert abs((full * v[i]).sum().item() - want[i]) <= tol[i]
        got = (grads[i].double().cpu() * v[i]).sum().item()
        assert abs(got - want[i]) <= tol[i], (i, got, want[i], tol[i])
    rstd = 1 / torch.sqrt((x - x.mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + 1e-5)
    gw = c * w
    for wrong in (rstd * (gw - hat * (gw * hat).mean(-1, keepdim=True)), rstd * (gw - gw.mean(-1, keepdim=True)), rstd * gw, 0 * gw):
        assert abs((wrong * v[0]).sum().item() - want[0]) > 100 * tol[0]
    assert abs(want[1]) > 100 * tol[1] and abs(want[2]) > 100 * tol[2]

"""keypoints_amd.lowp on the GPU against the format's definition in 64 bits (tests/blocks8.py)."""
import pytest
import torch

from blocks8 import quantise, same, to_type

pytestmark = pytest.mark.gpu

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def data(*shape, dtype='bf16', seed=0, spread=2.0):
    """Numbers whose size differs from row to row and inside a row, some zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    x = x * torch.exp(torch.randn(*shape, generator=g))
    x = torch.where(torch.rand(*shape, generator=g) < 0.05, torch.zeros_like(x), x)
    return x.to(TYPES[dtype]).cuda()


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('rows,width', [(1, 1), (1, 128), (3, 127), (5, 129), (7, 64), (33, 200), (130, 1000), (2, 4096), (1000, 8)])
def test_pack8_values(rows, width, dtype, fmt):
    from keypoints_amd import lowp
    x = data(rows, width, dtype=dtype)
    p = lowp.pack8(x, fmt)
    want, exps = quantise(x, fmt)
    assert same(p.unpack(torch.float32), want.float())     # (4 significant bits and 2^s: exact in fp32 above 2^-149)
    blocks = (width + 127) // 128
    assert torch.equal(p.scales[:, :blocks].cpu().int() - 127, exps.int())
    assert p.values.shape == (rows, blocks * 128) and int(p.values[:, width:].sum()) == 0
    assert same(p.unpack(), to_type(want, TYPES[dtype]))


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
def test_special_values(fmt):
    """Zero blocks, the format's border, subnormal inputs, infinities and not-a-numbers, alone and among numbers."""
    from keypoints_amd import lowp
    inf, nan, top = float('inf'), float('nan'), 448.0 if fmt == 'e4m3' else 57344.0
    rows = torch.zeros(14, 256)
    rows[1, 3] = top
    rows[2, 3] = top * (1 + 2.0 ** -20)
    rows[3, :4] = torch.tensor([1.0, inf, -inf, 2.0])
    rows[4, :3] = torch.tensor([nan, -3.0, 0.3])
    rows[5, :2] = torch.tensor([nan, inf])
    rows[6, 0] = 1e-40
    rows[7, :2] = torch.tensor([3.4e38, -1.0])
    rows[8, :3] = torch.tensor([2.0 ** -149, -2.0 ** -149, 2.0 ** -140])
    rows[9, :128] = torch.linspace(-1, 1, 128)
    rows[9, 128:] = torch.linspace(1, 1 + 2.0 ** -3, 128)                 # ties and their neighbours
    rows[10, :128] = 2.0 ** -torch.arange(128.)
    rows[11, :8] = -0.0
    rows[12, 200] = -inf
    rows[13] = 2.0 ** -130
    p = lowp.pack8(rows.cuda(), fmt)
    want, exps = quantise(rows, fmt)
    assert same(p.unpack(), to_type(want, torch.float32))
    assert torch.equal(p.scales[:, :2].cpu().int() - 127, exps.int())


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
def test_largest_numbers_stay_finite(dtype, fmt):
    from keypoints_amd import lowp
    top = torch.finfo(TYPES[dtype]).max
    x = torch.tensor([top, -top, top / 2, 1.0, -1.0, float('nan'), float('inf')], dtype=torch.float64).to(TYPES[dtype])
    want = to_type(quantise(x, fmt)[0], TYPES[dtype])
    got = lowp.checkpoint8(x.cuda(), fmt).unpack()
    assert same(got, want) and bool(got[:5].isfinite().all())


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('shape', [(1,), (127,), (128,), (129,), (3, 5, 7), (2, 64, 6, 10), (16, 1000), (1 << 18,)])
def test_checkpoint8(shape, dtype, fmt):
    from keypoints_amd import lowp
    x = data(*shape, 1, dtype=dtype).squeeze(-1)
    kept = lowp.checkpoint8(x, fmt)
    want, _ = quantise(x.reshape(-1), fmt)
    assert same(kept.unpack(), to_type(want, TYPES[dtype]).view(shape))
    assert kept.nbytes == x.numel() + (x.numel() + 127) // 128
    assert same(kept.unpack(torch.float32), want.float().view(shape))


def test_checkpoint8_keeps_strides():
    from keypoints_amd import lowp
    x = data(4, 6, 10, 24)
    for view in (x.permute(0, 3, 1, 2), x.transpose(0, 3), x[:, :, ::2], x[1:3], x.flatten(0, 2).t(), x[:, :1].expand(4, 3, 10, 24)):
        back = lowp.checkpoint8(view).unpack()
        dense = view if view.permute(sorted(range(view.dim()), key=lambda d: -view.stride(d))).is_contiguous() else view.contiguous()
        assert back.stride() == dense.stride() and back.shape == view.shape
        flat = dense.permute(sorted(range(dense.dim()), key=lambda d: -dense.stride(d))).reshape(-1)
        want = torch.empty_strided(dense.shape, dense.stride(), dtype=torch.float64)
        want.as_strided((flat.numel(),), (1,)).copy_(quantise(flat, 'e4m3')[0])
        assert same(back, want)


def product(a, b, dtype, bias=None):
    """(a b^T + bias, bound of its accumulation): every one of the K additions off by at most 2^-23 of the sum of magnitudes.  Results in
    16 bits come from the 8-bit matrix instruction, which aligns the products of 8 neighbouring elements to their largest and cuts each
    of the others off below 2^-13 of it: at most 7 * 2^-13 of the group's largest product, hence of the sum of magnitudes."""
    y = a @ b.t()
    bound = (a.abs() @ b.abs().t()) * ((a.shape[1] + 16) * 2.0 ** -23 + (0.0 if dtype == 'fp32' else 7 * 2.0 ** -13))
    if bias is not None:
        y = y + bias.double().cpu()
        bound = bound + (y.abs() + bias.double().cpu().abs()) * 2.0 ** -23
    return y, bound


def close(got, want, bound, dtype):
    """Within the bound and half a step of the output's type (its smallest subnormal where that is more)."""
    got = got.detach().cpu().double()
    info = torch.finfo(TYPES[dtype])
    tol = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps
    worst = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert got.shape == want.shape and worst <= 0.0, f'off by {worst} beyond the bound'


@pytest.mark.parametrize('fmts', [('e4m3', 'e4m3'), ('e5m2', 'e4m3'), ('e4m3', 'e5m2'), ('e5m2', 'e5m2')])
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (1, 64, 128), (2, 17, 129), (33, 31, 300), (64, 64, 512), (65, 70, 640), (129, 130, 1000),
                                   (200, 300, 256), (300, 260, 2048), (257, 513, 1100), (16, 500, 4096), (700, 16, 130)])
def test_matmul8(M, N, K, fmts):
    from keypoints_amd import lowp
    a, b = data(M, K, seed=1), data(N, K, seed=2)
    bias = torch.randn(N).cuda()
    qa, qb = quantise(a, fmts[0])[0], quantise(b, fmts[1])[0]
    pa, pb = lowp.pack8(a, fmts[0]), lowp.pack8(b, fmts[1])
    want, bound = product(qa, qb, 'fp32')
    close(lowp.matmul8(pa, pb, dtype=torch.float32), want, bound, 'fp32')
    want, bound = product(qa, qb, 'bf16', bias)
    close(lowp.matmul8(pa, pb, bias), want, bound, 'bf16')


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (1, 48, 200), (3, 1000, 512), (15, 33, 4096), (17, 130, 700), (130, 257, 129), (600, 300, 512)])
def test_linear8_serving(M, N, K, dtype):
    from keypoints_amd import lowp
    x, w = data(M, K, dtype=dtype, seed=3, spread=0.5), data(N, K, dtype='fp32', seed=4, spread=0.5) / K ** 0.5
    bias = torch.randn(N).cuda()
    for fmt in ('e4m3', 'e5m2'):
        packed = lowp.pack8(w, fmt)
        want, bound = product(quantise(x, fmt)[0], quantise(w, fmt)[0], dtype, bias)
        close(lowp.linear8(x, packed, bias, fmt=fmt), want, bound, dtype)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K', [(17, 1, 2100), (64, 16, 128), (65, 17, 1300), (300, 33, 4100), (129, 64, 2000), (1000, 65, 520), (2500, 100, 129), (5000, 128, 512)])
def test_linear8_few_columns(M, N, K, dtype):
    """The kernel that reads x once (N <= 128), also where the rule would take another, with rows at odd addresses."""
    from keypoints_amd import _lib, lowp
    from keypoints_amd.lowp import DTYPES, FORMATS
    from keypoints_amd._lib import call, ptr
    from keypoints_amd.runtime import stream_ptr
    wide = data(M, K + 3, dtype=dtype, seed=3, spread=0.5)
    x, w, bias = wide[:, 1:1 + K], data(N, K, dtype='fp32', seed=4, spread=0.5) / K ** 0.5, torch.randn(N).cuda()
    for fmt, wfmt in (('e4m3', 'e4m3'), ('e5m2', 'e4m3'), ('e4m3', 'e5m2')):
        packed = lowp.pack8(w, wfmt)
        want, bound = product(quantise(x, fmt)[0], quantise(w, wfmt)[0], dtype, bias)
        close(lowp.linear8(x, packed, bias, fmt=fmt), want, bound, dtype)
        y = torch.full((M, N + 2), -7.0, device='cuda', dtype=TYPES[dtype])   # rows further apart than they are long
        call('kp_q8_linear', ptr(wide) + wide.element_size(), K + 3, FORMATS[fmt], ptr(packed.values), packed.values.shape[1], ptr(packed.scales),
             packed.scales.shape[1], FORMATS[wfmt], ptr(bias), ptr(y), N + 2, M, N, K, DTYPES[x.dtype], stream_ptr())
        close(y[:, :N].contiguous(), want, bound, dtype)
        assert bool((y[:, N:] == -7.0).all())


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K', [(12301, 1, 1), (12300, 17, 100), (12500, 128, 128), (13000, 70, 255), (12289, 33, 384), (12290, 16, 520), (12400, 100, 1024)])
def test_linear8_few_columns_many_rows(M, N, K, dtype):
    """From no whole block to eight of them, each at a count of rows that takes the kernel by its rule."""
    from keypoints_amd import _lib, lowp
    assert _lib.lib().kp_q8_linear_suits(M, N, K, lowp.DTYPES[TYPES[dtype]]) and not (K <= 1024 and ((N + 15) // 16) * ((M + 15) // 16) <= 512)
    x, w, bias = data(M, K, dtype=dtype, seed=3, spread=0.5), data(N, K, dtype='fp32', seed=4, spread=0.5) / K ** 0.5, torch.randn(N).cuda()
    want, bound = product(quantise(x, 'e4m3')[0], quantise(w, 'e4m3')[0], dtype, bias)
    close(lowp.linear8(x, lowp.pack8(w), bias), want, bound, dtype)


@pytest.mark.parametrize('dtype,wtype', [('fp32', 'fp32'), ('bf16', 'fp32'), ('fp16', 'fp32'), ('bf16', 'bf16')])
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (1, 33, 130), (5, 128, 64), (129, 40, 257), (300, 520, 200), (1000, 70, 130)])
def test_linear8_training(M, N, K, dtype, wtype):
    """y and all gradients against the products of the definition's operands."""
    from keypoints_amd import lowp
    for fmt, gfmt in (('e4m3', 'e5m2'), ('e5m2', 'e4m3')):
        x = data(M, K, dtype=dtype, seed=5, spread=0.5).requires_grad_()
        w = (data(N, K, dtype='fp32', seed=6, spread=0.5) / K ** 0.5).to(TYPES[wtype]).requires_grad_()
        bias = torch.randn(N).cuda().requires_grad_()
        dy = data(M, N, dtype=dtype, seed=7, spread=0.5)
        y = lowp.linear8(x, w, bias, fmt=fmt, grad_fmt=gfmt)
        close(y, *product(quantise(x, fmt)[0], quantise(w, fmt)[0], dtype, bias.detach()), dtype)
        dx, dw, db = torch.autograd.grad(y, (x, w, bias), dy)
        close(dx, *product(quantise(dy, gfmt)[0], quantise(w, fmt, 0)[0].t(), dtype), dtype)
        close(dw, *product(quantise(dy, gfmt, 0)[0].t(), quantise(x, fmt, 0)[0].t(), wtype), wtype)
        d = dy.double().cpu()
        close(db, d.sum(0), d.abs().sum(0) * (M + 16) * 2.0 ** -24, 'fp32')
        assert dx.dtype == x.dtype and dw.dtype == w.dtype

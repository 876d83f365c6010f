"""Every kernel of the 8-bit products on whole numbers, where its answer is exact: the operands are small whole numbers times a power of two
that changes from block to block, so packing rounds nothing, no product is cut (see include/kp_hip.h: 13 bits below a group's largest; here all
are multiples of one and below 2^11) and every partial sum is a whole number below 2^24.  What comes out is the 64-bit product, rounded once:
one element too many, too few, twice or with its neighbour's exponent changes it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
FMTS = [('e4m3', 'e4m3'), ('e5m2', 'e4m3'), ('e4m3', 'e5m2'), ('e5m2', 'e5m2')]


def whole(rows, K, seed, dtype=torch.bfloat16):
    """Whole numbers -top .. top times 1, 2 or 4 by the block: rows differ, blocks differ.  top^2 * 4^2 * K < 2^24."""
    top = 7 if K <= 20000 else 5
    assert top * top * 16 * K + 64 < 1 << 24
    g = torch.Generator(device='cuda').manual_seed(seed)
    blocks = (K + 127) // 128
    x = torch.randint(-top, top + 1, (rows, blocks * 128), generator=g, device='cuda').float()
    two = 2.0 ** torch.randint(0, 3, (rows, blocks, 1), generator=g, device='cuda')
    return (x.view(rows, blocks, 128) * two).view(rows, -1)[:, :K].to(dtype).contiguous()


def exact(a, b, bias, dtype):
    y = torch.mm(a.double(), b.double().t().contiguous())   # (whole numbers below 2^53: exact in any order)
    return (y if bias is None else y + bias.double()).to(torch.float32).to(dtype)


# (tile, splits) of each case is the library's own answer, asserted: a rule that moves a case to another kernel fails here
@pytest.mark.parametrize('fmts', FMTS)
@pytest.mark.parametrize('tile,splits,M,N,K,dtype', [
    (64, 1, 65, 70, 1100, 'bf16'), (64, 1, 129, 63, 640, 'fp16'), (64, 1, 100, 257, 513, 'fp32'), (64, 7, 100, 70, 6300, 'bf16'), (64, 3, 70, 100, 2100, 'fp32'),
    (128, 1, 2000, 1540, 640, 'bf16'), (128, 1, 2000, 1540, 1000, 'fp16'), (128, 1, 2049, 1537, 1100, 'bf16'), (128, 6, 1000, 520, 8300, 'fp16'),
    (128, 1, 2000, 2570, 640, 'fp32'), (128, 1, 2000, 2570, 1100, 'fp32'), (128, 9, 1000, 777, 8300, 'fp32'),
    (256, 1, 3100, 4100, 640, 'bf16'), (256, 1, 3100, 4100, 1000, 'fp16'), (256, 1, 3329, 4097, 1100, 'bf16'), (256, 11, 700, 1540, 16500, 'bf16'),
    (256, 1, 5200, 1540, 640, 'fp32'), (256, 1, 5200, 1540, 1100, 'fp32'), (256, 6, 1300, 1540, 8300, 'fp32')])
def test_matmul8_tiles(tile, splits, M, N, K, dtype, fmts):
    from keypoints_amd import _lib, lowp
    code = lowp.DTYPES[TYPES[dtype]]
    assert _lib.lib().kp_q8_matmul_tile(M, N, K, code) == tile
    assert (_lib.lib().kp_q8_matmul_ws_floats(M, N, K, code) or M * N) == splits * M * N
    a, b = whole(M, K, 1), whole(N, K, 2)
    bias = torch.randint(-64, 65, (N,), device='cuda').float()
    pa, pb = lowp.pack8(a, fmts[0]), lowp.pack8(b, fmts[1])
    assert torch.equal(pa.unpack(), a) and torch.equal(pb.unpack(), b)
    for t in (None, bias):
        assert torch.equal(lowp.matmul8(pa, pb, t, dtype=TYPES[dtype]), exact(a, b, t, TYPES[dtype]))


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K', [(1, 300, 4096), (1, 33, 5000), (3, 8200, 1029), (16, 70, 4096), (13, 8193, 700), (40, 300, 1000)])
def test_few_rows(M, N, K, dtype):
    from keypoints_amd import _lib, lowp
    assert _lib.lib().kp_q8_linear_suits(M, N, K, lowp.DTYPES[TYPES[dtype]])
    x, w, bias = whole(M, K, 3, TYPES[dtype]), whole(N, K, 4), torch.randint(-64, 65, (N,), device='cuda').float()
    for fmt, wfmt in FMTS:
        for t in (None, bias):
            assert torch.equal(lowp.linear8(x, lowp.pack8(w, wfmt), t, fmt=fmt), exact(x, w, t, TYPES[dtype]))


@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K', [(12301, 1, 1000), (12300, 16, 129), (12355, 17, 1100), (13000, 32, 520), (12999, 33, 640), (12500, 64, 127), (12289, 100, 1300),
                                   (12400, 128, 1024)])
def test_few_columns(M, N, K, dtype):
    from keypoints_amd import _lib, lowp
    assert _lib.lib().kp_q8_linear_suits(M, N, K, lowp.DTYPES[TYPES[dtype]])
    x, w, bias = whole(M, K, 5, TYPES[dtype]), whole(N, K, 6), torch.randint(-64, 65, (N,), device='cuda').float()
    for fmt, wfmt in FMTS:
        assert torch.equal(lowp.linear8(x, lowp.pack8(w, wfmt), bias, fmt=fmt), exact(x, w, bias, TYPES[dtype]))


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('M,N,K', [(1100, 5200, 1540), (8300, 777, 1030)])
def test_training_step(M, N, K, dtype):
    """The three products of a step and the bias's gradient.  The forms along the batch mix the powers of two inside a block: whole numbers of 3
    bits times 1, 2 or 4, exact in both formats under one scale."""
    from keypoints_amd import lowp
    x, w, dy = whole(M, K, 7, TYPES[dtype]), whole(N, K, 8, torch.float32), whole(M, N, 9, TYPES[dtype])
    bias = torch.randint(-64, 65, (N,), device='cuda').float()
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    for fmt, gfmt in FMTS:
        y = lowp.linear8(*leaves, fmt=fmt, grad_fmt=gfmt)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        xd, wd = x.detach(), w.detach()
        assert torch.equal(y.detach(), exact(xd, wd, bias.detach(), TYPES[dtype]))
        assert torch.equal(dx, exact(dy, wd.t(), None, TYPES[dtype]))
        assert torch.equal(dw, exact(dy.t(), xd.t(), None, torch.float32))
        assert torch.equal(db, dy.double().sum(0).float())

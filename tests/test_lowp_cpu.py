"""CPU: the 8-bit format's oracle against torch's own 8-bit types, and what keypoints_amd.lowp / norm and their C entries refuse (nothing is
launched)."""
import ctypes

import pytest
import torch

from blocks8 import quantise

from keypoints_amd import lowp, norm
import keypoints_amd as ka


@pytest.mark.parametrize('fmt,kind', [('e4m3', torch.float8_e4m3fn), ('e5m2', torch.float8_e5m2)])
def test_oracle_rounds_as_the_types_do(fmt, kind):
    x = torch.cat([torch.randn(40, 300) * 10, torch.randn(40, 300) * torch.exp(4 * torch.randn(40, 300)), torch.linspace(-2, 2, 12000).view(40, 300)])
    values, s = quantise(x, fmt)
    two = torch.ldexp(torch.ones(1, dtype=torch.float64), s).repeat_interleave(128, 1)[:, :300]
    assert torch.equal((x.double() / two).float().to(kind).double() * two, values)
    peak = torch.stack([b.abs().amax(1) for b in x.double().split(128, 1)], 1) / torch.ldexp(torch.ones(1, dtype=torch.float64), s)
    top = 448.0 if fmt == 'e4m3' else 57344.0
    assert bool(((peak <= top) & (peak > top / 2)).all())      # the smallest exponent that fits


def refuses(kind, text, fn, *args, **kw):
    with pytest.raises(kind, match=text):
        fn(*args, **kw)


def test_lowp_refuses_what_it_cannot_take():
    x = torch.zeros(4, 8)
    for fn in (lowp.checkpoint8, lowp.pack8, lambda t: lowp.linear8(t, torch.zeros(3, 8))):
        refuses(RuntimeError, 'HIP device', fn, x)
    refuses(ValueError, 'format', lowp.checkpoint8, x, 'fp8')
    refuses(ValueError, 'format', lowp.pack8, x, 'e3m4')
    refuses(TypeError, 'HIP kernel', lowp.pack8, x.long())
    refuses(TypeError, 'HIP kernel', lowp.checkpoint8, x.double())
    refuses(TypeError, 'pack8 operand', lowp.matmul8, x, x)


def packed(shape, flat=False, fmt='e4m3', dtype=torch.bfloat16):
    """A Packed8 of zero bytes on the CPU: enough for what is checked before a launch."""
    rows, width = (1, 1) if flat else (torch.Size(shape[:-1]).numel(), shape[-1])
    return lowp.Packed8(torch.zeros(rows, (width + 127) // 128 * 128, dtype=torch.uint8), torch.zeros(rows, 4, dtype=torch.uint8), torch.Size(shape),
                        (1,), dtype, fmt, flat)


def test_matmul8_refusals():
    a, b = packed((4, 200)), packed((6, 200))
    refuses(TypeError, 'pack8 operand', lowp.matmul8, a, packed((800,), flat=True))
    refuses(ValueError, 'cannot multiply', lowp.matmul8, a, packed((6, 199)))
    refuses(ValueError, 'cannot multiply', lowp.matmul8, a, packed((2, 3, 200)))
    refuses(TypeError, 'HIP kernel', lowp.matmul8, a, b, None, torch.float64)
    refuses(ValueError, 'bias', lowp.matmul8, a, b, torch.zeros(5))
    refuses(ValueError, 'bias', lowp.matmul8, a, b, torch.zeros(6, dtype=torch.long))


def test_norm_and_switch_refusals():
    x = torch.zeros(4, 8)
    refuses(RuntimeError, 'HIP device', norm.layer_norm, x)
    refuses(ValueError, 'saved activations', ka.set_saved_activations, 'fp8')
    assert ka.runtime.saved_activations() is None


def test_c_entries_refuse_bad_arguments():
    """Host-side checks of the C entries (pointers are never followed): the code and a text that names the entry."""
    from keypoints_amd import _lib
    L = _lib.lib()
    p = ctypes.c_void_p(256)   # a non-null, aligned address that nothing reads
    E = -1

    def bad(name, *args):
        assert getattr(L, name)(*args) == E and name in L.kp_last_error().decode(), (name, args)

    bad('kp_q8_pack', None, 8, p, 128, p, 4, 1, 8, 1, 1, None)
    bad('kp_q8_pack', p, 8, p, 128, p, 4, 1, 8, 7, 1, None)          # unknown dtype
    bad('kp_q8_pack', p, 8, p, 128, p, 4, 1, 8, 1, 3, None)          # unknown format
    bad('kp_q8_pack', p, 8, p, 128, p, 4, 0, 8, 1, 1, None)          # no rows
    bad('kp_q8_pack', p, 4, p, 128, p, 4, 2, 8, 1, 1, None)          # rows overlap
    bad('kp_q8_pack', p, 8, p, 9, p, 4, 2, 8, 1, 1, None)            # neither padded nor back to back
    bad('kp_q8_pack', p, 1 << 40, p, 1 << 40, p, 1 << 34, 1, 1 << 40, 1, 1, None)   # 2^33 blocks
    bad('kp_q8_unpack', p, 128, p, 4, p, 4, 2, 8, 1, 1, None)
    bad('kp_q8_unpack', p, 128, p, 4, p, 8, 2, 8, 1, 0, None)
    bad('kp_q8_pack_both', p, 8, None, 0, None, 0, None, 0, None, 0, None, None, 4, 8, 1, 1, None)       # nothing asked for
    bad('kp_q8_pack_both', p, 8, p, 64, p, 4, None, 0, None, 0, None, None, 4, 8, 1, 1, None)            # row form not padded
    bad('kp_q8_pack_both', p, 8, None, 0, None, 0, p, 100, p, 4, None, None, 4, 8, 1, 1, None)           # column form not padded
    bad('kp_q8_pack_both', p, 8, None, 0, None, 0, ctypes.c_void_p(264), 128, p, 4, None, None, 4, 8, 1, 1, None)   # ... or not aligned
    bad('kp_q8_pack_both', p, 8, None, 0, None, 0, None, 0, None, 0, None, p, 4, 8, 1, 1, None)          # sums without a workspace
    bad('kp_q8_pack_both', p, 8, p, 128, p, 4, None, 0, None, 0, None, None, 1 << 24, 8, 1, 1, None)     # too many rows
    ok = dict(lda=128, sa=4, fa=1, ldb=128, sb=4, fb=1, ldc=8, M=4, N=8, K=100, dt=1)

    def mm(**kw):
        v = dict(ok, a=p, b=p, c=p, **kw)
        return (v['a'], v['lda'], p, v['sa'], v['fa'], v['b'], v['ldb'], p, v['sb'], v['fb'], None, v['c'], v['ldc'], None, v['M'], v['N'], v['K'],
                v['dt'], None)
    for kw in (dict(M=0), dict(N=0), dict(K=0), dict(lda=100), dict(ldb=96), dict(sa=1), dict(sb=6), dict(fa=0), dict(fb=3), dict(ldc=7), dict(dt=3),
               dict(N=1 << 30, ldc=1 << 30), dict(K=1 << 24, lda=1 << 24, ldb=1 << 24, sa=1 << 20, sb=1 << 20)):
        bad('kp_q8_matmul', *mm(**kw))
    v = list(mm())
    v[0] = ctypes.c_void_p(264)
    bad('kp_q8_matmul', *v)                                                                               # rows not on 16 bytes
    assert L.kp_q8_matmul_ws_floats(64, 64, 1 << 16, 1) > 0
    bad('kp_q8_matmul', *mm(M=64, N=64, K=1 << 16, lda=1 << 16, ldb=1 << 16, sa=512, sb=512, ldc=64))     # a workspace is needed
    bad('kp_q8_linear', p, 8, 1, p, 128, p, 1, 0, None, p, 8, 2, 8, 8, 1, None)
    bad('kp_q8_linear', p, 4, 1, p, 128, p, 1, 1, None, p, 8, 2, 8, 8, 1, None)
    bad('kp_q8_linear', p, 8, 1, p, 120, p, 1, 1, None, p, 8, 2, 8, 8, 1, None)
    bad('kp_q8_linear', p, 8, 1, p, 128, p, 1, 1, None, p, 200, 1 << 20, 200, 8, 1, None)
    bad('kp_layer_norm_fwd', p, 8, None, None, -1.0, p, 8, None, None, None, None, 0, 2, 8, 1, None)      # negative eps
    bad('kp_layer_norm_fwd', p, 8, None, None, 1e-5, p, 8, p, None, None, None, 0, 2, 8, 1, None)         # mean without rstd
    bad('kp_layer_norm_fwd', p, 8, None, None, 1e-5, p, 8, None, None, p, None, 1, 2, 8, 1, None)
    bad('kp_layer_norm_fwd', p, 4, None, None, 1e-5, p, 8, None, None, None, None, 0, 2, 8, 1, None)
    bad('kp_layer_norm_fwd', p, 8, None, None, 1e-5, p, 8, None, None, None, None, 0, 2, 0, 1, None)
    bad('kp_layer_norm_bwd', p, 8, p, 8, p, p, 1, None, p, p, p, 8, None, None, None, 2, 8, 1, None)      # x and its 8-bit form
    bad('kp_layer_norm_bwd', p, 8, None, 8, None, None, 0, None, p, p, p, 8, None, None, None, 2, 8, 1, None)
    bad('kp_layer_norm_bwd', p, 8, p, 8, None, None, 0, None, p, p, p, 8, None, p, None, 2, 8, 1, None)   # no workspace
    bad('kp_layer_norm_bwd', p, 8, p, 8, None, None, 0, None, p, p, None, 8, None, None, None, 2, 8, 1, None)   # nothing asked for


def test_products_plan_covers_every_block():
    """kp_q8_matmul_ws_floats is a whole number of partial matrices, at most 32 of them, and none for large outputs."""
    from keypoints_amd import _lib
    ws = _lib.lib().kp_q8_matmul_ws_floats
    for M, N, K in [(1, 1, 1), (64, 64, 65536), (1, 4096, 8191), (300, 300, 8192), (777, 1234, 1000), (100000, 64, 64), (4096, 2048, 16384)]:
        for dtype in (0, 1, 2):
            n = ws(M, N, K, dtype)
            assert n == 0 or (n % (M * N) == 0 and 2 <= n // (M * N) <= 32)
    assert ws(8192, 8192, 8192, 1) == 0 and ws(0, 4, 4, 1) == 0 and ws(4, 4, 1 << 40, 1) == 0


def test_packed_tensors_off_the_device():
    """A Packed8 that was brought to the CPU (a loaded file) is refused, not launched on."""
    a, b = packed((4, 200)), packed((6, 200))
    refuses(RuntimeError, 'HIP device', lowp.matmul8, a, b)
    refuses(RuntimeError, 'HIP device', a.unpack)
    refuses(RuntimeError, 'HIP device', packed((1,), flat=True).unpack)


def test_matmul8_refuses_a_bias_that_wants_a_gradient():
    a, b = packed((4, 200)), packed((6, 200))
    bias = torch.zeros(6, requires_grad=True)
    refuses(RuntimeError, 'carry no gradient', lowp.matmul8, a, b, bias)
    with torch.no_grad():
        refuses(RuntimeError, 'HIP device', lowp.matmul8, a, b, bias)

"""CPU: the calls that keypoints_amd.lowp and norm make of a user's calls, with the launches noted instead of made (tests/launch_stub.py)."""
import ctypes

import pytest
import torch

from launch_stub import stub

from keypoints_amd import _lib, lowp, norm


@pytest.fixture
def made(monkeypatch):
    return stub(monkeypatch)


def lazy(requires_grad=True):
    """(source, the map a network returns): the fp32 image of a padded bf16 tensor, made when somebody looks at it."""
    from keypoints_amd.models.functional import LazyNCHW
    source = torch.zeros(1, 6, 10, 3, dtype=torch.bfloat16, requires_grad=requires_grad)
    return source, LazyNCHW(source * 1, 1, _lib.KP_BF16)


@pytest.mark.parametrize('op', ['norm', 'kept', 'linear'])
def test_a_lazy_map_passes_its_gradient_on(made, op):
    """TransporterNet.forward returns its blend as a wrapper that carries no graph itself: the operators run on the tensor behind it."""
    source, x = lazy()
    w = torch.zeros(5, 8, requires_grad=True)
    y = lowp.linear8(x, w) if op == 'linear' else norm.layer_norm(x, keep='e4m3' if op == 'kept' else None)
    assert y.requires_grad
    y.sum().backward()
    assert source.grad is not None and source.grad.shape == source.shape


def test_lazy_weights_and_biases(made):
    source, m = lazy()
    x = torch.zeros(2, 8)
    for fn in (lambda t: norm.layer_norm(x, t), lambda t: norm.layer_norm(x, None, t), lambda t: lowp.linear8(x, torch.zeros(8, 8), t)):
        from keypoints_amd.models.functional import LazyNCHW

        class Row(LazyNCHW):
            """A lazy tensor of the shape these arguments have."""
            @staticmethod
            def __new__(cls):
                return torch.Tensor._make_wrapper_subclass(cls, (8,), dtype=torch.float32)

            def __init__(self):
                pass

            def materialize(self):
                return source.float()[0, 1, 1:9, 0]

        source.grad = None
        fn(Row()).sum().backward()
        assert source.grad is not None
    with pytest.raises(RuntimeError, match='carries no gradient'):
        lowp.linear8(m, lowp.pack8(torch.zeros(5, 8)))


def test_packing_a_lazy_map_reads_the_map(made):
    _, x = lazy()
    for fn in (lowp.checkpoint8, lowp.pack8):
        made.clear()
        fn(x)
        assert made[-1][0] == 'kp_q8_pack' and made[-1][1][0] == x.materialize().data_ptr() != 0


def test_forward_mode_is_refused_not_lost(made):
    """A dual tensor's tangent goes through none of the operators: a call that would return its result without one says so."""
    import torch.autograd.forward_ad as fwd
    x, w, v = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(8)
    packed = lowp.pack8(w)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        calls = [lambda: norm.layer_norm(dual(x)), lambda: norm.layer_norm(x, dual(v)), lambda: norm.layer_norm(x, None, dual(v)),
                 lambda: norm.layer_norm(dual(x), keep='e4m3'), lambda: lowp.linear8(dual(x), w), lambda: lowp.linear8(x, dual(w)),
                 lambda: lowp.linear8(x, w, dual(torch.zeros(5))), lambda: lowp.linear8(dual(x), packed),
                 lambda: lowp.linear8(x, packed, dual(torch.zeros(5))), lambda: lowp.matmul8(packed, packed, dual(torch.zeros(5)))]
        for grad in (True, False):
            for fn in calls:
                made.clear()
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    fn()
                assert not any(name != 'kp_q8_pack' for name, _ in made)
        for plain in (lambda: norm.layer_norm(x, v, v), lambda: lowp.linear8(x, packed), lambda: lowp.linear8(x, w), lambda: lowp.matmul8(packed, packed)):
            plain()   # (nothing carries a tangent)
    for transform in (lambda f: torch.func.jvp(f, (x,), (torch.ones_like(x),)), lambda f: torch.func.grad(lambda t: f(t).sum())(x)):
        for f in (norm.layer_norm, lambda t: lowp.linear8(t, w), lambda t: lowp.linear8(t, packed)):
            with pytest.raises(RuntimeError):
                transform(f)


def test_rows_longer_than_the_kernels_count(made):
    """Sizes that 32 bits do not hold arrive whole and are refused (2^32 + 8 columns are not 8); the largest row that is taken has 2^30."""
    L, p = _lib.lib(), ctypes.c_void_p(256)   # a non-null address that nothing reads

    def bad(name, *args):
        assert getattr(L, name)(*args) == -1 and name in L.kp_last_error().decode()
    for C in ((1 << 30) + 1, (1 << 31) - 8, (1 << 31) + 8, (1 << 32) + 8):
        bad('kp_layer_norm_fwd', p, C, None, None, 1e-5, p, C, None, None, None, None, 0, 2, C, 1, None)
        bad('kp_layer_norm_bwd', p, C, p, C, None, None, 0, None, p, p, p, C, p, p, p, 2, C, 1, None)
        assert L.kp_layer_norm_bwd_ws_floats(2, C) == 0
        long = torch.zeros(1).expand(1, C)   # (no memory behind it)
        made.clear()
        for call in (lambda: norm.layer_norm(long), lambda: norm.layer_norm(long, keep='e4m3')):
            with pytest.raises(ValueError, match='last dimension'):
                call()
        assert not made
    assert L.kp_layer_norm_bwd_ws_floats(2, 1 << 30) == 2 * 2 * (1 << 30)


def names(made):
    return [name for name, _ in made]


def test_a_layer_evaluated_without_gradients_packs_rows_only(made):
    """torch.no_grad() around a layer whose weight is a Parameter: no column form, nothing kept, and any number of rows."""
    x, b = torch.zeros(300, 64), torch.nn.Parameter(torch.zeros(40))
    w = torch.nn.Parameter(torch.zeros(40, 64))
    with torch.no_grad():
        for leaf in (x, x.clone().requires_grad_()):
            made.clear()
            y = lowp.linear8(leaf, w, b)
            assert names(made) == ['kp_q8_pack', 'kp_q8_pack', 'kp_q8_matmul'] and not y.requires_grad
    made.clear()
    assert not lowp.linear8(x, w.detach(), b.detach()).requires_grad and names(made) == ['kp_q8_pack', 'kp_q8_pack', 'kp_q8_matmul']
    made.clear()
    y = lowp.linear8(x, w, b)
    assert names(made) == ['kp_q8_pack_both', 'kp_q8_pack', 'kp_q8_matmul']
    y.sum().backward()
    assert w.grad is not None and b.grad is not None
    with torch.inference_mode():
        made.clear()
        assert lowp.linear8(x[:0], w, b).shape == (0, 40) and not made


@pytest.mark.parametrize('rows,width,inner,wants', [(3, 8388481, 4, 'x'), (5, 3, 8388481, ''), (5, 3, 8388481, 'w'), (40, 1 << 29, 1, '')])
def test_products_longer_than_one_call_takes(made, rows, width, inner, wants):
    """A sum over more than 8388480 elements is refused by the call itself, not between its launches or in the backward."""
    x = torch.zeros(1, dtype=torch.bfloat16).expand(rows, inner).requires_grad_('x' in wants)   # (no memory behind it)
    w = torch.zeros(1).expand(width, inner).requires_grad_('w' in wants)
    b = torch.zeros(width).requires_grad_('b' in wants) if width < 10 else None
    with pytest.raises(ValueError, match='8388480|2\\^29'):
        lowp.linear8(x, w, b)
    assert not made


@pytest.mark.parametrize('shape', [(300,), (2, 3, 50), (512,), (513,)])
@pytest.mark.parametrize('wants', ['x', 'w', 'b', 'xb', 'xwb'])
def test_more_rows_than_one_sum_takes(made, monkeypatch, shape, wants):
    """A training step of more rows than a product sums over packs the batch along itself in parts that begin on whole blocks; the parts' gradients
    are added.  Every byte of the forms is written by exactly one part."""
    monkeypatch.setattr(lowp, 'MOST', 256)
    rows = torch.Size(shape).numel()
    sizes = [256] * (rows // 256) + ([rows % 256] if rows % 256 else [])
    x, w, b = torch.zeros(*shape, 140), torch.zeros(5, 140), torch.zeros(5)
    leaves = [t.requires_grad_(k in wants) for t, k in ((x, 'x'), (w, 'w'), (b, 'b'))]
    y = lowp.linear8(*leaves)
    if 'w' in wants:
        calls = [a for name, a in made if name == 'kp_q8_pack_both' and a[12] != 5]
        assert [a[12] for a in calls] == sizes and all(a[13] == 140 for a in calls)
        at = 0
        for a in calls:   # x, ldx, q, ldq, s, lds, qt, ldqt, ...
            assert a[0] == x.data_ptr() + at * 140 * 4 and a[2] == calls[0][2] + at * 256 and a[4] == calls[0][4] + at * 4 and a[7] % 128 == 0 and a[7] >= a[12]
            at += a[12]
        spans = sorted((a[6], a[6] + 140 * a[7]) for a in calls)
        assert all(e <= b for (_, e), (b, _) in zip(spans, spans[1:]))
    else:
        assert [(name, a[6]) for name, a in made if name == 'kp_q8_pack'][0] == ('kp_q8_pack', rows)
    made.clear()
    g = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], torch.zeros_like(y))
    both = [a for name, a in made if name == 'kp_q8_pack_both']
    if 'w' in wants or 'b' in wants:
        assert [a[12] for a in both] == sizes
    assert [a[14:17] for name, a in made if name == 'kp_q8_matmul'] == ([(rows, 140, 5)] if 'x' in wants else []) + ([(5, 140, n) for n in sizes] if 'w' in wants else [])
    assert [t.shape for t in g] == [t.shape for t in leaves if t.requires_grad]


def test_lengths_that_are_refused(made, monkeypatch):
    monkeypatch.setattr(lowp, 'MOST', 256)
    leaf = lambda t: t.clone().requires_grad_()
    for args in ((leaf(torch.zeros(3, 8)), torch.zeros(300, 8), None), (torch.zeros(3, 300), torch.zeros(5, 300), None)):
        made.clear()
        with pytest.raises(ValueError, match='256'):
            lowp.linear8(*args)
        assert not made
    for rows, refused in ((4, False), (20, True)):   # serving: a few rows are summed by a kernel without that limit
        x, packed = torch.zeros(rows, 600, dtype=torch.bfloat16), lowp.pack8(torch.zeros(300, 600))
        monkeypatch.setattr(lowp, '_suits', lambda M, N, K, code: M <= 4)
        made.clear()
        if not refused:
            lowp.linear8(x, packed)
        else:
            with pytest.raises(ValueError, match='256'):
                lowp.linear8(x, packed)
            assert not made
    with pytest.raises(ValueError, match='256'):
        lowp.matmul8(packed, packed)


HOOKS = {   # what a saved tensor may come back as: (still the same numbers, or refused)
    'columns of a wider one': (True, lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]]),
    'every second row': (True, lambda t: torch.stack([t, t], 1).flatten(0, 1)[::2]),
    'transposed': (True, lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()),
    'another type': (False, lambda t: t.to(torch.float64)),
    'fewer elements': (False, lambda t: t[..., :-1].contiguous()),
    'off the device': (False, lambda t: t.to('meta')),
}


@pytest.mark.parametrize('how', HOOKS)
@pytest.mark.parametrize('op', ['norm', 'kept', 'linear'])
def test_saved_tensors_as_hooks_give_them_back(made, monkeypatch, op, how):
    """Saved-tensor hooks may hand a backward any tensor: it reads what has the right numbers where they lie, and refuses the rest."""
    same, change = HOOKS[how]
    x, w = torch.randn(6, 140, requires_grad=True), torch.randn(140, requires_grad=True)
    weight = torch.randn(5, 140, requires_grad=True)
    given = []
    keep = lambda t: t.detach().clone().random_(1, 100) if t.dtype == torch.uint8 or t.shape == (2, 6) else t.detach().clone()   # (not written: no launch)
    with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: given.append((t, change(t))) or given[-1][1]):
        y = lowp.linear8(x, weight) if op == 'linear' else norm.layer_norm(x, w, keep='e4m3' if op == 'kept' else None)
    made.clear()
    if not same:
        with pytest.raises(RuntimeError, match='saved'):
            y.sum().backward()
        assert not made
        return
    by = lambda shape, dtype: next(t for t, _ in given if tuple(t.shape) == shape and t.dtype == dtype)

    def numbers(address, shape, dtype, stride=None):
        rows, width = shape if len(shape) == 2 else (1, shape[0])
        flat = torch.frombuffer(bytearray((ctypes.c_char * (((rows - 1) * (stride or width) + width) * dtype.itemsize)).from_address(address)), dtype=dtype)
        return flat.as_strided((rows, width), (stride or width, 1)).reshape(shape)

    def look(name, *a):   # (while the call's own copies live)
        made.append((name, a))
        if name == 'kp_layer_norm_bwd':
            _, _, xp, ldx, q, s, _, wp, mean, rstd = a[:10]
            if op == 'kept':
                assert torch.equal(numbers(q, (6, 140), torch.uint8), by((6, 140), torch.uint8)) and torch.equal(numbers(s, (6, 2), torch.uint8), by((6, 2), torch.uint8))
            else:
                assert torch.equal(numbers(xp, (6, 140), torch.float32, ldx), x)
            st = by((2, 6), torch.float32)
            assert torch.equal(numbers(wp, (140,), torch.float32), w)
            assert torch.equal(numbers(mean, (6,), torch.float32), st[0]) and torch.equal(numbers(rstd, (6,), torch.float32), st[1])
        if name == 'kp_q8_matmul':   # dx = P(dy) P'(w), dw = P'(dy)^T P'(x): the second operand is what was kept
            blob = given[0][0]
            first = len([m for m in made if m[0] == 'kp_q8_matmul']) == 1   # (x's column form lies first: 140 rows of 128 bytes and their exponents)
            at = 140 * 128 + 768 if first else 0
            assert torch.equal(numbers(a[5], (140 * 128,), torch.uint8), blob[at:at + 140 * 128]) and a[5] % 16 == 0

    for module in (lowp, norm):
        monkeypatch.setattr(module, 'call', look)
    y.sum().backward()
    assert names(made) == (['kp_q8_pack_both', 'kp_q8_matmul', 'kp_q8_matmul'] if op == 'linear' else ['kp_layer_norm_bwd'])

"""Tensors in 8 bits with a power-of-two scale for each block of 128 elements (include/kp_hip.h): activation checkpoints and matrix products.

    kept = checkpoint8(x)                  # 1 byte an element (+ 1 / 128) instead of 2 or 4, between a forward and its backward
    x = kept.unpack()

    packed = pack8(weight)                 # once, for serving
    y = linear8(x, packed, bias)
    y = linear8(x, weight, bias)           # training: three 8-bit products a step; what it keeps of x IS the weight gradient's operand

    c = matmul8(pack8(a), pack8(b))        # a @ b.T

A block's scale is 2^s with the smallest s that brings the block's largest finite magnitude to at most 448 ('e4m3') or 57344 ('e5m2'); an
element is rounded once, by at most 2^-4 ('e4m3') or 2^-3 ('e5m2') of itself (elements more than 2^14 / 2^29 below their block's largest lose
more, down to zero).  Not-a-numbers stay what they are, so an overflowing fp16 step still reaches the loss scaler; infinities stay in
'e5m2' and become not-a-numbers in 'e4m3'.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, ptr
from .runtime import device_of, require_device, stream_ptr

BLOCK = 128
FORMATS = {'e4m3': _lib.KP_E4M3, 'e5m2': _lib.KP_E5M2}
MOST = 65535 * BLOCK   # elements a product's sum runs over (kp_q8_matmul, and the rows that kp_q8_pack_both turns): 8388480
DTYPES = {torch.float32: _lib.KP_F32, torch.bfloat16: _lib.KP_BF16, torch.float16: _lib.KP_F16}


def format_code(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f'format must be one of {sorted(FORMATS)}, not {fmt!r}')
    return FORMATS[fmt]


def dtype_code(dtype: torch.dtype) -> int:
    if dtype not in DTYPES:
        raise TypeError(f'{dtype} has no HIP kernel: float32, bfloat16 or float16')
    return DTYPES[dtype]


def real(t):
    """t itself, or the tensor behind a map that a network returned unmade (models.functional.LazyNCHW): the wrapper carries no graph, so an
    autograd Function that was handed it would pass no gradient on.  (Plain tensors leave by their type, without the import.)"""
    if type(t) in PLAIN:
        return t
    from .models.functional import unlazy
    return unlazy(t)


def no_tangents(op, *tensors):
    """(Inside a level of forward-mode differentiation: forward_ad._current_level >= 0.)  Refuses inputs of forward-mode differentiation: the operators have no formula for it, and a result without a tangent would read as a
    derivative of zero."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f'{op}: no forward-mode derivative; take the reverse one, or hand over the primal tensors')


def as_rows(x: torch.Tensor):
    """x [..., width] as (tensor, rows, row stride): x itself where its rows lie one stride apart (a column slice of a matrix does), else a
    contiguous copy."""
    width = x.shape[-1]
    if not x.is_contiguous():
        if x.dim() == 2 and (width <= 1 or x.stride(1) == 1) and x.stride(0) >= width:
            return x, x.shape[0], x.stride(0)
        x = x.contiguous()
    return x, x.numel() // width, width


def as_vector(t):
    """A weight or bias vector as the kernels read it: fp32, dense (differentiable; itself where it already is; None stays None)."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def saved(t: torch.Tensor, shape, dtype, device):
    """A saved tensor as the backward got it.  Saved-tensor hooks (offloading, compression) may give back another one: with other strides,
    which is fine, or of another size, type or place, of which the kernels would read past the end."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise RuntimeError(f'a saved tensor of shape {tuple(shape)}, {dtype}, on {device} came back from its hook as {tuple(t.shape)}, {t.dtype}, on {t.device}')
    return t


class Packed8:
    """A tensor in the 8-bit block format: `values` (bytes), `scales` (exponent bytes), the `shape` and `dtype` it stands for.

    Operand form (pack8): values [rows][width rounded up to 128], scales [rows][blocks rounded up to 4], blocks along the last dimension.
    Checkpoint form (checkpoint8, `flat`): the tensor's elements in memory order as one row, nothing padded; `stride` brings the order back."""

    __slots__ = ('values', 'scales', 'shape', 'stride', 'dtype', 'fmt', 'flat')

    def __init__(self, values, scales, shape, stride, dtype, fmt, flat):
        self.values, self.scales, self.shape, self.stride = values, scales, shape, stride
        self.dtype, self.fmt, self.flat = dtype, fmt, flat

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.scales.numel()

    def unpack(self, dtype: torch.dtype = None) -> torch.Tensor:
        """The tensor again (in `dtype`, its own by default), each element rounded once to that type (to its largest number where the format
        rounded a finite element past the type's range)."""
        dtype = self.dtype if dtype is None else dtype
        code = dtype_code(dtype)
        v, s = self.values, self.scales
        require_device(v, s)
        if self.flat:
            y = torch.empty_strided(self.shape, self.stride, dtype=dtype, device=v.device)
            rows, width, ldq, lds = 1, y.numel(), v.numel(), s.numel()
        else:
            y = torch.empty(self.shape, dtype=dtype, device=v.device)
            rows, width, ldq, lds = v.shape[0], self.shape[-1], v.shape[1], s.shape[1]
        if y.numel():
            with device_of(v):
                call('kp_q8_unpack', ptr(v), ldq, ptr(s), lds, ptr(y), width, rows, width, code, FORMATS[self.fmt], stream_ptr())
        return y


PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None), Packed8))


def _dense(x: torch.Tensor) -> bool:
    """True if x's elements fill one run of memory in some order of its dimensions (channels_last, a transpose, ...)."""
    if x.is_contiguous():
        return True
    run = 1
    for stride, size in sorted((st, n) for st, n in zip(x.stride(), x.shape) if n > 1):
        if stride != run:
            return False
        run *= size
    return True


def checkpoint8(x: torch.Tensor, fmt: str = 'e4m3') -> Packed8:
    """x in 8 bits, to be kept between a forward and its backward: `.unpack()` gives it back with its shape, strides (a tensor with gaps or
    repeated elements: dense ones) and type.  The blocks run over the elements in memory order, across rows, whatever the shape; no gradient flows through it."""
    x = real(x)
    code, dcode = format_code(fmt), dtype_code(x.dtype)
    require_device(x)
    if not _dense(x):
        x = x.contiguous()
    n = x.numel()
    values, scales = x.new_empty(n, dtype=torch.uint8), x.new_empty((n + BLOCK - 1) // BLOCK, dtype=torch.uint8)
    if n:
        with device_of(x):
            call('kp_q8_pack', ptr(x), n, ptr(values), n, ptr(scales), scales.numel(), 1, n, dcode, code, stream_ptr())
    return Packed8(values, scales, x.shape, x.stride(), x.dtype, fmt, True)


def _sizes(rows, width):
    """Row strides of an operand form: values padded to whole blocks, exponent bytes to whole words."""
    blocks = (width + BLOCK - 1) // BLOCK
    return blocks * BLOCK, (blocks + 3) // 4 * 4


def pack8(x: torch.Tensor, fmt: str = 'e4m3') -> Packed8:
    """x [..., width] as a product's operand, blocks along the last dimension.  No gradient flows through it (linear8 has its own)."""
    x = real(x)
    code, dcode = format_code(fmt), dtype_code(x.dtype)
    require_device(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'pack8: the last dimension must hold at least one element, got shape {tuple(x.shape)}')
    m, rows, ld = as_rows(x.detach())
    width = x.shape[-1]
    ldv, lds = _sizes(rows, width)
    values, scales = x.new_empty((rows, ldv), dtype=torch.uint8), x.new_empty((rows, lds), dtype=torch.uint8)
    if rows:
        with device_of(x):
            call('kp_q8_pack', ptr(m), ld, ptr(values), ldv, ptr(scales), lds, rows, width, dcode, code, stream_ptr())
    return Packed8(values, scales, x.shape, None, x.dtype, fmt, False)


class _Forms:
    """Operand forms (and a workspace) of one call in ONE allocation: a linear layer's step has ten of them, and an allocation costs a
    microsecond of host time, three in a backward.  A form is (address, stride of values, address, stride of exponents, rows, width)."""
    __slots__ = ('bytes', 'parts', 'memory')

    def __init__(self):
        self.bytes, self.parts, self.memory = 0, [], None

    def _take(self, n):
        at = self.bytes
        self.bytes = at + (n + 255) // 256 * 256
        return at

    def form(self, rows, width, wanted=True):
        if not wanted:
            return None
        ldv, lds = _sizes(rows, width)
        f = [self._take(rows * ldv), ldv, self._take(rows * lds), lds, rows, width]
        self.parts.append(f)
        return f

    def floats(self, n, wanted=True):
        if not wanted:
            return None
        f = [self._take(4 * n)]
        self.parts.append(f)
        return f

    def allocate(self, like):
        return self.rebase(like.new_empty(self.bytes, dtype=torch.uint8))

    def rebase(self, memory):
        self.memory = memory   # (held here: what a saved-tensor hook gives back has no other owner)
        base = memory.data_ptr()
        for f in self.parts:
            f[0] += base
            if len(f) > 1:
                f[2] += base
        return memory


_NO_FORM = (None, 0, None, 0)


def _pack_both(m, rows, ld, width, dcode, code, q, qt, ws=None, colsum=None):
    """A matrix into a row form, a column form and column sums (each may be None): kp_q8_pack_both, or kp_q8_pack for rows alone."""
    if qt is None and colsum is None:
        if q is not None:
            call('kp_q8_pack', ptr(m), ld, q[0], q[1], q[2], q[3], rows, width, dcode, code, stream_ptr())
        return
    v, ldv, s, lds = q[:4] if q is not None else _NO_FORM
    vt, ldvt, st, ldst = qt[:4] if qt is not None else _NO_FORM
    call('kp_q8_pack_both', ptr(m), ld, v, ldv, s, lds, vt, ldvt, st, ldst, ws[0] if ws is not None else None, ptr(colsum), rows, width, dcode,
         code, stream_ptr())


def _product(a, fmta, b, fmtb, bias, like, shape, dtype):
    """kp_q8_matmul of two operand forms into a new tensor of `shape` = [..., rows of b] on `like`'s device."""
    M, N, K, code = a[4], b[4], a[5], DTYPES[dtype]
    c = like.new_empty(shape, dtype=dtype)
    floats = _lib.lib().kp_q8_matmul_ws_floats(M, N, K, code)
    ws = like.new_empty(floats, dtype=torch.float32) if floats else None
    call('kp_q8_matmul', a[0], a[1], a[2], a[3], fmta, b[0], b[1], b[2], b[3], fmtb, ptr(bias), ptr(c), N, ptr(ws), M, N, K, code, stream_ptr())
    return c


def _form_of(p: Packed8):
    v, s = p.values, p.scales
    return ptr(v), v.shape[1], ptr(s), s.shape[1], v.shape[0], p.shape[-1]


def _check_bias(bias, width, device):
    if bias is not None and (bias.shape != (width,) or bias.device != device or bias.dtype not in DTYPES):
        raise ValueError(f'the bias must be a vector of {width} floats on {device}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}')


def _check_sizes(op, rows, columns, *sums):
    """What kp_q8_matmul and kp_q8_pack_both take in one call; `sums`: (name, length) of every sum that a product of this call runs over."""
    for name, n in sums:
        if n > MOST:
            raise ValueError(f'{op}: the sum over {n} {name} is longer than one product takes ({MOST}): split it')
    if rows > 0x7fffff00 or columns > 0x1fffff00:
        raise ValueError(f'{op}: {rows} x {columns} results are more than one product takes (2^31 - 256 rows, 2^29 - 256 columns)')


def matmul8(a: Packed8, b: Packed8, bias: torch.Tensor = None, dtype: torch.dtype = None) -> torch.Tensor:
    """a @ b.T (+ bias) of two operand forms: a [..., k], b [n, k] -> [..., n] in `dtype` (a's by default).  The formats may differ.

    float32 results are fp32 sums of exact products.  16-bit results come from the 8-bit matrix instruction, which cuts what lies 13 bits below
    the largest of 8 neighbouring products before it adds them up in fp32: off by less than 7 * 2^-13 of the sum of those largest products,
    then rounded once -- at twice the rate."""
    bias = real(bias)
    if forward_ad._current_level >= 0:
        no_tangents('matmul8', bias)
    for name, p in (('a', a), ('b', b)):
        if not isinstance(p, Packed8) or p.flat:
            raise TypeError(f'matmul8: {name} must be a pack8 operand')
    if len(b.shape) != 2 or a.shape[-1] != b.shape[-1]:
        raise ValueError(f'matmul8: cannot multiply {tuple(a.shape)} with the transpose of {tuple(b.shape)}')
    if a.values.device != b.values.device:
        raise ValueError(f'matmul8: operands on {a.values.device} and {b.values.device}')
    dtype = a.dtype if dtype is None else dtype
    dtype_code(dtype)
    _check_bias(bias, b.shape[0], a.values.device)
    _check_sizes('matmul8', a.values.shape[0], b.shape[0], ('inner elements', b.shape[1]))
    if torch.is_grad_enabled() and bias is not None and bias.requires_grad:
        raise RuntimeError('matmul8: packed operands carry no gradient, and none would reach the bias; run under torch.no_grad()')
    require_device(a.values, a.scales, b.values, b.scales)
    shape = (*a.shape[:-1], b.shape[0])
    if a.values.shape[0] == 0 or b.shape[0] == 0:
        return torch.empty(shape, device=a.values.device, dtype=dtype)
    bias = as_vector(bias)
    with device_of(a.values):
        return _product(_form_of(a), FORMATS[a.fmt], _form_of(b), FORMATS[b.fmt], bias, a.values, shape, dtype)


def _parts(rows):
    """(first row, rows) of the parts in which a batch of more than MOST rows is packed along itself.  They begin on whole blocks, so the blocks are
    the whole batch's; the weight's and bias's gradients add up over the parts."""
    return [(at, min(MOST, rows - at)) for at in range(0, rows, MOST)]


def _pack_parts(m, rows, ld, width, dcode, code, q, qts, wss=None, colsums=None):
    """_pack_both for such a batch: a column form, workspace and column sums for each part (q, and whole lists, may be None)."""
    m = m if m.dim() == 2 else m.view(rows, width)
    for i, (at, n) in enumerate(_parts(rows)):
        part = None if q is None else (q[0] + at * q[1], q[1], q[2] + at * q[3], q[3])
        _pack_both(m[at:at + n], n, ld, width, dcode, code, part, qts and qts[i], wss and wss[i], colsums and colsums[i])


def _total(tensors):
    """Their sum, in their order (into the first)."""
    tensors = iter(tensors)
    total = next(tensors)
    for t in tensors:
        total += t
    return total


def _forward(x, weight, bias, code, need_x, need_w):
    """-> y = P(x) P(w)^T + b and what a backward reads: P'(x) where the weight's gradient is wanted, P'(w) where x's is (None: neither)."""
    m, rows, ld = as_rows(x)
    N, K = weight.shape
    shape = (*x.shape[:-1], N)
    if rows == 0 or N == 0:
        return torch.empty(shape, device=x.device, dtype=x.dtype), None
    with device_of(x):
        w2, _, wld = as_rows(weight)
        now, later = _Forms(), _Forms()
        qx, qw = now.form(rows, K), now.form(N, K)
        long = need_w and rows > MOST
        qxt = [later.form(K, n) for _, n in _parts(rows)] if long else later.form(K, rows, need_w)
        qwt = later.form(K, N, need_x)
        now.allocate(x)
        kept = later.allocate(x) if need_x or need_w else None
        (_pack_parts if long else _pack_both)(m, rows, ld, K, DTYPES[x.dtype], code, qx, qxt)
        _pack_both(w2, N, wld, K, DTYPES[weight.dtype], code, qw, qwt)
        return _product(qx, code, qw, code, bias, x, shape, x.dtype), kept


class _Linear8(torch.autograd.Function):
    """y = P(x) P(w)^T + b;  dx = P(dy) P'(w),  dw = P'(dy)^T P'(x),  db = column sums of dy.  P: blocks along the product's inner index, P':
    along the other one (w along its rows, x and dy along the batch), so that every product's operands have their blocks along its own
    inner index.  P'(x) -- a byte an element -- is what waits for the backward, and P'(w)."""

    @staticmethod
    def forward(ctx, x, weight, bias, fmt, grad_fmt):
        ctx.args = (x.shape, x.dtype, weight.shape, weight.dtype, FORMATS[fmt], FORMATS[grad_fmt])
        y, kept = _forward(x, weight, bias, FORMATS[fmt], *ctx.needs_input_grad[:2])
        if kept is not None:
            ctx.save_for_backward(kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xshape, xdtype, wshape, wdtype, code, grad_code = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        N, dev = wshape[0], dy.device
        if dy.numel() == 0:   # no rows, or no columns: nothing was launched
            return (torch.zeros(xshape, device=dev, dtype=xdtype) if need_x else None,
                    torch.zeros(wshape, device=dev, dtype=wdtype) if need_w else None,
                    torch.zeros(N, device=dev, dtype=torch.float32) if need_b else None, None, None)
        m, rows, ld = as_rows(dy)
        K = wshape[1]
        with device_of(dy):
            later, now = _Forms(), _Forms()
            parts = _parts(rows) if rows > MOST else None
            qxt = later.form(K, rows, need_w) if parts is None or not need_w else [later.form(K, n) for _, n in parts]
            qwt = later.form(K, N, need_x)
            if need_x or need_w:
                kept = saved(ctx.saved_tensors[0], (later.bytes,), torch.uint8, dev).contiguous()
                later.rebase(kept if kept.data_ptr() % 16 == 0 else kept.clone())   # (what the products take)
            qd, dw = now.form(rows, N, need_x), None
            ws_floats, dcode = _lib.lib().kp_q8_pack_both_ws_floats, DTYPES[dy.dtype]
            if parts is None:
                qdt = now.form(N, rows, need_w)
                ws = now.floats(ws_floats(rows, N), need_b)
                now.allocate(dy)
                db = dy.new_empty(N, dtype=torch.float32) if need_b else None
                _pack_both(m, rows, ld, N, dcode, grad_code, qd, qdt, ws, db)
            else:
                qdt = [now.form(N, n) for _, n in parts] if need_w else None
                wss = [now.floats(ws_floats(n, N)) for _, n in parts] if need_b else None
                now.allocate(dy)
                dbs = [dy.new_empty(N, dtype=torch.float32) for _ in parts] if need_b else None
                if need_w or need_b:
                    _pack_parts(m, rows, ld, N, dcode, grad_code, qd, qdt, wss, dbs)
                else:
                    _pack_both(m, rows, ld, N, dcode, grad_code, qd, None)
                db = _total(dbs) if need_b else None
            dx = _product(qd, grad_code, qwt, code, None, dy, xshape, xdtype) if need_x else None
            if need_w and parts is None:
                dw = _product(qdt, grad_code, qxt, code, None, dy, wshape, wdtype)
            elif need_w:   # (added in fp32, rounded once)
                dw = _total(_product(a, grad_code, b, code, None, dy, wshape, torch.float32) for a, b in zip(qdt, qxt)).to(wdtype)
        return dx, dw, db, None, None


def _suits(rows, N, K, code):
    """Whether x goes to the product as it is (kp_q8_linear)."""
    return _lib.lib().kp_q8_linear_suits(rows, N, K, code) != 0


def linear8(x: torch.Tensor, weight, bias: torch.Tensor = None, fmt: str = 'e4m3', grad_fmt: str = 'e4m3') -> torch.Tensor:
    """x [..., k] @ weight.T (+ bias) in 8-bit products: [..., n] in x's type.

    weight a tensor [n, k] (fp32 master weights, or 16 bits): every call packs x and the weight in `fmt`; differentiable in x, weight and
    bias.  The backward packs the output gradient in `grad_fmt` and takes dx and dw from two more 8-bit products; between the passes only
    8-bit forms wait (a byte an element of x and of the weight).  Gradients come in the types of what they belong to.  A product sums over at
    most 8388480 elements; the weight's gradient of more rows is the sum of such parts.
    weight a Packed8 (pack8): serving.  `fmt` is x's format; no gradient.

    Each product is matmul8's: y and dx as x's type has it, dw as the weight's has it.  A float32 x takes the exact sums."""
    if not (type(x) in PLAIN and type(weight) in PLAIN and type(bias) in PLAIN):
        x, weight, bias = real(x), real(weight), real(bias)
    if forward_ad._current_level >= 0:
        no_tangents('linear8', x, weight, bias)
    require_device(x, bias)
    code = format_code(fmt)
    format_code(grad_fmt)
    dtype_code(x.dtype)
    packed = isinstance(weight, Packed8)
    if packed and weight.flat:
        raise TypeError('linear8: the weight must be a pack8 operand, not a checkpoint')
    if not packed:
        require_device(weight)
        dtype_code(weight.dtype)
    if len(weight.shape) != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.shape[1] < 1:
        raise ValueError(f'linear8: cannot multiply {tuple(x.shape)} with the transpose of {tuple(weight.shape)}')
    dev = weight.values.device if packed else weight.device
    if dev != x.device:
        raise ValueError(f'linear8: x on {x.device}, the weight on {dev}')
    N = weight.shape[0]
    _check_bias(bias, N, x.device)
    grad = torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad) or (not packed and weight.requires_grad))
    if not packed:
        K = weight.shape[1]
        rows = x.numel() // K
        if rows > MOST or N > MOST or K > MOST:
            _check_sizes('linear8', rows, N, ('inner elements', K), ("outputs (x's gradient)", N if grad and x.requires_grad else 0))
        bias = as_vector(bias)
        return _Linear8.apply(x, weight, bias, fmt, grad_fmt) if grad else _forward(x, weight, bias, code, False, False)[0]
    if grad:
        raise RuntimeError('linear8: a packed weight carries no gradient; pass the weight itself, or run under torch.no_grad()')
    shape = (*x.shape[:-1], N)
    K = x.shape[-1]
    rows = x.numel() // K
    if rows == 0 or N == 0:
        return torch.empty(shape, device=x.device, dtype=x.dtype)
    suits = _suits(rows, N, K, DTYPES[x.dtype])
    if not suits and (rows > MOST or N > MOST or K > MOST):
        _check_sizes('linear8', rows, N, ('inner elements', K))
    bias = as_vector(bias)
    m, _, ld = as_rows(x)
    with device_of(x):
        if suits:
            y = x.new_empty(shape)
            v, s = weight.values, weight.scales
            call('kp_q8_linear', ptr(m), ld, code, ptr(v), v.shape[1], ptr(s), s.shape[1], FORMATS[weight.fmt], ptr(bias), ptr(y), N,
                 rows, N, K, DTYPES[x.dtype], stream_ptr())
            return y
        forms = _Forms()
        q = forms.form(rows, K)
        forms.allocate(x)
        _pack_both(m, rows, ld, K, DTYPES[x.dtype], code, q, None)
        return _product(q, code, _form_of(weight), FORMATS[weight.fmt], bias, x, shape, x.dtype)

"""Layer norm over the last dimension (kp_layer_norm_*, include/kp_hip.h): the batch-independent normalisation beside the Units' BatchNorm --
the same in training and inference, no running statistics, nothing to synchronise between ranks.

    y = layer_norm(x, weight, bias)                  # x [..., C], fp32 / bf16 / fp16; weight, bias [C]
    y = layer_norm(x, weight, bias, keep='e4m3')     # the backward reads x from an 8-bit copy the forward writes on its way
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, ptr
from .lowp import BLOCK, DTYPES, FORMATS, PLAIN, as_rows, as_vector, dtype_code, format_code, no_tangents, real, saved
from .runtime import device_of, require_device, stream_ptr


def _forward(x, weight, bias, eps, stats, fmt):
    """-> y, x as rows, its row stride, [means | deviations' reciprocals], 8-bit copy, its exponents (each None where not asked for)."""
    m, rows, ld = as_rows(x)
    C = x.shape[-1]
    y = torch.empty_like(m) if m is x and ld == C else x.new_empty(x.shape)
    st = q = s = None
    if stats:
        st = x.new_empty((2, rows), dtype=torch.float32)
    if fmt:
        q = x.new_empty((rows, C), dtype=torch.uint8)
        s = x.new_empty((rows, (C + BLOCK - 1) // BLOCK), dtype=torch.uint8)
    if rows:
        at = ptr(st)
        with device_of(x):
            call('kp_layer_norm_fwd', ptr(m), ld, ptr(weight), ptr(bias), eps, ptr(y), C, at, at + 4 * rows if stats else None, ptr(q), ptr(s),
                 FORMATS[fmt] if fmt else 0, rows, C, DTYPES[x.dtype], stream_ptr())
    return y, m, ld, st, q, s


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        y, m, ld, st, q, s = _forward(x, weight, bias, eps, True, keep)
        ctx.keep = keep
        ctx.save_for_backward(weight, st, q if keep else m, s)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        keep = ctx.keep
        weight, st, kept, s = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        g, rows, ldg = as_rows(dy)
        C, dev, f32 = dy.shape[-1], dy.device, torch.float32
        st = saved(st, (2, rows), f32, dev).contiguous()
        if weight is not None:
            weight = saved(weight, (C,), f32, dev).contiguous()
        if keep:
            kept = saved(kept, (rows, C), torch.uint8, dev).contiguous()
            s = saved(s, (rows, (C + BLOCK - 1) // BLOCK), torch.uint8, dev).contiguous()
            ldx = C
        else:
            kept, _, ldx = as_rows(saved(kept, dy.shape, dy.dtype, dev))
        make = st.new_empty if rows else st.new_zeros   # (no rows: nothing is launched)
        dx = dy.new_empty(dy.shape) if need_x else None
        dw = make(C) if need_w else None
        db = make(C) if need_b else None
        if rows:
            ws = st.new_empty(_lib.lib().kp_layer_norm_bwd_ws_floats(rows, C)) if need_w or need_b else None
            at = ptr(st)
            with device_of(dy):
                call('kp_layer_norm_bwd', ptr(g), ldg, None if keep else ptr(kept), ldx, ptr(kept) if keep else None, ptr(s),
                     FORMATS[keep] if keep else 0, ptr(weight), at, at + 4 * rows, ptr(dx), C, ptr(ws), ptr(dw), ptr(db), rows, C,
                     DTYPES[dy.dtype], stream_ptr())
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, eps: float = 1e-5, keep: str = None) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension, in x's type; statistics in fp32.  weight and bias are
    vectors of x.shape[-1] floats or None.  keep: None -- the backward reads x itself -- or the 8-bit format ('e4m3', 'e5m2'; keypoints_amd.lowp)
    in which a copy of x waits for it: half the memory of a 16-bit x, and the gradients of x and weight are taken with
    the copy's values (each off from x by at most 2^-4 / 2^-3 of itself) and x's own statistics."""
    if not (type(x) in PLAIN and type(weight) in PLAIN and type(bias) in PLAIN):
        x, weight, bias = real(x), real(weight), real(bias)
    if forward_ad._current_level >= 0:
        no_tangents('layer_norm', x, weight, bias)
    eps = float(eps)
    C = x.shape[-1] if x.dim() else 0
    if not (x.is_cuda and 0 < C <= MOST and x.dtype in DTYPES and 0.0 <= eps < _INF and (keep is None or keep in FORMATS)
            and _plain_vector(weight, C, x) and _plain_vector(bias, C, x)):
        weight, bias = _checked(x, weight, bias, eps, keep, C)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, keep)
    return _forward(x, weight, bias, eps, False, None)[0]


_INF = float('inf')
MOST = 1 << 30   # columns


def _plain_vector(t, C, x):
    """None, or a vector as the kernels read it, where x is."""
    return t is None or (t.dtype is torch.float32 and t.dim() == 1 and t.numel() == C and t.is_cuda and t.is_contiguous() and t.device == x.device)


def _checked(x, weight, bias, eps, keep, C):
    """weight and bias as the kernels read them, or the refusal that says what is wrong (off the path of calls that need neither)."""
    require_device(x, weight, bias)
    dtype_code(x.dtype)
    if keep is not None:
        format_code(keep)
    if not 1 <= C <= MOST:
        raise ValueError(f'layer_norm: the last dimension must hold at least one element and at most 2^30, got shape {tuple(x.shape)}')
    if not 0.0 <= eps < _INF:
        raise ValueError(f'layer_norm: eps must be a number that is not negative, got {eps}')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and (t.shape != x.shape[-1:] or t.dtype not in DTYPES or t.device != x.device):
            raise ValueError(f'layer_norm: {name} must be a vector of {C} floats on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}')
    return as_vector(weight), as_vector(bias)

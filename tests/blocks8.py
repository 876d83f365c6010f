"""The 8-bit block format from its definition, in 64 bits on the CPU (the oracle of the lowp / norm tests)."""
import torch

GRID = {'e4m3': (3, -6, 448.0), 'e5m2': (2, -14, 57344.0)}   # mantissa bits, exponent of the smallest normal number, largest value
STEP = {'e4m3': 2.0 ** -4, 'e5m2': 2.0 ** -3}                # half a step, relative


def scale_exponent(peak, fmt):
    """Smallest whole s >= -127 with peak * 2^-s <= the format's largest value (0 for a peak of zero); peak: fp64 tensor."""
    mantissa, exponent = torch.frexp(peak)                   # peak = mantissa * 2^exponent, mantissa in [0.5, 1)
    _, top = torch.frexp(torch.tensor(GRID[fmt][2], dtype=torch.float64))   # the largest value is 0.875 * 2^top
    s = exponent - top + (mantissa > 0.875).to(torch.int32)
    return torch.where(peak > 0, s.clamp_min(-127), torch.zeros_like(s))


def quantise(x, fmt, axis=-1):
    """(values, exponents) of x with blocks of 128 along `axis`; values fp64 in x's shape, exponents with the blocks along `axis`."""
    bits, lowest, _ = GRID[fmt]
    x = x.detach().cpu().double().movedim(axis, -1)
    out, exps = torch.empty_like(x), []
    for c in range(0, x.shape[-1], 128):
        part = x[..., c:c + 128]
        finite = torch.where(torch.isfinite(part), part.abs(), torch.zeros_like(part))
        s = scale_exponent(finite.amax(-1, keepdim=True), fmt)
        exps.append(s)
        two = torch.ldexp(torch.ones_like(s, dtype=torch.float64), s)
        u = torch.where(torch.isfinite(part), part / two, torch.zeros_like(part))
        _, e = torch.frexp(u)
        step = torch.ldexp(torch.ones_like(u), (e - 1).clamp_min(lowest) - bits)
        v = torch.round(u / step) * step * two               # (torch.round: halves to even)
        if fmt == 'e5m2':
            v = torch.where(torch.isinf(part), part, v)
        else:
            v = torch.where(torch.isinf(part), torch.full_like(v, float('nan')), v)
        out[..., c:c + 128] = torch.where(torch.isnan(part), part, v)
    return out.movedim(-1, axis), torch.cat(exps, -1).movedim(-1, axis)


def same(a, b):
    """Equal numbers, with not-a-numbers in the same places."""
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def to_type(v, dtype):
    """fp64 values in a storage type, finite ones past its range as its largest number."""
    top = torch.finfo(dtype).max
    return torch.where(v.isfinite(), v.clamp(-top, top), v).to(dtype)

"""8-bit values with scales, plainly and in 64 bits: the rule of the scales, the rounding to e4m3, products and gates."""
import math

import torch

GROUP = 128


def groups(k):
    return -(-k // GROUP)


def two_to(exponent):
    """2^e to the bit."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def scale_of(largest):
    """The smallest power of two that brings `largest` (float64) to 448 or less, 2^-126 at least; 1 for zero, NaN for what is
    not finite."""
    mantissa, exponent = torch.frexp(largest)          # in [1/2, 1): 448 = 0.875 * 2^9
    e = (exponent - 9 + (mantissa > 0.875).int()).clamp(-126, 200)
    s = torch.where(largest == 0, torch.ones_like(largest), two_to(e))
    return torch.where(torch.isfinite(largest), s, torch.full_like(s, math.nan))


def round_e4m3(y):
    """Float64 to the nearest e4m3 value, the even one of two, for magnitudes of at most 448."""
    step = two_to((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def quantize_rows(x):
    """(values, scales) in float64 of rows of any type."""
    x = x.double()
    m, k = x.shape
    p = torch.nn.functional.pad(x, (0, groups(k) * GROUP - k)).view(m, -1, GROUP)
    s = scale_of(torch.where(torch.isfinite(p), p.abs(), torch.full_like(p, math.inf)).amax(2))
    q = torch.where(torch.isnan(s)[:, :, None], torch.zeros_like(p), round_e4m3(torch.nan_to_num(p / s[:, :, None])))
    return q.view(m, -1)[:, :k], s


def quantize_weight(w):
    w = w.double()
    n, k = w.shape
    p = torch.nn.functional.pad(w, (0, groups(k) * GROUP - k, 0, groups(n) * GROUP - n)).view(groups(n), GROUP, groups(k), GROUP)
    s = scale_of(torch.where(torch.isfinite(p), p.abs(), torch.full_like(p, math.inf)).amax((1, 3)))
    q = torch.where(torch.isnan(s)[:, None, :, None], torch.zeros_like(p), round_e4m3(torch.nan_to_num(p / s[:, None, :, None])))
    return q.view(groups(n) * GROUP, -1)[:n, :k], s


def row_values(a, scales):
    """What 8-bit rows stand for."""
    return a.double() * scales.double().repeat_interleave(GROUP, 1)[:, : a.shape[1]]


def weight_values(w, scales):
    n, k = w.shape
    return w.double() * scales.double().repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]


def product(a, a_scales, w, w_scales):
    """(a w^T in float64, what 32-bit sums may be away from it).  The tensor cores add the products of a group in four
    instructions, each with at most two units of truncation of its sizes (2^-22); a product of the scales, a product with it and
    an addition to the running sum per group, 2^-24 each, in sizes |a w| added up."""
    x, y = row_values(a, a_scales), weight_values(w, w_scales)
    size = x.abs() @ y.abs().T
    return x @ y.T, (4 * 2.0 ** -22 + (groups(a.shape[1]) + 2) * 2.0 ** -24) * size


def gate(g, u, act, limit=0.0):
    if act == "silu":
        return g * torch.sigmoid(g) * u
    if act == "relu":
        return g.clamp(min=0) * u
    if act == "clamped":
        g = g.clamp(max=limit)
        return g * torch.sigmoid(1.702 * g) * (u.clamp(-limit, limit) + 1)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u


def gated(a, a_scales, w, w_scales, width, act, limit=0.0):
    """(act(gate) * up in float64, what it may be away): no gate is steeper than 1.2, none is larger than its input; the clamped
    one's up side is at most limit + 1; the gate itself is worked out in 32 bits with errors of a few units (2^-20 of the value)."""
    y, off = product(a, a_scales, w, w_scales)
    y, off = y.view(y.shape[0], -1, 2, GROUP), off.view(off.shape[0], -1, 2, GROUP)
    g, u, dg, du = (t[:, :, side].reshape(y.shape[0], -1)[:, :width] for t in (y, off) for side in (0, 1))
    h = gate(g, u, act, limit)
    return h, 1.2 * (u.abs() + 1) * dg + g.abs() * du + 1.2 * dg * du + 2.0 ** -20 * h.abs()


def between_roundings(data, scales, want, off):
    """Whether 8-bit rows are roundings of values at most `off` away from `want`, with the scales that such values have."""
    k = want.shape[1]
    pad = (0, groups(k) * GROUP - k)
    low, high = (torch.nn.functional.pad(t, pad).view(want.shape[0], -1, GROUP).amax(2) for t in ((want.abs() - off).clamp(min=0), want.abs() + off))
    s = scales.double()
    if not bool(((s >= torch.where(low == 0, torch.zeros_like(low), scale_of(low))) & ((s <= scale_of(high)) | (s == 1) & (low == 0))).all()):
        return False
    each = s.repeat_interleave(GROUP, 1)[:, :k]
    top = torch.full_like(want, 448.0)
    lo, hi = (round_e4m3(torch.minimum(torch.maximum((want + sign * off) / each, -top), top)) for sign in (-1, 1))
    q = data.double()
    return bool(((q >= lo) & (q <= hi)).all())

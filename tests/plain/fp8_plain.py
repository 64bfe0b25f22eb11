"""Numbers in 8 bits and products with them, restated in 64 bits.

A code is one of the 253 finite e4m3 values; a group's scale is ``max(float32(a / 448), 2^-100)``.
Which code a number gets is decided without a quotient: middles of neighbouring codes times a float32
scale fit 64 bits exactly, so ``|x|`` is compared with them.
"""
import torch

F32, F64 = torch.float32, torch.float64
GROUP, LARGEST, FLOOR = 128, 448.0, 2.0 ** -100


def values(device="cpu"):
    """The values of the codes 0 .. 126, float64."""
    return torch.arange(127, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn).to(F64)


def nearest(x, s):
    """Codes' values (float64, signed) of ``x`` for scales ``s`` of its shape, ties to the even code."""
    v = values(x.device)
    a, mid = x.to(F64).abs(), (v[1:] + v[:-1]) / 2
    at = torch.zeros(x.shape, dtype=torch.long, device=x.device)
    for step in (64, 32, 16, 8, 4, 2, 1):             # the last code whose lower middle is not above a
        t = (at + step).clamp_max(126)
        low = mid[(t - 1).clamp_min(0)] * s.to(F64)
        above = (a > low) | ((a == low) & (t % 2 == 0))
        at = torch.where((at + step <= 126) & above, t, at)
    return torch.where(x < 0, -v[at], v[at])


def scale(largest):
    s = (largest.to(F64) / torch.full_like(largest, LARGEST, dtype=F64)).to(F32).clamp_min(FLOOR)
    return torch.where(torch.isfinite(largest), s, torch.full_like(s, float("nan")))


def hold(x, rows):
    """``(values of the codes [T, K] float64, scales float32 [ceil(T / rows), ceil(K / 128)])`` of groups of
    ``rows`` x 128 numbers."""
    T, K = x.shape
    pad = torch.nn.functional.pad(x.to(F32), [0, -K % GROUP, 0, -T % rows])
    g = pad.reshape(pad.shape[0] // rows, rows, pad.shape[1] // GROUP, GROUP)
    s = scale(g.abs().amax(dim=(1, 3)))
    each = s.repeat_interleave(rows, 0).repeat_interleave(GROUP, 1)[:T, :K]
    return torch.where(torch.isnan(each), torch.nan, nearest(x, each)), s


def hold_weight(w, gated=False):
    if not gated:
        return hold(w, GROUP)
    n = w.shape[0] // 2
    a, b = hold(w[:n], GROUP), hold(w[n:], GROUP)
    return torch.cat([a[0], b[0]]), torch.cat([a[1], b[1]])


def spread(scales, rows, shape):
    return scales.to(F64).repeat_interleave(rows, 0)[:shape[0]].repeat_interleave(GROUP, 1)[:, :shape[1]]


def dense(codes, scales, rows, gated=False):
    """What codes (their values) and scales stand for, float64."""
    if gated:
        n, b = codes.shape[0] // 2, scales.shape[0] // 2
        return torch.cat([dense(codes[:n], scales[:b], rows), dense(codes[n:], scales[b:], rows)])
    return codes.to(F64) * spread(scales, rows, codes.shape)


def product(x, w_codes, w_scales, gated=False, act=None):
    """``(result float64, how far a sum in float may be off)`` of rows ``x`` against a held weight.

    The bound: 128 products of codes are whole multiples of 2^-18 below 2^25, added up by the tensor
    cores with at most 2^-23 of the sizes' sum lost each; then a factor (two roundings) and an addition
    per group.  (128 + 2 + groups) 2^-23 of the sum of the sizes is above all of it."""
    cx, sx = hold(x, 1)
    a, b = dense(cx, sx, 1), dense(w_codes, w_scales, GROUP, gated)
    y = a @ b.t()
    off = (a.abs() @ b.abs().t()) * ((130 + sx.shape[1]) * 2.0 ** -23)
    if not gated:
        return y, off
    g, u = y.chunk(2, dim=1)
    og, ou = off.chunk(2, dim=1)
    act = act or (lambda g, u: (g * torch.sigmoid(g), u))
    ag, au = act(g, u)
    # (the activations' slopes are at most 1.1; exp and the quotient are good to 2^-20 in the kernels)
    return ag * au, 1.1 * og * au.abs() + ou * ag.abs() + 1.1 * og * ou + (ag * au).abs() * 2.0 ** -19

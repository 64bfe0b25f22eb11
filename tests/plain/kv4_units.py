"""Attention over a cache in 4 bits with values that show which keys were counted.

Keys come to the kernels sixteen at a time (a unit).  Values are +1 or -1, drawn per unit, head and channel, so that the
result of U units of about equal weight is of size 1 / sqrt(U) and a unit that is left out or counted twice changes it by
1 / U in every channel: 2 % of it at 40,000 keys, 10 % at 1,500.

``attend`` returns the result in 64 bits and how far off a row and kv head may be, in the root mean square over its numbers:
the result's rounding to bfloat16, at most half a step (2^-8) of each number, and that of the probabilities times the value
scales, whose error meets a code's distance from 8, at most 8 of 15 steps of a range of 2.  That is 2^-8 * 16 / 15 of
the whole weight at worst; of more than 32 keys, whose roundings are independent of each other and uniform, twice
2^-8 / sqrt(3) * 16 / 15 of the root of the squared weights' sum."""
import math

import torch

F64, BF16 = torch.float64, torch.bfloat16
HALF_STEP = 2.0 ** -8
UNIT = 16


def values(n, nkv, d, device, seed):
    g = torch.Generator(device).manual_seed(seed)
    s = torch.randint(0, 2, (-(-n // UNIT), nkv, d), generator=g, device=device)
    return (2 * s - 1).to(BF16).repeat_interleave(UNIT, 0)[:n].contiguous()


def keys(n, nkv, d, device, seed):
    return torch.randn((n, nkv, d), generator=torch.Generator(device).manual_seed(seed), device=device).to(BF16)


def attend(q, k, v, positions, window, keep, scale, weight=None):
    """``q [T, nh, d]`` over ``k, v [n, nkv, d]`` (float64): the result ``[T, nh, d]`` and what is allowed
    ``[T, nkv]``.  ``weight [n]``: how often a key counts (once; for mistakes that a test plants)."""
    T, nh, d = q.shape
    n, nkv = k.shape[:2]
    p, j = positions[:, None], torch.arange(n, device=q.device)[None]
    seen = j <= p
    if window is not None:
        seen &= (j > p - window) | (j < keep)
    out = torch.empty((T, nh, d), dtype=F64, device=q.device)
    allowed = torch.empty((T, nkv), dtype=F64, device=q.device)
    group = nh // nkv
    for h in range(nkv):
        s = torch.einsum("tgd,jd->gtj", q[:, h * group:(h + 1) * group], k[:, h]) * scale
        s = s.masked_fill(~seen, -math.inf)
        w = (s - s.amax(-1, keepdim=True)).exp()
        if weight is not None:
            w = w * weight
        w = w / w.sum(-1, keepdim=True)
        o = torch.einsum("gtj,jd->tgd", w, v[:, h])
        out[:, h * group:(h + 1) * group] = o
        spread = torch.where(seen.sum(-1) > 32, 2 / math.sqrt(3) * w.square().sum(-1).sqrt(), 1.0)      # [group, T]
        allowed[:, h] = HALF_STEP * (o.square().mean((1, 2)).sqrt() + 16 / 15 * spread.square().mean(0).sqrt())
    return out, allowed


def off(got, ref, nkv):
    """Root mean square of the difference per row and kv head ``[T, nkv]``."""
    T = ref.shape[0]
    return (got.reshape(ref.shape).to(F64) - ref).view(T, nkv, -1).square().mean(-1).sqrt()


def check(got, ref, allowed):
    far = off(got, ref, allowed.shape[1]) / allowed
    assert (far <= 1).all(), f"{int((~(far <= 1)).sum())} of {far.numel()} too far off, worst {float(far.max()):.3g}"

"""A cache held in 4 bits, restated in plain torch and 64 bits.

What numbers stand for once they are held (``held``), what the bytes of a cache stand for
(``unpack``), attention over such numbers with the error that roundings to bfloat16 may make
(``attend``), and a step's description from lengths and pages (``describe``).
"""
import math

import torch

F64, BF16 = torch.float64, torch.bfloat16
HALF_STEP = 2.0 ** -8            # of bfloat16, relative


def held(x):
    """``x [..., d]`` bfloat16 -> what its codes stand for, float64; a group of 64 numbers with one that
    is not finite is NaN."""
    g = x.to(F64).unflatten(-1, (-1, 64))
    finite = torch.isfinite(g).all(-1, keepdim=True)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).to(BF16).to(F64)
    c = torch.where(s > 0, torch.round((g - lo) / torch.where(s > 0, s, 1.0)).clamp(0, 15), 0.0)
    return torch.where(finite, lo + s * c, math.nan).flatten(-2)


def unpack(cache):
    """Every token of a cache, number by number: ``(k, v)`` float64 ``[pages, kv_heads, page_size, d]``."""
    c = cache.cpu()
    pages, nkv, eighths, rec = c.shape
    d = rec // 9
    k = torch.empty((pages, nkv, eighths, 8, d), dtype=F64)
    v = torch.empty_like(k)
    for at, out in ((8 * d, k), (8 * d + d // 2, v)):
        par = c[..., at:at + d // 2].contiguous().view(BF16).to(F64).view(pages, nkv, eighths, 8, d // 64, 2)
        for i in range(d):
            for tok in range(8):
                e = i % 64
                if out is k:
                    byte = tok * (d // 2) + (e // 16) * (d // 8) + (i // 64) * 8 + (e % 16) // 2
                else:
                    byte = 4 * d + (e // 8) * (d // 2) + tok * (d // 16) + (i // 64) * 4 + (e % 8) // 2
                code = (c[..., byte].to(torch.int64) >> (4 * (i % 2))) & 15
                p = par[:, :, :, tok, i // 64]
                out[:, :, :, tok, i] = p[..., 1] + p[..., 0] * code
    shape = (pages, nkv, eighths * 8, d)
    return k.reshape(shape), v.reshape(shape)


def seen(positions, n, window, keep):
    """bool ``[rows, n]``: which keys rows at these positions see."""
    p, j = positions[:, None], torch.arange(n, device=positions.device)[None]
    m = j <= p
    if window is not None:
        m &= (j > p - window) | (j < keep)
    return m


def attend(q, k, v, positions, window, keep, scale):
    """Rows ``q [T, nh, d]`` over keys and values ``[n, nkv, d]`` (float64): the result ``[T, nh, d]`` and
    the error allowed.  Roundings to bfloat16 that a kernel may make: the result; the probabilities before
    the product with the values, whose error meets a value's distance from the middle of its group's codes,
    at most 8 of 15 steps of the group's range (a range lies within twice the largest |v|); and, where
    keys and values pass through bfloat16, each of them.  Independent roundings of a score's terms add
    up like a random walk: six standard deviations, a rounding's being 1 / sqrt(3) of half a step.
    A score that is off by e moves a probability by e times itself."""
    T, nh, d = q.shape
    group = nh // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("thd,jhd->htj", q, kk) * scale
    s = s.masked_fill(~seen(positions, k.shape[0], window, keep)[None], -math.inf)
    p = torch.softmax(s, -1)
    o = torch.einsum("htj,jhd->thd", p, vv)
    sp = 6 / math.sqrt(3) * HALF_STEP * abs(scale) * torch.sqrt(torch.einsum("thd,jhd->htj", q * q, kk * kk))
    mag = torch.einsum("htj,jhd->thd", p * (sp + HALF_STEP), vv.abs() + o.abs().amax())
    biggest = vv.abs().amax(-1).T[:, None, :].expand(nh, T, -1)              # [nh, T, n]
    mid = torch.einsum("htj,htj->th", p, biggest) * (16 / 15) * HALF_STEP
    return o, HALF_STEP * o.abs() + mag + mid[..., None] + 1e-30


def describe(master, entries, new_pages, page_size, width):
    """``step_tables`` in Python: a dict of lists (master changed in place)."""
    out = dict(q_start=[0], positions=[], seq=[], ctx_lens=[], slots=[], tables=[], decode_rows=[], items=[])
    for b, (row, start, count, have, off) in enumerate(entries):
        need = 0 if row < 0 else -(-(start + count) // page_size)
        for i in range(have, need):
            master[row][i] = new_pages[off + i - have]
        table = [master[row][i] for i in range(need)]
        first = out["q_start"][-1]
        for p in range(start, start + count):
            page = table[p // page_size] if row >= 0 else 0
            out["positions"].append(p)
            out["seq"].append(b)
            out["slots"].append(page * page_size + p % page_size)
        if count == 1:
            out["decode_rows"].append(first)
        if count > 1:
            out["items"].append([b, first, count, start])
        out["q_start"].append(first + count)
        out["ctx_lens"].append(start + count)
        out["tables"].append(table + [0] * (width - need))
    return out

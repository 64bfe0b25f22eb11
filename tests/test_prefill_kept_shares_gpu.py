"""Portions over bfloat16 pages behind a window that keeps first tokens, their keys shared out over several blocks."""
import math
import random

import pytest
import torch

import kv4_units as U

pytestmark = pytest.mark.gpu

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32


@pytest.mark.parametrize("nh,nkv,ps", [(4, 2, 16), (2, 2, 8), (6, 1, 64)])
@pytest.mark.parametrize("window,keep", [(64, 4), (1, 64), (200, 100), (700, 300), (90, 1), (1500, 5000)])
@pytest.mark.parametrize("splits", [2, 3, 8])
@pytest.mark.parametrize("sinks", [False, True])
def test_kept_tokens_with_keys_shared_out(cuda_device, nh, nkv, ps, window, keep, splits, sinks):
    """Values that show a unit left out or counted twice; pages that no row sees have been given back."""
    from binfer_b200.csrc import ops
    dev, d, lens, new = cuda_device, 128, [300, 70, 1800, 2, 257], [300, 37, 260, 2, 129]
    g = torch.Generator(dev).manual_seed(nh + ps)
    sink = torch.randn(nh, generator=g, device=dev) * 2
    need = [-(-n // ps) for n in lens]
    ids = list(range(1, sum(need) + 4))
    random.Random(ps).shuffle(ids)
    kc, vc = torch.full((2, len(ids) + 1, nkv, ps, d), math.nan, dtype=BF16, device=dev)
    tables = torch.full((len(lens), max(need)), -1, dtype=I32)
    ks, vs, items, row = [], [], [], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = U.keys(n, nkv, d, dev, 2 * b), U.values(n, nkv, d, dev, 2 * b + 1)
        first = max(0, n - m - window + 1) // ps
        for x in range(need[b]):
            if x >= -(-keep // ps) and x < first:
                continue
            page = ids.pop()
            tables[b, x] = page
            for c, rows in ((kc, k), (vc, v)):
                part = rows[x * ps:x * ps + ps].transpose(0, 1)
                c[page] = 0                      # (places behind a context are finite)
                c[page, :, :part.shape[1]] = part
        ks.append(k), vs.append(v)
        items.append((b, row, m, n - m))
        row += m
    q = torch.randn((row, nh * d), generator=g, device=dev).to(BF16)
    out, err = torch.full_like(q, math.nan), torch.zeros(1, dtype=I32, device=dev)
    ops.prefill_attention(q, kc, vc, torch.tensor(items, dtype=I32, device=dev), len(items), max(new), tables.to(dev), out,
                          nh, nkv, d, window, d ** -0.5, err, variant="umma2", splits=splits, keep_first=keep,
                          sinks=sink if sinks else None)
    assert int(err.item()) == 0
    for b, at, m, first in items:
        where = torch.arange(first, first + m, device=dev)
        k, v, x = ks[b].to(F64), vs[b].to(F64), q[at:at + m].view(m, nh, d).to(F64)
        ref, allowed = U.attend(x, k, v, where, window, keep, d ** -0.5)
        if sinks:                                # every head's result times its keys' share of the sum
            j = torch.arange(lens[b], device=dev)
            seen = (j <= where[:, None]) & ((j > where[:, None] - window) | (j < keep))
            s = torch.einsum("thd,jhd->htj", x, k.repeat_interleave(nh // nkv, 1)) * d ** -0.5
            total = torch.logsumexp(s.masked_fill(~seen, -math.inf), -1)
            ref = ref * torch.sigmoid(total - sink.to(F64)[:, None]).T[..., None]
        U.check(out[at:at + m], ref, allowed)

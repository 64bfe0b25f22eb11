"""Which keys the attention kernels over a cache in 4 bits count: values that show a unit of sixteen that is left out or
counted twice (``kv4_units``), in every form and at every place where work is cut."""
import math

import pytest
import torch

import kv4_plain as K4
import kv4_units as U
from test_kv4_gpu import Cache, _attention, _queries

pytestmark = pytest.mark.gpu

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32


@pytest.fixture(params=[1, 200, 1 << 12])
def tables(request, monkeypatch):
    monkeypatch.setattr(Cache, "places", request.param)


def _cache(lens, nkv, d, ps, dev, seed=0):
    from binfer_b200.csrc import ops
    c = Cache(lens, nkv, d, ps, dev, seed=seed)
    for i, n in enumerate(lens):
        c.k[i], c.v[i] = U.keys(n, nkv, d, dev, 7 * seed + 2 * i), U.values(n, nkv, d, dev, 7 * seed + 2 * i + 1)
        ops.kv4_store(c.k[i].flatten(1), c.v[i].flatten(1), c.slots[i], c.cache, c.err)
    return c


def _check(c, q, out, nh, jobs, window, keep, scale, pick=None):
    at = 0
    for x, (b, n, p) in enumerate(jobs):
        if pick is None or x in pick:
            k, v = c.held(b)
            ref, allowed = U.attend(q[at:at + n].view(n, nh, c.d).to(F64), k[:n + p], v[:n + p],
                                    torch.arange(p, p + n, device=q.device), window, keep, scale)
            U.check(out[at:at + n], ref, allowed)
        at += n
    assert int(c.err.item()) == 0


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("nh,nkv,d,ps", [(32, 8, 128, 16), (16, 8, 128, 8), (64, 8, 128, 64), (5, 1, 128, 128),
                                         (12, 4, 64, 16), (20, 1, 64, 8), (6, 6, 256, 128), (32, 2, 256, 16)])
@pytest.mark.parametrize("window,keep", [(None, 0), (40, 0), (1000, 70)])
@pytest.mark.parametrize("lens", [[2063], [1, 17, 700, 129, 1500, 64, 33], [4096, 31, 2730]])
def test_single_tokens(cuda_device, nh, nkv, d, ps, window, keep, lens):
    c = _cache(lens, nkv, d, ps, cuda_device, seed=nh + ps)
    q = _queries(len(lens), nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    jobs = [(b, 1, n - 1) for b, n in enumerate(lens)]
    _attention(c, q, out, nh, jobs, True, window, keep, d ** -0.5)
    _check(c, q, out, nh, jobs, window, keep, d ** -0.5)


def test_many_rows_and_a_long_one(cuda_device):
    nh, nkv, d = 4, 1, 128
    lens = [1 + i % 40 for i in range(598)] + [40000, 9000]
    c = _cache(lens, nkv, d, 16, cuda_device)
    q = _queries(600, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    jobs = [(b, 1, n - 1) for b, n in enumerate(lens)]
    _attention(c, q, out, nh, jobs, True, None, 0, d ** -0.5)
    _check(c, q, out, nh, jobs, None, 0, d ** -0.5, pick={0, 1, 39, 511, 512, 513, 598, 599})


def test_a_full_batch(cuda_device):
    """Stretches that cross heads and rows, their ends anywhere in a row."""
    nh, nkv, d = 64, 8, 128
    lens = [1500 - 19 * i for i in range(64)]
    c = _cache(lens, nkv, d, 16, cuda_device)
    q = _queries(64, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    jobs = [(b, 1, n - 1) for b, n in enumerate(lens)]
    _attention(c, q, out, nh, jobs, True, None, 0, d ** -0.5)
    _check(c, q, out, nh, jobs, None, 0, d ** -0.5)


@pytest.mark.parametrize("variant", ["stretches", "load"])
@pytest.mark.parametrize("nh,nkv,d,ps", [(8, 2, 128, 16), (16, 1, 128, 8), (6, 3, 64, 32), (4, 1, 256, 128)])
@pytest.mark.parametrize("window,keep", [(None, 0), (120, 9), (900, 70)])
@pytest.mark.parametrize("jobs", [[(0, 2, 698)], [(2, 7, 0), (0, 5, 400), (1, 1, 3), (3, 3, 997)],
                                  [(0, 700, 0), (3, 300, 700)], [(4, 130, 2000), (1, 33, 0)], [(4, 40, 4200)]])
def test_portions(cuda_device, variant, nh, nkv, d, ps, window, keep, jobs):
    from binfer_b200.csrc import ops
    c = _cache([700, 33, 7, 1000, 4240], nkv, d, ps, cuda_device, seed=d + ps)
    T = sum(n for _, n, _ in jobs)
    q = _queries(T, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    items, at = [], 0
    for b, n, p in jobs:
        items.append((b, at, n, p))
        at += n
    ops.kv4_prefill_attention(q, c.cache, torch.tensor(items, dtype=I32, device=cuda_device), len(items),
                              max(n for _, n, _ in jobs), c.tables, out, nh, nkv, d, window, d ** -0.5, c.err,
                              ctx_rows=sum(-(-(n + p) // 64) * 64 for _, n, p in jobs),
                              max_ctx=max(n + p for _, n, p in jobs), keep_first=keep, variant=variant)
    _check(c, q, out, nh, jobs, window, keep, d ** -0.5)

"""The operators of a paged cache held in 4 bits against their restatement in 64 bits."""
import gc
import math
import random

import pytest
import torch

import kv4_plain as K4

pytestmark = pytest.mark.gpu

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32


def _err(dev):
    return torch.zeros(1, dtype=I32, device=dev)


def _rows(T, nkv, d, dev, seed, size=1.0):
    g = torch.Generator(dev).manual_seed(seed)
    x = torch.randn((T, nkv, d), generator=g, device=dev) * size
    return (x + 0.7 * torch.randn((nkv, d), generator=g, device=dev)).to(BF16)


class Cache:
    """Requests of given lengths in a shuffled pool; keys and values as rows and as held."""

    places = 1          # of the tables beyond what the longest request needs

    def __init__(self, lens, nkv, d, ps, dev, seed=0, spare=3):
        from binfer_b200.csrc import ops
        self.lens, self.ps, self.nkv, self.d, self.dev = lens, ps, nkv, d, dev
        need = [-(-n // ps) for n in lens]
        ids = list(range(1, sum(need) + spare + 1))
        random.Random(seed).shuffle(ids)
        self.pages = len(ids) + 1
        self.cache = ops.kv4_cache(self.pages, nkv, ps, d, dev)
        self.err = _err(dev)
        self.tables = torch.full((len(lens), max(need) + self.places), -1, dtype=I32)
        self.k, self.v, self.slots = [], [], []
        for i, n in enumerate(lens):
            pg = [ids.pop() for _ in range(need[i])]
            self.tables[i, :need[i]] = torch.tensor(pg, dtype=I32)
            p = torch.arange(n)
            self.slots.append((torch.tensor(pg)[p // ps] * ps + p % ps).to(I32).to(dev))
            self.k.append(_rows(n, nkv, d, dev, 100 * seed + 2 * i))
            self.v.append(_rows(n, nkv, d, dev, 100 * seed + 2 * i + 1))
            ops.kv4_store(self.k[i].flatten(1), self.v[i].flatten(1), self.slots[i], self.cache, self.err)
        self.tables = self.tables.to(dev)

    def held(self, i):
        return K4.held(self.k[i]), K4.held(self.v[i])


@pytest.fixture(params=[1, 200, 1 << 12])
def tables(request, monkeypatch):
    """Single tokens and short portions take one of several forms by how many keys the tables have room for: a
    block a head, a cluster of two to eight, stretches."""
    monkeypatch.setattr(Cache, "places", request.param)


def _check(got, ref, allowed):
    off = (got.to(F64) - ref).abs()
    bad = ~(off <= allowed)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} too far off, worst "
                           f"{float((off / allowed).max()):.3g} of what is allowed")


# ------------------------------------------------------------------------------ store and load
@pytest.mark.parametrize("d,ps,nkv,T", [(128, 16, 8, 1), (128, 16, 2, 333), (64, 8, 1, 77), (256, 128, 3, 130),
                                        (64, 64, 5, 200), (128, 32, 1, 31)])
def test_store_holds_what_the_formula_says(cuda_device, d, ps, nkv, T):
    from binfer_b200.csrc import ops
    c = Cache([T], nkv, d, ps, cuda_device, seed=d + T)
    k, v = K4.unpack(c.cache)
    at = c.slots[0].long().cpu()
    for x, got in ((c.k[0], k), (c.v[0], v)):
        got = got.permute(0, 2, 1, 3).reshape(-1, nkv, d)
        assert torch.equal(got[at], K4.held(x).cpu())
        other = torch.ones(got.shape[0], dtype=torch.bool)
        other[at] = False
        assert not got[other].any()                     # no other place was written
    assert int(c.err.item()) == 0


def test_store_of_rows_in_a_wider_buffer_and_off_alignment(cuda_device):
    from binfer_b200.csrc import ops
    T, nkv, d, ps = 21, 2, 128, 16
    k, v = _rows(T, nkv, d, cuda_device, 1), _rows(T, nkv, d, cuda_device, 2)
    slots = torch.arange(16, 16 + T, dtype=I32, device=cuda_device)
    want = ops.kv4_cache(4, nkv, ps, d, cuda_device)
    ops.kv4_store(k.flatten(1), v.flatten(1), slots, want, _err(cuda_device))
    for shift in (0, 1, 2, 4):
        wide = torch.full((T, 3 * nkv * d + 13), 9.0, dtype=BF16, device=cuda_device)
        a, b = wide[:, shift:shift + nkv * d], wide[:, nkv * d + 5:2 * nkv * d + 5]
        a.copy_(k.flatten(1)), b.copy_(v.flatten(1))
        got = ops.kv4_cache(4, nkv, ps, d, cuda_device)
        ops.kv4_store(a, b, slots, got, _err(cuda_device))
        assert torch.equal(got, want)


def test_store_of_hard_numbers(cuda_device):
    """Ties, constant groups, the largest and smallest bfloat16 numbers, numbers that are not finite."""
    from binfer_b200.csrc import ops
    rows = torch.zeros((8, 64))
    rows[0, 1], rows[0, 2:18] = 15.0, torch.arange(16) + 0.5 - 0.5 * (torch.arange(16) % 3 == 0)
    rows[1] = -3.25
    rows[2, 0], rows[2, 5], rows[2, 6] = 3.38e38, -3.38e38, 1e38
    rows[3] = torch.arange(64) * 2.0 ** -133
    rows[4, 7] = math.nan
    rows[5, 9] = math.inf
    rows[6, 9] = -math.inf
    rows[7] = torch.linspace(1000.0, 1007.0, 64)
    x = rows.to(BF16).to(cuda_device)
    c = ops.kv4_cache(2, 1, 8, 64, cuda_device)
    err = _err(cuda_device)
    ops.kv4_store(x, x.flip(0), torch.arange(8, 16, dtype=I32, device=cuda_device), c, err)
    k, v = K4.unpack(c)
    want = K4.held(x).cpu()
    for got, w in ((k[1, 0], want), (v[1, 0], want.flip(0))):
        assert torch.equal(torch.nan_to_num(got, nan=123.0), torch.nan_to_num(w, nan=123.0))
    assert torch.isnan(want[4:7]).all() and torch.isfinite(want[[0, 1, 2, 3, 7]]).all()


def test_store_leaves_out_negative_slots_and_flags_bad_ones(cuda_device):
    from binfer_b200.csrc import ops
    k = _rows(4, 1, 64, cuda_device, 3)
    c, err = ops.kv4_cache(3, 1, 8, 64, cuda_device), _err(cuda_device)
    slots = torch.tensor([-1, 9, 24, 2 ** 31 - 1], dtype=I32, device=cuda_device)
    ops.kv4_store(k.flatten(1), k.flatten(1), slots, c, err)
    assert int(err.item()) == 2
    got = K4.unpack(c)[0].reshape(24, 64)
    assert torch.equal(got[9], K4.held(k[1, 0]).cpu())
    assert not got[torch.arange(24) != 9].any()
    before = c.clone()
    ops.kv4_store(k[:0].flatten(1), k[:0].flatten(1), slots[:0], c, err)     # no tokens
    assert torch.equal(c, before)


@pytest.mark.parametrize("d,ps,nkv", [(128, 16, 2), (64, 8, 3), (256, 128, 1), (128, 64, 8)])
@pytest.mark.parametrize("window,keep", [(None, 0), (70, 0), (33, 5), (1, 130)])
def test_load(cuda_device, d, ps, nkv, window, keep):
    from binfer_b200.csrc import ops
    lens, new = [300, 1, 64, 449], [17, 1, 64, 200]
    c = Cache(lens, nkv, d, ps, cuda_device, seed=ps)
    order = [3, 0, 2, 1]                                # portions in another order than the requests
    items = torch.tensor([(b, 5 * i, new[b], lens[b] - new[b]) for i, b in enumerate(order)], dtype=I32,
                         device=cuda_device)
    each = [-(-lens[b] // 64) for b in order]
    moved = torch.zeros_like(items)
    k, v, tables = ops.kv4_load(c.cache, c.tables, items, 4, 64 * (sum(each) + 2), c.err, window, keep,
                                items_out=moved)
    assert int(c.err.item()) == 0
    want_items = items.clone()
    want_items[:, 0] = torch.arange(4)
    assert torch.equal(moved, want_items)
    for x in (k, v):
        assert not x[0].any() and not x[1 + sum(each):].any()
    page = 1
    for i, b in enumerate(order):
        n = each[i]
        vis = K4.seen(torch.arange(lens[b] - new[b], lens[b]), 64 * n, window, keep).any(0).view(n, 64)
        want = torch.where(vis.any(1), torch.arange(page, page + n), 0)
        assert torch.equal(tables[i, :n].cpu(), want.to(I32)) and not tables[i, n:].any()
        for x, h in ((k, c.held(b)[0]), (v, c.held(b)[1])):
            for j in range(n):
                if not vis[j].any():
                    continue
                got = x[page + j].transpose(0, 1).to(F64).cpu()                # [64, nkv, d]
                ref = torch.zeros_like(got)
                part = h[64 * j:64 * j + 64].cpu()
                ref[:part.shape[0]] = part
                ref[~vis[j]] = 0
                assert ((got - ref).abs() <= 1.001 * K4.HALF_STEP * ref.abs()).all()
        page += n


def test_load_flags_pages_and_rows_that_do_not_fit(cuda_device):
    from binfer_b200.csrc import ops
    c = Cache([100], 1, 64, 16, cuda_device)
    items = torch.tensor([[0, 0, 100, 0]], dtype=I32, device=cuda_device)
    bad = c.tables.clone()
    bad[0, 2] = c.pages
    k, v, _ = ops.kv4_load(c.cache, bad, items, 1, 128, c.err)
    assert int(c.err.item()) == 4 and not k[1, 0, 32:48].any() and k[1, 0, 48:].any()
    c.err.zero_()
    ops.kv4_load(c.cache, c.tables, items, 1, 64, c.err)          # room for one of the two pages
    assert int(c.err.item()) == 16


@pytest.mark.parametrize("T,nh,nkv,d,ps,rot,norms,scaled", [
    (1, 32, 8, 128, 16, 64, True, False), (1, 2, 2, 128, 8, 64, False, True), (65, 16, 8, 128, 64, 64, True, True),
    (700, 4, 2, 128, 16, 64, True, False), (33, 6, 3, 128, 128, 32, True, False), (17, 4, 4, 64, 32, 32, True, True),
    (40, 3, 1, 256, 16, 0, False, False)])
def test_norm_rotation_and_store_in_one(cuda_device, T, nh, nkv, d, ps, rot, norms, scaled):
    """The same bits as head norms and rotation into rows of bfloat16, and those stored."""
    from binfer_b200.csrc import ops
    dev = cuda_device
    g = torch.Generator(dev).manual_seed(T)
    width = (nh + 2 * nkv) * d
    qkv = torch.randn((T, width + 64), generator=g, device=dev).to(BF16)[:, :width]
    w = [torch.rand(d, generator=g, device=dev) + 0.5 if norms else None for _ in range(2)]
    freq = 10000.0 ** (-torch.arange(rot, device=dev) / max(rot, 1)) if rot else None
    scale = ops.RowScale(torch.rand((T, 3), generator=g, device=dev) + 0.1, 5, 1e-6) if scaled else None
    positions = torch.randint(0, 9000, (T,), generator=g, device=dev, dtype=I32)
    pages = -(-T // ps) + 2
    slots = torch.randperm(pages * ps, generator=g, device=dev)[:T].to(I32)
    if T > 20:
        qkv[3, nh * d + 5], qkv[4, -3], qkv[5, nh * d:], qkv[6, -d:-d + 64] = math.inf, math.nan, 0, 3e38
        qkv[7, -d::2], qkv[8, -d:] = -3e38, 1e-38
        slots[9], slots[10] = -1, pages * ps
    want_q, got_q = torch.empty((2, T, nh * d), dtype=BF16, device=dev)
    k, v = torch.zeros((2, T, nkv, 1, d), dtype=BF16, device=dev)
    want, got = ops.kv4_cache(pages, nkv, ps, d, dev), ops.kv4_cache(pages, nkv, ps, d, dev)
    err, err2 = _err(dev), _err(dev)
    ops.qk_norm_rope_kv_write(qkv, w[0], w[1], freq, positions, torch.arange(T, dtype=I32, device=dev), want_q, k, v,
                              nh, nkv, d, 1e-6, err, row_scale=scale)
    ops.kv4_store(k.flatten(1), v.flatten(1), slots, want, err)
    n = ops.launches()
    ops.qk_norm_rope_kv4_store(qkv, w[0], w[1], freq, positions, slots, got_q, got, nh, nkv, d, 1e-6, err2, row_scale=scale)
    assert ops.launches() - n == 1
    assert got_q.view(torch.int16).equal(want_q.view(torch.int16)) and int(err.item()) == int(err2.item()) == (2 if T > 20 else 0)
    assert torch.equal(got, want)
    assert T < 21 or got.any()


def test_token_rows_first_asked_for_in_a_capture(cuda_device):
    from binfer_b200.csrc import ops
    ops._token_rows.clear()
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = ops.token_rows(100, cuda_device) + 1
    assert ops.token_rows(100, cuda_device).tolist() == list(range(100))
    graph.replay()
    torch.cuda.synchronize()
    assert inside.tolist() == list(range(1, 101)) and ops.token_rows(70, cuda_device).tolist() == list(range(70))


# ------------------------------------------------------------------------------ attention
def _attention(c, q, out, nh, jobs, decode, window, keep, scale):
    """``jobs``: (request, rows, first position)."""
    from binfer_b200.csrc import ops
    dev, at, items = q.device, 0, []
    for b, n, p in jobs:
        items.append((b, at, n, p))
        at += n
    if decode:
        seq = torch.tensor([b for b, _, _ in jobs], dtype=I32, device=dev)
        pos = torch.tensor([p for _, _, p in jobs], dtype=I32, device=dev)
        ops.kv4_decode_attention(q, c.cache, None, len(jobs), seq, pos, c.tables, out, nh, c.nkv, c.d, window,
                                 scale, c.err, keep_first=keep)
    else:
        ctx = sum(-(-(n + p) // 64) * 64 for _, n, p in jobs)
        ops.kv4_prefill_attention(q, c.cache, torch.tensor(items, dtype=I32, device=dev), len(items),
                                  max(n for _, n, _ in jobs), c.tables, out, nh, c.nkv, c.d, window, scale,
                                  c.err, ctx_rows=ctx, max_ctx=max(n + p for _, n, p in jobs), keep_first=keep)


def _compare(c, q, out, nh, jobs, window, keep, scale):
    at = 0
    for b, n, p in jobs:
        k, v = c.held(b)
        ref, allowed = K4.attend(q[at:at + n].view(n, nh, c.d).to(F64), k[:n + p], v[:n + p],
                                 torch.arange(p, p + n, device=q.device), window, keep, scale)
        _check(out[at:at + n].view(n, nh, c.d), ref, allowed)
        at += n
    assert int(c.err.item()) == 0


def _queries(T, nh, d, dev, seed=5):
    return torch.randn((T, nh * d), generator=torch.Generator(dev).manual_seed(seed), device=dev).to(BF16)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("nh,nkv,d,ps", [(32, 8, 128, 16), (16, 8, 128, 8), (64, 8, 128, 64), (5, 1, 128, 16),
                                         (16, 1, 128, 32), (12, 4, 64, 16), (6, 6, 256, 128), (20, 1, 64, 8),
                                         (32, 2, 256, 16)])
@pytest.mark.parametrize("window,keep", [(None, 0), (40, 0), (200, 7), (1, 20)])
def test_decode_attention(cuda_device, nh, nkv, d, ps, window, keep):
    lens = [1, 2, 15, 16, 17, 700, 129, 1500, 64]
    c = Cache(lens, nkv, d, ps, cuda_device, seed=nh + ps)
    q = _queries(len(lens), nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    jobs = [(b, 1, n - 1) for b, n in enumerate(lens)]
    _attention(c, q, out, nh, jobs, True, window, keep, d ** -0.5)
    _compare(c, q, out, nh, jobs, window, keep, d ** -0.5)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("nh,nkv,d,ps", [(8, 2, 128, 16), (16, 1, 128, 8), (6, 3, 64, 32), (4, 1, 256, 128),
                                         (3, 3, 128, 128), (18, 1, 64, 16)])
@pytest.mark.parametrize("window,keep", [(None, 0), (50, 0), (120, 9), (1, 0)])
@pytest.mark.parametrize("jobs", [[(0, 2, 698)], [(2, 7, 0), (0, 5, 400), (1, 1, 3), (3, 3, 997)],
                                  [(0, 700, 0), (3, 300, 700)], [(4, 130, 2000), (1, 33, 0)]])
def test_prefill_attention(cuda_device, nh, nkv, d, ps, window, keep, jobs):
    c = Cache([700, 33, 7, 1000, 2130], nkv, d, ps, cuda_device, seed=d + ps)
    T = sum(n for _, n, _ in jobs)
    q = _queries(T, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    _attention(c, q, out, nh, jobs, False, window, keep, d ** -0.5)
    _compare(c, q, out, nh, jobs, window, keep, d ** -0.5)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("decode", [True, False])
def test_attention_of_scores_far_apart(cuda_device, decode):
    """Scores of some hundreds, growing and falling along the context, in both signs of the scale."""
    nh, nkv, d, ps = 4, 1, 128, 16
    c = Cache([900], nkv, d, ps, cuda_device)
    q = _queries(3, nh, d, cuda_device) * 12
    for scale in (0.5, -0.5, 0.0):
        out = torch.empty_like(q)
        jobs = [(0, 1, 899), (0, 1, 500), (0, 1, 20)] if decode else [(0, 3, 897)]
        _attention(c, q, out, nh, jobs, decode, None, 0, scale)
        _compare(c, q, out, nh, jobs, None, 0, scale)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("size", [2.0 ** 40, 2.0 ** -40])
@pytest.mark.parametrize("decode", [True, False])
def test_attention_of_large_and_small_numbers(cuda_device, decode, size):
    nh, nkv, d, ps = 8, 2, 64, 16
    c = Cache([333], nkv, d, ps, cuda_device)
    from binfer_b200.csrc import ops
    c.v[0] = (c.v[0].float() * size).to(BF16)
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(2, nh, d, cuda_device)
    out = torch.empty_like(q)
    jobs = [(0, 1, 332), (0, 1, 100)] if decode else [(0, 2, 331)]
    _attention(c, q, out, nh, jobs, decode, None, 0, d ** -0.5)
    _compare(c, q, out, nh, jobs, None, 0, d ** -0.5)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("rows_new", [1, 3, 90])
def test_numbers_that_are_not_finite_reach_the_rows_that_see_them(cuda_device, rows_new):
    """A token whose key (head 0) or value (head 1) is not finite: rows that see it have NaN there, all
    others are as without it; a place behind the context or a window may hold anything."""
    from binfer_b200.csrc import ops
    nh, nkv, d, ps, n = 6, 3, 128, 16, 300
    c = Cache([n + 20], nkv, d, ps, cuda_device)
    q = _queries(rows_new, nh, d, cuda_device)
    first = n - rows_new
    jobs = [(0, rows_new, first)]

    def run(window, keep, poison):
        k, v = c.k[0].clone(), c.v[0].clone()
        for j in poison:
            k[j, 0, 5], v[j, 1, 70] = math.nan, math.inf
        ops.kv4_store(k.flatten(1), v.flatten(1), c.slots[0], c.cache, c.err)
        out = torch.empty_like(q)
        _attention(c, q, out, nh, jobs, rows_new == 1, window, keep, d ** -0.5)
        return out.view(rows_new, nkv, nh // nkv, d)

    clean = run(100, 4, [])
    assert torch.isfinite(clean).all()
    assert torch.equal(run(100, 4, [5, 20, first - 100, n, n + 7, n + 19]), clean)
    at = n - 1 - rows_new // 3                          # seen by the rows from `at` on
    got = run(100, 4, [at])
    sees = torch.arange(first, n, device=q.device) >= at
    assert torch.equal(got[~sees], clean[~sees])
    assert torch.isnan(got[sees][:, 0]).all()
    assert torch.isnan(got[sees][:, 1, :, 64:]).all() and torch.equal(got[sees][:, 1, :, :64], clean[sees][:, 1, :, :64])
    assert torch.equal(got[sees][:, 2], clean[sees][:, 2])


@pytest.mark.usefixtures("tables")
def test_decode_attention_of_listed_rows(cuda_device):
    """Rows in any order, out in a column block; other rows and columns stay as they were."""
    from binfer_b200.csrc import ops
    nh, nkv, d = 8, 2, 128
    c = Cache([77, 401, 5], nkv, d, 16, cuda_device)
    wide = torch.randn((9, 3 * nh * d), device=cuda_device).to(BF16)
    q, out_wide = wide[:, nh * d:2 * nh * d], torch.full((9, 2 * nh * d), 7.0, dtype=BF16, device=cuda_device)
    out = out_wide[:, :nh * d]
    seq = torch.tensor([9, 0, 9, 9, 1, 9, 9, 2, 9], dtype=I32, device=cuda_device)
    pos = torch.tensor([0, 76, 0, 0, 400, 0, 0, 4, 0], dtype=I32, device=cuda_device)
    rows = torch.tensor([7, 1, 4], dtype=I32, device=cuda_device)
    ops.kv4_decode_attention(q, c.cache, rows, 3, seq, pos, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err)
    for t, b in ((7, 2), (1, 0), (4, 1)):
        k, v = c.held(b)
        ref, allowed = K4.attend(q[t:t + 1].reshape(1, nh, d).to(F64), k, v, pos[t:t + 1].long(), None, 0, d ** -0.5)
        _check(out[t:t + 1].reshape(1, nh, d), ref, allowed)
    rest = [0, 2, 3, 5, 6, 8]
    assert (out_wide[rest] == 7).all() and (out_wide[:, nh * d:] == 7).all() and int(c.err.item()) == 0


@pytest.mark.parametrize("decode", [True, False])
def test_attention_flags_bad_pages_and_requests(cuda_device, decode):
    nh, nkv, d = 4, 2, 64
    c = Cache([200, 90], nkv, d, 16, cuda_device)
    q = _queries(2, nh, d, cuda_device)
    jobs = [(0, 1, 199), (1, 1, 89)] if decode else [(1, 2, 88)]
    good = c.tables.clone()
    for bad in (-1, c.pages, 2 ** 31 - 1):
        out = torch.zeros_like(q)
        c.tables = good.clone()
        c.tables[1, 3] = bad
        c.err.zero_()
        _attention(c, q, out, nh, jobs, decode, None, 0, 0.1)
        assert int(c.err.item()) & 4 and torch.isfinite(out.float()).all()
    c.tables = good
    c.err.zero_()
    _attention(c, q, torch.zeros_like(q), nh, [(b + 2, n, p) for b, n, p in jobs], decode, None, 0, 0.1)
    assert int(c.err.item()) & 4                         # no such request
    c.err.zero_()
    _attention(c, q, torch.zeros_like(q), nh, [(b, n, p + 5000) for b, n, p in jobs], decode, None, 0, 0.1)
    assert int(c.err.item()) & 4                         # keys behind the table's end


def test_many_rows_and_long_contexts(cuda_device):
    """700 rows in one call, contexts from one token on; one row of 40,000 keys among short ones."""
    nh, nkv, d = 4, 1, 128
    lens = [1 + i % 40 for i in range(699)] + [40000]
    c = Cache(lens, nkv, d, 16, cuda_device)
    q = _queries(700, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    jobs = [(b, 1, n - 1) for b, n in enumerate(lens)]
    _attention(c, q, out, nh, jobs, True, None, 0, d ** -0.5)
    pick = [0, 1, 39, 511, 512, 513, 698, 699]
    for b in pick:
        k, v = c.held(b)
        ref, allowed = K4.attend(q[b:b + 1].view(1, nh, d).to(F64), k, v, torch.tensor([lens[b] - 1], device=q.device),
                                 None, 0, d ** -0.5)
        _check(out[b:b + 1].view(1, nh, d), ref, allowed)
    assert torch.isfinite(out.float()).all() and int(c.err.item()) == 0


def test_offsets_past_32_bits(cuda_device):
    """A pool of more than 4 GiB whose last pages hold the request."""
    from binfer_b200.csrc import ops
    nkv, d, ps, pages, n = 8, 128, 128, 30000, 300
    cache, err = ops.kv4_cache(pages, nkv, ps, d, cuda_device), _err(cuda_device)
    assert cache.numel() > 1 << 32
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=I32, device=cuda_device)
    k, v = _rows(n, nkv, d, cuda_device, 1), _rows(n, nkv, d, cuda_device, 2)
    p = torch.arange(n, device=cuda_device)
    slots = (table[0, p // ps].long() * ps + p % ps).to(I32)
    ops.kv4_store(k.flatten(1), v.flatten(1), slots, cache, err)
    q, out = _queries(1, 32, d, cuda_device), torch.empty((1, 32 * d), dtype=BF16, device=cuda_device)
    ops.kv4_decode_attention(q, cache, None, 1, torch.zeros(1, dtype=I32, device=cuda_device),
                             torch.tensor([n - 1], dtype=I32, device=cuda_device), table, out, 32, nkv, d, None,
                             d ** -0.5, err)
    ref, allowed = K4.attend(q.view(1, 32, d).to(F64), K4.held(k), K4.held(v), torch.tensor([n - 1], device=q.device),
                             None, 0, d ** -0.5)
    _check(out.view(1, 32, d), ref, allowed)
    items = torch.tensor([[0, 0, n, 0]], dtype=I32, device=cuda_device)
    k2, v2, _ = ops.kv4_load(cache, table, items, 1, 320, err)
    got = k2[1:].transpose(1, 2).reshape(-1, nkv, d)[:n].to(F64)
    assert ((got - K4.held(k)).abs() <= 1.001 * K4.HALF_STEP * K4.held(k).abs()).all()
    assert int(err.item()) == 0


@pytest.mark.usefixtures("tables")
# ------------------------------------------------------------------------------ streams and graphs
def test_two_graphs_and_an_eager_call_share_nothing(cuda_device):
    """Captured calls replayed in turn, with other positions than at the capture, beside an eager call."""
    from binfer_b200.csrc import ops
    nh, nkv, d, ps = 16, 4, 128, 16
    c = Cache([3000, 1200, 40, 900], nkv, d, ps, cuda_device)
    pos = torch.zeros(4, dtype=I32, device=cuda_device)
    seq = torch.arange(4, dtype=I32, device=cuda_device)
    q = _queries(4, nh, d, cuda_device)
    items = torch.tensor([[1, 0, 4, 100]], dtype=I32, device=cuda_device)

    def decode(out):
        ops.kv4_decode_attention(q, c.cache, None, 4, seq, pos, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err)

    def prefill(out):
        ops.kv4_prefill_attention(q, c.cache, items, 1, 4, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                                  ctx_rows=1216, max_ctx=1200)

    outs = [torch.zeros_like(q) for _ in range(2)]
    graphs = []
    for f, o in ((decode, outs[0]), (prefill, outs[1])):
        f(o)
        torch.cuda.synchronize()
        gc.collect()                          # (not in the middle of the capture)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f(o)
        graphs.append(g)
    side = torch.cuda.Stream()
    for lens, first in (([3000, 1200, 40, 900], 1196), ([1, 700, 33, 2], 50), ([2222, 3, 40, 899], 900)):
        pos.copy_(torch.tensor(lens, dtype=I32) - 1)
        items[0, 3] = first
        torch.cuda.synchronize()
        eager = torch.zeros_like(q)
        for g, o in zip(graphs, outs):
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        decode(eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, outs[0])
        _compare(c, q, outs[0], nh, [(b, 1, n - 1) for b, n in enumerate(lens)], None, 0, d ** -0.5)
        _compare(c, q, outs[1], nh, [(1, 4, first)], None, 0, d ** -0.5)


@pytest.mark.usefixtures("tables")
def test_results_are_the_same_every_time(cuda_device):
    c = Cache([2500, 17, 800], 4, 128, 16, cuda_device)
    q = _queries(3, 32, 128, cuda_device)
    outs = []
    for _ in range(5):
        out = torch.empty_like(q)
        _attention(c, q, out, 32, [(0, 1, 2499), (1, 1, 16), (2, 1, 799)], True, None, 0, 0.1)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("rows_new", [1, 5])
def test_a_chain_of_layers_described_once(cuda_device, rows_new):
    """Store and attention of several layers in a graph, each reading what the kernel ahead wrote; the rows'
    description read early or not makes no difference."""
    from binfer_b200.csrc import ops
    nh, nkv, d, layers, lens = 8, 2, 128, 6, [700, 70, 2100]
    c = Cache(lens, nkv, d, 16, cuda_device)
    T = rows_new * len(lens)
    slots = torch.cat([c.slots[i][-rows_new:] for i in range(len(lens))])
    seq = torch.arange(len(lens), device=cuda_device).repeat_interleave(rows_new).to(I32)
    pos = torch.cat([torch.arange(n - rows_new, n) for n in lens]).to(I32).to(cuda_device)
    items = torch.tensor([(i, i * rows_new, rows_new, n - rows_new) for i, n in enumerate(lens)], dtype=I32,
                         device=cuda_device)
    first = _queries(T, nh, d, cuda_device)

    def run(described):
        x = first
        for _ in range(layers):
            k = x[:, :nkv * d]
            ops.kv4_store(k, x[:, nkv * d:2 * nkv * d], slots, c.cache, c.err)
            out = torch.empty_like(x)
            if rows_new == 1:
                ops.kv4_decode_attention(x, c.cache, None, T, seq, pos, c.tables, out, nh, nkv, d, None, 0.2, c.err,
                                         described=described)
            else:
                ops.kv4_prefill_attention(x, c.cache, items, len(lens), rows_new, c.tables, out, nh, nkv, d, None, 0.2,
                                          c.err, ctx_rows=704 + 128 + 2112, max_ctx=2100, described=described)
            x = out
        return x

    want = run(False).clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = run(True)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        gc.collect()                          # (not in the middle of the capture)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = run(True)
        for _ in range(20):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
    assert int(c.err.item()) == 0 and torch.isfinite(want.float()).all()


# ------------------------------------------------------------------------------ a step's description
def _describe(dev, master, entries, new_pages, ps, num_pages, width, T=None, n_dec=None, n_pf=None, B=None):
    from binfer_b200.csrc import ops
    T = sum(e[2] for e in entries) if T is None else T
    n_dec = sum(e[2] == 1 for e in entries) if n_dec is None else n_dec
    n_pf = sum(e[2] > 1 for e in entries) if n_pf is None else n_pf
    full = lambda *s: torch.full(s, -77, dtype=I32, device=dev)
    B = len(entries)
    out = dict(q_start=full(B + 1), positions=full(T + 3), seq=full(T + 3), ctx_lens=full(B), slots=full(T + 3),
               tables=full(B, width), decode_rows=full(n_dec), items=full(n_pf, 4))
    err = _err(dev)
    ops.step_tables(master, torch.tensor(entries, dtype=I32, device=dev).view(-1, 5),
                    torch.tensor(new_pages, dtype=I32, device=dev), ps, num_pages, out["q_start"],
                    out["positions"][:T], out["seq"][:T], out["ctx_lens"], out["slots"][:T], out["tables"], err,
                    decode_rows=out["decode_rows"], prefill_items=out["items"])
    return out, int(err.item())


@pytest.mark.parametrize("B,ps,longest", [(1, 16, 1), (3, 8, 40), (33, 16, 700), (300, 1, 3), (64, 128, 5000),
                                          (130, 5, 90)])
def test_step_tables(cuda_device, B, ps, longest):
    rng = random.Random(B + ps)
    rows = rng.sample(range(B + 4), B)
    pool = list(range(1, 40000))
    rng.shuffle(pool)
    width = -(-2 * longest // ps) + 2
    master = [[-5] * width for _ in range(B + 4)]
    entries, new_pages = [], []
    for b in range(B):
        start, count = rng.randint(0, longest), rng.choice([1, 1, 1, 0, 2, rng.randint(1, longest)])
        if b % 7 == 6:
            entries.append((-1, 0, 1, 0, 0))             # padding
            continue
        need = -(-(start + count) // ps)
        have = rng.randint(0, need + 1)                  # also more than the step needs
        have = min(have, width)
        for i in range(have):
            master[rows[b]][i] = pool.pop()
        entries.append((rows[b], start, count, have, len(new_pages)))
        new_pages += [pool.pop() for _ in range(max(0, need - have))]
    dev_master = torch.tensor(master, dtype=I32, device=cuda_device)
    got, err = _describe(cuda_device, dev_master, entries, new_pages + [0], ps, 40000, width)
    want = K4.describe(master, entries, new_pages, ps, width)
    assert err == 0
    T = want["q_start"][-1]
    for name in ("positions", "seq", "slots"):
        assert got[name].tolist() == want[name] + [-77] * 3
    for name in ("q_start", "ctx_lens", "tables", "decode_rows", "items"):
        assert got[name].tolist() == want[name], name
    assert dev_master.tolist() == master and T == sum(e[2] for e in entries)


@pytest.mark.parametrize("entry,new_pages", [((9, 0, 4, 0, 0), [1]),          # no such row
                                             ((1, 60, 10, 0, 0), [1] * 5),    # more places than a table has
                                             ((1, 0, 20, 0, 0), [1]),         # new pages that are not there
                                             ((1, 0, 20, 0, -1), [1, 2, 3]), ((1, -3, 4, 0, 0), [1]),
                                             ((1, 0, 4, -1, 0), [1]), ((1, 0, 4, 0, 0), [50]),
                                             ((1, 0, 4, 0, 0), [-2])])
def test_step_tables_flags_what_does_not_fit(cuda_device, entry, new_pages):
    master = torch.full((3, 4), 2, dtype=I32, device=cuda_device)
    good = (0, 3, 2, 1, 0)
    got, err = _describe(cuda_device, master, [good, entry, (2, 0, 1, 1, 0)], new_pages, 16, 10, 4)
    assert err == 4
    n = max(entry[2], 0)
    assert got["slots"][:2].tolist() == [35, 36] and got["slots"][2 + n].item() == 32
    assert (got["slots"][2:2 + n] == -1).all()
    assert got["tables"][0].tolist() == [2, 0, 0, 0] and got["tables"][2].tolist() == [2, 0, 0, 0]


@pytest.mark.parametrize("start", [2 ** 31 - 2, 2 ** 31 - 4, 2 ** 31 - 5])
def test_step_tables_flags_positions_past_31_bits(cuda_device, start):
    """Pages of one token, where the places needed are as many as the tokens."""
    master = torch.full((3, 4), 2, dtype=I32, device=cuda_device)
    got, err = _describe(cuda_device, master, [(0, 1, 2, 2, 0), (1, start, 4, 0, 0), (2, 0, 1, 1, 0)], [5], 1, 10, 4)
    assert err == 4 and got["slots"][:7].tolist() == [2, 5, -1, -1, -1, -1, 2]
    assert got["tables"].tolist() == [[2, 2, 5, 0], [0] * 4, [2, 0, 0, 0]]


def test_step_tables_with_less_room_than_tokens(cuda_device):
    master = torch.full((2, 4), 3, dtype=I32, device=cuda_device)
    got, err = _describe(cuda_device, master, [(0, 0, 3, 1, 0), (1, 0, 6, 1, 0)], [0], 16, 10, 4, T=5)
    assert err == 4 and got["positions"].tolist()[:3] == [0, 1, 2] and (got["positions"][5:] == -77).all()
    got, err = _describe(cuda_device, master, [(0, 0, 1, 1, 0), (1, 0, 1, 1, 0)], [0], 16, 10, 4, n_dec=1)
    assert err == 4 and got["decode_rows"].tolist() == [0]


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("window,keep", [(None, 0), (90, 3)])
def test_a_run_of_steps(cuda_device, window, keep):
    """Requests that come in portions and go on with single tokens, each step described, stored and
    attended on the device; every row against the attention over its request's tokens so far."""
    from binfer_b200.csrc import ops
    nh, nkv, d, ps, num_pages, width, slots = 8, 2, 128, 16, 200, 24, 6
    rng, dev = random.Random(4), cuda_device
    cache, err = ops.kv4_cache(num_pages, nkv, ps, d, dev), _err(dev)
    master = torch.zeros((slots, width), dtype=I32, device=dev)
    lens, have, row = [0] * 4, [0] * 4, [5, 0, 3, 2]
    total = [330, 47, 120, 16]
    ks = [_rows(n, nkv, d, dev, 10 + i) for i, n in enumerate(total)]
    vs = [_rows(n, nkv, d, dev, 20 + i) for i, n in enumerate(total)]
    pool = list(range(1, num_pages))
    rng.shuffle(pool)
    step = 0
    while any(l < t for l, t in zip(lens, total)):
        step += 1
        counts = []
        for b in range(4):
            left = total[b] - lens[b]
            counts.append(min(left, rng.choice([1, 1, 5, 64, 130]) if step > 1 else 30))
        counts[step % 4] = 0                              # one request sits out
        live = [b for b in range(4) if counts[b]]
        if not live:
            continue
        entries, new_pages = [], []
        for b in live:
            need = -(-(lens[b] + counts[b]) // ps)
            entries.append((row[b], lens[b], counts[b], have[b], len(new_pages)))
            new_pages += [pool.pop() for _ in range(need - have[b])]
            have[b] = max(have[b], need)
        o, flag = _describe(dev, master, entries, new_pages + [0], ps, num_pages, width)
        assert flag == 0
        T = sum(counts)
        k = torch.cat([ks[b][lens[b]:lens[b] + counts[b]] for b in live]).flatten(1)
        v = torch.cat([vs[b][lens[b]:lens[b] + counts[b]] for b in live]).flatten(1)
        ops.kv4_store(k, v, o["slots"][:T], cache, err)
        q = _queries(T, nh, d, dev, seed=step)
        out = torch.full_like(q, math.nan)
        tail = (o["tables"], out, nh, nkv, d, window, d ** -0.5, err)
        n_dec, n_pf = o["decode_rows"].numel(), o["items"].shape[0]
        if n_dec:
            ops.kv4_decode_attention(q, cache, o["decode_rows"], n_dec, o["seq"][:T], o["positions"][:T], *tail,
                                     keep_first=keep)
        if n_pf:
            many = [b for b in live if counts[b] > 1]
            ops.kv4_prefill_attention(q, cache, o["items"], n_pf, max(counts), *tail,
                                      ctx_rows=sum(-(-(lens[b] + counts[b]) // 64) * 64 for b in many),
                                      max_ctx=max(lens[b] + counts[b] for b in many), keep_first=keep)
        at = 0
        for b in live:
            n = lens[b] + counts[b]
            ref, allowed = K4.attend(q[at:at + counts[b]].view(-1, nh, d).to(F64), K4.held(ks[b][:n]),
                                     K4.held(vs[b][:n]), torch.arange(lens[b], n, device=dev), window, keep, d ** -0.5)
            _check(out[at:at + counts[b]].view(-1, nh, d), ref, allowed)
            at += counts[b]
            lens[b] = n
        assert int(err.item()) == 0


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("variant", ["stretches", "load"])
@pytest.mark.parametrize("nh,nkv,d,ps", [(8, 2, 128, 16), (4, 4, 64, 8), (6, 2, 256, 64), (17, 1, 128, 32)])
@pytest.mark.parametrize("window,keep", [(None, 0), (64, 0), (100, 11)])
def test_both_ways_of_a_portion(cuda_device, variant, nh, nkv, d, ps, window, keep):
    from binfer_b200.csrc import ops
    c = Cache([300, 70, 1], nkv, d, ps, cuda_device, seed=nh)
    jobs = [(1, 70, 0), (0, 33, 267), (2, 1, 0)]
    q = _queries(104, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    items = torch.tensor([(1, 0, 70, 0), (0, 70, 33, 267), (2, 103, 1, 0)], dtype=I32, device=cuda_device)
    ops.kv4_prefill_attention(q, c.cache, items, 3, 70, c.tables, out, nh, nkv, d, window, d ** -0.5, c.err,
                              ctx_rows=128 + 320 + 64, max_ctx=300, keep_first=keep, variant=variant)
    _compare(c, q, out, nh, jobs, window, keep, d ** -0.5)


def test_load_without_room_attends_what_fits(cuda_device):
    """``ctx_rows`` smaller than the contexts: the portions that have no room are flagged and left out."""
    from binfer_b200.csrc import ops
    nh, nkv, d = 4, 2, 128
    c = Cache([100, 200], nkv, d, 16, cuda_device)
    q = _queries(150, nh, d, cuda_device)
    out = torch.zeros_like(q)
    items = torch.tensor([(0, 0, 50, 50), (1, 50, 100, 100)], dtype=I32, device=cuda_device)
    ops.kv4_prefill_attention(q, c.cache, items, 2, 100, c.tables, out, nh, nkv, d, None, 0.1, c.err, ctx_rows=256,
                              max_ctx=200, variant="load")
    assert int(c.err.item()) == 16 and not out[50:].any()
    c.err.zero_()
    _compare(c, q[:50], out[:50], nh, [(0, 50, 50)], None, 0, 0.1)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("variant", ["stretches", "load"])
@pytest.mark.parametrize("item", [(-1, 40, 30, 20), (2, 40, 30, 20), (2 ** 31 - 1, 40, 30, 20), (1, -1, 30, 20),
                                  (1, 41, 30, 20), (1, 2 ** 31 - 1, 30, 20), (1, 40, 30, -10), (1, 40, 30, 2 ** 21),
                                  (1, 40, 30, 2 ** 31 - 10)])
def test_portions_that_are_not_there(cuda_device, variant, item):
    """A request, token rows or places outside of what the call is given: flagged, and the rows left as they were;
    the portion beside it is attended, one value that is not finite and all."""
    from binfer_b200.csrc import ops
    nh, nkv, d = 4, 2, 128
    c = Cache([140, 90], nkv, d, 16, cuda_device)
    c.v[0][120, 1, 3] = math.inf
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(70, nh, d, cuda_device)
    out = torch.full_like(q, 7.0)
    items = torch.tensor([(0, 0, 40, 100), item], dtype=I32, device=cuda_device)
    ops.kv4_prefill_attention(q, c.cache, items, 2, 40, c.tables, out, nh, nkv, d, None, 0.1, c.err, ctx_rows=384,
                              max_ctx=192, variant=variant)
    assert int(c.err.item()) == 4 and (out[40:] == 7).all()
    c.err.zero_()
    k, v = c.held(0)
    ref, allowed = K4.attend(q[:40].view(40, nh, d).to(F64), k, v.nan_to_num(), torch.arange(100, 140, device=q.device),
                             None, 0, 0.1)
    got, lost = out[:40].view(40, nh, d), torch.zeros_like(ref, dtype=torch.bool)
    lost[20:, nh // nkv:, :64] = True
    assert torch.isnan(got[lost]).all()
    _check(got[~lost], ref[~lost], allowed[~lost])


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("variant", ["stretches", "load"])
def test_a_window_of_any_size(cuda_device, variant):
    from binfer_b200.csrc import ops
    nh, nkv, d = 4, 2, 128
    c = Cache([140], nkv, d, 16, cuda_device)
    q = _queries(40, nh, d, cuda_device)
    items = torch.tensor([(0, 0, 40, 100)], dtype=I32, device=cuda_device)
    for window, keep in ((2 ** 31 - 1, 2 ** 31 - 1), (2 ** 40, 2 ** 40), (1, 2 ** 40)):
        out = torch.zeros_like(q)
        ops.kv4_prefill_attention(q, c.cache, items, 1, 40, c.tables, out, nh, nkv, d, window, 0.1, c.err,
                                  ctx_rows=192, max_ctx=140, keep_first=keep, variant=variant)
        _compare(c, q, out, nh, [(0, 40, 100)], None, 0, 0.1)


@pytest.mark.parametrize("what", ["queries", "keys", "both", "one key"])
@pytest.mark.parametrize("window,keep,d", [(None, 0, 128), (150, 4, 128), (None, 0, 64), (None, 0, 256), (150, 4, 256)])
def test_loaded_keys_and_queries_beyond_fp16(cuda_device, what, window, keep, d):
    """Numbers that fp16 has no room for, with a scale that makes ordinary scores of them."""
    from binfer_b200.csrc import ops
    nh, nkv, n, new = 6, 3, 400, 100
    c = Cache([n], nkv, d, 16, cuda_device, seed=9)
    q = _queries(new, nh, d, cuda_device)
    scale = d ** -0.5
    if what in ("queries", "both"):
        q, scale = (q.float() * 2.0 ** 17).to(BF16), scale * 2.0 ** -17
    if what in ("keys", "both"):
        c.k[0], scale = (c.k[0].float() * 2.0 ** 18).to(BF16), scale * 2.0 ** -18
    if what == "one key":
        c.k[0][350, 1, 7] = 70000.0
        q[:, nh // 3 * d + 7:2 * nh // 3 * d:d] = 2.0 ** -14
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    out = torch.full_like(q, math.nan)
    items = torch.tensor([(0, 0, new, n - new)], dtype=I32, device=cuda_device)
    ops.kv4_prefill_attention(q, c.cache, items, 1, new, c.tables, out, nh, nkv, d, window, scale, c.err,
                              ctx_rows=448, max_ctx=n, keep_first=keep, variant="load")
    _compare(c, q, out, nh, [(0, new, n - new)], window, keep, scale)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_loaded_portions_are_as_close_as_stretches(cuda_device, d):
    """Keys in fp16: what is left of the error is that of the probabilities, the values and the result
    in bfloat16, 1.7e-3 and twice 1.1e-3 of the result's rms (each half a step uniform, 2^-8 / sqrt(3) of a
    number's upper bound, 0.75 of it on average); 2.3e-3 together, where bfloat16 keys add 2.5e-3 or more."""
    from binfer_b200.csrc import ops
    nh, nkv, n = 8, 2, 600
    c = Cache([n], nkv, d, 16, cuda_device, seed=2)
    q = _queries(300, nh, d, cuda_device) * 1.5
    items = torch.tensor([(0, 0, 300, 300)], dtype=I32, device=cuda_device)
    k, v = c.held(0)
    ref, _ = K4.attend(q.view(300, nh, d).to(F64), k, v, torch.arange(300, 600, device=q.device), None, 0, d ** -0.5)
    for variant in ("stretches", "load"):
        out = torch.empty_like(q)
        ops.kv4_prefill_attention(q, c.cache, items, 1, 300, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                                  ctx_rows=640, max_ctx=n, variant=variant)
        off = (out.view(300, nh, d).to(F64) - ref).square().mean().sqrt() / ref.square().mean().sqrt()
        assert off <= 2.8e-3, (variant, float(off))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [600, 9000])
def test_loaded_portions_lose_little_but_the_result_s_rounding(cuda_device, d, n):
    """Queries, keys, values and probabilities in fp16 are off by 2^-11 / sqrt(3) each, 5e-4 together; the result's
    rounding to bfloat16 by 2^-8 / sqrt(3) of a number's upper bound, 1.7e-3 of its rms on average."""
    from binfer_b200.csrc import ops
    nh, nkv, new = 8, 2, 300
    c = Cache([n], nkv, d, 16, cuda_device, seed=2)
    q = _queries(new, nh, d, cuda_device) * 1.5
    items = torch.tensor([(0, 0, new, n - new)], dtype=I32, device=cuda_device)
    k, v = c.held(0)
    ref, _ = K4.attend(q.view(new, nh, d).to(F64), k, v, torch.arange(n - new, n, device=q.device), None, 0, d ** -0.5)
    out = torch.empty_like(q)
    ops.kv4_prefill_attention(q, c.cache, items, 1, new, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                              ctx_rows=-(-n // 64) * 64, max_ctx=n, variant="load")
    off = (out.view(new, nh, d).to(F64) - ref).square().mean().sqrt() / ref.square().mean().sqrt()
    assert off <= 2e-3, float(off)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** -20, 2.0 ** -16, 2.0 ** -8, 2.0 ** 8, 2.0 ** 11, 2.0 ** 30])
def test_loaded_values_of_any_size(cuda_device, d, size):
    """Values that fp16 has no room for, or few bits, among them; the first tokens' are ordinary."""
    from binfer_b200.csrc import ops
    nh, nkv, n, new = 4, 2, 300, 100
    c = Cache([n], nkv, d, 16, cuda_device, seed=4)
    c.v[0][40:] = (c.v[0][40:].float() * size).to(BF16)
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(new, nh, d, cuda_device)
    items = torch.tensor([(0, 0, new, n - new)], dtype=I32, device=cuda_device)
    for window in (None, 120):                  # (with it no row sees an ordinary value)
        out = torch.full_like(q, math.nan)
        ops.kv4_prefill_attention(q, c.cache, items, 1, new, c.tables, out, nh, nkv, d, window, 0.1, c.err,
                                  ctx_rows=320, max_ctx=n, variant="load")
        _compare(c, q, out, nh, [(0, new, n - new)], window, 0, 0.1)


@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 64), (6, 6, 128), (16, 1, 64), (8, 2, 256), (9, 3, 256)])
@pytest.mark.parametrize("window,keep", [(None, 0), (300, 0), (500, 70)])
def test_loaded_long_portions(cuda_device, nh, nkv, d, window, keep):
    """Several query blocks of 256 rows, tiles that end inside, values and keys of two portions."""
    from binfer_b200.csrc import ops
    c = Cache([1500, 700], nkv, d, 32, cuda_device, seed=d)
    q = _queries(1300, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    items = torch.tensor([(0, 0, 900, 600), (1, 900, 400, 300)], dtype=I32, device=cuda_device)
    ops.kv4_prefill_attention(q, c.cache, items, 2, 900, c.tables, out, nh, nkv, d, window, d ** -0.5, c.err,
                              ctx_rows=1536 + 704, max_ctx=1500, keep_first=keep, variant="load")
    _compare(c, q, out, nh, [(0, 900, 600), (1, 400, 300)], window, keep, d ** -0.5)


@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("window,keep", [(None, 0), (2500, 0), (2500, 70), (2100, 300), (4000, 3000)])
def test_loaded_portions_with_their_keys_shared_out(cuda_device, nh, nkv, d, window, keep):
    """Few blocks and some thousand keys each, the kept first tokens among them."""
    from binfer_b200.csrc import ops
    assert ops._kv4_splits(2, 300, 4500, window or 0, keep, nh, d, ops.num_sms(cuda_device))[2] > 1
    c = Cache([4500, 900], nkv, d, 32, cuda_device, seed=d)
    q = _queries(500, nh, d, cuda_device)
    out = torch.full_like(q, math.nan)
    items = torch.tensor([(0, 0, 300, 4200), (1, 300, 200, 700)], dtype=I32, device=cuda_device)
    ops.kv4_prefill_attention(q, c.cache, items, 2, 300, c.tables, out, nh, nkv, d, window, d ** -0.5, c.err,
                              ctx_rows=4544 + 960, max_ctx=4500, keep_first=keep, variant="load")
    _compare(c, q, out, nh, [(0, 300, 4200), (1, 200, 700)], window, keep, d ** -0.5)

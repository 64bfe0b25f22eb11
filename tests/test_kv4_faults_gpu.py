"""The operators of a cache in 4 bits where they were once wrong."""
import math
from fractions import Fraction

import pytest
import torch

import kv4_plain as K4
import kv4_units as U
from test_kv4_gpu import Cache, _err, _queries

pytestmark = pytest.mark.gpu

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32


# ------------------------------------------------------------------------------ portions without room
@pytest.fixture
def filled(monkeypatch):
    """Memory that a call takes is full of what it does not want: 77, and NaN."""
    real = torch.empty_strided

    def empty(*a, **kw):
        t = real(*a, **kw)
        return t.fill_(math.nan) if t.dtype == BF16 else t.fill_(77) if t.dtype == I32 else t
    monkeypatch.setattr(torch, "empty_strided", empty)


@pytest.mark.parametrize("d,ps,nkv", [(128, 16, 2), (64, 8, 1), (256, 128, 3)])
@pytest.mark.parametrize("lens,rows", [([128, 128], 128), ([100, 128], 192), ([128], 64), ([200, 60], 128),
                                       ([60, 200, 60], 192), ([64, 64, 64], 192)])
@pytest.mark.parametrize("places", [0, 9])
def test_load_of_portions_without_room(cuda_device, filled, d, ps, nkv, lens, rows, places):
    """A portion without room, or with room for a part of it: page 0 everywhere in its row of the tables, its error bit,
    no rows; the others whole, and zeros where no portion lies.  A portion that its row of the tables has no places for takes
    no room from those behind it."""
    from binfer_b200.csrc import ops
    width, fit, taken = places or rows // 64, [], 0
    for n in lens:
        own = -(-n // 64)
        taken += own if own <= width else 0
        fit.append(own <= width and taken <= rows // 64)
    c = Cache(lens, nkv, d, ps, cuda_device, seed=ps)
    n = len(lens)
    items = torch.tensor([(b, 2 * b, 2, lens[b] - 2) for b in range(n)], dtype=I32, device=cuda_device)
    moved = torch.full_like(items, 77)
    k, v, tables = ops.kv4_load(c.cache, c.tables, items, n, rows, c.err, items_out=moved, places=places)
    assert int(c.err.item()) == (0 if all(fit) else 16)
    assert moved.tolist() == [[b, 2 * b, 2 if fit[b] else 0, lens[b] - 2] for b in range(n)]
    page = 1
    for b in range(n):
        own = -(-lens[b] // 64)
        want = [page + i if fit[b] and i < own else 0 for i in range(width)]
        assert tables[b].tolist() == want, b
        if fit[b]:
            for x, h in ((k, c.held(b)[0]), (v, c.held(b)[1])):
                got = x[page:page + own].transpose(1, 2).reshape(-1, nkv, d).to(F64)
                assert ((got[:lens[b]] - h).abs() <= 1.001 * K4.HALF_STEP * h.abs()).all() and not got[lens[b]:].any()
            page += own
    for x in (k, v):
        assert not x[0].any() and not x[page:].any()


# ------------------------------------------------------------------------------ a portion beside others
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [100, 300])
def test_a_portion_s_bits_do_not_depend_on_the_rows_behind_it(cuda_device, d, rows):
    """The next request's queries, which the same tile of 128 rows reads: beyond fp16, infinite, not a number."""
    from binfer_b200.csrc import ops
    nh, nkv, n = 4, 2, 400
    c = Cache([n, 50], nkv, d, 16, cuda_device, seed=3)
    q = _queries(rows + 50, nh, d, cuda_device)
    items = torch.tensor([(0, 0, rows, n - rows), (1, rows, 50, 0)], dtype=I32, device=cuda_device)

    def run(q):
        out = torch.zeros_like(q)
        ops.kv4_prefill_attention(q, c.cache, items, 2, rows, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                                  ctx_rows=448 + 64, max_ctx=n, variant="load")
        return out[:rows]

    alone = run(q)
    for what in (2.0 ** 20, math.inf, math.nan):
        other = q.clone()
        other[rows:] = what
        assert torch.equal(run(other), alone), what
    assert int(c.err.item()) == 0


# ------------------------------------------------------------------------------ numbers that fp16 has few bits for
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("variant", ["load", "auto", "stretches"])
@pytest.mark.parametrize("key_size,query_size", [(-30, 0), (0, -30), (-20, 0), (0, -18), (-16, -16), (-20, -20), (12, -40),
                                                 (-40, 12)])
def test_small_keys_and_queries_with_a_large_scale(cuda_device, d, variant, key_size, query_size):
    """Numbers below fp16's, whose scores a scale makes ordinary."""
    from binfer_b200.csrc import ops
    nh, nkv, n, new = 6, 3, 400, 100
    c = Cache([n], nkv, d, 16, cuda_device, seed=9)
    c.k[0] = U.keys(n, nkv, d, cuda_device, 1) * 2.0 ** key_size
    c.v[0] = U.values(n, nkv, d, cuda_device, 2)
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(new, nh, d, cuda_device) * 2.0 ** query_size
    scale = d ** -0.5 * 2.0 ** -(key_size + query_size)
    items = torch.tensor([(0, 0, new, n - new)], dtype=I32, device=cuda_device)
    out = torch.full_like(q, math.nan)
    ops.kv4_prefill_attention(q, c.cache, items, 1, new, c.tables, out, nh, nkv, d, None, scale, c.err, ctx_rows=448,
                              max_ctx=n, variant=variant)
    k, v = c.held(0)
    ref, allowed = U.attend(q.view(new, nh, d).to(F64), k, v, torch.arange(n - new, n, device=q.device), None, 0, scale)
    U.check(out, ref, allowed)
    assert int(c.err.item()) == 0


@pytest.mark.parametrize("what", ["a row of queries", "a key", "a group of keys"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_some_small_keys_and_queries_with_a_large_scale(cuda_device, what, d):
    """A few small numbers among ordinary ones; zeros, which fp16 has, beside them."""
    from binfer_b200.csrc import ops
    nh, nkv, n, new, scale = 4, 2, 300, 140, 64.0
    c = Cache([n], nkv, d, 16, cuda_device, seed=9)
    k, q = U.keys(n, nkv, d, cuda_device, 1) * d ** -0.5 / 64, _queries(new, nh, d, cuda_device)
    c.v[0] = U.values(n, nkv, d, cuda_device, 2)
    k[::7] = 0
    q[5] = 0
    if what == "a row of queries":                      # (the keys that it meets are as much larger)
        q, k = q * 2.0 ** -10, k * 2.0 ** 10
        q[133, d:2 * d] *= 2.0 ** -9
    elif what == "a key":
        k[201, 1] *= 2.0 ** -11
        q = q * 2.0 ** 5
    else:
        k[:, 1, -64:] *= 2.0 ** -14
        q.view(new, nh, d)[:, 2:, -64:] *= 2.0 ** 14
    c.k[0] = k
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    items = torch.tensor([(0, 0, new, n - new)], dtype=I32, device=cuda_device)
    kk, v = c.held(0)
    ref, allowed = U.attend(q.view(new, nh, d).to(F64), kk, v, torch.arange(n - new, n, device=q.device), None, 0, scale)
    out = torch.full_like(q, math.nan)
    ops.kv4_prefill_attention(q, c.cache, items, 1, new, c.tables, out, nh, nkv, d, None, scale, c.err, ctx_rows=320,
                              max_ctx=n, variant="load")
    U.check(out, ref, allowed)
    assert int(c.err.item()) == 0


# ------------------------------------------------------------------------------ codes
def _border_rows():
    """Groups whose lowest number is a whole number and a half of steps, with numbers beside zero that no float holds
    beside it, so that the quotient is next to a border; and lowest numbers beside zero with numbers on a border."""
    rows = torch.zeros((12, 64), dtype=F64)
    for r, (low, step) in enumerate([(-3.0, 2.0), (-1.0, 2.0), (-5.0, 2.0), (-0.75, 0.5), (-3.0 * 2.0 ** 40, 2.0 ** 41),
                                     (-3.0 * 2.0 ** -60, 2.0 ** -59)]):
        rows[r, 0], rows[r, 1] = low, low + 15 * step
        tiny = abs(low) * 2.0 ** -torch.arange(20.0, 50.0, dtype=F64)
        rows[r, 2:32], rows[r, 32:62] = tiny, -tiny
    for r, (low, step) in enumerate([(-2.0 ** -40, 2.0), (2.0 ** -40, 2.0), (-2.0 ** -60, 0.25), (2.0 ** -60, 0.25),
                                     (-1e-36, 1e-3), (-2.0 ** 60, 2.0 ** 124)], 6):
        rows[r] = step * (torch.arange(64, dtype=F64) % 15 + 0.5)
        rows[r, 0], rows[r, 1] = low, 15 * step
    return rows.to(torch.float32).to(BF16)


def _held_exactly(x):
    """``K4.held`` with quotients as fractions: 64 bits do not hold 0.125 + 2^-60 either."""
    out = torch.empty(x.shape, dtype=F64)
    for r, row in enumerate(x.cpu().to(F64).unflatten(-1, (-1, 64)).flatten(0, -2)):
        low, high = row.min(), row.max()
        s = ((high - low) / 15).to(BF16).to(F64)
        codes = [min(15, round((Fraction(float(n)) - Fraction(float(low))) / Fraction(float(s)))) for n in row]
        out.view(-1, 64)[r] = low + s * torch.tensor(codes, dtype=F64)
    return out


def test_codes_next_to_a_border(cuda_device):
    from binfer_b200.csrc import ops
    x = _border_rows().to(cuda_device)
    T = x.shape[0]
    c, err = ops.kv4_cache(3, 1, 8, 64, cuda_device), _err(cuda_device)
    ops.kv4_store(x, x.flip(0).contiguous(), torch.arange(8, 8 + T, dtype=I32, device=cuda_device), c, err)
    k, v = K4.unpack(c)
    want = _held_exactly(x)
    assert torch.equal(k.reshape(-1, 64)[8:8 + T], want) and torch.equal(v.reshape(-1, 64)[8:8 + T], want.flip(0))


@pytest.mark.parametrize("d", [64, 128])
def test_codes_next_to_a_border_behind_norms_and_rotation(cuda_device, d):
    """The kernel of a model's layers, heads of 128 by a kernel of their own: the same codes."""
    from binfer_b200.csrc import ops
    rows = _border_rows()
    if d == 128:
        rows = torch.cat([rows, rows.flip(0)], 1)
    x = rows.to(cuda_device)
    T = x.shape[0]
    qkv = torch.cat([x, x, x], 1)
    freq = torch.zeros(d // 2, dtype=torch.float32, device=cuda_device)
    want, got = ops.kv4_cache(3, 1, 8, d, cuda_device), ops.kv4_cache(3, 1, 8, d, cuda_device)
    slots, err = torch.arange(8, 8 + T, dtype=I32, device=cuda_device), _err(cuda_device)
    ops.kv4_store(x, x, slots, want, err)
    ops.qk_norm_rope_kv4_store(qkv, None, None, freq, torch.zeros(T, dtype=I32, device=cuda_device), slots,
                               torch.empty_like(x), got, 1, 1, d, 1e-6, err)
    assert torch.equal(got, want)
    assert torch.equal(K4.unpack(got)[0].reshape(-1, d)[8:8 + T], _held_exactly(x))


# ------------------------------------------------------------------------------ what fp16 has no room for
@pytest.mark.parametrize("nh,nkv,d,ps", [(8, 2, 128, 16), (16, 1, 128, 8), (6, 3, 64, 32), (20, 1, 64, 16), (4, 4, 64, 8),
                                         (4, 1, 256, 128), (18, 2, 256, 16), (3, 3, 128, 64)])
@pytest.mark.parametrize("window,keep", [(None, 0), (120, 9), (900, 70)])
@pytest.mark.parametrize("jobs", [[(0, 2, 698)], [(2, 7, 0), (0, 5, 400), (1, 1, 3), (3, 3, 997)],
                                  [(0, 700, 0), (3, 300, 700)], [(4, 40, 4200), (1, 33, 0)]])
def test_portions_that_are_computed_from_the_codes(cuda_device, nh, nkv, d, ps, window, keep, jobs):
    """Keys beyond fp16 in every kv head but the second, whose bits are what they are beside ordinary ones."""
    from binfer_b200.csrc import ops
    c = Cache([700, 33, 7, 1000, 4240], nkv, d, ps, cuda_device, seed=d + ps)
    T, scale = sum(n for _, n, _ in jobs), d ** -0.5
    q = _queries(T, nh, d, cuda_device)
    items, at = [], 0
    for b, n, p in jobs:
        items.append((b, at, n, p))
        at += n
    for i, n in enumerate(c.lens):
        c.k[i], c.v[i] = U.keys(n, nkv, d, cuda_device, 2 * i), U.values(n, nkv, d, cuda_device, 2 * i + 1)

    def run():
        for i in range(len(c.lens)):
            ops.kv4_store(c.k[i].flatten(1), c.v[i].flatten(1), c.slots[i], c.cache, c.err)
        out = torch.full_like(q, math.nan)
        ops.kv4_prefill_attention(q, c.cache, torch.tensor(items, dtype=I32, device=cuda_device), len(items),
                                  max(n for _, n, _ in jobs), c.tables, out, nh, nkv, d, window, scale, c.err,
                                  ctx_rows=sum(-(-(n + p) // 64) * 64 for _, n, p in jobs),
                                  max_ctx=max(n + p for _, n, p in jobs), keep_first=keep, variant="load")
        assert int(c.err.item()) == 0
        return out

    ordinary = run()
    up = torch.full((nkv, 1), 2.0 ** 18, device=cuda_device)
    if nkv > 1:
        up[1] = 1
    q = (q.view(T, nkv, -1, d) / up[:, None]).to(BF16).view(T, -1)
    for i in range(len(c.lens)):
        c.k[i] = (c.k[i] * up).to(BF16)
    out = run()
    at = 0
    for b, n, p in jobs:
        k, v = c.held(b)
        ref, allowed = U.attend(q[at:at + n].view(n, nh, d).to(F64), k[:n + p], v[:n + p],
                                torch.arange(p, p + n, device=q.device), window, keep, scale)
        U.check(out[at:at + n], ref, allowed)
        at += n
    if nkv > 1:
        other = slice(nh // nkv * d, 2 * nh // nkv * d)
        assert torch.equal(out[:, other], ordinary[:, other])


@pytest.mark.parametrize("rows,ctx,nh,nkv,d", [(256, 4096, 16, 4, 128), (1024, 1024, 8, 2, 64), (300, 2000, 8, 2, 256)])
def test_a_value_beyond_fp16_costs_little_more_than_reading_the_codes(cuda_device, rows, ctx, nh, nkv, d):
    """One value in one token of each head; the kernel that reads the codes of every head takes the same way.  (It was a
    walk over the keys, one after the other, of some hundred times that.)"""
    from binfer_b200.csrc import ops
    c = Cache([ctx], nkv, d, 16, cuda_device)
    c.v[0][ctx // 2, :, 5] = 5000.0
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(rows, nh, d, cuda_device)
    out = torch.empty_like(q)
    items = torch.tensor([(0, 0, rows, ctx - rows)], dtype=I32, device=cuda_device)

    def time(variant):
        took = []
        for _ in range(7):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.kv4_prefill_attention(q, c.cache, items, 1, rows, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                                      ctx_rows=-(-ctx // 64) * 64, max_ctx=ctx, variant=variant)
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b))
        return min(took)

    assert time("load") <= 10 * time("stretches")


# ------------------------------------------------------------------------------ scratch
def test_portions_with_room_for_more_than_is_kept_free_are_not_loaded(cuda_device):
    """``ctx_rows`` of 2^30 tokens, 4 TiB loaded: the choice reads the codes instead."""
    from binfer_b200.csrc import ops
    nh, nkv, d, n, rows = 32, 8, 128, 2000, 600
    c = Cache([n], nkv, d, 16, cuda_device)
    c.k[0], c.v[0] = U.keys(n, nkv, d, cuda_device, 1), U.values(n, nkv, d, cuda_device, 2)
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(rows, nh, d, cuda_device)
    items = torch.tensor([(0, 0, rows, n - rows)], dtype=I32, device=cuda_device)
    assert ops._kv4_load_pays(1, rows, n, 0, 0, nh, nkv, d)
    out = torch.full_like(q, math.nan)
    ops.kv4_prefill_attention(q, c.cache, items, 1, rows, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                              ctx_rows=1 << 30, max_ctx=n)
    ref, allowed = U.attend(q.view(rows, nh, d).to(F64), *c.held(0), torch.arange(n - rows, n, device=q.device), None, 0,
                            d ** -0.5)
    U.check(out, ref, allowed)
    assert int(c.err.item()) == 0


def test_loaded_portions_in_a_graph_with_other_items_and_numbers(cuda_device):
    """A captured call replayed with other portions, with and without numbers beyond fp16, with more context than its room,
    beside another graph of the same call."""
    import gc
    from binfer_b200.csrc import ops
    nh, nkv, d, lens = 8, 2, 128, [900, 500]
    c = Cache(lens, nkv, d, 16, cuda_device)
    q = _queries(300, nh, d, cuda_device)
    items = torch.tensor([(0, 0, 200, 100), (1, 200, 100, 100)], dtype=I32, device=cuda_device)

    def call(out):
        ops.kv4_prefill_attention(q, c.cache, items, 2, 200, c.tables, out, nh, nkv, d, None, d ** -0.5, c.err,
                                  ctx_rows=960 + 512, max_ctx=900, variant="load")

    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    for o in outs:
        call(o)
        torch.cuda.synchronize()
        gc.collect()                          # (not in the middle of the capture)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(o)
        graphs.append(g)
    for jobs, large in (([(0, 0, 200, 700), (1, 200, 100, 400)], 0), ([(1, 0, 100, 400), (0, 100, 200, 700)], 2.0 ** 18),
                        ([(0, 0, 150, 0), (1, 150, 1, 499)], 0), ([(0, 0, 200, 700), (1, 200, 100, 399)], 2.0 ** 18),
                        ([(0, 0, 200, 700), (0, 200, 100, 800)], 0)):
        for i, n in enumerate(lens):
            c.k[i], c.v[i] = U.keys(n, nkv, d, cuda_device, i), U.values(n, nkv, d, cuda_device, 5 + i)
            if large:                        # (in one token of one head)
                c.k[i][17, 1], c.v[i][17, 1] = 0, 0
                c.v[i][17, 1, 0] = large
            ops.kv4_store(c.k[i].flatten(1), c.v[i].flatten(1), c.slots[i], c.cache, c.err)
        items.copy_(torch.tensor(jobs, dtype=I32))
        c.err.zero_()
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
        torch.cuda.synchronize()
        fits = sum(-(-(n + p) // 64) * 64 for _, _, n, p in jobs) <= 960 + 512
        assert int(c.err.item()) == (0 if fits else 16) and torch.equal(outs[0], outs[1])
        for i, (b, at, n, p) in enumerate(jobs):
            if not fits and i:
                assert not outs[0][at:at + n].any()
                continue
            k, v = c.held(b)
            ref, allowed = U.attend(q[at:at + n].view(n, nh, d).to(F64), k[:n + p], v[:n + p],
                                    torch.arange(p, p + n, device=q.device), None, 0, d ** -0.5)
            if large:                        # the numbers that the large one reaches are as far off as it is large
                ref, got = ref.view(n, nh, d).clone(), outs[0][at:at + n].view(n, nh, d).clone()
                ref[:, nh // 2:, :64] = got[:, nh // 2:, :64] = 0
                U.check(got, ref, allowed)
            else:
                U.check(outs[0][at:at + n], ref, allowed)

"""The operators of a paged cache held in 4 bits, as cases that can be timed and compared.

Keys and values lie in pages ``uint8 [pages, kv_heads, page_size / 8, 9 d]``.  Every 64 numbers of a
key or value row share a scale s and a lowest value m (bfloat16); a number is m + s c with a code c of
0 to 15.  The 9 d bytes of eight tokens are the keys' codes, the values' codes, the keys' (s, m) and
the values' (s, m); ``_key_places`` and ``_value_places`` say which byte and half a code lies in.

Kinds of pass:

* ``store``: a step's keys and values into the pages, then the whole contexts out of them as
  bfloat16 pages of 64 tokens (what a prompt portion does);
* ``decode``: attention of rows that bring one token each over the pages;
* ``prefill``: causal attention of prompt portions over the pages;
* ``tables``: what a step's kernels need to know of its batch (positions, places, block tables),
  from the requests' lengths and the pages they were given.

``own`` False computes a pass in plain torch, True through the package's entry points.
"""
import math
import zlib

import torch

own = False

DEVICE = "cuda:0"
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
GROUP = 64
LOAD_PAGE = 64


# --------------------------------------------------------------------------------- cases
def _case(name, kind, **kw):
    c = dict(name=name, kind=kind, heads=32, kv_heads=8, dim=128, page=16, requests=1, tokens=1,
             context=0, window=0, keep=0)
    c.update(kw)
    return c


def listed():
    """``requests`` requests bring up to ``tokens`` tokens each behind up to ``context`` cached ones."""
    return [
        # the first tokens of a chat: nothing but latency
        _case("store_small", "store", tokens=13, context=40),
        # a prompt's second portion: its keys and values in, its whole context out
        _case("store_prompt", "store", tokens=2048, context=2048),
        # portions of several users at odd lengths, heads of 64
        _case("store_portions", "store", heads=16, dim=64, requests=5, tokens=333, context=1500,
              page=32),
        # one user's decode step in a short conversation
        _case("decode_one", "decode", context=519),
        # eight requests with 4k tokens of context each
        _case("decode_eight", "decode", requests=8, context=4096),
        # a full batch of a model with 64 heads, contexts up to 4k
        _case("decode_many", "decode", heads=64, requests=64, context=4096),
        # long documents behind a window that keeps the first tokens visible
        _case("decode_window", "decode", heads=16, requests=12, context=30000, window=4096, keep=4,
              page=64),
        # a prompt from its first token on
        _case("prefill_prompt", "prefill", tokens=2048),
        # a portion of a long prompt
        _case("prefill_portion", "prefill", tokens=256, context=8192),
        # a few drafted tokens per request to be checked at once
        _case("prefill_drafts", "prefill", heads=16, requests=6, tokens=5, context=3000),
        # a serving step's description: two prompt portions beside thirty decoded tokens
        _case("tables_step", "tables", requests=32, tokens=1013, context=900),
        # a captured decode step's description: many requests, tables wide enough for 32k tokens
        _case("tables_decode", "tables", requests=256, context=32000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Heads of 64, 128 and 256 in groups of 1 to 16, pages of 8 to 128 tokens; stores of 1 to 2,048
    tokens a request behind up to 8,192; single tokens of 1 to 64 requests behind 1 to 32,000 tokens
    (at most 250,000 in all); portions of 2 to 2,048 tokens behind up to 8,192; descriptions of 1 to
    256 requests."""
    kind = rng.choice(["store", "decode", "decode", "prefill", "prefill", "tables"])
    heads, kv, d = rng.choice([(16, 8, 128), (32, 8, 128), (64, 8, 128), (20, 4, 128), (6, 6, 128),
                               (16, 1, 128), (16, 4, 64), (12, 2, 64), (8, 2, 256), (9, 3, 256)])
    c = dict(kind=kind, heads=heads, kv_heads=kv, dim=d, page=rng.choice([8, 16, 16, 32, 64, 128]),
             requests=1, tokens=1, context=0, window=0, keep=0)
    if kind == "tables":
        c["requests"] = _log(rng, 1, 256)
        c["context"] = _log(rng, 1, 32000)
        if c["requests"] <= 40 and rng.random() < 0.6:
            c["tokens"] = _log(rng, 2, 2048)
        return c
    if kind == "decode":
        c["requests"] = _log(rng, 1, 64)
        c["context"] = _log(rng, 1, min(32000, 250000 // c["requests"]))
    else:
        c["requests"] = rng.choice([1, 1, 2, 3, 5])
        c["tokens"] = _log(rng, 2 if kind == "prefill" else 1, 2048 // c["requests"])
        c["context"] = rng.choice([0, _log(rng, 1, 8192 // c["requests"])])
    if kind != "store" and rng.random() < 0.3:
        c["window"] = _log(rng, 16, 4096)
        c["keep"] = rng.choice([0, 1, 4, 70])
    return c


def _requests(c):
    """(cached tokens, tokens of this step) of every request: contexts and portions get shorter from
    one request to the next; of a described step two requests bring portions, the others one token."""
    n, out = c["requests"], []
    for i in range(n):
        if c["kind"] == "tables":
            new = c["tokens"] * (8 - 3 * i) // 8 if i < 2 else 1
        else:
            new = c["tokens"] * (2 * n - i) // (2 * n)
        out.append((c["context"] * (3 * n - i) // (3 * n), max(1, new)))
    return out


def _generator(seed, name):
    g = torch.Generator(DEVICE)
    g.manual_seed((int(seed) * 1_000_003 + zlib.crc32(name.encode())) & 0x7FFF_FFFF_FFFF)
    return g


# --------------------------------------------------------------- the pages' layout, in plain torch
def _key_places(d, device):
    """Of every number of a key row: its code's byte in the row's d / 2, and the shift in that byte."""
    i = torch.arange(d, device=device)
    e = i % GROUP
    return e // 16 * (d // 8) + i // GROUP * 8 + e % 16 // 2, e % 2 * 4


def _value_places(d, device):
    """Of every number of a value row: its code's byte among the eight tokens' (the token's own share
    of a part is d / 16 bytes further for each token), and the shift in that byte."""
    i = torch.arange(d, device=device)
    e = i % GROUP
    return e // 8 * (d // 2) + i // GROUP * 4 + e % 8 // 2, e % 2 * 4


def _codes(x):
    """Codes (uint8), scales and lowest values (bfloat16) of rows ``x [..., d]`` (bfloat16)."""
    g = x.float().unflatten(-1, (-1, GROUP)) * 0.25             # (no difference overflows)
    low, high = g.amin(-1), g.amax(-1)
    s = ((high - low) / 3.75).to(BF16)
    c = torch.round((g - low[..., None]) / (s.float() * 0.25)[..., None])
    c = torch.where(s[..., None] > 0, c, torch.zeros_like(c)).clamp_(0, 15)
    return c.to(torch.uint8).flatten(-2), s, (low * 4).to(BF16)


def _store(cache, slots, k, v):
    """Rows ``k``, ``v`` ``[T, kv_heads, d]`` into the pages at ``slots [T]``."""
    pages, nkv, eighths, rec = cache.shape
    d = k.shape[-1]
    flat = cache.view(-1)
    head = torch.arange(nkv, device=cache.device)
    slot = slots.long()
    page, off = slot // (eighths * 8), slot % (eighths * 8)
    base = ((page[:, None] * nkv + head) * eighths + (off // 8)[:, None]) * rec       # [T, nkv]
    tok = (off % 8)[:, None]
    for x, at in ((k, 0), (v, 1)):
        c, s, low = _codes(x)
        if at == 0:
            place, _ = _key_places(d, cache.device)
            where = base + tok * (d // 2)
        else:
            place, _ = _value_places(d, cache.device)
            where = base + 4 * d + tok * (d // 16)
        byte = c[..., 0::2] | (c[..., 1::2] << 4)               # neighbours share a byte
        flat[where[..., None] + place[0::2]] = byte
        par = torch.stack([s, low], -1).contiguous().view(torch.uint8).flatten(-2)    # [T, nkv, d / 16]
        where = base + 8 * d + at * (d // 2) + tok * (d // 16)
        flat[where[..., None] + torch.arange(d // 16, device=cache.device)] = par


def _read(cache, table, n):
    """The keys and values of a request's first ``n`` tokens, float32 ``[n, kv_heads, d]`` each."""
    nkv, eighths, rec = cache.shape[1:]
    d = rec // 9
    pages = -(-n // (eighths * 8))
    b = cache[table[:pages].long()].permute(0, 2, 1, 3).reshape(pages * eighths, nkv, rec)
    out = []
    for at, places in ((0, _key_places), (1, _value_places)):
        place, shift = places(d, cache.device)
        tok = torch.arange(8, device=cache.device)[:, None]
        where = 4 * d * at + tok * (d // 16 if at else d // 2) + place                # [8, d]
        c = (b[:, :, where.flatten()].view(-1, nkv, 8, d) >> shift.to(torch.uint8)) & 15
        at_par = 8 * d + at * (d // 2)
        par = b[:, :, at_par:at_par + d // 2].contiguous().view(BF16).view(-1, nkv, 8, d // GROUP, 2)
        par = par.float()
        x = c.float().unflatten(-1, (-1, GROUP)) * par[..., :1] + par[..., 1:]
        out.append(x.flatten(-2).permute(0, 2, 1, 3).reshape(-1, nkv, d)[:n])
    return out


# --------------------------------------------------------------------------------- prepare
def _rows(c, seed, name, n):
    """Keys: channels of different size and mean, as norms and rotations leave them; values."""
    g = _generator(seed, name)
    k = torch.randn((n, c["kv_heads"], c["dim"]), generator=g, device=DEVICE)
    v = torch.randn((n, c["kv_heads"], c["dim"]), generator=g, device=DEVICE)
    h = _generator(seed, "channels")
    size = torch.randn((c["kv_heads"], c["dim"]), generator=h, device=DEVICE).mul_(0.4).exp_()
    mean = torch.randn((c["kv_heads"], c["dim"]), generator=h, device=DEVICE).mul_(0.5)
    return (k * size + mean).to(BF16), v.to(BF16)


def prepare(case, seed):
    c, reqs = case, _requests(case)
    ps, nkv, d = c["page"], c["kv_heads"], c["dim"]
    B, T = len(reqs), sum(n for _, n in reqs)
    held = [-(-(b + n) // ps) for b, n in reqs]
    pages = 1 + sum(held)
    # pages of a request mostly follow one another, in runs that lie anywhere in the pool
    g = _generator(seed, "pages")
    run = max(1, 128 // ps)
    starts = [s for s in range(1, pages, run)]
    order = torch.randperm(len(starts), generator=g, device=DEVICE).tolist()
    ids = [p for i in order for p in range(starts[i], min(pages, starts[i] + run))]
    own_pages, at = [], 0
    for n in held:
        own_pages.append(ids[at:at + n])
        at += n
    if c["kind"] == "tables":
        return _prepare_tables(c, reqs, held, own_pages, pages)
    tables = torch.zeros((B, max(held)), dtype=torch.int32)
    for i, p in enumerate(own_pages):
        tables[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    tables = tables.to(DEVICE)
    cache = torch.zeros((pages, nkv, ps // 8, 9 * d), dtype=torch.uint8, device=DEVICE)
    slots, ks, vs = [], [], []
    for i, (before, new) in enumerate(reqs):
        k, v = _rows(c, seed, "request %d" % i, before + new)
        p = torch.arange(before + new, device=DEVICE)
        slot = (tables[i][p // ps] * ps + p % ps).int()
        stored = before if c["kind"] == "store" else before + new
        for a in range(0, stored, 8192):
            e = min(stored, a + 8192)
            _store(cache, slot[a:e], k[a:e], v[a:e])
        slots.append(slot[before:])
        ks.append(k[before:])
        vs.append(v[before:])
    first = [sum(n for _, n in reqs[:i]) for i in range(B)]
    items = torch.tensor([(i, first[i], n, b) for i, (b, n) in enumerate(reqs)], dtype=torch.int32)
    s = dict(case=c, cache=cache, tables=tables, items=items.to(DEVICE), max_rows=max(n for _, n in reqs),
             ctx_rows=sum(-(-(b + n) // LOAD_PAGE) * LOAD_PAGE for b, n in reqs),
             max_ctx=max(b + n for b, n in reqs), reqs=reqs, first=first,
             err=torch.zeros(1, dtype=torch.int32, device=DEVICE))
    if c["kind"] == "store":
        # as the products leave them: a token's keys and values side by side behind its queries
        qkv = torch.zeros((T, (c["heads"] + 2 * nkv) * d), dtype=BF16, device=DEVICE)
        qkv[:, -2 * nkv * d:-nkv * d] = torch.cat(ks).flatten(1)
        qkv[:, -nkv * d:] = torch.cat(vs).flatten(1)
        return dict(s, slots=torch.cat(slots), k=qkv[:, -2 * nkv * d:-nkv * d], v=qkv[:, -nkv * d:])
    q = torch.randn((T, c["heads"] * d), generator=_generator(seed, "queries"), device=DEVICE)
    s["q"] = q.mul_(1.3).to(BF16)
    s["out"] = torch.empty_like(s["q"])
    s["positions"] = torch.cat([torch.arange(b, b + n) for b, n in reqs]).int().to(DEVICE)
    s["seq"] = torch.cat([torch.full((n,), i) for i, (_, n) in enumerate(reqs)]).int().to(DEVICE)
    return s


def _prepare_tables(c, reqs, held, own_pages, pages):
    """The requests' pages of earlier steps lie in ``master`` (a row per request that the server may
    hold); a step brings each request's row, lengths, pages held so far and its newly given pages."""
    ps, B, T = c["page"], len(reqs), sum(n for _, n in reqs)
    width = max(held) + 3
    master = torch.zeros((B + 5, width), dtype=torch.int32)
    entries, new_pages = [], []
    for i, (before, new) in enumerate(reqs):
        row, have = (i * 7 + 3) % (B + 5) if math.gcd(7, B + 5) == 1 else i + 2, -(-before // ps)
        master[row, :have] = torch.tensor(own_pages[i][:have], dtype=torch.int32)
        entries.append((row, before, new, have, len(new_pages)))
        new_pages += own_pages[i][have:]
    n_dec = sum(n == 1 for _, n in reqs)
    empty = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEVICE)
    return dict(case=c, master=master.to(DEVICE), width=width, pages=pages, T=T, n_dec=n_dec,
                entries=torch.tensor(entries, dtype=torch.int32).to(DEVICE),
                new_pages=torch.tensor(new_pages + [0], dtype=torch.int32).to(DEVICE),
                q_start=empty(B + 1), positions=empty(T), seq=empty(T), ctx_lens=empty(B),
                slots=empty(T), tables=empty(B, width), decode_rows=empty(n_dec),
                portions=empty(B - n_dec, 4), err=empty(1))


# ------------------------------------------------------------------------------------- run
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from binfer_b200.csrc import ops
    c = s["case"]
    if c["kind"] == "tables":
        ops.step_tables(s["master"], s["entries"], s["new_pages"], c["page"], s["pages"], s["q_start"],
                        s["positions"], s["seq"], s["ctx_lens"], s["slots"], s["tables"], s["err"],
                        decode_rows=s["decode_rows"], prefill_items=s["portions"])
        return [s[n] for n in ("q_start", "positions", "seq", "ctx_lens", "slots", "tables",
                               "decode_rows", "portions", "master")]
    if c["kind"] == "store":
        ops.kv4_store(s["k"], s["v"], s["slots"], s["cache"], s["err"])
        return ops.kv4_load(s["cache"], s["tables"], s["items"], len(s["reqs"]), s["ctx_rows"], s["err"])
    common = (s["tables"], s["out"], c["heads"], c["kv_heads"], c["dim"], c["window"] or None,
              c["dim"] ** -0.5, s["err"])
    if c["kind"] == "decode":
        ops.kv4_decode_attention(s["q"], s["cache"], None, len(s["reqs"]), s["seq"], s["positions"],
                                 *common, keep_first=c["keep"])
    else:
        ops.kv4_prefill_attention(s["q"], s["cache"], s["items"], len(s["reqs"]), s["max_rows"],
                                  *common, ctx_rows=s["ctx_rows"], max_ctx=s["max_ctx"],
                                  keep_first=c["keep"])
    return s["out"]


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "tables":
        return _plain_tables(s)
    if c["kind"] == "store":
        T = s["k"].shape[0]
        shape = (T, c["kv_heads"], c["dim"])
        _store(s["cache"], s["slots"], s["k"].reshape(shape), s["v"].reshape(shape))
        contexts = [_read(s["cache"], s["tables"][i], b + n) for i, (b, n) in enumerate(s["reqs"])]
        return _as_pages(s["reqs"], contexts, BF16)
    out = s["out"]
    for i, (before, new) in enumerate(s["reqs"]):
        k, v = _read(s["cache"], s["tables"][i], before + new)
        a = s["first"][i]
        out[a:a + new] = _attend(c, s["q"][a:a + new].float(), k, v, before).to(BF16)
    return out


def _as_pages(reqs, contexts, dtype):
    """Contexts ``(k, v)`` one behind the other in pages of 64 tokens, page 0 zero; and the pages of
    each request."""
    each = [-(-(b + n) // LOAD_PAGE) for b, n in reqs]
    total = 1 + sum(each)
    nkv, d = contexts[0][0].shape[1:]
    out = []
    for at in (0, 1):
        x = torch.zeros((total * LOAD_PAGE, nkv, d), dtype=dtype, device=DEVICE)
        row = LOAD_PAGE
        for n, kv in zip(each, contexts):
            x[row:row + kv[at].shape[0]] = kv[at].to(dtype)
            row += n * LOAD_PAGE
        out.append(x.view(total, LOAD_PAGE, nkv, d).transpose(1, 2).contiguous())
    w = torch.arange(sum(each), device=DEVICE)
    base = [1 + sum(each[:i]) for i in range(len(each))]
    tables = torch.stack([torch.where(w < n, w + b, torch.zeros_like(w)) for n, b in zip(each, base)])
    return out[0], out[1], tables.int()


def _attend(c, q, k, v, before):
    """softmax(q k / sqrt(d)) v of rows at positions ``before ..``; head h reads kv head h // group."""
    new, d, group = q.shape[0], c["dim"], c["heads"] // c["kv_heads"]
    q = q.view(new, c["kv_heads"], group, d)
    p = torch.arange(before, before + new, device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)
    seen = j <= p
    if c["window"]:
        seen &= (j > p - c["window"]) | (j < c["keep"])
    outs = []
    for g in range(c["kv_heads"]):                       # a kv head at a time: the scores fit
        score = torch.einsum("tgd,jd->gtj", q[:, g], k[:, g]) * d ** -0.5
        score = score.masked_fill(~seen, float("-inf"))
        score = (score - score.amax(-1, keepdim=True)).exp_()
        score /= score.sum(-1, keepdim=True)
        outs.append(torch.einsum("gtj,jd->tgd", score, v[:, g]))
    return torch.stack(outs, 1).reshape(new, -1)


def _plain_tables(s):
    c, ps, T, width = s["case"], s["case"]["page"], s["T"], s["width"]
    row, start, count, have, off = s["entries"].long().unbind(1)
    dev, B = row.device, row.shape[0]
    w = torch.arange(width, device=dev)
    need = (start + count + ps - 1) // ps
    fresh = (w >= have[:, None]) & (w < need[:, None])
    given = s["new_pages"][torch.where(fresh, off[:, None] + w - have[:, None], torch.zeros_like(w))]
    table = torch.where(fresh, given, s["master"][row])
    s["master"][row] = table
    table = torch.where(w < need[:, None], table, torch.zeros_like(table))
    ends = count.cumsum(0)
    q_start = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(T, device=dev)
    seq = (t[:, None] >= ends).sum(1)
    pos = start[seq] + t - q_start[seq]
    slots = table[seq, pos // ps] * ps + pos % ps
    b = torch.arange(B, device=dev)
    single = count == 1
    rank = torch.where(single, single.long().cumsum(0) - 1, (~single).long().cumsum(0) - 1)
    dec = torch.zeros(B, dtype=torch.long, device=dev)
    por = torch.zeros((B, 4), dtype=torch.long, device=dev)
    first = q_start[:B]
    dec.scatter_add_(0, rank, torch.where(single, first, torch.zeros_like(first)))
    item = torch.stack([b, first, count, start], 1) * (~single)[:, None]
    por.scatter_add_(0, rank[:, None].expand(-1, 4), item)
    out = [q_start, pos, seq, start + count, slots, table, dec[:s["n_dec"]], por[:B - s["n_dec"]]]
    return [x.int() for x in out] + [s["master"]]


# ------------------------------------------------------------------------------------ work
def _keys(c, before, new):
    """Keys that some row of a request sees, and pairs of a row and a key it sees."""
    n = before + new
    if not c["window"]:
        return n, new * before + new * (new + 1) // 2
    w, keep = c["window"], c["keep"]
    first = max(0, before - w + 1)
    seen = n - first + min(keep, first)
    pairs = 0
    for p in range(before, n):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(keep, lo)
    return seen, pairs


def work(case):
    c, reqs = case, _requests(case)
    nkv, d, ps = c["kv_heads"], c["dim"], c["page"]
    T, B = sum(n for _, n in reqs), len(reqs)
    if c["kind"] == "tables":
        ints = 5 * B + (B + 1) + 3 * T + B
        pages = sum(-(-(b + n) // ps) for b, n in reqs)
        width = max(-(-(b + n) // ps) for b, n in reqs) + 3
        return {"bytes": 4 * (ints + pages + B * width), "flops": 0}
    token = nkv * d * 9 // 8                             # codes and (s, m) of a token's keys and values
    if c["kind"] == "store":
        ctx = sum(b + n for b, n in reqs)
        rows = sum(-(-(b + n) // LOAD_PAGE) * LOAD_PAGE for b, n in reqs)
        return {"bytes": T * (4 * nkv * d + token) + ctx * token + (rows + LOAD_PAGE) * nkv * d * 4,
                "flops": 0}
    seen = [_keys(c, b, n) for b, n in reqs]
    return {"bytes": sum(k for k, _ in seen) * token + 4 * T * c["heads"] * d,
            "flops": 4 * d * c["heads"] * sum(p for _, p in seen)}


# ------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """The same from the definitions in 64 bits: the numbers that the codes stand for are worked out
    from the rows, never from the pages' bytes."""
    c, reqs = case, _requests(case)
    if c["kind"] == "tables":
        return None
    outs, contexts = [], []
    T = sum(n for _, n in reqs)
    if c["kind"] != "store":
        q = torch.randn((T, c["heads"] * c["dim"]), generator=_generator(seed, "queries"), device=DEVICE)
        q = q.mul_(1.3).to(BF16).to(F64)
    at = 0
    for i, (before, new) in enumerate(reqs):
        held = [_held64(x) for x in _rows(c, seed, "request %d" % i, before + new)]
        if c["kind"] == "store":
            contexts.append(held)
            continue
        outs.append(_attend64(c, q[at:at + new], held[0], held[1], before))
        at += new
    if c["kind"] != "store":
        return torch.cat(outs)
    k, v, _ = _as_pages(reqs, contexts, F64)
    return k, v, None


def _held64(x):
    """What rows stand for once they are held in 4 bits."""
    g = x.to(F64).view(x.shape[0], x.shape[1], -1, GROUP)
    low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    step = ((high - low) / 15).to(BF16).to(F64)
    code = ((g - low) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(max=15)
    return (low + step * code).view(x.shape)


def _attend64(c, q, k, v, before):
    new, d, group = q.shape[0], c["dim"], c["heads"] // c["kv_heads"]
    out = torch.empty((new, c["heads"], d), dtype=F64, device=q.device)
    key = torch.arange(k.shape[0], device=q.device)
    for a in range(0, new, 512):
        e = min(new, a + 512)
        at = torch.arange(before + a, before + e, device=q.device).view(-1, 1)
        hidden = key > at
        if c["window"]:
            hidden |= (at - key >= c["window"]) & (key >= c["keep"])
        for h in range(c["heads"]):
            g = h // group
            logit = q[a:e].view(e - a, c["heads"], d)[:, h] @ k[:, g].T / math.sqrt(d)
            logit[hidden] = -math.inf
            out[a:e, h] = torch.softmax(logit, -1) @ v[:, g]
    return out.view(new, -1)

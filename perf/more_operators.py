"""Matrix products with weights in 8 bits, as cases that can be timed and compared.

A number is held as an e4m3 code (1 sign, 4 exponent, 3 fraction bits, largest value 448) times a
float32 scale.  Weights ``[N, K]`` share a scale over blocks of 128 x 128, activations ``[T, K]`` over
128 neighbouring numbers of a row.  With a the largest size of such a group, its scale is
``s = max(float32(a / 448), 2^-100)`` and a number's code the e4m3 value nearest to ``x / s`` (ties to
even).  A stacked gate/up weight ``[2 I, K]`` is two weights of I rows: the up rows' blocks begin anew.

Kinds of pass:

* ``rows``: activations into codes and scales, and back out of them;
* ``blocks``: the same of a weight;
* ``linear``: activations times a held weight, the activations put into 8 bits within the call: with t
  over the groups of 128, ``out[m, n] = sum_t sx[m, t] sw[n / 128, t] sum_k cx[m, k] cw[n, k]``;
  ``gated``: ``silu(g) u`` of the two halves g and u of the result;
* ``experts``: the same of rows that are sorted by expert, each expert's against its own weight;
  ``weighted``: every row of the result times its token's weight for the expert.

``own`` False computes a pass in plain torch, True through the package's entry points.
"""
import math
import zlib

import torch

own = False

DEVICE = "cuda:0"
F32, F64, BF16, E4M3 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn
GROUP = 128
LARGEST = 448.0
FLOOR = 2.0 ** -100


# --------------------------------------------------------------------------------- cases
def _case(name, kind, **kw):
    c = dict(name=name, kind=kind, tokens=1, width=4096, features=4096, gated=False, experts=0,
             top=0, weighted=False, wide=False)
    c.update(kw)
    return c


def listed():
    """``tokens`` rows of ``width`` numbers against ``features`` outputs (a gated weight has twice as
    many rows); ``top`` of ``experts`` experts for every token; ``wide``: results in 32 bits."""
    return [
        # what a decode step of eight requests hands to a projection
        _case("rows_step", "rows", tokens=8, width=4096),
        # a prompt portion's feed-forward activations
        _case("rows_prompt", "rows", tokens=2048, width=12288),
        # a small head's weight at odd sizes, and a feed-forward's: what loading a model does
        _case("blocks_odd", "blocks", features=1000, width=1111),
        _case("blocks_weight", "blocks", features=12288, width=4096),
        # one user's decode step: the q/k/v projection
        _case("linear_one", "linear", tokens=1, width=4096, features=6144),
        # a decode step of eight requests: the down projection
        _case("linear_step", "linear", tokens=8, width=12288, features=4096),
        # a large decode batch with a short prompt portion in it
        _case("linear_mixed", "linear", tokens=157, width=4096, features=6144),
        # a decode step of eight requests: gate and up projections
        _case("gated_step", "linear", tokens=8, width=4096, features=12288, gated=True),
        # a prompt portion's gate and up projections
        _case("gated_prompt", "linear", tokens=2048, width=4096, features=12288, gated=True),
        # a decode step of a mixture: few rows an expert, some experts without any
        _case("experts_step", "experts", tokens=8, width=2048, features=1024, experts=64, top=8,
              gated=True),
        # a prompt portion through a mixture's down projections, whose width is no multiple of 128
        _case("experts_down", "experts", tokens=1011, width=704, features=1024, experts=64, top=8,
              weighted=True, wide=True),
        # a prompt portion through a mixture of few large experts
        _case("experts_prompt", "experts", tokens=2048, width=4096, features=2048, experts=8, top=2,
              gated=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Mostly whole groups of 128, some multiples of 16, some odd."""
    n = _log(rng, lo, hi)
    step = rng.choice([128, 128, 128, 16, 1])
    return max(lo, n // step * step)


def draw(rng):
    """1 to 4,096 rows of 16 to 12,288 numbers against 16 to 12,288 outputs; 2 to 64 experts of which a
    token takes 1 to 8."""
    kind = rng.choice(["rows", "blocks", "linear", "linear", "linear", "experts", "experts"])
    c = dict(kind=kind, tokens=_log(rng, 1, 4096), width=_size(rng, 16, 12288),
             features=_size(rng, 16, 12288), gated=False, experts=0, top=0, weighted=False,
             wide=rng.random() < 0.3)
    if kind in ("linear", "experts"):
        c["gated"] = rng.random() < 0.4
    if kind == "experts":
        c["experts"] = _log(rng, 2, 64)
        c["top"] = min(c["experts"], rng.choice([1, 2, 4, 8]))
        c["weighted"] = rng.random() < 0.4
        # every expert's weight fits: at most 2^30 numbers in all
        c["width"] = min(c["width"], 4096)
        c["features"] = max(16, min(c["features"], (1 << 28) // (c["experts"] * c["width"])))
        c["tokens"] = max(1, min(c["tokens"], 8192 // c["top"]))
    if c["gated"]:
        c["wide"] = False
    cost = c["tokens"] * max(1, c["top"]) * c["width"] * c["features"] * (2 if c["gated"] else 1)
    if kind in ("linear", "experts") and cost > 2e11:
        c["tokens"] = max(1, int(c["tokens"] * 2e11 / cost))
    return c


def _generator(seed, name):
    g = torch.Generator(DEVICE)
    g.manual_seed((int(seed) * 1_000_003 + zlib.crc32(name.encode())) & 0x7FFF_FFFF_FFFF)
    return g


# ------------------------------------------------------------------- inputs
def _activations(c, seed, rows):
    """Normal numbers whose columns differ in size, with a few columns far larger than the others, as
    behind a norm's weight."""
    g = _generator(seed, "x")
    x = torch.randn((rows, c["width"]), generator=g, device=DEVICE)
    size = torch.exp(0.5 * torch.randn(c["width"], generator=g, device=DEVICE))
    size = size * torch.where(torch.rand(c["width"], generator=g, device=DEVICE) < 0.005, 20.0, 1.0)
    return (x * size).to(BF16)


def _weight(c, seed):
    """bfloat16 ``[N, K]`` or ``[E, N, K]``, the rows of different sizes."""
    g = _generator(seed, "w")
    n = c["features"] * (2 if c["gated"] else 1)
    shape = (c["experts"], n, c["width"]) if c["experts"] else (n, c["width"])
    w = torch.randn(shape, generator=g, device=DEVICE, dtype=BF16)
    size = torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=g, device=DEVICE))
    return w.mul_((size / math.sqrt(c["width"])).to(BF16))


def _choices(c, seed):
    """The experts' first rows (``experts + 1`` of them): every token takes ``top`` experts, some of
    which are far more popular than others."""
    g = _generator(seed, "choices")
    taste = 0.7 * torch.randn(c["experts"], generator=g, device=DEVICE)
    z = taste + torch.randn((c["tokens"], c["experts"]), generator=g, device=DEVICE)
    ids = z.topk(c["top"], dim=1).indices.reshape(-1)
    count = torch.bincount(ids, minlength=c["experts"])
    return torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)


def prepare(case, seed):
    c = case
    s = {"case": c}
    if c["kind"] == "blocks":
        s["w"] = _weight(c, seed)
        return s
    if c["kind"] == "rows":
        s["x"] = _activations(c, seed, c["tokens"])
        return s
    rows = c["tokens"] * max(1, c["top"])
    s["x"] = _activations(c, seed, rows)
    w = _weight(c, seed)
    # the weight as a checkpoint holds it (an expert at a time: the plain form takes room)
    parts = [_hold_blocks(p, c["gated"]) for p in (w if c["experts"] else [w])]
    codes = torch.stack([p[0] for p in parts]).to(E4M3)
    scales = torch.stack([p[1] for p in parts])
    if not c["experts"]:
        codes, scales = codes[0], scales[0]
    s["out_type"] = F32 if c["wide"] else BF16
    if c["experts"]:
        s["starts"] = _choices(c, seed)
        s["starts_host"] = s["starts"].tolist()
        if c["weighted"]:
            s["row_w"] = torch.rand(rows, generator=_generator(seed, "row_w"), device=DEVICE)
    if own:
        from binfer_b200.csrc import ops
        s["w"] = ops.Fp8Weight(codes, scales, gated=c["gated"])
    else:
        s["codes"], s["scales"] = codes, scales
    return s


# ------------------------------------------------------------------- the plain form
def _nearest(q):
    """The e4m3 values nearest to ``q`` (float64, at most 448 in size), ties to even: numbers of one
    power of two lie an eighth of it apart, those below 2^-6 lie 2^-9 apart."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(q / step) * step).clamp(-LARGEST, LARGEST)


def _padded(x, rows, cols):
    pad = [0, -x.shape[1] % cols, 0, -x.shape[0] % rows]
    return torch.nn.functional.pad(x.to(F32), pad)


def _hold(x, rows):
    """(values of the codes float32 [T, K], scales [T / rows, K / 128]) of groups of rows x 128."""
    T, K = x.shape
    g = _padded(x, rows, GROUP)
    g = g.reshape(g.shape[0] // rows, rows, g.shape[1] // GROUP, GROUP)
    # (the quotient in 64 bits: by a plain number, 32 bits are multiplied by its reciprocal)
    scales = (g.abs().amax(dim=(1, 3)).to(F64) / LARGEST).to(F32).clamp_min(FLOOR)
    v = _nearest(g.to(F64) / scales.to(F64)[:, None, :, None]).to(F32)
    return v.reshape(v.shape[0] * rows, -1)[:T, :K], scales


def _hold_blocks(w, gated):
    if gated:
        n = w.shape[0] // 2
        halves = [_hold(w[:n], GROUP), _hold(w[n:], GROUP)]
        return torch.cat([h[0] for h in halves]), torch.cat([h[1] for h in halves])
    return _hold(w, GROUP)


def _values(codes, scales, rows, dtype):
    """What codes and scales stand for."""
    T, K = codes.shape
    s = scales.to(dtype).repeat_interleave(rows, 0)[:T].repeat_interleave(GROUP, 1)[:, :K]
    return codes.to(F32).to(dtype) * s


def _weight_values(codes, scales, gated, dtype):
    if gated:
        n, b = codes.shape[0] // 2, scales.shape[0] // 2
        return torch.cat([_values(codes[:n], scales[:b], GROUP, dtype),
                          _values(codes[n:], scales[b:], GROUP, dtype)])
    return _values(codes, scales, GROUP, dtype)


def _finish(y, gated):
    if gated:
        g, u = y.chunk(2, dim=1)
        y = g / (1 + torch.exp(-g)) * u
    return y


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "rows":
        codes, scales = _hold(s["x"], 1)
        return {"values": _values(codes, scales, 1, F32), "scales": scales.t().contiguous()}
    if c["kind"] == "blocks":
        codes, scales = _hold(s["w"], GROUP)
        return {"values": _values(codes, scales, GROUP, F32), "scales": scales}
    codes, scales = _hold(s["x"], 1)
    x = _values(codes, scales, 1, F32)
    if c["kind"] == "linear":
        w = _weight_values(s["codes"], s["scales"], c["gated"], F32)
        return _finish(x @ w.t(), c["gated"]).to(s["out_type"])
    out = torch.empty((x.shape[0], c["features"]), dtype=s["out_type"], device=DEVICE)
    for e, (a, b) in enumerate(zip(s["starts_host"], s["starts_host"][1:])):
        if b > a:
            w = _weight_values(s["codes"][e], s["scales"][e], c["gated"], F32)
            y = _finish(x[a:b] @ w.t(), c["gated"])
            if c["weighted"]:
                y = y * s["row_w"][a:b, None]
            out[a:b] = y.to(out.dtype)
    return out


# ------------------------------------------------------------------- a pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from binfer_b200.csrc import ops
    c = s["case"]
    if c["kind"] == "rows":
        codes, scales = ops.fp8_rows(s["x"])
        values = torch.empty(s["x"].shape, dtype=F32, device=DEVICE)
        ops.fp8_rows_read(codes, scales, values)
        return {"values": values, "scales": scales}
    if c["kind"] == "blocks":
        w = ops.fp8_weight(s["w"])
        values = torch.empty(s["w"].shape, dtype=F32, device=DEVICE)
        ops.fp8_weight_read(w, values)
        return {"values": values, "scales": w.scales}
    out = torch.empty((s["x"].shape[0], c["features"]), dtype=s["out_type"], device=DEVICE)
    if c["kind"] == "linear":
        ops.fp8_linear(s["x"], s["w"], out)
    else:
        ops.fp8_experts(s["x"], s["w"], s["starts"], out, row_w=s.get("row_w"))
    return out


def work(case):
    c = case
    t, k, n = c["tokens"], c["width"], c["features"]
    groups = -(-k // GROUP)
    if c["kind"] == "rows":
        # in, codes out and in, values out, scales out and in
        return {"bytes": t * k * (2 + 1 + 1 + 4) + 8 * t * groups, "flops": 4 * t * k}
    if c["kind"] == "blocks":
        return {"bytes": n * k * (2 + 1 + 1 + 4) + 8 * groups * -(-n // GROUP), "flops": 4 * n * k}
    rows, held = t * max(1, c["top"]), n * (2 if c["gated"] else 1)
    used = 1.0
    if c["experts"]:
        used = c["experts"] * (1 - (1 - 1 / c["experts"]) ** rows)
    return {"bytes": int(2 * rows * k + used * held * (k + 4 * groups / GROUP)
                         + rows * n * (4 if c["wide"] else 2)),
            "flops": 2 * rows * held * k}


# ------------------------------------------------------------------- in 64 bits
def _table(device):
    """The 127 e4m3 values from 0 on, by code, in float64."""
    c = torch.arange(127, device=device)
    e, f = c // 8, (c % 8).to(F64)
    return torch.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * torch.exp2(e.to(F64) - 7))


def _hold64(x, rows):
    """(values float64, scales float64): a number lies above the middle of two neighbouring codes or
    not, by x against middle times scale, which float64 holds exactly."""
    T, K = x.shape
    table = _table(x.device)
    middle = (table[1:] + table[:-1]) / 2
    values = torch.empty((T, K), dtype=F64, device=x.device)
    scales = torch.empty((-(-T // rows), -(-K // GROUP)), dtype=F64, device=x.device)
    step = rows * max(1, (1 << 24) // (rows * max(K, 1)))
    for t0 in range(0, T, step):
        part = x[t0:t0 + step].to(F64)
        for i, k0 in enumerate(range(0, K, GROUP)):
            p = part[:, k0:k0 + GROUP]
            biggest = p.abs().amax(dim=1)
            n = -(-p.shape[0] // rows)
            full = biggest.new_zeros(n * rows)
            full[:p.shape[0]] = biggest
            s = (full.view(n, rows).amax(dim=1) / LARGEST).to(F32).to(F64).clamp_min(FLOOR)
            scales[t0 // rows:t0 // rows + n, i] = s
            each = s.repeat_interleave(rows)[:p.shape[0], None]
            # first by the quotient, then put right where x lies on the other side of a middle
            at = torch.bucketize((p.abs() / each).contiguous(), middle)
            low = middle[(at - 1).clamp_min(0)] * each
            at = torch.where((at > 0) & (p.abs() < low), at - 1, at)
            high = middle[at.clamp_max(125)] * each
            at = torch.where((at < 126) & (p.abs() > high), at + 1, at)
            low = middle[(at - 1).clamp_min(0)] * each
            high = middle[at.clamp_max(125)] * each
            at = torch.where((at > 0) & (p.abs() == low) & (at % 2 == 1), at - 1, at)
            at = torch.where((at < 126) & (p.abs() == high) & (at % 2 == 1), at + 1, at)
            values[t0:t0 + step, k0:k0 + GROUP] = torch.sign(p) * table[at] * each
    return values, scales


def _weight64(w, gated):
    if gated:
        n = w.shape[0] // 2
        return torch.cat([_hold64(w[:n], GROUP)[0], _hold64(w[n:], GROUP)[0]])
    return _hold64(w, GROUP)[0]


def exact(case, seed):
    c = case
    if c["kind"] == "blocks":
        values, scales = _hold64(_weight(c, seed), GROUP)
        return {"values": values, "scales": scales}
    rows = c["tokens"] * max(1, c["top"])
    x, scales = _hold64(_activations(c, seed, rows), 1)
    if c["kind"] == "rows":
        return {"values": x, "scales": scales.t().contiguous()}
    w = _weight(c, seed)

    def product(a, weight):
        y = a @ _weight64(weight, c["gated"]).t()
        if c["gated"]:
            n = y.shape[1] // 2
            y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
        return y

    if c["kind"] == "linear":
        return product(x, w)
    starts = _choices(c, seed).tolist()
    out = torch.empty((rows, c["features"]), dtype=F64, device=DEVICE)
    for e in range(c["experts"]):
        a, b = starts[e], starts[e + 1]
        if b > a:
            out[a:b] = product(x[a:b], w[e])
    if c["weighted"]:
        out *= torch.rand(rows, generator=_generator(seed, "row_w"), device=DEVICE).to(F64)[:, None]
    return out

"""Weights in 8 bits: quantising, reading back and the products against their restatement in 64 bits."""
import copy
import gc
import pickle

import pytest
import torch

import fp8_plain as P8

pytestmark = pytest.mark.gpu

BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


def _x(T, K, dev, seed=0, dtype=BF16):
    g = torch.Generator(dev).manual_seed(seed)
    x = torch.randn((T, K), generator=g, device=dev) * torch.exp(torch.randn(K, generator=g, device=dev))
    return x.to(dtype)


def _w(shape, dev, seed=0):
    g = torch.Generator(dev).manual_seed(1000 + seed)
    return (torch.randn(shape, generator=g, device=dev) * shape[-1] ** -0.5).to(BF16)


def _same(a, b):
    """Equal, NaN where the other is."""
    return torch.equal(torch.nan_to_num(a, nan=-1234.5), torch.nan_to_num(b, nan=-1234.5))


def _check(got, ref, off):
    # a result is rounded to its type: half a step
    allowed = off + ref.abs() * (torch.finfo(got.dtype).eps / 2)
    diff = (got.to(F64) - ref).abs()
    bad = ~(diff <= allowed)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} too far off, worst "
                           f"{float((diff / allowed).nan_to_num(0).max()):.3g} of what is allowed")


# ------------------------------------------------------------------------- into 8 bits and back
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 129), (7, 16), (33, 1000), (5, 4096), (130, 333)])
def test_rows(cuda_device, T, K, dtype):
    from binfer_b200.csrc import ops
    x = _x(T, K, cuda_device, T + K, dtype)
    codes, scales = ops.fp8_rows(x)
    v, s = P8.hold(x, 1)
    assert torch.equal(scales.t(), s)
    assert torch.equal(codes.to(F32).to(F64), v)
    for out_type in (F32, BF16):
        out = torch.empty((T, K), dtype=out_type, device=cuda_device)
        ops.fp8_rows_read(codes, scales, out)
        assert torch.equal(out, P8.dense(v, s, 1).to(F32).to(out_type))


@pytest.mark.parametrize("K,off", [(256, 1), (250, 3), (77, 5)])
def test_rows_of_a_wider_buffer(cuda_device, K, off):
    from binfer_b200.csrc import ops
    wide = _x(9, K + 17, cuda_device, K)
    codes, scales = ops.fp8_rows(wide[:, off:off + K])
    ref, s = ops.fp8_rows(wide[:, off:off + K].contiguous())
    assert torch.equal(codes.view(torch.uint8), ref.view(torch.uint8)) and torch.equal(scales, s)
    out = torch.full((9, K + 17), 7.0, device=cuda_device)
    ops.fp8_rows_read(codes, scales, out[:, off:off + K])
    assert (out[:, :off] == 7).all() and (out[:, off + K:] == 7).all()
    assert torch.equal(out[:, off:off + K], P8.dense(*P8.hold(wide[:, off:off + K], 1), 1).to(F32))


def test_rows_next_to_a_border(cuda_device):
    """Numbers on the middle of two codes and one place to either side of it, for scales of every kind."""
    from binfer_b200.csrc import ops
    g = torch.Generator().manual_seed(5)
    v = P8.values()
    mid = (v[1:] + v[:-1]) / 2                                    # 126 of them
    rows = []
    for i in range(600):
        top = torch.rand(1, generator=g).item() * 2.0 ** ((i % 60) - 30)
        s = P8.scale(torch.tensor([top]))
        x = (mid * s.to(F64)).to(F32)
        x = torch.nextafter(x, x + [0, 1e30, -1e30][i % 3])
        rows.append(torch.cat([torch.tensor([top, -top]), x * (1 - 2 * (torch.arange(126) % 2))]).to(F32))
    x = torch.stack(rows).to(cuda_device)
    codes, scales = ops.fp8_rows(x)
    v, s = P8.hold(x, 1)
    assert torch.equal(scales.t(), s) and torch.equal(codes.to(F32).to(F64), v)


@pytest.mark.parametrize("size", [2.0 ** -149, 2.0 ** -130, 2.0 ** -101, 2.0 ** -93, 2.0 ** -60, 2.0 ** 100,
                                  2.0 ** 127])
def test_rows_of_any_size(cuda_device, size):
    from binfer_b200.csrc import ops
    g = torch.Generator().manual_seed(int(abs(torch.tensor(size).log2())))
    x = ((torch.rand((8, 256), generator=g, dtype=F64) * 2 - 1) * size * 1.9).to(F32).to(cuda_device)
    codes, scales = ops.fp8_rows(x)
    v, s = P8.hold(x, 1)
    assert torch.equal(scales.t(), s) and torch.equal(codes.to(F32).to(F64), v)


def test_rows_that_are_not_finite(cuda_device):
    from binfer_b200.csrc import ops
    x = _x(6, 300, cuda_device, 3)
    x[1, 5], x[2, 140], x[3, 299], x[4] = float("inf"), float("nan"), float("-inf"), 0
    codes, scales = ops.fp8_rows(x)
    v, s = P8.hold(x, 1)
    assert _same(scales.t(), s) and _same(codes.to(F32).to(F64), v)
    assert int(torch.isnan(s).sum()) == 3 and not codes[4].to(F32).any()


@pytest.mark.parametrize("shape,gated", [((1, 1), False), ((128, 128), False), ((300, 200), False),
                                         ((129, 77), False), ((300, 200), True), ((3, 130, 260), False),
                                         ((2, 260, 100), True), ((1000, 1111), False)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_weight(cuda_device, shape, gated, dtype):
    from binfer_b200.csrc import ops
    w = _w(shape, cuda_device, sum(shape)).to(dtype) * 3
    h = ops.fp8_weight(w, gated)
    mats = [w] if w.dim() == 2 else list(w)
    for i, m in enumerate(mats):
        v, s = P8.hold_weight(m, gated)
        hs, hc = (h.scales, h.codes) if w.dim() == 2 else (h.scales[i], h.codes[i])
        assert torch.equal(hs, s) and torch.equal(hc.to(F32).to(F64), v)
    for out_type in (F32, BF16):
        out = torch.empty(shape, dtype=out_type, device=cuda_device)
        ops.fp8_weight_read(h, out)
        for i, m in enumerate(mats):
            ref = P8.dense(*P8.hold_weight(m, gated), 128, gated).to(F32).to(out_type)
            assert torch.equal(out if w.dim() == 2 else out[i], ref)


def test_weight_of_a_wider_buffer(cuda_device):
    from binfer_b200.csrc import ops
    wide = _w((300, 263), cuda_device)
    a, b = ops.fp8_weight(wide[:, 5:205]), ops.fp8_weight(wide[:, 5:205].contiguous())
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    with pytest.raises(ops.KernelError):
        ops.fp8_weight(wide[:200].view(2, 100, 263)[:, :99])          # the matrices lie further apart


# --------------------------------------------------------------------------------- products
def _linear(dev, M, K, N, gated=False, out_type=BF16, seed=0, **kw):
    from binfer_b200.csrc import ops
    x, w = _x(M, K, dev, seed), _w(((2 if gated else 1) * N, K), dev, seed)
    out = torch.full((M, N), float("nan"), dtype=out_type, device=dev)
    ops.fp8_linear(x, ops.fp8_weight(w, gated), out, **kw)
    assert ops.error_word(dev).item() == 0
    return out, P8.product(x, *P8.hold_weight(w, gated), gated)


SIZES = [(1, 128, 128), (1, 16, 16), (3, 1, 5), (8, 384, 640), (16, 1000, 130), (17, 256, 257), (33, 130, 96),
         (64, 512, 300), (65, 2048, 128), (129, 640, 200), (200, 100, 1000), (257, 384, 513), (300, 1024, 64)]


@pytest.mark.parametrize("tile", [16, 32, 64, -1])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_of_every_tile(cuda_device, M, K, N, tile):
    out, ref = _linear(cuda_device, M, K, N, out_type=F32, seed=M + N, tile=tile)
    _check(out, *ref)


@pytest.mark.parametrize("tile", [16, 32, 64, -1])
@pytest.mark.parametrize("M,K,N", [(1, 128, 64), (5, 300, 100), (16, 512, 128), (40, 256, 200), (130, 640, 65),
                                   (300, 384, 300), (520, 256, 130)])
def test_gated_linear_of_every_tile(cuda_device, M, K, N, tile):
    out, ref = _linear(cuda_device, M, K, N, gated=True, seed=M + N, tile=tile)
    _check(out, *ref)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("split", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("M,K,N", [(1, 1024, 128), (7, 1100, 300), (16, 2048, 640), (33, 1024, 200), (64, 4096, 128)])
def test_linear_shared_by_a_cluster(cuda_device, M, K, N, split, gated):
    out, ref = _linear(cuda_device, M, K, N, gated=gated, seed=split, split=split)
    _check(out, *ref)


@pytest.mark.parametrize("M,K,N,gated", [(1, 4096, 6144, False), (8, 12288, 4096, False), (8, 4096, 12288, True),
                                         (100, 4096, 1024, False), (1030, 2048, 2048, True), (2048, 1024, 4096, False)])
def test_linear_as_chosen(cuda_device, M, K, N, gated):
    out, ref = _linear(cuda_device, M, K, N, gated=gated)
    _check(out, *ref)


@pytest.mark.parametrize("M", [3, 40, 150, 300])
def test_linear_of_strided_rows(cuda_device, M):
    """Column blocks of wider buffers, at odd offsets, on both sides; what lies beside the result stays."""
    from binfer_b200.csrc import ops
    wide, w = _x(M, 400, cuda_device, M), _w((203, 333), cuda_device)
    x, held = wide[:, 13:346], ops.fp8_weight(w)
    for out_type, off in ((BF16, 3), (F32, 1), (BF16, 8)):
        out = torch.full((M, 230), 5.0, dtype=out_type, device=cuda_device)
        ops.fp8_linear(x, held, out[:, off:off + 203])
        _check(out[:, off:off + 203], *P8.product(x, *P8.hold_weight(w)))
        assert (out[:, :off] == 5).all() and (out[:, off + 203:] == 5).all()


@pytest.mark.parametrize("M", [4, 50, 300])
def test_clamped_activation(cuda_device, M):
    from binfer_b200.csrc import ops
    x, w = _x(M, 256, cuda_device, M) * 2, _w((400, 256), cuda_device)
    out = torch.empty((M, 200), dtype=BF16, device=cuda_device)
    ops.fp8_linear(x, ops.fp8_weight(w, True), out, activation="clamped", limit=1.5, slope=1.7, up_offset=1.0)

    def act(g, u):
        g, u = g.clamp_max(1.5), u.clamp(-1.5, 1.5) + 1.0
        return g * torch.sigmoid(1.7 * g), u
    ref, off = P8.product(x, *P8.hold_weight(w, True), True, act)
    _check(out, ref, off)


@pytest.mark.parametrize("M", [6, 70, 300])
def test_rows_do_not_touch_one_another(cuda_device, M):
    """A row with an infinity or a NaN is NaN; the others are what they were.  A row of zeros is zero."""
    from binfer_b200.csrc import ops
    x, w = _x(M, 384, cuda_device, M), ops.fp8_weight(_w((300, 384), cuda_device))
    x[2] = 0
    a = torch.empty((M, 300), dtype=BF16, device=cuda_device)
    ops.fp8_linear(x, w, a)
    assert not a[2].any()
    x[1, 7], x[4, 300], x[5, 383] = float("inf"), float("nan"), float("-inf")
    b = torch.empty_like(a)
    ops.fp8_linear(x, w, b)
    bad = torch.tensor([1, 4, 5], device=cuda_device)
    assert torch.isnan(b[bad]).all()
    rest = torch.ones(M, dtype=torch.bool, device=cuda_device)
    rest[bad] = False
    assert torch.equal(a[rest], b[rest])


def test_scales_of_any_size(cuda_device):
    """Products of scales that a float has no room for count with the largest float and leave zeros zero."""
    from binfer_b200.csrc import ops
    for M in (3, 300):
        x = torch.zeros((M, 256), dtype=BF16, device=cuda_device)
        x[:, 0], x[1, 0] = 2.0 ** 120, 2.0 ** -120
        w = torch.zeros((128, 256), device=cuda_device)
        w[:, 1] = 2.0 ** 100
        w[5, 0] = 2.0 ** -60
        w[:, 200], x[:, 200] = 1.0, 3.0
        out = torch.empty((M, 128), dtype=F32, device=cuda_device)
        ops.fp8_linear(x, ops.fp8_weight(w), out)
        # (2^-60 is far below a code's step beside 2^100: it reads as zero.  448 x 448 times two scales,
        # each rounded, their product and the sum too)
        assert ((out - 3.0).abs() <= 3.0 * 2.0 ** -21).all()


def test_empty_calls(cuda_device):
    from binfer_b200.csrc import ops
    w = ops.fp8_weight(_w((300, 200), cuda_device))
    ops.fp8_linear(torch.empty((0, 200), dtype=BF16, device=cuda_device), w,
                   torch.empty((0, 300), dtype=BF16, device=cuda_device))
    codes, scales = ops.fp8_rows(torch.empty((0, 200), dtype=BF16, device=cuda_device))
    assert codes.shape == (0, 200) and scales.shape == (2, 0)
    ops.fp8_rows_read(codes, scales, torch.empty((0, 200), device=cuda_device))


# ---------------------------------------------------------------------------------- experts
def _experts(dev, counts, K, N, gated=False, out_type=BF16, before=0, behind=0, weighted=False, seed=0, tile=0):
    from binfer_b200.csrc import ops
    E, R = len(counts), before + sum(counts) + behind
    x, w = _x(R, K, dev, seed), _w((E, (2 if gated else 1) * N, K), dev, seed)
    starts = [before]
    for c in counts:
        starts.append(starts[-1] + c)
    row_w = torch.rand(R, device=dev) if weighted else None
    out = torch.full((R, N), 9.0, dtype=out_type, device=dev)
    ops.fp8_experts(x, ops.fp8_weight(w, gated), torch.tensor(starts, dtype=torch.int32, device=dev), out,
                    row_w=row_w, tile=tile)
    assert ops.error_word(dev).item() == 0
    assert (out[:before] == 9).all() and (out[R - behind:] == 9).all()
    for e, (a, b) in enumerate(zip(starts, starts[1:])):
        if b > a:
            ref, off = P8.product(x[a:b], *P8.hold_weight(w[e], gated), gated)
            if weighted:
                ref, off = ref * row_w[a:b, None].to(F64), (off + ref.abs() * 2.0 ** -23) * row_w[a:b, None].to(F64)
            _check(out[a:b], ref, off)


@pytest.mark.parametrize("tile", [0, 16, 32, 64, -1])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts", [[1], [0, 0, 3], [5, 0, 17, 1, 16, 0], [40, 300, 0, 129, 64], [600, 2]])
def test_experts(cuda_device, counts, gated, tile):
    _experts(cuda_device, counts, 384, 200, gated=gated, seed=len(counts), tile=tile)


@pytest.mark.parametrize("K,N", [(100, 16), (704, 130), (129, 1)])
@pytest.mark.parametrize("tile", [0, -1])
def test_experts_in_part_of_the_rows(cuda_device, K, N, tile):
    _experts(cuda_device, [7, 0, 30, 260], K, N, before=5, behind=11, weighted=True, out_type=F32, tile=tile)
    _experts(cuda_device, [3, 4], K, N, before=1, behind=2, weighted=True, gated=True, tile=tile)


def test_many_experts(cuda_device):
    _experts(cuda_device, [(i * 7) % 5 for i in range(512)], 128, 64)


def test_no_rows_at_all(cuda_device):
    _experts(cuda_device, [0, 0, 0], 256, 128, before=4, behind=3)
    _experts(cuda_device, [0, 0, 0], 256, 128, before=4, behind=3, gated=True, tile=-1)


@pytest.mark.parametrize("tile", [16, -1])
def test_starts_outside_the_rows(cuda_device, tile):
    """Whatever the starts hold, what is read and written lies inside the rows."""
    from binfer_b200.csrc import ops
    x, w = _x(20, 128, cuda_device), ops.fp8_weight(_w((3, 64, 128), cuda_device))
    out = torch.full((20, 64), 9.0, dtype=BF16, device=cuda_device)
    s = torch.tensor([-5, 4, 2, 1000], dtype=torch.int32, device=cuda_device)
    ops.fp8_experts(x, w, s, out, tile=tile)
    # (the first expert has rows 0 .. 3, the second none, the third 2 .. 19, two rows of which are both's)
    _check(out[:2], *P8.product(x[:2], w.codes[0].to(F32).to(F64), w.scales[0]))
    _check(out[4:], *P8.product(x[4:], w.codes[2].to(F32).to(F64), w.scales[2]))


# ------------------------------------------------------------------------ streams, graphs, together
def test_on_another_stream(cuda_device):
    from binfer_b200.csrc import ops
    x, w = _x(8, 512, cuda_device), _w((256, 512), cuda_device)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty((8, 256), dtype=BF16, device=cuda_device)
        for _ in range(20):
            h = ops.fp8_weight(w * 1.0)               # the weight made right before the product
            ops.fp8_linear(x, h, out)
    side.synchronize()
    _check(out, *P8.product(x, *P8.hold_weight(w)))


@pytest.mark.parametrize("M", [8, 300])
def test_captured_and_replayed(cuda_device, M):
    """Two graphs of one weight, replayed in turn with other rows."""
    from binfer_b200.csrc import ops
    w, e = _w((256, 512), cuda_device), _w((4, 256, 256), cuda_device)
    held, held_e = ops.fp8_weight(w), ops.fp8_weight(e, True)
    starts = torch.tensor([0, 2, 2, 5, M], dtype=torch.int32, device=cuda_device)

    def step(x, y, z):
        ops.fp8_linear(x, held, y)
        ops.fp8_experts(y, held_e, starts, z)
    graphs = []
    for seed in range(2):
        x = _x(M, 512, cuda_device, seed)
        y = torch.empty((M, 256), dtype=BF16, device=cuda_device)
        z = torch.empty((M, 128), dtype=BF16, device=cuda_device)
        step(x, y, z)
        torch.cuda.synchronize()
        gc.collect()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(x, y, z)
        graphs.append((g, x, y, z))
    for seed in range(4):
        g, x, y, z = graphs[seed % 2]
        x.copy_(_x(M, 512, cuda_device, 50 + seed))
        g.replay()
        _check(y, *P8.product(x, *P8.hold_weight(w)))
        s = starts.tolist()
        for i, (a, b) in enumerate(zip(s, s[1:])):
            if b > a:
                _check(z[a:b], *P8.product(y[a:b], *P8.hold_weight(e[i], True), True))


def test_a_feed_forward(cuda_device):
    """The operators one behind the other, as a mixture uses them: rows sorted by expert, gate and up, down."""
    from binfer_b200.csrc import ops
    counts = [9, 0, 40, 3]
    R, starts = sum(counts), torch.tensor([0, 9, 9, 49, 52], dtype=torch.int32, device=cuda_device)
    x, row_w = _x(R, 256, cuda_device), torch.rand(52, device=cuda_device)
    gu, dn = _w((4, 384, 256), cuda_device, 1), _w((4, 256, 192), cuda_device, 2)
    h = torch.empty((R, 192), dtype=BF16, device=cuda_device)
    y = torch.empty((R, 256), dtype=F32, device=cuda_device)
    ops.fp8_experts(x, ops.fp8_weight(gu, True), starts, h)
    ops.fp8_experts(h, ops.fp8_weight(dn), starts, y, row_w=row_w)
    s = starts.tolist()
    for e, (a, b) in enumerate(zip(s, s[1:])):
        if b > a:
            _check(h[a:b], *P8.product(x[a:b], *P8.hold_weight(gu[e], True), True))
            ref, off = P8.product(h[a:b], *P8.hold_weight(dn[e]))
            k = row_w[a:b, None].to(F64)
            _check(y[a:b], ref * k, (off + ref.abs() * 2.0 ** -23) * k)


def test_repeats_bit_for_bit(cuda_device):
    from binfer_b200.csrc import ops
    for M in (5, 100, 600):
        x, w = _x(M, 2048, cuda_device), ops.fp8_weight(_w((512, 2048), cuda_device))
        outs = [torch.empty((M, 512), dtype=F32, device=cuda_device) for _ in range(5)]
        for o in outs:
            ops.fp8_linear(x, w, o)
        assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 300), (3, 1000, 130), (8, 12288, 256), (9, 4096, 128), (16, 2048, 5000),
                                   (20, 640, 4000), (32, 4096, 640)])
def test_one_kernel_or_two(cuda_device, monkeypatch, M, K, N, gated):
    """Few rows as one kernel and as two: the same codes, the same sums."""
    from binfer_b200.csrc import ops
    x, w = _x(M, K + 8, cuda_device, M)[:, 3:3 + K], ops.fp8_weight(_w(((1 + gated) * N, K), cuda_device), gated)
    for rows in (x, x.contiguous()):
        outs = []
        for resident in (True, False):
            monkeypatch.setattr(ops, "FP8_RESIDENT", resident)
            out = torch.empty((M, N), dtype=BF16, device=cuda_device)
            ops.fp8_linear(rows, w, out)
            outs.append(out)
        assert torch.equal(*outs)


@pytest.mark.parametrize("T,H", [(1, 8), (3, 200), (8, 4096), (17, 2048), (300, 1000), (5, 8192)])
def test_norm_into_8_bits(cuda_device, T, H):
    """The codes and scales of the norm's bfloat16 output, and the stream as the norm leaves it."""
    from binfer_b200.csrc import ops
    g = torch.Generator(cuda_device).manual_seed(T + H)
    w = 1 + 0.1 * torch.randn(H, generator=g, device=cuda_device)
    for delta in (None, _x(T, H, cuda_device, 5)):
        a = torch.randn((T, H), generator=g, device=cuda_device)
        b, y = a.clone(), torch.empty((T, H), dtype=BF16, device=cuda_device)
        ops.add_rmsnorm(a, delta, w, y, 1e-6)
        rows = ops.add_rmsnorm_fp8(b, delta, w, 1e-6)
        ref = ops.fp8_rows(y)
        assert torch.equal(a, b) and torch.equal(rows.scales, ref.scales)
        assert torch.equal(rows.codes.view(torch.uint8), ref.codes.view(torch.uint8))


@pytest.mark.parametrize("M", [1, 8, 40, 300])
def test_rows_that_are_there_already(cuda_device, M):
    from binfer_b200.csrc import ops
    for K in (384, 1000):
        x, w = _x(M, K, cuda_device, M), ops.fp8_weight(_w((300, K), cuda_device))
        e, starts = ops.fp8_weight(_w((2, 64, K), cuda_device)), torch.tensor([0, M // 2, M], dtype=torch.int32,
                                                                              device=cuda_device)
        rows = ops.fp8_rows(x)
        for call in (lambda r, o: ops.fp8_linear(r, w, o[:, :300]), lambda r, o: ops.fp8_experts(r, e, starts, o[:, :64])):
            a, b = (torch.zeros((M, 304), dtype=BF16, device=cuda_device) for _ in range(2))
            call(x, a)
            call(rows, b)
            assert torch.equal(a, b) and a.any()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("split", [2, 4])
@pytest.mark.parametrize("M,K,N", [(1, 512, 128), (157, 1100, 300), (256, 2048, 1024), (300, 640, 130), (513, 4096, 256)])
def test_linear_shared_by_pairs(cuda_device, M, K, N, split, gated):
    out, ref = _linear(cuda_device, M, K, N, gated=gated, seed=split, tile=-1, split=split)
    _check(out, *ref)


@pytest.mark.parametrize("M,K,N", [(157, 4096, 6144), (300, 12288, 4096), (512, 2048, 1024), (700, 4096, 4096)])
def test_middle_sizes_as_chosen(cuda_device, M, K, N):
    for out_type in (BF16, F32):
        out, ref = _linear(cuda_device, M, K, N, out_type=out_type)
        _check(out, *ref)


@pytest.mark.parametrize("M", [1, 8, 40, 300])
def test_result_in_the_rows_place(cuda_device, M):
    from binfer_b200.csrc import ops
    w = ops.fp8_weight(_w((512, 512), cuda_device))
    wide = torch.empty((M, 1024), dtype=BF16, device=cuda_device)
    x, ref = _x(M, 512, cuda_device, M), torch.empty((M, 512), dtype=BF16, device=cuda_device)
    ops.fp8_linear(x, w, ref)
    wide[:, 256:768] = x
    ops.fp8_linear(wide[:, 256:768], w, wide[:, 512:])       # half of it over the rows
    assert torch.equal(wide[:, 512:], ref)
    ops.fp8_linear(x, w, x)
    assert torch.equal(x, ref)


@pytest.mark.parametrize("M", [3, 40])
def test_copies_of_a_weight(cuda_device, M):
    """A deep copy, or a weight read back, has its own numbers; a shallow one has those of its source."""
    from binfer_b200.csrc import ops
    dev = cuda_device
    w = ops.fp8_weight(_w((300, 200), dev, 5))
    x = _x(M, 200, dev, 6)
    want, got = (torch.empty((M, 300), dtype=F32, device=dev) for _ in range(2))
    ops.fp8_linear(x, w, want)
    copies = [copy.deepcopy(w), pickle.loads(pickle.dumps(w)), copy.copy(w)]
    w.codes.view(torch.uint8).zero_()
    for c in copies[:2]:
        ops.fp8_linear(x, c, got)
        assert torch.equal(got, want)
    ops.fp8_linear(x, copies[2], got)
    assert not got.any()


@pytest.mark.parametrize("resident", [True, False])
@pytest.mark.parametrize("M", [1, 8, 20, 60, 300])
def test_a_weight_that_the_kernel_ahead_writes(cuda_device, monkeypatch, M, resident):
    """Codes that a kernel writes which lets its successor begin early: the product waits for them."""
    from binfer_b200.csrc import ops
    monkeypatch.setattr(ops, "FP8_RESIDENT", resident)
    N, K = 19000, 512
    x, scales = _x(M, K, cuda_device, M), torch.full((-(-N // 128), K // 128), 2.0 ** -6, device=cuda_device)
    makes = [_w((N, K), cuda_device, i).mul_(9) for i in range(3)]
    held = [ops.fp8_rows(m).codes.view(torch.uint8).clone() for m in makes]
    want = [P8.product(x, h.view(E4M3).to(F32).to(F64), scales) for h in held]
    torch.cuda.synchronize()
    out = torch.empty((M, N), dtype=F32, device=cuda_device)
    for i in [0, 1, 2] * 4:
        # (the codes' memory is that of the turn before, which the allocator gives out again)
        ops.fp8_linear(x, ops.Fp8Weight(ops.fp8_rows(makes[i]).codes, scales), out)
        _check(out, *want[i])


@pytest.mark.parametrize("H", [512, 4096])
def test_a_norm_s_weight_that_the_kernel_ahead_writes(cuda_device, H):
    """The norm's weight as the last row of what a kernel makes that lets its successor begin early."""
    from binfer_b200.csrc import ops
    T = 8192
    made = torch.zeros((T, H), device=cuda_device)
    g = torch.Generator(cuda_device).manual_seed(H)
    resid = torch.randn((3, H), generator=g, device=cuda_device)
    rows = [ops.fp8_rows(_x(T, H, cuda_device, i)) for i in range(2)]
    want = []
    for r in rows:
        w, y = torch.empty((T, H), device=cuda_device), torch.empty((3, H), dtype=BF16, device=cuda_device)
        ops.fp8_rows_read(*r, w)
        torch.cuda.synchronize()
        ops.add_rmsnorm(resid.clone(), None, w[-1], y, 1e-6)
        want.append(ops.fp8_rows(y))
    torch.cuda.synchronize()
    for i in [0, 1] * 6:
        ops.fp8_rows_read(*rows[i], made)
        got = ops.add_rmsnorm_fp8(resid, None, made[-1], 1e-6)
        assert torch.equal(got.scales, want[i].scales)
        assert torch.equal(got.codes.view(torch.uint8), want[i].codes.view(torch.uint8))


@pytest.mark.parametrize("act", [dict(), dict(activation="clamped", limit=1.5, slope=1.7, up_offset=1.0)])
@pytest.mark.parametrize("M,kw", [(6, {}), (70, {}), (300, {}), (6, dict(split=1)), (8, dict(split=2)), (20, dict(split=3)),
                                  (300, dict(tile=-1, split=2)), (300, dict(tile=-1, split=1)), (300, dict(tile=64))])
def test_gated_rows_that_are_not_finite(cuda_device, M, kw, act):
    """A row with an infinity or a NaN is NaN behind either activation, by every kernel; the others are what they were."""
    from binfer_b200.csrc import ops
    x, w = _x(M, 1024, cuda_device, M), ops.fp8_weight(_w((400, 1024), cuda_device), True)
    a, b = (torch.empty((M, 200), dtype=BF16, device=cuda_device) for _ in range(2))
    ops.fp8_linear(x, w, a, **act, **kw)
    assert torch.isfinite(a).all()
    x[1, 7], x[4, 900], x[5, 1023] = float("inf"), float("nan"), float("-inf")
    ops.fp8_linear(x, w, b, **act, **kw)
    bad = torch.tensor([1, 4, 5], device=cuda_device)
    assert torch.isnan(b[bad]).all()
    b[bad] = a[bad]
    assert torch.equal(a, b)


@pytest.mark.parametrize("tile", [0, 16, -1])
def test_experts_rows_that_are_not_finite(cuda_device, tile):
    from binfer_b200.csrc import ops
    x, w = _x(90, 256, cuda_device, 1), ops.fp8_weight(_w((3, 200, 256), cuda_device), True)
    starts, out = torch.tensor([0, 20, 21, 90], dtype=torch.int32, device=cuda_device), torch.empty((90, 100), dtype=BF16,
                                                                                                   device=cuda_device)
    x[20, 3] = x[89, 255] = float("nan")
    ops.fp8_experts(x, w, starts, out, activation="clamped", limit=2.0, up_offset=1.0, tile=tile)
    assert torch.isnan(out[[20, 89]]).all() and torch.isfinite(out[:20]).all() and torch.isfinite(out[21:89]).all()


def _scaled(dev, M, K, N, gated, sx, sw, seed=0):
    """Rows and a weight of codes of every size, zeros among them, with the scales 2^sx[t] and 2^sw[t] of their groups of
    columns, up to a factor of two."""
    from binfer_b200.csrc import ops
    g = torch.Generator(dev).manual_seed(seed)
    T, B = K // 128, -(-N // 128) * (2 if gated else 1)

    def codes(n):
        c = torch.randint(0, 0x7f, (n, K), generator=g, device=dev, dtype=torch.uint8)
        return (c | (torch.randint(0, 2, c.shape, generator=g, device=dev, dtype=torch.uint8) << 7)).view(E4M3)

    def scales(n, e):
        e = torch.tensor(e, dtype=F64, device=dev)
        return (torch.exp2(e) * (1 + torch.rand((n, T), generator=g, device=dev, dtype=F64))).to(F32)
    x = ops.Fp8Rows(codes(M), scales(M, sx).t().contiguous())
    return x, ops.Fp8Weight(codes((2 if gated else 1) * N), scales(B, sw), gated)


def _by_hand(x, w, gated):
    """The product in 64 bits of rows that are in 8 bits (P8.product's sums and bounds)."""
    a = P8.dense(x.codes.to(F32).to(F64), x.scales.t(), 1)
    b = P8.dense(w.codes.to(F32).to(F64), w.scales, 128, gated)
    return a @ b.t(), (a.abs() @ b.abs().t()) * ((131 + x.scales.shape[0]) * 2.0 ** -23)


@pytest.mark.parametrize("kw", [dict(tile=16), dict(tile=16, split=3), dict(tile=32, split=1), dict(tile=64),
                                dict(tile=-1, split=1), dict(tile=-1, split=2), dict()])
@pytest.mark.parametrize("M", [1, 7, 61, 300])
@pytest.mark.parametrize("sx,sw", [([-70] * 6, [-69] * 6), ([-99] * 6, [-60] * 6), ([-65, -20, -70, -100, -66, -68], [-66] * 6),
                                   ([-100] * 6, [-30, -27, -26, -25, -24, -23]), ([70] * 6, [48] * 6)])
def test_scales_whose_product_is_no_float(cuda_device, M, kw, sx, sw):
    """Results that a float has room for, of scales whose product it has none for (or only some of its bits): 131
    where P8.product has 130, for one more rounding a group; results below a float's smallest step, 2^-149, are off
    by a step a group more."""
    from binfer_b200.csrc import ops
    for N in (130, 640):
        x, w = _scaled(cuda_device, M, 768, N, False, sx, sw, M + N)
        out = torch.full((M, N), 9.0, dtype=F32, device=cuda_device)
        ops.fp8_linear(x, w, out, **kw)
        ref, off = _by_hand(x, w, False)
        # (no partial sum is above the sum of the sizes; a result above all floats is infinite, or NaN where partial
        # sums of both signs are)
        fits, above = off / ((131 + 6) * 2.0 ** -23) < 2.0 ** 127, ref.abs() - off >= 2.0 ** 128
        assert (fits | above).float().mean() > 0.5 and not torch.isfinite(out[above]).any()
        _check(out[fits], ref[fits], off[fits] + 7 * 2.0 ** -149)


@pytest.mark.parametrize("kw", [dict(tile=16), dict(tile=16, split=2), dict(tile=32), dict(tile=64), dict(tile=-1, split=1),
                                dict(tile=-1, split=2)])
@pytest.mark.parametrize("M", [3, 200])
@pytest.mark.parametrize("sx,sw", [(80, 70), (63, 66)])
def test_scales_whose_product_is_too_large(cuda_device, M, kw, sx, sw):
    """Sums that are not zero times a product above all floats: infinity, or a float where the sum is small.  (Each row
    has one code that is not zero: its results are one product each.  Codes of 2^-9 at least: 2^150 times them is above
    the floats; of 1.375 2^-5 and 1.625 2^-4 at most: 2^131 times them is not.)"""
    from binfer_b200.csrc import ops
    N, K = 200, 256
    x, w = _scaled(cuda_device, M, K, N, False, [sx, -3], [sw, 2])
    one = torch.zeros((M, K), dtype=torch.uint8, device=cuda_device)
    one[:, 5] = torch.arange(M, device=cuda_device) % 20          # codes of 0 to 1.5 * 2^-6 in the first group
    w.codes.view(torch.uint8)[:, 5] = (torch.arange(N, device=cuda_device) % 30).to(torch.uint8)
    x = ops.Fp8Rows(one.view(E4M3), x.scales)
    ref, _ = _by_hand(x, w, False)
    out = torch.empty((M, N), dtype=F32, device=cuda_device)
    ops.fp8_linear(x, w, out, **kw)
    inf = ref.abs() >= 2.0 ** 128
    near = (ref.abs() > 2.0 ** 128 * (1 - 2.0 ** -20)) & (ref.abs() < 2.0 ** 128 * (1 + 2.0 ** -20))
    assert not near.any() and (ref == 0).any() and torch.equal(inf, (ref != 0) if sx == 80 else inf & False)
    assert torch.isinf(out[inf & ~near]).all()
    rest = ~inf & ~near
    # (two scales and a factor: at most three roundings, and the multiply-add's)
    assert ((out.to(F64) - ref).abs()[rest] <= ref.abs()[rest] * (4 * 2.0 ** -24)).all()


def test_a_row_s_scales_do_not_touch_the_others(cuda_device):
    from binfer_b200.csrc import ops
    for M, kw in ((7, {}), (7, dict(split=2)), (40, dict(tile=64)), (300, dict(tile=-1, split=1))):
        x, w = _scaled(cuda_device, M, 512, 150, True, [-3, -5, -2, -4], [-6] * 4, M)
        a, b = (torch.empty((M, 150), dtype=BF16, device=cuda_device) for _ in range(2))
        ops.fp8_linear(x, w, a, **kw)
        x.scales[1, 2], x.scales[3, 0] = 2.0 ** -127, float("nan")
        x.scales[0, 4] = 2.0 ** 127
        ops.fp8_linear(x, w, b, **kw)
        keep = torch.ones(M, dtype=torch.bool, device=cuda_device)
        keep[[0, 2, 4]] = False
        assert torch.isnan(b[0]).all() and not torch.equal(a[2], b[2])
        assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,kw", [(1, {}), (5, {}), (5, dict(tile=16, split=2)), (40, dict(tile=32)), (40, dict(tile=64)),
                                  (290, dict(tile=-1, split=1)), (290, dict(tile=-1, split=2))])
def test_tiny_rows_and_weights(cuda_device, M, kw, gated):
    """Numbers whose scales' product is below the floats of full precision, from their bfloat16 rows on and with a last
    group that ends inside a word.  (One rounding a group more than P8.product counts.)"""
    from binfer_b200.csrc import ops
    K, N = 333, 200
    x, w = (_x(M, K, cuda_device, M).to(F32) * 2.0 ** -60).to(BF16), _w(((1 + gated) * N, K), cuda_device, M)
    w[:N] *= 2.0 ** -60
    if gated:
        w[N:] *= 2.0 ** 110
    out = torch.empty((M, N), dtype=BF16 if gated else F32, device=cuda_device)
    ops.fp8_linear(x, ops.fp8_weight(w, gated), out, **kw)
    ref, off = P8.product(x, *P8.hold_weight(w, gated), gated)
    assert ref.abs().max() > 2.0 ** -125
    _check(out, ref, off * (134 / 133) + 2.0 ** -148)


@pytest.mark.parametrize("tile", [0, 16, 64, -1])
def test_experts_with_tiny_numbers(cuda_device, tile):
    """An expert's weight and some rows so small that the scales' products are below the floats of full precision; the
    other experts, and the rows beside, as they are without them."""
    from binfer_b200.csrc import ops
    counts, K, N = [30, 0, 300, 7], 300, 136
    starts, R = torch.tensor([0, 30, 30, 330, 337], dtype=torch.int32, device=cuda_device), 337
    x, w = _x(R, K, cuda_device, 1), _w((4, N, K), cuda_device, 1)
    row_w = torch.rand(R, device=cuda_device) + 0.5
    a, b = (torch.empty((R, N), dtype=F32, device=cuda_device) for _ in range(2))
    ops.fp8_experts(x, ops.fp8_weight(w), starts, a, row_w=row_w, tile=tile)
    w[2] *= 2.0 ** -58
    small = torch.arange(R, device=cuda_device) % 3 == 1
    x[small] *= 2.0 ** -58
    ops.fp8_experts(x, ops.fp8_weight(w), starts, b, row_w=row_w, tile=tile)
    for e, (i, j) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
        if j > i:
            ref, off = P8.product(x[i:j], *P8.hold_weight(w[e]))
            k = row_w[i:j, None].to(F64)
            _check(b[i:j], ref * k, (off * (134 / 133) + ref.abs() * 2.0 ** -23) * k + 2.0 ** -148)
    rest = ~small
    rest[30:330] = False
    assert torch.equal(a[rest], b[rest]) and b[small].any()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,groups,N,fits", [
    # clusters of eight: 1 to 5 groups a CTA, in one or two turns
    (1, 32, 300, True), (2, 32, 300, True), (3, 40, 128, True), (5, 32, 130, True), (8, 40, 300, True),
    # a tile for every SM: a CTA has all groups, in one to four turns of 32, 16, 8 or 4 ...
    (1, 32, 19200, True), (2, 20, 19200, True), (3, 32, 19200, True), (4, 9, 19200, True), (7, 16, 19200, True),
    (8, 12, 19200, True), (8, 16, 19200, True),
    # ... five, or more than there is room for beside four stages of the weight; more than eight rows
    (8, 17, 19200, False), (4, 33, 19200, False), (1, 48, 19200, False), (9, 32, 300, False)])
def test_rows_that_stay_in_the_product_s_kernel(cuda_device, monkeypatch, M, groups, N, fits, gated):
    """One kernel where the rows fit and two elsewhere, with the same results; an odd last group either way."""
    from binfer_b200.csrc import ops
    if gated and N == 19200:
        N = 9600
    for K in (groups * 128, groups * 128 - 37):
        x, w = _x(M, K + 3, cuda_device, M)[:, 3:], ops.fp8_weight(_w(((1 + gated) * N, K), cuda_device), gated)
        for rows in (x, x.contiguous()):
            outs = []
            for resident in (True, False):
                monkeypatch.setattr(ops, "FP8_RESIDENT", resident)
                out = torch.full((M, N), float("nan"), dtype=BF16, device=cuda_device)
                before = ops.launches()
                ops.fp8_linear(rows, w, out)
                assert ops.launches() - before == (1 if resident and fits else 2)
                outs.append(out)
            assert torch.equal(*outs)
    assert ops.error_word(cuda_device).item() == 0


@pytest.mark.parametrize("R", [40, 900])
def test_captured_experts_with_other_rows_each_time(cuda_device, R):
    """A captured call replayed with other rows, other shares of the experts and other weights of the rows."""
    from binfer_b200.csrc import ops
    E, K, N = 6, 384, 200
    w = _w((E, 2 * N, K), cuda_device)
    held, x = ops.fp8_weight(w, True), _x(R, K, cuda_device)
    starts, row_w = torch.zeros(E + 1, dtype=torch.int32, device=cuda_device), torch.ones(R, device=cuda_device)
    out = torch.empty((R, N), dtype=BF16, device=cuda_device)
    ops.fp8_experts(x, held, starts, out, row_w=row_w)
    torch.cuda.synchronize()
    gc.collect()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.fp8_experts(x, held, starts, out, row_w=row_w)
    for i, cuts in enumerate(([0, 0, 1, 1, 1, 1, 1], [0, .1, .1, .5, .9, .9, 1], [.2, .3, .4, .5, .6, .7, .8],
                              [1, 1, 1, 1, 1, 1, 1], [0, 0, 0, 0, 0, 0, 1])):
        s = [round(c * R) for c in cuts]
        x.copy_(_x(R, K, cuda_device, 20 + i))
        row_w.copy_(torch.rand(R, device=cuda_device))
        starts.copy_(torch.tensor(s, dtype=torch.int32))
        out.fill_(9.0)
        g.replay()
        for e, (a, b) in enumerate(zip(s, s[1:])):
            if b > a:
                ref, off = P8.product(x[a:b], *P8.hold_weight(w[e], True), True)
                k = row_w[a:b, None].to(F64)
                _check(out[a:b], ref * k, (off + ref.abs() * 2.0 ** -23) * k)
        assert (out[:s[0]] == 9).all() and (out[s[-1]:] == 9).all()


@pytest.mark.parametrize("M", [1, 8])
def test_one_kernel_in_a_graph_too(cuda_device, M):
    """Which kernels a call takes depends on its sizes, not on how it is launched."""
    from binfer_b200.csrc import ops
    w = _w((300, 1024), cuda_device)
    held, x = ops.fp8_weight(w), _x(M, 1024, cuda_device)
    out, eager = (torch.empty((M, 300), dtype=F32, device=cuda_device) for _ in range(2))
    ops.fp8_linear(x, held, out)
    torch.cuda.synchronize()
    gc.collect()
    g, before = torch.cuda.CUDAGraph(), ops.launches()
    with torch.cuda.graph(g):
        ops.fp8_linear(x, held, out)
    assert ops.launches() - before == 1
    for seed in range(3):
        x.copy_(_x(M, 1024, cuda_device, 30 + seed))
        g.replay()
        ops.fp8_linear(x, held, eager)
        assert torch.equal(out, eager)
        _check(out, *P8.product(x, *P8.hold_weight(w)))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,kw", [(6, {}), (6, dict(split=1, tile=32)), (100, dict(tile=64)), (300, dict(tile=-1, split=1)),
                                  (300, dict(tile=-1, split=2))])
def test_rows_of_zeros_beside_tiny_weights(cuda_device, M, kw, gated):
    """Zeros' scale is the smallest there is, so that its product with a small weight's is no float: such rows, and groups
    of zeros within others, count as zeros, and results of the others are what they are."""
    from binfer_b200.csrc import ops
    x, w = _x(M, 640, cuda_device, M), _w(((1 + gated) * 200, 640), cuda_device, M)
    w[:, 128:256] *= 2.0 ** -40
    x[::2] = 0
    x[1::4, 128:256] = 0
    out = torch.empty((M, 200), dtype=BF16 if gated else F32, device=cuda_device)
    ops.fp8_linear(x, ops.fp8_weight(w, gated), out, **kw)
    _check(out, *P8.product(x, *P8.hold_weight(w, gated), gated))
    assert not out[::2].any() and out[1::2].any(dim=1).all()

"""Weights in 8 bits: the restatement, and what the operators refuse before anything reaches a GPU."""
import copy
import pickle

import pytest
import torch

import fp8_plain as P8

BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn


@pytest.fixture
def ops():
    from binfer_b200.csrc import ops
    return ops


def test_values_are_e4m3s():
    v = P8.values()
    assert v[0] == 0 and v[126] == 448 and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6 and bool((v[1:] > v[:-1]).all())


def test_nearest_ties_to_even_codes():
    one = torch.ones(1)
    for x, want in ((1.0625, 1.0), (1.1875, 1.25), (1.0625 + 2.0 ** -20, 1.125), (2.0 ** -10, 0.0),
                    (3 * 2.0 ** -10, 2.0 ** -8), (447.9, 448.0), (432.0, 448.0), (431.9, 416.0), (-1.1875, -1.25)):
        assert P8.nearest(torch.tensor([x]), one).item() == want


def test_nearest_is_the_nearest():
    g = torch.Generator().manual_seed(1)
    x, s = torch.randn(4000, generator=g), torch.rand(4000, generator=g) * 0.01 + 0.01
    got, v = P8.nearest(x, s), P8.values()
    v = torch.cat([-v.flip(0), v])
    best = (x.to(F64)[:, None] - v * s.to(F64)[:, None]).abs().amin(dim=1)
    assert torch.equal((x.to(F64) - got * s.to(F64)).abs(), best)


def test_hold_groups():
    x = torch.randn(3, 300)
    x[1, 128:256] = 0
    x[2, 256:] = float("inf")
    v, s = P8.hold(x, 1)
    assert s.shape == (3, 3) and s[1, 1] == 2.0 ** -100 and torch.isnan(s[2, 2])
    assert torch.isnan(v[2, 256:]).all() and not torch.isnan(v[2, :256]).any() and not v[1, 128:256].any()


# --------------------------------------------------------------------------- refusals
def _codes(*shape):
    return torch.zeros(shape).to(E4M3)


def test_weight_object(ops):
    w = ops.Fp8Weight(_codes(300, 200), torch.ones(3, 2))
    # rows of 200 bytes do not lie on 16-byte boundaries: they are laid out anew
    assert w.codes.stride() == (208, 1) and w.features == 300 and w.rows == 300 and w.K == 200 and not w.experts
    codes = _codes(300, 256)
    assert ops.Fp8Weight(codes, torch.ones(3, 2)).codes is codes
    g = ops.Fp8Weight(_codes(300, 200), torch.ones(4, 2), gated=True)
    assert g.features == 150 and g.rows == 300
    e = ops.Fp8Weight(_codes(5, 300, 200), torch.ones(5, 3, 2))
    assert e.experts == 5 and e.codes.stride() == (300 * 208, 208, 1)
    odd = (torch.randn(4, 33) * 3).to(E4M3)
    assert torch.equal(ops.Fp8Weight(odd, torch.ones(1, 1)).codes.view(torch.uint8), odd.view(torch.uint8))


@pytest.mark.parametrize("codes,scales,gated", [
    (torch.zeros(300, 200), torch.ones(3, 2), False),
    (_codes(200), torch.ones(1, 2), False),
    (_codes(0, 200), torch.ones(0, 2), False),
    (_codes(2, 2, 300, 200), torch.ones(2, 2, 3, 2), False),
    (_codes(300, 200), torch.ones(2, 2), False),
    (_codes(300, 200), torch.ones(3, 2), True),
    (_codes(301, 200), torch.ones(4, 2), True),
    (_codes(300, 200), torch.ones(3, 2, dtype=F64), False),
    (_codes(300, 200), torch.ones(2, 3).t(), False),
    (_codes(513, 2, 8), torch.ones(513, 1, 1), False),
])
def test_weight_object_refuses(ops, codes, scales, gated):
    with pytest.raises(ops.KernelError):
        ops.Fp8Weight(codes, scales, gated=gated)


def test_no_cpu_path(ops):
    x, out = torch.zeros(2, 200, dtype=BF16), torch.zeros(2, 300, dtype=BF16)
    w = ops.Fp8Weight(_codes(300, 200), torch.ones(3, 2))
    for call in (lambda: ops.fp8_rows(x), lambda: ops.fp8_weight(x),
                 lambda: ops.fp8_rows_read(w.codes, torch.ones(2, 300), torch.zeros(300, 200)),
                 lambda: ops.fp8_weight_read(w, torch.zeros(300, 200))):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(2, 200)), dict(x=torch.zeros(2, 201, dtype=BF16)), dict(x=torch.zeros(200, dtype=BF16)),
    dict(x=torch.zeros(200, 2, dtype=BF16).t()), dict(out=torch.zeros(2, 300, dtype=torch.float16)),
    dict(out=torch.zeros(3, 300, dtype=BF16)), dict(out=torch.zeros(2, 299, dtype=BF16)),
    dict(out=torch.zeros(300, 2, dtype=BF16).t()), dict(tile=48), dict(split=9), dict(split=-1),
])
def test_linear_refuses(ops, change):
    args = dict(x=torch.zeros(2, 200, dtype=BF16), w=ops.Fp8Weight(_codes(300, 200), torch.ones(3, 2)),
                out=torch.zeros(2, 300, dtype=BF16))
    args.update(change)
    with pytest.raises(ops.KernelError) as e:
        ops.fp8_linear(**args)
    assert "CUDA" not in str(e.value)


def test_gated_linear_refuses(ops):
    x, w = torch.zeros(2, 200, dtype=BF16), ops.Fp8Weight(_codes(300, 200), torch.ones(4, 2), gated=True)
    with pytest.raises(ops.KernelError, match="bfloat16 result"):
        ops.fp8_linear(x, w, torch.zeros(2, 150))
    with pytest.raises(ops.KernelError, match="activations"):
        ops.fp8_linear(x, w, torch.zeros(2, 150, dtype=BF16), activation="gelu_tanh")


@pytest.mark.parametrize("change", [
    dict(starts=torch.zeros(6)), dict(starts=torch.zeros(5, dtype=torch.int32)),
    dict(starts=torch.zeros(12, dtype=torch.int32)[::2]), dict(row_w=torch.zeros(3)),
    dict(row_w=torch.zeros(2, dtype=BF16)), dict(row_w=torch.zeros(4)[::2]),
    dict(w=lambda ops: ops.Fp8Weight(_codes(300, 200), torch.ones(3, 2))),
])
def test_experts_refuse(ops, change):
    args = dict(x=torch.zeros(2, 200, dtype=BF16), w=ops.Fp8Weight(_codes(5, 300, 200), torch.ones(5, 3, 2)),
                starts=torch.zeros(6, dtype=torch.int32), out=torch.zeros(2, 300, dtype=BF16))
    args.update({k: v(ops) if callable(v) else v for k, v in change.items()})
    with pytest.raises(ops.KernelError) as e:
        ops.fp8_experts(**args)
    assert "CUDA" not in str(e.value)
    with pytest.raises(ops.KernelError, match="has experts"):
        ops.fp8_linear(args["x"], ops.Fp8Weight(_codes(5, 300, 200), torch.ones(5, 3, 2)), args["out"])


@pytest.mark.parametrize("bad", [torch.zeros(2, 8, dtype=torch.float16), torch.zeros(8, dtype=BF16),
                                 torch.zeros(8, 2, dtype=BF16).t(), torch.zeros(2, 0, dtype=BF16)])
def test_rows_and_weight_refuse(ops, bad):
    for fn in (ops.fp8_rows, ops.fp8_weight):
        with pytest.raises(ops.KernelError) as e:
            fn(bad)
        assert "CUDA" not in str(e.value)


def test_read_refuses(ops):
    codes, scales = _codes(4, 32), torch.ones(1, 4)
    for c, s, o in ((codes.view(torch.uint8), scales, torch.zeros(4, 32)), (codes, torch.ones(4, 1), torch.zeros(4, 32)),
                    (codes, scales, torch.zeros(4, 31)), (codes[:, 1:], scales, torch.zeros(4, 31)),
                    (codes, scales.to(F64), torch.zeros(4, 32)), (codes, scales, torch.zeros(4, 32, dtype=F64))):
        with pytest.raises(ops.KernelError) as e:
            ops.fp8_rows_read(c, s, o)
        assert "CUDA" not in str(e.value)
    w = ops.Fp8Weight(_codes(4, 32), torch.ones(1, 1))
    with pytest.raises(ops.KernelError, match="shape"):
        ops.fp8_weight_read(w, torch.zeros(4, 31))


def test_rows_in_8_bits_refused(ops):
    w, out = ops.Fp8Weight(_codes(300, 256), torch.ones(3, 2)), torch.zeros(2, 300, dtype=BF16)
    for codes, scales in ((_codes(2, 256), torch.ones(2, 3)), (_codes(2, 256), torch.ones(2, 2, dtype=F64)),
                          (_codes(2, 255), torch.ones(2, 2)), (_codes(2, 256).view(torch.uint8), torch.ones(2, 2)),
                          (_codes(2, 512)[:, 1:257], torch.ones(2, 2)), (_codes(256, 2).t(), torch.ones(2, 2))):
        with pytest.raises(ops.KernelError) as e:
            ops.fp8_linear(ops.Fp8Rows(codes, scales), w, out)
        assert "CUDA" not in str(e.value)


def test_norm_into_8_bits_refuses(ops):
    ok = dict(resid=torch.zeros(2, 64), delta=torch.zeros(2, 64, dtype=BF16), weight=torch.ones(64), eps=1e-6)
    for change in (dict(resid=torch.zeros(2, 60), delta=None, weight=torch.ones(60)), dict(weight=torch.ones(32)),
                   dict(delta=torch.zeros(2, 64)), dict(delta=torch.zeros(3, 64, dtype=BF16)),
                   dict(resid=torch.zeros(2, 64, dtype=BF16)), dict(resid=torch.zeros(64)),
                   dict(resid=torch.zeros(130)[1:129].view(2, 64)),
                   dict(resid=torch.zeros(2, 8200), delta=None, weight=torch.ones(8200))):
        with pytest.raises(ops.KernelError) as e:
            ops.add_rmsnorm_fp8(**dict(ok, **change))
        assert "CUDA" not in str(e.value)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.add_rmsnorm_fp8(**ok)


def test_copies_have_tensors_of_their_own(ops):
    w = ops.Fp8Weight((torch.randn(300, 200) * 3).to(E4M3), torch.rand(4, 2), gated=True)
    for c in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert c.gated and c.features == 150 and c.K == 200
        assert c.codes.data_ptr() != w.codes.data_ptr() and c.scales.data_ptr() != w.scales.data_ptr()
        assert c._held == (c.codes.data_ptr(), 208, c.scales.data_ptr())
        assert torch.equal(c.codes.view(torch.uint8), w.codes.view(torch.uint8)) and torch.equal(c.scales, w.scales)
    c = copy.copy(w)
    assert c.codes is w.codes and c.scales is w.scales and c._held == w._held
    for name in ("codes", "scales"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name).clone())


def test_results_in_rows_that_share_memory_refused(ops):
    w, x = ops.Fp8Weight(_codes(300, 200), torch.ones(3, 2)), torch.zeros(2, 200, dtype=BF16)
    for fn in (lambda out: ops.fp8_linear(x, w, out),
               lambda out: ops.fp8_linear(ops.Fp8Rows(_codes(2, 208)[:, :200], torch.ones(2, 2)), w, out)):
        for out in (torch.zeros(300, dtype=BF16).expand(2, 300),
                    torch.zeros(700, dtype=BF16).as_strided((2, 300), (299, 1))):
            with pytest.raises(ops.KernelError, match="of their own"):
                fn(out)
    with pytest.raises(ops.KernelError, match="share memory"):
        ops.fp8_rows_read(_codes(4, 32), torch.ones(1, 4), torch.zeros(32).expand(4, 32))
    with pytest.raises(ops.KernelError, match="share memory"):
        ops.fp8_weight_read(w, torch.zeros(200).expand(300, 200))


def test_no_fused_epilogue_takes_a_weight_in_8_bits(ops):
    """The products with the next norm in their epilogue leave such a weight to the plain product."""
    from binfer_b200.parts.linear import linear_add_norm, linear_add_tanh
    x, w = torch.zeros(2, 256, dtype=BF16), ops.Fp8Weight(_codes(128, 256), torch.ones(1, 2))
    resid, norm_w = torch.zeros(2, 128), torch.ones(128)
    assert linear_add_norm(x, w, resid, norm_w, 1e-6) is None
    for assign in (False, True):
        assert linear_add_tanh(x, w, resid, None, 0.5, norm_w, None, assign=assign) is None


def test_weights_whose_memory_went_elsewhere_are_refused(ops):
    """The addresses taken when the weight was made are not read where its tensors have others by now."""
    for change in (lambda w: setattr(w.codes, "data", w.codes.clone()), lambda w: setattr(w.scales, "data", w.scales.clone()),
                   lambda w: w.codes.untyped_storage().resize_(0), lambda w: w.scales.set_(torch.ones(3, 2))):
        w = ops.Fp8Weight(_codes(300, 208), torch.ones(3, 2))
        x, out = torch.zeros(2, 208, dtype=BF16), torch.zeros(2, 300, dtype=BF16)
        for call in (lambda: ops.fp8_linear(x, w, out), lambda: ops.fp8_weight_read(w, torch.zeros(300, 208))):
            with pytest.raises(ops.KernelError, match="CUDA"):
                call()
        change(w)
        for call in (lambda: ops.fp8_linear(x, w, out), lambda: ops.fp8_weight_read(w, torch.zeros(300, 208))):
            with pytest.raises(ops.KernelError, match="elsewhere"):
                call()


def test_more_rows_than_the_kernels_count_are_refused(ops):
    n = 2 ** 31 - 100
    x, y = torch.zeros(1, 1, dtype=BF16).expand(n, 1), torch.zeros(1, 1).expand(n, 1)
    w = ops.Fp8Weight(_codes(1, 1), torch.ones(1, 1))
    e = ops.Fp8Weight(_codes(2, 1, 1), torch.ones(2, 1, 1))
    for call in (lambda: ops.fp8_rows(x), lambda: ops.fp8_rows(y), lambda: ops.fp8_weight(x), lambda: ops.fp8_weight(y),
                 lambda: ops.fp8_linear(x, w, x), lambda: ops.fp8_experts(x, e, torch.zeros(3, dtype=torch.int32), x),
                 lambda: ops.fp8_rows_read(_codes(1, 1).expand(n, 1), torch.ones(1, 1).expand(1, n), y)):
        with pytest.raises(ops.KernelError, match="at most"):
            call()

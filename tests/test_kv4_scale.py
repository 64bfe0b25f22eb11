"""How large a scale the attention kernels over a cache in 4 bits take."""
import math

import pytest
import torch

BF16, I32 = torch.bfloat16, torch.int32


def _i(*shape):
    return torch.zeros(shape, dtype=I32)


@pytest.mark.parametrize("scale", [2.0 ** 41, -2.0 ** 41, 2.0 ** 80, math.inf, -math.inf, math.nan])
def test_a_scale_beyond_what_the_products_take_is_refused(scale):
    from binfer_b200.csrc import ops
    c, k = ops.kv4_cache(3, 1, 16, 64, "cpu"), torch.zeros((2, 64), dtype=BF16)
    with pytest.raises(ops.KernelError, match="scale"):
        ops.kv4_decode_attention(k, c, None, 2, _i(2), _i(2), _i(1, 2), k, 1, 1, 64, None, scale, _i(1))
    with pytest.raises(ops.KernelError, match="scale"):
        ops.kv4_prefill_attention(k, c, _i(1, 4), 1, 2, _i(1, 2), k, 1, 1, 64, None, scale, _i(1), 64, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("key_size,query_size", [(0, -40), (-40, 0), (-20, -20), (8, -48), (-100, 60)])
def test_the_largest_scale(cuda_device, d, sign, key_size, query_size):
    """Scores of ordinary size out of numbers whose products are 2^-40."""
    import kv4_plain as K4
    import kv4_units as U
    from binfer_b200.csrc import ops
    from test_kv4_gpu import Cache, _attention, _queries
    nh, nkv, n = 4, 2, 600
    c = Cache([n], nkv, d, 16, cuda_device)
    c.k[0] = U.keys(n, nkv, d, cuda_device, 1) * (d ** -0.5 * 2.0 ** key_size)
    c.v[0] = U.values(n, nkv, d, cuda_device, 2)
    ops.kv4_store(c.k[0].flatten(1), c.v[0].flatten(1), c.slots[0], c.cache, c.err)
    q = _queries(1, nh, d, cuda_device) * 2.0 ** query_size
    out = torch.full_like(q, math.nan)
    scale = sign * 2.0 ** 40
    _attention(c, q, out, nh, [(0, 1, n - 1)], True, None, 0, scale)
    ref, allowed = U.attend(q.view(1, nh, d).double(), *c.held(0), torch.tensor([n - 1], device=q.device), None, 0, scale)
    U.check(out, ref, allowed)
    assert int(c.err.item()) == 0

"""That the bound of ``kv4_units`` sees a unit of keys that is left out or counted twice."""
import pytest
import torch

import kv4_plain as K4
import kv4_units as U


@pytest.mark.parametrize("n,nh,nkv,d", [(33, 3, 3, 64), (700, 4, 1, 128), (1500, 5, 1, 64), (1500, 2, 2, 256),
                                        (40000, 4, 1, 128)])
def test_a_unit_left_out_or_counted_twice_is_seen(n, nh, nkv, d):
    k, v = K4.held(U.keys(n, nkv, d, "cpu", n)), K4.held(U.values(n, nkv, d, "cpu", n + 1))
    q = torch.randn((1, nh, d), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(torch.float64)
    at = torch.tensor([n - 1])
    ref, allowed = U.attend(q, k, v, at, None, 0, d ** -0.5)
    # (whole units: the one key of a last one may weigh less than half a step)
    units = range(n // 16) if n < 5000 else range(0, n // 16, 97)
    for u in units:
        for times in (0.0, 2.0):
            weight = torch.ones(n, dtype=torch.float64)
            weight[16 * u:16 * u + 16] = times
            got, _ = U.attend(q, k, v, at, None, 0, d ** -0.5, weight)
            assert (U.off(got, ref, nkv) > allowed).all(), (u, times, U.off(got, ref, nkv) / allowed)
    rounded = ref.to(torch.bfloat16)
    U.check(rounded, ref, allowed)

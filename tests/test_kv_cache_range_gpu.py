"""The 4-bit cache at the ends of its types' ranges: half steps beside values that vanish in a difference, rows of queries and
value scales whose sizes lie far apart. Bounds are those of the other tests of the cache (derived there); where what an outlier
adds to the answer is itself negligible, its size does not enter them."""
import numpy as np
import pytest
import torch

from ferro_kittens_b200 import kv_cache

from kv_cache_plain import key_nibble, value_nibble
from test_kv_cache_gpu import _by_slot, _expect_rows

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- writing

@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_steps_beside_values_that_vanish(device, dtype, group):
    """Rows whose smallest value lies half a step below zero, of a tiny value that the difference rounds away, and beside it in the
    same eight channels one a little larger that it does not: below and above the border, each on its own side."""
    lost, kept = (2.0 ** -30, 2.0 ** -20) if dtype == torch.bfloat16 else (2.0 ** -24, 2.0 ** -10)
    unit = 1.0 if dtype == torch.bfloat16 else 64.0  # half a step: large beside fp16's smallest value
    rng = np.random.default_rng(0)
    rows = []
    for below in (0, 1, 3, 6, 9, 14):  # codes of zero less a little
        for channel in range(8):
            x = rng.integers(-2 * below, 2 * (14 - below) + 1, 128).astype(np.float64) * unit
            for g in range(0, 128, group):
                x[g + 8], x[g + 9] = -(2 * below + 1) * unit, (30 - (2 * below + 1)) * unit
                at = g + 16 + rng.permutation(8)
                x[g + 16 + channel] = -lost
                others = [i for i in at if i != g + 16 + channel]
                x[others[0]], x[others[1]], x[others[2]] = kept, lost, -kept
            rows.append(x)
    x = torch.from_numpy(np.array(rows)).to(dtype).view(len(rows), 1, 128)
    cache = kv_cache.new(1, len(rows), 1, 128, group, dtype, device)
    slots = torch.arange(len(rows), device=device)
    kv_cache.write(cache, x.to(device), x.flip(0).to(device), slots)
    for y, codes, params, place in ((x, cache.k_codes, cache.k_params, key_nibble), (x.flip(0), cache.v_codes, cache.v_params, value_nibble)):
        want_codes, want_params = _expect_rows(y, group, dtype, place)
        assert (want_params[..., 0] == 2 * unit).all()
        assert np.array_equal(_by_slot(params).double().numpy(), want_params)
        assert np.array_equal(_by_slot(codes).numpy(), want_codes)

"""The 4-bit cache at the ends of its types' ranges: half steps beside values that vanish in a difference, rows of queries and
value scales whose sizes lie far apart. Bounds are those of the other tests of the cache (derived there); where what an outlier
adds to the answer is itself negligible, its size does not enter them."""
import numpy as np
import pytest
import torch

from ferro_kittens_b200 import gemm, kv_cache

from kv_cache_plain import key_nibble, value_nibble
from test_kv_cache_gpu import _by_slot, _compare, _expect_rows, _random_cache, _tables

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


# ---------------------------------------------------------------- queries

@pytest.mark.parametrize("ratio,queries", [(4, 1), (12, 1), (4, 3)])
@pytest.mark.parametrize("dtype,far,size,keys", [(torch.bfloat16, 3e38, 1.0, 1.0), (torch.bfloat16, 2.0 ** 60, 1.0, 1.0),
                                                 (torch.bfloat16, 2.0 ** 40, 2.0 ** -20, 2.0 ** 20), (torch.float16, 6e4, 2.0 ** -11, 1.0),
                                                 (torch.float16, 6e4, 2.0 ** -14, 64.0)])
def test_a_row_keeps_its_precision_beside_rows_of_any_size(device, dtype, far, size, keys, ratio, queries):
    """Every other query head is `far` larger than the rest, whose scores are ordinary (small queries, large keys)."""
    kv_heads, heads = 2, 2 * ratio
    cache = _random_cache(device, 30, 16, kv_heads, 128, 64, dtype, 12)
    cache.k_params.mul_(keys)
    table, lengths = _tables(device, 3, 10, 30), torch.tensor([150, 9, 64], dtype=torch.int32, device=device)
    q = (torch.randn(3, queries, heads, 128, device=device) * 1.5 * size).to(dtype)
    large = torch.arange(heads, device=device) % 2 == 1
    bad = q.clone()
    bad[:, :, large] = (far * (torch.rand(3, queries, ratio, 128, device=device) - 0.5).sign()).to(dtype)
    status = gemm.new_status(device)
    out, lse = kv_cache.attend(bad, cache, lengths, table, status=status)
    gemm.check_status(status)
    clean, clean_lse = kv_cache.attend(q, cache, lengths, table)
    out[:, :, large], lse[:, :, large] = clean[:, :, large], clean_lse[:, :, large]
    _compare(cache, q, lengths, table, None, None, 0, out, lse)


@pytest.mark.parametrize("ratio", [2, 6])
def test_places_of_a_batch_that_hold_no_query_may_hold_anything(device, ratio):
    """A sequence shorter than its queries: the rows before its first token see nothing, whatever lies there."""
    cache = _random_cache(device, 9, 16, 2, 128, 64, torch.bfloat16, 12)
    table, lengths = _tables(device, 3, 3, 9), torch.tensor([2, 1, 40], dtype=torch.int32, device=device)
    q = torch.randn(3, 4, 2 * ratio, 128, device=device).bfloat16()
    for value in (3.3e38, float("inf"), float("nan"), 1e-40):
        bad = q.clone()
        bad[0, :2], bad[1, :3] = value, -value
        out, lse = kv_cache.attend(bad, cache, lengths, table)
        _compare(cache, q, lengths, table, None, None, 0, out, lse)


@pytest.mark.parametrize("scale", [1e-30, 3e30, -2.0 ** 40])
def test_queries_of_one_end_of_the_range_and_a_scale_of_the_other(device, scale):
    cache = _random_cache(device, 4, 16, 1, 128, 64, torch.bfloat16, 12)
    table, lengths = _tables(device, 1, 4, 4), torch.tensor([60], dtype=torch.int32, device=device)
    q = (torch.randn(1, 1, 4, 128, device=device) * 0.1 / abs(scale)).bfloat16()
    out, lse = kv_cache.attend(q, cache, lengths, table, scale=scale)
    _compare(cache, q, lengths, table, scale, None, 0, out, lse)


def test_a_scale_of_zero_weighs_all_alike(device):
    """However large the keys are."""
    cache = _random_cache(device, 4, 16, 1, 128, 64, torch.bfloat16, 12)
    cache.k_params.mul_(2.0 ** 123)
    table, lengths = _tables(device, 1, 4, 4), torch.tensor([60], dtype=torch.int32, device=device)
    q = torch.randn(1, 1, 4, 128, device=device).bfloat16()
    out, lse = kv_cache.attend(q, cache, lengths, table, scale=0.0)
    assert torch.allclose(lse, torch.full_like(lse, float(np.log(60))), rtol=0, atol=2.0 ** -16)
    cache.k_params.mul_(2.0 ** -123)
    _compare(cache, q, lengths, table, 0.0, None, 0, out, lse)

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


# ---------------------------------------------------------------- value scales

def _ordinary(device, dtype, head_dim, group, seed, page_size=16, pages=30):
    return _random_cache(device, pages, page_size, 1, head_dim, group, dtype, seed)


@pytest.mark.parametrize("head_dim,group,dtype", [(128, 64, torch.bfloat16), (128, 32, torch.bfloat16), (64, 32, torch.bfloat16),
                                                  (128, 64, torch.float16), (64, 32, torch.float16)])
@pytest.mark.parametrize("apart", [12, 16, 20, 24, 30, 60])
@pytest.mark.parametrize("ratio", [4, 12])
def test_groups_of_a_head_whose_scales_lie_far_apart(device, head_dim, group, dtype, apart, ratio):
    """Each group of channels keeps its own precision, whatever the scales of the groups beside it."""
    cache = _ordinary(device, dtype, head_dim, group, 21)
    if dtype == torch.float16:  # what its range holds: one group near the top, the others far below
        apart = min(apart, 22)
        cache.v_params[..., 0, :].mul_(2.0 ** min(apart, 13))
        cache.v_params[..., 1:, :].mul_(2.0 ** min(13 - apart, 0))
    else:
        cache.v_params[..., -1, :].mul_(2.0 ** apart)
    table, lengths = _tables(device, 3, 10, 30), torch.tensor([150, 9, 64], dtype=torch.int32, device=device)
    q = (torch.randn(3, 1, ratio, head_dim, device=device) * 1.5).to(dtype)
    out, lse = kv_cache.attend(q, cache, lengths, table)
    _compare(cache, q, lengths, table, None, None, 0, out, lse)


def _token(table, b, j, page_size=16):
    return int(table[b, j // page_size]), 0, j % page_size


@pytest.mark.parametrize("head_dim,group", [(128, 64), (128, 128), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("apart", [10, 24, 32, 60, 100])
@pytest.mark.parametrize("count,ratio", [(1, 4), (7, 12), (40, 4)])
def test_tokens_of_far_scales_and_no_weight(device, head_dim, group, apart, count, ratio):
    """Tokens whose values are 2^apart times the others' and whose weight is e^-100 or less: the answer is the others'."""
    cache = _ordinary(device, torch.bfloat16, head_dim, group, 22)
    table, lengths = _tables(device, 2, 14, 30), torch.tensor([211, 64], dtype=torch.int32, device=device)
    q = (1.0 + torch.rand(2, 1, ratio, head_dim, device=device)).bfloat16()
    rng = np.random.default_rng(apart)
    for b, n in enumerate(lengths.tolist()):
        for j in rng.permutation(n)[:min(count, n - 4)].tolist() + ([0] if count > 1 else []):
            page, head, place = _token(table, b, j)
            cache.v_params[page, head, place] *= 2.0 ** apart
            # Keys of -16 to -15.4 in every channel: scores of -120 and less, the others' within 40 of 0.
            cache.k_params[page, head, place, :, 0], cache.k_params[page, head, place, :, 1] = 0.04, -16.0
    out, lse = kv_cache.attend(q, cache, lengths, table)
    _compare(cache, q, lengths, table, None, None, 0, out, lse)


@pytest.mark.parametrize("apart", [9, 20, 60, 100])
@pytest.mark.parametrize("ratio", [4, 12])
def test_tokens_of_far_scales_with_weight(device, apart, ratio):
    """A few tokens whose scales are far above or below the others', with a weight like theirs."""
    for sign in (1, -1):
        cache = _ordinary(device, torch.bfloat16, 128, 64, 23)
        table, lengths = _tables(device, 2, 14, 30), torch.tensor([211, 64], dtype=torch.int32, device=device)
        if sign < 0:
            cache.v_params.mul_(2.0 ** apart)
        for b, j in ((0, 3), (0, 100), (0, 210), (1, 0), (1, 33)):
            cache.v_params[_token(table, b, j)] *= 2.0 ** (sign * apart)
        q = torch.randn(2, 1, ratio, 128, device=device).bfloat16()
        out, lse = kv_cache.attend(q, cache, lengths, table)
        _compare(cache, q, lengths, table, None, None, 0, out, lse)


@pytest.mark.parametrize("ratio", [4, 12])
def test_tokens_of_far_scales_of_which_one_decides(device, ratio):
    """The far token beside one of nearly all the weight whose own scale is small: fp16 over its whole range."""
    cache = _ordinary(device, torch.float16, 128, 64, 24)
    cache.v_params.mul_(2.0 ** -11)
    table, lengths = _tables(device, 1, 14, 30), torch.tensor([211], dtype=torch.int32, device=device)
    for j in (0, 50, 120):
        at = _token(table, 0, j)
        cache.v_params[at][:, 0], cache.v_params[at][:, 1] = 4000.0, -30000.0
        cache.k_params[at][:, 0], cache.k_params[at][:, 1] = 0.04, -16.0
    q = (1.0 + torch.rand(1, 1, ratio, 128, device=device)).half()
    out, lse = kv_cache.attend(q, cache, lengths, table)
    _compare(cache, q, lengths, table, None, None, 0, out, lse)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 100), (torch.bfloat16, 2.0 ** 30), (torch.float16, 2.0 ** 13)])
@pytest.mark.parametrize("ratio", [2, 5])
def test_newer_tokens_of_far_scales_leave_earlier_queries_alone(device, dtype, size, ratio):
    """A guess's later tokens, which its earlier queries do not see, hold values far above the others'."""
    cache = _ordinary(device, dtype, 128, 64, 25)
    if dtype == torch.float16:
        cache.v_params.mul_(2.0 ** -8)
    table, lengths = _tables(device, 2, 14, 30), torch.tensor([211, 64], dtype=torch.int32, device=device)
    q = torch.randn(2, 3, ratio, 128, device=device).to(dtype)
    for window, sinks in ((None, 0), (40, 3)):
        for b, n in enumerate(lengths.tolist()):
            for j in (n - 1, n - 2):
                cache.v_params[_token(table, b, j)] = torch.tensor([size / 8, -size], device=device).to(dtype)
        out, lse = kv_cache.attend(q, cache, lengths, table, window=window, sinks=sinks)
        _compare(cache, q[:, :1], lengths - 2, table, None, window, sinks, out[:, :1], lse[:, :1])
        _compare(cache, q, lengths, table, None, window, sinks, out, lse)


@pytest.mark.parametrize("page_size", [16, 20])
@pytest.mark.parametrize("window,sinks,queries", [(21, 0, 1), (33, 2, 1), (30, 17, 3)])
@pytest.mark.parametrize("scale,low", [(2.0 ** 100, 1.0), (3e38, 3e38), (-3e38, -3e38), (float("inf"), 0.0)])
def test_tokens_that_no_row_sees_may_be_of_any_scale(device, page_size, window, sinks, queries, scale, low):
    """Those that fill up 16 at the sinks' end and the window's beginning, and those behind the lengths: the same bits."""
    per = -(-224 // page_size)
    cache = _ordinary(device, torch.bfloat16, 128, 64, 26, page_size, 2 * per)
    table, lengths = _tables(device, 2, per, 2 * per), torch.tensor([211, 64], dtype=torch.int32, device=device)
    q = torch.randn(2, queries, 4, 128, device=device).bfloat16()
    want = kv_cache.attend(q, cache, lengths, table, window=window, sinks=sinks)
    for b, n in enumerate(lengths.tolist()):
        for j in range(per * page_size):
            if j >= n or (j >= sinks and j <= n - queries - window):
                for params in (cache.k_params, cache.v_params):
                    params[_token(table, b, j, page_size)] = torch.tensor([scale, low], device=device).bfloat16()
    got = kv_cache.attend(q, cache, lengths, table, window=window, sinks=sinks)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("ratio", [4, 12])
def test_later_queries_tokens_may_hold_anything_for_earlier_ones(device, ratio):
    """Parameters that no written row has (their middle is past the type's range), seen by the last query alone."""
    cache = _ordinary(device, torch.bfloat16, 128, 64, 27)
    table, lengths = _tables(device, 1, 14, 30), torch.tensor([211], dtype=torch.int32, device=device)
    q = torch.randn(1, 2, ratio, 128, device=device).bfloat16()
    want = kv_cache.attend(q, cache, lengths, table)
    for scale, low in ((3e38, 3e38), (-3e38, -3e38), (float("inf"), 0.0), (0.0, float("nan"))):
        cache.v_params[_token(table, 0, 210)] = torch.tensor([scale, low], device=device).bfloat16()
        out, lse = kv_cache.attend(q, cache, lengths, table)
        assert torch.equal(lse, want[1])
        assert not torch.isfinite(out[0, 1]).any()
        _compare(cache, q[:, :1], lengths - 1, table, None, None, 0, out[:, :1], lse[:, :1])


@pytest.mark.parametrize("rise", [-3.0, 3.0])
@pytest.mark.parametrize("ratio", [4, 12])
def test_scores_and_scales_that_drift_along_the_sequence(device, rise, ratio):
    """Scores rise (or fall) by 3 nats every 16 tokens while scales change by 2^3: references and windows move with them."""
    cache = _ordinary(device, torch.bfloat16, 128, 64, 28)
    table, lengths = _tables(device, 1, 28, 30), torch.tensor([441], dtype=torch.int32, device=device)
    q = torch.full((1, 1, ratio, 128), 0.25, device=device) + 0.1 * torch.rand(1, 1, ratio, 128, device=device)
    for i in range(28):
        page = int(table[0, i])
        cache.v_params[page].mul_(2.0 ** (3 * (i if rise < 0 else 27 - i)))
        cache.k_params[page, ..., 1] += rise * i / (0.3 * 128 ** 0.5)
    for order in (table, table[:, :28].flip(1).contiguous()):
        out, lse = kv_cache.attend(q.bfloat16(), cache, lengths, order)
        _compare(cache, q.bfloat16(), lengths, order, None, None, 0, out, lse)


@pytest.mark.parametrize("length,batch,ratio", [(9000, 1, 4), (9000, 1, 12), (2500, 5, 12), (700, 160, 3), (700, 310, 12)])
def test_far_scales_in_parts_of_long_sequences(device, length, batch, ratio):
    """Scales that drift over 2^40 along the sequence, differ by 2^12 between groups and jump by 2^25 at one token in a hundred, put
    together from the parts of warps and blocks."""
    page_size, per = 64, -(-length // 64)
    cache = _ordinary(device, torch.bfloat16, 128, 64, 29, page_size, per)
    drift = torch.linspace(-20, 20, per * page_size, device=device).view(per, 1, page_size, 1, 1)
    jump = 25.0 * (torch.rand(per, 1, page_size, 1, 1, device=device) < 0.01)
    between = torch.tensor([0.0, 12.0], device=device).view(1, 1, 1, 2, 1)
    cache.v_params.copy_((cache.v_params.float() * torch.exp2(drift + jump + between)).bfloat16())
    table = torch.arange(per, dtype=torch.int32, device=device).view(1, per).repeat(batch, 1)
    lengths = torch.tensor([length - (i * 331) % length for i in range(batch)], dtype=torch.int32, device=device)
    q = torch.randn(batch, 1, ratio, 128, device=device).bfloat16()
    out, lse = kv_cache.attend(q, cache, lengths, table)
    some = sorted({0, batch // 2, batch - 1})
    _compare(cache, q[some], lengths[some], table[some], None, None, 0, out[some], lse[some])

"""The 4-bit key/value cache on the GPU: bytes written, values read and attention against plain 64-bit arithmetic, at the
sizes, masks and contents where each can go wrong.

Tolerances. Codes, parameters and values read back are exact. An output of the attention may be off by
  - half a step of its type (bf16 2^-8, fp16 2^-11 of the value, and half the smallest fp16 subnormal);
  - what rounding each weight to fp16 moves it by: 2^-11 of sum p * scale * |code - 8| (`room`);
  - fp32 arithmetic: a score of magnitude `size` = sum |q| |k| is a sum of at most 128 + 8 terms, each a few roundings of 2^-24,
    which tensor cores may truncate (2^-23); with 2^-23 * 64 for terms that do not all err one way, a weight is off by
    2^-17 * (size + 1) of itself, and an output by twice that of sum p |v| (`slack`): above and below the line."""
import numpy as np
import pytest
import torch

from ferro_kittens_b200 import FerroKittensError, flash_forward, gemm, kv_cache

from kv_cache_plain import Plain, attention, key_nibble, pack, quantise, value_nibble

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FORMATS = [(128, 64, torch.bfloat16), (128, 128, torch.float16), (128, 32, torch.bfloat16), (64, 64, torch.float16),
           (64, 32, torch.bfloat16)]


def _random_cache(device, pages, page_size, kv_heads, head_dim, group, dtype, seed):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    cache = kv_cache.new(pages, page_size, kv_heads, head_dim, group, dtype, device)
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        codes.copy_(torch.randint(0, 256, codes.shape, device=device, generator=g, dtype=torch.uint8))
        scale = 0.3 * (0.3 + torch.rand(params.shape[:-1], device=device, generator=g))
        params[..., 0] = scale
        params[..., 1] = -7.5 * scale + torch.randn(params.shape[:-1], device=device, generator=g)
    return cache


def _awkward(dtype, head_dim, tokens, heads, seed):
    """Rows of every kind the rounding rule meets: ordinary, far off centre, constant, zero, ties, spans that underflow or
    overflow, values tiny beside their group's."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((tokens, heads, head_dim))
    far = 60000.0 if dtype == torch.float16 else 3.3e38
    tiny = 6e-8 if dtype == torch.float16 else 1e-39
    flat = x.reshape(-1, head_dim)
    for r in range(len(flat)):
        kind = r % 11
        if kind == 1:
            flat[r] += 37.0
        elif kind == 2:
            flat[r] = 1.75
        elif kind == 3:
            flat[r] = 0.0
        elif kind == 4:  # every half step of a scale of 2^-3 over [-1, 0.875], and the ends
            flat[r] = rng.integers(0, 31, head_dim) / 16 - 1.0
            flat[r, ::16], flat[r, 1::16] = -1.0, 0.875
        elif kind == 5:
            flat[r] *= tiny
        elif kind == 6:
            flat[r] = rng.choice([-far, far, 0.0, far / 3], head_dim)
        elif kind == 7:  # beside a span of 15/8, borders at zero and values that vanish in the difference
            flat[r] = rng.choice([0.9375, -0.9375, 2.0 ** -20, -2.0 ** -20, 2.0 ** -24, 0.0], head_dim)
            flat[r, ::16], flat[r, 1::16] = -0.9375, 0.9375
        elif kind == 8:
            flat[r] *= 2.0 ** rng.integers(-14, 5, head_dim)
        elif kind == 9:
            flat[r] = rng.integers(-8, 8, head_dim)
        elif kind == 10:
            flat[r] = 1.0 + rng.integers(0, 3, head_dim) * (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -10)
    return torch.from_numpy(x).to(dtype)


def _expect_rows(x, group, dtype, place):
    """Packed codes and parameters of every row of x [tokens, heads, dim]."""
    codes = np.zeros(x.shape[:2] + (x.shape[2] // 2,), np.uint8)
    params = np.zeros(x.shape[:2] + (x.shape[2] // group, 2))
    for t in range(x.shape[0]):
        for h in range(x.shape[1]):
            c, scale, low = quantise(x[t, h].double().numpy(), group, dtype)
            codes[t, h] = pack(c, place)
            params[t, h, :, 0], params[t, h, :, 1] = scale, low
    return codes, params


def _by_slot(t):
    return t.transpose(1, 2).reshape(-1, t.shape[1], *t.shape[3:]).cpu()


@pytest.mark.parametrize("head_dim,group,dtype", FORMATS)
@pytest.mark.parametrize("tokens,heads,page_size,wide", [(1, 1, 16, False), (13, 3, 5, True), (70, 2, 64, False)])
def test_written_bytes_are_exact(device, head_dim, group, dtype, tokens, heads, page_size, wide):
    pages = -(-tokens // page_size) + 2
    cache = kv_cache.new(pages, page_size, heads, head_dim, group, dtype, device)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0xa5)
    for t in (cache.k_params, cache.v_params):
        t.fill_(7.0)
    k, v = (_awkward(dtype, head_dim, tokens, heads, seed) for seed in (1, 2))
    slots = torch.randperm(pages * page_size, generator=torch.Generator().manual_seed(3))[:tokens]
    if tokens > 3:
        slots[tokens // 2] = -1
    status = gemm.new_status(device)
    kv_cache.write(cache, k.to(device), v.to(device), slots.to(device, torch.int64 if wide else torch.int32), status)
    gemm.check_status(status)
    kept = [i for i in range(tokens) if slots[i] >= 0]
    others = sorted(set(range(pages * page_size)) - set(slots.tolist()))
    for x, codes, params, place in ((k, cache.k_codes, cache.k_params, key_nibble),
                                    (v, cache.v_codes, cache.v_params, value_nibble)):
        want_codes, want_params = _expect_rows(x[kept], group, dtype, place)
        got_params, got_codes = _by_slot(params).double(), _by_slot(codes)
        at = slots[kept]
        assert np.array_equal(got_params[at].numpy(), want_params)
        assert np.array_equal(got_codes[at].numpy(), want_codes)
        assert (got_codes[others] == 0xa5).all() and (got_params[others] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
def test_a_group_that_is_not_finite_reads_back_as_nan(device, dtype, poison):
    cache = kv_cache.new(2, 16, 2, 128, 32, dtype, device)
    x = torch.randn(5, 2, 128, device=device).to(dtype)
    bad = x.clone()
    bad[3, 1, 40] = poison
    slots = torch.arange(5, dtype=torch.int32, device=device)
    kv_cache.write(cache, x, x, slots)
    clean = kv_cache.read(cache, slots)
    kv_cache.write(cache, bad, bad, slots)
    for got, want in zip(kv_cache.read(cache, slots), clean):
        assert torch.isnan(got[3, 1, 32:64]).all()
        rest = torch.ones_like(got, dtype=torch.bool)
        rest[3, 1, 32:64] = False
        assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("head_dim,group,dtype", FORMATS)
def test_values_read_back_are_rounded_once(device, head_dim, group, dtype):
    cache = _random_cache(device, 4, 9, 3, head_dim, group, dtype, 5)
    slots = torch.tensor([7, 0, 35, 7, -1, 20, -9], dtype=torch.int32, device=device)
    plain = Plain(cache)
    k, v = kv_cache.read(cache, slots)
    for which, got in (("k", k), ("v", v)):
        want, _ = plain.values(which, np.maximum(slots.cpu().numpy(), 0))
        want = torch.from_numpy(want)
        got = got.cpu().double()
        assert (got[[4, 6]] == 0).all()
        kept = [0, 1, 2, 3, 5]
        # One rounding: nothing of the type lies nearer. Half a step at the value's binade, and exactly.
        bits = {torch.bfloat16: 8, torch.float16: 11}[dtype]
        step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -13))) + 1 - bits)
        assert ((got - want).abs()[kept] <= step[kept] / 2).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_is_read_stays_inside_its_group_and_half_a_step_near(device, dtype):
    cache = kv_cache.new(9, 16, 2, 128, 64, dtype, device)
    x = _awkward(dtype, 128, 132, 2, 8).to(device)
    slots = torch.arange(132, device=device)
    kv_cache.write(cache, x, x, slots)
    for got in kv_cache.read(cache, slots):
        wide, back = (t.double().unflatten(-1, (2, 64)) for t in (x, got))
        low, high = wide.amin(-1, keepdim=True), wide.amax(-1, keepdim=True)
        assert ((back >= low) & (back <= high)).all()
        # Half a scale, the rounding of the sum to the type, and the span a scale that underflows leaves (15 subnormals).
        room = (high - low) / 30 + HALF_STEP[dtype] * back.abs() + 16 * 2.0 ** (BITS_LEAST[dtype])
        assert ((back - wide).abs() <= room).all()


BITS_LEAST = {torch.bfloat16: -133, torch.float16: -24}


@pytest.mark.parametrize("head_dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_strided_tensors_and_rows_left_as_they_were(device, head_dim, dtype):
    heads, tokens = 3, 21
    cache = kv_cache.new(3, 16, heads, head_dim, 32, dtype, device)
    wide = torch.randn(tokens, 4 * heads, head_dim, device=device).to(dtype)
    k, v = wide[:, heads:2 * heads], wide[:, 2 * heads:3 * heads]
    slots = torch.randperm(48, device=device)[:tokens].to(torch.int32)
    kv_cache.write(cache, k, v, slots)
    want = kv_cache.read(cache, slots)
    packed = kv_cache.new(3, 16, heads, head_dim, 32, dtype, device)
    kv_cache.write(packed, k.contiguous(), v.contiguous(), slots)
    for name in ("k_codes", "k_params", "v_codes", "v_params"):
        assert torch.equal(getattr(packed, name), getattr(cache, name))
    # Into planes [heads, tokens, head_dim], two tokens skipped.
    slots[4], slots[20] = -1, -7
    planes = [torch.full((heads, tokens + 2, head_dim), 3.0, dtype=dtype, device=device) for _ in range(2)]
    kv_cache.read(cache, slots, *(p[:, 1:-1].transpose(0, 1) for p in planes))
    for plane, rows in zip(planes, want):
        expected = torch.full_like(plane, 3.0)
        expected[:, 1:-1] = rows.transpose(0, 1)
        expected[:, 1 + 4] = expected[:, 1 + 20] = 3.0
        assert torch.equal(plane, expected)


def test_slots_outside_the_cache_are_skipped_and_noted(device):
    cache = kv_cache.new(2, 8, 1, device=device)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0x5a)
    x = torch.randn(3, 1, 128, device=device).bfloat16()
    for slots in (torch.tensor([16, 3, -1], dtype=torch.int32), torch.tensor([1 << 40, 3, -1])):
        status = gemm.new_status(device)
        kv_cache.write(cache, x, x, slots.to(device), status)
        with pytest.raises(FerroKittensError, match="token 0 lies outside the cache"):
            gemm.check_status(status)
        assert (_by_slot(cache.k_codes)[[i for i in range(16) if i != 3]] == 0x5a).all()
        status = gemm.new_status(device)
        k, _ = kv_cache.read(cache, slots.to(device), status=status)
        with pytest.raises(FerroKittensError, match="token 0 lies outside the cache"):
            gemm.check_status(status)
        assert (k[[0, 2]] == 0).all() and (k[1] != 0).any()


# ---------------------------------------------------------------- attention

def _check_attention(device, cache, q, lengths, table, scale=None, window=None, sinks=0, workspace=None):
    status = gemm.new_status(device)
    out, lse = kv_cache.attend(q, cache, lengths, table, scale, window, sinks, workspace, status=status)
    gemm.check_status(status)
    assert out.dtype == cache.dtype and lse.dtype == torch.float32
    _compare(cache, q, lengths, table, scale, window, sinks, out, lse)
    return out, lse


def _compare(cache, q, lengths, table, scale, window, sinks, out, lse):
    plain = Plain(cache)
    dtype = cache.dtype
    factor = cache.head_dim ** -0.5 if scale is None else scale
    for b, length in enumerate(lengths.tolist()):
        pages = table[b].tolist() if table is not None else [b]
        want, want_lse, room, slack, size = attention(plain, q[b].cpu().double().numpy(), max(length, 0), pages, factor, window,
                                                      sinks)
        got, got_lse = out[b].cpu().double().numpy(), lse[b].cpu().double().numpy()
        assert np.array_equal(np.isneginf(got_lse), np.isneginf(want_lse)), (b, got_lse, want_lse)
        weight = 2.0 ** -17 * (size + 1)
        fine = np.isfinite(want_lse)
        off = np.abs(got_lse[fine] - want_lse[fine]) - weight[fine]
        assert (off <= 0).all(), (b, off.max())
        allowed = HALF_STEP[dtype] * np.abs(want) + 2.0 ** -11 * room + 2 * weight[..., None] * slack + 2.0 ** -25
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= allowed).all(), (b, (np.abs(got - want) / allowed).max())
        assert (got[~fine] == 0).all()


def _tables(device, batch, per, pages, seed=0):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * per]
    return order.to(device, torch.int32).view(batch, per)


@pytest.mark.parametrize("head_dim,group,dtype", FORMATS)
@pytest.mark.parametrize("kv_heads,ratio,queries", [(2, 1, 1), (1, 8, 1), (2, 7, 1), (1, 4, 3), (2, 16, 1), (1, 5, 8), (3, 2, 40)])
def test_attention_formats_and_heads(device, head_dim, group, dtype, kv_heads, ratio, queries):
    lengths = torch.tensor([150, 0, 1, 131, queries], dtype=torch.int32, device=device)
    per, page_size = 10, 16
    cache = _random_cache(device, 55, page_size, kv_heads, head_dim, group, dtype, 11)
    q = torch.randn(5, queries, kv_heads * ratio, head_dim, device=device).to(dtype) * 1.5
    _check_attention(device, cache, q, lengths, _tables(device, 5, per, 55), workspace=kv_cache.workspace(device))


@pytest.mark.parametrize("page_size", [1, 3, 16, 100, 128, 1000])
@pytest.mark.parametrize("length", [1, 2, 31, 33, 127, 128, 129, 257, 700])
def test_attention_lengths_and_pages(device, page_size, length):
    per = -(-length // page_size)
    cache = _random_cache(device, per + 2, page_size, 1, 128, 64, torch.bfloat16, length)
    q = torch.randn(1, 1, 4, 128, device=device).bfloat16()
    lengths = torch.tensor([length], dtype=torch.int32, device=device)
    _check_attention(device, cache, q, lengths, _tables(device, 1, per, per + 2, length))


@pytest.mark.parametrize("head_dim,group", [(128, 128), (128, 32), (64, 64)])
@pytest.mark.parametrize("page_size,window,sinks", [(1, None, 0), (5, 90, 3), (10, None, 0), (24, 200, 33), (100, 37, 1)])
def test_attention_rows_that_do_not_begin_on_16_bytes(device, head_dim, group, page_size, window, sinks):
    """Parameters of 4 and 8 bytes a row whose runs begin and end anywhere."""
    lengths = torch.tensor([333, 12, 480], dtype=torch.int32, device=device)
    per = -(-480 // page_size)
    cache = _random_cache(device, 3 * per, page_size, 3, head_dim, group, torch.bfloat16, 17)
    q = torch.randn(3, 2, 9, head_dim, device=device).bfloat16()
    _check_attention(device, cache, q, lengths, _tables(device, 3, per, 3 * per), window=window, sinks=sinks)


@pytest.mark.parametrize("seed", range(30))
def test_attention_drawn(device, seed):
    """Everything at once, drawn: formats, heads, ragged lengths with empty ones, pages, windows, strides of the table."""
    rng = np.random.default_rng(seed)
    head_dim, group, dtype = FORMATS[seed % len(FORMATS)]
    kv_heads, ratio, queries = int(rng.integers(1, 4)), int(rng.choice([1, 2, 3, 6, 8, 12])), int(rng.choice([1, 1, 2, 5]))
    batch, page_size = int(rng.choice([1, 3, 9])), int(rng.choice([1, 7, 16, 32, 48, 64, 200]))
    lengths = [int(n) for n in np.exp(rng.uniform(0, np.log(900), batch))]
    if batch > 1:
        lengths[int(rng.integers(batch))] = 0
    per = -(-max(lengths) // page_size) + int(rng.integers(0, 3))
    per = max(per, 1)
    cache = _random_cache(device, batch * per + 1, page_size, kv_heads, head_dim, group, dtype, seed)
    wide = torch.full((batch, per + 3), 1 << 30, dtype=torch.int32, device=device)
    wide[:, :per] = _tables(device, batch, per, batch * per + 1, seed)
    window, sinks = (int(rng.integers(1, 400)), int(rng.choice([0, 1, 4, 60]))) if rng.random() < 0.4 else (None, 0)
    q = torch.randn(batch, queries, kv_heads * ratio, head_dim, device=device).to(dtype) * float(rng.choice([0.3, 1.5, 4.0]))
    _check_attention(device, cache, q, torch.tensor(lengths, dtype=torch.int32, device=device), wide[:, :per], window=window,
                     sinks=sinks)


@pytest.mark.parametrize("head_dim,group,dtype", FORMATS)
@pytest.mark.parametrize("ratio", [3, 12])
def test_a_token_of_nearly_all_the_weight_whose_value_is_zero(device, head_dim, group, dtype, ratio):
    """Its code is the middle, 8, and its smallest value -8 scales: what the others add must not drown in what cancels."""
    g = torch.Generator(device=device)
    g.manual_seed(5)
    cache = _random_cache(device, 3, 64, 1, head_dim, group, dtype, 5)
    for page, token in ((0, 46), (1, 7), (2, 30)):
        cache.k_codes[page, 0, token] = 0xff
        cache.v_codes[page, 0, token] = 0x88
        cache.k_params[page, 0, token, :, 0], cache.k_params[page, 0, token, :, 1] = 0.25, -1.5
        cache.v_params[page, 0, token, :, 0], cache.v_params[page, 0, token, :, 1] = 0.25, -2.0
    # The token's key is 2.25 in every channel, so that queries of one sign give it scores 5 to 12 above the others'.
    for size in (0.2, 0.3, 0.45):
        q = (size * 128 / head_dim * (0.5 + torch.rand(3, 1, ratio, head_dim, device=device, generator=g))).to(dtype)
        _check_attention(device, cache, q, torch.tensor([50, 31, 64], dtype=torch.int32, device=device),
                         torch.tensor([[0], [1], [2]], dtype=torch.int32, device=device))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (64, 4), (100, 0), (128, 130), (5000, 4), (37, 1000)])
@pytest.mark.parametrize("queries", [1, 4])
def test_attention_window_and_sinks(device, window, sinks, queries):
    lengths = torch.tensor([500, 36, 3, 1, 130], dtype=torch.int32, device=device)
    cache = _random_cache(device, 170, 16, 2, 128, 64, torch.float16, 2)
    q = torch.randn(5, queries, 6, 128, device=device).half()
    _check_attention(device, cache, q, lengths, _tables(device, 5, 32, 170), window=window, sinks=sinks)


def test_what_a_row_does_not_see_may_hold_anything(device):
    """NaN parameters behind the lengths, outside the window and, for a guess's earlier rows, in its later tokens."""
    page_size, per = 16, 12
    lengths = [150, 40, 0, 17]
    cache = _random_cache(device, 50, page_size, 2, 128, 64, torch.bfloat16, 4)
    table = _tables(device, 4, per, 50)
    q = torch.randn(4, 3, 8, 128, device=device).bfloat16()
    at = torch.tensor(lengths, dtype=torch.int32, device=device)
    want = kv_cache.attend(q, cache, at, table, window=20, sinks=2)
    unseen = torch.ones(50 * page_size, dtype=torch.bool)
    newest = torch.zeros(50 * page_size, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for j in range(n):
            slot = int(table[b, j // page_size]) * page_size + j % page_size
            if j > n - 3 - 20 or j < 2:
                unseen[slot] = False
            if j >= n - 2:
                newest[slot] = True
    def spoil(which):
        rows = which.view(50, page_size).to(device)
        for t in (cache.k_params, cache.v_params):
            t.masked_fill_(rows[:, None, :, None, None], float("nan"))
    spoil(unseen)
    for x, y in zip(kv_cache.attend(q, cache, at, table, window=20, sinks=2), want):
        assert torch.equal(x, y)
    # Only rows of later queries see the two newest tokens.
    spoil(newest)
    got = kv_cache.attend(q, cache, at, table, window=20, sinks=2)
    for x, y in zip(got, want):
        assert torch.equal(x[:, 0], y[:, 0])
    assert torch.isnan(got[0][[0, 1, 3], 2]).all()
    # Table entries behind the lengths are never looked at.
    for b, n in enumerate(lengths):
        table[b, -(-n // page_size):] = 1 << 30
    status = gemm.new_status(device)
    again = kv_cache.attend(q, cache, at, table, window=20, sinks=2, status=status)
    gemm.check_status(status)
    assert torch.equal(again[0][:, 0], want[0][:, 0])


@pytest.mark.parametrize("page_size", [1, 4, 20, 64])
@pytest.mark.parametrize("window,sinks,queries", [(21, 0, 1), (21, 2, 1), (1, 5, 1), (30, 17, 3)])
def test_pages_that_no_row_sees_may_be_gone(device, page_size, window, sinks, queries):
    lengths = [200, 199, 64]
    per = -(-200 // page_size)
    cache = _random_cache(device, 3 * per, page_size, 2, 128, 64, torch.bfloat16, 4)
    table = _tables(device, 3, per, 3 * per)
    q = torch.randn(3, queries, 8, 128, device=device).bfloat16()
    at = torch.tensor(lengths, dtype=torch.int32, device=device)
    want = kv_cache.attend(q, cache, at, table, window=window, sinks=sinks)
    first, last = {}, {}
    for b, n in enumerate(lengths):
        for page in range(per):
            tokens = range(page * page_size, min((page + 1) * page_size, n))
            seen = [j for j in tokens if j < sinks or j > n - queries - window]
            if not seen:
                table[b, page] = -1 if page % 2 else 1 << 30
            elif tokens[0] > n - queries - window:
                last[b] = page
            else:
                first[b] = page
    status = gemm.new_status(device)
    for x, y in zip(kv_cache.attend(q, cache, at, table, window=window, sinks=sinks, status=status), want):
        assert torch.equal(x, y)
    gemm.check_status(status)
    # One that some row sees may not.
    page = last.get(1, first.get(1))
    table[1, page] = -1
    status = gemm.new_status(device)
    kv_cache.attend(q, cache, at, table, window=window, sinks=sinks, status=status)
    with pytest.raises(FerroKittensError, match="in the table of sequence 1"):
        gemm.check_status(status)


def test_bad_pages_and_lengths_are_noted_and_skipped(device):
    cache = _random_cache(device, 8, 16, 1, 128, 64, torch.bfloat16, 4)
    table = torch.tensor([[1, 2, 3], [4, 8, 5]], dtype=torch.int32, device=device)
    q = torch.randn(2, 1, 4, 128, device=device).bfloat16()
    status = gemm.new_status(device)
    out, _ = kv_cache.attend(q, cache, torch.tensor([48, 40], dtype=torch.int32, device=device), table, status=status)
    with pytest.raises(FerroKittensError, match="page 8 in the table of sequence 1"):
        gemm.check_status(status)
    assert torch.isfinite(out).all()
    table[1, 1] = -1
    status = gemm.new_status(device)
    kv_cache.attend(q, cache, torch.tensor([48, 40], dtype=torch.int32, device=device), table, status=status)
    with pytest.raises(FerroKittensError, match="page 4294967295 in the table of sequence 1"):
        gemm.check_status(status)
    status = gemm.new_status(device)
    want, _ = kv_cache.attend(q[:1], cache, torch.tensor([48], dtype=torch.int32, device=device), table[:1])
    out, _ = kv_cache.attend(q, cache, torch.tensor([49, 16], dtype=torch.int32, device=device), table, status=status)
    with pytest.raises(FerroKittensError, match="length 49 of sequence 0"):
        gemm.check_status(status)
    assert torch.equal(out[:1], want)


def test_scales_of_every_size(device):
    """Parameters and queries whose sizes lie far apart: the products' ranges are followed, not assumed."""
    cache = _random_cache(device, 6, 64, 1, 128, 64, torch.bfloat16, 9)
    size = 2.0 ** torch.arange(-60, 60, 120 / (6 * 64), device=device)[:6 * 64].view(6, 1, 64, 1, 1)
    cache.v_params.copy_((cache.v_params.float() * size).bfloat16())
    cache.k_params.mul_(0.05)
    lengths = torch.tensor([384], dtype=torch.int32, device=device)
    table = torch.arange(6, dtype=torch.int32, device=device).view(1, 6)
    q = torch.randn(1, 1, 4, 128, device=device).bfloat16()
    _check_attention(device, cache, q, lengths, table)
    _check_attention(device, cache, q, lengths, table.flip(1).contiguous())
    cache.k_params.mul_(2.0 ** -70)
    big = (q.float() * 2.0 ** 70).bfloat16()
    big[0, 0, 0] *= 2.0 ** -90
    big[0, 0, 1] = 0
    _check_attention(device, cache, big, lengths, table)


def test_scale_signs(device):
    cache = _random_cache(device, 10, 16, 2, 64, 32, torch.float16, 9)
    lengths = torch.tensor([100, 50], dtype=torch.int32, device=device)
    table = _tables(device, 2, 5, 10)
    table = torch.cat([table, table], 1)
    q = torch.randn(2, 2, 4, 64, device=device).half()
    for scale in (-0.3, 0.0, 1.0):
        _check_attention(device, cache, q, lengths, table, scale=scale)


def test_one_page_a_sequence_without_a_table(device):
    cache = _random_cache(device, 4, 300, 2, 128, 128, torch.bfloat16, 3)
    q = torch.randn(3, 4, 128, device=device).bfloat16()
    lengths = torch.tensor([300, 7, 128], dtype=torch.int32, device=device)
    out, lse = kv_cache.attend(q, cache, lengths)
    assert out.shape == q.shape and lse.shape == q.shape[:2]
    _compare(cache, q.unsqueeze(1), lengths, None, None, None, 0, out.unsqueeze(1), lse.unsqueeze(1))


def test_strided_queries_and_a_given_output(device):
    cache = _random_cache(device, 20, 16, 2, 128, 64, torch.bfloat16, 3)
    lengths = torch.tensor([90, 33], dtype=torch.int32, device=device)
    table = _tables(device, 2, 10, 20)
    wide = torch.randn(2, 3, 12, 128, device=device).bfloat16()
    q = wide[:, :, 2:10]
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device=device)
    got, lse = kv_cache.attend(q, cache, lengths, table[:, :8], out=out)
    assert got.data_ptr() == out.data_ptr()
    _compare(cache, q, lengths, table, None, None, 0, out, lse)


def _serve(device, batch, kv_heads, ratio, length, ragged, seed, **more):
    page_size = 64
    per = -(-length // page_size)
    cache = _random_cache(device, batch * per, page_size, kv_heads, 128, 64, torch.bfloat16, seed)
    lengths = [length - (i * 977) % length if ragged else length for i in range(batch)]
    q = torch.randn(batch, 1, kv_heads * ratio, 128, device=device).bfloat16()
    return cache, q, torch.tensor(lengths, dtype=torch.int32, device=device), _tables(device, batch, per, batch * per)


@pytest.mark.parametrize("batch,kv_heads,ratio,length,ragged", [(1, 1, 8, 40000, False), (3, 2, 4, 9000, True), (300, 1, 2, 90, True)])
def test_long_and_many_sequences(device, batch, kv_heads, ratio, length, ragged):
    cache, q, lengths, table = _serve(device, batch, kv_heads, ratio, length, ragged, 6)
    workspace = kv_cache.workspace(device)
    out, lse = _check_attention(device, cache, q, lengths, table, workspace=workspace)
    for _ in range(3):  # the same bits every time, through a workspace that is used again
        again, lse_again = kv_cache.attend(q, cache, lengths, table, workspace=workspace)
        assert torch.equal(again, out) and torch.equal(lse_again, lse)


def test_more_sequences_than_blocks_count(device):
    """Thousands of sequences, most of them empty or of a token or two."""
    batch = 5000
    cache = _random_cache(device, 40, 16, 1, 64, 32, torch.bfloat16, 6)
    lengths = torch.zeros(batch, dtype=torch.int32)
    lengths[::7], lengths[3::1000], lengths[-1] = 1, 300, 2
    table = (torch.arange(batch)[:, None] * 3 + torch.arange(20)).remainder(40).int()
    q = torch.randn(batch, 1, 3, 64, device=device).bfloat16()
    out, lse = kv_cache.attend(q, cache, lengths.to(device), table.to(device))
    some = [0, 1, 3, 7, 1003, 2499, 3003, 4900, 4998, 4999]
    _compare(cache, q[some], lengths[some], table[some], None, None, 0, out[some], lse[some])
    empty = lengths == 0
    assert (out[empty.to(device)] == 0).all() and torch.isneginf(lse[empty.to(device)]).all()


def test_rows_that_hold_nan_or_infinite_queries_spoil_no_others(device):
    cache = _random_cache(device, 10, 16, 2, 128, 64, torch.bfloat16, 3)
    table, lengths = _tables(device, 2, 5, 10), torch.tensor([77, 30], dtype=torch.int32, device=device)
    for heads in (8, 24):
        q = torch.randn(2, 1, heads, 128, device=device).bfloat16()
        want = kv_cache.attend(q, cache, lengths, table)
        bad = q.clone()
        bad[0, 0, 1, 5], bad[1, 0, heads - 1, 0] = float("nan"), float("inf")
        out, lse = kv_cache.attend(bad, cache, lengths, table)
        assert torch.isnan(out[0, 0, 1]).all() and torch.isnan(out[1, 0, heads - 1]).all()
        rest = torch.ones(2, 1, heads, dtype=torch.bool, device=device)
        rest[0, 0, 1] = rest[1, 0, heads - 1] = False
        # The others' queries may be scaled by another power of two: the same numbers but for fp32 sums' last bits.
        assert torch.allclose(out[rest].float(), want[0][rest].float(), rtol=2.0 ** -7, atol=2.0 ** -12)
        assert torch.allclose(lse[rest], want[1][rest], rtol=0, atol=2.0 ** -14)


@pytest.mark.parametrize("heads", [4, 20])
@pytest.mark.parametrize("length", [1, 600, 3000, 20000])
def test_a_row_of_nothing_but_nan_stays_nan(device, heads, length):
    """However many parts its segment is put together from, and whether the query or all keys made it NaN."""
    page_size = 64
    per = -(-length // page_size)
    cache = _random_cache(device, per, page_size, 1, 128, 64, torch.bfloat16, 3)
    table = _tables(device, 1, per, per)
    at = torch.tensor([length], dtype=torch.int32, device=device)
    q = torch.randn(1, 1, heads, 128, device=device).bfloat16()
    q[0, 0, 2, 7] = float("nan")
    out, lse = kv_cache.attend(q, cache, at, table)
    bad = torch.arange(heads, device=device) == 2
    assert torch.isnan(out[0, 0, bad]).all() and torch.isnan(lse[0, 0, bad]).all()
    assert torch.isfinite(out[0, 0, ~bad]).all() and torch.isfinite(lse[0, 0, ~bad]).all()
    cache.k_params[..., 0, :] = float("nan")
    out, lse = kv_cache.attend(q, cache, at, table)
    assert torch.isnan(out).all() and torch.isnan(lse).all()


def test_rows_past_four_gibibytes(device):
    """A cache whose codes pass 2^32 bytes on each side: the last pages, written, read and attended to."""
    page_size, kv_heads = 1024, 8
    pages = (1 << 32) // (page_size * kv_heads * 64) + 40
    cache = kv_cache.Cache(*(torch.empty((pages, kv_heads, page_size, 64), dtype=torch.uint8, device=device) if i % 2 == 0 else
                             torch.empty((pages, kv_heads, page_size, 2, 2), dtype=torch.bfloat16, device=device) for i in range(4)))
    small = kv_cache.new(3, page_size, kv_heads, device=device)
    table = torch.tensor([[pages - 1, 0, pages - 30]], dtype=torch.int32, device=device)
    tokens = 2 * page_size + 100
    at = torch.arange(tokens, device=device)
    x, y = (torch.randn(tokens, kv_heads, 128, device=device).bfloat16() for _ in range(2))
    slots = table[0].long()[at // page_size] * page_size + at % page_size
    kv_cache.write(cache, x, y, slots)
    kv_cache.write(small, x, y, at)
    for a, b in zip(kv_cache.read(cache, slots), kv_cache.read(small, at)):
        assert torch.equal(a, b)
    q = torch.randn(1, 1, 16, 128, device=device).bfloat16()
    lengths = torch.tensor([tokens], dtype=torch.int32, device=device)
    got = kv_cache.attend(q, cache, lengths, table)
    want = kv_cache.attend(q, small, lengths, torch.tensor([[0, 1, 2]], dtype=torch.int32, device=device))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- together, as they are used

def test_a_prompt_then_decoding_steps(device):
    """Prompts of two sequences written, then tokens appended one by one, each step attending over what was written so far."""
    batch, kv_heads, ratio, page_size, per = 2, 2, 4, 16, 6
    cache = kv_cache.new(batch * per + 1, page_size, kv_heads, device=device)
    table = _tables(device, batch, per, batch * per)
    workspace = kv_cache.workspace(device)
    lengths = torch.tensor([37, 60], dtype=torch.int32, device=device)
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(n, device=device)
        slots = table[b].long()[at // page_size] * page_size + at % page_size
        kv_cache.write(cache, *(torch.randn(n, kv_heads, 128, device=device).bfloat16() for _ in range(2)), slots)
    for step in range(20):
        place = lengths.long()
        slots = table.long()[torch.arange(batch, device=device), place // page_size] * page_size + place % page_size
        kv_cache.write(cache, *(torch.randn(batch, kv_heads, 128, device=device).bfloat16() for _ in range(2)), slots)
        lengths += 1
        q = torch.randn(batch, 1, kv_heads * ratio, 128, device=device).bfloat16()
        _check_attention(device, cache, q, lengths, table, window=32 if step % 2 else None, sinks=4, workspace=workspace)


def test_a_prefix_read_into_planes_for_the_prompt_attention(device):
    """A prefix read back feeds flash_forward.run, whose last row agrees with the cache's own attention."""
    kv_heads, tokens = 2, 256
    cache = kv_cache.new(4, 64, kv_heads, device=device)
    slots = torch.arange(tokens, device=device)
    kv_cache.write(cache, *(torch.randn(tokens, kv_heads, 128, device=device).bfloat16() for _ in range(2)), slots)
    k, v = (torch.empty(kv_heads, tokens, 128, dtype=torch.bfloat16, device=device) for _ in range(2))
    kv_cache.read(cache, slots, k.transpose(0, 1), v.transpose(0, 1))
    q = torch.randn(kv_heads, tokens, 128, device=device).bfloat16()
    prompt, prompt_lse = flash_forward.run(q, k, v, causal=True)
    out, lse = kv_cache.attend(q[:, -1].unsqueeze(0), cache, torch.tensor([tokens], dtype=torch.int32, device=device),
                               torch.arange(4, dtype=torch.int32, device=device).view(1, 4))
    # Keys and values rounded to bf16 on one side: scores off by 2^-8 of sum |q| |k| / sqrt(128) <= 2^-8 * 16 in the lse;
    # outputs of unit values by that of themselves and by P's and the values' own roundings.
    assert (lse[0] - prompt_lse[:, -1]).abs().max() < 2.0 ** -4
    assert (out[0].float() - prompt[:, -1].float()).abs().max() < 2.0 ** -4


def test_streams_and_captured_graphs(device):
    """Two streams with a workspace each, and a captured write-and-attend step replayed with other tokens in its buffers."""
    cache, q, lengths, table = _serve(device, 5, 2, 4, 3000, True, 8)
    want, want_lse = kv_cache.attend(q, cache, lengths, table)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    spaces = [kv_cache.workspace(device) for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for stream, space in zip(streams, spaces):
            with torch.cuda.stream(stream):
                results.append(kv_cache.attend(q, cache, lengths, table, workspace=space))
    torch.cuda.synchronize()
    for out, lse in results:
        assert torch.equal(out, want) and torch.equal(lse, want_lse)

    k, v = (torch.randn(5, 2, 128, device=device).bfloat16() for _ in range(2))
    place = lengths.long() - 1
    slots = table.long()[torch.arange(5, device=device), place // 64] * 64 + place % 64
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_cache.write(cache, k, v, slots)
        out, lse = kv_cache.attend(q, cache, lengths, table, workspace=spaces[0])
    for _ in range(3):
        k.copy_(torch.randn_like(k))
        v.copy_(torch.randn_like(v))
        q.copy_(torch.randn_like(q))
        lengths.copy_(torch.clamp(lengths - 64, min=1))
        place = lengths.long() - 1
        slots.copy_(table.long()[torch.arange(5, device=device), place // 64] * 64 + place % 64)
        graph.replay()
        torch.cuda.synchronize()
        fresh, fresh_lse = kv_cache.attend(q, cache, lengths, table)
        assert torch.equal(out, fresh) and torch.equal(lse, fresh_lse)
        again = kv_cache.read(cache, slots)
        kv_cache.write(cache, k, v, slots)
        for a, b in zip(kv_cache.read(cache, slots), again):
            assert torch.equal(a, b)


def test_empty_calls(device):
    cache = kv_cache.new(2, 16, 2, device=device)
    none = torch.empty(0, dtype=torch.int32, device=device)
    rows = torch.empty(0, 2, 128, dtype=torch.bfloat16, device=device)
    kv_cache.write(cache, rows, rows, none)
    assert kv_cache.read(cache, none)[0].shape == (0, 2, 128)
    out, lse = kv_cache.attend(torch.empty(0, 1, 4, 128, dtype=torch.bfloat16, device=device), cache, none,
                               torch.empty(0, 2, dtype=torch.int32, device=device))
    assert out.shape == (0, 1, 4, 128) and lse.shape == (0, 1, 4)


def test_refusals_with_tensors(device):
    cache = kv_cache.new(2, 16, 2, device=device)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=device)
    slots = torch.arange(4, device=device)
    for bad in (x.half(), x[:, :1], x[:3], x[..., :64], x.flatten(1)):
        with pytest.raises(ValueError):
            kv_cache.write(cache, bad, x, slots)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv_cache.write(cache, x.cpu(), x, slots)
    for bad in (slots.float(), slots.view(2, 2), torch.arange(8, device=device)[::2]):
        with pytest.raises(ValueError):
            kv_cache.write(cache, x, x, bad)
    odd = torch.zeros(4 * 300, dtype=torch.bfloat16, device=device)
    with pytest.raises(FerroKittensError, match="no multiple of 8"):
        kv_cache.write(cache, odd.as_strided((4, 2, 128), (300, 128, 1)), x, slots)
    with pytest.raises(FerroKittensError, match="16-byte aligned"):
        kv_cache.write(cache, odd[4:4 + 1024].view(4, 2, 128), x, slots)
    with pytest.raises(ValueError, match="together"):
        kv_cache.read(cache, slots, k=x)
    lengths = torch.ones(4, dtype=torch.int32, device=device)
    table = torch.zeros(4, 2, dtype=torch.int32, device=device)
    q = torch.zeros(4, 1, 4, 128, dtype=torch.bfloat16, device=device)
    for bad in (q.half(), q[:, :, :3], q[..., :64], q[0]):
        with pytest.raises((ValueError, FerroKittensError)):
            kv_cache.attend(bad, cache, lengths, table)
    for bad in (lengths.long(), lengths[:3], lengths[::2]):
        with pytest.raises(ValueError):
            kv_cache.attend(q, cache, bad, table)
    for bad in (table.long(), table[:3], table.t(), torch.zeros(4, 4, dtype=torch.int32, device=device)[:, ::2]):
        with pytest.raises(ValueError):
            kv_cache.attend(q, cache, lengths, bad)
    with pytest.raises(FerroKittensError, match="own a page each"):
        kv_cache.attend(q, cache, lengths)
    with pytest.raises(ValueError):
        kv_cache.attend(q, cache, lengths, table[:, :0])
    for more in ({"window": 0}, {"window": -1}, {"sinks": -1}, {"workspace": torch.zeros(16, device="cpu")},
                 {"out": q.half()}, {"out": q[:, :, :2]}, {"out": q}, {"scale": float("nan")}):
        with pytest.raises((ValueError, RuntimeError)):  # FerroKittensError is a RuntimeError
            kv_cache.attend(q, cache, lengths, table, **more)
    with pytest.raises(FerroKittensError, match="over one another"):
        kv_cache.read(cache, slots, x[:1].expand(4, 2, 128), x)
    with pytest.raises(FerroKittensError, match="workspace of 16 bytes"):
        kv_cache.attend(q, cache, lengths, table, workspace=torch.zeros(16, dtype=torch.uint8, device=device))
    for sizes in ({"head_dim": 96}, {"group": 16}, {"head_dim": 64, "group": 128}, {"dtype": torch.float32}):
        with pytest.raises(ValueError):
            kv_cache.new(1, 16, 1, device=device, **sizes)

"""What the 4-bit cache's entries refuse before they reach a device, and the plain definition the GPU tests compare with."""
import ctypes
import re
import types

import numpy as np
import pytest
import torch

from ferro_kittens_b200 import kv_cache
from ferro_kittens_b200._lib import FK_BF16, FK_ERR_ALIGNMENT, FK_ERR_INVALID, FK_ERR_SHAPE, FK_F32, FK_OK, CacheView, last_error, library

from kv_cache_plain import key_nibble, quantise, value_nibble

BASE = 0x7F00_0000  # a device address is never dereferenced on the host


def _cache(**changed):
    fields = {"k_codes": BASE, "k_params": BASE, "v_codes": BASE, "v_params": BASE, "pages": 4, "page_size": 16,
              "kv_heads": 2, "head_dim": 128, "group": 64, "element": FK_BF16} | changed
    return CacheView(*fields.values())


def _write(cache, k=BASE, v=BASE, strides=(256, 128, 256, 128), slots=BASE, slot_bytes=4, tokens=3):
    return library().fk_cache_write(ctypes.byref(cache) if cache else None, k, v, *strides, slots, slot_bytes, tokens, None, None)


def _read(cache, k=BASE, v=BASE, strides=(256, 128, 256, 128), slots=BASE, slot_bytes=4, tokens=3):
    return library().fk_cache_read(ctypes.byref(cache) if cache else None, k, v, *strides, slots, slot_bytes, tokens, 0, None, None)


def _attend(cache, q=BASE, strides=(1024, 1024, 128), out=BASE + (1 << 20), lse=BASE, lengths=BASE, table=BASE, table_pages=2, batch=3,
            queries=1, heads=8, scale=0.1, workspace=BASE, workspace_bytes=1 << 30):
    return library().fk_cache_attention(ctypes.byref(cache) if cache else None, q, *strides, out, lse, lengths, table, table_pages,
                                        table_pages, batch, queries, heads, scale, 0, 0, workspace, workspace_bytes, None, None)


@pytest.mark.parametrize("entry", [_write, _read, _attend])
@pytest.mark.parametrize("changed,code,word", [
    ({"k_codes": None}, FK_ERR_INVALID, "buffer is null"), ({"v_params": None}, FK_ERR_INVALID, "buffer is null"),
    ({"v_codes": BASE + 8}, FK_ERR_ALIGNMENT, "16-byte"), ({"element": FK_F32}, FK_ERR_INVALID, "bf16 or fp16"),
    ({"head_dim": 96}, FK_ERR_SHAPE, "head_dim 96"), ({"group": 16}, FK_ERR_SHAPE, "groups of 16"),
    ({"head_dim": 64, "group": 128}, FK_ERR_SHAPE, "groups of 128"), ({"pages": 0}, FK_ERR_SHAPE, "is empty"),
    ({"page_size": 0}, FK_ERR_SHAPE, "is empty"), ({"kv_heads": 0}, FK_ERR_SHAPE, "is empty"),
    ({"pages": 1 << 31, "page_size": 1 << 31, "kv_heads": 1 << 31}, FK_ERR_SHAPE, "more than 2\\^31"),
    ({"pages": 1 << 20, "page_size": 1 << 10}, FK_ERR_SHAPE, "more than 2\\^31")])
def test_caches_refused(entry, changed, code, word):
    assert entry(_cache(**changed)) == code
    assert re.search(word, last_error()), last_error()


def test_a_null_cache_is_refused():
    for entry in (_write, _read, _attend):
        assert entry(None) == FK_ERR_INVALID and "null" in last_error()


@pytest.mark.parametrize("entry", [_write, _read])
@pytest.mark.parametrize("changed,code,word", [
    ({"k": None}, FK_ERR_INVALID, "null"), ({"slots": None}, FK_ERR_INVALID, "null"), ({"v": BASE + 2}, FK_ERR_ALIGNMENT, "16-byte"),
    ({"slot_bytes": 2}, FK_ERR_INVALID, "4 or 8"), ({"slots": BASE + 4, "slot_bytes": 8}, FK_ERR_ALIGNMENT, "8 bytes"),
    ({"strides": (256, 132, 256, 128)}, FK_ERR_ALIGNMENT, "132"), ({"strides": (256, 128, 257, 128)}, FK_ERR_ALIGNMENT, "257"),
    ({"tokens": 1 << 30}, FK_ERR_SHAPE, "more than 2^31")])
def test_rows_refused(entry, changed, code, word):
    assert entry(_cache(), **changed) == code
    assert word in last_error()


@pytest.mark.parametrize("changed,code,word", [
    ({"heads": 7}, FK_ERR_SHAPE, "7 query heads"), ({"heads": 0}, FK_ERR_SHAPE, "0 query heads"), ({"q": None}, FK_ERR_INVALID, "null"),
    ({"out": None}, FK_ERR_INVALID, "null"), ({"lengths": None}, FK_ERR_INVALID, "null"), ({"workspace": None}, FK_ERR_INVALID, "null"),
    ({"out": BASE}, FK_ERR_INVALID, "over the queries"), ({"q": BASE + 8}, FK_ERR_ALIGNMENT, "16-byte"), ({"lse": BASE + 2}, FK_ERR_ALIGNMENT, "4-byte"),
    ({"strides": (1024, 1020, 128)}, FK_ERR_ALIGNMENT, "1020"), ({"table_pages": 0}, FK_ERR_SHAPE, "no columns"),
    ({"table": None, "batch": 5}, FK_ERR_SHAPE, "own a page each"), ({"table_pages": 1 << 30}, FK_ERR_SHAPE, "tokens a sequence")])
def test_attention_refused(changed, code, word):
    assert _attend(_cache(), **changed) == code
    assert word in last_error()


@pytest.mark.parametrize("strides", [(0, 128, 256, 128), (256, 128, 256, 0), (64, 128, 256, 128), (256, 128, 256, 120)])
def test_rows_read_over_one_another_are_refused(strides):
    assert _read(_cache(), strides=strides) == FK_ERR_SHAPE and "over one another" in last_error()


@pytest.mark.parametrize("strides", [(128, 128, 256, 128), (256, 128, 128, 128), (256, 128, 192, 128), (256, 128, -128, 128),
                                     (256, 128, 136, 256), (384, 256, 1 << 62, 64), (256, 128, 256, 256), (256, 128, 0, 128)])
def test_strides_that_only_together_lay_rows_over_one_another_are_refused(strides):
    """Tokens and heads each a row or more apart, but one token's last head on another token's first."""
    assert _read(_cache(), strides=strides, v=BASE + (1 << 30), tokens=5) == FK_ERR_SHAPE and "over one another" in last_error()


@pytest.mark.parametrize("heads,tokens", [(1, 4), (2, 3), (3, 5), (5, 2)])
def test_rows_apart_are_told_from_rows_that_meet(heads, tokens):
    """Every pair of strides up to some rows, against the elements themselves; what is let through fails for want of a device, or
    (as keys over values) on purpose."""
    for token in range(-640, 641, 64):
        for head in range(-640, 641, 64):
            firsts = sorted(token * t + head * h for t in range(tokens) for h in range(heads))
            apart = all(y - x >= 64 for x, y in zip(firsts, firsts[1:]))
            # Values elsewhere meet nothing; the keys' own place is refused in other words.
            code = _read(_cache(head_dim=64, kv_heads=heads), strides=(token, head, token, head), tokens=tokens)
            assert code == (FK_ERR_INVALID if apart else FK_ERR_SHAPE), (token, head)
            assert "over one another" in last_error()


@pytest.mark.parametrize("offset,strides", [(0, (256, 128, 256, 128)), (0, (256, 128, 512, 128)), (256, (256, 128, 256, 128)),
                                            (16, (512, 128, 512, 128)), (-512, (256, 128, 256, 128)), (2 * 1024, (512, 256, 512, 256))])
def test_keys_read_over_values_are_refused(offset, strides):
    assert _read(_cache(), v=BASE + offset, strides=strides, tokens=5) == FK_ERR_INVALID
    assert "keys and values" in last_error()


@pytest.mark.parametrize("changed,word", [
    ({"out": BASE + 16}, "output may not lie over the queries"), ({"out": BASE + 3 * 2048 - 16}, "output may not lie over the queries"),
    ({"out": BASE - 3 * 2048 + 16}, "output may not lie over the queries"),
    ({"out": BASE, "strides": (4096, 1024, 128)}, "output may not lie over the queries"),
    ({"out": BASE + 3 * 2048, "strides": (-1024, 1024, 128), "q": BASE + 6 * 2048}, "output may not lie over the queries"),
    ({"lse": BASE + 64}, "lse may not lie over the queries"), ({"lse": BASE + 3 * 2048 - 4}, "lse may not lie over the queries"),
    ({"lse": BASE + (1 << 20) + 16}, "lse may not lie over the output"), ({"lse": BASE + (1 << 20) - 4}, "lse may not lie over the output")])
def test_outputs_that_begin_inside_something_are_refused(changed, word):
    """Three sequences of one query, 8 heads of 128: 2048 bytes each."""
    assert _attend(_cache(), **changed) == FK_ERR_INVALID
    assert word in last_error()


@pytest.mark.parametrize("sizes", [{"queries": 1 << 28}, {"batch": 1 << 20, "queries": 1 << 12}, {"batch": 0xffffffff, "queries": 0xffffffff}])
def test_more_rows_than_memory_holds_are_refused(sizes):
    assert _attend(_cache(), **sizes) == FK_ERR_SHAPE and "more rows" in last_error()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scales_that_are_not_finite_are_refused(scale):
    assert _attend(_cache(), scale=scale) == FK_ERR_INVALID and "not finite" in last_error()


def test_empty_calls_need_no_device():
    assert _write(_cache(), tokens=0) == FK_OK and _read(_cache(), tokens=0) == FK_OK
    assert _attend(_cache(), batch=0) == FK_OK and _attend(_cache(), queries=0) == FK_OK


def test_tensors_on_the_cpu_are_refused():
    codes, params = torch.zeros(1, 1, 16, 64, dtype=torch.uint8), torch.zeros(1, 1, 16, 2, 2, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv_cache.Cache(codes, params, codes, params)


@pytest.mark.parametrize("dim", [64, 128])
def test_the_layouts_place_every_channel_once(dim):
    for place in (key_nibble, value_nibble):
        assert sorted(place(d, dim) for d in range(dim)) == list(range(dim))


def test_the_plain_rule():
    """Ends read back near themselves, every value within half a scale, ties upwards."""
    x = np.array([-1.0, 0.875, -0.9375, -0.8125] + [0.0] * 28)
    codes, scale, low = quantise(x, 32, torch.bfloat16)
    assert scale[0] == 0.125 and low[0] == -1.0
    assert codes[:4].tolist() == [0, 15, 1, 2] and (codes[4:] == 8).all()
    rng = np.random.default_rng(0)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.from_numpy(rng.standard_normal(128)).to(dtype).double().numpy()
        codes, scale, low = quantise(x, 64, dtype)
        back = np.repeat(low, 64) + codes * np.repeat(scale, 64)
        assert (np.abs(back - x) <= np.repeat(scale, 64) / 2).all() and codes.max() == 15 and codes.min() == 0


def test_status_words_that_a_kernel_cannot_write_are_refused():
    there, here = torch.device("cuda", 0), torch.device("cpu")
    assert kv_cache._status_words(None, there) is None
    with pytest.raises(RuntimeError, match="status must live on the cache's device cuda:0"):
        kv_cache._status_words(torch.zeros(8, dtype=torch.int32), there)
    for bad in (torch.zeros(8), torch.zeros(8, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="4 words or more"):
            kv_cache._status_words(bad, here)
    words = torch.zeros(8, dtype=torch.int32)
    assert kv_cache._status_words(words[4:], here) == words.data_ptr() + 16


def _sizes_alone():
    """What the checks look at of a cache, on the device whose tensors have sizes and no content."""
    return types.SimpleNamespace(device=torch.device("meta"), dtype=torch.bfloat16, kv_heads=2, head_dim=128, view=None)


def test_counts_past_32_bits_are_refused():
    """They would reach the entries as what is left of them: 2^32 + 3 tokens as 3."""
    cache, many = _sizes_alone(), (1 << 32) + 3
    rows = torch.empty(1, 2, 128, dtype=torch.bfloat16, device="meta").expand(many, 2, 128)
    slots = torch.empty(many, dtype=torch.int32, device="meta")
    for call in (lambda: kv_cache.write(cache, rows, rows, slots), lambda: kv_cache.read(cache, slots, rows, rows)):
        with pytest.raises(ValueError, match="4294967299 tokens are more than a call counts"):
            call()
    def attend(batch=1, queries=1, heads=4, pages=2):
        q = torch.empty(1, 1, 1, 128, dtype=torch.bfloat16, device="meta").expand(batch, queries, heads, 128)
        kv_cache.attend(q, cache, torch.empty(batch, dtype=torch.int32, device="meta"),
                        torch.empty(batch, pages, dtype=torch.int32, device="meta"))
    for name, count in (("batch", many), ("queries", many), ("heads", many + 1), ("pages", many)):
        with pytest.raises(ValueError, match="more than a call counts"):
            attend(**{name: count})


@pytest.mark.parametrize("places", [(0, 2, 1, 3), (0, 1, 0, 3), (0, 1, 2, 1), (0, 0, 2, 3), (0, 1, 2, 2)])
@pytest.mark.parametrize("shift", [0, -16, 16])
def test_writes_to_buffers_over_one_another_are_refused(places, shift):
    """Codes of 4 x 16 x 2 rows of 64 bytes and parameters of 8: buffers 8192 bytes apart, but for two."""
    names = ("k_codes", "k_params", "v_codes", "v_params")
    at = {name: BASE + (1 << 20) + 8192 * place for name, place in zip(names, places)}
    if places == (0, 2, 1, 3):  # all apart: moved into a neighbour
        at["v_codes"] -= 16 + abs(shift)
    else:
        at[names[max(i for i in range(4) if places.count(places[i]) > 1)]] += shift
    assert _write(_cache(**at)) == FK_ERR_INVALID
    assert "buffers lie over one another" in last_error()

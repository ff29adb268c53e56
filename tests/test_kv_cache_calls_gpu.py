"""The 4-bit cache's calls: outputs beside one another in memory, what a bad index is reported as, and every variant of the attention
that the device's size and the number of segments choose."""
import pytest
import torch

from ferro_kittens_b200 import FerroKittensError, kv_cache

pytestmark = pytest.mark.gpu


def test_keys_and_values_read_side_by_side(device):
    """Into one buffer, [tokens, 2, heads, 128] for instance: near one another, but not over."""
    heads, tokens = 3, 9
    cache = kv_cache.new(2, 16, heads, device=device)
    slots = torch.arange(tokens, device=device)
    kv_cache.write(cache, *(torch.randn(tokens, heads, 128, device=device).bfloat16() for _ in range(2)), slots)
    want = kv_cache.read(cache, slots)
    for shape, dim in (((tokens, 2, heads, 128), 1), ((tokens, heads, 2, 128), 2), ((2, tokens, heads, 128), 0)):
        both = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        k, v = both.unbind(dim)
        kv_cache.read(cache, slots, k, v)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    with pytest.raises(FerroKittensError, match="keys and values"):
        kv_cache.read(cache, slots, k, k)

"""The 4-bit cache's calls: outputs beside one another in memory, what a bad index is reported as, and every variant of the attention
that the device's size and the number of segments choose."""
import numpy as np
import pytest
import torch

from ferro_kittens_b200 import FerroKittensError, gemm, kv_cache

from test_kv_cache_gpu import _compare, _random_cache

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


def test_an_output_between_the_queries_of_a_projection(device):
    """Of [queries, keys, values] side by side, one sequence: the output may take the keys' place, and not a part of the queries'."""
    cache = kv_cache.new(2, 64, 2, device=device)
    slots = torch.arange(90, device=device)
    kv_cache.write(cache, *(torch.randn(90, 2, 128, device=device).bfloat16() for _ in range(2)), slots)
    lengths, table = torch.tensor([90], dtype=torch.int32, device=device), torch.tensor([[0, 1]], dtype=torch.int32, device=device)
    wide = torch.randn(1, 1, 12, 128, device=device).bfloat16()
    q = wide[:, :, :4]
    want, _ = kv_cache.attend(q, cache, lengths, table)
    got, _ = kv_cache.attend(q, cache, lengths, table, out=wide[:, :, 4:8])
    assert got.data_ptr() == wide[:, :, 4:8].data_ptr() and torch.equal(got, want)
    for begin in (0, 1, 3):
        with pytest.raises(FerroKittensError, match="over the queries"):
            kv_cache.attend(q, cache, lengths, table, out=wide[:, :, begin:begin + 4])
    # Two sequences whose queries lie far apart: the output fits in the gap.
    lengths, table = torch.tensor([90, 33], dtype=torch.int32, device=device), table.expand(2, 2).contiguous()
    far = torch.randn(2, 5, 4, 128, device=device).bfloat16()
    q = far[:, :1]
    want, _ = kv_cache.attend(q, cache, lengths, table)
    got, _ = kv_cache.attend(q, cache, lengths, table, out=far[0, 2:4].unsqueeze(1))
    assert torch.equal(got, want)


@pytest.mark.parametrize("slot,wide", [(1 << 40, True), ((7 << 32) + 3, True), ((1 << 63) - 1, True), (16, True), (16, False), ((1 << 31) - 1, False)])
def test_a_bad_slot_is_reported_whole(device, slot, wide):
    cache = kv_cache.new(2, 8, 1, device=device)
    x = torch.randn(2, 1, 128, device=device).bfloat16()
    slots = torch.tensor([3, slot], dtype=torch.int64 if wide else torch.int32, device=device)
    for call in (lambda status: kv_cache.write(cache, x, x, slots, status), lambda status: kv_cache.read(cache, slots, status=status)):
        status = gemm.new_status(device)
        call(status)
        with pytest.raises(FerroKittensError, match=f"slot {slot} of token 1 lies outside the cache"):
            gemm.check_status(status)


def test_status_words_elsewhere_are_refused_by_every_call(device):
    cache = kv_cache.new(2, 8, 1, device=device)
    x = torch.randn(2, 1, 128, device=device).bfloat16()
    slots, lengths = torch.arange(2, device=device), torch.ones(2, dtype=torch.int32, device=device)
    for status, error in ((torch.zeros(8, dtype=torch.int32), RuntimeError), (torch.zeros(8, dtype=torch.int64, device=device), ValueError),
                          (torch.zeros(2, dtype=torch.int32, device=device), ValueError)):
        for call in (lambda: kv_cache.write(cache, x, x, slots, status), lambda: kv_cache.read(cache, slots, status=status),
                     lambda: kv_cache.attend(x, cache, lengths, status=status)):
            with pytest.raises(error, match="status must"):
                call()


@pytest.mark.parametrize("ratio", [4, 12])
def test_calls_in_a_row_see_what_those_before_them_wrote(device, ratio):
    """Tables, lengths, slots, queries and rows that change in place between calls which follow each other without a pause, against the
    same calls with a pause after each."""
    batch, kv_heads, page_size, per, steps = 6, 2, 16, 12, 60
    g = torch.Generator(device=device)
    g.manual_seed(3)
    def draw(*shape):
        return torch.randn(*shape, device=device, generator=g).bfloat16()
    orders = [torch.randperm(batch * per, device=device, generator=g).to(torch.int32).view(batch, per) for _ in range(steps)]
    counts = [torch.randint(1, per * page_size, (batch,), device=device, generator=g, dtype=torch.int32) for _ in range(steps)]
    places = [torch.randperm(batch * per * page_size, device=device, generator=g)[:50] for _ in range(steps)]
    keys, values, asked = ([draw(*shape) for _ in range(steps)] for shape in ((50, kv_heads, 128), (50, kv_heads, 128),
                                                                              (batch, 1, kv_heads * ratio, 128)))
    rows = draw(batch * per * page_size, kv_heads, 128)

    def run(pause):
        cache, workspace = kv_cache.new(batch * per, page_size, kv_heads, device=device), kv_cache.workspace(device)
        kv_cache.write(cache, rows, rows, torch.arange(batch * per * page_size, device=device))
        table, lengths, slots, k, v, q = (torch.empty_like(x[0]) for x in (orders, counts, places, keys, values, asked))
        seen = []
        torch.cuda.synchronize()
        for i in range(steps):
            for ours, theirs in ((table, orders), (lengths, counts), (slots, places), (k, keys), (v, values), (q, asked)):
                ours.copy_(theirs[i])
            pause()
            kv_cache.write(cache, k, v, slots)
            pause()
            seen += kv_cache.attend(q, cache, lengths, table, workspace=workspace)
            pause()
            seen += kv_cache.read(cache, slots)
            pause()
            q.mul_(0.5)
            seen += kv_cache.attend(q, cache, lengths, table, window=20, sinks=3, workspace=workspace)
            pause()
        torch.cuda.synchronize()
        return seen

    for x, y in zip(run(lambda: None), run(torch.cuda.synchronize)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("ratio", [3, 12])
@pytest.mark.parametrize("plan", ["one block", "one block for long tables", "two blocks", "three blocks"])
def test_every_plan_of_the_attention(device, head_dim, group, dtype, ratio, plan):
    """Segments (a sequence's kv head) up to the number of SMs, up to twice it with tables of more and of less than 8192 tokens, and
    beyond: blocks alone on an SM, two and three of them, for 8 rows and for 16."""
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    kv_heads = 2 if ratio == 3 else 1
    segments = {"one block": sms - 3, "one block for long tables": 2 * sms - 2, "two blocks": sms + 2, "three blocks": 2 * sms + 9}[plan]
    batch = -(-segments // kv_heads)
    seed = 2 * head_dim + group + ratio + len(plan)
    rng = np.random.default_rng(seed)
    for page_size, window, sinks in ((16, None, 0), (48, 100, 5), (7, None, 0), (10, 37, 20)):
        per = -(-(9000 if plan == "one block for long tables" else 400) // page_size)
        pool = 6 * 48 // page_size
        cache = _random_cache(device, pool, page_size, kv_heads, head_dim, group, dtype, seed)
        lengths = torch.from_numpy(np.exp(rng.uniform(0, np.log(400), batch)).astype(np.int32))
        lengths[rng.integers(batch)], lengths[-1] = 0, 399
        table = torch.full((batch, per), -1, dtype=torch.int32)
        used = -(-400 // page_size)
        table[:, :used] = torch.from_numpy(rng.integers(0, pool, (batch, used)).astype(np.int32))
        q = torch.randn(batch, 1, kv_heads * ratio, head_dim, device=device).to(dtype)
        ours, workspace = table.to(device), kv_cache.workspace(device)
        status = gemm.new_status(device)
        out, lse = kv_cache.attend(q, cache, lengths.to(device), ours, window=window, sinks=sinks, workspace=workspace, status=status)
        gemm.check_status(status)
        some = sorted({0, batch - 1, int(lengths.argmin()), *rng.integers(0, batch, 5).tolist()})
        _compare(cache, q[some], lengths[some], table[some], None, window, sinks, out[some], lse[some])
        # A page outside the cache, of the newest tokens of one sequence: noted, and nothing to the others.
        bad = int(rng.integers(batch))
        bad = bad if int(lengths[bad]) else batch - 1
        ours[bad, (int(lengths[bad]) - 1) // page_size] = pool
        status = gemm.new_status(device)
        again, lse_again = kv_cache.attend(q, cache, lengths.to(device), ours, window=window, sinks=sinks, workspace=workspace, status=status)
        with pytest.raises(FerroKittensError, match=f"page {pool} in the table of sequence {bad} lies"):
            gemm.check_status(status)
        others = torch.arange(batch) != bad
        assert torch.equal(again[others], out[others]) and torch.equal(lse_again[others], lse[others])
        assert torch.isfinite(again).all()


def test_a_captured_step_on_two_streams(device):
    """A step captured as two branches, copies and kernels in turn on each, that meet in an attention over what both wrote: replayed
    with other contents, against the same calls one by one. (Its kernels' first calls, if no test ran before, fall into the capture.)"""
    batch, kv_heads, ratio, page_size, per = 4, 2, 6, 16, 20
    cache, plain = (kv_cache.new(batch * per, page_size, kv_heads, 64, 64, device=device) for _ in range(2))
    table = torch.randperm(batch * per, device=device).to(torch.int32).view(batch, per)
    lengths = torch.tensor([300, 1, 77, 320], dtype=torch.int32, device=device)
    spaces = [kv_cache.workspace(device) for _ in range(2)]
    half = batch * per * page_size // 2
    slots = torch.randperm(2 * half, device=device)
    source, rows = (torch.zeros(2 * half, kv_heads, 64, dtype=torch.bfloat16, device=device) for _ in range(2))
    asked, q = (torch.zeros(batch, 2, kv_heads * ratio, 64, dtype=torch.bfloat16, device=device) for _ in range(2))
    side = torch.cuda.Stream(device)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        rows.copy_(source)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            kv_cache.write(cache, rows[half:], rows[half:], slots[half:])
            q.copy_(asked)
            early = kv_cache.attend(q, plain, lengths, table, workspace=spaces[1])
        kv_cache.write(cache, rows[:half], rows[:half], slots[:half])
        back = kv_cache.read(cache, slots[:half])
        main.wait_stream(side)
        late = kv_cache.attend(q, cache, lengths, table, window=100, sinks=4, workspace=spaces[0])
        late_too = kv_cache.attend(q, cache, lengths, table, workspace=spaces[0])
    for _ in range(4):
        source.copy_(torch.randn_like(source))
        asked.copy_(torch.randn_like(asked))
        graph.replay()
        torch.cuda.synchronize()
        kv_cache.write(plain, source, source, slots)
        for x, y in zip((*late, *late_too, *back),
                        (*kv_cache.attend(asked, plain, lengths, table, window=100, sinks=4), *kv_cache.attend(asked, plain, lengths, table),
                         *kv_cache.read(plain, slots[:half]))):
            assert torch.equal(x, y)
        assert torch.isfinite(early[0]).all()

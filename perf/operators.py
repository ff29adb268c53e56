"""A key/value cache held in 4 bits: writing it, reading it back, and attention over it, case by case.

``listed()`` and ``draw()`` say what is run, ``prepare()`` makes the inputs, and ``run()`` makes one pass:
with ``own`` false in elementary torch operations, with ``own`` true through ``ferro_kittens_b200.kv_cache``.

The cache holds one row per (page, kv head, place in the page). A row of ``head_dim`` channels is cut into
groups of ``group`` channels; a group keeps its smallest value ``low`` and ``scale`` = the largest value of the
cache's type that is not above (high - low) / 15, and each channel a code 0..15: the number of k in 0..14
with x - low >= (k + 1/2) * scale. It stands for low + code * scale.

A row's codes, ``head_dim / 2`` bytes, low nibble of a byte first:
  keys    as a matrix [4][head_dim / 32] of runs of 8 nibbles; run [c][w] holds channels 8 * (4 w + c) + 0..7
  values  as a matrix [8][head_dim / 8] of nibbles; nibble [l][n] is channel 8 n + l
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(name, kind, **given):
    base = {"name": name, "kind": kind, "dtype": "bf16", "kv_heads": 8, "head_dim": 128, "group": 64, "page": 64}
    if kind == "attend":
        base |= {"batch": 1, "length": 1024, "ragged": True, "queries": 1, "ratio": 4, "window": 0, "sinks": 0}
    else:
        base |= {"tokens": 1024, "padded": 0}
    return base | given


def listed():
    return [
        # One decoding step of a small batch: the new tokens of 37 sequences, written and read back.
        _case("write_step", "write", tokens=37, padded=3),
        # A prompt's keys and values on their way into the cache, an odd number of tokens, eight kv heads.
        _case("write_prompt", "write", tokens=8191, page=16),
        # Many prompts at once, narrow heads and short groups, fp16.
        _case("write_many", "write", tokens=150001, head_dim=64, group=32, dtype="f16", page=128),
        # A short shared prefix fetched for a new request.
        _case("read_short", "read", tokens=500, kv_heads=2, group=128, dtype="f16", page=16),
        # A long prefix fetched as keys and values for a prompt that continues it.
        _case("read_prefix", "read", tokens=65536, padded=7),
        # One user, a short conversation: the smallest call, where latency counts.
        _case("attend_short", "attend", length=777, ragged=False, page=16),
        # A serving batch of ragged conversations, grouped queries.
        _case("attend_batch", "attend", batch=48, length=4096, ratio=8),
        # Every head with keys of its own, groups as wide as the head.
        _case("attend_heads", "attend", batch=20, length=2000, kv_heads=32, ratio=1, group=128, page=32),
        # One long document: few rows, so the length has to be split.
        _case("attend_long", "attend", length=131072, ragged=False, ratio=8),
        # Guessed tokens checked four at a time, narrow heads, fp16.
        _case("attend_guess", "attend", batch=16, length=8192, queries=4, head_dim=64, group=32, dtype="f16"),
        # A sliding window with the first tokens kept visible, over long histories.
        _case("attend_window", "attend", batch=24, length=32768, ratio=7, kv_heads=4, window=4096, sinks=4),
        # The largest: a full batch of long histories.
        _case("attend_large", "attend", batch=32, length=30000, ratio=8, page=128),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    head_dim = rng.choice([64, 128, 128])
    case = {
        "kind": rng.choice(["write", "read", "attend", "attend", "attend"]),
        "dtype": rng.choice(["bf16", "f16"]),
        "head_dim": head_dim,
        "group": rng.choice([g for g in (32, 64, 128) if g <= head_dim]),
        "kv_heads": rng.choice([1, 2, 3, 4, 5, 8, 8, 16, 32]),
        "page": rng.choice([16, 24, 32, 64, 100, 128, 256]),
    }
    if case["kind"] != "attend":
        case["tokens"] = min(_spread(rng, 1, 150000), 76000000 // (case["kv_heads"] * head_dim))
        case["padded"] = rng.choice([0, 0, 1, 5])
        return case
    case["ratio"] = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    case["queries"] = min(rng.choice([1, 1, 1, 2, 3, 4, 8]), 32 // case["ratio"])
    case["batch"] = _spread(rng, 1, 128)
    # No more rows of the cache, and no more products, than the largest listed case has.
    most = min(3800000, 31000000 // (case["queries"] * case["ratio"])) // (case["batch"] * case["kv_heads"])
    case["length"] = max(case["queries"], _spread(rng, 1, min(131072, most)))
    case["ragged"] = rng.random() < 0.7
    windowed = rng.random() < 0.35
    case["window"] = _spread(rng, 1, 8192) if windowed else 0
    case["sinks"] = rng.choice([0, 1, 4, 37, 128]) if windowed else 0
    return case


def _lengths(case):
    """Tokens of each sequence: all of `length`, or spread between the new tokens and `length`."""
    n, low = case["length"], case["queries"]
    if not case["ragged"]:
        return [n] * case["batch"]
    return [n - int((n - low) * ((i * 0.6180339887498949) % 1.0)) for i in range(case["batch"])]


def _pages_of(case):
    return -(-case["length"] // case["page"])


def _random_cache(case, pages, generator):
    """Codes and parameters of a cache in use: codes bell-shaped over 0..15, groups of unit spread with channels off
    centre, some of them far."""
    device, dtype = "cuda", TYPES[case["dtype"]]
    rows = (pages, case["kv_heads"], case["page"])
    half, groups = case["head_dim"] // 2, case["head_dim"] // case["group"]
    # 16 equally likely codes of a normal variable over [-2.4, 2.4]
    bell = torch.tensor([0, 2, 4, 5, 5, 6, 7, 7, 8, 8, 9, 10, 10, 11, 13, 15], dtype=torch.uint8, device=device)
    pairs = (bell[:, None] * 16 + bell[None, :]).reshape(-1)
    made = []
    for _ in range(2):
        codes = torch.randint(0, 256, rows + (half,), dtype=torch.uint8, device=device, generator=generator)
        codes = pairs[codes.int()]
        scale = 0.32 * (0.7 + 0.6 * torch.rand(rows + (groups,), device=device, generator=generator))
        low = -7.5 * scale + 0.6 * torch.randn(rows + (groups,), device=device, generator=generator)
        made += [codes, torch.stack((scale, low), -1).to(dtype)]
    return {"k_codes": made[0], "k_params": made[1], "v_codes": made[2], "v_params": made[3]}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, page = TYPES[case["dtype"]], case["page"]
    state = {"case": case}
    if case["kind"] == "attend":
        batch, per = case["batch"], _pages_of(case)
        pages = batch * per + 3
        state["cache"] = _random_cache(case, pages, g)
        state["table"] = torch.randperm(pages, device="cuda", generator=g)[: batch * per].to(torch.int32).view(batch, per)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        heads = case["kv_heads"] * case["ratio"]
        state["q"] = torch.randn(batch, case["queries"], heads, case["head_dim"], device="cuda", generator=g).to(dtype)
        state["q"] *= 1.5
    else:
        tokens = case["tokens"]
        pages = -(-tokens // page) + 2
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(tokens, device="cuda")
        slots = (order[at // page] * page + at % page).to(torch.int32)
        slots[tokens - min(case["padded"], tokens - 1):] = -1  # places of a padded batch that hold no token
        state["slots"] = slots
        if case["kind"] == "read":
            state["cache"] = _random_cache(case, pages, g)
        else:
            # The heads' keys and values lie side by side in one projection's output, behind its queries.
            heads = case["kv_heads"]
            wide = torch.randn(tokens, 3 * heads, case["head_dim"], device="cuda", generator=g)
            off = torch.randn(3 * heads, case["head_dim"], device="cuda", generator=g)
            wide += off * (off.abs() > 2) * 3  # a few channels that sit far off centre, as keys have them
            wide = wide.to(dtype)
            state["k"], state["v"] = wide[:, heads:2 * heads], wide[:, 2 * heads:]
            rows = (pages, heads, page)
            state["cache"] = {
                "k_codes": torch.zeros(rows + (case["head_dim"] // 2,), dtype=torch.uint8, device="cuda"),
                "k_params": torch.zeros(rows + (case["head_dim"] // case["group"], 2), dtype=dtype, device="cuda")}
            state["cache"] |= {"v" + name[1:]: torch.zeros_like(t) for name, t in list(state["cache"].items())}
    if own:
        from ferro_kittens_b200 import kv_cache

        # What a serving program makes once and keeps: the cache's handle and the attention's workspace.
        state["handle"] = kv_cache.Cache(**state["cache"])
        state["workspace"] = kv_cache.workspace("cuda")
    return state


def run(state):
    case = state["case"]
    if own:
        from ferro_kittens_b200 import kv_cache

        cache = state["handle"]
        if case["kind"] == "attend":
            return kv_cache.attend(state["q"], cache, state["lengths"], state["table"], window=case["window"] or None,
                                   sinks=case["sinks"], workspace=state["workspace"])
        if case["kind"] == "write":
            kv_cache.write(cache, state["k"], state["v"], state["slots"])
        return kv_cache.read(cache, state["slots"])
    if case["kind"] == "attend":
        return _attend(state)
    if case["kind"] == "write":
        _write(state)
    return _read(state)


# ---------------------------------------------------------------- plain forms

def _unpack_keys(codes):
    """Codes of key rows [..., head_dim / 2] as whole numbers [..., head_dim] in channel order."""
    nibbles = torch.stack((codes & 15, codes >> 4), -1)
    runs = nibbles.reshape(*codes.shape[:-1], 4, codes.shape[-1] // 16, 8)
    return runs.transpose(-3, -2).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def _unpack_values(codes):
    nibbles = torch.stack((codes & 15, codes >> 4), -1)
    matrix = nibbles.reshape(*codes.shape[:-1], 8, codes.shape[-1] // 4)
    return matrix.transpose(-2, -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def _pack_keys(codes):
    runs = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 32, 4, 8).transpose(-3, -2)
    nibbles = runs.reshape(*codes.shape[:-1], codes.shape[-1] // 2, 2)
    return nibbles[..., 0] | (nibbles[..., 1] << 4)


def _pack_values(codes):
    matrix = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 8, 8).transpose(-2, -1)
    nibbles = matrix.reshape(*codes.shape[:-1], codes.shape[-1] // 2, 2)
    return nibbles[..., 0] | (nibbles[..., 1] << 4)


def _values_of(codes, params):
    """low + code * scale in 32 bits; codes [..., head_dim], params [..., groups, 2]."""
    grouped = codes.reshape(*params.shape[:-1], -1).float()
    scale, low = params.float().unbind(-1)
    return (grouped * scale.unsqueeze(-1) + low.unsqueeze(-1)).reshape(codes.shape)


def _quantise(x, group):
    """Codes [..., head_dim] (uint8) and params [..., groups, 2] of rows x; in 64 bits, for values next to a border."""
    wide = x.double().reshape(*x.shape[:-1], -1, group)
    low, span = wide.amin(-1), wide.amax(-1) - wide.amin(-1)
    scale = (span / 15).to(x.dtype)
    below = (scale.view(torch.int16) - 1).view(x.dtype)
    scale = torch.where(scale.double() * 15 > span, below, scale)
    step = scale.double().unsqueeze(-1)
    codes = torch.floor((wide - low.unsqueeze(-1)) / torch.where(step > 0, step, 1.0) + 0.5).clamp(0, 15)
    codes = torch.where(step > 0, codes, 0.0)
    return codes.to(torch.uint8).reshape(x.shape), torch.stack((scale, low.to(x.dtype)), -1)


def _write(state):
    case, cache = state["case"], state["cache"]
    kept = state["slots"] >= 0
    slots = state["slots"][kept].long()
    page, place = slots // case["page"], slots % case["page"]
    for name, pack in (("k", _pack_keys), ("v", _pack_values)):
        codes, params = _quantise(state[name][kept], case["group"])
        cache[name + "_codes"][page, :, place] = pack(codes)
        cache[name + "_params"][page, :, place] = params


def _read(state):
    case, cache = state["case"], state["cache"]
    kept = (state["slots"] >= 0)[:, None, None]
    slots = state["slots"].clamp(min=0).long()
    page, place = slots // case["page"], slots % case["page"]
    k = _values_of(_unpack_keys(cache["k_codes"][page, :, place]), cache["k_params"][page, :, place])
    v = _values_of(_unpack_values(cache["v_codes"][page, :, place]), cache["v_params"][page, :, place])
    dtype = TYPES[case["dtype"]]
    return torch.where(kept, k, 0.0).to(dtype), torch.where(kept, v, 0.0).to(dtype)


def _visible(case, lengths, longest):
    """[batch, queries, longest]: which tokens each query sees; the queries are a sequence's last tokens."""
    at = torch.arange(longest, device=lengths.device)
    of = lengths.long()[:, None] - case["queries"] + torch.arange(case["queries"], device=lengths.device)
    seen = at <= of[..., None]
    if case["window"]:
        seen &= (at > of[..., None] - case["window"]) | (at < case["sinks"])
    return seen


def _attend(state):
    case, cache, q = state["case"], state["cache"], state["q"]
    batch, queries, heads, dim = q.shape
    longest = case["length"]
    at = torch.arange(longest, device=q.device)
    page, place = state["table"].long()[:, at // case["page"]], at % case["page"]
    k = _values_of(_unpack_keys(cache["k_codes"][page, :, place]), cache["k_params"][page, :, place])
    scores = q.float().view(batch, queries, case["kv_heads"], case["ratio"], dim).permute(0, 2, 1, 3, 4)
    scores = scores.reshape(batch, case["kv_heads"], queries * case["ratio"], dim) @ k.permute(0, 2, 3, 1)
    del k
    scores = scores.view(batch, case["kv_heads"], queries, case["ratio"], longest) * dim ** -0.5
    seen = _visible(case, state["lengths"], longest)[:, None, :, None, :]
    scores = scores.masked_fill(~seen, -math.inf)
    peak = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weights = torch.exp(scores - peak)
    total = weights.sum(-1, keepdim=True)
    lse = (peak + torch.log(total)).squeeze(-1)
    v = _values_of(_unpack_values(cache["v_codes"][page, :, place]), cache["v_params"][page, :, place])
    out = weights.view(batch, case["kv_heads"], queries * case["ratio"], longest) @ v.permute(0, 2, 1, 3)
    out = out.view(batch, case["kv_heads"], queries, case["ratio"], dim) / total.clamp(min=1e-38)
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, queries, heads, dim).to(q.dtype)
    return out, lse.permute(0, 2, 1, 3).reshape(batch, queries, heads)


# ---------------------------------------------------------------- what a pass cannot do without

def _row_bytes(case):
    """One token's keys and values of one kv head: codes and parameters."""
    return case["head_dim"] + 2 * 4 * (case["head_dim"] // case["group"])


def work(case):
    dim, kv = case["head_dim"], case["kv_heads"]
    if case["kind"] != "attend":
        kept = case["tokens"] - min(case["padded"], case["tokens"] - 1)
        raw = 2 * kv * dim * 2
        moved = kept * kv * _row_bytes(case) + case["tokens"] * raw + 4 * case["tokens"]  # read back
        if case["kind"] == "write":
            moved += kept * (raw + kv * _row_bytes(case)) + 4 * case["tokens"]
        return {"bytes": moved, "flops": 0}
    heads, rows, pairs = kv * case["ratio"], 0, 0
    for n in _lengths(case):
        first = n - case["queries"]
        if not case["window"]:
            rows += n
            pairs += sum(first + i + 1 for i in range(case["queries"]))
            continue
        begin = max(0, first + 1 - case["window"])
        rows += n - begin + min(case["sinks"], begin)
        for i in range(first, n):
            begin = max(0, i + 1 - case["window"])
            pairs += i + 1 - begin + min(case["sinks"], begin)
    asked = case["batch"] * case["queries"] * heads
    return {"bytes": rows * kv * _row_bytes(case) + asked * (2 * dim * 2 + 4) + 4 * case["batch"] * (1 + _pages_of(case)),
            "flops": 4 * dim * heads * pairs}


# ---------------------------------------------------------------- the definition in 64 bits

def _code_at(codes, channel, keys, dim):
    """The codes of one channel of rows [..., head_dim / 2], by the place the layout gives it."""
    if keys:
        run, inside = divmod(channel, 8)
        nibble = ((run % 4) * (dim // 32) + run // 4) * 8 + inside
    else:
        nibble = (channel % 8) * (dim // 8) + channel // 8
    byte = codes[..., nibble // 2]
    return byte // 16 if nibble % 2 else byte % 16


def _rows_64(cache, name, page, place, case):
    """The values of rows (page[i], every head, place[i]) in 64 bits: [rows, heads, head_dim]."""
    codes, params = cache[name + "_codes"], cache[name + "_params"].double()
    codes, params = codes[page, :, place].long(), params[page, :, place]
    columns = [_code_at(codes, d, name == "k", case["head_dim"]) for d in range(case["head_dim"])]
    columns = [params[..., d // case["group"], 1] + c * params[..., d // case["group"], 0] for d, c in enumerate(columns)]
    return torch.stack(columns, -1)


def _rounded_64(x, case):
    """What a written row stands for, in 64 bits."""
    bits, least = (8, -133) if case["dtype"] == "bf16" else (11, -24)
    x = x.double().unflatten(-1, (-1, case["group"]))
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    fine = (high - low) / 15
    unit = torch.exp2(torch.clamp(torch.frexp(fine).exponent.double() - bits, min=float(least)))
    scale = torch.floor(fine / unit) * unit
    code = torch.zeros_like(x)
    for k in range(15):
        code += ((x - low) * 2 >= (2 * k + 1) * scale) & (scale > 0)
    return (low + code * scale).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "write":
        kept = (state["slots"] >= 0)[:, None, None]
        return tuple(torch.where(kept, _rounded_64(state[name], case), 0.0) for name in ("k", "v"))
    cache, size = state["cache"], case["page"]
    if case["kind"] == "read":
        slots = state["slots"].tolist()
        page = torch.tensor([s // size if s >= 0 else 0 for s in slots], device="cuda")
        place = torch.tensor([s % size if s >= 0 else 0 for s in slots], device="cuda")
        kept = (state["slots"] >= 0)[:, None, None]
        return tuple(torch.where(kept, _rows_64(cache, name, page, place, case), 0.0) for name in ("k", "v"))
    batch, queries, heads, dim = state["q"].shape
    out = torch.zeros(batch, queries, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, queries, heads), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        at = torch.arange(n, device="cuda")
        page, place = state["table"][b].long()[at // size], at % size
        k = _rows_64(cache, "k", page, place, case).transpose(0, 1)  # [kv, n, dim]
        v = _rows_64(cache, "v", page, place, case).transpose(0, 1)
        for t in range(queries):
            here = n - queries + t
            hidden = at > here
            if case["window"]:
                hidden = hidden | ((at <= here - case["window"]) & (at >= case["sinks"]))
            q = state["q"][b, t].double().view(case["kv_heads"], case["ratio"], dim)
            s = torch.einsum("hrd,hnd->hrn", q, k) / math.sqrt(dim)
            s = s.masked_fill(hidden, -math.inf)
            total = torch.logsumexp(s, -1)
            lse[b, t] = total.reshape(-1)
            out[b, t] = torch.einsum("hrn,hnd->hrd", torch.exp(s - total[..., None]), v).reshape(heads, dim)
    return out, lse

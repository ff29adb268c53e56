"""The 4-bit key/value cache in plain 64-bit arithmetic, row by row from its definition, for the tests."""
import math

import numpy as np
import torch

BITS = {torch.bfloat16: (8, -133), torch.float16: (11, -24)}  # significand bits, exponent of the smallest value


def at_most(x: float, dtype) -> float:
    """The largest value of the type not above x >= 0."""
    if x == 0:
        return 0.0
    bits, least = BITS[dtype]
    unit = 2.0 ** max(math.frexp(x)[1] - bits, least)
    return math.floor(x / unit) * unit


def quantise(x: np.ndarray, group: int, dtype):
    """(codes [D], scale [D / group], low [D / group]) of one row of float64 values of the type."""
    codes, scales, lows = [], [], []
    for g in x.reshape(-1, group):
        if not np.isfinite(g).all():
            codes += [0] * group
            scales.append(0.0)
            lows.append(math.nan)
            continue
        low, high = g.min(), g.max()
        scale = at_most((high - low) / 15 if high - low < 1e308 else math.inf, dtype)
        for v in g:
            # Exact: sums of three values of at most 11 significant bits are compared through fractions of powers of two.
            codes.append(sum(_not_below(v, low, (k + 0.5) * scale) for k in range(15)) if scale > 0 else 0)
        scales.append(scale)
        lows.append(low)
    return np.array(codes), np.array(scales), np.array(lows)


def _not_below(v: float, low: float, border: float) -> bool:
    """v - low >= border, exactly."""
    return math.fsum((v, -low, -border)) >= 0


def key_nibble(d: int, dim: int) -> int:
    """Where channel d's code stands in a row of keys: runs of 8 channels in a matrix [4][dim / 32]."""
    w, c = divmod(d // 8, 4)
    return (c * (dim // 32) + w) * 8 + d % 8


def value_nibble(d: int, dim: int) -> int:
    """Where channel d's code stands in a row of values: a matrix [8][dim / 8] of nibbles."""
    return (d % 8) * (dim // 8) + d // 8


def pack(codes: np.ndarray, place) -> np.ndarray:
    row = np.zeros(len(codes) // 2, np.uint8)
    for d, c in enumerate(codes):
        n = place(d, len(codes))
        row[n // 2] |= int(c) << (4 * (n % 2))
    return row


def unpack(rows: np.ndarray, place) -> np.ndarray:
    """Codes [..., dim] in channel order of packed rows [..., dim / 2]."""
    dim = 2 * rows.shape[-1]
    n = np.array([place(d, dim) for d in range(dim)])
    return (rows[..., n // 2] >> (4 * (n % 2))) & 15


class Plain:
    """A cache's content on the CPU in 64 bits: codes, scale and low of every row, by slot."""

    def __init__(self, cache):
        self.page_size, self.group, self.dim = cache.page_size, cache.group, cache.head_dim
        def by_slot(t):
            return t.transpose(1, 2).reshape(-1, cache.kv_heads, *t.shape[3:]).cpu()
        self.k_codes = unpack(by_slot(cache.k_codes).numpy(), key_nibble)
        self.v_codes = unpack(by_slot(cache.v_codes).numpy(), value_nibble)
        self.k_params = by_slot(cache.k_params).double().numpy()
        self.v_params = by_slot(cache.v_params).double().numpy()

    def values(self, which: str, slots):
        """(values, scales) [tokens, kv_heads, dim] of the rows at `slots`."""
        codes, params = (self.k_codes, self.k_params) if which == "k" else (self.v_codes, self.v_params)
        scale, low = (np.repeat(params[slots][..., i], self.group, -1) for i in (0, 1))
        return low + codes[slots] * scale, scale


def attention(plain: Plain, q: np.ndarray, length: int, pages, scale: float, window: int | None, sinks: int):
    """(out, lse, room, slack) of one sequence; q [queries, heads, dim]. `room` is sum p * scale * |code - 8|, what a relative
    error of every weight moves an output by; `slack` the same for sum p |v|; both [queries, heads, dim]."""
    queries, heads, dim = q.shape
    out, room, slack = (np.zeros(q.shape) for _ in range(3))
    lse = np.full((queries, heads), -math.inf)
    size = np.zeros((queries, heads))
    kv = plain.k_codes.shape[1]
    for t in range(queries):
        i = length - queries + t
        seen = [j for j in range(min(i + 1, length)) if window is None or j > i - window or j < sinks]
        if not seen:
            continue
        slots = np.array([pages[j // plain.page_size] * plain.page_size + j % plain.page_size for j in seen])
        k, _ = plain.values("k", slots)
        v, v_scale = plain.values("v", slots)
        v_off = v_scale * np.abs(plain.v_codes[slots].astype(np.float64) - 8)
        for h in range(heads):
            g = h // (heads // kv)
            s = scale * (k[:, g] @ q[t, h])
            size[t, h] = (abs(scale) * (np.abs(k[:, g]) @ np.abs(q[t, h]))).max()
            peak = s.max()
            p = np.exp(s - peak)
            lse[t, h] = peak + math.log(p.sum())
            p /= p.sum()
            out[t, h], room[t, h], slack[t, h] = p @ v[:, g], p @ v_off[:, g], p @ np.abs(v[:, g])
    return out, lse, room, slack, size

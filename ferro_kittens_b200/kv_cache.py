"""A key/value cache in 4 bits through the C ABI: tokens quantised as they are written, rows read back, and
attention of each sequence's newest tokens over its rows (decoding, and the short runs of tokens of a guess
being checked), paged, with grouped heads, and a sliding window that keeps the first tokens visible.

No counterpart in the reference, whose attention (``examples/src/flash_forward.rs``) reads whole planes. The
format stands beside ``fk_cache_t`` in ``include/ferro_kittens.h``. torch supplies memory and streams only; there
is no CPU path.

    cache = kv_cache.new(pages, page_size, kv_heads)
    workspace = kv_cache.workspace(device)                       # kept, like the cache
    kv_cache.write(cache, k, v, slots)                           # k, v [tokens, kv_heads, 128]; slot = page * page_size + place
    out, lse = kv_cache.attend(q, cache, lengths, table, workspace=workspace)
    k, v = kv_cache.read(cache, slots)
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import FK_BF16, FK_F16, CacheView, check, library

#: Channels that share a scale and a smallest value, unless a cache asks for another number.
GROUP = 64
HEAD_DIMS = (64, 128)
GROUPS = (32, 64, 128)
_ELEMENTS = {torch.bfloat16: FK_BF16, torch.float16: FK_F16}


class Cache:
    """The four tensors of a cache and what the kernels need to know of them.

    ``k_codes``, ``v_codes``: uint8 ``[pages, kv_heads, page_size, head_dim / 2]``; ``k_params``, ``v_params``: bf16 or fp16
    ``[pages, kv_heads, page_size, head_dim / group, 2]`` (scale, smallest value). All contiguous, on one device."""

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "pages", "page_size", "kv_heads", "head_dim", "group",
                 "dtype", "device", "view")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor):
        for name, tensor in (("k_codes", k_codes), ("k_params", k_params), ("v_codes", v_codes), ("v_params", v_params)):
            if not tensor.is_cuda:
                raise RuntimeError(f"{name} must live on a CUDA device: there is no CPU path")
            if tensor.device != k_codes.device:
                raise ValueError("a cache's tensors must live on one device")
            if not tensor.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        if k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8:
            raise ValueError("codes must be uint8 tensors")
        if k_params.dtype not in _ELEMENTS or v_params.dtype != k_params.dtype:
            raise ValueError("k_params and v_params must share bfloat16 or float16")
        if k_codes.dim() != 4 or k_codes.shape != v_codes.shape:
            raise ValueError("k_codes and v_codes must share one [pages, kv_heads, page_size, head_dim / 2] shape")
        if (k_params.dim() != 5 or k_params.shape != v_params.shape or k_params.shape[:3] != k_codes.shape[:3]
                or k_params.shape[4] != 2):
            raise ValueError("k_params and v_params must share the shape [pages, kv_heads, page_size, head_dim / group, 2]")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.pages, self.kv_heads, self.page_size, half = k_codes.shape
        self.head_dim = 2 * half
        groups = k_params.shape[3]
        if self.head_dim not in HEAD_DIMS or groups == 0 or self.head_dim % groups or self.head_dim // groups not in GROUPS:
            raise ValueError(f"heads of {self.head_dim} in {groups} groups: head_dim is 64 or 128, a group 32, 64 or 128 channels")
        self.group = self.head_dim // groups
        self.dtype, self.device = k_params.dtype, k_codes.device
        self.view = ctypes.byref(CacheView(k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(),
                                           self.pages, self.page_size, self.kv_heads, self.head_dim, self.group,
                                           _ELEMENTS[self.dtype]))


def new(pages: int, page_size: int, kv_heads: int, head_dim: int = 128, group: int = GROUP,
        dtype: torch.dtype = torch.bfloat16, device="cuda") -> Cache:
    """An empty cache (every row reads back as zeros)."""
    if head_dim not in HEAD_DIMS or group not in GROUPS or group > head_dim:
        raise ValueError(f"head_dim {head_dim} in groups of {group}: head_dim is 64 or 128, a group 32, 64 or 128 channels")
    if dtype not in _ELEMENTS:
        raise ValueError("a cache is of bfloat16 or float16")
    rows = (pages, kv_heads, page_size)
    codes = [torch.zeros(rows + (head_dim // 2,), dtype=torch.uint8, device=device) for _ in range(2)]
    params = [torch.zeros(rows + (head_dim // group, 2), dtype=dtype, device=device) for _ in range(2)]
    return Cache(codes[0], params[0], codes[1], params[1])


def workspace(device="cuda") -> torch.Tensor:
    """The zeroed workspace of :func:`attend` on ``device``, for calls of any shape. Every call leaves its counters zero
    again; calls that share one must not overlap on the device."""
    sm_count = torch.cuda.get_device_properties(device).multi_processor_count
    return torch.zeros(library().fk_cache_attention_workspace_bytes(sm_count), dtype=torch.uint8, device=device)


def _on(device: torch.device, call) -> None:
    """``call(stream handle)`` with ``device`` current, on torch's current stream of it. (The raw handle: a step of a small
    batch takes the device some ten microseconds, and a stream object alone takes the host three.)"""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if torch._C._cuda_getDevice() == device.index:
        check(call(stream))
    else:
        with torch.cuda.device(device):
            check(call(stream))


def _require(name: str, tensor: torch.Tensor, cache: Cache, dims: int) -> None:
    if tensor.device != cache.device:
        raise RuntimeError(f"{name} must live on the cache's device {cache.device}: there is no CPU path")
    if (tensor.dtype is not cache.dtype or tensor.dim() != dims or tensor.shape[-1] != cache.head_dim
            or tensor.stride(-1) != 1):
        raise ValueError(f"{name} must be a {dims}-dimensional {cache.dtype} tensor of contiguous rows of {cache.head_dim}")


def _require_indices(name: str, tensor: torch.Tensor, cache: Cache, count: int | None = None, wide: bool = False) -> None:
    if tensor.device != cache.device:
        raise RuntimeError(f"{name} must live on the cache's device {cache.device}: there is no CPU path")
    if (not (tensor.dtype is torch.int32 or wide and tensor.dtype is torch.int64) or tensor.dim() != 1
            or count is not None and tensor.shape[0] != count or not tensor.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {'int32 or int64' if wide else 'int32'} vector"
                         + (f" of {count} entries" if count is not None else ""))


def _require_counts(**counts: int) -> None:
    for name, count in counts.items():  # the entries take 32 bits, and would be given the rest of a longer number
        if count >= 1 << 32:
            raise ValueError(f"{count} {name} are more than a call counts")


def _status_words(status: torch.Tensor | None, device: torch.device) -> int | None:
    """The address of a call's status words, which the kernels write where they find them."""
    if status is None:
        return None
    if status.device != device:
        raise RuntimeError(f"status must live on the cache's device {device}: its kernels write it")
    if status.dtype is not torch.int32 or not status.is_contiguous() or status.numel() < 4:
        raise ValueError("status must be a contiguous int32 tensor of 4 words or more (gemm.new_status makes one)")
    return status.data_ptr()


def _rows(entry, cache: Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, status, *more) -> None:
    tokens = slots.shape[0]
    for name, tensor in (("k", k), ("v", v)):
        _require(name, tensor, cache, 3)
        if tensor.shape[1] != cache.kv_heads or tensor.shape[0] != tokens:
            raise ValueError(f"{name} must hold {tokens} tokens of {cache.kv_heads} heads, one token a slot")
    _require_counts(tokens=tokens)
    k_strides, v_strides, words = k.stride(), v.stride(), _status_words(status, cache.device)
    _on(cache.device, lambda stream: entry(
        cache.view, k.data_ptr(), v.data_ptr(), k_strides[0], k_strides[1], v_strides[0], v_strides[1], slots.data_ptr(),
        4 if slots.dtype is torch.int32 else 8, tokens, *more, stream, words))


def write(cache: Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, status: torch.Tensor | None = None) -> None:
    """Quantise the tokens ``k[i], v[i]`` (``[tokens, kv_heads, head_dim]``, any strides that are multiples of 8 elements) into
    the slots ``slots[i]`` = page * page_size + place (int32 or int64); a negative slot skips its token. Slots that are not
    negative must be distinct: of one named twice the row is unspecified."""
    _require_indices("slots", slots, cache, wide=True)
    _rows(library().fk_cache_write, cache, k, v, slots, status)


def read(cache: Cache, slots: torch.Tensor, k: torch.Tensor | None = None, v: torch.Tensor | None = None,
         status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, ``[tokens, kv_heads, head_dim]``: what the rows at ``slots`` (int32 or int64, may repeat) stand for, rounded once.
    Rows of negative slots are zero in new tensors and left as they were in ``k`` and ``v`` that are given (which may be
    strided, as views of the planes ``flash_forward.run`` takes, but not lie over one another)."""
    _require_indices("slots", slots, cache, wide=True)
    if (k is None) != (v is None):
        raise ValueError("k and v are given together or not at all")
    fresh = k is None
    if fresh:
        k = slots.new_empty((slots.shape[0], cache.kv_heads, cache.head_dim), dtype=cache.dtype)
        v = torch.empty_like(k)
    _rows(library().fk_cache_read, cache, k, v, slots, status, int(fresh))
    return k, v


def attend(q: torch.Tensor, cache: Cache, lengths: torch.Tensor, table: torch.Tensor | None = None,
           scale: float | None = None, window: int | None = None, sinks: int = 0, workspace: torch.Tensor | None = None,
           out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``softmax(scale * q K^T + mask) V`` of each sequence's newest tokens over its rows of the cache.

    ``q`` is ``[batch, queries, heads, head_dim]``, or ``[batch, heads, head_dim]`` for single tokens, with strides that are
    multiples of 8 elements; head h reads kv head ``h // (heads // kv_heads)``. ``lengths`` (int32 ``[batch]``) counts each
    sequence's tokens, the ``queries`` newest included, whose keys and values have been written; ``table`` (int32
    ``[batch, pages]``) names its pages in order (any number will do for pages that no row sees), and without one sequence b
    owns page b. Query t sits at
    ``i = length - queries + t`` and sees the tokens ``j <= i``; with a ``window``, those with ``j > i - window`` and the first
    ``sinks``. Returns ``(out, lse)``: ``out`` like ``q``, packed, and ``lse`` fp32 natural-log normalisers ``[batch, (queries,) heads]``;
    a row that sees nothing is zero, its lse -inf.

    ``out`` may not lie over ``q``. Each 16 rows (queries times heads per kv head) read the sequence once more: this is for few
    new tokens, not for long prompts. ``table`` wants no more columns than the longest sequence has: past 8192 tokens the launch is planned
    for long ones.

    A serving loop passes a ``workspace`` that it keeps (see :func:`workspace`); without one each call makes its own."""
    squeeze = q.dim() == 3
    if squeeze:
        q = q.unsqueeze(1)
    _require("q", q, cache, 4)
    batch, queries, heads, head_dim = q.shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads do not divide over {cache.kv_heads} kv heads")
    _require_indices("lengths", lengths, cache, batch)
    if table is not None:
        if table.device != cache.device:
            raise RuntimeError(f"table must live on the cache's device {cache.device}: there is no CPU path")
        if (table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != batch or table.shape[1] == 0
                or (table.shape[1] > 1 and table.stride(1) != 1)):
            raise ValueError("table must be an int32 [batch, pages] tensor of contiguous rows of one page or more")
    _require_counts(sequences=batch, queries=queries, heads=heads, pages=table.shape[1] if table is not None else 0)
    if window is not None and not 1 <= window < 1 << 31:
        raise ValueError("a window is at least one token")
    if not 0 <= sinks < 1 << 31:
        raise ValueError("sinks is a number of tokens")
    if workspace is None:
        workspace = globals()["workspace"](cache.device)
    elif workspace.device != cache.device or not workspace.is_contiguous():
        raise ValueError(f"the workspace must be a contiguous tensor on {cache.device}")
    shape = (batch, queries, heads, head_dim)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        if squeeze and out.dim() == 3:
            out = out.unsqueeze(1)
        _require("out", out, cache, 4)
        if out.shape != shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and of q's shape")
    lse = lengths.new_empty(shape[:3], dtype=torch.float32)
    strides, words = q.stride(), _status_words(status, cache.device)
    _on(cache.device, lambda stream: library().fk_cache_attention(
        cache.view, q.data_ptr(), strides[0], strides[1], strides[2], out.data_ptr(), lse.data_ptr(),
        lengths.data_ptr(), table.data_ptr() if table is not None else None, table.stride(0) if table is not None else 0,
        table.shape[1] if table is not None else 0, batch, queries, heads,
        head_dim ** -0.5 if scale is None else scale, window or 0, sinks, workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), stream, words))
    return (out.squeeze(1), lse.squeeze(1)) if squeeze else (out, lse)

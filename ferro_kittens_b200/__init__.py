"""B200-native (sm_100a) implementation of ferro-kittens' two dense-contraction
hot paths -- the two-CTA-cluster bf16 GEMM and flash-attention forward -- behind
a C ABI, with this package as the thin host-side mirror of the crate's surface;
and beside them the key/value cache in 4 bits that serving needs after a prompt.
"""
from . import (_lib, flash_backward, flash_forward, gemm, global_layout, kv_cache, plan, rows, shard,  # noqa: F401
               watchdog)
from ._lib import FerroKittensError  # noqa: F401

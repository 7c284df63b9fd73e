"""MI355X (gfx950) int8-KV paged attention: the `_gfx906_pth_dec` decode operator and the
`_gfx906_fa_pth` chunked-prefill operator of 0c33/mi50-vllm-lab rebuilt for CDNA4, the KV-cache
writer that produces their rows, and the vLLM routing shim.

The directory name is not a Python identifier; load it with `load_package()` from
`__graft_entry__` / `tests/conftest.py`, which registers it as `mi50_vllm_lab_amd`.
"""
from . import kvcache, pth_dec, rotary, vllm_shim  # noqa: F401
from .pth_dec import (cache_write, compact_pages, decode, decode_shared, evict, fork_pages, forward_pth, forward_window,  # noqa: F401
                      key_weights, norm_rotary_cache_write, rotary_cache_write, supported_layout)
from .rotary import rotary_table  # noqa: F401

__all__ = ["cache_write", "compact_pages", "decode", "decode_shared", "evict", "fork_pages", "forward_pth", "forward_window", "key_weights",
           "norm_rotary_cache_write", "rotary_cache_write", "rotary_table", "supported_layout", "kvcache", "pth_dec", "rotary", "vllm_shim"]

"""flash_lab for MI355X (gfx950): FlashAttention-2 prefill, split-KV decode and the operators of a
served key-value cache as hand-written HIP kernels behind the reference's flash_lab API (reference
flash_lab/__init__.py:1-5).

The reference also exports its fp64 test oracle as flash_lab.reference; in this build the oracle
is test infrastructure and lives outside the package (oracle/reference.py at the repository root).
"""

from flash_lab.ops import (
    attention,
    attention_cached,
    available_impls,
    decode,
    read_cache,
    write_cache,
)

__version__ = "0.1.0"
__all__ = ["attention", "attention_cached", "available_impls", "decode", "read_cache", "write_cache"]

"""Input validation shared by the public API (flash_lab.ops) and the test oracle.

Same contract as the reference's flash_lab/layouts.py:1-167 (its tests match these messages):
prefill tensors are [B, S, H, D] (batch, sequence, heads, head_dim); K and V may have fewer heads
than Q, query head h reading KV head h // (H // H_kv). Decode takes q [B, 1, H, D] or [B, H, D]
and a [B, S_max, H_kv, D] cache, or a paged [num_blocks, page_size, H_kv, D] pool with
block_tables [B, max_blocks]. Errors are raised before any kernel runs.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass(frozen=True)
class AttnShape:
    """Problem size of one prefill call (reference flash_lab/layouts.py:12-23)."""

    batch: int
    seqlen_q: int
    seqlen_k: int
    heads: int
    heads_kv: int
    head_dim: int

    @property
    def group(self) -> int:
        return self.heads // self.heads_kv


@dataclass(frozen=True)
class DecodeShape:
    """Problem size of one decode call (reference flash_lab/layouts.py:26-41). max_seqlen is S_max
    of a contiguous cache, or max_blocks * page_size of a paged one; page_size is 0 when the cache
    is contiguous."""

    batch: int
    heads: int
    heads_kv: int
    head_dim: int
    max_seqlen: int
    page_size: int

    @property
    def group(self) -> int:
        return self.heads // self.heads_kv

    @property
    def paged(self) -> bool:
        return self.page_size > 0


@dataclass(frozen=True)
class CacheShape:
    """Sizes of a key-value cache. max_seqlen is S_max of slabs, or max_blocks * page_size of a pool;
    page_size is 0 for slabs. quantized: e4m3 codes with scales."""

    batch: int
    heads_kv: int
    head_dim: int
    max_seqlen: int
    page_size: int
    quantized: bool

    @property
    def paged(self) -> bool:
        return self.page_size > 0


def _shape(x: torch.Tensor) -> tuple:
    return tuple(x.shape)


def _tensor_or_raise(name: str, x: object) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(x).__name__}")


def _heads_divide(heads: int, heads_kv: int) -> None:
    if heads_kv <= 0 or heads % heads_kv:
        raise ValueError(
            f"the number of query heads ({heads}) must be a multiple of KV heads ({heads_kv})"
        )


def _unit_stride_in_d(tensors: dict[str, torch.Tensor]) -> None:
    for name, x in tensors.items():
        if x.stride(-1) != 1:
            raise ValueError(
                f"{name} must be contiguous in its last dimension, got strides {tuple(x.stride())}"
            )


def check_attention_inputs(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, require_unit_stride: bool = True
) -> AttnShape:
    """Validates prefill inputs (reference flash_lab/layouts.py:64-92) and returns their shape."""
    tensors = {"q": q, "k": k, "v": v}
    for name, x in tensors.items():
        _tensor_or_raise(name, x)
        if x.dim() != 4:
            raise ValueError(f"{name} must be 4-D [B, S, H, D], got shape {_shape(x)}")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise TypeError(f"q, k, v must share a dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.device != k.device or q.device != v.device:
        raise ValueError(f"q, k, v must be on one device, got {q.device}, {k.device}, {v.device}")
    if k.shape != v.shape:
        raise ValueError(f"k and v must have the same shape, got {_shape(k)} and {_shape(v)}")

    batch, seqlen_q, heads, head_dim = q.shape
    kv_batch, seqlen_k, heads_kv, kv_head_dim = k.shape
    if kv_batch != batch:
        raise ValueError(f"batch size mismatch: q has {batch}, k and v have {kv_batch}")
    if kv_head_dim != head_dim:
        raise ValueError(f"head_dim mismatch: q has {head_dim}, k and v have {kv_head_dim}")
    if 0 in (batch, seqlen_q, seqlen_k, heads, head_dim):
        raise ValueError(f"empty input: q {_shape(q)}, k {_shape(k)}")
    _heads_divide(heads, heads_kv)
    if require_unit_stride:
        _unit_stride_in_d(tensors)
    return AttnShape(batch, seqlen_q, seqlen_k, heads, heads_kv, head_dim)


def check_decode_inputs(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    block_tables: torch.Tensor | None = None,
    *,
    require_unit_stride: bool = True,
) -> tuple[torch.Tensor, DecodeShape]:
    """Validates decode inputs (reference flash_lab/layouts.py:95-167). Returns q as a [B, H, D]
    view and the problem shape. seq_lens [B] int32 counts each sequence's valid keys, the token
    being decoded included; its values stay on the device and are not checked here."""
    tensors = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "seq_lens": seq_lens}
    if block_tables is not None:
        tensors["block_tables"] = block_tables
    for name, x in tensors.items():
        _tensor_or_raise(name, x)
    devices = {str(x.device) for x in tensors.values()}
    if len(devices) != 1:
        where = {name: str(x.device) for name, x in tensors.items()}
        raise ValueError(f"decode inputs must be on one device, got {where}")

    if q.dim() == 4:
        if q.shape[1] != 1:
            raise ValueError(f"decode takes one query token per sequence, got q {_shape(q)}")
        q = q.select(1, 0)
    elif q.dim() != 3:
        raise ValueError(f"q must be [B, 1, H, D] or [B, H, D], got shape {_shape(q)}")
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be 4-D, got shape {_shape(k_cache)}")
    if k_cache.shape != v_cache.shape:
        raise ValueError(
            "k_cache and v_cache must have the same shape, "
            f"got {_shape(k_cache)} and {_shape(v_cache)}"
        )
    if q.dtype != k_cache.dtype or q.dtype != v_cache.dtype:
        raise TypeError(
            f"q and the caches must share a dtype, got {q.dtype}, {k_cache.dtype}, {v_cache.dtype}"
        )

    batch, heads, head_dim = q.shape
    if seq_lens.dtype != torch.int32:
        raise TypeError(f"seq_lens must be int32, got {seq_lens.dtype}")
    if _shape(seq_lens) != (batch,):
        raise ValueError(f"seq_lens must have shape ({batch},), got {_shape(seq_lens)}")
    if not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be contiguous, got stride {seq_lens.stride()}")

    if block_tables is None:
        cache_batch, max_seqlen, heads_kv, cache_head_dim = k_cache.shape
        page_size = 0
        if cache_batch != batch:
            raise ValueError(f"batch size mismatch: q has {batch}, the cache has {cache_batch}")
    else:
        if block_tables.dtype != torch.int32:
            raise TypeError(f"block_tables must be int32, got {block_tables.dtype}")
        if block_tables.dim() != 2 or block_tables.shape[0] != batch:
            raise ValueError(
                f"block_tables must be [{batch}, max_blocks], got {_shape(block_tables)}"
            )
        _, page_size, heads_kv, cache_head_dim = k_cache.shape
        max_seqlen = block_tables.shape[1] * page_size

    if cache_head_dim != head_dim:
        raise ValueError(f"head_dim mismatch: q has {head_dim}, the cache has {cache_head_dim}")
    if 0 in (batch, heads, head_dim, max_seqlen):
        raise ValueError(f"empty input: q {_shape(q)}, k_cache {_shape(k_cache)}")
    _heads_divide(heads, heads_kv)
    if require_unit_stride:
        _unit_stride_in_d({"q": q, "k_cache": k_cache, "v_cache": v_cache})
    return q, DecodeShape(batch, heads, heads_kv, head_dim, max_seqlen, page_size)


# A cache in 8 bits: e4m3 codes [..., H_kv, D], and for each row the exponent byte [..., H_kv] of its scale,
# 2^(byte - 127). (Plain bytes rather than torch.float8_e8m0fnu, which torch.compile cannot pass through.)
CODE_DTYPE = torch.float8_e4m3fn
SCALE_DTYPE = torch.uint8


def check_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    block_tables: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
) -> CacheShape:
    """Validates a cache and its sequences: slabs [B, S_max, H_kv, D], or a pool [num_blocks, page_size,
    H_kv, D] with block_tables [B, max_blocks] int32, in a floating type, or in float8_e4m3fn with
    uint8 scales of the same shape without D. seq_lens [B] and cu_seqlens [B + 1] are int32;
    their values stay on the device and are not checked here."""
    tensors = {"k_cache": k_cache, "v_cache": v_cache, "seq_lens": seq_lens}
    for name, x in (("block_tables", block_tables), ("k_scales", k_scales), ("v_scales", v_scales),
                    ("cu_seqlens", cu_seqlens)):
        if x is not None:
            tensors[name] = x
    for name, x in tensors.items():
        _tensor_or_raise(name, x)
    if len({x.device for x in tensors.values()}) != 1:
        where = {name: str(x.device) for name, x in tensors.items()}
        raise ValueError(f"a cache's tensors must be on one device, got {where}")
    if k_cache.dim() != 4:
        raise ValueError(f"k_cache must be 4-D, got shape {_shape(k_cache)}")
    if k_cache.shape != v_cache.shape:
        raise ValueError(
            "k_cache and v_cache must have the same shape, "
            f"got {_shape(k_cache)} and {_shape(v_cache)}"
        )
    if k_cache.dtype != v_cache.dtype:
        raise TypeError(f"the caches must share a dtype, got {k_cache.dtype} and {v_cache.dtype}")
    quantized = k_cache.dtype == CODE_DTYPE
    if quantized != (k_scales is not None) or quantized != (v_scales is not None):
        raise ValueError(f"k_scales and v_scales go with {CODE_DTYPE} caches, and with no other")
    if quantized:
        for name, x in (("k_scales", k_scales), ("v_scales", v_scales)):
            if x.dtype != SCALE_DTYPE:
                raise TypeError(f"{name} must be {SCALE_DTYPE}, got {x.dtype}")
            if x.shape != k_cache.shape[:3]:
                raise ValueError(
                    f"{name} must have the caches' shape without D, {_shape(k_cache)[:3]}, got {_shape(x)}"
                )
    if seq_lens.dtype != torch.int32:
        raise TypeError(f"seq_lens must be int32, got {seq_lens.dtype}")
    if seq_lens.dim() != 1 or not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be a contiguous [B], got shape {_shape(seq_lens)}, "
                         f"stride {seq_lens.stride()}")
    batch = seq_lens.shape[0]
    if cu_seqlens is not None:
        if cu_seqlens.dtype != torch.int32:
            raise TypeError(f"cu_seqlens must be int32, got {cu_seqlens.dtype}")
        if _shape(cu_seqlens) != (batch + 1,) or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must be a contiguous [{batch + 1}], got shape {_shape(cu_seqlens)}")
    outer, rows, heads_kv, head_dim = k_cache.shape
    page_size, max_seqlen = 0, rows
    if block_tables is not None:
        if block_tables.dtype != torch.int32:
            raise TypeError(f"block_tables must be int32, got {block_tables.dtype}")
        if block_tables.dim() != 2 or block_tables.shape[0] != batch or block_tables.stride(1) != 1:
            raise ValueError(
                f"block_tables must be [{batch}, max_blocks] with unit stride in its last dimension, "
                f"got {_shape(block_tables)}"
            )
        page_size, max_seqlen = rows, block_tables.shape[1] * rows
    elif outer != batch:
        raise ValueError(f"batch size mismatch: seq_lens has {batch}, the cache has {outer}")
    if 0 in (batch, outer, heads_kv, head_dim, max_seqlen):
        raise ValueError(f"empty input: k_cache {_shape(k_cache)}, {batch} sequences")
    _unit_stride_in_d({"k_cache": k_cache, "v_cache": v_cache})
    return CacheShape(batch, heads_kv, head_dim, max_seqlen, page_size, quantized)


def check_token_rows(
    name: str, x: torch.Tensor, cache: CacheShape, k_cache: torch.Tensor, cu_seqlens: torch.Tensor | None
) -> None:
    """Validates a tensor of the call's tokens against a checked cache: [tokens, heads, D] with cu_seqlens,
    [B, S, heads, D] without."""
    _tensor_or_raise(name, x)
    if x.device != k_cache.device:
        raise ValueError(f"{name} is on {x.device}, the cache on {k_cache.device}")
    if cu_seqlens is None:
        if x.dim() != 4:
            raise ValueError(f"{name} must be 4-D [B, S, H, D] without cu_seqlens, got shape {_shape(x)}")
        if x.shape[0] != cache.batch:
            raise ValueError(f"batch size mismatch: {name} has {x.shape[0]}, seq_lens has {cache.batch}")
    elif x.dim() != 3:
        raise ValueError(f"{name} must be 3-D [tokens, H, D] with cu_seqlens, got shape {_shape(x)}")
    if x.shape[-1] != cache.head_dim:
        raise ValueError(f"head_dim mismatch: {name} has {x.shape[-1]}, the cache has {cache.head_dim}")
    if not cache.quantized and x.dtype != k_cache.dtype:
        raise TypeError(f"{name} must have the caches' dtype {k_cache.dtype}, or they {CODE_DTYPE}, got {x.dtype}")
    _unit_stride_in_d({name: x})


def check_query_heads(heads: int, heads_kv: int) -> None:
    _heads_divide(heads, heads_kv)
    if heads == 0:
        raise ValueError("empty input: no query heads")

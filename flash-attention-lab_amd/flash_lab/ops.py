"""Public entry points: flash_lab.attention, flash_lab.decode, flash_lab.available_impls, and the cache
operators flash_lab.write_cache, flash_lab.read_cache and flash_lab.attention_cached, which the reference
lacks.

Same API, selection rules and errors as the reference's flash_lab/ops.py:1-226. Each call
validates its inputs, picks an implementation from the tables below (impl="auto" takes the first
built entry that supports the input), and calls torch.ops.flash_lab.<op>. The ops are the gfx950
HIP kernels registered by flash_lab._hip; impl names the reference also ships as other kernels
(Triton, the fp32 CUDA-core progression, the copy-based decode baseline) are kept in the tables so
that code naming them gets a clear "not available in this build" error instead of "unknown impl".
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from flash_lab.layouts import (
    AttnShape,
    CacheShape,
    DecodeShape,
    check_attention_inputs,
    check_cache,
    check_decode_inputs,
    check_query_heads,
    check_token_rows,
)

try:
    from flash_lab import _hip  # noqa: F401  (loading the library registers the ops)
except ImportError as exc:
    HAS_EXTENSION = False
    EXTENSION_ERROR = str(exc)
else:
    HAS_EXTENSION = True
    EXTENSION_ERROR = ""


@dataclass(frozen=True)
class PrefillImpl:
    """One prefill kernel and what it supports (reference flash_lab/ops.py:33-50)."""

    op: str
    dtypes: tuple[torch.dtype, ...]
    head_dims: tuple[int, ...]
    gqa: bool = True
    causal_unequal_lengths: bool = True  # causal with S_q != S_k, bottom-right aligned

    def unsupported_reason(self, shape: AttnShape, dtype: torch.dtype, causal: bool) -> str | None:
        if dtype not in self.dtypes:
            return f"dtype {dtype} is not one of {self.dtypes}"
        if shape.head_dim not in self.head_dims:
            return f"head_dim {shape.head_dim} is not one of {self.head_dims}"
        if shape.group > 1 and not self.gqa:
            return "grouped-query attention (H_kv < H) is not supported"
        if causal and shape.seqlen_q != shape.seqlen_k and not self.causal_unequal_lengths:
            return "causal attention requires S_q == S_k"
        return None


@dataclass(frozen=True)
class DecodeImpl:
    """One decode kernel and what it supports (reference flash_lab/ops.py:53-68)."""

    op: str
    dtypes: tuple[torch.dtype, ...]
    head_dims: tuple[int, ...]
    paged_op: str | None = None  # the op serving paged caches (None: paged caches unsupported)
    in_auto: bool = True  # False for baselines kept for comparison only

    @property
    def paged(self) -> bool:
        return self.paged_op is not None

    def unsupported_reason(self, shape: DecodeShape, dtype: torch.dtype) -> str | None:
        if dtype not in self.dtypes:
            return f"dtype {dtype} is not one of {self.dtypes}"
        if shape.head_dim not in self.head_dims:
            return f"head_dim {shape.head_dim} is not one of {self.head_dims}"
        if shape.paged and not self.paged:
            return "paged KV caches are not supported"
        return None


@dataclass(frozen=True)
class CachedImpl:
    """One kernel for attention over a cache and what it supports."""

    op: str
    dtypes: tuple[torch.dtype, ...]
    head_dims: tuple[int, ...]

    def unsupported_reason(self, cache: CacheShape, dtype: torch.dtype) -> str | None:
        if dtype not in self.dtypes:
            return f"dtype {dtype} is not one of {self.dtypes}"
        if cache.head_dim not in self.head_dims:
            return f"head_dim {cache.head_dim} is not one of {self.head_dims}"
        return None


_HALF = (torch.bfloat16, torch.float16)
_FP32 = (torch.float32,)
_DIMS = (64, 128)

# In order of preference. The gfx950 MFMA kernel serves both tensor-core names of the reference.
PREFILL_IMPLS: dict[str, PrefillImpl] = {
    "mma_pipelined": PrefillImpl(op="attention_mma_pipelined", dtypes=_HALF, head_dims=_DIMS),
    "mma": PrefillImpl(op="attention_mma", dtypes=_HALF, head_dims=_DIMS),
    # Reference kernels that this build does not ship (Triton, fp32 CUDA-core progression).
    "triton": PrefillImpl(op="attention_triton", dtypes=_HALF, head_dims=_DIMS),
    "fp32_regtile": PrefillImpl(op="attention_fp32_regtile", dtypes=_FP32, head_dims=_DIMS),
    "fp32_fused": PrefillImpl(op="attention_fp32_fused", dtypes=_FP32, head_dims=_DIMS),
    "naive": PrefillImpl(op="attention_naive", dtypes=_FP32, head_dims=_DIMS),
}
_DECODE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
DECODE_IMPLS: dict[str, DecodeImpl] = {
    "splitkv": DecodeImpl(
        op="decode_splitkv", dtypes=_DECODE_DTYPES, head_dims=_DIMS, paged_op="decode_splitkv_paged"
    ),
    "decode_inplace": DecodeImpl(
        op="decode_inplace", dtypes=_DECODE_DTYPES, head_dims=_DIMS, paged_op="decode_inplace_paged"
    ),
    # The reference's copy-based baseline; not shipped by this build.
    "decode_copy": DecodeImpl(
        op="decode_copy", dtypes=_DECODE_DTYPES, head_dims=_DIMS, in_auto=False
    ),
}
CACHED_IMPLS: dict[str, CachedImpl] = {
    "cached_mma": CachedImpl(op="attention_cached", dtypes=_HALF, head_dims=_DIMS),
}
# Writing and reading a cache: one kernel each.
CACHE_OPS = ("write_cache", "read_cache")


def _op_exists(op: str) -> bool:
    return hasattr(torch.ops.flash_lab, op)


def _register_fakes() -> None:
    """Shape-only versions of the ops, so torch.compile can trace through them
    (reference flash_lab/ops.py:100-118)."""

    def prefill_fake(q, k, v, causal, softmax_scale):
        batch, seqlen_q, heads, _ = q.shape
        return q.new_empty(q.shape), q.new_empty((batch, heads, seqlen_q), dtype=torch.float32)

    def decode_fake(q, k_cache, v_cache, seq_lens, softmax_scale, num_splits):
        return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)

    def paged_decode_fake(q, k_cache, v_cache, seq_lens, block_tables, softmax_scale, num_splits):
        return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)

    def cached_fake(q, k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables, causal,
                    softmax_scale, num_splits):
        return q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32)

    def write_cache_fake(k, v, k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables):
        return None

    def read_cache_fake(k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables, num_tokens,
                        dtype):
        shape = (num_tokens, *k_cache.shape[2:])
        return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)

    for name, fake in (("attention_cached", cached_fake), ("write_cache", write_cache_fake),
                       ("read_cache", read_cache_fake)):
        if _op_exists(name):
            torch.library.register_fake(f"flash_lab::{name}")(fake)
    for spec in PREFILL_IMPLS.values():
        if _op_exists(spec.op):
            torch.library.register_fake(f"flash_lab::{spec.op}")(prefill_fake)
    for spec in DECODE_IMPLS.values():
        if _op_exists(spec.op):
            torch.library.register_fake(f"flash_lab::{spec.op}")(decode_fake)
        if spec.paged_op and _op_exists(spec.paged_op):
            torch.library.register_fake(f"flash_lab::{spec.paged_op}")(paged_decode_fake)


if HAS_EXTENSION:
    _register_fakes()

# All ops are registered by the import above, so availability is looked up once.
_BUILT_OPS = frozenset(
    op
    for spec in (*PREFILL_IMPLS.values(), *DECODE_IMPLS.values(), *CACHED_IMPLS.values())
    for op in (spec.op, getattr(spec, "paged_op", None), *CACHE_OPS)
    if op and HAS_EXTENSION and _op_exists(op)
)


# The ops' overloads, looked up once: the packet's own lookup takes a call about 2 us.
_OVERLOADS = {op: getattr(torch.ops.flash_lab, op).default for op in _BUILT_OPS}


def available_impls() -> dict[str, list[str]]:
    """Implementations compiled into this build, by entry point."""
    return {
        "attention": [name for name, spec in PREFILL_IMPLS.items() if spec.op in _BUILT_OPS],
        "decode": [name for name, spec in DECODE_IMPLS.items() if spec.op in _BUILT_OPS],
    }


def _select(table: dict, impl: str, device: torch.device, describe, reason_of):
    """The implementation to run (reference flash_lab/ops.py:139-159). describe() names the
    problem in error messages and is only called on failure."""
    if impl != "auto" and impl not in table:
        raise ValueError(f"unknown impl {impl!r}; choose from {['auto', *table]}")
    if device.type != "cuda":
        raise ValueError(f"flash_lab kernels take CUDA tensors, got device {device}")
    missing = "" if HAS_EXTENSION else f" (the HIP extension did not load: {EXTENSION_ERROR})"
    if impl != "auto":
        spec = table[impl]
        reason = reason_of(spec)
        if reason is not None:
            raise ValueError(f"impl {impl!r} cannot run {describe()}: {reason}")
        if spec.op not in _BUILT_OPS:
            raise RuntimeError(f"impl {impl!r} is not available in this build{missing}")
        return spec
    candidates = [s for s in table.values() if getattr(s, "in_auto", True) and s.op in _BUILT_OPS]
    for spec in candidates:
        if reason_of(spec) is None:
            return spec
    raise ValueError(f"no available implementation supports {describe()}{missing}")


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    causal: bool = False,
    softmax_scale: float | None = None,
    impl: str = "auto",
    return_lse: bool = False,
):
    """Attention forward. q is [B, S_q, H, D]; k and v are [B, S_k, H_kv, D] with H % H_kv == 0.

    Returns o [B, S_q, H, D] in the input dtype and, with return_lse=True, the natural-log
    log-sum-exp of each score row as fp32 [B, H, S_q]. Causal masking with S_q != S_k is aligned
    to the bottom-right corner: query i sees key j iff j <= i + (S_k - S_q).
    """
    shape = check_attention_inputs(q, k, v)
    scale = 1.0 / math.sqrt(shape.head_dim) if softmax_scale is None else softmax_scale
    if not scale > 0:
        raise ValueError(f"softmax_scale must be positive, got {scale}")
    spec = _select(
        PREFILL_IMPLS,
        impl,
        q.device,
        lambda: (
            f"dtype={q.dtype}, head_dim={shape.head_dim}, heads={shape.heads}/{shape.heads_kv}, "
            f"S_q={shape.seqlen_q}, S_k={shape.seqlen_k}, causal={causal}"
        ),
        lambda s: s.unsupported_reason(shape, q.dtype, causal),
    )
    out, lse = _OVERLOADS[spec.op](q, k, v, causal, scale)
    return (out, lse) if return_lse else out


def decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    block_tables: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    impl: str = "auto",
    num_splits: int | None = None,
    return_lse: bool = False,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
):
    """One decode step: each sequence's single query token attends to its first seq_lens[b] keys.

    The cache is [B, S_max, H_kv, D], or [num_blocks, page_size, H_kv, D] with block_tables. With k_scales
    and v_scales it holds 8 bits (float8_e4m3fn codes, see write_cache) under q in bf16 or fp16; impl is
    then "auto" or "splitkv".
    seq_lens values are not checked on the host (that would force a device sync).
    num_splits=None lets the library choose how many workgroups share one sequence's keys; a large
    paged batch then shares all sequences' keys evenly, so a sequence's last bits can depend on the
    other lengths of the batch and on the cache's layout. A num_splits of one's own pins them.
    """
    if k_scales is not None or v_scales is not None:
        return _decode_quantized(q, k_cache, v_cache, seq_lens, block_tables, softmax_scale, impl,
                                 num_splits, return_lse, k_scales, v_scales)
    q3, shape = check_decode_inputs(q, k_cache, v_cache, seq_lens, block_tables)
    scale = 1.0 / math.sqrt(shape.head_dim) if softmax_scale is None else softmax_scale
    if num_splits is not None and num_splits < 1:
        raise ValueError(f"num_splits must be positive, got {num_splits}")
    spec = _select(
        DECODE_IMPLS,
        impl,
        q.device,
        lambda: (
            f"dtype={q.dtype}, head_dim={shape.head_dim}, heads={shape.heads}/{shape.heads_kv}, "
            f"paged={shape.paged}"
        ),
        lambda s: s.unsupported_reason(shape, q.dtype),
    )
    if block_tables is not None:
        out, lse = _OVERLOADS[spec.paged_op](
            q3, k_cache, v_cache, seq_lens, block_tables, scale, num_splits or 0
        )
    else:
        out, lse = _OVERLOADS[spec.op](
            q3, k_cache, v_cache, seq_lens, scale, num_splits or 0
        )
    if q.dim() == 4:
        out = out.unsqueeze(1)
    return (out, lse) if return_lse else out


# The native ops check their arguments themselves, and a call of one costs less than the checks here: so the
# cache operators call the op first, and find out what was wrong (and raise as the other entry points do)
# when it refuses. Under torch.compile, where the ops are not run, the checks come first.


def _decode_quantized(q, k_cache, v_cache, seq_lens, block_tables, softmax_scale, impl, num_splits, return_lse,
                      k_scales, v_scales):
    """decode() over a cache in 8 bits: attention_cached with one token per sequence."""
    if impl not in ("auto", "splitkv"):
        if impl not in DECODE_IMPLS:
            raise ValueError(f"unknown impl {impl!r}; choose from {['auto', *DECODE_IMPLS]}")
        raise ValueError(f"impl {impl!r} cannot run a cache in 8 bits; choose 'auto' or 'splitkv'")
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
    rank = q.dim()
    if rank == 4 and q.shape[1] != 1:
        raise ValueError(f"decode takes one query token per sequence, got q {tuple(q.shape)}")
    if rank not in (3, 4):
        raise ValueError(f"q must be [B, 1, H, D] or [B, H, D], got shape {tuple(q.shape)}")
    if num_splits is not None and num_splits < 1:
        raise ValueError(f"num_splits must be positive, got {num_splits}")
    out, lse = _attention_cached(q if rank == 4 else q.unsqueeze(1), k_cache, v_cache, seq_lens, None, block_tables,
                                 k_scales, v_scales, True, softmax_scale, "auto", num_splits or 0)
    out = out if rank == 4 else out.squeeze(1)
    return (out, lse.squeeze(1)) if return_lse else out


def _check_attention_cached(q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scales, v_scales,
                            softmax_scale, impl) -> None:
    cache = check_cache(k_cache, v_cache, seq_lens, block_tables, k_scales, v_scales, cu_seqlens)
    check_token_rows("q", q, cache, k_cache, cu_seqlens)
    check_query_heads(q.shape[-2], cache.heads_kv)
    if softmax_scale is not None and not softmax_scale > 0:
        raise ValueError(f"softmax_scale must be positive, got {softmax_scale}")
    _select(
        CACHED_IMPLS,
        impl,
        q.device,
        lambda: (
            f"dtype={q.dtype}, head_dim={cache.head_dim}, heads={q.shape[-2]}/{cache.heads_kv}, "
            f"paged={cache.paged}, quantized={cache.quantized}"
        ),
        lambda s: s.unsupported_reason(cache, q.dtype),
    )


def _attention_cached(q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scales, v_scales, causal,
                      softmax_scale, impl, num_splits):
    checked = (q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scales, v_scales, softmax_scale, impl)
    if impl not in ("auto", "cached_mma") or torch.compiler.is_compiling():
        _check_attention_cached(*checked)
    try:
        scale = 1.0 / math.sqrt(q.shape[-1]) if softmax_scale is None else softmax_scale
        return _OVERLOADS["attention_cached"](q, k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens,
                                              block_tables, causal, scale, num_splits)
    except Exception:
        _check_attention_cached(*checked)
        raise


def attention_cached(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    block_tables: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    causal: bool = True,
    softmax_scale: float | None = None,
    impl: str = "auto",
    return_lse: bool = False,
):
    """Attention of new tokens to the caches of their sequences: chunks of prompts, next turns, drafted
    tokens, single tokens, in one ragged batch; or, with causal=False, cross attention to an encoder's
    states of a length per sequence.

    q is [tokens, H, D], in which tokens cu_seqlens[b] .. cu_seqlens[b + 1] - 1 are sequence b's (cu_seqlens
    [B + 1] int32), or [B, S_q, H, D] without cu_seqlens, in bf16 or fp16. The cache is [B, S_max, H_kv, D],
    or [num_blocks, page_size, H_kv, D] with block_tables [B, max_blocks], in q's dtype, or in
    float8_e4m3fn with k_scales and v_scales (see write_cache). It holds seq_lens[b] (int32) tokens of
    sequence b; with causal=True the call's tokens are the last of them (write_cache comes first) and see
    the keys up to their own.

    Returns o like q and, with return_lse=True, the natural-log log-sum-exp of each score row as fp32 of q's
    shape without D. A token that sees no key gets o = 0 and lse = -inf, and so do rows of q behind the last
    sequence. Values of seq_lens, cu_seqlens and block_tables are not checked on the host (that would force
    a device sync): the kernels clamp them, so that a wrong one gives wrong rows and no access out of
    bounds. Keys and values that a token does not see do not reach it, whatever they hold. A token's last bits
    can depend on the other sequences' lengths. A batch with one token for every sequence is faster as [B, 1, H, D]
    without cu_seqlens, or through decode: then no longer sequences are prepared for.
    """
    out, lse = _attention_cached(q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scales, v_scales,
                                 causal, softmax_scale, impl, 0)
    return (out, lse) if return_lse else out


def _check_cache_op(name: str, cache: CacheShape, dtype: torch.dtype, device: torch.device) -> None:
    if dtype not in _DECODE_DTYPES:
        raise TypeError(f"token rows must be one of {_DECODE_DTYPES}, got {dtype}")
    if cache.head_dim not in _DIMS:
        raise ValueError(f"head_dim {cache.head_dim} is not one of {_DIMS}")
    if device.type != "cuda":
        raise ValueError(f"flash_lab kernels take CUDA tensors, got device {device}")
    if name not in _BUILT_OPS:
        missing = "" if HAS_EXTENSION else f" (the HIP extension did not load: {EXTENSION_ERROR})"
        raise RuntimeError(f"{name} is not available in this build{missing}")


def _check_write_cache(k, v, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scales, v_scales) -> None:
    cache = check_cache(k_cache, v_cache, seq_lens, block_tables, k_scales, v_scales, cu_seqlens)
    for name, x in (("k", k), ("v", v)):
        check_token_rows(name, x, cache, k_cache, cu_seqlens)
        if x.shape[-2] != cache.heads_kv:
            raise ValueError(f"{name} has {x.shape[-2]} heads, the cache has {cache.heads_kv}")
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k and v must have the same shape and dtype, got {tuple(k.shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    _check_cache_op("write_cache", cache, k.dtype, k.device)


def _check_read_cache(k_cache, v_cache, seq_lens, cu_seqlens, num_tokens, block_tables, k_scales, v_scales,
                      dtype) -> None:
    cache = check_cache(k_cache, v_cache, seq_lens, block_tables, k_scales, v_scales, cu_seqlens)
    if cu_seqlens is None:
        raise TypeError("cu_seqlens must be a torch.Tensor, got NoneType")
    if num_tokens < 0:
        raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
    if dtype is None:
        dtype = torch.bfloat16 if cache.quantized else k_cache.dtype
    if not cache.quantized and dtype != k_cache.dtype:
        raise TypeError(f"a cache of {k_cache.dtype} is read in its own dtype, got {dtype}")
    _check_cache_op("read_cache", cache, dtype, k_cache.device)


def write_cache(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    block_tables: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
) -> None:
    """Writes new tokens' keys and values into the cache, in place, quantising them where it holds 8 bits.

    k and v are [tokens, H_kv, D] with cu_seqlens [B + 1], or [B, S, H_kv, D] without, in bf16, fp16 or fp32;
    seq_lens [B] counts each sequence's tokens with the new ones, which are its last. The cache is [B, S_max,
    H_kv, D], or [num_blocks, page_size, H_kv, D] with block_tables [B, max_blocks]: in the rows' dtype, or
    in 8 bits, float8_e4m3fn with k_scales and v_scales, uint8 of the cache's shape without D.

    A row (one token's D values of one KV head) is then stored as codes times a power of two, 2^(scale byte -
    127): the least that brings its largest finite magnitude to at most 448, so that a value is off by at most 1/16 of itself, or
    2^-10 of the scale if that is more. Infinities and NaN become NaN, and magnitudes are held to the largest
    that the rows' type holds after the rounding too (61,440 in fp16).

    Tokens whose position is outside the cache, or whose table entry is outside the pool, are not written.
    Sequences must not write to a block that they share (its rows would hold a mixture).
    """
    checked = (k, v, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scales, v_scales)
    if torch.compiler.is_compiling():
        _check_write_cache(*checked)
    try:
        _OVERLOADS["write_cache"](k, v, k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables)
    except Exception:
        _check_write_cache(*checked)
        raise


def read_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    num_tokens: int,
    block_tables: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Reads rows of the cache back as contiguous k and v [num_tokens, H_kv, D].

    Rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of the result are the last tokens of sequence b's
    seq_lens[b]: whole sequences where cu_seqlens is the running sum of seq_lens. num_tokens is the number
    of rows to allocate, cu_seqlens[B] or more. The cache and its scales are write_cache's. A cache in 8 bits
    gives `dtype` (bf16 by default; values that fp16 cannot hold are rounded to it), any other its own.
    Rows behind the last sequence, and rows of positions that the cache does not have, are zero.
    """
    checked = (k_cache, v_cache, seq_lens, cu_seqlens, num_tokens, block_tables, k_scales, v_scales, dtype)
    if torch.compiler.is_compiling():
        _check_read_cache(*checked)
    try:
        if dtype is None:
            dtype = torch.bfloat16 if k_scales is not None else k_cache.dtype
        return _OVERLOADS["read_cache"](k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables,
                                        num_tokens, dtype)
    except Exception:
        _check_read_cache(*checked)
        raise

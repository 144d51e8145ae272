"""What the cache operators refuse, on the CPU: the public entry points' checks (raised before anything runs)
and the C entry points', which return before any launch."""

import ctypes

import pytest
import torch

import flash_lab
from flash_lab import _hip
from flash_lab.layouts import check_cache, check_token_rows


def cache(dtype=torch.bfloat16, quantized=False, page=0, batch=2):
    outer, rows = (7, page) if page else (batch, 40)
    shape = (outer, rows, 2, 64)
    lens = torch.tensor([20] * batch, dtype=torch.int32)
    tables = torch.zeros(batch, 3, dtype=torch.int32) if page else None
    if quantized:
        k = torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
        scales = torch.full(shape[:3], 127, dtype=torch.uint8)
        return dict(k_cache=k, v_cache=k.clone(), seq_lens=lens, block_tables=tables, k_scales=scales,
                    v_scales=scales.clone())
    k = torch.zeros(shape, dtype=dtype)
    return dict(k_cache=k, v_cache=k.clone(), seq_lens=lens, block_tables=tables, k_scales=None, v_scales=None)


def q(dtype=torch.bfloat16, heads=4, head_dim=64):
    return torch.zeros(6, heads, head_dim, dtype=dtype)


CU = torch.tensor([0, 2, 6], dtype=torch.int32)


def test_shapes_that_are_taken():
    c = cache()
    shape = check_cache(**c, cu_seqlens=CU)
    assert (shape.max_seqlen, shape.page_size, shape.paged, shape.quantized) == (40, 0, False, False)
    c = cache(quantized=True, page=16)
    shape = check_cache(**c)
    assert (shape.max_seqlen, shape.page_size, shape.paged, shape.quantized) == (48, 16, True, True)
    check_token_rows("q", q(torch.float16), shape, c["k_cache"], CU)
    check_token_rows("k", torch.zeros(2, 3, 2, 64), shape, c["k_cache"], None)


@pytest.mark.parametrize("change,error,message", [
    (dict(k_cache=None), TypeError, "k_cache must be a torch.Tensor"),
    (dict(k_cache=lambda x: x[0]), ValueError, "4-D"),
    (dict(v_cache=lambda x: x[:, :8]), ValueError, "same shape"),
    (dict(v_cache=lambda x: x.to(torch.float16)), TypeError, "share a dtype"),
    (dict(k_cache=lambda x: x.transpose(1, 3).contiguous().transpose(1, 3)), ValueError, "last dimension"),
    (dict(seq_lens=lambda x: x.long()), TypeError, "seq_lens must be int32"),
    (dict(seq_lens=lambda x: x[None]), ValueError, "seq_lens must be a contiguous"),
    (dict(seq_lens=lambda x: x.repeat(2)), ValueError, "batch size mismatch|contiguous"),
    (dict(cu_seqlens=lambda x: x[:2]), ValueError, "cu_seqlens must be a contiguous"),
    (dict(cu_seqlens=lambda x: x.long()), TypeError, "cu_seqlens must be int32"),
    (dict(k_scales=torch.zeros(2, 40, 2, dtype=torch.uint8)), ValueError, "go with torch.float8_e4m3fn"),
], ids=lambda x: next(iter(x)) if isinstance(x, dict) else "")
def test_bad_caches(change, error, message):
    args = dict(cache(), cu_seqlens=CU)
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    for call in (lambda: flash_lab.attention_cached(q(), **args), lambda: flash_lab.write_cache(
            torch.zeros(6, 2, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 64, dtype=torch.bfloat16), **args),
            lambda: flash_lab.read_cache(num_tokens=6, **args)):
        with pytest.raises(error, match=message):
            call()


@pytest.mark.parametrize("change,error,message", [
    (dict(k_scales=None), ValueError, "go with torch.float8_e4m3fn"),
    (dict(k_scales=lambda x: x.float()), TypeError, "k_scales must be torch.uint8"),
    (dict(v_scales=lambda x: x[:, :, :1]), ValueError, "without D"),
    (dict(block_tables=lambda x: x.long()), TypeError, "block_tables must be int32"),
    (dict(block_tables=lambda x: x[:1]), ValueError, "block_tables must be"),
    (dict(block_tables=lambda x: x.t().contiguous().t()), ValueError, "unit stride"),
    (dict(block_tables=lambda x: x[:, :0]), ValueError, "empty input"),
], ids=lambda x: next(iter(x)) if isinstance(x, dict) else "")
def test_bad_quantized_pools(change, error, message):
    args = dict(cache(quantized=True, page=16), cu_seqlens=CU)
    for name, f in change.items():
        args[name] = f(args[name]) if callable(f) else f
    with pytest.raises(error, match=message):
        flash_lab.attention_cached(q(), **args)


@pytest.mark.parametrize("x,cu,error,message", [
    (q()[0], CU, ValueError, "3-D"),
    (q(), None, ValueError, "4-D"),
    (torch.zeros(3, 2, 4, 64, dtype=torch.bfloat16), None, ValueError, "batch size mismatch"),
    (q(torch.float16), CU, TypeError, "caches' dtype"),
    (q(head_dim=128), CU, ValueError, "head_dim mismatch"),
    (q(heads=3), CU, ValueError, "multiple of KV heads"),
    (q(heads=0), CU, ValueError, "no query heads"),
    (q().transpose(1, 2).contiguous().transpose(1, 2), CU, ValueError, "last dimension"),
    (q(), CU, ValueError, "CUDA tensors"),
])
def test_bad_queries(x, cu, error, message):
    with pytest.raises(error, match=message):
        flash_lab.attention_cached(x, cu_seqlens=cu, **cache())


def test_bad_options():
    with pytest.raises(ValueError, match="unknown impl 'fast'"):
        flash_lab.attention_cached(q(), cu_seqlens=CU, impl="fast", **cache())
    with pytest.raises(ValueError, match="softmax_scale must be positive"):
        flash_lab.attention_cached(q(), cu_seqlens=CU, softmax_scale=0.0, **cache())
    with pytest.raises(ValueError, match="softmax_scale must be positive"):
        flash_lab.attention_cached(q(), cu_seqlens=CU, softmax_scale=float("nan"), **cache())
    with pytest.raises(ValueError, match="num_tokens must not be negative"):
        flash_lab.read_cache(num_tokens=-1, cu_seqlens=CU, **cache())
    with pytest.raises(TypeError, match="read in its own dtype"):
        flash_lab.read_cache(num_tokens=6, cu_seqlens=CU, dtype=torch.float32, **cache())
    with pytest.raises(TypeError, match="must be one of"):
        flash_lab.read_cache(num_tokens=6, cu_seqlens=CU, dtype=torch.float64, **cache(quantized=True))
    with pytest.raises(TypeError, match="cu_seqlens"):
        flash_lab.read_cache(num_tokens=6, cu_seqlens=None, **cache())
    k = torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k has 3 heads"):
        flash_lab.write_cache(torch.zeros(6, 3, 64, dtype=torch.bfloat16), k, cu_seqlens=CU, **cache())
    with pytest.raises(ValueError, match="same shape and dtype"):
        flash_lab.write_cache(k[:5], k, cu_seqlens=CU, **cache())
    with pytest.raises(TypeError, match="must be one of"):
        flash_lab.write_cache(k.double(), k.double(), cu_seqlens=CU, **cache(quantized=True))


def test_bad_quantized_decodes():
    c = cache(quantized=True)
    step = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one query token"):
        flash_lab.decode(step.repeat(1, 2, 1, 1), **c)
    with pytest.raises(ValueError, match=r"\[B, 1, H, D\]"):
        flash_lab.decode(step[0, 0], **c)
    with pytest.raises(ValueError, match="cannot run a cache in 8 bits"):
        flash_lab.decode(step, impl="decode_inplace", **c)
    with pytest.raises(ValueError, match="unknown impl"):
        flash_lab.decode(step, impl="fast", **c)
    with pytest.raises(ValueError, match="num_splits must be positive"):
        flash_lab.decode(step, num_splits=0, **c)
    with pytest.raises(ValueError, match="CUDA tensors"):
        flash_lab.decode(step, **c)
    # Codes without scales are no cache of decode's.
    with pytest.raises(TypeError, match="share a dtype"):
        flash_lab.decode(step, **dict(c, k_scales=None, v_scales=None))


# ----------------------------------------------------------------------------------------------
# The C entry points. Pointers are never followed: every call here is refused first, or has no tokens.


def c_cache(**over):
    c = _hip.KvCache()
    c.k = c.v = c.seq_lens = c.cu_seqlens = 256
    c.batch = c.outer = 2
    c.rows, c.heads_kv, c.head_dim, c.dtype, c.tokens = 40, 2, 64, 0, 6
    c.k_batch_stride = c.v_batch_stride = 40 * 2 * 64
    c.k_seq_stride = c.v_seq_stride = 2 * 64
    c.k_head_stride = c.v_head_stride = 64
    for name, value in over.items():
        setattr(c, name, value)
    return c


def c_rows(**over):
    r = _hip.TokenRows()
    r.k = r.v = 256
    r.k_seq_stride = r.v_seq_stride = 2 * 64
    r.k_head_stride = r.v_head_stride = 64
    for name, value in over.items():
        setattr(r, name, value)
    return r


def c_attn(cache=None, **over):
    p = _hip.CachedAttnParams()
    p.cache = c_cache() if cache is None else cache
    p.q = p.o = p.lse = p.workspace = 256
    p.workspace_bytes = 1 << 40
    p.q_seq_stride = p.o_seq_stride = 4 * 64
    p.q_head_stride = p.o_head_stride = 64
    p.heads, p.causal, p.softmax_scale = 4, 1, 0.125
    for name, value in over.items():
        setattr(p, name, value)
    return p


def refused(rc, message):
    assert rc != 0
    assert message in _hip.LIB.fl_last_error().decode()


BAD_CACHES = [
    (dict(dtype=4), "bf16, fp16, fp32 or e4m3"),
    (dict(head_dim=96), "unsupported head_dim 96"),
    (dict(batch=0), "empty input"),
    (dict(rows=0), "empty input"),
    (dict(tokens=-1), "empty input"),
    (dict(outer=3), "batch size mismatch"),
    (dict(block_tables=256, max_blocks=0), "at least one block"),
    (dict(block_tables=256, max_blocks=1 << 30), "too long"),
    (dict(cu_seqlens=0, tokens_per_seq=4), "tokens_per_seq"),
    (dict(tokens=(1 << 31) - 1), "too large"),
    (dict(k=0), "null tensor pointer"),
    (dict(dtype=3), "go with an e4m3 cache"),
    (dict(k_scales=256), "go with an e4m3 cache"),
    (dict(k=264), "k_cache must have 16-byte aligned rows"),
    (dict(v_seq_stride=132), "v_cache must have 16-byte aligned rows"),
    (dict(dtype=3, k_scales=256, v_scales=256, k_seq_stride=136), "k_cache must have 16-byte aligned rows"),
    (dict(seq_lens=258), "4-byte aligned"),
    (dict(cu_seqlens=258), "4-byte aligned"),
    (dict(block_tables=257, max_blocks=1), "4-byte aligned"),
]


@pytest.mark.parametrize("over,message", BAD_CACHES, ids=[m for _, m in BAD_CACHES])
def test_c_entries_refuse_a_bad_cache(over, message):
    c = c_cache(**over)
    for call in (_hip.LIB.fl_cache_write, _hip.LIB.fl_cache_read):
        refused(call(ctypes.byref(c), ctypes.byref(c_rows()), None), message)
    refused(_hip.LIB.fl_cached_attention(ctypes.byref(c_attn(c)), 256, None), message)


def test_c_entries_refuse_bad_rows():
    c = c_cache()
    call = lambda **over: _hip.LIB.fl_cache_write(ctypes.byref(c), ctypes.byref(c_rows(**over)), None)
    refused(call(dtype=3), "token rows are bf16, fp16, or fp32")
    refused(call(dtype=1), "the cache's dtype")
    refused(call(k=0), "null tensor pointer")
    refused(call(k=260), "k must have 16-byte aligned rows")
    refused(call(v_head_stride=66), "v must have 16-byte aligned rows")
    refused(_hip.LIB.fl_cache_write(None, None, None), "null cache parameters")
    # (no tokens: nothing to do, and no pointer of theirs is needed)
    assert _hip.LIB.fl_cache_write(ctypes.byref(c_cache(tokens=0)), ctypes.byref(c_rows(k=0, v=0)), None) == 0


def test_c_attention_refuses_bad_calls():
    call = lambda p: _hip.LIB.fl_cached_attention(ctypes.byref(p), 256, None)
    refused(call(c_attn(dtype=2)), "takes bf16 or fp16")
    refused(call(c_attn(dtype=1)), "q's dtype")
    refused(call(c_attn(heads=0)), "empty input")
    refused(call(c_attn(heads=3)), "multiple of KV heads")
    refused(call(c_attn(num_splits=129)), "num_splits must be in [0, 128]")
    refused(call(c_attn(softmax_scale=0.0)), "softmax_scale must be positive")
    refused(call(c_attn(q=0)), "null tensor pointer")
    refused(call(c_attn(q=264)), "q must have 16-byte aligned rows")
    refused(call(c_attn(o_head_stride=68)), "o must have 16-byte aligned rows")
    refused(call(c_attn(lse=258)), "lse must be 4-byte aligned")
    refused(call(c_attn(num_splits=2, workspace_bytes=64)), "workspace is missing or smaller")
    refused(call(c_attn(num_splits=2, workspace=0)), "workspace is missing or smaller")
    refused(call(c_attn(num_splits=2, workspace=264)), "16-byte aligned")
    refused(_hip.LIB.fl_cached_attention(None, 256, None), "null attention parameters")
    refused(call(c_attn(c_cache(tokens=(1 << 29)), heads=4)), "too large")
    size = ctypes.c_size_t()
    p = c_attn(c_cache(tokens=1 << 22, heads_kv=4), heads=4, num_splits=128)
    refused(_hip.LIB.fl_cached_attention_plan(ctypes.byref(p), 256, ctypes.byref(size)), "grid limit")
    assert call(c_attn(c_cache(tokens=0))) == 0


def test_struct_layouts():
    # Natural C alignment: 7 pointers + 13 int64 + 9 int32 (+4 pad) = 200 bytes; 2 pointers + 6 int64 + int32
    # (+4 pad) = 72; 200 + 3 pointers + 6 int64 + 4 int32 + double + pointer + size_t = 312.
    assert ctypes.sizeof(_hip.KvCache) == 200
    assert ctypes.sizeof(_hip.TokenRows) == 72
    assert ctypes.sizeof(_hip.CachedAttnParams) == 312


def test_c_attention_refuses_sizes_beyond_its_counters():
    call = lambda p: _hip.LIB.fl_cached_attention(ctypes.byref(p), 256, None)
    far = 1 << 32
    refused(call(c_attn(c_cache(k_seq_stride=far))), "stride too large")
    pool = dict(block_tables=256, max_blocks=4)
    refused(call(c_attn(c_cache(v_batch_stride=far, **pool))), "stride too large")
    codes = dict(dtype=3, k_scales=256, v_scales=256)
    refused(call(c_attn(c_cache(ks_seq_stride=far, **codes))), "scales stride too large")
    refused(call(c_attn(c_cache(block_tables=256, max_blocks=(1 << 31) // 40))), "cache too long")
    refused(call(c_attn(c_cache(rows=(1 << 31) - 1))), "cache too long")
    # A grid has less than 2^32 threads, that of the merge too.
    refused(call(c_attn(c_cache(tokens=1 << 26), heads=16, num_splits=128)), "grid limit")
    refused(call(c_attn(c_cache(batch=1 << 17, outer=1 << 17, tokens=1 << 17), heads=2, num_splits=128)), "grid limit")
    size = ctypes.c_size_t()
    refused(_hip.LIB.fl_cached_attention_plan(ctypes.byref(c_attn(c_cache(tokens=1 << 26), heads=16, num_splits=128)), 256,
                                              ctypes.byref(size)), "grid limit")

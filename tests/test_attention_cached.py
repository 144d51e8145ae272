"""flash_lab.attention_cached and decode over a cache in 8 bits against the float64 oracle
(oracle/cache.py), with the bounds of cache_cases.check_attention. Unwritten rows of every cache hold NaN.
"""

import pytest
import torch

import flash_lab
from cache_cases import check_attention, cumulative, make_cache

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
TYPES = {"bf16": (torch.bfloat16, False), "fp16": (torch.float16, False), "bf16-e4m3": (torch.bfloat16, True),
         "fp16-e4m3": (torch.float16, True)}

# lens, new tokens, heads, heads_kv, head_dim, page (0: slabs)
RAGGED = {
    "one-token-each": ([1, 17, 300], [1, 1, 1], 8, 2, 128, 16),
    "prompt-and-steps": ([130, 65, 700, 64], [130, 1, 33, 0], 8, 2, 128, 16),
    "empty-sequences": ([0, 5, 0, 90], [0, 5, 3, 0], 4, 4, 64, 5),
    "more-new-than-held": ([10, 200], [40, 199], 8, 8, 64, 0),
    "group-of-3": ([333, 257], [70, 257], 6, 2, 128, 48),
    "group-of-16": ([500, 31], [9, 31], 16, 1, 64, 64),
    "group-of-160": ([90], [3], 160, 1, 64, 16),
    "page-of-1": ([77, 130], [20, 2], 4, 2, 128, 1),
    "tile-edges": ([63, 64, 65, 127, 128, 129], [63, 64, 65, 1, 2, 128], 4, 1, 64, 16),
    "slabs": ([400, 1, 129], [128, 1, 129], 8, 2, 128, 0),
    "long": ([2500, 40], [2, 40], 4, 2, 128, 64),
    "many-rows": ([600, 520], [600, 300], 16, 2, 64, 16),
}


@pytest.mark.parametrize("case", RAGGED, ids=list(RAGGED))
@pytest.mark.parametrize("types", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_ragged_batches(case, types, causal):
    lens, counts, heads, heads_kv, head_dim, page = RAGGED[case]
    dtype, quantized = TYPES[types]
    print(f"attention_cached {case} {types} causal={causal}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = make_cache(lens, max(lens) + 70, heads_kv, head_dim, dtype, quantized, page, gen)
    q = torch.randn(sum(counts) + 2, heads, head_dim, device="cuda", dtype=dtype, generator=gen)
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative(counts), causal=causal, return_lse=True, **cache)
    check_attention(out, lse, q, cache, counts, causal)


@pytest.mark.parametrize("types", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("seqlen_q", [1, 5, 100])
def test_the_same_number_of_tokens_each(types, head_dim, seqlen_q):
    # [B, S_q, H, D] queries without cu_seqlens, cross attention to states of a length each, one of them 0.
    dtype, quantized = TYPES[types]
    gen = torch.Generator(device="cuda").manual_seed(2)
    cache = make_cache([150, 0, 1, 333], 333, 4, head_dim, dtype, quantized, 0, gen, layout="bhsd")
    q = torch.randn(4, 8, seqlen_q, head_dim, device="cuda", dtype=dtype, generator=gen).transpose(1, 2)
    for causal in (False, True):
        out, lse = flash_lab.attention_cached(q, causal=causal, return_lse=True, **cache)
        assert out.shape == q.shape and lse.shape == q.shape[:3]
        check_attention(out, lse, q, cache, [seqlen_q] * 4, causal)


@pytest.mark.parametrize("batch", [65, 130, 300])
def test_more_sequences_than_lanes(batch):
    gen = torch.Generator(device="cuda").manual_seed(3)
    lens = torch.randint(0, 200, (batch,), generator=torch.Generator().manual_seed(batch)).tolist()
    counts = [min(n, i % 4) for i, n in enumerate(lens)]
    cache = make_cache(lens, 300, 2, 64, torch.bfloat16, True, 16, gen)
    q = torch.randn(sum(counts) + 1, 8, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative(counts), return_lse=True, **cache)
    check_attention(out, lse, q, cache, counts)


@pytest.mark.parametrize("dtype", HALF, ids=["bf16", "fp16"])
@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("heads,heads_kv,head_dim", [(32, 8, 128), (8, 8, 64), (64, 4, 128), (3, 1, 64)])
def test_decode_over_8_bits(dtype, page, heads, heads_kv, head_dim):
    gen = torch.Generator(device="cuda").manual_seed(4)
    lens = [1, 700, 64, 2049]
    cache = make_cache(lens, 2100, heads_kv, head_dim, dtype, True, page, gen)
    q = torch.randn(4, 1, heads, head_dim, device="cuda", dtype=dtype, generator=gen)
    out, lse = flash_lab.decode(q, return_lse=True, **cache)
    assert out.shape == q.shape and lse.shape == (4, heads)
    check_attention(out, lse[:, None], q, cache, [1] * 4)
    out3, lse3 = flash_lab.decode(q[:, 0], return_lse=True, **cache)
    assert torch.equal(out3, out[:, 0]) and torch.equal(lse3, lse)


@pytest.mark.parametrize("num_splits", [1, 2, 7, 64, 128])
def test_split_counts(num_splits):
    # More splits than tiles leaves some without keys.
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = make_cache([2000, 40, 777, 1], 2048, 2, 128, torch.bfloat16, True, 16, gen)
    q = torch.randn(4, 1, 16, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    out, lse = flash_lab.decode(q, num_splits=num_splits, return_lse=True, **cache)
    check_attention(out, lse[:, None], q, cache, [1] * 4)
    # A count of one's own pins a sequence's bits, whatever else is in the batch.
    one = {name: x if x is None or name in ("k_cache", "v_cache", "k_scales", "v_scales") else x[2:3]
           for name, x in cache.items()}
    assert torch.equal(flash_lab.decode(q[2:3], num_splits=num_splits, **one), out[2:3])


def test_the_same_call_gives_the_same_bits():
    gen = torch.Generator(device="cuda").manual_seed(6)
    counts = [3, 0, 64, 1, 190]
    cache = make_cache([3000, 10, 900, 2500, 190], 3000, 2, 128, torch.bfloat16, True, 16, gen)
    q = torch.randn(sum(counts), 8, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    first = flash_lab.attention_cached(q, cu_seqlens=cumulative(counts), return_lse=True, **cache)
    for _ in range(3):
        again = flash_lab.attention_cached(q, cu_seqlens=cumulative(counts), return_lse=True, **cache)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    check_attention(*first, q, cache, counts)


def test_rows_before_and_behind_the_sequences():
    gen = torch.Generator(device="cuda").manual_seed(7)
    cache = make_cache([90, 33], 100, 2, 64, torch.float16, False, 16, gen)
    q = torch.randn(40, 4, 64, device="cuda", dtype=torch.float16, generator=gen)
    q[:7] = float("nan")
    q[20:] = float("nan")
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative([10, 3], start=7), return_lse=True, **cache)
    check_attention(out, lse, q.nan_to_num(0.0), cache, [10, 3], start=7)


def test_no_tokens_at_all():
    gen = torch.Generator(device="cuda").manual_seed(8)
    cache = make_cache([9, 3], 20, 2, 64, torch.bfloat16, True, 16, gen)
    q = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative([0, 0]), return_lse=True, **cache)
    assert out.shape == q.shape and lse.shape == (0, 4)


def test_strides():
    # q and the caches are slices of larger tensors; the table is a column range of a wider one.
    gen = torch.Generator(device="cuda").manual_seed(9)
    cache = make_cache([150, 70], 160, 2, 64, torch.bfloat16, False, 16, gen)
    wide_q = torch.randn(30, 3, 8, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    q = wide_q[:, 1]
    both = torch.stack([cache["k_cache"], cache["v_cache"]], dim=2)  # [N, P, 2, H_kv, D]
    tables = torch.full((2, 40), 1 << 30, device="cuda", dtype=torch.int32)
    tables[:, 5:15] = cache["block_tables"]
    strided = dict(cache, k_cache=both[:, :, 0], v_cache=both[:, :, 1], block_tables=tables[:, 5:15])
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative([20, 10]), return_lse=True, **strided)
    want = flash_lab.attention_cached(q.contiguous(), cu_seqlens=cumulative([20, 10]), return_lse=True, **cache)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    check_attention(out, lse, q, cache, [20, 10])


def test_lengths_beyond_the_cache_are_held_to_it():
    gen = torch.Generator(device="cuda").manual_seed(10)
    cache = make_cache([64, 64], 64, 2, 64, torch.bfloat16, True, 0, gen)
    q = torch.randn(2, 1, 4, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    want = flash_lab.decode(q, **cache)
    cache["seq_lens"] = torch.tensor([1 << 30, 64], device="cuda", dtype=torch.int32)
    assert torch.equal(flash_lab.decode(q, **cache), want)
    cache["seq_lens"] = torch.tensor([-5, 64], device="cuda", dtype=torch.int32)
    out, lse = flash_lab.decode(q, return_lse=True, **cache)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and torch.equal(out[1], want[1])


@pytest.mark.parametrize("quantized", [False, True], ids=["same", "e4m3"])
def test_dominant_scores_and_large_values(quantized):
    # One key far above the rest, early and late; scores of +-200; a scale of one's own.
    gen = torch.Generator(device="cuda").manual_seed(11)
    cache = make_cache([700], 704, 1, 64, torch.bfloat16, quantized, 16, gen)
    q = 6 * torch.randn(33, 2, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative([33]), softmax_scale=0.5, return_lse=True, **cache)
    check_attention(out, lse, q, cache, [33], scale=0.5)


def test_a_nan_query_stays_its_own_rows():
    gen = torch.Generator(device="cuda").manual_seed(12)
    cache = make_cache([300], 304, 2, 128, torch.bfloat16, True, 16, gen)
    q = torch.randn(20, 8, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    want = flash_lab.attention_cached(q, cu_seqlens=cumulative([20]), **cache)
    bad = q.clone()
    bad[5, 3] = float("nan")
    out = flash_lab.attention_cached(bad, cu_seqlens=cumulative([20]), **cache)
    assert torch.isnan(out[5, 3]).all()
    keep = torch.ones(20, 8, dtype=torch.bool, device="cuda")
    keep[5, 3] = False
    assert torch.equal(out[keep], want[keep])


@pytest.mark.slow
@pytest.mark.parametrize("quantized", [False, True], ids=["same", "e4m3"])
def test_offsets_past_32_bits(quantized):
    # The sequence's blocks lie at both ends of a pool of more than 2^32 elements.
    page, heads_kv, head_dim = 64, 8, 128
    blocks = (1 << 32) // (page * heads_kv * head_dim) + 600
    gen = torch.Generator(device="cuda").manual_seed(13)
    small = make_cache([1000, 400], 1024, heads_kv, head_dim, torch.bfloat16, quantized, page, gen, spare=0)
    used = small["k_cache"].shape[0]
    place = torch.cat([torch.arange(used // 2), torch.arange(blocks - used + used // 2, blocks)]).cuda()
    big = dict(small, block_tables=place[small["block_tables"].long()].to(torch.int32))
    for name in ("k_cache", "v_cache", "k_scales", "v_scales"):
        x = small[name]
        if x is not None:
            pool = torch.zeros((blocks, *x.shape[1:]), device="cuda",
                               dtype=torch.uint8 if quantized else torch.int16)
            pool[place] = x.view(pool.dtype)
            big[name] = pool.view(x.dtype)
    q = torch.randn(30, 16, head_dim, device="cuda", dtype=torch.bfloat16, generator=gen)
    got = flash_lab.attention_cached(q, cu_seqlens=cumulative([29, 1]), return_lse=True, **big)
    want = flash_lab.attention_cached(q, cu_seqlens=cumulative([29, 1]), return_lse=True, **small)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cu = cumulative([1000, 400])
    got = flash_lab.read_cache(big.pop("k_cache"), big.pop("v_cache"), big.pop("seq_lens"), cu, 1400, **big)
    want = flash_lab.read_cache(small.pop("k_cache"), small.pop("v_cache"), small.pop("seq_lens"), cu, 1400, **small)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_replays_in_a_hip_graph_with_new_lengths():
    # The call reads lengths and tables on the device: a captured one follows them.
    gen = torch.Generator(device="cuda").manual_seed(14)
    cache = make_cache([1500, 900], 1600, 2, 128, torch.bfloat16, True, 16, gen)
    cache["k_cache"].view(torch.uint8)[cache["k_cache"].view(torch.uint8) == 0x7F] = 0x20
    cache["v_cache"].view(torch.uint8)[cache["v_cache"].view(torch.uint8) == 0x7F] = 0x20
    cache["k_scales"].fill_(120)
    cache["v_scales"].fill_(120)
    q = torch.randn(12, 8, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    cu = cumulative([8, 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flash_lab.attention_cached(q, cu_seqlens=cu, **cache)  # warm the allocator
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **cache)
    for lens, counts in (([1500, 900], [8, 4]), ([20, 1601], [1, 11]), ([700, 700], [12, 0]), ([1500, 900], [8, 4])):
        cache["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(cumulative(counts))
        eager = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **cache)
        captured[0].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1])
        _ = (q.float() * 2).sum().item()  # eager work between replays


def test_two_calls_on_two_streams():
    gen = torch.Generator(device="cuda").manual_seed(15)
    cache = make_cache([3000, 2000], 3008, 2, 128, torch.bfloat16, True, 16, gen)
    q = [torch.randn(2, 1, 8, 128, device="cuda", dtype=torch.bfloat16, generator=gen) for _ in range(2)]
    want = [flash_lab.decode(x, **cache) for x in q]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, s in zip(q, streams):
            with torch.cuda.stream(s):
                got.append(flash_lab.decode(x, **cache))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_traces_without_graph_breaks():
    torch._dynamo.reset()
    gen = torch.Generator(device="cuda").manual_seed(16)
    cache = make_cache([90, 33], 100, 2, 64, torch.bfloat16, True, 16, gen)
    q = torch.randn(13, 4, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    k, v = torch.randn(2, 13, 2, 64, device="cuda", dtype=torch.bfloat16, generator=gen)

    def step(q, k, v, cu, cache):
        flash_lab.write_cache(k, v, cu_seqlens=cu, **cache)
        out, lse = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **cache)
        return out * 2, lse

    cu = cumulative([10, 3])
    copy = {name: None if x is None else x.clone() for name, x in cache.items()}
    want = step(q, k, v, cu, cache)
    got = torch.compile(step, fullgraph=True)(q, k, v, cu, copy)
    assert torch.equal(copy["k_cache"].view(torch.uint8), cache["k_cache"].view(torch.uint8))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)


def test_refused_types():
    gen = torch.Generator(device="cuda").manual_seed(18)
    cache = make_cache([40], 48, 2, 64, torch.bfloat16, True, 16, gen)
    for dtype in (torch.float32, torch.float64):
        with pytest.raises(ValueError, match="no available implementation supports"):
            flash_lab.decode(torch.zeros(1, 1, 4, 64, device="cuda", dtype=dtype), **cache)
    wide = make_cache([40], 48, 2, 64, torch.float32, False, 16, gen)
    with pytest.raises(ValueError, match="is not one of"):
        flash_lab.attention_cached(torch.zeros(1, 1, 4, 64, device="cuda"), impl="cached_mma", **wide)
    with pytest.raises(ValueError, match="one device"):
        flash_lab.attention_cached(torch.zeros(1, 1, 4, 64, device="cuda", dtype=torch.bfloat16),
                                   **dict(cache, seq_lens=cache["seq_lens"].cpu()))


def test_a_backward_is_refused():
    gen = torch.Generator(device="cuda").manual_seed(17)
    cache = make_cache([40], 48, 2, 64, torch.bfloat16, False, 16, gen)
    q = torch.randn(4, 4, 64, device="cuda", dtype=torch.bfloat16, generator=gen).requires_grad_()
    out = flash_lab.attention_cached(q, cu_seqlens=cumulative([4]), **cache)
    with pytest.raises(RuntimeError, match="no autograd formula was registered"):
        out.sum().backward()
    k = torch.randn(4, 2, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError, match="write_cache has no gradient"):
        flash_lab.write_cache(k, k, cu_seqlens=cumulative([4]), **cache)
    # A graph that saved the cache notices the write.
    w = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = (cache["k_cache"] * w)
    flash_lab.write_cache(k.detach(), k.detach(), cu_seqlens=cumulative([4]), **cache)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()

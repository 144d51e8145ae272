"""How flash_lab.attention_cached shares out its work, against the float64 oracle with the bounds of
cache_cases.check_attention: batches that take each of its schedules (equal shares, a line of tiles, whole
blocks), sequences of few and of many rows in one call, and values that are not finite in places that some
rows do not see."""

import math

import pytest
import torch

import flash_lab
from cache_cases import NAN_CODE, check_attention, cumulative, make_cache

pytestmark = pytest.mark.gpu

TYPES = {"bf16": (torch.bfloat16, False), "fp16": (torch.float16, False), "bf16-e4m3": (torch.bfloat16, True),
         "fp16-e4m3": (torch.float16, True)}


def ints(n, low, high, seed):
    return torch.randint(low, high, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def run(lens, counts, heads, heads_kv, head_dim, types, page, seed, ragged=True, causal=True):
    dtype, quantized = TYPES[types]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache = make_cache(lens, max(lens) + 10, heads_kv, head_dim, dtype, quantized, page, gen)
    if ragged:
        q = torch.randn(sum(counts), heads, head_dim, device="cuda", dtype=dtype, generator=gen)
        got = flash_lab.attention_cached(q, cu_seqlens=cumulative(counts), causal=causal, return_lse=True, **cache)
    else:
        q = torch.randn(len(lens), counts[0], heads, head_dim, device="cuda", dtype=dtype, generator=gen)
        got = flash_lab.attention_cached(q, causal=causal, return_lse=True, **cache)
    check_attention(*got, q, cache, counts, causal)


@pytest.mark.parametrize("types", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("head_dim", [64, 128])
def test_more_blocks_than_workgroups(types, head_dim):
    # 20 sequences of 50 to 500 tokens, 8 KV heads: some 500 blocks of rows of different lengths, on the line.
    counts = ints(20, 50, 500, 1)
    lens = [c + more for c, more in zip(counts, ints(20, 0, 700, 2))]
    run(lens, counts, 16, 8, head_dim, types, 16, 3)


@pytest.mark.parametrize("types", ["bf16", "fp16-e4m3"])
def test_many_rounds_of_blocks(types):
    # 200 sequences of 8 heads with a block each, more than six rounds of workgroups: whole blocks, longest first.
    run([70 + n for n in ints(200, 0, 60, 4)], [65] * 200, 8, 8, 64, types, 16, 5)


@pytest.mark.parametrize("ragged", [True, False], ids=["ragged", "uniform"])
@pytest.mark.parametrize("types", ["bf16", "bf16-e4m3"])
def test_one_long_sequence(types, ragged):
    # Few blocks over many keys: split, and the partials merged.
    run([9000], [300], 8, 2, 128, types, 16, 6, ragged)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("types", TYPES, ids=list(TYPES))
def test_steps_drafts_and_chunks_in_one_call(types, causal):
    # One row block, three, and large blocks; idle and empty sequences between them.
    counts = [1, 300, 0, 5, 12, 1, 0, 700, 3, 49]
    lens = [3000, 2200, 50, 777, 12, 64, 0, 700, 1029, 2048]
    run(lens, counts, 8, 2, 64, types, 16, 7, causal=causal)


@pytest.mark.parametrize("types", ["bf16", "bf16-e4m3"])
def test_tables_longer_than_an_item_keeps(types):
    # Blocks of one row: 2,600 entries for one block of rows without splits (32 sequences of 8 KV heads fill the chip).
    run([2600] + [30] * 31, [17] * 32, 32, 8, 64, types, 1, 8)


@pytest.mark.parametrize("batch", [65, 200])
def test_wide_sequences_beyond_a_wave_of_lanes(batch):
    counts = [n if n > 40 else n % 3 for n in ints(batch, 0, 70, 9)]
    lens = [c + more for c, more in zip(counts, ints(batch, 0, 200, 10))]
    run(lens, counts, 4, 2, 64, "bf16-e4m3", 16, 11)


@pytest.mark.parametrize("hidden", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("types", TYPES, ids=list(TYPES))
@pytest.mark.parametrize("length,count,bad", [
    (90, 5, 87), (2500, 5, 2497), (2500, 40, 2461), (300, 130, 180), (2500, 130, 2400), (5000, 300, 4701)])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(length, count, bad, types, hidden):
    # Keys and values of one of the new tokens. In e4m3 only NaN is one.
    dtype, quantized = TYPES[types]
    if quantized and not math.isnan(hidden):
        pytest.skip("e4m3 has no infinities")
    gen = torch.Generator(device="cuda").manual_seed(12)
    clean = make_cache([length, 700], 5008, 2, 128, dtype, quantized, 16, gen)
    q = torch.randn(count + 20, 8, 128, device="cuda", dtype=dtype, generator=gen)
    cu = cumulative([count, 20])
    block, row = clean["block_tables"][0, bad // 16].item(), bad % 16
    dims = slice(3, 90, 7)
    dirty = dict(clean)
    for t in "kv":
        x = clean[f"{t}_cache"].clone()
        if quantized:
            clean[f"{t}_cache"].view(torch.uint8)[block, row, :, dims] = 0
            x.view(torch.uint8)[block, row, :, dims] = NAN_CODE
        else:
            clean[f"{t}_cache"][block, row, :, dims] = 0.0
            x[block, row, :, dims] = hidden
        dirty[f"{t}_cache"] = x
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **dirty)
    want, want_lse = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **clean)
    first = bad - (length - count)  # token whose row sees the key
    assert not torch.isfinite(out[first:count][..., dims]).any()
    # The rows before it, and the other sequence, are what they are without it.
    out[first:count], lse[first:count] = want[first:count], want_lse[first:count]
    check_attention(out, lse, q, clean, [count, 20])
    # With the values alone, the row sums stay, and with them all other dims of the rows that see them.
    only_v = dict(clean, v_cache=dirty["v_cache"])
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **only_v)
    assert torch.equal(lse, want_lse)
    assert not torch.isfinite(out[first:count][..., dims]).any()
    out[first:count][..., dims] = want[first:count][..., dims]
    check_attention(out, lse, q, clean, [count, 20])


def test_sequences_that_overlap_leave_the_next_call_alone():
    # cu_seqlens that descends is not a batch: such a call writes nothing that is read here, and harms nothing.
    gen = torch.Generator(device="cuda").manual_seed(13)
    cache = make_cache([400, 300, 500], 500, 2, 128, torch.bfloat16, True, 16, gen)
    q = torch.randn(90, 8, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    for ends in ([0, 80, 10, 90], [90, 60, 30, 0], [0, 1 << 30, -5, 1 << 30], [-(1 << 31), -7, 0, 0]):
        flash_lab.attention_cached(q, cu_seqlens=torch.tensor(ends, device="cuda", dtype=torch.int32), **cache)
    torch.cuda.synchronize()
    out, lse = flash_lab.attention_cached(q, cu_seqlens=cumulative([70, 1, 19]), return_lse=True, **cache)
    check_attention(out, lse, q, cache, [70, 1, 19])


def test_two_captured_graphs_of_a_ragged_call():
    # Each has a workspace of its own, and replays follow one another in any order.
    gen = torch.Generator(device="cuda").manual_seed(14)
    caches = [make_cache([2500, 900, 64], 2512, 2, 128, torch.bfloat16, quantized, 16, gen) for quantized in (True, False)]
    q = torch.randn(341, 8, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    cu = cumulative([300, 1, 40])
    want = [flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **c) for c in caches]
    torch.cuda.synchronize()
    graphs, got = [], []
    for c in caches:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **c))
    for order in ((0, 1), (1, 0), (1, 1, 0, 0)):
        for i in order:
            got[i][0].fill_(7.0)
            graphs[i].replay()
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
        _ = (q.float() * 2).sum().item()  # eager work between replays

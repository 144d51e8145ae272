"""flash_lab.write_cache and read_cache, bit for bit against the definition (oracle/cache.py), and the whole
run of a served sequence: chunks written, attended to, decoded from."""

import math

import pytest
import torch

import flash_lab
from cache_cases import NAN_CODE, NAN_SCALE, check_attention, cumulative, make_cache
from oracle import cache as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def empty_cache(outer, rows, heads_kv, head_dim, dtype, quantized):
    """Filled with a pattern that no write leaves behind."""
    shape = (outer, rows, heads_kv, head_dim)
    if not quantized:
        full = torch.full(shape, math.nan, device="cuda", dtype=dtype)
        return dict(k_cache=full, v_cache=full.clone(), k_scales=None, v_scales=None)
    codes = torch.full(shape, 0xAA, device="cuda", dtype=torch.uint8)
    scales = torch.full(shape[:3], 0xBB, device="cuda", dtype=torch.uint8)
    return dict(k_cache=codes.view(torch.float8_e4m3fn), v_cache=codes.clone().view(torch.float8_e4m3fn),
                k_scales=scales, v_scales=scales.clone())


def bits(x):
    return x.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()]).cpu()


def check_rows(codes, scales, x):
    """codes [n, H_kv, D] and scales [n, H_kv] are x's rows, to the bit."""
    want, exponents = oracle.quantize_rows(x)
    assert torch.equal(scales.cpu().int(), exponents + 127)
    got = oracle.values(codes, scales)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("page", [0, 1, 5, 16])
@pytest.mark.parametrize("quantized", [False, True], ids=["same", "e4m3"])
def test_round_trip(dtype, head_dim, page, quantized):
    # Every row of the cache that is not written keeps its bytes; positions before the first and behind
    # the last row, and rows of no sequence, are dropped.
    print(f"write and read {dtype} {head_dim} {page} {quantized}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(0)
    capacity, heads_kv = 60, 3
    lens, counts = [7, 60, 0, 63, 2, 33], [7, 1, 0, 10, 5, 0]
    batch = len(lens)
    rows = page or capacity
    blocks = -(-capacity // rows)
    capacity = blocks * rows
    cache = empty_cache(batch * blocks if page else batch, rows, heads_kv, head_dim, dtype, quantized)
    tables = None
    if page:
        tables = torch.randperm(batch * blocks, device="cuda", generator=gen).to(torch.int32).view(batch, blocks)
    start, total = 2, 2 + sum(counts) + 3
    k, v = torch.randn(2, total, heads_kv, head_dim, device="cuda", dtype=dtype, generator=gen)
    cache.update(seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), block_tables=tables)
    before = {name: None if x is None else x.clone() for name, x in cache.items()}
    cu = cumulative(counts, start)
    assert flash_lab.write_cache(k, v, cu_seqlens=cu, **cache) is None

    untouched = torch.ones(cache["k_cache"].shape[:2], dtype=torch.bool)
    expected = {"k": torch.zeros(total, heads_kv, head_dim, dtype=torch.float64),
                "v": torch.zeros(total, heads_kv, head_dim, dtype=torch.float64)}
    for b, (n, c) in enumerate(zip(lens, counts)):
        for i in range(c):
            position = n - c + i
            if not 0 <= position < capacity:
                continue
            outer, row = (b, position) if not page else (int(tables[b, position // page]), position % page)
            untouched[outer, row] = False
            token = int(cu[b]) + i
            for name, x in (("k", k), ("v", v)):
                cell, scale = cache[f"{name}_cache"][outer, row], cache[f"{name}_scales"]
                if quantized:
                    check_rows(cell, scale[outer, row], x[token])
                    expected[name][token] = oracle.values(cell, scale[outer, row])
                else:
                    assert torch.equal(bits(cell), bits(x[token]))
                    expected[name][token] = x[token].cpu().double()
    for name in ("k_cache", "v_cache", "k_scales", "v_scales"):
        if cache[name] is not None:
            assert torch.equal(bits(cache[name])[untouched], bits(before[name])[untouched])

    args = dict(cache)
    got = flash_lab.read_cache(args.pop("k_cache"), args.pop("v_cache"), args.pop("seq_lens"), cu, total, dtype=dtype,
                               **args)
    for name, x in zip("kv", got):
        assert x.dtype == dtype and torch.equal(x.cpu().double(), expected[name])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("head_dim", [64, 128])
def test_every_magnitude(dtype, head_dim):
    # Rows from the type's least values to its largest, rows whose largest value lies next to 1.75 2^n (where
    # the scale changes), ties, zeros, and rows with infinities and NaN.
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(400, 2, head_dim, device="cuda", generator=gen)
    info = torch.finfo(dtype)
    powers = torch.linspace(math.log2(info.smallest_normal) - 3, math.log2(info.max) - 3, 300, device="cuda")
    x[:300] *= torch.exp2(powers)[:, None, None]
    x = x.to(dtype)
    edge = torch.tensor([1.75, 1.75 + info.eps, 1.75 - info.eps, 1.0, 2.0 - info.eps, 1.875], device="cuda", dtype=dtype)
    x[300:306] = x[300:306].clamp(-1, 1)
    x[300:306, :, 5] = edge[:, None]
    x[306] = 0
    x[307, 0] = -0.0
    x[308] = (torch.arange(2 * head_dim, device="cuda").view(2, head_dim) * 0.5 + 8.5).to(dtype)  # ties on the way
    x[309, :, 3] = math.inf
    x[310, :, 0] = -math.inf
    x[311, :, 7] = math.nan
    x[312] = math.nan
    x[313] = math.inf
    x[314] = info.max
    x[315] = -info.max
    x[316] = info.smallest_normal / 4
    cache = empty_cache(1, 400, 2, head_dim, dtype, True)
    lens = torch.tensor([400], dtype=torch.int32, device="cuda")
    flash_lab.write_cache(x[None], x.flip(0)[None], seq_lens=lens, **cache)
    check_rows(cache["k_cache"][0], cache["k_scales"][0], x)
    check_rows(cache["v_cache"][0], cache["v_scales"][0], x.flip(0))
    args = dict(cache)
    k, v = flash_lab.read_cache(args.pop("k_cache"), args.pop("v_cache"), lens, cumulative([400]), 400,
                                dtype=torch.float32, **args)
    want = oracle.values(cache["k_cache"][0], cache["k_scales"][0])
    # (float32 holds every code times every scale, down to 2^-126 2^-9 rounded to its own least step)
    assert torch.equal(k.cpu(), want.float()) or torch.equal(k.cpu().isnan(), want.isnan()) and torch.equal(
        k.cpu().nan_to_num(0.0), want.float().nan_to_num(0.0))
    if dtype != torch.float32:
        k, _ = flash_lab.read_cache(cache["k_cache"], cache["v_cache"], lens, cumulative([400]), 400, dtype=dtype,
                                    k_scales=cache["k_scales"], v_scales=cache["v_scales"])
        finite = torch.isfinite(want)
        assert torch.equal(torch.isfinite(k.cpu()), finite)  # nothing that the type held overflows in it
        assert torch.equal(k.cpu()[finite], want.to(dtype)[finite])


def test_every_code_and_scale_is_read_as_what_it_stands_for():
    codes = torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).view(4, 1, 64).expand(4, 254, 64)
    codes = codes.transpose(0, 1).contiguous()  # [254 rows, 4 heads, 64]
    scales = torch.arange(1, 255, device="cuda", dtype=torch.int32).to(torch.uint8).view(254, 1).expand(254, 4).contiguous()
    cache = dict(k_cache=codes[None].view(torch.float8_e4m3fn), v_cache=codes[None].view(torch.float8_e4m3fn),
                 k_scales=scales[None], v_scales=scales[None])
    lens = torch.tensor([254], dtype=torch.int32, device="cuda")
    want = oracle.values(cache["k_cache"][0], cache["k_scales"][0])
    for dtype in DTYPES:
        args = dict(cache)
        k, v = flash_lab.read_cache(args.pop("k_cache"), args.pop("v_cache"), lens, cumulative([254]), 254, dtype=dtype,
                                    **args)
        for x in (k, v):
            x = x.cpu()
            assert torch.equal(x.isnan(), want.isnan())
            assert torch.equal(x.nan_to_num(0.0, math.inf, -math.inf), want.to(dtype).nan_to_num(0.0, math.inf, -math.inf))


@pytest.mark.parametrize("batch", [63, 64, 65, 200])
@pytest.mark.parametrize("heads_kv", [1, 5])
def test_more_sequences_than_lanes(batch, heads_kv):
    gen = torch.Generator(device="cuda").manual_seed(2)
    counts = [i % 3 for i in range(batch)]
    lens = [c + i % 7 for i, c in enumerate(counts)]
    cache = empty_cache(batch, 16, heads_kv, 64, torch.bfloat16, True)
    k, v = torch.randn(2, sum(counts), heads_kv, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    flash_lab.write_cache(k, v, cu_seqlens=cumulative(counts), seq_lens=lens_t, **cache)
    at = 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        check_rows(cache["k_cache"][b, n - c : n], cache["k_scales"][b, n - c : n], k[at : at + c])
        check_rows(cache["v_cache"][b, n - c : n], cache["v_scales"][b, n - c : n], v[at : at + c])
        at += c


def test_strided_rows_and_caches():
    # Rows sliced out of a packed projection; a cache that is a transposed view, its scales another one.
    gen = torch.Generator(device="cuda").manual_seed(3)
    packed = torch.randn(2, 30, 4, 5, 128, device="cuda", dtype=torch.float16, generator=gen)
    k, v = packed[:, :, 1], packed[:, :, 3]
    base = empty_cache(2, 50, 5, 128, torch.float16, True)
    cache = {name: x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(x.dtype)
             for name, x in base.items()}
    lens = torch.tensor([50, 31], dtype=torch.int32, device="cuda")
    flash_lab.write_cache(k, v, seq_lens=lens, **cache)
    for b, n in enumerate((50, 31)):
        check_rows(cache["k_cache"][b, n - 30 : n], cache["k_scales"][b, n - 30 : n], k[b])
        check_rows(cache["v_cache"][b, n - 30 : n], cache["v_scales"][b, n - 30 : n], v[b])


def test_table_entries_outside_the_pool():
    # A write drops their tokens, a read takes the pool's first or last block.
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache = empty_cache(3, 4, 2, 64, torch.bfloat16, True)
    before = cache["k_cache"].clone()
    tables = torch.tensor([[1, -7, 1 << 30]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([12], dtype=torch.int32, device="cuda")
    k, v = torch.randn(2, 1, 12, 2, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    flash_lab.write_cache(k, v, seq_lens=lens, block_tables=tables, **cache)
    check_rows(cache["k_cache"][1], cache["k_scales"][1], k[0, :4])
    for block in (0, 2):
        assert torch.equal(bits(cache["k_cache"][block]), bits(before[block]))
    args = dict(cache)
    got, _ = flash_lab.read_cache(args.pop("k_cache"), args.pop("v_cache"), lens, cumulative([12]), 12,
                                  block_tables=tables, **args)
    want = oracle.values(cache["k_cache"], cache["k_scales"])
    assert torch.equal(got.cpu().double(), torch.cat([want[1], want[0], want[2]]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("quantized", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("page", [0, 16])
def test_a_served_batch(dtype, quantized, page):
    """Prompts in chunks, then steps: each call writes its tokens and attends to all so far. What the last
    call sees is compared with the prefill operator on the rows read back, and every call with float64."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    heads, heads_kv, head_dim, capacity = 8, 2, 128, 320
    calls = [[100, 7, 0], [60, 0, 129], [1, 1, 1], [5, 1, 30], [1, 1, 1]]
    cache = make_cache([0, 0, 0], capacity, heads_kv, head_dim, dtype, quantized, page, gen)
    lens = [0, 0, 0]
    kept = [[], [], []]
    for counts in calls:
        lens = [n + c for n, c in zip(lens, counts)]
        cache["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        total = sum(counts)
        q = torch.randn(total, heads, head_dim, device="cuda", dtype=dtype, generator=gen)
        k, v = torch.randn(2, total, heads_kv, head_dim, device="cuda", dtype=dtype, generator=gen)
        cu = cumulative(counts)
        flash_lab.write_cache(k, v, cu_seqlens=cu, **cache)
        out, lse = flash_lab.attention_cached(q, cu_seqlens=cu, return_lse=True, **cache)
        check_attention(out, lse, q, cache, counts)
        for b in range(3):
            kept[b].append((q[int(cu[b]) : int(cu[b + 1])], out[int(cu[b]) : int(cu[b + 1])]))
    # One token per sequence through decode as well.
    step = q[:, None] if total == 3 else None
    decoded, decoded_lse = flash_lab.decode(step, return_lse=True, **cache)
    check_attention(decoded, decoded_lse[:, None], step, cache, [1, 1, 1])
    args = dict(cache)
    args.pop("seq_lens")
    rows = flash_lab.read_cache(args.pop("k_cache"), args.pop("v_cache"), cache["seq_lens"], cumulative(lens), sum(lens),
                                dtype=dtype, **args)
    at = 0
    u = torch.finfo(dtype).eps / 2
    for b, n in enumerate(lens):
        q = torch.cat([x for x, _ in kept[b]])[None]
        out = torch.cat([x for _, x in kept[b]])[None]
        k, v = (x[at : at + n][None] for x in rows)
        at += n
        want = flash_lab.attention(q, k, v, causal=True)
        # Both are within u sum p |v| + u |o| (and 1% for fp32) of the same values: sum p |v| <= max |v|.
        assert ((out.double() - want.double()).abs() <= 2.02 * u * (v.abs().max() + want.abs()).double()).all()


def test_write_and_read_replay_in_a_hip_graph():
    gen = torch.Generator(device="cuda").manual_seed(6)
    cache = empty_cache(10, 16, 2, 128, torch.bfloat16, True)
    tables = torch.randperm(10, device="cuda", generator=gen).to(torch.int32).view(2, 5)
    lens = torch.tensor([30, 12], dtype=torch.int32, device="cuda")
    k, v = torch.randn(2, 2, 1, 2, 128, device="cuda", dtype=torch.bfloat16, generator=gen)
    cu = cumulative([1, 1])

    def step():
        flash_lab.write_cache(k, v, seq_lens=lens, block_tables=tables, **cache)
        return flash_lab.read_cache(cache["k_cache"], cache["v_cache"], lens, cu, 2, block_tables=tables,
                                    k_scales=cache["k_scales"], v_scales=cache["v_scales"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        lens.add_(3)
        k.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        want, _ = oracle.quantize_rows(k[:, 0])
        assert torch.equal(captured[0].cpu().double(), want)
        for b in range(2):
            n = int(lens[b]) - 1
            block, row = int(tables[b, n // 16]), n % 16
            check_rows(cache["k_cache"][block, row], cache["k_scales"][block, row], k[b, 0])


def test_opcheck():
    gen = torch.Generator(device="cuda").manual_seed(7)
    c = make_cache([20, 5], 32, 2, 64, torch.bfloat16, True, 16, gen)
    k = torch.randn(3, 2, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    c["k_cache"].view(torch.uint8)[c["k_cache"].view(torch.uint8) == NAN_CODE] = 0
    c["v_cache"].view(torch.uint8)[c["v_cache"].view(torch.uint8) == NAN_CODE] = 0
    c["k_scales"][c["k_scales"] == NAN_SCALE] = 127
    c["v_scales"][c["v_scales"] == NAN_SCALE] = 127
    cu = cumulative([2, 1])
    names = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(torch.ops.flash_lab.read_cache.default,
                          (c["k_cache"], c["v_cache"], c["k_scales"], c["v_scales"], c["seq_lens"], cu,
                           c["block_tables"], 3, torch.bfloat16), test_utils=names[2:])
    q = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16, generator=gen)
    torch.library.opcheck(torch.ops.flash_lab.attention_cached.default,
                          (q, c["k_cache"], c["v_cache"], c["k_scales"], c["v_scales"], c["seq_lens"], cu,
                           c["block_tables"], True, 0.125, 0), test_utils=names[2:])
    plain = make_cache([20, 5], 32, 2, 64, torch.bfloat16, False, 16, gen)
    torch.library.opcheck(torch.ops.flash_lab.write_cache.default,
                          (k, k, plain["k_cache"].nan_to_num(0.0), plain["v_cache"].nan_to_num(0.0), None, None,
                           plain["seq_lens"], cu, plain["block_tables"]), test_utils=names)

"""Caches, tokens and error bounds for the tests of the cache operators."""

import math

import torch

from oracle import cache as oracle

NAN_CODE, NAN_SCALE = 0x7F, 0xFF


def make_cache(lens, capacity, heads_kv, head_dim, dtype, quantized, page=0, gen=None, layout="bshd", spare=3):
    """A cache whose sequences hold lens[b] rows and NaN everywhere else. Returns a dict of the operators'
    cache arguments. layout "bhsd": views of [.., H_kv, rows, D] tensors; scales of pools lie the same way."""
    batch = len(lens)
    dev = "cuda"
    if page:
        blocks = -(-capacity // page)
        outer, rows = batch * blocks + spare, page
        tables = torch.randperm(outer, generator=gen, device=dev)[: batch * blocks]
        tables = tables.to(torch.int32).view(batch, blocks)
    else:
        outer, rows, tables = batch, capacity, None
    held = torch.zeros((outer, rows), dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        if page:
            for i in range(-(-n // page)):
                held[tables[b, i], : min(page, n - i * page)] = True
        else:
            held[b, :n] = True

    def one():
        shape = (outer, heads_kv, rows, head_dim) if layout == "bhsd" else (outer, rows, heads_kv, head_dim)
        x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)
        x *= torch.exp(0.5 * torch.randn(head_dim, generator=gen, device=dev))
        x = x.to(dtype)
        x = x.transpose(1, 2) if layout == "bhsd" else x
        if not quantized:
            x.masked_fill_(~held[..., None, None], math.nan)
            return x, None
        top = x.float().abs().amax(dim=-1)
        exponent = torch.ceil(torch.log2(top / 448.0)).clamp(-100, 100).to(torch.int32)
        codes = (x.float() * (127 - exponent << 23).view(torch.float32).unsqueeze(-1)).clamp(-448, 448)
        codes = codes.to(torch.float8_e4m3fn).view(torch.uint8)
        scales = (exponent + 127).to(torch.uint8)
        if layout == "bhsd":  # keep the strides
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
            scales = scales.transpose(1, 2).contiguous().transpose(1, 2)
        codes.masked_fill_(~held[..., None, None], NAN_CODE)
        scales.masked_fill_(~held[..., None], NAN_SCALE)
        return codes.view(torch.float8_e4m3fn), scales

    (k, ks), (v, vs) = one(), one()
    return dict(k_cache=k, v_cache=v, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                block_tables=tables, k_scales=ks, v_scales=vs)


def cumulative(counts, start=0):
    ends = [start]
    for n in counts:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


def check_attention(out, lse, q, cache, counts, causal=True, start=0, scale=None):
    """Every token of every sequence against float64, and rows of no sequence against (0, -inf).

    Bounds, with u half a step of the output type (2^-8 bf16, 2^-11 fp16), n keys, S the row's largest
    scale sum |q_d k_d| and A = sum_j p_j |v_j|:
      * a score is a sum of D products in fp32 (each addition off by 2^-24 of at most S), then scaled and
        shifted: off by d = (D + 8) 2^-24 S in natural-log units; with the exponential's own 2^-22, p and
        the sum of p are off by at most e = d + 2^-22 relative, their quotient by 2 e;
      * p is rounded to the input type (u A), and in fp16, below 2^-14, by at most 2^-25 against the largest
        p of at least 2^-3 (the reference point lags by at most 3): 2^-22 per key, n 2^-22 max |v|;
      * sums of n terms in fp32, and those of the merge: n 2^-24 each for o and for l;
      * codes times scales are exact in bf16 and, in these tests, in fp16;
      * the output is rounded: u |o|, or half of fp16's least step, 2^-25.
    """
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    out, lse, qd = out.cpu().double(), lse.cpu().double(), q.cpu().double()
    if q.dim() == 4:
        out, lse, qd = out.flatten(0, 1), lse.flatten(0, 1), qd.flatten(0, 1)
    head_dim = q.shape[-1]
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    capacity = cache["k_cache"].shape[1]
    if cache["block_tables"] is not None:
        capacity *= cache["block_tables"].shape[1]
    at = start
    assert (out[:start] == 0).all() and torch.isneginf(lse[:start]).all()
    for b, (n, c) in enumerate(zip(cache["seq_lens"].tolist(), counts)):
        n = min(max(n, 0), capacity)
        k, v = (oracle.rows_of(cache[f"{t}_cache"], cache[f"{t}_scales"], cache["block_tables"], b, n) for t in "kv")
        rows = slice(at, at + c)
        at += c
        o, want_lse, weight, size = oracle.attention(qd[rows], k, v, torch.arange(n - c, n), causal, scale)
        e = (head_dim + 8) * 2.0**-24 * size + 2.0**-22
        sums = (n + 16) * 2.0**-24
        bound = (u * (1 + u) + (2 * e + 2 * sums)[..., None]) * weight + u * o.abs()
        if dtype == torch.float16:
            bound += 2.0**-25 + (n * 2.0**-22 * v.abs().max() if n else 0.0)
        err = (out[rows] - o).abs()
        assert (err <= bound).all(), f"sequence {b}: {(err / bound.clamp(min=1e-300)).max():.3g} of the bound"
        seen = torch.isfinite(want_lse)
        assert torch.equal(torch.isneginf(lse[rows]), ~seen)
        lse_bound = 2 * e + sums + 2.0**-22 * want_lse.abs()
        assert ((lse[rows] - want_lse).abs() <= lse_bound)[seen].all()
    assert (out[at:] == 0).all() and torch.isneginf(lse[at:]).all()

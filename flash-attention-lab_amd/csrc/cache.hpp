// Device-side view of a key-value cache (CacheArgs): which sequence a token of the call belongs to, where
// a position's row lies, and e4m3 codes as values of the matrix cores' types.
#pragma once

#include "gfx950.hpp"
#include "launch.hpp"

namespace fl {
namespace cache {

// The call's tokens of one sequence, held to the call's and the cache's sizes whatever the arrays say.
struct Sequence {
  int start, count;  // tokens start .. start + count - 1 of the call
  int len;           // keys
};
__device__ __forceinline__ Sequence sequence(const CacheArgs& c, int b) {
  Sequence s;
  if (c.cu_seqlens != nullptr) {
    s.start = min(max(c.cu_seqlens[b], 0), c.tokens);
    s.count = min(max(c.cu_seqlens[b + 1], s.start), c.tokens) - s.start;
  } else {
    s.start = b * c.tokens_per_seq;
    s.count = c.tokens_per_seq;
  }
  s.len = min(max(c.seq_lens[b], 0), c.capacity);
  return s;
}

// A token's sequence, its index among the sequence's tokens and their number, and the sequence's length as
// the array has it. b < 0: the token belongs to none.
struct Token {
  int b, index, count, len;
};
// Every aligned group of kLanes lanes asks for a token of its own. All lanes of the wave take part.
template <int kLanes>
__device__ __forceinline__ Token find_token(const CacheArgs& c, int token) {
  Token t{-1, 0, 0, 0};
  if (c.cu_seqlens == nullptr) {
    t.b = token / c.tokens_per_seq;
    t.index = token - t.b * c.tokens_per_seq;
    t.count = c.tokens_per_seq;
    t.len = c.seq_lens[t.b];
    return t;
  }
  // The first sequence that ends behind the token, 64 ends at a time. Everything that is asked of a
  // sequence is loaded with its end: one memory latency in a batch of up to 64.
  const int lane = __lane_id();
  bool open = true;
  for (int base = 0; base < c.batch; base += 64) {
    const int b = min(base + lane, c.batch - 1);
    const int start = c.cu_seqlens[b];
    const int end = base + lane < c.batch ? c.cu_seqlens[b + 1] : INT32_MAX;
    const int len = c.seq_lens[b];
    int at = 64;
#pragma unroll
    for (int r = 0; r < 64 / kLanes; ++r) {
      const uint64_t behind = __builtin_amdgcn_ballot_w64(end > __builtin_amdgcn_readlane(token, r * kLanes));
      const int first = behind ? __builtin_ctzll(behind) : 64;
      at = lane / kLanes == r ? first : at;
    }
    const int from = at < 64 ? at : 0;
    const int s = __shfl(start, from);
    const int e = __shfl(end, from);
    const int n = __shfl(len, from);
    if (open && at < 64) {
      open = false;
      if (base + at < c.batch && s >= 0 && s <= token) t = Token{base + at, token - s, e - s, n};
    }
    if (!wave_any(open)) break;
  }
  return t;
}

// Where the row of a position in [0, capacity) lies: its slab or block, and the row in it. A table entry
// is not checked here.
struct Place {
  int outer, row;
};
__device__ __forceinline__ int row_in_block(const CacheArgs& c, int position) {
  return c.page_shift >= 0 ? position & (c.rows - 1) : position % c.rows;
}
__device__ __forceinline__ Place place(const CacheArgs& c, int b, int position) {
  if (c.block_tables == nullptr) return Place{b, position};
  const int page = c.page_shift >= 0 ? position >> c.page_shift : position / c.rows;
  return Place{c.block_tables[b * c.block_tables_stride + page], position - page * c.rows};
}

// 2^(byte - 127), the scale that an exponent byte stands for.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Four e4m3 codes (the bytes of `codes`, lowest first) times a power of two, as two packed pairs of Tag's
// elements. One instruction converts and scales a pair; in bf16 the result is exact (four significant
// bits), in fp16 it is where fp16 holds the value.
template <typename Tag>
__device__ __forceinline__ u32x2 values4(uint32_t codes, float scale) {
  if constexpr (std::is_same_v<Tag, bf16_tag>) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
  } else {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true))};
  }
}

}  // namespace cache
}  // namespace fl

// Pieces shared by the kernels of attention over a cache (cached_attn.hip: plan and merge; cached_narrow.hip:
// sequences with few rows; cached_pp.hip and cached_wide.hip: the
// others, at head_dim 128 and 64): the rows of a sequence, the items that the
// workgroups of a kernel share out, and the offsets of cache rows.
#pragma once

#include <type_traits>

#include "cache.hpp"
#include "decode_sched.hpp"
#include "prefill_tile.hpp"

namespace fl {
namespace cached {

// Kinds of sequences, by their rows (tokens x query heads of a KV head).
enum Kind { kNarrow, kWide };
constexpr int kNarrowRows = 48;  // most rows of a narrow sequence
constexpr int kKeys = 64;        // keys of a tile: splits are whole tiles
constexpr int kStartTiles = 4;   // tiles that starting and ending an item costs as much as
constexpr int kMaxRounds = 3;
// Rows of a block.
__host__ __device__ __forceinline__ constexpr int block_rows(Kind kind, int head_dim) {
  return kind == kNarrow ? kNarrowRows : head_dim == 128 ? 256 : 128;
}
// Workgroups of the wide kernel per CU.
constexpr int wide_resident(int head_dim) { return head_dim == 128 ? 1 : 2; }

namespace {

using cache::Sequence;
using decode::wave_inclusive_sum;

constexpr float kLn2 = 0.693147180559945309f;
// Running max before the first key: finite, so that a masked score (-inf) gives p = 0.
constexpr float kNoRef = -1e30f;

__device__ __forceinline__ int token_of_row(const CachedAttnArgs& a, int row) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(row)) * a.group_mul) >> a.group_shift);
}

__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_inclusive_sum(x), 63); }
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) x += __shfl_xor(x, m);
  return x;
}

// A workgroup's item: one split of one block of rows of one KV head of one sequence.
struct Item {
  int b, hkv, block, split, splits;
  int slot;        // of its partials, splits > 1
  int first_slot;  // of the sequence
  bool first;      // the sequence's first item
  Sequence seq;
};

// Blocks of rows and key tiles of a sequence; no blocks, if it is of the other kind.
struct Load {
  int blocks, tiles;
};
template <Kind kKind, int D>
__device__ __forceinline__ Load load_of(const CachedAttnArgs& a, const Sequence& s) {
  const int rows = s.count * a.group;
  const bool mine = (rows <= kNarrowRows) == (kKind == kNarrow);
  return Load{mine ? (rows + block_rows(kKind, D) - 1) / block_rows(kKind, D) : 0, (s.len + kKeys - 1) / kKeys};
}

// The items of a kernel, over the sequences of its kind: sequence b has blocks_b splits_b H_kv of them, with splits_b = ceil(tiles_b / share). a.slots
// workgroups run at once, so items of up to `share` tiles that fill r rounds of slots end after about
// r (share + what starting an item costs): share and r are chosen for the least of that, with the least
// share for which no more than r slots items result. Within a chunk of 64 sequences longer items come
// first where there is more than one round, so that the last ones to start are short. Lane l holds sequence
// 64 i + l of chunk i; chunks behind the first are read again in every pass.
template <Kind kKind, int D>
__device__ __forceinline__ bool find_item(const CachedAttnArgs& a, int id, Item& item) {
  const int lane = __lane_id();
  const int batch = a.c.batch;
  auto sequence_at = [&](int b) {
    Sequence s{0, 0, 0};
    if (b < batch) s = cache::sequence(a.c, b);
    return s;
  };
  const Sequence first = sequence_at(lane);
  const Load first_load = load_of<kKind, D>(a, first);
  // f(blocks, tiles) summed over all sequences.
  auto sum = [&](auto f) {
    auto total = f(first_load);
    for (int base = 64; base < batch; base += 64) total += f(load_of<kKind, D>(a, sequence_at(base + lane)));
    return wave_sum(total);
  };
  // Sequences that overlap (cu_seqlens does not ascend) could have more items than the grid and the
  // workspace are made for: no item is run then.
  if (a.c.cu_seqlens != nullptr) {
    float tokens = first.count;
    for (int base = 64; base < batch; base += 64) tokens += sequence_at(base + lane).count;
    if (wave_sum(tokens) > 1.001f * a.c.tokens) return false;
  }
  int share = 1 << 30;  // tiles of a split
  int rounds = 2;       // (more than one)
  if (a.num_splits == 0 && a.slots > 0) {
    const int blocks = a.c.heads_kv * sum([](const Load& l) { return l.blocks; });
    const float work = a.c.heads_kv * sum([](const Load& l) { return float(l.blocks) * float(l.tiles); });
    auto items = [&](int t) {
      return a.c.heads_kv * sum([t](const Load& l) { return l.blocks * max((l.tiles + t - 1) / t, 1); });
    };
    float least = INFINITY;
    for (int r = 1; r <= a.max_rounds; ++r) {
      const int slots = r * a.slots;
      if (blocks > slots) continue;
      // sum of ceil(x / t) is at most work / t + blocks.
      int low = max(a.min_tiles, static_cast<int>(work / slots));
      int high = blocks < slots ? max(low, static_cast<int>(work / (slots - blocks) * 1.001f) + 1) : 1 << 28;
      while (low < high) {
        const int mid = low + (high - low) / 2;
        if (items(mid) <= slots) {
          high = mid;
        } else {
          low = mid + 1;
        }
      }
      if (items(low) > slots) continue;
      const float time = r * static_cast<float>(low + kStartTiles);
      if (time < least) {
        least = time;
        share = low;
        rounds = r;
      }
      // (More rounds can't gain on one that is close to an even share.)
      if (low <= work / a.slots + kStartTiles) break;
    }
  }
  auto splits_of = [&](const Load& l) {
    return a.num_splits > 0 ? a.num_splits : max((l.tiles + share - 1) / share, 1);
  };
  int before = 0;       // items of earlier chunks
  int before_slot = 0;  // slots of earlier chunks
  for (int base = 0; base < batch; base += 64) {
    const Sequence s = base == 0 ? first : sequence_at(base + lane);
    const Load l = load_of<kKind, D>(a, s);
    const int splits = splits_of(l);
    const int items = l.blocks * splits * a.c.heads_kv;
    const int slots = splits > 1 ? items : 0;
    const int all = wave_inclusive_sum(items);
    const int all_slots = wave_inclusive_sum(slots);
    int from = all - items;  // items and slots of the chunk before the lane's
    int from_slot = all_slots - slots;
    if (rounds > 1) {
      const int length = l.tiles / splits;
      from = from_slot = 0;
      const int here = min(batch - base, 64);
      for (int j = 0; j < here; ++j) {
        const int other = __builtin_amdgcn_readlane(length, j);
        const bool ahead = other > length || (other == length && j < lane);
        from += ahead ? __builtin_amdgcn_readlane(items, j) : 0;
        from_slot += ahead ? __builtin_amdgcn_readlane(slots, j) : 0;
      }
    }
    const int local = id - before - from;
    const uint64_t mask = __builtin_amdgcn_ballot_w64(local >= 0 && local < items);
    if (mask) {
      const int owner = __builtin_ctzll(mask);
      auto of_owner = [&](int x) { return __builtin_amdgcn_readlane(x, owner); };
      item.b = base + owner;
      item.seq = Sequence{of_owner(s.start), of_owner(s.count), of_owner(s.len)};
      item.splits = of_owner(splits);
      const int at = of_owner(local);
      const int units = a.c.heads_kv * item.splits;  // items of a block
      const int turn = at / units;                   // blocks with more keys first
      const int unit = at - turn * units;
      item.hkv = unit / item.splits;
      item.split = unit - item.hkv * item.splits;
      item.block = of_owner(l.blocks) - 1 - turn;
      item.first_slot = before_slot + of_owner(from_slot);
      item.slot = item.first_slot + at;
      item.first = at == 0;
      return true;
    }
    before += __builtin_amdgcn_readlane(all, 63);
    before_slot += __builtin_amdgcn_readlane(all_slots, 63);
  }
  return false;
}

// Rows are moved in 16-byte pieces, kPerRow of them to a row.
template <int D, bool kE4M3>
struct Piece {
  static constexpr int kElem = kE4M3 ? 1 : 2;
  static constexpr int kElems = 16 / kElem;
  static constexpr int kPerRow = D / kElems;
};
// Where the rows of one sequence and KV head lie in a tensor (bytes, or scales): `base` and the strides between
// blocks (0 in a slab) and between rows, in bytes that fit 32 bits (checked on the host), so that an offset is
// two 32-bit products. It is worked out by one lane for all that move the row's pieces.
struct RowSpace {
  const char* base;
  uint32_t block_stride, row_stride;
  __device__ __forceinline__ uint64_t offset(const CacheArgs& c, const cache::Place& p) const {
    const uint32_t block = static_cast<uint32_t>(min(max(p.outer, 0), c.outer - 1));
    return static_cast<uint64_t>(block) * block_stride + static_cast<uint64_t>(static_cast<uint32_t>(p.row)) * row_stride;
  }
};
__device__ __forceinline__ RowSpace row_space(const CacheArgs& c, const void* tensor, int b, int hkv, int64_t bs,
                                              int64_t ss, int64_t hs, int elem) {
  const bool slab = c.block_tables == nullptr;
  return RowSpace{static_cast<const char*>(tensor) + (hkv * hs + (slab ? b * bs : 0)) * elem,
                  slab ? 0u : static_cast<uint32_t>(bs * elem), static_cast<uint32_t>(ss * elem)};
}
// The spaces of K's (or V's) rows and of their scales.
__device__ __forceinline__ RowSpace rows_of(const CacheArgs& c, bool v, int b, int hkv, int elem) {
  return v ? row_space(c, c.v, b, hkv, c.v_bs, c.v_ss, c.v_hs, elem) : row_space(c, c.k, b, hkv, c.k_bs, c.k_ss, c.k_hs, elem);
}
__device__ __forceinline__ RowSpace scales_of(const CacheArgs& c, bool v, int b, int hkv) {
  return v ? row_space(c, c.v_scales, b, hkv, c.vs_bs, c.vs_ss, c.vs_hs, 1)
           : row_space(c, c.k_scales, b, hkv, c.ks_bs, c.ks_ss, c.ks_hs, 1);
}

// The merge of partials and what they leave: (reference point, sum) of a row. A sum of zero means that no key
// was seen; a NaN stays one.
__device__ __forceinline__ f32pair point_and_sum(float ref, float l) {
  return f32pair{l == 0.f ? -INFINITY : ref, l};
}
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float ref, float l) { return l == 0.f ? -INFINITY : ref * kLn2 + logf(l); }

// This split's share of `tiles` key tiles.
struct TileRange {
  int begin, end;
};
__device__ __forceinline__ TileRange tile_range(const Item& item, int tiles) {
  return TileRange{static_cast<int>(static_cast<int64_t>(tiles) * item.split / item.splits),
                   static_cast<int>(static_cast<int64_t>(tiles) * (item.split + 1) / item.splits)};
}

}  // namespace
}  // namespace cached
}  // namespace fl

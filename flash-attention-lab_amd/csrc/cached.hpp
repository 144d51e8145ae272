// Pieces shared by the kernels of attention over a cache (cached_attn.hip: plan and merge; cached_narrow.hpp:
// sequences with few rows; cached_wide.hip: the others, and ragged batches of both): the rows of a sequence, the
// items of work that workgroups share out, and the offsets of cache rows.
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
// Tiles that starting and ending an item of a wide block costs as much as (about 7 us before the first tile is done
// and 2 us behind the last, at 2 us a tile of 16-bit keys at head_dim 128). 3 / 6 / 10, us: 8 sequences, 64/8 heads,
// 1,914 tokens, bf16 268-274 / 245-253 / 242-247; 24, 32/32 heads of 64, 5,975 tokens, bf16 394-401 / 376-382 / 379-381;
// 8, 16/16 heads of 64, 2,377 tokens, e4m3 102 / 97 / 100.
constexpr int kStartTiles = 6;
// From so many rounds of blocks on they run whole, as they come, the longest first: what the line evens out no
// longer pays for its partials. us with the merge, whole / line, bf16 if not said: 3.1 rounds (16 sequences, 64/8 heads
// of 128, 3,135 tokens on up to 8,000, e4m3) 663-681 / 685; 3.2 (12, 32/32 heads of 64, up to 700 tokens on 2,200)
// 103 / 108; 3.5 (16, 32/8 of 128) 180 / 184; 4.3 (24, 32/32 of 64, on up to 8,000) 355-360 / 361-381; 12.5 406-420 / 403.
constexpr int kWholeRounds = 3;
// Rows of a block.
__host__ __device__ __forceinline__ constexpr int block_rows(Kind kind) { return kind == kNarrow ? kNarrowRows : 256; }

namespace {

using cache::Sequence;
using decode::wave_inclusive_sum;

constexpr float kLn2 = 0.693147180559945309f;
// Running max before the first key: finite, so that a masked score (-inf) gives p = 0.
constexpr float kNoRef = -1e30f;

// The kernel's arguments (its only parameter), for the compiler to load again from here on: kept in scalar registers
// from the kernel's start, with what follows from them, a hundred and more were spilled.
__device__ __forceinline__ const CachedAttnArgs& reload_args() {
  typedef const CachedAttnArgs __attribute__((address_space(4))) ConstantArgs;
  ConstantArgs* p = (ConstantArgs*)(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return *(const CachedAttnArgs*)(p);
}

__device__ __forceinline__ int token_of_row(const CachedAttnArgs& a, int row) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(row)) * a.group_mul) >> a.group_shift);
}

__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_inclusive_sum(x), 63); }
// (The steps of wave_inclusive_sum: a tree of lane permutes through LDS took 0.25 us.)
__device__ __forceinline__ float wave_sum(float x) {
  auto step = [&](auto ctrl, auto rows) {
    const int from = __builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    x += __int_as_float(from);
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// n / c for 0 <= n < 2^31 - c and 1 <= c, by a reciprocal: the first quotient is off by at most 1 + n 2^-21 / c, so
// what it leaves is below c + n 2^-21 in magnitude, whose quotient brings it to one off. (The integer division is some
// forty instructions on the way to a workgroup's first load.)
struct Quotient {
  int c;
  float r;
  __device__ __forceinline__ explicit Quotient(int divisor)
      : c(divisor), r(__builtin_amdgcn_rcpf(static_cast<float>(divisor))) {}
  __device__ __forceinline__ int of(int n) const {
    auto left_of = [&](int q) { return static_cast<int>(static_cast<uint32_t>(n) - static_cast<uint32_t>(q) * c); };
    int q = static_cast<int>(static_cast<float>(n) * r);
    q += static_cast<int>(static_cast<float>(left_of(q)) * r);
    const int left = left_of(q);
    return q + (left >= c ? 1 : 0) - (left < 0 ? 1 : 0);
  }
  __device__ __forceinline__ int ceil_of(int n) const { return of(n + c - 1); }
};

// The sequences of a batch: lane l holds sequence 64 i + l of chunk i; chunks behind the first are read again
// in every pass.
struct Batch {
  const CachedAttnArgs* args;
  Sequence first;
  __device__ __forceinline__ explicit Batch(const CachedAttnArgs& a) { read(a); }
  __device__ __forceinline__ void read(const CachedAttnArgs& a) {
    args = &a;
    first = at(__lane_id());
  }
  __device__ __forceinline__ Sequence at(int b) const {
    Sequence s{0, 0, 0};
    if (b < args->c.batch) s = cache::sequence(args->c, b);
    return s;
  }
  __device__ __forceinline__ Sequence lane_of(int base) const { return base == 0 ? first : at(base + __lane_id()); }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    f(first);
    for (int base = 64; base < args->c.batch; base += 64) f(at(base + __lane_id()));
  }
  // Sequences that overlap (cu_seqlens does not ascend) could have more items than the grid and the
  // workspace are made for: no item is run then.
  __device__ __forceinline__ bool sound() const {
    if (args->c.cu_seqlens == nullptr) return true;
    bool back = false;
    for (int b = __lane_id(); b < args->c.batch; b += 64) back |= args->c.cu_seqlens[b + 1] < args->c.cu_seqlens[b];
    return !wave_any(back);
  }
};

// Blocks of rows of a sequence (none, if it is of the other kind), and its key tiles.
template <Kind kKind, int D>
__device__ __forceinline__ int blocks_of(const CachedAttnArgs& a, const Sequence& s) {
  const int rows = s.count * a.group;
  const bool mine = (rows <= kNarrowRows) == (kKind == kNarrow);
  return mine ? (rows + block_rows(kKind) - 1) / block_rows(kKind) : 0;
}
__device__ __forceinline__ int tiles_of(const Sequence& s) { return (s.len + kKeys - 1) / kKeys; }
// Key tiles that block i of a sequence sees any key of.
template <Kind kKind, int D>
__device__ __forceinline__ int block_tiles(const CachedAttnArgs& a, const Sequence& s, int i) {
  int end = s.len;
  if (a.causal) {
    const int rows = min((i + 1) * block_rows(kKind), s.count * a.group);
    end = max(min(end, token_of_row(a, max(rows - 1, 0)) + 1 + s.len - s.count), 0);
  }
  return (end + kKeys - 1) / kKeys;
}

// A workgroup's item: key tiles begin .. end - 1 of one block of rows of one KV head of one sequence. Not all
// of the block's: what it leaves are partials, in slot `slot`.
struct Item {
  int b, hkv, block, begin, end;
  bool partial;
  int slot;
  Sequence seq;
};

// The same values, for the compiler to keep in scalar registers.
__device__ __forceinline__ Item uniform(const Item& i) {
  auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return Item{u(i.b), u(i.hkv), u(i.block), u(i.begin), u(i.end), u(i.partial) != 0, u(i.slot),
              Sequence{u(i.seq.start), u(i.seq.count), u(i.seq.len)}};
}

// What the merge needs of a block whose first partial the workgroup leaves (cached_attn.hip): in the workgroup's own
// place of the list.
template <Kind kKind>
__device__ __forceinline__ void leave(const CachedAttnArgs& a, const Item& item, int splits) {
  if (threadIdx.x == 0 && static_cast<int>(blockIdx.x) < a.parts[kKind].merges)
    a.parts[kKind].merge_blocks[blockIdx.x] = MergeBlock{splits, item.slot, item.b, item.hkv, item.block, item.seq.start, item.seq.count, 0};
}

// No block whose partials start with this workgroup, until there is one. Every kernel does this first of all.
template <Kind kKind>
__device__ __forceinline__ void clear_list(const CachedAttnArgs& a) {
  if (threadIdx.x == 0 && static_cast<int>(blockIdx.x) < a.parts[kKind].merges)
    a.parts[kKind].merge_blocks[blockIdx.x].splits = 0;
}

// Items of equal shares: sequence b has blocks_b splits_b H_kv of them, with splits_b = ceil(tiles_b / share).
// The least share for which no more than `slots` items result (which run at once), 0 if there are more blocks.
template <Kind kKind, int D>
__device__ __forceinline__ int even_share(const CachedAttnArgs& a, const Batch& batch, int blocks, float work, int slots) {
  if (blocks > slots) return 0;
  auto items = [&](int t) {
    const Quotient by(t);
    int total = 0;
    batch.each([&](const Sequence& s) { total += blocks_of<kKind, D>(a, s) * max(by.ceil_of(tiles_of(s)), 1); });
    return a.c.heads_kv * wave_sum(total);
  };
  // sum of ceil(x / t) is at most work / t + blocks.
  int low = max(a.parts[kKind].min_tiles, static_cast<int>(work / slots));
  int high = blocks < slots ? max(low, static_cast<int>(work / (slots - blocks) * 1.001f) + 1) : 1 << 28;
  while (low < high) {
    const int mid = low + (high - low) / 2;
    if (items(mid) <= slots) {
      high = mid;
    } else {
      low = mid + 1;
    }
  }
  return items(low) <= slots ? low : 0;
}

// Item `id` of the equal shares (or of a.num_splits splits of every block; share 0: one each). Within a chunk
// of 64 sequences longer items come first with `sorted`, and within a sequence the blocks that see more keys.
// The partials of a block lie in consecutive slots.
template <Kind kKind, int D>
__device__ __forceinline__ bool find_item(const CachedAttnArgs& a, const Batch& batch, int id, int share, bool sorted,
                                          Item& item) {
  int before = 0;       // items of earlier chunks
  int before_slot = 0;  // slots of earlier chunks
  for (int base = 0; base < a.c.batch; base += 64) {
    const int lane = __lane_id();
    const Sequence s = batch.lane_of(base);
    const int tiles = tiles_of(s);
    const int splits = a.num_splits > 0 ? a.num_splits : share > 0 ? max(Quotient(share).ceil_of(tiles), 1) : 1;
    const int items = blocks_of<kKind, D>(a, s) * splits * a.c.heads_kv;
    const int slots = splits > 1 ? items : 0;
    const int all = wave_inclusive_sum(items);
    const int all_slots = wave_inclusive_sum(slots);
    int from = all - items;  // items and slots of the chunk before the lane's
    int from_slot = all_slots - slots;
    if (sorted) {
      const int length = Quotient(splits).of(tiles);
      from = from_slot = 0;
      const int here = min(a.c.batch - base, 64);
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
      const int n = of_owner(splits);
      const int at = of_owner(local);
      const int units = a.c.heads_kv * n;  // items of a block
      const int turn = Quotient(units).of(at);
      const int unit = at - turn * units;
      const Quotient by_splits(n);
      item.hkv = by_splits.of(unit);
      const int split = unit - item.hkv * n;
      item.block = Quotient(units).of(of_owner(items)) - 1 - turn;
      // The first `more` splits have one tile more than the others.
      const int all_tiles = block_tiles<kKind, D>(a, item.seq, item.block);
      const int each = by_splits.of(all_tiles);
      const int more = all_tiles - each * n;
      item.begin = each * split + min(split, more);
      item.end = item.begin + each + (split < more ? 1 : 0);
      item.partial = n > 1;
      item.slot = before_slot + of_owner(from_slot) + at;
      if (item.partial && split == 0) leave<kKind>(a, item, n);
      return true;
    }
    before += __builtin_amdgcn_readlane(all, 63);
    before_slot += __builtin_amdgcn_readlane(all_slots, 63);
  }
  return false;
}

// The line: the blocks of all sequences of a kind one after the other, a block as long as its tiles and what
// starting it costs, cut into equal chunks for the workgroups: all end together, and no more than two
// partials a workgroup result. A sequence's blocks go in pairs from its two ends, i and n - 1 - i, the one that
// sees more keys first: under a causal mask a pair's tiles are about the same for all i (the lighter block
// counts as what is missing to that), so that a position's block follows without a search.
template <Kind kKind, int D>
struct SequenceLine {
  int n, pairs, pair_tiles, pair_length, length;  // blocks, pairs, tiles and length of a pair, length of a KV head's line
  static constexpr int kStart = kStartTiles;
  __device__ __forceinline__ SequenceLine(const CachedAttnArgs& a, const Sequence& s) {
    n = blocks_of<kKind, D>(a, s);
    pairs = n / 2;
    pair_tiles = block_tiles<kKind, D>(a, s, n - 1) + block_tiles<kKind, D>(a, s, 0);
    pair_length = pair_tiles + 2 * kStart;
    length = pairs * pair_length + (n & 1 ? block_tiles<kKind, D>(a, s, pairs) + kStart : 0);
  }
  // A block's place: where it starts, and the tiles that it counts as.
  struct Span {
    int block, start, tiles;
  };
  __device__ __forceinline__ Span span_of(const CachedAttnArgs& a, const Sequence& s, int block) const {
    const bool light = block < pairs;
    const int heavy = block_tiles<kKind, D>(a, s, light ? n - 1 - block : block);
    if (light) return Span{block, block * pair_length + heavy + kStart, pair_tiles - heavy};
    return Span{block, (n - 1 - block) * pair_length, heavy};
  }
  __device__ __forceinline__ Span span_at(const CachedAttnArgs& a, const Sequence& s, int position) const {
    const int pair = min(Quotient(pair_length).of(position), pairs);
    const Span heavy = span_of(a, s, n - 1 - pair);
    return pair < pairs && position >= heavy.start + heavy.tiles + kStart ? span_of(a, s, pair) : heavy;
  }
};

// The segments that a workgroup runs, of one schedule or the other, which every workgroup derives from the
// lengths alike:
//  * equal shares, one item a workgroup, where the blocks are few and divide evenly enough;
//  * a chunk of the line;
//  * whole blocks as they come, where there are many rounds of them (or no workspace).
template <Kind kKind, int D>
struct Segments {
  enum { kShares, kLine, kWhole, kDone };
  int mode, share, chunk, position, end;
  __device__ __forceinline__ Segments(const CachedAttnArgs& a, const Batch& batch)
      : mode(kWhole), share(0), chunk(0), position(0), end(0) {
    int lane_blocks = 0;
    int lane_line = 0;
    float lane_work = 0.f;
    batch.each([&](const Sequence& s) {
      const int n = blocks_of<kKind, D>(a, s);
      lane_blocks += n;
      lane_work += static_cast<float>(n) * static_cast<float>(tiles_of(s));
      if (kKind == kWide && a.parts[kKind].line) lane_line += SequenceLine<kKind, D>(a, s).length;
    });
    const int blocks = a.c.heads_kv * wave_sum(lane_blocks);
    if (blocks == 0 || !batch.sound()) {
      mode = kDone;
      return;
    }
    if (a.num_splits > 0 || a.parts[kKind].slots == 0 || blocks > kWholeRounds * a.parts[kKind].slots) return;
    // (The grid is made for whole blocks too, which can be more; a workgroup that comes behind the slots starts
    // when another has ended, and has nothing to do unless blocks stay whole.)
    if (static_cast<int>(blockIdx.x) >= a.parts[kKind].slots && (a.parts[kKind].line || blocks <= a.parts[kKind].slots)) {
      mode = kDone;
      return;
    }
    const float work = a.c.heads_kv * wave_sum(lane_work);
    const int total = a.c.heads_kv * wave_sum(lane_line);
    chunk = max((total + a.parts[kKind].slots - 1) / a.parts[kKind].slots, a.parts[kKind].min_tiles + kStartTiles);
    share = even_share<kKind, D>(a, batch, blocks, work, a.parts[kKind].slots);
    // (A chunk's workgroup starts one more segment than its length counts, and leaves two partials: the line has
    // to gain more than that.)
    if (share > 0 && (!a.parts[kKind].line || share <= chunk + 2 * kStartTiles)) {
      mode = kShares;
    } else if (kKind == kWide && a.parts[kKind].line) {
      mode = kLine;
      position = min(static_cast<int>(blockIdx.x) * chunk, total);  // (the product is below total + chunk and a few)
      end = min(position + chunk, total);
      position = __builtin_amdgcn_readfirstlane(position);
      end = __builtin_amdgcn_readfirstlane(end);
      chunk = __builtin_amdgcn_readfirstlane(chunk);
    }
  }
  __device__ __forceinline__ bool more() const { return mode != kDone && (mode != kLine || position < end); }
  __device__ __forceinline__ bool next(const CachedAttnArgs& a, const Batch& batch, Item& item) {
    if (!more()) return false;
    if (kKind == kNarrow || mode != kLine) {
      const bool found = find_item<kKind, D>(a, batch, blockIdx.x, share, mode == kWhole, item);
      mode = kDone;
      return found;
    }
    while (position < end) {
      int before = 0;
      for (int base = 0; base < a.c.batch; base += 64) {
        const Sequence s = batch.lane_of(base);
        const int length = SequenceLine<kKind, D>(a, s).length * a.c.heads_kv;
        const int through = before + wave_inclusive_sum(length);
        const uint64_t mask = __builtin_amdgcn_ballot_w64(position < through);
        if (mask == 0) {
          before = __builtin_amdgcn_readlane(through, 63);
          continue;
        }
        const int owner = __builtin_ctzll(mask);
        auto of_owner = [&](int x) { return __builtin_amdgcn_readlane(x, owner); };
        item.b = base + owner;
        item.seq = Sequence{of_owner(s.start), of_owner(s.count), of_owner(s.len)};
        const int origin = of_owner(through) - of_owner(length);  // of the sequence
        const SequenceLine<kKind, D> line(a, item.seq);
        item.hkv = Quotient(line.length).of(position - origin);
        const int start = origin + item.hkv * line.length;  // of the KV head
        const auto span = line.span_at(a, item.seq, position - start);
        item.block = span.block;
        const int from = position - start - span.start;
        const int to = min(from + end - position, span.tiles);
        const int tiles = block_tiles<kKind, D>(a, item.seq, span.block);
        // (The last segment takes what the block has; a lighter block can count as a tile more or less.)
        item.begin = min(from, tiles);
        item.end = to == span.tiles ? tiles : min(to, tiles);
        item.partial = from > 0 || to < span.tiles;
        item.slot = 2 * static_cast<int>(blockIdx.x) + (from == 0 ? 1 : 0);
        const bool any = from == 0 || from < span.tiles;  // (not only what a start costs)
        if (item.partial && from == 0) {
          const int at = position;
          leave<kKind>(a, item, -(Quotient(chunk).of(at + span.tiles - 1) - static_cast<int>(blockIdx.x) + 1));
        }
        position = __builtin_amdgcn_readfirstlane(min(end, start + span.start + span.tiles + kStartTiles));
        if (any) return true;
        break;
      }
    }
    return false;
  }
};

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

// Four consecutive dims of row `key` of a sequence's K (or V), from the one that `at` bytes lead to.
template <typename Tag, bool kE4M3>
__device__ __forceinline__ f32x4 four_of(const CacheArgs& c, const RowSpace& rows, const RowSpace& scales,
                                         const cache::Place& p, int dim) {
  u32x2 x;
  if constexpr (kE4M3) {
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(rows.base + rows.offset(c, p) + dim);
    x = cache::values4<Tag>(codes, cache::scale_of(static_cast<uint8_t>(scales.base[scales.offset(c, p)])));
  } else {
    x = *reinterpret_cast<const u32x2*>(rows.base + rows.offset(c, p) + 2 * dim);
  }
  using E = Elem<Tag>;
  return f32x4{E::to_float(x.x & 0xffff), E::to_float(x.x >> 16), E::to_float(x.y & 0xffff), E::to_float(x.y >> 16)};
}

// A value that is not finite reaches the rows that do not see its key too, where they share a tile with rows that
// do: 0 times it is NaN. Rows of a causal call whose sum is not finite are therefore summed again, over their own
// keys alone: the sum over the item's keys of 2^(s - ref) v, by D / 4 lanes with four dims each. (Slow, a key at a
// time; reached only with such values in the cache.)
template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ f32x4 sum_again(const CachedAttnArgs& a, const Item& item, int row, float ref, int lane) {
  using E = Elem<Tag>;
  constexpr int kLanes = D / 4;
  constexpr int kElem = kE4M3 ? 1 : 2;
  const int dim = 4 * (lane % kLanes);
  const int token = token_of_row(a, row);
  const int head = item.hkv * a.group + row - token * a.group;
  const int64_t q_row = a.c.cu_seqlens ? (item.seq.start + token) * a.q_ss : item.b * a.q_bs + token * a.q_ss;
  const u32x2 q = *reinterpret_cast<const u32x2*>(a.q + q_row + head * a.q_hs + dim);
  const RowSpace k = rows_of(a.c, false, item.b, item.hkv, kElem), v = rows_of(a.c, true, item.b, item.hkv, kElem);
  const RowSpace ks = scales_of(a.c, false, item.b, item.hkv), vs = scales_of(a.c, true, item.b, item.hkv);
  const int end = min(min(item.end * kKeys, item.seq.len), item.seq.len - item.seq.count + token + 1);
  f32x4 o = {};
  for (int key = item.begin * kKeys; key < end; ++key) {
    const cache::Place p = cache::place(a.c, item.b, key);
    const f32x4 x = four_of<Tag, kE4M3>(a.c, k, ks, p, dim);
    float s = E::to_float(q.x & 0xffff) * x[0] + E::to_float(q.x >> 16) * x[1] + E::to_float(q.y & 0xffff) * x[2] +
              E::to_float(q.y >> 16) * x[3];
#pragma unroll
    for (int m = kLanes / 2; m >= 1; m /= 2) s += __shfl_xor(s, m);
    o += four_of<Tag, kE4M3>(a.c, v, vs, p, dim) * exp2_fast(fmaf(s, a.scale_log2, -ref));
  }
  return o;
}

}  // namespace
}  // namespace cached
}  // namespace fl

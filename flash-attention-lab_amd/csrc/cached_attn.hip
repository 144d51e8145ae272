// Attention of new tokens to the caches of their sequences (fl_cached_attention): a ragged batch whose
// sequences have any number of new tokens each, over slabs or a pool of blocks, in the tokens' type or in
// e4m3 codes with a power-of-two scale per row.
//
// For token i of sequence b, query head h, KV head h / group, with the n_b new tokens the last of the
// sequence's len_b:
//   s_j = scale q . k_j for j < len_b (causal: and j <= len_b - n_b + i),
//   o = sum_j softmax(s)_j v_j, lse = log sum_j e^(s_j); no such j: o = 0, lse = -inf.
// One pass over the keys with a running reference point and sum per row, on the lane layouts of
// prefill_tile.hpp (scores and outputs transposed, a lane per query row).
//
//  * The query heads of a KV head are packed: row r of a sequence is token r / group, head r % group. A
//    workgroup has 4 waves of 32 rows and streams key tiles of 64 through LDS, two slots each for K and V.
//  * Tiles go through registers: a thread loads 16-byte pieces of the tile after the next one and, an
//    iteration later, puts them into the other slot; codes become bf16 or fp16 on the way, pairs per
//    conversion instruction with the scale in it (exact in bf16). So the matrix cores see the tokens' type
//    whatever the cache holds, and a row's codes are converted once per workgroup.
//  * Lengths are known on the device only. Every workgroup derives the same list of items from them
//    (schedule, below) and takes the one of its own number; the grid is an upper bound from the sizes.
//    Where the blocks are fewer than the workgroups that the CUs hold, the keys of every sequence are cut
//    into equal splits, as many as still run at once; partials are merged by a second kernel in order.
#include <type_traits>

#include "cache.hpp"
#include "decode_sched.hpp"
#include "prefill_tile.hpp"

namespace fl {
namespace cached {
namespace {

using cache::Sequence;
using prefill::acc_key;
using prefill::k_lane_offset;
using prefill::kKeyBlockBytes;
using prefill::kKeyStepBytes;
using prefill::kMoveSlack;
using prefill::kTileElems;
using prefill::max_of;
using prefill::p_frag;
using prefill::tile_offset;
using prefill::v_frag_at;
using prefill::v_lane_offset;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;  // query rows of a block
constexpr int kKeys = 64;                  // keys of a tile
constexpr int kStartTiles = 4;             // tiles that starting and ending an item costs as much as
constexpr int kMaxRounds = 3;
constexpr float kLn2 = 0.693147180559945309f;
// Running max before the first key: finite, so that a masked score (-inf) gives p = 0.
constexpr float kNoRef = -1e30f;
constexpr int max(int a, int b) { return a > b ? a : b; }

__device__ __forceinline__ int token_of_row(const CachedAttnArgs& a, int row) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(row)) * a.group_mul) >> a.group_shift);
}

using decode::wave_inclusive_sum;

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

// Blocks of rows and key tiles of a sequence.
struct Load {
  int blocks, tiles;
};
__device__ __forceinline__ Load load_of(const CachedAttnArgs& a, const Sequence& s) {
  return Load{(s.count * a.group + kRows - 1) / kRows, (s.len + kKeys - 1) / kKeys};
}

// The items: sequence b has blocks_b splits_b H_kv of them, with splits_b = ceil(tiles_b / share). a.slots
// workgroups run at once, so items of up to `share` tiles that fill r rounds of slots end after about
// r (share + what starting an item costs): share and r are chosen for the least of that, with the least
// share for which no more than r slots items result. Within a chunk of 64 sequences longer items come
// first where there is more than one round, so that the last ones to start are short. Lane l holds sequence
// 64 i + l of chunk i; chunks behind the first are read again in every pass.
__device__ __forceinline__ bool find_item(const CachedAttnArgs& a, int id, Item& item) {
  const int lane = __lane_id();
  const int batch = a.c.batch;
  auto sequence_at = [&](int b) {
    Sequence s{0, 0, 0};
    if (b < batch) s = cache::sequence(a.c, b);
    return s;
  };
  const Sequence first = sequence_at(lane);
  const Load first_load = load_of(a, first);
  // f(blocks, tiles) summed over all sequences.
  auto sum = [&](auto f) {
    auto total = f(first_load);
    for (int base = 64; base < batch; base += 64) total += f(load_of(a, sequence_at(base + lane)));
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
    const Load l = load_of(a, s);
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

// o = 0 and lse = -inf in the rows of the call that belong to no sequence.
template <int D>
__device__ __forceinline__ void clear_unowned(const CachedAttnArgs& a) {
  if (a.c.cu_seqlens == nullptr) return;
  const int begin = min(max(a.c.cu_seqlens[0], 0), a.c.tokens);
  const int end = min(max(a.c.cu_seqlens[a.c.batch], begin), a.c.tokens);
  const int rows = begin + a.c.tokens - end;
  for (int i = blockIdx.x; i < rows; i += gridDim.x) {
    const int t = i < begin ? i : end + i - begin;
    for (int h = 0; h < a.heads; ++h) {
      if (threadIdx.x < D / 8)
        *reinterpret_cast<u32x4*>(a.o + t * a.o_ss + h * a.o_hs + 8 * threadIdx.x) = u32x4{0, 0, 0, 0};
      if (threadIdx.x == 0) a.lse[static_cast<int64_t>(t) * a.heads + h] = -INFINITY;
    }
  }
}

// Rows are moved in 16-byte pieces, kPerRow of them to a row.
template <int D, bool kE4M3>
struct Piece {
  static constexpr int kElem = kE4M3 ? 1 : 2;
  static constexpr int kElems = 16 / kElem;
  static constexpr int kPerRow = D / kElems;
};
// Where a tensor's rows lie: bytes, or scales. A row's offset is worked out by one lane for all that move
// its pieces (two 64-bit products, which the pieces' lanes would repeat).
struct RowSpace {
  int64_t outer_stride, row_stride;
  __device__ __forceinline__ int64_t offset(const CacheArgs& c, const cache::Place& p) const {
    return min(max(p.outer, 0), c.outer - 1) * outer_stride + p.row * row_stride;
  }
};

// A piece into a tile in LDS, as Tag's elements.
template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void put_piece(uint16_t* tile, int row, int col, const u32x4& piece, float scale) {
  if constexpr (kE4M3) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 lo = cache::values4<Tag>(piece[2 * h], scale);
      const u32x2 hi = cache::values4<Tag>(piece[2 * h + 1], scale);
      *reinterpret_cast<u32x4*>(tile + tile_offset<D>(row, col + 8 * h)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  } else {
    *reinterpret_cast<u32x4*>(tile + tile_offset<D>(row, col)) = piece;
  }
}

// The merge of partials and what they leave: (reference point, sum) of a row. A sum of zero means that no key
// was seen; a NaN stays one.
__device__ __forceinline__ f32pair point_and_sum(float ref, float l) {
  return f32pair{l == 0.f ? -INFINITY : ref, l};
}
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float ref, float l) { return l == 0.f ? -INFINITY : ref * kLn2 + logf(l); }

// An item with more than 32 rows in its block: a wave per 32 rows, all on the same tiles.
template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void wide_item(const CachedAttnArgs& a, const Item& item, uint16_t* smem) {
  using E = Elem<Tag>;
  constexpr int kTile = kTileElems<D>;
  // Two slots of K tiles, of V tiles, of rows' offsets (K, V) and of scales (K, V).
  int64_t* offsets = reinterpret_cast<int64_t*>(smem + 4 * kTile);
  float* scales = reinterpret_cast<float*>(offsets + 4 * kKeys);
  auto k_lds = [&](int slot) { return smem + slot * kTile; };
  auto v_lds = [&](int slot) { return smem + (2 + slot) * kTile; };

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;

  const Sequence& seq = item.seq;
  const int rows = seq.count * a.group;
  const int offset = seq.len - seq.count;  // position of the first new token
  const int row0 = item.block * kRows + wave * kWaveRows;
  const int my_row = row0 + (lane & 31);
  const int my_token = token_of_row(a, my_row);
  const int my_head = item.hkv * a.group + my_row - my_token * a.group;
  const bool mine = my_row < rows;

  // Keys of the block, and this split's tiles of them.
  int kv_end = seq.len;
  if (a.causal)
    kv_end = min(kv_end, token_of_row(a, min(item.block * kRows + kRows, rows) - 1) + 1 + offset);
  const int all_tiles = kv_end > 0 ? (kv_end + kKeys - 1) / kKeys : 0;
  const int t_begin = static_cast<int>(static_cast<int64_t>(all_tiles) * item.split / item.splits);
  const int t_end = static_cast<int>(static_cast<int64_t>(all_tiles) * (item.split + 1) / item.splits);

  const int64_t q_base = a.c.cu_seqlens ? seq.start * a.q_ss : item.b * a.q_bs;
  u32x4 qf[D / 16];
  {
    const uint16_t* src = a.q + q_base + (mine ? my_token : 0) * a.q_ss +
                          (mine ? my_head : item.hkv * a.group) * a.q_hs + 8 * half;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = mine ? load16(src + 16 * ks) : u32x4{0, 0, 0, 0};
  }

  int k_off[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) k_off[ks] = k_lane_offset<D>(ks, lane);
  int v_off[D / 32][2];
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) {
    v_off[nb][0] = v_lane_offset<D>(nb, 0, lane);
    v_off[nb][1] = v_lane_offset<D>(nb, 1, lane);
  }

  // Tile loads: piece j of a tensor's tile gives this thread 16 bytes of row load_row + j kRowStep. Lane l of
  // waves 0 to 3 works out where key l's K row, V row, K scale and V scale lie, and leaves the offset, or
  // the scale itself, in LDS.
  using P = Piece<D, kE4M3>;
  constexpr int kRowStep = kThreads / P::kPerRow;
  constexpr int kPieces = kKeys / kRowStep;
  const int load_row = tid / P::kPerRow;
  const int load_col = tid % P::kPerRow * P::kElems;
  const int last = seq.len - 1;  // rows behind it are not read: it takes their place in K, zeros in V
  const char* kp = a.c.k + (item.hkv * a.c.k_hs + load_col) * P::kElem;
  const char* vp = a.c.v + (item.hkv * a.c.v_hs + load_col) * P::kElem;
  const bool for_v = wave & 1;
  const bool for_scale = wave >> 1;
  const uint8_t* my_scales = for_v ? a.c.v_scales + item.hkv * a.c.vs_hs : a.c.k_scales + item.hkv * a.c.ks_hs;
  RowSpace space{(for_v ? a.c.v_bs : a.c.k_bs) * P::kElem, (for_v ? a.c.v_ss : a.c.k_ss) * P::kElem};
  if (kE4M3 && for_scale) space = for_v ? RowSpace{a.c.vs_bs, a.c.vs_ss} : RowSpace{a.c.ks_bs, a.c.ks_ss};
  struct Pieces {
    u32x4 k[kPieces], v[kPieces];
  };
  auto find = [&](int tile) { return cache::place(a.c, item.b, min(tile * kKeys + lane, last)); };
  // The offsets of a tile's rows into LDS; the scale waves ask for their bytes.
  auto locate = [&](int tile, const cache::Place& at, uint32_t& byte) {
    if (!for_scale) {
      offsets[((tile & 1) * 2 + wave) * kKeys + lane] = space.offset(a.c, at);
    } else if constexpr (kE4M3) {
      byte = my_scales[space.offset(a.c, at)];
    }
  };
  auto put_scales = [&](int tile, uint32_t byte) {
    if constexpr (kE4M3) {
      if (for_scale) scales[((tile & 1) * 2 + for_v) * kKeys + lane] = cache::scale_of(byte);
    }
  };
  auto load = [&](int tile, Pieces& r) {
    const int64_t* at = offsets + (tile & 1) * 2 * kKeys + load_row;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      r.k[j] = load16(kp + at[j * kRowStep]);
      r.v[j] = load16(vp + at[kKeys + j * kRowStep]);
    }
  };
  auto store = [&](int tile, Pieces& r) {
    if (tile * kKeys + kKeys - 1 > last) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        if (tile * kKeys + load_row + j * kRowStep > last) r.v[j] = u32x4{0, 0, 0, 0};
    }
    const float* sc = scales + (tile & 1) * 2 * kKeys + load_row;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int row = load_row + j * kRowStep;
      put_piece<Tag, D, kE4M3>(k_lds(tile & 1), row, load_col, r.k[j], kE4M3 ? sc[j * kRowStep] : 0.f);
      put_piece<Tag, D, kE4M3>(v_lds(tile & 1), row, load_col, r.v[j], kE4M3 ? sc[kKeys + j * kRowStep] : 0.f);
    }
  };

  f32x16 o[D / 32];
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) o[nb] = f32x16{};
  float ref = -INFINITY;  // reference point of o and l, log2 units; -inf until a key is seen
  float l = 0.f;
  const float sl2 = a.scale_log2;
  // Last key that this lane's row, the wave's first and the wave's last row see.
  const int last_key = a.causal ? min(last, my_token + offset) : last;
  const int first_limit = a.causal ? min(last, token_of_row(a, row0) + offset) : last;
  const int wave_limit = row0 >= rows ? -1 : a.causal ? min(last, token_of_row(a, row0 + kWaveRows - 1) + offset) : last;

  auto tile_step = [&](int t, int slot) {
    const int k0 = t * kKeys;
    if (k0 > wave_limit) return;
    const char* kt = reinterpret_cast<const char*>(k_lds(slot));
    const char* vt = reinterpret_cast<const char*>(v_lds(slot));
    f32x16 s0 = f32x16{};
    f32x16 s1 = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      s0 = E::mfma32(prefill::lds_load16(kt, k_off[ks]), qf[ks], s0);
      s1 = E::mfma32(prefill::lds_load16(kt + kKeyBlockBytes<D>, k_off[ks]), qf[ks], s1);
    }
    if (k0 + kKeys - 1 > first_limit) {
      const int lim = last_key - k0 - 4 * half;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int kj = acc_key(j, 0);
        if (kj > lim) s0[j] = -INFINITY;
        if (kj + 32 > lim) s1[j] = -INFINITY;
      }
    }
    // The reference point moves to the row's running max when that has grown by more than kMoveSlack over
    // it (prefill_tile.hpp).
    const float top = max_halves(max_of(s0, s1)) * sl2;
    const bool move = top > ref + kMoveSlack;
    if (wave_any(move)) {
      const float alpha = move ? exp2_fast(ref - top) : 1.f;  // ref = -inf gives 0
      ref = move ? top : ref;
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < D / 32; ++nb) o[nb] *= alpha;
    }
    const float shift = ref == -INFINITY ? 0.f : ref;
    float r0 = 0.f;
    float r1 = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s0[j] = exp2_fast(fmaf(s0[j], sl2, -shift));
      r0 += s0[j];
      s1[j] = exp2_fast(fmaf(s1[j], sl2, -shift));
      r1 += s1[j];
    }
    l += r0 + r1;
    const u32x4 pf[4] = {p_frag<Tag, 0>(s0), p_frag<Tag, 1>(s0), p_frag<Tag, 0>(s1), p_frag<Tag, 1>(s1)};
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
      for (int nb = 0; nb < D / 32; ++nb)
        o[nb] = E::mfma32(v_frag_at(vt + kk * kKeyStepBytes<D>, v_off[nb][0], v_off[nb][1]), pf[kk], o[nb]);
    }
  };

  if (t_begin < t_end) {
    // Iteration t multiplies tile t. Before it, tile t + 1's pieces go into the other slot, tile t + 2's are
    // asked for, tile t + 3's rows are located and tile t + 4's table entries are asked for; scales run one
    // iteration behind the offsets. Tiles past the end repeat the last row and are not used.
    Pieces in;
    uint32_t byte = 0;
    cache::Place at = find(t_begin);
    locate(t_begin, at, byte);
    put_scales(t_begin, byte);
    at = find(t_begin + 1);
    locate(t_begin + 1, at, byte);
    put_scales(t_begin + 1, byte);
    __syncthreads();
    load(t_begin, in);
    at = find(t_begin + 2);
    store(t_begin, in);
    load(t_begin + 1, in);
    __syncthreads();
    locate(t_begin + 2, at, byte);
    at = find(t_begin + 3);
    __syncthreads();
    for (int t = t_begin; t < t_end; ++t) {
      store(t + 1, in);
      load(t + 2, in);
      put_scales(t + 2, byte);
      locate(t + 3, at, byte);
      at = find(t + 4);
      tile_step(t, t & 1);
      __syncthreads();
    }
  }

  const float lt = sum_halves(l);
  if (item.splits > 1) {
    if (mine) {
      const int64_t slot_row = static_cast<int64_t>(item.slot) * kRows + wave * kWaveRows + (lane & 31);
      float* po = a.partial_o + slot_row * D + 4 * half;
#pragma unroll
      for (int nb = 0; nb < D / 32; ++nb) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(po + 32 * nb + 8 * g) =
              f32x4{o[nb][4 * g], o[nb][4 * g + 1], o[nb][4 * g + 2], o[nb][4 * g + 3]};
      }
      if (half == 0) a.partial_ml[slot_row] = point_and_sum(ref, lt);
    }
    return;
  }
  if (!mine) return;
  const float inv = inverse(lt);
  const int64_t o_base = a.c.cu_seqlens ? seq.start * a.o_ss : item.b * a.o_bs;
  uint16_t* orow = a.o + o_base + my_token * a.o_ss + my_head * a.o_hs;
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<u32x2*>(orow + 32 * nb + 8 * g + 4 * half) =
          u32x2{E::pack2(o[nb][4 * g] * inv, o[nb][4 * g + 1] * inv),
                E::pack2(o[nb][4 * g + 2] * inv, o[nb][4 * g + 3] * inv)};
  }
  if (half == 0)
    a.lse[(static_cast<int64_t>(seq.start) + my_token) * a.heads + my_head] =
        log_sum(ref, lt);
}

// An item with at most 32 rows (few tokens, or a decode step): bound by reading the cache, so the waves take
// tiles of 32 keys of their own, w, w + 4, .., in registers up to kAhead tiles early, through LDS that no
// other wave touches (no barriers), and their states are merged at the end.
#ifndef FL_NARROW_AHEAD
#define FL_NARROW_AHEAD 1
#endif
template <typename Tag, int D, bool kE4M3>
constexpr int kNarrowAhead = kE4M3 ? FL_NARROW_AHEAD : 1;
constexpr int kNarrowKeys = 32;
template <int D>
constexpr int kNarrowTileBytes = kNarrowKeys * D * 2;
template <int D>
constexpr int kRedPitch = D + 1;  // (conflict-free stores from the 32 columns)
template <int D>
constexpr int kRedBytes = 4 * kWaves * kWaveRows * (2 + kRedPitch<D>);

template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void narrow_item(const CachedAttnArgs& a, const Item& item, uint16_t* smem) {
  using E = Elem<Tag>;
  constexpr int kAhead = kNarrowAhead<Tag, D, kE4M3>;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int col = lane & 31;

  const Sequence& seq = item.seq;
  const int rows = seq.count * a.group;  // <= 32
  const int offset = seq.len - seq.count;
  const bool mine = col < rows;
  const int my_token = token_of_row(a, mine ? col : 0);
  const int my_head = item.hkv * a.group + (mine ? col : 0) - my_token * a.group;
  const int last = seq.len - 1;
  const int all_tiles = (seq.len + kKeys - 1) / kKeys;
  const int t_begin = static_cast<int>(static_cast<int64_t>(all_tiles) * item.split / item.splits);
  const int t_end = static_cast<int>(static_cast<int64_t>(all_tiles) * (item.split + 1) / item.splits);
  // In tiles of 32 keys.
  const int begin = 2 * t_begin + wave;
  const int end = min(2 * t_end, (seq.len + kNarrowKeys - 1) / kNarrowKeys);
  const int tiles = end > begin ? (end - begin + kWaves - 1) / kWaves : 0;

  const int64_t q_base = a.c.cu_seqlens ? seq.start * a.q_ss : item.b * a.q_bs;
  u32x4 qf[D / 16];
  {
    const uint16_t* src = a.q + q_base + my_token * a.q_ss + my_head * a.q_hs + 8 * half;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = mine ? load16(src + 16 * ks) : u32x4{0, 0, 0, 0};
  }

  // Lane l works out where the K row (lower half) or V row (upper half) of key l % 32 of a tile lies, and its
  // scale; piece j of a tensor's tile gives the lane 16 bytes of row load_row + j kRowStep.
  using P = Piece<D, kE4M3>;
  constexpr int kRowStep = 64 / P::kPerRow;
  constexpr int kPieces = kNarrowKeys / kRowStep;
  const int load_row = lane / P::kPerRow;
  const int load_col = lane % P::kPerRow * P::kElems;
  const char* kp = a.c.k + (item.hkv * a.c.k_hs + load_col) * P::kElem;
  const char* vp = a.c.v + (item.hkv * a.c.v_hs + load_col) * P::kElem;
  const RowSpace space{(half ? a.c.v_bs : a.c.k_bs) * P::kElem, (half ? a.c.v_ss : a.c.k_ss) * P::kElem};
  const RowSpace scale_space = half ? RowSpace{a.c.vs_bs, a.c.vs_ss} : RowSpace{a.c.ks_bs, a.c.ks_ss};
  const uint8_t* my_scales = half ? a.c.v_scales + item.hkv * a.c.vs_hs : a.c.k_scales + item.hkv * a.c.ks_hs;
  uint16_t* k_lds = smem + wave * kNarrowTileBytes<D>;  // (K and V: kNarrowTileBytes elements)
  uint16_t* v_lds = k_lds + kNarrowTileBytes<D> / 2;
  int64_t* offsets = reinterpret_cast<int64_t*>(smem + kWaves * kNarrowTileBytes<D>) + wave * 64;
  auto first_key = [&](int i) { return (begin + kWaves * i) * kNarrowKeys; };
  struct Pieces {
    u32x4 k[kPieces], v[kPieces];
    uint32_t scale;
  };
  auto find = [&](int i) { return cache::place(a.c, item.b, min(first_key(i) + col, last)); };
  auto load = [&](const cache::Place& p, Pieces& r) {
    offsets[lane] = space.offset(a.c, p);
    if constexpr (kE4M3) r.scale = my_scales[scale_space.offset(a.c, p)];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      r.k[j] = load16_stream(kp + offsets[load_row + j * kRowStep]);
      r.v[j] = load16_stream(vp + offsets[32 + load_row + j * kRowStep]);
    }
  };

  f32x16 o[D / 32];
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) o[nb] = f32x16{};
  float ref = kNoRef;
  float l = 0.f;
  const float sl2 = a.scale_log2;
  const int last_key = a.causal ? min(last, my_token + offset) : last;
  const int first_limit = a.causal ? min(last, offset) : last;  // of the first token

  cache::Place at;
  auto step = [&](int i, Pieces& r) __attribute__((always_inline)) {
    const int k0 = first_key(i);
    if (k0 + kNarrowKeys - 1 > last) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        if (k0 + load_row + j * kRowStep > last) r.v[j] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int row = load_row + j * kRowStep;
      const float ks = kE4M3 ? cache::scale_of(__shfl(static_cast<int>(r.scale), row)) : 0.f;
      const float vs = kE4M3 ? cache::scale_of(__shfl(static_cast<int>(r.scale), 32 + row)) : 0.f;
      put_piece<Tag, D, kE4M3>(k_lds, row, load_col, r.k[j], ks);
      put_piece<Tag, D, kE4M3>(v_lds, row, load_col, r.v[j], vs);
    }
    // (Unconditional, past the end on the last row: a load skipped on some path leaves the compiler unsure
    // how many are in flight, and it waits for all of them.)
    load(at, r);
    at = find(i + kAhead + 1);
    __builtin_amdgcn_sched_barrier(0);

    f32x16 s = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) s = E::mfma32(prefill::k_frag<D>(k_lds, 0, ks, lane), qf[ks], s);
    if (k0 + kNarrowKeys - 1 > first_limit) {
      const int lim = last_key - k0 - 4 * half;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (acc_key(j, 0) > lim) s[j] = -INFINITY;
      }
    }
    u32x4 vf[2][D / 32];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int nb = 0; nb < D / 32; ++nb) vf[kk][nb] = prefill::v_frag<D>(v_lds, nb, kk, lane);
    }
    const float top = max_halves(max_of(s)) * sl2;
    if (wave_any(top > ref)) {
      const float moved = fmaxf(ref, top);
      const float alpha = exp2_fast(ref - moved);  // 0 for a row's first key
      ref = moved;
#pragma unroll
      for (int nb = 0; nb < D / 32; ++nb) o[nb] *= alpha;
      l *= alpha;
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[j] = exp2_fast(fmaf(s[j], sl2, -ref));
      sum += s[j];
    }
    l += sum;
    const u32x4 p0 = p_frag<Tag, 0>(s);
    const u32x4 p1 = p_frag<Tag, 1>(s);
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb) {
      o[nb] = E::mfma32(vf[0][nb], p0, o[nb]);
      o[nb] = E::mfma32(vf[1][nb], p1, o[nb]);
    }
  };

  if (tiles > 0) {
    Pieces r[kAhead];
    at = find(0);
    static_for<0, kAhead>([&](auto t) __attribute__((always_inline)) {
      load(at, r[decltype(t)::value]);
      at = find(decltype(t)::value + 1);
    });
    int i = 0;
    for (; i + kAhead <= tiles; i += kAhead) {
      static_for<0, kAhead>([&](auto t) __attribute__((always_inline)) {
        step(i + decltype(t)::value, r[decltype(t)::value]);
      });
    }
    static_for<0, kAhead>([&](auto t) __attribute__((always_inline)) {
      if (i + decltype(t)::value < tiles) step(i + decltype(t)::value, r[decltype(t)::value]);
    });
  }

  // Merge the four waves in order; the tiles are free after the barrier.
  __syncthreads();
  f32pair* red_ml = reinterpret_cast<f32pair*>(smem);                       // [kWaves][32]
  float* red_o = reinterpret_cast<float*>(red_ml + kWaves * kWaveRows);     // [kWaves][32][kRedPitch]
  const float lt = sum_halves(l);
  if (mine) {
    if (half == 0) red_ml[wave * kWaveRows + col] = point_and_sum(ref, lt);
    float* row = red_o + (wave * kWaveRows + col) * kRedPitch<D>;
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb) {
#pragma unroll
      for (int j = 0; j < 16; ++j) row[32 * nb + acc_key(j, half)] = o[nb][j];
    }
  }
  __syncthreads();
  const int64_t o_base = a.c.cu_seqlens ? seq.start * a.o_ss : item.b * a.o_bs;
  for (int i = tid; i < rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4);
    const int d = i % (D / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, red_ml[w * kWaveRows + r].x);
    f32x4 num = {};
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const f32pair p = red_ml[w * kWaveRows + r];
      const float f = p.x == -INFINITY ? 0.f : exp2_fast(p.x - m);
      const float* row = red_o + (w * kWaveRows + r) * kRedPitch<D> + d;
      num += f32x4{row[0], row[1], row[2], row[3]} * f;
      den += p.y * f;
    }
    if (item.splits > 1) {
      const int64_t slot_row = static_cast<int64_t>(item.slot) * kRows + r;
      *reinterpret_cast<f32x4*>(a.partial_o + slot_row * D + d) = num;
      if (d == 0) a.partial_ml[slot_row] = f32pair{m, den};
      continue;
    }
    const float inv = inverse(den);
    const int token = token_of_row(a, r);
    const int head = item.hkv * a.group + r - token * a.group;
    *reinterpret_cast<u32x2*>(a.o + o_base + token * a.o_ss + head * a.o_hs + d) =
        u32x2{E::pack2(num[0] * inv, num[1] * inv), E::pack2(num[2] * inv, num[3] * inv)};
    if (d == 0) a.lse[(static_cast<int64_t>(seq.start) + token) * a.heads + head] = log_sum(m, den);
  }
}

// kNarrow, kWide: which kinds of items the call can have (both, where only the device knows).
template <typename Tag, int D, bool kE4M3, bool kNarrow, bool kWide>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
    cached_attn_kernel(const CachedAttnArgs a) {
  constexpr int kWideBytes = 4 * 2 * kTileElems<D> + 4 * kKeys * (8 + 4);
  constexpr int kNarrowBytes = max(kWaves * (2 * kNarrowTileBytes<D> + 64 * 8), kRedBytes<D>);
  constexpr int kBytes = max(kWide ? kWideBytes : 0, kNarrow ? kNarrowBytes : 0);
  __shared__ __attribute__((aligned(16))) uint16_t smem[kBytes / 2];
  clear_unowned<D>(a);
  Item item;
  if (!find_item(a, blockIdx.x, item)) return;
  if (item.first && threadIdx.x == 0 && a.sequence_splits != nullptr)
    a.sequence_splits[item.b] = int2{item.splits, item.first_slot};
  if (kNarrow && (!kWide || item.seq.count * a.group <= kWaveRows)) {
    narrow_item<Tag, D, kE4M3>(a, item, smem);
  } else if constexpr (kWide) {
    wide_item<Tag, D, kE4M3>(a, item, smem);
  }
}

// Merge pass: D / 4 lanes per row (token, head). With M = max_s m_s, o = sum_s o_s 2^(m_s - M) / sum_s l_s
// 2^(m_s - M), the splits in order. Splits in which a row sees no key (m = -inf) contribute nothing.
template <typename Tag, int D>
__global__ void __launch_bounds__(kThreads) cached_merge_kernel(const CachedAttnArgs a) {
  using E = Elem<Tag>;
  constexpr int kLanes = D / 4;
  const int64_t all = static_cast<int64_t>(a.c.tokens) * a.heads;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  const int64_t row = min(at, all - 1);
  const int token = static_cast<int>(row / a.heads);
  const int head = static_cast<int>(row - static_cast<int64_t>(token) * a.heads);
  const cache::Token t = cache::find_token<kLanes>(a.c, token);
  if (at >= all || t.b < 0) return;
  const int2 info = a.sequence_splits[t.b];
  const int n = info.x;
  if (n <= 1) return;
  const int hkv = head / a.group;
  const int r = t.index * a.group + head - hkv * a.group;
  const int blocks = (t.count * a.group + kRows - 1) / kRows;
  const int64_t slot = info.y + (static_cast<int64_t>(blocks - 1 - r / kRows) * a.c.heads_kv + hkv) * n;
  const int64_t first = slot * kRows + r % kRows;
  const f32pair* ml = a.partial_ml + first;
  const f32x4* po = reinterpret_cast<const f32x4*>(a.partial_o + first * D) + threadIdx.x % kLanes;
  float m = -INFINITY;
  for (int s = 0; s < n; ++s) m = fmaxf(m, ml[s * kRows].x);
  float l = 0.f;
  f32x4 o = {};
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const f32pair p = ml[s * kRows];
    const float f = p.x == -INFINITY ? 0.f : exp2_fast(p.x - m);
    l += p.y * f;
    o += po[static_cast<int64_t>(s) * (kRows * D / 4)] * f;
  }
  const float inv = inverse(l);
  const int64_t base = a.c.cu_seqlens ? token * a.o_ss : t.b * a.o_bs + t.index * a.o_ss;
  *reinterpret_cast<u32x2*>(a.o + base + head * a.o_hs + 4 * (threadIdx.x % kLanes)) =
      u32x2{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  if (threadIdx.x % kLanes == 0) a.lse[row] = log_sum(m, l);
}

template <typename Tag, int D, bool kE4M3>
void launch_kinds(const CachedAttnArgs& args, const CachedPlan& plan, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(plan.workgroups));
  if (!plan.wide) {
    hipLaunchKernelGGL((cached_attn_kernel<Tag, D, kE4M3, true, false>), grid, dim3(kThreads), 0, stream, args);
  } else if (!plan.narrow) {
    hipLaunchKernelGGL((cached_attn_kernel<Tag, D, kE4M3, false, true>), grid, dim3(kThreads), 0, stream, args);
  } else {
    hipLaunchKernelGGL((cached_attn_kernel<Tag, D, kE4M3, true, true>), grid, dim3(kThreads), 0, stream, args);
  }
}

template <typename Tag, int D>
hipError_t launch_typed(const CachedAttnArgs& args, const CachedPlan& plan, bool e4m3, hipStream_t stream) {
  if (e4m3) {
    launch_kinds<Tag, D, true>(args, plan, stream);
  } else {
    launch_kinds<Tag, D, false>(args, plan, stream);
  }
  if (hipError_t err = hipGetLastError()) return err;
  if (plan.partial_rows == 0) return hipSuccess;
  const int64_t lanes = static_cast<int64_t>(args.c.tokens) * args.heads * (D / 4);
  hipLaunchKernelGGL((cached_merge_kernel<Tag, D>), dim3(static_cast<uint32_t>((lanes + kThreads - 1) / kThreads)),
                     dim3(kThreads), 0, stream, args);
  return hipGetLastError();
}

}  // namespace
}  // namespace cached

CachedPlan plan_cached_attn(CachedAttnArgs& args, int head_dim, int cu_count) {
  using namespace cached;
  const int64_t cus = cu_count > 0 ? cu_count : 256;
  const CacheArgs& c = args.c;
  const int64_t rows = static_cast<int64_t>(c.tokens) * args.group;
  // Blocks that the lengths can lead to at least and at most.
  const int64_t per_seq = (static_cast<int64_t>(c.tokens_per_seq) * args.group + kRows - 1) / kRows;
  const int64_t least = (c.cu_seqlens ? (rows + kRows - 1) / kRows : per_seq * c.batch) * c.heads_kv;
  const int64_t most = (c.cu_seqlens ? rows / kRows + c.batch : per_seq * c.batch) * c.heads_kv;
  const int64_t tiles = (c.capacity + kKeys - 1) / kKeys;
  CachedPlan plan{};
  // Which kinds of items there can be: without cu_seqlens all sequences have the same rows.
  plan.narrow = c.cu_seqlens != nullptr || static_cast<int64_t>(c.tokens_per_seq) * args.group <= kWaveRows;
  plan.wide = c.cu_seqlens != nullptr ? rows > kWaveRows : !plan.narrow;
  plan.workgroups = most;
  args.min_tiles = plan.wide ? 4 : 2;
  args.slots = 0;
  args.max_rounds = 1;
  int64_t slots = 0;
  if (args.num_splits > 1) {
    plan.workgroups = slots = most * args.num_splits;
  } else if (args.num_splits == 0 && tiles > args.min_tiles && least < kMaxRounds * 2 * cus) {
    args.slots = static_cast<int>(2 * cus);
    // (With few blocks one round of splits is even enough.)
    args.max_rounds = 4 * most <= args.slots ? 1 : kMaxRounds;
    const int64_t splits = (tiles + args.min_tiles - 1) / args.min_tiles;
    const int64_t split_items = static_cast<int64_t>(args.max_rounds) * args.slots;
    slots = most * splits < split_items ? most * splits : split_items;
    plan.workgroups = slots > most ? slots : most;
  }
  plan.partial_rows = slots * kRows;
  if (slots > 0) plan.floats = plan.partial_rows * (head_dim + 2) + 2 * static_cast<int64_t>(c.batch);
  return plan;
}

hipError_t launch_cached_attn(const CachedAttnArgs& args, const CachedPlan& plan, DType dtype, bool e4m3,
                              int head_dim, hipStream_t stream) {
  using namespace cached;
  if (dtype == DType::bf16) {
    return head_dim == 64 ? launch_typed<bf16_tag, 64>(args, plan, e4m3, stream)
                          : launch_typed<bf16_tag, 128>(args, plan, e4m3, stream);
  }
  if (dtype == DType::f16) {
    return head_dim == 64 ? launch_typed<f16_tag, 64>(args, plan, e4m3, stream)
                          : launch_typed<f16_tag, 128>(args, plan, e4m3, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace fl

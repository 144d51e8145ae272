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
constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ int token_of_row(const CachedAttnArgs& a, int row) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(row)) * a.group_mul) >> a.group_shift);
}

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) x += __shfl_xor(x, m);
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m /= 2) x += __shfl_xor(x, m);
  return x;
}
__device__ __forceinline__ int wave_inclusive_sum(int x) {
  const int lane = __lane_id();
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const int y = __shfl_up(x, m);
    x += lane >= m ? y : 0;
  }
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

// The items, sequence after sequence: sequence b has blocks_b splits_b H_kv of them, and splits_b =
// ceil(tiles_b / share), with the least share of tiles for which no more than a.slots items result (1
// split each, where there are as many blocks). Lane l holds sequence 64 i + l of chunk i; chunks behind
// the first are read again in every pass.
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
  int share = 1 << 30;  // tiles of a split
  if (a.num_splits == 0 && a.slots > 0) {
    const int blocks = a.c.heads_kv * sum([](const Load& l) { return l.blocks; });
    if (blocks < a.slots) {
      const float work = a.c.heads_kv * sum([](const Load& l) { return float(l.blocks) * float(l.tiles); });
      auto items = [&](int t) {
        return a.c.heads_kv * sum([t](const Load& l) { return l.blocks * max((l.tiles + t - 1) / t, 1); });
      };
      // sum of ceil(x / t) is at most work / t + blocks.
      int low = max(a.min_tiles, static_cast<int>(work / a.slots));
      int high = max(low, static_cast<int>(work / (a.slots - blocks) * 1.001f) + 1);
      while (low < high) {
        const int mid = (low + high) / 2;
        if (items(mid) <= a.slots) {
          high = mid;
        } else {
          low = mid + 1;
        }
      }
      if (items(low) <= a.slots) share = low;
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
    const int through = wave_inclusive_sum(items);
    const int through_slot = wave_inclusive_sum(slots);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(before + through > id);
    if (mask) {
      const int owner = __builtin_ctzll(mask);
      auto of_owner = [&](int x) { return __builtin_amdgcn_readlane(x, owner); };
      item.b = base + owner;
      item.seq = Sequence{of_owner(s.start), of_owner(s.count), of_owner(s.len)};
      item.splits = of_owner(splits);
      const int local = id - (before + of_owner(through) - of_owner(items));
      const int units = a.c.heads_kv * item.splits;  // items of a block
      const int turn = local / units;                // blocks with more keys first
      const int unit = local - turn * units;
      item.hkv = unit / item.splits;
      item.split = unit - item.hkv * item.splits;
      item.block = of_owner(l.blocks) - 1 - turn;
      item.first_slot = before_slot + of_owner(through_slot) - of_owner(slots);
      item.slot = item.first_slot + local;
      item.first = local == 0;
      return true;
    }
    before += __builtin_amdgcn_readlane(through, 63);
    before_slot += __builtin_amdgcn_readlane(through_slot, 63);
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

template <typename Tag, int D, bool kE4M3>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
    cached_attn_kernel(const CachedAttnArgs a) {
  using E = Elem<Tag>;
  constexpr int kTile = kTileElems<D>;
  __shared__ __attribute__((aligned(16))) uint16_t k_lds[2][kTile];
  __shared__ __attribute__((aligned(16))) uint16_t v_lds[2][kTile];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;

  clear_unowned<D>(a);
  Item item;
  if (!find_item(a, blockIdx.x, item)) return;
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

  // Tile loads: piece j of a tensor's tile gives this thread 16 bytes of row load_row + j kRowStep.
  constexpr int kElem = kE4M3 ? 1 : 2;
  constexpr int kPieceElems = 16 / kElem;
  constexpr int kPiecesPerRow = D / kPieceElems;
  constexpr int kRowStep = kThreads / kPiecesPerRow;
  constexpr int kPieces = kKeys / kRowStep;
  const int load_row = tid / kPiecesPerRow;
  const int load_col = tid % kPiecesPerRow * kPieceElems;
  const char* kp = a.c.k + (item.hkv * a.c.k_hs + load_col) * kElem;
  const char* vp = a.c.v + (item.hkv * a.c.v_hs + load_col) * kElem;
  const uint8_t* ksp = kE4M3 ? a.c.k_scales + item.hkv * a.c.ks_hs : nullptr;
  const uint8_t* vsp = kE4M3 ? a.c.v_scales + item.hkv * a.c.vs_hs : nullptr;
  const int last = seq.len - 1;  // rows behind it are not read: they take its place, and are masked
  struct Places {
    cache::Place at[kPieces];
  };
  auto find = [&](int tile, Places& p) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      p.at[j] = cache::place(a.c, item.b, min(tile * kKeys + load_row + j * kRowStep, last));
  };
  struct Pieces {
    u32x4 k[kPieces], v[kPieces];
    uint8_t ks[kPieces], vs[kPieces];
  };
  auto load = [&](const Places& p, Pieces& r) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int64_t outer = min(max(p.at[j].outer, 0), a.c.outer - 1);
      const int64_t row = p.at[j].row;
      r.k[j] = load16(kp + (outer * a.c.k_bs + row * a.c.k_ss) * kElem);
      r.v[j] = load16(vp + (outer * a.c.v_bs + row * a.c.v_ss) * kElem);
      if constexpr (kE4M3) {
        r.ks[j] = ksp[outer * a.c.ks_bs + row * a.c.ks_ss];
        r.vs[j] = vsp[outer * a.c.vs_bs + row * a.c.vs_ss];
      }
    }
  };
  auto put = [&](uint16_t* tile, int row, const u32x4& piece, uint8_t byte) {
    if constexpr (kE4M3) {
      const float scale = cache::scale_of(byte);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x2 lo = cache::values4<Tag>(piece[2 * h], scale);
        const u32x2 hi = cache::values4<Tag>(piece[2 * h + 1], scale);
        *reinterpret_cast<u32x4*>(tile + tile_offset<D>(row, load_col + 8 * h)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    } else {
      *reinterpret_cast<u32x4*>(tile + tile_offset<D>(row, load_col)) = piece;
    }
  };
  auto store = [&](int slot, const Pieces& r) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      put(k_lds[slot], load_row + j * kRowStep, r.k[j], r.ks[j]);
      put(v_lds[slot], load_row + j * kRowStep, r.v[j], r.vs[j]);
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
    const char* kt = reinterpret_cast<const char*>(k_lds[slot]);
    const char* vt = reinterpret_cast<const char*>(v_lds[slot]);
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
    Places at;
    Pieces in;
    find(t_begin, at);
    load(at, in);
    find(t_begin + 1, at);
    store(t_begin & 1, in);
    load(at, in);
    find(t_begin + 2, at);
    __syncthreads();
    for (int t = t_begin; t < t_end; ++t) {
      store((t + 1) & 1, in);  // (tiles past the end repeat the last row and are not used)
      load(at, in);
      find(t + 3, at);
      tile_step(t, t & 1);
      __syncthreads();
    }
  }

  const float lt = sum_halves(l);
  if (item.splits > 1) {
    if (item.first && tid == 0) a.sequence_splits[item.b] = int2{item.splits, item.first_slot};
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
      if (half == 0) a.partial_ml[slot_row] = f32pair{lt > 0.f ? ref : -INFINITY, lt};
    }
    return;
  }
  if (item.first && tid == 0 && a.sequence_splits != nullptr) a.sequence_splits[item.b] = int2{1, 0};
  if (!mine) return;
  const float inv = lt > 0.f ? 1.f / lt : 0.f;
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
        lt > 0.f ? ref * kLn2 + logf(lt) : -INFINITY;
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
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int64_t base = a.c.cu_seqlens ? token * a.o_ss : t.b * a.o_bs + t.index * a.o_ss;
  *reinterpret_cast<u32x2*>(a.o + base + head * a.o_hs + 4 * (threadIdx.x % kLanes)) =
      u32x2{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  if (threadIdx.x % kLanes == 0) a.lse[row] = l > 0.f ? m * kLn2 + logf(l) : -INFINITY;
}

template <typename Tag, int D>
hipError_t launch_typed(const CachedAttnArgs& args, const CachedPlan& plan, bool e4m3, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(plan.workgroups));
  if (e4m3) {
    hipLaunchKernelGGL((cached_attn_kernel<Tag, D, true>), grid, dim3(kThreads), 0, stream, args);
  } else {
    hipLaunchKernelGGL((cached_attn_kernel<Tag, D, false>), grid, dim3(kThreads), 0, stream, args);
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
  args.min_tiles = 4;
  args.slots = 0;
  CachedPlan plan{most, 0, 0};
  int64_t slots = 0;
  if (args.num_splits > 1) {
    plan.workgroups = slots = most * args.num_splits;
  } else if (args.num_splits == 0 && tiles > args.min_tiles && least < 2 * cus) {
    args.slots = static_cast<int>(2 * cus);
    const int64_t splits = (tiles + args.min_tiles - 1) / args.min_tiles;
    slots = most * splits < args.slots ? most * splits : args.slots;
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

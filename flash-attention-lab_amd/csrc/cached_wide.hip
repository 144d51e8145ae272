// Attention over a cache for sequences with many rows (fl_cached_attention, cached.hpp): chunks of prompts.
// One pass over the keys with a running reference point and sum per row, on the lane layouts of
// prefill_tile.hpp (scores and outputs transposed, a lane per query row).
//
//  * The query heads of a KV head are packed: row r of a sequence is token r / group, head r % group. A
//    workgroup has 4 waves of 32 rows and streams key tiles of 64 through LDS, two slots each for K and V.
//  * Tiles go through registers: a thread loads 16-byte pieces of the tile after the next one and, an
//    iteration later, puts them into the other slot; codes become bf16 or fp16 on the way, pairs per
//    conversion instruction with the scale in it (exact in bf16). So the matrix cores see the tokens' type
//    whatever the cache holds, and a row's codes are converted once per workgroup.
#include "cached.hpp"
#include "prefill_pp.hpp"

namespace fl {
namespace cached {
namespace {

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
using prefill::pp::phase_barrier;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveRows = 32;
constexpr int kRows = block_rows(kWide, 64);
static_assert(kRows == kWaves * kWaveRows, "a wave per 32 rows");

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

template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void wide_item(const CachedAttnArgs& a, const Item& item, uint16_t* smem) {
  using E = Elem<Tag>;
  constexpr int kTile = kTileElems<D>;
  // Two slots of K tiles, of V tiles, of rows' offsets (K, V) and of scales (K, V).
  uint64_t* offsets = reinterpret_cast<uint64_t*>(smem + 4 * kTile);
  float* scales = reinterpret_cast<float*>(offsets + 4 * kKeys);
  auto k_lds = [&](int slot) { return smem + slot * kTile; };
  auto v_lds = [&](int slot) { return smem + (2 + slot) * kTile; };

  // (Opaque: what follows from it is worked out again for every item instead of being kept, which took 127 more
  // registers than there are.)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
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

  const int t_begin = item.begin;
  const int t_end = item.end;
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
  const bool for_v = wave & 1;
  const bool for_scale = wave >> 1;
  const RowSpace space = kE4M3 && for_scale ? scales_of(a.c, for_v, item.b, item.hkv)
                                            : rows_of(a.c, for_v, item.b, item.hkv, P::kElem);
  const char* kp = rows_of(a.c, false, item.b, item.hkv, P::kElem).base + load_col * P::kElem;
  const char* vp = rows_of(a.c, true, item.b, item.hkv, P::kElem).base + load_col * P::kElem;
  struct Pieces {
    u32x4 k[kPieces], v[kPieces];
  };
  auto find = [&](int tile) { return cache::place(a.c, item.b, min(tile * kKeys + lane, last)); };
  // The offsets of a tile's rows into LDS; the scale waves ask for their bytes.
  auto locate = [&](int tile, const cache::Place& at, uint32_t& byte) {
    if (!for_scale) {
      offsets[((tile & 1) * 2 + wave) * kKeys + lane] = space.offset(a.c, at);
    } else if constexpr (kE4M3) {
      byte = static_cast<uint8_t>(space.base[space.offset(a.c, at)]);
    }
  };
  auto put_scales = [&](int tile, uint32_t byte) {
    if constexpr (kE4M3) {
      if (for_scale) scales[((tile & 1) * 2 + for_v) * kKeys + lane] = cache::scale_of(byte);
    }
  };
  auto load = [&](int tile, Pieces& r) {
    const uint64_t* at = offsets + (tile & 1) * 2 * kKeys + load_row;
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
    // (K fragments two steps ahead of their MFMAs: prefill_fwd.hip)
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
    for (int ks = 0; ks < D / 16 - 2; ++ks) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
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
      phase_barrier();  // (the loads in flight need not have come back)
    }
  }

  const float lt = sum_halves(l);
  if (item.partial) {
    if (mine) {
      const int64_t slot_row = a.wide_partials + static_cast<int64_t>(item.slot) * kRows + wave * kWaveRows + (lane & 31);
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

template <typename Tag, int D, bool kE4M3>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
    cached_wide_kernel(const CachedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t smem[4 * kTileElems<D> + 4 * kKeys * (8 + 4) / 2];
  Segments<kWide, D> segments(a);
  Item item;
  while (segments.next(a, item)) {
    wide_item<Tag, D, kE4M3>(a, uniform(item), smem);
    __syncthreads();  // (the next item uses the LDS again)
  }
}

template <typename Tag, int D>
hipError_t launch_typed(const CachedAttnArgs& args, int64_t workgroups, bool e4m3, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(workgroups));
  if (e4m3) {
    hipLaunchKernelGGL((cached_wide_kernel<Tag, D, true>), grid, dim3(kThreads), 0, stream, args);
  } else {
    hipLaunchKernelGGL((cached_wide_kernel<Tag, D, false>), grid, dim3(kThreads), 0, stream, args);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace cached

hipError_t launch_cached_wide(const CachedAttnArgs& args, int64_t workgroups, DType dtype, bool e4m3, int head_dim,
                              hipStream_t stream) {
  using namespace cached;
  if (head_dim == 128) return launch_cached_pp(args, workgroups, dtype, e4m3, stream);
  return dtype == DType::bf16 ? launch_typed<bf16_tag, 64>(args, workgroups, e4m3, stream)
                              : launch_typed<f16_tag, 64>(args, workgroups, e4m3, stream);
}

}  // namespace fl

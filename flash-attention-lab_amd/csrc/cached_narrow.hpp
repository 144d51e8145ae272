// Attention over a cache for sequences with at most 48 rows (fl_cached_attention, cached.hpp): decode steps,
// drafted tokens, short turns. Such a call is bound by reading the cache: 2 x (D + 1) bytes a key and KV head
// in e4m3, against 4 D operations per row.
//
//  * A workgroup has one item, a key range of one KV head of one sequence. Its waves (4, or 8 where a CU holds
//    one workgroup) take tiles of 32 keys of their own, w, w + waves, .., loaded into registers a tile early; no
//    barriers until the waves' states are merged at the end.
//  * Products are on v_mfma_f32_16x16x32, 16 rows to a column block (kCols blocks): with 16 rows or fewer
//    (most decode steps) that is half the 32 x 32 form's work and registers, and four workgroups fit a CU
//    instead of two. Scores are transposed, S^T = K Q^T: lane l holds row l % 16 and keys 4 (l / 16) .. + 3
//    of each 16-key block, and the output O^T = V^T P^T, so softmax state and rescaling are per lane.
//  * Every load instruction of a wave covers whole rows: reading half of each row's 128 bytes per instruction
//    took 142 us for 8 sequences of 32K keys of 8 KV heads in e4m3, 173 with the streaming hint, whole rows 94-100
//    (5.5-5.8 TB/s). So both tensors go through LDS to get to the lanes that multiply them, 8 KiB of the wave's
//    own that holds K's tile, as it is in memory, and then V's (a wave's LDS operations keep their order).
//  * Latency bounds short caches (1 sequence of 640 keys, 9.4 us on eight waves, 10.5 on four) and the start of
//    all calls: 1.7 us for the schedule, 0.9 for the item, 1.8 to the first loads, 2.5 to their rows.
//  * K's A operand: lane (m, g) = (l % 16, l / 16) takes 16 bytes of every 64 of key m's row. The products
//    sum over dims in any order, and Q's fragments are read in the same one (step_dim).
//  * V^T's operand needs keys across, so V goes into LDS in the tokens' type and comes back by
//    ds_read_b64_tr_b16. P^T's operand element e of lane group g is key 4 g + e (e < 4) or 16 + 4 g + e - 4
//    of the tile, the ones the lane holds; V is read in that order.
//  * Codes become bf16 or fp16 in registers, with their scales (cache::values4).
#pragma once

#include "cached.hpp"
#include "prefill_pp.hpp"

namespace fl {
namespace cached {
namespace {

constexpr int kTileKeys = 32;

// Swizzles of the tiles' 16-byte chunks. K, whose rows have kPerRow of them: 16 lanes read one chunk of 16 rows,
// at 16 distinct places of the 16 that the banks hold.
template <int kPerRow>
__device__ __forceinline__ int k_offset(int row, int chunk) {  // bytes
  return 16 * (row * kPerRow + (chunk ^ ((row / (16 / kPerRow)) & (kPerRow - 1))));
}
// V: 32 lanes of a transpose read take an aligned pair of chunks of 8 rows (8 distinct pairs at D = 128, 4 of
// either half of the banks at 64).
template <int D>
__device__ __forceinline__ int v_swz(int row) {
  return D == 128 ? 2 * (row & 7) + ((row >> 3) & 1) : 2 * ((row >> 1) & 3) + ((row >> 3) & 1);
}
template <int D>
__device__ __forceinline__ int v_offset(int row, int chunk) {  // bytes
  return row * (2 * D) + 16 * (chunk ^ v_swz<D>(row));
}

// LDS of a workgroup: Q where it does not stay in registers, then each wave's tile and row offsets, in whose place
// the waves are merged afterwards, 16 rows of each at a time.
template <int D, int kCols, int kWaves>
struct NarrowLds {
  static constexpr bool kQ = kCols > 2;  // (48 rows' Q would take 48 registers)
  static constexpr int kTileBytes = kTileKeys * D * 2;
  static constexpr int kRedPitch = D + 4;  // floats
  static constexpr int kQBytes = kQ ? kCols * 16 * D * 2 : 0;
  static constexpr int kWaveBytes = kTileBytes + 64 * 8;
  static constexpr int kRedBytes = 16 * (8 + 4 * kRedPitch);  // of a wave
  static constexpr int kBytes = kQBytes + kWaves * (kRedBytes > kWaveBytes ? kRedBytes : kWaveBytes);
};

// First of the 8 dims that lane group g holds for step ks of K Q^T.
template <bool kE4M3>
__device__ __forceinline__ constexpr int step_dim(int ks, int g) {
  return kE4M3 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
}

template <typename Tag, int D, bool kE4M3, int kCols, int kWaves>
__device__ __forceinline__ void narrow_item(const CachedAttnArgs& a, const Item& item, char* smem) {
  using E = Elem<Tag>;
  using P = Piece<D, kE4M3>;
  using L = NarrowLds<D, kCols, kWaves>;
  constexpr int kSteps = D / 32;              // of K Q^T
  constexpr int kBlocks = D / 16;             // dim blocks of the output
  constexpr int kRowStep = 64 / P::kPerRow;   // rows of a load instruction
  constexpr int kPieces = kTileKeys / kRowStep;
  constexpr int kParts = P::kPerRow / 4;      // 16-byte parts of a K row in a lane
  // (Opaque: what follows from it is worked out here and not at the kernel's start, to be kept over other items.)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15;
  const int g = lane >> 4;
  const int half = lane >> 5;

  const Sequence& seq = item.seq;
  const int rows = seq.count * a.group;  // <= 16 kCols
  const int offset = seq.len - seq.count;
  const int last = seq.len - 1;
  // In tiles of 32 keys.
  const int begin = 2 * item.begin + wave;
  const int end = min(2 * item.end, (seq.len + kTileKeys - 1) / kTileKeys);
  const int tiles = end > begin ? (end - begin + kWaves - 1) / kWaves : 0;

  char* work = smem + L::kQBytes;
  char* tile = work + wave * L::kTileBytes;
  uint64_t* offsets = reinterpret_cast<uint64_t*>(work + kWaves * L::kTileBytes) + wave * 64;

  // Q^T, the B operand: lane (n, g) holds row 16 c + n, dims step_dim(ks, g) .. + 7.
  const int64_t q_base = a.c.cu_seqlens ? seq.start * a.q_ss : item.b * a.q_bs;
  auto load_q = [&](int c, int ks) {
    const int row = 16 * c + n;
    const bool in = row < rows;
    const int token = token_of_row(a, in ? row : 0);
    const int head = item.hkv * a.group + (in ? row : 0) - token * a.group;
    const u32x4 x = load16(a.q + q_base + token * a.q_ss + head * a.q_hs + step_dim<kE4M3>(ks, g));
    return in ? x : u32x4{0, 0, 0, 0};
  };
  // Lane l works out where the K row (lower half) or V row (upper half) of key l % 32 of a tile lies, and
  // loads its scale.
  const int load_row = lane / P::kPerRow;
  const int load_piece = lane % P::kPerRow;
  const RowSpace space = rows_of(a.c, half != 0, item.b, item.hkv, P::kElem);
  const RowSpace scale_space = scales_of(a.c, half != 0, item.b, item.hkv);
  const char* kp = rows_of(a.c, false, item.b, item.hkv, P::kElem).base + 16 * load_piece;
  const char* vp = rows_of(a.c, true, item.b, item.hkv, P::kElem).base + 16 * load_piece;
  auto first_key = [&](int i) { return (begin + kWaves * i) * kTileKeys; };
  auto find = [&](int i) { return cache::place(a.c, item.b, max(min(first_key(i) + (lane & 31), last), 0)); };
  u32x4 k[kPieces], v[kPieces];
  uint32_t byte = 0;
  auto load = [&](const cache::Place& p) __attribute__((always_inline)) {
    offsets[lane] = space.offset(a.c, p);
    if constexpr (kE4M3) byte = static_cast<uint8_t>(scale_space.base[scale_space.offset(a.c, p)]);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      k[j] = load16_stream(kp + offsets[load_row + j * kRowStep]);
      v[j] = load16_stream(vp + offsets[32 + load_row + j * kRowStep]);
    }
  };

  // The first tile's loads leave before Q is waited for. (They are made for any item, of no key too.)
  const cache::Place first = find(0);
  u32x4 qf[L::kQ ? 1 : kCols][kSteps];
  u32x4* q_lds = reinterpret_cast<u32x4*>(smem) + lane;  // [c][ks][64]
  constexpr int kFrags = kCols * kSteps;
  constexpr int kMine = (kFrags + kWaves - 1) / kWaves;  // that a wave brings into LDS
  auto my_frag = [&](int i) { return min(kMine * wave + i, kFrags - 1); };
  if constexpr (L::kQ) {
    u32x4 mine[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) mine[i] = load_q(my_frag(i) / kSteps, my_frag(i) % kSteps);
    load(first);
#pragma unroll
    for (int i = 0; i < kMine; ++i) q_lds[64 * my_frag(i)] = mine[i];
    prefill::pp::phase_barrier();
  } else {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) qf[c][ks] = load_q(c, ks);
    }
    load(first);
  }

  f32x4 o[kCols][kBlocks];
  float ref[kCols], l[kCols];
  int last_key[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) o[c][db] = f32x4{};
    ref[c] = kNoRef;
    l[c] = 0.f;
    last_key[c] = a.causal ? min(last, token_of_row(a, 16 * c + n) + offset) : last;
  }
  const float sl2 = a.scale_log2;
  const int first_limit = a.causal ? min(last, offset) : last;  // of the first token
  int v_get[kBlocks];
#pragma unroll
  for (int db = 0; db < kBlocks; ++db) v_get[db] = v_offset<D>(4 * g + (n >> 2), 2 * db + ((n >> 1) & 1)) + 8 * (n & 1);

  cache::Place at;
  auto step = [&](int i) __attribute__((always_inline)) {
    const int k0 = first_key(i);
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      *reinterpret_cast<u32x4*>(tile + k_offset<P::kPerRow>(load_row + j * kRowStep, load_piece)) = k[j];
    u32x4 kr[2][kParts];
    float k_scale[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int i = 0; i < kParts; ++i)
        kr[kb][i] = *reinterpret_cast<const u32x4*>(tile + k_offset<P::kPerRow>(16 * kb + n, 4 * i + g));
      k_scale[kb] = kE4M3 ? cache::scale_of(__shfl(static_cast<int>(byte), 16 * kb + n)) : 0.f;
    }
    // V rows behind the sequence's last one took its place: zeros, so that its values count once.
    if (k0 + kTileKeys - 1 > last) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        if (k0 + load_row + j * kRowStep > last) v[j] = u32x4{0, 0, 0, 0};
    }
    auto eight = [](const u32x4& x, int h, float scale) -> u32x4 {  // 8 codes as values
      const u32x2 lo = cache::values4<Tag>(x[2 * h], scale);
      const u32x2 hi = cache::values4<Tag>(x[2 * h + 1], scale);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int row = load_row + j * kRowStep;
      if constexpr (kE4M3) {
        const float scale = cache::scale_of(__shfl(static_cast<int>(byte), 32 + row));
        *reinterpret_cast<u32x4*>(tile + v_offset<D>(row, 2 * load_piece)) = eight(v[j], 0, scale);
        *reinterpret_cast<u32x4*>(tile + v_offset<D>(row, 2 * load_piece + 1)) = eight(v[j], 1, scale);
      } else {
        *reinterpret_cast<u32x4*>(tile + v_offset<D>(row, load_piece)) = v[j];
      }
    }
    f32x4 s[kCols][2];
#pragma unroll
    for (int c = 0; c < kCols; ++c) s[c][0] = s[c][1] = f32x4{};
    static_for<0, 2 * kSteps>([&](auto t) __attribute__((always_inline)) {
      constexpr int kb = decltype(t)::value % 2, ks = decltype(t)::value / 2;
      u32x4 kf;
      if constexpr (kE4M3) {
        kf = eight(kr[kb][ks / 2], ks % 2, k_scale[kb]);
      } else {
        kf = kr[kb][ks];
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        u32x4 q;
        if constexpr (L::kQ) {
          q = q_lds[64 * (c * kSteps + ks)];
        } else {
          q = qf[c][ks];
        }
        s[c][kb] = E::mfma16(kf, q, s[c][kb]);
      }
    });
    // (Unconditional, past the end on the last row: a load skipped on some path leaves the compiler unsure
    // how many are in flight, and it waits for all of them.)
    load(at);
    at = find(i + 2);
    __builtin_amdgcn_sched_barrier(0);
    if (k0 + kTileKeys - 1 > first_limit) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int lim = last_key[c] - k0 - 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r > lim) s[c][0][r] = -INFINITY;
          if (16 + r > lim) s[c][1][r] = -INFINITY;
        }
      }
    }
    u32x4 pf[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      float top = max2_f32(max3_f32(s[c][0][0], s[c][0][1], s[c][0][2]), max3_f32(s[c][0][3], s[c][1][0], s[c][1][1]));
      top = max_quarters(max3_f32(top, s[c][1][2], s[c][1][3])) * sl2;
      // The running max moves (and O and l are rescaled, a wave-uniform branch) only where some row's grows.
      if (wave_any(top > ref[c])) {
        const float moved = fmaxf(ref[c], top);
        const float alpha = exp2_fast(ref[c] - moved);  // 0 for a row's first key
        ref[c] = moved;
#pragma unroll
        for (int db = 0; db < kBlocks; ++db) o[c][db] *= alpha;
        l[c] *= alpha;
      }
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp2_fast(fmaf(s[c][e / 4][e % 4], sl2, -ref[c]));
        l[c] += p[e];
      }
      pf[c] = u32x4{E::pack2(p[0], p[1]), E::pack2(p[2], p[3]), E::pack2(p[4], p[5]), E::pack2(p[6], p[7])};
    }
#pragma unroll
    for (int db = 0; db < kBlocks; ++db) {
      const u32x2 lo = __builtin_bit_cast(u32x2, lds_read_tr16(tile + v_get[db]));
      const u32x2 hi = __builtin_bit_cast(u32x2, lds_read_tr16(tile + v_get[db] + 16 * 2 * D));
      const u32x4 vf{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[c][db] = E::mfma16(vf, pf[c], o[c][db]);
    }
  };

  at = find(1);
  for (int i = 0; i < tiles; ++i) step(i);

  // Merge the waves in order, 16 rows at a time.
  f32pair* red_ml = reinterpret_cast<f32pair*>(work);                // [kWaves][16]
  float* red_o = reinterpret_cast<float*>(red_ml + kWaves * 16);     // [kWaves][16][kRedPitch]
  const int64_t o_base = a.c.cu_seqlens ? seq.start * a.o_ss : item.b * a.o_bs;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    if (16 * c >= rows) break;
    __syncthreads();
    const float lt = sum_quarters(l[c]);
    if (g == 0) red_ml[wave * 16 + n] = point_and_sum(ref[c], lt);
#pragma unroll
    for (int db = 0; db < kBlocks; ++db)
      *reinterpret_cast<f32x4*>(red_o + (wave * 16 + n) * L::kRedPitch + 16 * db + 4 * g) = o[c][db];
    __syncthreads();
    const int here = min(rows - 16 * c, 16);
    for (int i = tid; i < here * (D / 4); i += 64 * kWaves) {
      const int r = i / (D / 4);
      const int d = i % (D / 4) * 4;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, red_ml[w * 16 + r].x);
      f32x4 num = {};
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f32pair x = red_ml[w * 16 + r];
        const float f = x.x == -INFINITY ? 0.f : exp2_fast(x.x - m);
        num += *reinterpret_cast<const f32x4*>(red_o + (w * 16 + r) * L::kRedPitch + d) * f;
        den += x.y * f;
      }
      const int row = 16 * c + r;
      if (a.causal && seq.count > 1 && den == den) {
        // (All D / 4 lanes of a row, or none.)
        const uint64_t bad = __builtin_amdgcn_ballot_w64((num[0] + num[1] + num[2] + num[3]) * 0.f != 0.f);
        if (bad >> (lane & ~(D / 4 - 1)) & ((uint64_t{1} << D / 4) - 1)) num = sum_again<Tag, D, kE4M3>(a, item, row, m, lane);
      }
      if (item.partial) {
        const int64_t slot_row = static_cast<int64_t>(item.slot) * kNarrowRows + row;
        *reinterpret_cast<f32x4*>(a.partial_o + slot_row * D + d) = num;
        if (d == 0) a.partial_ml[slot_row] = f32pair{m, den};
        continue;
      }
      const float inv = inverse(den);
      const int token = token_of_row(a, row);
      const int head = item.hkv * a.group + row - token * a.group;
      *reinterpret_cast<u32x2*>(a.o + o_base + token * a.o_ss + head * a.o_hs + d) =
          u32x2{E::pack2(num[0] * inv, num[1] * inv), E::pack2(num[2] * inv, num[3] * inv)};
      if (d == 0) a.lse[(static_cast<int64_t>(seq.start) + token) * a.heads + head] = log_sum(m, den);
    }
  }
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

}  // namespace
}  // namespace cached
}  // namespace fl

// Attention over a cache for sequences with many rows (fl_cached_attention, cached.hpp): chunks
// of prompts, bound by the matrix cores. The arithmetic, lane layouts and phases are those of the prefill
// kernel (prefill_pp.hip): 8 waves of 32 rows, two to a SIMD in two groups that take turns, one group's
// MFMAs running beside the other's softmax, one barrier per tile of 64 keys. What differs is where keys
// come from and how the work is found:
//
//  * Rows may lie anywhere (a pool's blocks of any size). Group 0 moves K, group 1 V, 16 rows a wave, in its
//    MFMA phase, between the MFMAs: one lane works out a row's address, the lanes that move its 16-byte
//    pieces get it by a lane permute. Rows in the tokens' type go straight into LDS, asked for two (V) or three (K)
//    tiles ahead; codes go into LDS three tiles ahead as they are, and a period before their use become
//    the tokens' type (a pair per instruction, scale included), once per workgroup.
//  * A workgroup's items are shares of blocks' tiles (cached.hpp), with the rows of all query heads of
//    a KV head.
//
// A period (a tile of 64 keys against 256 rows at head_dim 128) takes about 3,900 cycles in 16 bits and 4,640 in e4m3,
// of them 2,048 of MFMAs: the rate of the prefill kernel in 16 bits, and the codes' conversion and second way through
// LDS on top. (1 sequence, 2,048 new of 16,384 tokens, 32/8 heads, e4m3 pool: 485-575 us by box, 897-1,060 TFLOP/s; the
// clock settles at 1.85-2.2 GHz under this load.) Short calls are bound by starts: 3 us of schedule, 2 of tables and
// query rows, 2 until the first tile, 2 for the rows' way out.
#include "cached_narrow.hpp"

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

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;
static_assert(kRows == block_rows(kWide), "a wave per 32 rows");
// LDS slots for K and for V: in period m the tiles m - 1 (V), m and m + 1, and in the tokens' type one more that
// loads bring in (codes arrive in a place of their own, where they are three tiles).
template <bool kE4M3>
constexpr int kStagesOf = kE4M3 ? 3 : 4;
constexpr int kAhead = 2;        // fragments read ahead of their MFMAs
constexpr int kTableEntries = 2048;  // of the block table that an item keeps in LDS

// LDS: the K ring, the V ring, each wave's codes of three tiles and their scales, and the item's part of the
// block table.
template <int D, bool kE4M3>
struct Lds {
  static constexpr int kSlotBytes = 2 * kTileElems<D>;
  static constexpr int kRingBytes = kStagesOf<kE4M3> * kSlotBytes;
  static constexpr int kCodeBytes = 16 * D;    // a wave's rows of a tile, as codes
  static constexpr int kScaleBytes = 64 * 4;
  static constexpr int kCodes = 2 * kRingBytes;
  static constexpr int kScales = kCodes + (kE4M3 ? kWaves * 3 * kCodeBytes : 0);
  static constexpr int kTable = kScales + (kE4M3 ? kWaves * 3 * kScaleBytes : 0);
  static constexpr int kBytes = kTable + 4 * kTableEntries;
};
static_assert(Lds<128, true>::kBytes <= 160 * 1024 && Lds<128, false>::kBytes <= 160 * 1024, "a CU's LDS");

// What V's rows behind a sequence's last one are read as.
__device__ const u32x4 zero_row[16] = {};

template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void pp_item(const CachedAttnArgs& a, const Item& item, char* smem) {
  using E = Elem<Tag>;
  using P = Piece<D, kE4M3>;
  using L = Lds<D, kE4M3>;
  constexpr int kStages = kStagesOf<kE4M3>;
  constexpr int kSlotBytes = L::kSlotBytes;
  constexpr int kVRingBytes = L::kRingBytes;
  const char* lds_bytes = smem;

  // (Opaque: what follows from it is worked out again for every item instead of being kept, which took 127 more
  // registers than there are.)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = wave >> 2;
  const int half = lane >> 5;

  const Sequence& seq = item.seq;
  const int rows = seq.count * a.group;
  const int q0 = item.block * kRows;
  const int row0 = q0 + wave * kWaveRows;
  const int my_row = row0 + (lane & 31);
  const int last = seq.len - 1;

  // Keys and positions count from the item's first tile.
  const int num_tiles = item.end - item.begin;
  const int key0 = item.begin * kKeys;
  const int offset = seq.len - seq.count - key0;
  const int seqlen_k = seq.len - key0;
  // Tiles this wave sees any key of, and the first whose scores need masking.
  int my_tiles = num_tiles;
  int mask_from = seqlen_k / kKeys;
  if (a.causal) {
    const int end = token_of_row(a, row0 + kWaveRows - 1) + offset;
    my_tiles = end < 0 ? 0 : min(num_tiles, end / kKeys + 1);
    const int x = token_of_row(a, row0) + offset - (kKeys - 1);
    mask_from = min(mask_from, x < 0 ? 0 : x / kKeys + 1);
  }
  if (row0 >= rows) my_tiles = 0;
  const int last_key = a.causal ? min(seqlen_k - 1, token_of_row(a, my_row) + offset) : seqlen_k - 1;

  u32x4 qf[D / 16];
  {
    const bool in = my_row < rows;
    const int token = token_of_row(a, in ? my_row : 0);
    const int head = item.hkv * a.group + (in ? my_row : 0) - token * a.group;
    const uint16_t* src = a.q + (a.c.cu_seqlens ? seq.start * a.q_ss : item.b * a.q_bs) + token * a.q_ss +
                          head * a.q_hs + 8 * half;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = in ? load16(src + 16 * ks) : u32x4{0, 0, 0, 0};
  }

  int k_lds[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) k_lds[ks] = k_lane_offset<D>(ks, lane);
  // (V offsets are biased by the K ring's size, so that every slot is an immediate.)
  int v_lds[D / 32][2];
  int v_bias = kVRingBytes;
  asm volatile("" : "+v"(v_bias));
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) {
    v_lds[nb][0] = v_lane_offset<D>(nb, 0, lane) + v_bias;
    v_lds[nb][1] = v_lane_offset<D>(nb, 1, lane) + v_bias;
  }

  // The blocks that hold the item's keys, as the table has them (kept in LDS while they fit; a load here would
  // wait for all tile loads before it).
  const bool paged = a.c.block_tables != nullptr;
  const int32_t* table_row = a.c.block_tables + item.b * a.c.block_tables_stride;
  int* table = reinterpret_cast<int*>(smem + L::kTable);
  auto block_of = [&](int key) { return a.c.page_shift >= 0 ? key >> a.c.page_shift : key / a.c.rows; };
  int first_block = 0;
  bool in_lds = false;
  if (paged && num_tiles > 0) {
    first_block = block_of(key0);
    const int blocks = block_of(min(item.end * kKeys - 1, last)) - first_block + 1;
    in_lds = blocks <= kTableEntries;
    if (in_lds) {
      for (int i = tid; i < blocks; i += kThreads) table[i] = table_row[first_block + i];
    }
    __syncthreads();
  }

  // This wave's 16 rows of its group's tensor in every tile: lane l works out where row l % 16 lies, and
  // piece j of the lane is 16 bytes of row kRowStep j + l / kPerRow.
  constexpr int kRowStep = 64 / P::kPerRow;
  constexpr int kPieces = 16 / kRowStep;
  constexpr int kLoads = kPieces + (kE4M3 ? 1 : 0);  // of a tile and wave
  const int tile_row0 = 16 * (wave & 3);
  const int piece_row = lane / P::kPerRow;
  const int piece = lane % P::kPerRow;
  const bool for_v = group == 1;
  const RowSpace space = rows_of(a.c, for_v, item.b, item.hkv, P::kElem);
  const RowSpace scale_space = scales_of(a.c, for_v, item.b, item.hkv);
  const int ring = for_v ? kVRingBytes : 0;
  // Tile t's pieces go into its ring slot, codes and their scales into places of the wave's own.
  const int my_codes = L::kCodes + wave * 3 * L::kCodeBytes;
  const int my_scales = L::kScales + wave * 3 * L::kScaleBytes;
  const uint32_t lds_base = lds_address(smem);
  uint64_t row_at = 0;  // address of the lane's row of the tile being asked for
  // Rows behind the sequence's last one are not read: it takes their place in K, zeros in V.
  auto locate = [&](int t, int slot) {
    const int at_key = key0 + t * kKeys + tile_row0 + (lane & 15);
    const int key = min(at_key, last);
    cache::Place at{0, key};
    if (paged) {
      const int block = block_of(key);
      // (Past the item's last tile the entry is not used; it is kept within the table's place.)
      at.outer = in_lds ? table[min(block - first_block, kTableEntries - 1)] : table_row[block];
      at.row = cache::row_in_block(a.c, key);
    }
    row_at = reinterpret_cast<uint64_t>(space.base) + space.offset(a.c, at);
    if constexpr (kE4M3)
      global_load_u8_to_lds_asm(scale_space.base + scale_space.offset(a.c, at),
                                lds_base + my_scales + (static_cast<unsigned>(slot) % 3) * L::kScaleBytes);
    if (for_v && at_key > last) row_at = reinterpret_cast<uint64_t>(zero_row);
  };
  auto ask = [&](int slot, int j) {
    const int from = kRowStep * j + piece_row;
    const uint32_t lo = __shfl(static_cast<int>(row_at), from);
    const uint32_t hi = __shfl(static_cast<int>(row_at >> 32), from);
    // (LDS chunk `piece` of a row of 16-bit elements holds the row's chunk piece ^ swz.)
    const int chunk = kE4M3 ? piece : piece ^ prefill::swz<D>(tile_row0 + from);
    const uint32_t to = kE4M3 ? my_codes + (static_cast<unsigned>(slot) % 3) * L::kCodeBytes
                              : ring + tile_row0 * 2 * D + (static_cast<unsigned>(slot) % kStages) * kSlotBytes;
    global_load16_to_lds_asm(reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo) + 16 * chunk,
                             lds_base + to + 1024 * j);
  };
  // Codes: a piece of a tile's, with its row's scale, becomes two 16-byte stores.
  constexpr int kPuts = kE4M3 ? 2 * kPieces : 0;
  u32x4 code{};
  float scale = 0.f;
  auto take = [&](int slot, int j) {
    const unsigned s = static_cast<unsigned>(slot) % 3;
    code = *reinterpret_cast<const u32x4*>(smem + my_codes + s * L::kCodeBytes + 1024 * j + 16 * lane);
    scale = cache::scale_of(
        *reinterpret_cast<const uint32_t*>(smem + my_scales + s * L::kScaleBytes + 4 * (kRowStep * j + piece_row)));
  };
  auto put = [&](int slot, int i) {
    const int row = tile_row0 + kRowStep * (i / 2) + piece_row;
    uint16_t* tile = reinterpret_cast<uint16_t*>(smem + ring + (static_cast<unsigned>(slot) % kStages) * kSlotBytes);
    const u32x2 lo = cache::values4<Tag>(code[2 * (i % 2)], scale);
    const u32x2 hi = cache::values4<Tag>(code[2 * (i % 2) + 1], scale);
    *reinterpret_cast<u32x4*>(tile + tile_offset<D>(row, 16 * piece + 8 * (i % 2))) = u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  f32x16 o[D / 32];
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) o[nb] = f32x16{};
  f32x16 s0 = f32x16{};
  f32x16 s1 = f32x16{};
  u32x4 pf[4] = {};
  float ref = kNoRef;
  float l = 0.f;
  const float sl2 = a.scale_log2;

  // The MFMA phase of a period (prefill_pp.hip): P V of the tile before, K Q^T of this one, 12 P V steps
  // first, the row max of the new scores between the last 4.
  constexpr int kPv = 4 * (D / 32);
  constexpr int kQk = 2 * (D / 16);
  constexpr int kSteps = kPv + kQk;
  constexpr int kTail = 4;
  constexpr int kLeadPv = kPv - kTail;
  auto step_at = [](auto n_tag, auto full_tag) constexpr {
    constexpr int n = decltype(n_tag)::value;
    if constexpr (!decltype(full_tag)::value) {
      return n;
    } else {
      return n < kLeadPv ? n : n < kLeadPv + kQk ? kPv + (n - kLeadPv) : n - kQk;
    }
  };
  auto read_frag = [&](int slot, auto i_tag) -> u32x4 {
    constexpr int i = decltype(i_tag)::value;
    if constexpr (i < kPv) {
      constexpr int kk = i / (D / 32), nb = i % (D / 32);
      const char* vt = lds_bytes + (static_cast<unsigned>(slot + kStages - 1) % kStages) * kSlotBytes;
      return v_frag_at(vt + kk * kKeyStepBytes<D>, v_lds[nb][0], v_lds[nb][1]);
    } else {
      constexpr int j = i - kPv, ks = j / 2, blk = j % 2;
      const char* kt = lds_bytes + (static_cast<unsigned>(slot) % kStages) * kSlotBytes;
      return prefill::lds_load16(kt + blk * kKeyBlockBytes<D>, k_lds[ks]);
    }
  };
  u32x4 pre[kAhead];
  auto prefetch = [&](int slot) {
    static_for<0, kAhead>([&](auto i) { pre[decltype(i)::value] = read_frag(slot, i); });
  };
  auto prefetch_qk = [&](int slot) {
    static_for<0, kAhead>([&](auto i) {
      pre[decltype(i)::value] = read_frag(slot, std::integral_constant<int, kPv + decltype(i)::value>{});
    });
  };
  float tile_mx = kNoRef;
  float mx_t[10], mx_u[4], mx_w = 0.f;
  auto max_op = [&](auto k_tag) {
    constexpr int k = decltype(k_tag)::value;
    if constexpr (k < 5) {
      mx_t[k] = max3_f32(s0[3 * k], s0[3 * k + 1], s0[3 * k + 2]);
    } else if constexpr (k < 10) {
      mx_t[k] = max3_f32(s1[3 * (k - 5)], s1[3 * (k - 5) + 1], s1[3 * (k - 5) + 2]);
    } else if constexpr (k < 13) {
      mx_u[k - 10] = max3_f32(mx_t[3 * (k - 10)], mx_t[3 * (k - 10) + 1], mx_t[3 * (k - 10) + 2]);
    } else if constexpr (k == 13) {
      mx_u[3] = max3_f32(mx_t[9], s0[15], s1[15]);
    } else if constexpr (k == 14) {
      mx_w = max3_f32(mx_u[0], mx_u[1], mx_u[2]);
    } else if constexpr (k == 15) {
      mx_w = max2_f32(mx_w, mx_u[3]);
    } else if constexpr (k == 16) {
      mx_w = max_halves(mx_w);
    } else {
      tile_mx = mx_w * sl2;
    }
  };
  constexpr int kMaxOps = 18;
  auto mfma_phase = [&](int slot, auto pv_tag, auto qk_tag, auto&& hook) {
    constexpr bool kDoPv = decltype(pv_tag)::value;
    constexpr bool kDoQk = decltype(qk_tag)::value;
    constexpr bool kFull = kDoPv && kDoQk;
    constexpr int kFirstLive = kDoPv ? 0 : kPv;
    constexpr int kEndLive = kDoQk ? kSteps : kPv;
    u32x4 fr[kSteps];
    static_for<0, kAhead>([&](auto i) {
      constexpr int n = kFirstLive + decltype(i)::value;
      fr[step_at(std::integral_constant<int, n>{}, std::bool_constant<kFull>{})] = pre[decltype(i)::value];
    });
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
    static_for<0, kSteps>([&](auto n_tag) {
      constexpr int n = decltype(n_tag)::value;
      constexpr int i = step_at(n_tag, std::bool_constant<kFull>{});
      if constexpr (n >= kFirstLive && n < kEndLive) {
        if constexpr (i < kPv) {
          constexpr int kk = i / (D / 32), nb = i % (D / 32);
          o[nb] = E::mfma32(fr[i], pf[kk], o[nb]);
        } else {
          constexpr int j = i - kPv, ks = j / 2, blk = j % 2;
          f32x16& acc = blk == 0 ? s0 : s1;
          acc = E::mfma32(fr[i], qf[ks], ks == 0 ? f32x16{} : acc);
        }
      }
      constexpr int nx = n + kAhead;
      if constexpr (nx >= kFirstLive + kAhead && nx < kEndLive) {
        constexpr int ix = step_at(std::integral_constant<int, nx>{}, std::bool_constant<kFull>{});
        fr[ix] = read_frag(slot, std::integral_constant<int, ix>{});
      }
      hook(n_tag);
      if constexpr (kFull && n >= kLeadPv + kQk) {
        constexpr int k = n - (kLeadPv + kQk);
        static_for<k * kMaxOps / kTail, (k + 1) * kMaxOps / kTail>([&](auto op) { max_op(op); });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
    if constexpr (kDoQk && !kDoPv) static_for<0, kMaxOps>([&](auto op) { max_op(op); });
  };

  auto softmax_phase = [&](int t) {
    float mx = tile_mx;
    if (t >= mask_from) {
      asm volatile("" ::: "memory");
      const int lim = last_key - t * kKeys - 4 * half;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int kj = acc_key(j, 0);
        s0[j] = kj > lim ? -INFINITY : s0[j];
        s1[j] = kj + 32 > lim ? -INFINITY : s1[j];
        __builtin_amdgcn_sched_barrier(0);  // (one compare and one select at a time: prefill_pp.hip)
      }
      mx = max_halves(max_of(s0, s1)) * sl2;
    }
    if (wave_any(mx > ref + kMoveSlack)) {
      asm volatile("" ::: "memory");
      const float moved = max2_f32(ref, mx);
      const float alpha = exp2_fast(ref - moved);  // 0 for a row's first key
      ref = moved;
#pragma unroll
      for (int nb = 0; nb < D / 32; ++nb) o[nb] *= alpha;
      l *= alpha;
    }
    f32x16 p0, p1;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      p0[j] = exp2_fast(fmaf(s0[j], sl2, -ref));
      p1[j] = exp2_fast(fmaf(s1[j], sl2, -ref));
    }
    float r0 = p0[0];
    float r1 = p1[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) {
      r0 += p0[j];
      r1 += p1[j];
    }
    pf[0] = p_frag<Tag, 0>(p0);
    pf[1] = p_frag<Tag, 1>(p0);
    pf[2] = p_frag<Tag, 0>(p1);
    pf[3] = p_frag<Tag, 1>(p1);
    l += r0 + r1;
  };

  // Tiles that loads run ahead: in the tokens' type V's ring has no place for a third.
  constexpr auto kLeadOf = [](int g) { return kE4M3 || g == 0 ? 3 : 2; };
  using kFirstT = std::integral_constant<int, 0>;
  using kFullT = std::integral_constant<int, 1>;
  using kLastT = std::integral_constant<int, 2>;
  using kLoadsT = std::integral_constant<int, 3>;
  auto run = [&](auto group_tag) {
    constexpr int kGroup = decltype(group_tag)::value;
    constexpr int kLead = kLeadOf(kGroup);
    auto period = [&](int m, int slot, auto mode_tag) {
      constexpr int kMode = decltype(mode_tag)::value;
      constexpr bool kDoPv = kMode == kFullT::value || kMode == kLastT::value;
      constexpr bool kDoQk = kMode == kFirstT::value || kMode == kFullT::value;
      auto hook = [&](auto i_tag) {
        constexpr int i = decltype(i_tag)::value;
        // (Codes of tile m + 1 have landed, tile m + 2's are on their way.)
        if constexpr (kE4M3 && i == 0) prefill::pp::wait_vmcnt<kLoads>();
        if constexpr (i % 6 == 0 && i / 3 < kPuts) take(slot + 1, i / 6);
        if constexpr (i % 3 == 2 && i / 3 < kPuts) put(slot + 1, i / 3);
        constexpr int kAskFrom = 3 * kPuts + 1;
        if constexpr (i == kAskFrom) locate(m + kLead, slot + kLead);
        constexpr int k = i - kAskFrom - 2;
        if constexpr (k >= 0 && k % 3 == 0 && k / 3 < kPieces) ask(slot + kLead, k / 3);
        static_assert(kAskFrom + 2 + 3 * (kPieces - 1) < kSteps, "the tile's moves fit the phase");
      };
      auto mfma = [&]() {
        if constexpr (kMode == kLoadsT::value) {
          static_for<0, kSteps>([&](auto i) { hook(i); });
        } else {
          mfma_phase(slot, std::bool_constant<kDoPv>{}, std::bool_constant<kDoQk>{}, hook);
        }
      };
      if constexpr (kGroup == 0) {
        if constexpr (kMode == kFirstT::value) prefetch_qk(slot);
        mfma();
        if constexpr (kDoQk) {
          prefetch(slot + 1);
          softmax_phase(m);
        }
      } else {
        if constexpr (kMode == kFirstT::value) prefetch_qk(slot);
        if constexpr (kDoPv) {
          prefetch(slot);
          softmax_phase(m - 1);
        }
        mfma();
      }
      // In the tokens' type: tile m + 1's loads into LDS have landed, later ones are on their way; the barrier
      // publishes it.
      if constexpr (!kE4M3) prefill::pp::wait_vmcnt<(kLead - 1) * kLoads>();
      phase_barrier();
    };
    int m = 0;
    if (my_tiles > 0) {
      period(0, 0, kFirstT{});
      for (m = 1; m < my_tiles;) {
        bool done = false;
        static_for<0, kStages>([&](auto j) {
          if (done) return;
          period(m, (1 + decltype(j)::value) % kStages, kFullT{});
          done = ++m == my_tiles;
        });
      }
      period(m, m % kStages, kLastT{});
      ++m;
    }
    for (; m <= num_tiles; ++m) period(m, m % kStages, kLoadsT{});
  };
  if (num_tiles > 0) {
    auto ask_tile = [&](int i) {
      locate(i, i);
      static_for<0, kPieces>([&](auto j) { ask(i, decltype(j)::value); });
    };
    ask_tile(0);
    ask_tile(1);
    if (kE4M3 || group == 0) ask_tile(2);
    if constexpr (kE4M3) {
      prefill::pp::wait_vmcnt<2 * kLoads>();
      static_for<0, kPuts>([&](auto i) {
        if constexpr (decltype(i)::value % 2 == 0) take(0, decltype(i)::value / 2);
        put(0, decltype(i)::value);
      });
    } else if (group == 0) {
      prefill::pp::wait_vmcnt<2 * kLoads>();
    } else {
      prefill::pp::wait_vmcnt<kLoads>();
    }
    phase_barrier();
    if (group == 0) {
      run(std::integral_constant<int, 0>{});
    } else {
      run(std::integral_constant<int, 1>{});
    }
  }

  prefill::pp::wait_vmcnt<0>();  // (the loads of tiles past the end have landed before LDS is used again)
  phase_barrier();
  const CachedAttnArgs& e = reload_args();
  // Rows to sum again (sum_again): both halves of a row's lanes say which.
  uint32_t again = 0;
  if (e.causal && seq.count > 1) {
    float sum = 0.f;
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb) {
#pragma unroll
      for (int j = 0; j < 16; ++j) sum = fmaf(o[nb][j], 0.f, sum);
    }
    const uint64_t bad = __builtin_amdgcn_ballot_w64(sum != 0.f && my_row < rows);
    again = static_cast<uint32_t>(bad) | static_cast<uint32_t>(bad >> 32);
  }
  // f(row of the wave, its reference point, its sum, its four dims, which of them) for those rows, when the wave's stores have
  // been made.
  auto each_again = [&](float lt, auto&& f) {
    if (again == 0) return;
    prefill::pp::wait_vmcnt<0>();
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (as tid)
    const int lane_dim = 4 * (lane % (D / 4));
    while (again != 0) {
      const int r = __builtin_ctz(again);
      again &= again - 1;
      const float row_ref = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ref), r));
      const float row_sum = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lt), r));
      if (row_sum != row_sum) continue;  // (NaN whatever V is)
      const f32x4 x = sum_again<Tag, D, kE4M3>(reload_args(), item, row0 + r, row_ref, lane);
      if (lane < D / 4) f(r, row_sum, x, lane_dim);
    }
  };
  // Rows leave whole: each wave stages its 32 in its own part of the (free) rings, padded by 16 bytes.
  const float lt = sum_halves(l);
  constexpr int kStageRow = 4 * D + 16;
  static_assert(kWaves * 16 * kStageRow <= L::kBytes, "16 rows of each wave fit");
  char* stage = smem + wave * 16 * kStageRow;
  const float inv = inverse(lt);
  if (item.partial) {
    // (In two halves of 16 rows.)
    float* po = e.partial_o + (e.wide_partials + static_cast<int64_t>(item.slot) * kRows + wave * kWaveRows) * D;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (((lane >> 4) & 1) == part) {
        char* w = stage + (lane & 15) * kStageRow + 16 * half;
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(w + 32 * (4 * nb + g)) =
                f32x4{o[nb][4 * g], o[nb][4 * g + 1], o[nb][4 * g + 2], o[nb][4 * g + 3]};
        }
      }
      constexpr int kLanes = D / 4;  // of a row
      const int c = lane % kLanes;
#pragma unroll
      for (int j = 0; j < 16 * kLanes / 64; ++j) {
        const int r = j * (64 / kLanes) + lane / kLanes;
        const f32x4 x = *reinterpret_cast<const f32x4*>(stage + r * kStageRow + 16 * c);
        if (row0 + 16 * part + r < rows) *reinterpret_cast<f32x4*>(po + (16 * part + r) * D + 4 * c) = x;
      }
    }
    if (my_row < rows && half == 0)
      e.partial_ml[e.wide_partials + static_cast<int64_t>(item.slot) * kRows + my_row - q0] = point_and_sum(ref, lt);
    each_again(lt, [&](int r, float, const f32x4& x, int dim) { *reinterpret_cast<f32x4*>(po + r * D + dim) = x; });
    return;
  }
  constexpr int kOutRow = 2 * D + 16;
  stage = smem + wave * kWaveRows * kOutRow;
  {
    char* w = stage + (lane & 31) * kOutRow + 8 * half;
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<u32x2*>(w + 16 * (4 * nb + g)) =
            u32x2{E::pack2(o[nb][4 * g] * inv, o[nb][4 * g + 1] * inv),
                  E::pack2(o[nb][4 * g + 2] * inv, o[nb][4 * g + 3] * inv)};
    }
  }
  constexpr int kLanes = D / 8;  // of a row
  uint16_t* out = e.o + (e.c.cu_seqlens ? seq.start * e.o_ss : item.b * e.o_bs) + 8 * (lane % kLanes);
#pragma unroll
  for (int j = 0; j < kWaveRows * kLanes / 64; ++j) {
    const int r = j * (64 / kLanes) + lane / kLanes;
    const u32x4 x = *reinterpret_cast<const u32x4*>(stage + r * kOutRow + 16 * (lane % kLanes));
    if (row0 + r < rows) {
      const int token = token_of_row(e, row0 + r);
      const int head = item.hkv * e.group + row0 + r - token * e.group;
      *reinterpret_cast<u32x4*>(out + token * e.o_ss + head * e.o_hs) = x;
    }
  }
  if (my_row < rows && half == 0) {
    const int token = token_of_row(e, my_row);
    e.lse[(static_cast<int64_t>(seq.start) + token) * e.heads + item.hkv * e.group + my_row - token * e.group] =
        log_sum(ref, lt);
  }
  each_again(lt, [&](int r, float row_sum, const f32x4& x, int dim) {
    const float row_inv = inverse(row_sum);
    const int token = token_of_row(e, row0 + r);
    const int head = item.hkv * e.group + row0 + r - token * e.group;
    *reinterpret_cast<u32x2*>(e.o + (e.c.cu_seqlens ? seq.start * e.o_ss : item.b * e.o_bs) + token * e.o_ss +
                              head * e.o_hs + dim) =
        u32x2{E::pack2(x[0] * row_inv, x[1] * row_inv), E::pack2(x[2] * row_inv, x[3] * row_inv)};
  });
}

// The narrow sequences of a ragged batch run in the same launch: each workgroup takes its share of them too, with
// eight waves, every other workgroup first of all. So one half of the chip reads the cache while the other is on
// the matrix cores. (Two launches took 4.4 us more, where one had nothing to do.)
constexpr int kNarrowCols = (kNarrowRows + 15) / 16;

template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void run_wide(Batch& batch, char* smem) {
  const CachedAttnArgs& a = reload_args();
  batch.args = &a;
  Segments<kWide, D> segments(a, batch);
  Item item;
  while (segments.next(reload_args(), batch, item)) {
    pp_item<Tag, D, kE4M3>(reload_args(), uniform(item), smem);
    if (!segments.more()) break;
    phase_barrier();  // (the next item uses the LDS again)
    batch.read(reload_args());  // (kept, it would take registers from the item)
  }
}

template <typename Tag, int D, bool kE4M3>
__device__ __forceinline__ void run_narrow(Batch& batch, char* smem) {
  const CachedAttnArgs& a = reload_args();
  batch.args = &a;
  Segments<kNarrow, D> segments(a, batch);
  Item item;
  if (!segments.next(a, batch, item)) return;
  item = uniform(item);
  if (item.seq.count * a.group <= 16) {
    narrow_item<Tag, D, kE4M3, 1, kWaves>(reload_args(), item, smem);
  } else {
    narrow_item<Tag, D, kE4M3, kNarrowCols, kWaves>(reload_args(), item, smem);
  }
}

template <typename Tag, int D, bool kE4M3, bool kRagged>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
    cached_wide_kernel(const CachedAttnArgs a) {
  constexpr int kBytes = Lds<D, kE4M3>::kBytes, kNarrowBytes = NarrowLds<D, kNarrowCols, kWaves>::kBytes;
  __shared__ __attribute__((aligned(16))) char smem[kRagged && kNarrowBytes > kBytes ? kNarrowBytes : kBytes];
  Batch batch(a);
  clear_list<kWide>(a);
  if constexpr (!kRagged) {
    run_wide<Tag, D, kE4M3>(batch, smem);
  } else {
    clear_list<kNarrow>(a);
    clear_unowned<D>(a);
    bool lane_narrow = false;
    bool lane_wide = false;
    batch.each([&](const Sequence& s) {
      lane_narrow |= blocks_of<kNarrow, D>(a, s) > 0;
      lane_wide |= blocks_of<kWide, D>(a, s) > 0;
    });
    const bool any[2] = {wave_any(lane_narrow), wave_any(lane_wide)};
    const int narrow_at = any[kWide] ? (blockIdx.x >> 3) & 1 : 0;  // (neighbours run on different XCDs)
    for (int i = 0; i < 2; ++i) {
      if (i == narrow_at) {
        if (any[kNarrow]) run_narrow<Tag, D, kE4M3>(batch, smem);
      } else {
        if (any[kWide]) run_wide<Tag, D, kE4M3>(batch, smem);
      }
      if (i == 1 || !any[kNarrow] || !any[kWide]) continue;
      phase_barrier();  // (the other part uses the LDS again)
      batch.read(reload_args());  // (kept, it would take registers from the items)
    }
  }
}

template <typename Tag, int D, bool kE4M3>
void launch_ragged_or_not(const CachedAttnArgs& args, const CachedPlan& plan, hipStream_t stream) {
  if (args.c.cu_seqlens != nullptr) {
    const int64_t most = plan.wide.workgroups > plan.narrow.workgroups ? plan.wide.workgroups : plan.narrow.workgroups;
    hipLaunchKernelGGL((cached_wide_kernel<Tag, D, kE4M3, true>), dim3(static_cast<uint32_t>(most)), dim3(kThreads), 0, stream, args);
  } else {
    hipLaunchKernelGGL((cached_wide_kernel<Tag, D, kE4M3, false>), dim3(static_cast<uint32_t>(plan.wide.workgroups)), dim3(kThreads), 0,
                       stream, args);
  }
}

template <typename Tag, int D>
hipError_t launch_typed(const CachedAttnArgs& args, const CachedPlan& plan, bool e4m3, hipStream_t stream) {
  if (e4m3) {
    launch_ragged_or_not<Tag, D, true>(args, plan, stream);
  } else {
    launch_ragged_or_not<Tag, D, false>(args, plan, stream);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace cached

hipError_t launch_cached_wide(const CachedAttnArgs& args, const CachedPlan& plan, DType dtype, bool e4m3, int head_dim,
                              hipStream_t stream) {
  using namespace cached;
  if (dtype == DType::bf16) {
    return head_dim == 64 ? launch_typed<bf16_tag, 64>(args, plan, e4m3, stream)
                          : launch_typed<bf16_tag, 128>(args, plan, e4m3, stream);
  }
  return head_dim == 64 ? launch_typed<f16_tag, 64>(args, plan, e4m3, stream)
                        : launch_typed<f16_tag, 128>(args, plan, e4m3, stream);
}

}  // namespace fl

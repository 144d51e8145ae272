// Attention of new tokens to the caches of their sequences (fl_cached_attention): a ragged batch whose
// sequences have any number of new tokens each, over slabs or a pool of blocks, in the tokens' type or in
// e4m3 codes with a power-of-two scale per row.
//
// For token i of sequence b, query head h, KV head h / group, with the n_b new tokens the last of the
// sequence's len_b:
//   s_j = scale q . k_j for j < len_b (causal: and j <= len_b - n_b + i),
//   o = sum_j softmax(s)_j v_j, lse = log sum_j e^(s_j); no such j: o = 0, lse = -inf.
//
// Lengths are known on the device only. Sequences with few rows (tokens x heads of a group) are bound by
// reading the cache and run the narrow form (cached_narrow.hpp), those with many by the matrix cores and run the
// wide one (cached_wide.hip). The host knows which there can be: calls with only few rows launch
// cached_narrow.hip, calls without cu_seqlens and with many the wide kernel alone, and ragged batches the
// wide kernel with both. Every workgroup derives the same schedule from the lengths (Segments, cached.hpp) and
// takes its own part of it; the grid is an upper bound from the sizes. Where blocks of rows are few, their keys
// are split over several workgroups, and a last kernel, here, merges the partials in order.
#include "cached.hpp"

namespace fl {
namespace cached {
namespace {

// With M = max_s m_s, o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), the splits in a fixed order. Splits
// in which a row sees no key (m = -inf) contribute nothing. A workgroup takes 256 / (D / 4) rows of a
// block, D / 4 lanes to a row; where a block has fewer rows than it has room for, several groups of lanes
// share a row's splits and are added up in order through LDS. Bound by latency for few rows (list entry, then
// partials: 4.8 us for 64 blocks of 12 splits and 4 rows), by reading the partials for many (31 MB of them 9.3 us).
constexpr int kMergeThreads = 256;
template <int D>
constexpr int kMergeRows = kMergeThreads / (D / 4);
template <typename Tag, int D>
__global__ void __launch_bounds__(kMergeThreads)
    cached_merge_kernel(const CachedAttnArgs a, int narrow_groups, int narrow_chunks) {
  using E = Elem<Tag>;
  constexpr int kLanes = D / 4;
  constexpr int kGroups = kMergeRows<D>;
  __shared__ f32x4 sums[kGroups][kLanes];
  __shared__ float ls[kGroups];
  const bool wide = static_cast<int>(blockIdx.x) >= narrow_groups;
  const int id = wide ? blockIdx.x - narrow_groups : blockIdx.x;
  const int chunks = wide ? block_rows(kWide) / kGroups : narrow_chunks;
  const int at = id / chunks;
  const int chunk = id - at * chunks;
  const MergeBlock mb = a.parts[wide ? kWide : kNarrow].merge_blocks[at];
  if (mb.splits == 0) return;
  const int per_block = wide ? block_rows(kWide) : kNarrowRows;
  const int rows = min(per_block, mb.count * a.group - mb.block * per_block);
  const int first_row = chunk * kGroups;
  if (first_row >= rows) return;
  const int64_t base = wide ? a.wide_partials : 0;
  const bool line = mb.splits < 0;
  const int n = line ? -mb.splits : mb.splits;
  auto slot_row = [&](int s) { return base + static_cast<int64_t>(line && s > 0 ? 2 * (at + s) : mb.slot + s) * per_block; };
  const int d = threadIdx.x % kLanes;
  const int group = threadIdx.x / kLanes;
  // Groups to a row (a power of two), where all of the chunk's rows fit.
  int share = 1;
  while (!wide && 2 * share * min(rows - first_row, kGroups) <= kGroups) share *= 2;
  const int part = group & (share - 1);
  const int r = first_row + group / share;
  const bool in = r < rows;
  auto row_of = [&](int s) { return slot_row(s) + (in ? r : 0); };
  float m = -INFINITY;
  float l = 0.f;
  f32x4 o = {};
  // The first two partials of a lane are on their way before any maximum is known.
  const int s0 = part, s1 = part + share;
  const bool has0 = s0 < n, has1 = s1 < n;
  const f32x4 o0 = has0 ? reinterpret_cast<const f32x4*>(a.partial_o + row_of(s0) * D)[d] : f32x4{};
  const f32x4 o1 = has1 ? reinterpret_cast<const f32x4*>(a.partial_o + row_of(s1) * D)[d] : f32x4{};
#pragma unroll 4
  for (int s = 0; s < n; ++s) m = fmaxf(m, a.partial_ml[row_of(s)].x);
  auto add = [&](int s, const f32x4& x) {
    const f32pair p = a.partial_ml[row_of(s)];
    const float f = p.x == -INFINITY ? 0.f : exp2_fast(p.x - m);
    l += p.y * f;
    o += x * f;
  };
  if (has0) add(s0, o0);
  if (has1) add(s1, o1);
#pragma unroll 4
  for (int s = s1 + share; s < n; s += share) add(s, reinterpret_cast<const f32x4*>(a.partial_o + row_of(s) * D)[d]);
  if (share > 1) {
    sums[group][d] = o;
    if (d == 0) ls[group] = l;
    __syncthreads();
    if (part != 0) return;
    for (int k = 1; k < share; ++k) {
      o += sums[group + k][d];
      l += ls[group + k];
    }
  }
  if (!in) return;
  const float inv = inverse(l);
  const int place = mb.block * per_block + r;
  const int token = token_of_row(a, place);
  const int head = mb.hkv * a.group + place - token * a.group;
  const int64_t o_row = a.c.cu_seqlens ? (mb.start + token) * a.o_ss : mb.b * a.o_bs + token * a.o_ss;
  *reinterpret_cast<u32x2*>(a.o + o_row + head * a.o_hs + 4 * d) =
      u32x2{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  if (d == 0) a.lse[(static_cast<int64_t>(mb.start) + token) * a.heads + head] = log_sum(m, l);
}

// Workgroups of a narrow block, and of all.
int64_t narrow_chunks(const CachedPlan& plan, int head_dim) {
  const int rows = kMergeThreads / (head_dim / 4);
  return ((plan.most_rows < kNarrowRows ? plan.most_rows : kNarrowRows) + rows - 1) / rows;
}
int64_t merge_groups(const CachedPlan& plan, int head_dim) {
  return plan.narrow.merges * narrow_chunks(plan, head_dim) +
         plan.wide.merges * int64_t{block_rows(kWide) / (kMergeThreads / (head_dim / 4))};
}

template <typename Tag, int D>
hipError_t launch_merge(const CachedAttnArgs& args, const CachedPlan& plan, hipStream_t stream) {
  const int chunks = static_cast<int>(narrow_chunks(plan, D));
  hipLaunchKernelGGL((cached_merge_kernel<Tag, D>), dim3(static_cast<uint32_t>(plan.merge_groups)), dim3(kMergeThreads), 0,
                     stream, args, plan.narrow.merges * chunks, chunks);
  return hipGetLastError();
}

// Grid and slots of one kind's kernel, whose sequences have `least` to `most` blocks in all and which runs
// `resident` workgroups at once (Segments, cached.hpp).
CachedPlan::Part plan_part(const CachedAttnArgs& args, Kind kind, int64_t least, int64_t most, int64_t resident,
                           int min_tiles, bool whole) {
  CachedPlan::Part part{};
  part.workgroups = most;
  part.min_tiles = min_tiles;
  const int64_t tiles = (args.c.capacity + kKeys - 1) / kKeys;
  if (args.num_splits > 1) {
    part.workgroups = part.partials = part.merges = most * args.num_splits;
  } else if (args.num_splits == 0 && tiles > min_tiles && least <= kWholeRounds * resident && !whole) {
    part.slots = static_cast<int>(resident);
    // The line needs blocks enough, and positions that fit 32 bits.
    part.line = kind == kWide && 4 * most > resident && most * (tiles + kStartTiles + 1) < (int64_t{1} << 30);
    const int64_t shares = most * ((tiles + min_tiles - 1) / min_tiles);
    part.partials = part.line ? 2 * resident : shares < resident ? shares : resident;
    part.workgroups = part.line || part.partials == resident ? resident : part.partials;
    if (most > part.workgroups) part.workgroups = most;
    part.merges = static_cast<int>(part.line ? resident : part.partials);
  }
  return part;
}

}  // namespace
}  // namespace cached

CachedPlan plan_cached_attn(const CachedAttnArgs& args, int head_dim, bool e4m3, int cu_count) {
  using namespace cached;
  const int64_t cus = cu_count > 0 ? cu_count : 256;
  const CacheArgs& c = args.c;
  const bool ragged = c.cu_seqlens != nullptr;
  const int64_t rows = static_cast<int64_t>(c.tokens) * args.group;
  const int64_t per_seq = static_cast<int64_t>(c.tokens_per_seq) * args.group;
  CachedPlan plan{};
  // Rows of the largest sequence there can be, which kinds there can be, and their blocks.
  plan.most_rows = static_cast<int>(ragged ? rows : per_seq);
  // Short caches keep their blocks whole, one workgroup each (of eight waves, with up to 16 rows): its time goes up
  // by 5.3 us for 1,000 keys (9.5 with more rows, on four waves), a merge and its launch cost 5.5 us (7). In a large
  // batch splits gain less than that from longer caches too; but lengths can differ, which whole blocks do not even
  // out, so only part of it counts. us, whole / split + merge, 32/8 heads, head_dim 128, e4m3: B = 1, 640 keys 9.1 /
  // 6.5 + 4.1, 1,024 11.5 / 6.7 + 4.4, 1,536 14.3 / 6.5 + 4.7; B = 16, 1,024 14.6 / 12.6 + 4.4, 2,048 22.5 / 18.4 + 4.5;
  // bf16, B = 16, 2,048 32.0 / 29.6 + 4.1; 8 tokens each, e4m3: B = 1, 640 13.6 / 8.9 + 4.4, B = 16, 1,024 19.1 / 19.2 + 6.4.
  const double megabytes = 2e-6 * c.batch * c.heads_kv * c.capacity * head_dim * (e4m3 ? 1 : 2);
  plan.whole = plan.most_rows <= 16 ? 5.3e-3 * c.capacity < 5.5 + 0.06 * megabytes
                                    : plan.most_rows <= kNarrowRows && 9.5e-3 * c.capacity < 7.0 + 0.1 * megabytes;
  if (ragged || per_seq <= kNarrowRows) {
    const int64_t least = ragged ? 0 : c.batch * int64_t{c.heads_kv};
    // (In the kernel of the wide ones a workgroup has twice the waves, and a CU to itself.)
    const bool with_wide = plan.most_rows > kNarrowRows;
    plan.narrow = plan_part(args, kNarrow, least, c.batch * int64_t{c.heads_kv},
                            cus * (with_wide ? 1 : cached_narrow_resident(head_dim, e4m3, plan.most_rows)),
                            with_wide ? 4 : 2, plan.whole);
  }
  if (plan.most_rows > kNarrowRows) {
    const int64_t wide_rows = block_rows(kWide);
    const int64_t blocks = (per_seq + wide_rows - 1) / wide_rows * c.batch;
    const int64_t least = ragged ? 0 : blocks * c.heads_kv;
    const int64_t most = (ragged ? rows / wide_rows + (c.batch < rows / kNarrowRows + 1 ? c.batch : rows / kNarrowRows + 1)
                                 : blocks) * c.heads_kv;
    plan.wide = plan_part(args, kWide, least, most, cus, 4, false);
  }
  plan.wide_partials = plan.narrow.partials * kNarrowRows;
  plan.partial_rows = plan.wide_partials + plan.wide.partials * block_rows(kWide);
  plan.floats = plan.partial_rows * (head_dim + 2) +
                (plan.narrow.merges + static_cast<int64_t>(plan.wide.merges)) * (sizeof(MergeBlock) / sizeof(float));
  plan.merge_groups = merge_groups(plan, head_dim);
  return plan;
}

hipError_t launch_cached_attn(const CachedAttnArgs& args, const CachedPlan& plan, DType dtype, bool e4m3,
                              int head_dim, hipStream_t stream) {
  using namespace cached;
  const hipError_t err = plan.wide.workgroups > 0 ? launch_cached_wide(args, plan, dtype, e4m3, head_dim, stream)
                                                  : launch_cached_narrow(args, plan, dtype, e4m3, head_dim, stream);
  if (err != hipSuccess || plan.partial_rows == 0) return err;
  if (head_dim == 64) {
    return dtype == DType::bf16 ? launch_merge<bf16_tag, 64>(args, plan, stream)
                                : launch_merge<f16_tag, 64>(args, plan, stream);
  }
  return dtype == DType::bf16 ? launch_merge<bf16_tag, 128>(args, plan, stream)
                              : launch_merge<f16_tag, 128>(args, plan, stream);
}

}  // namespace fl

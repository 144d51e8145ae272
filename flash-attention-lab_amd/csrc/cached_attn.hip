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
// reading the cache and run on cached_narrow.hip, those with many by the matrix cores and run on
// cached_pp.hip (head_dim 128) or cached_wide.hip (64); without cu_seqlens the host knows which it is, and only that kernel is launched.
// Every workgroup of either derives the same list of items from the lengths (find_item, cached.hpp) and
// takes the one of its own number; the grid is an upper bound from the sizes. Where the items are few, keys
// are split over several workgroups, and a last kernel, here, merges the partials in order.
#include "cached.hpp"

namespace fl {
namespace cached {
namespace {

constexpr int kThreads = 256;

// The partials of a row.
struct Partials {
  int splits;
  int64_t first, step;  // rows of the workspace
};
__device__ __forceinline__ Partials partials_of(const CachedAttnArgs& a, const cache::Token& t, int head, int head_dim) {
  const int2 info = a.sequence_splits[t.b];
  const int hkv = head / a.group;
  const int rows = t.count * a.group;
  const int r = t.index * a.group + head - hkv * a.group;
  const Kind kind = rows <= kNarrowRows ? kNarrow : kWide;
  const int per_block = block_rows(kind, head_dim);
  const int blocks = (rows + per_block - 1) / per_block;
  const int block = r / per_block;
  const int64_t slot = info.y + (static_cast<int64_t>(blocks - 1 - block) * a.c.heads_kv + hkv) * info.x;
  return Partials{info.x, (kind == kWide ? a.wide_partials : 0) + slot * per_block + r - block * per_block, per_block};
}

// With M = max_s m_s, o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), the splits in a fixed order. Splits
// in which a row sees no key (m = -inf) contribute nothing. kGroups groups of D / 4 lanes take every
// kGroups-th split of a row and are added up in order through LDS: one for many rows of few splits, all of
// a workgroup for few rows of many, where the time is that of one row's dependent loads.
template <typename Tag, int D, int kGroups>
__global__ void __launch_bounds__(kThreads) cached_merge_kernel(const CachedAttnArgs a) {
  using E = Elem<Tag>;
  constexpr int kLanes = D / 4;
  constexpr int kRowThreads = kLanes * kGroups;
  static_assert(kGroups == 1 || kRowThreads == kThreads, "a row's groups are a workgroup or one group");
  const int64_t all = static_cast<int64_t>(a.c.tokens) * a.heads;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kRowThreads;
  const int64_t row = min(at, all - 1);
  const int token = static_cast<int>(row / a.heads);
  const int head = static_cast<int>(row - static_cast<int64_t>(token) * a.heads);
  const cache::Token t = cache::find_token<kGroups == 1 ? kLanes : 64>(a.c, token);
  if (at >= all || t.b < 0) return;
  const Partials p = partials_of(a, t, head, D);
  const int n = p.splits;
  if (n <= 1) return;
  const int d = threadIdx.x % kLanes;
  const int group = kGroups == 1 ? 0 : threadIdx.x / kLanes;
  const f32pair* ml = a.partial_ml + p.first;
  const f32x4* po = reinterpret_cast<const f32x4*>(a.partial_o + p.first * D) + d;
  float m = -INFINITY;
  if constexpr (kGroups == 1) {
    for (int s = 0; s < n; ++s) m = fmaxf(m, ml[s * p.step].x);
  } else {
    for (int s = threadIdx.x & 63; s < n; s += 64) m = fmaxf(m, ml[s * p.step].x);
#pragma unroll
    for (int k = 32; k >= 1; k /= 2) m = fmaxf(m, __shfl_xor(m, k));
  }
  float l = 0.f;
  f32x4 o = {};
#pragma unroll 4
  for (int s = group; s < n; s += kGroups) {
    const f32pair x = ml[s * p.step];
    const float f = x.x == -INFINITY ? 0.f : exp2_fast(x.x - m);
    l += x.y * f;
    o += po[s * p.step * kLanes] * f;
  }
  if constexpr (kGroups > 1) {
    __shared__ f32x4 sums[kGroups][kLanes];
    __shared__ float ls[kGroups];
    sums[group][d] = o;
    if (d == 0) ls[group] = l;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
      o += sums[k][d];
      l += ls[k];
    }
  }
  const float inv = inverse(l);
  const int64_t base = a.c.cu_seqlens ? token * a.o_ss : t.b * a.o_bs + t.index * a.o_ss;
  *reinterpret_cast<u32x2*>(a.o + base + head * a.o_hs + 4 * d) =
      u32x2{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  if (d == 0) a.lse[row] = log_sum(m, l);
}

template <typename Tag, int D>
hipError_t launch_merge(const CachedAttnArgs& args, const CachedPlan& plan, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(args.c.tokens) * args.heads;
  if (plan.many_splits) {
    hipLaunchKernelGGL((cached_merge_kernel<Tag, D, kThreads / (D / 4)>), dim3(static_cast<uint32_t>(rows)),
                       dim3(kThreads), 0, stream, args);
  } else {
    const int64_t lanes = rows * (D / 4);
    hipLaunchKernelGGL((cached_merge_kernel<Tag, D, 1>), dim3(static_cast<uint32_t>((lanes + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, stream, args);
  }
  return hipGetLastError();
}

// Grid, slots and rounds of one kind's kernel, whose sequences have `least` to `most` blocks in all and run
// on `slots` workgroups at once.
CachedPlan::Part plan_part(const CachedAttnArgs& args, int64_t least, int64_t most, int64_t resident, int min_tiles) {
  CachedPlan::Part part{};
  part.workgroups = most;
  part.min_tiles = min_tiles;
  part.max_rounds = 1;
  const int64_t tiles = (args.c.capacity + kKeys - 1) / kKeys;
  if (args.num_splits > 1) {
    part.workgroups = part.partials = most * args.num_splits;
  } else if (args.num_splits == 0 && tiles > min_tiles && least < kMaxRounds * resident) {
    part.slots = static_cast<int>(resident);
    // (With few blocks one round of splits is even enough.)
    part.max_rounds = 4 * most <= resident ? 1 : kMaxRounds;
    const int64_t splits = (tiles + min_tiles - 1) / min_tiles;
    const int64_t items = part.max_rounds * resident;
    part.partials = most * splits < items ? most * splits : items;
    part.workgroups = part.partials > most ? part.partials : most;
  }
  return part;
}

CachedAttnArgs with_part(CachedAttnArgs args, const CachedPlan::Part& part) {
  args.slots = part.slots;
  args.max_rounds = part.max_rounds;
  args.min_tiles = part.min_tiles;
  return args;
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
  if (ragged || per_seq <= kNarrowRows) {
    const int64_t least = ragged ? 0 : c.batch * int64_t{c.heads_kv};
    plan.narrow = plan_part(args, least, c.batch * int64_t{c.heads_kv},
                            cus * cached_narrow_resident(head_dim, e4m3, plan.most_rows), 2);
  }
  if (plan.most_rows > kNarrowRows) {
    const int64_t wide_rows = block_rows(kWide, head_dim);
    const int64_t blocks = (per_seq + wide_rows - 1) / wide_rows * c.batch;
    const int64_t least = ragged ? 0 : blocks * c.heads_kv;
    const int64_t most = (ragged ? rows / wide_rows + (c.batch < rows / kNarrowRows + 1 ? c.batch : rows / kNarrowRows + 1)
                                 : blocks) * c.heads_kv;
    plan.wide = plan_part(args, least, most, wide_resident(head_dim) * cus, 4);
  }
  plan.wide_partials = plan.narrow.partials * kNarrowRows;
  plan.partial_rows = plan.wide_partials + plan.wide.partials * block_rows(kWide, head_dim);
  if (plan.partial_rows > 0) plan.floats = plan.partial_rows * (head_dim + 2) + 2 * static_cast<int64_t>(c.batch);
  // One workgroup per row pays while the rows are about as few as the CUs and their splits many.
  plan.many_splits = static_cast<int64_t>(c.tokens) * args.heads <= 8 * cus;
  return plan;
}

hipError_t launch_cached_attn(const CachedAttnArgs& args, const CachedPlan& plan, DType dtype, bool e4m3,
                              int head_dim, hipStream_t stream) {
  using namespace cached;
  hipError_t err = hipSuccess;
  if (plan.wide.workgroups > 0)
    err = launch_cached_wide(with_part(args, plan.wide), plan.wide.workgroups, dtype, e4m3, head_dim, stream);
  if (err == hipSuccess && plan.narrow.workgroups > 0)
    err = launch_cached_narrow(with_part(args, plan.narrow), plan, dtype, e4m3, head_dim, stream);
  if (err != hipSuccess || plan.partial_rows == 0) return err;
  if (head_dim == 64) {
    return dtype == DType::bf16 ? launch_merge<bf16_tag, 64>(args, plan, stream)
                                : launch_merge<f16_tag, 64>(args, plan, stream);
  }
  return dtype == DType::bf16 ? launch_merge<bf16_tag, 128>(args, plan, stream)
                              : launch_merge<f16_tag, 128>(args, plan, stream);
}

}  // namespace fl

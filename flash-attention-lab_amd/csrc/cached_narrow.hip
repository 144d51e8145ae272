// The kernels of attention over a cache for calls whose sequences all have at most 48 rows (cached_narrow.hpp).
#include "cached_narrow.hpp"

namespace fl {
namespace cached {
namespace {

// Workgroups per CU (a wave of each per SIMD): by the registers of up to kCols column blocks. (One block at
// head_dim 128 does not fit the 128 registers of a fourth: 25 of them spilled, 162 us against 94 for 8 sequences of
// 32K keys in e4m3, and 105 with two.)
template <int D, bool kE4M3, int kCols>
constexpr int kResident = kCols > 1 || (D == 128 && !kE4M3) ? 2 : D == 128 ? 3 : 4;

template <int D, bool kE4M3, int kCols, int kWaves>
constexpr int kPerSimd = kWaves == 8 ? 2 : kResident<D, kE4M3, kCols>;

// kCols: column blocks of the largest sequence. With kMixed (ragged batches) sequences of one block run
// the one-block form.
template <typename Tag, int D, bool kE4M3, int kCols, bool kMixed, int kWaves = 4>
__global__ void __launch_bounds__(64 * kWaves)
    __attribute__((amdgpu_waves_per_eu(kPerSimd<D, kE4M3, kCols, kWaves>, kPerSimd<D, kE4M3, kCols, kWaves>)))
    cached_narrow_kernel(const CachedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[NarrowLds<D, kCols, kWaves>::kBytes];
  clear_list<kNarrow>(a);
  clear_unowned<D>(a);
  const Batch batch(a);
  Segments<kNarrow, D> segments(a, batch);
  Item item;
  if (!segments.next(a, batch, item)) return;
  item = uniform(item);
  if (kMixed && item.seq.count * a.group <= 16) {
    narrow_item<Tag, D, kE4M3, 1, kWaves>(reload_args(), item, smem);
  } else {
    narrow_item<Tag, D, kE4M3, kCols, kWaves>(reload_args(), item, smem);
  }
}

template <typename Tag, int D, bool kE4M3>
void launch_cols(const CachedAttnArgs& args, const CachedPlan& plan, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(plan.narrow.workgroups));
  constexpr int kThreads = 64 * 4;
  if (plan.most_rows <= 16 && plan.whole) {
    hipLaunchKernelGGL((cached_narrow_kernel<Tag, D, kE4M3, 1, false, 8>), grid, dim3(64 * 8), 0, stream, args);
  } else if (plan.most_rows <= 16) {
    hipLaunchKernelGGL((cached_narrow_kernel<Tag, D, kE4M3, 1, false>), grid, dim3(kThreads), 0, stream, args);
  } else if (args.c.cu_seqlens != nullptr) {
    hipLaunchKernelGGL((cached_narrow_kernel<Tag, D, kE4M3, 3, true>), grid, dim3(kThreads), 0, stream, args);
  } else if (plan.most_rows <= 32) {
    hipLaunchKernelGGL((cached_narrow_kernel<Tag, D, kE4M3, 2, false>), grid, dim3(kThreads), 0, stream, args);
  } else {
    hipLaunchKernelGGL((cached_narrow_kernel<Tag, D, kE4M3, 3, false>), grid, dim3(kThreads), 0, stream, args);
  }
}

template <typename Tag, int D>
hipError_t launch_typed(const CachedAttnArgs& args, const CachedPlan& plan, bool e4m3, hipStream_t stream) {
  if (e4m3) {
    launch_cols<Tag, D, true>(args, plan, stream);
  } else {
    launch_cols<Tag, D, false>(args, plan, stream);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace cached

int cached_narrow_resident(int head_dim, bool e4m3, int most_rows) {
  if (most_rows > 16 || (head_dim == 128 && !e4m3)) return 2;
  return head_dim == 128 ? 3 : 4;
}

hipError_t launch_cached_narrow(const CachedAttnArgs& args, const CachedPlan& plan, DType dtype, bool e4m3,
                                int head_dim, hipStream_t stream) {
  using namespace cached;
  if (dtype == DType::bf16) {
    return head_dim == 64 ? launch_typed<bf16_tag, 64>(args, plan, e4m3, stream)
                          : launch_typed<bf16_tag, 128>(args, plan, e4m3, stream);
  }
  return head_dim == 64 ? launch_typed<f16_tag, 64>(args, plan, e4m3, stream)
                        : launch_typed<f16_tag, 128>(args, plan, e4m3, stream);
}

}  // namespace fl

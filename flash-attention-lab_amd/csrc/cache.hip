// Writing rows of new tokens into a key-value cache and reading rows back (fl_cache_write, fl_cache_read).
//
// A cache of e4m3 codes has one power-of-two scale per row (a token's D values of one KV head): for a row
// with largest finite magnitude m the least e with m 2^-e <= 448 = 1.75 2^8, from m's exponent and
// mantissa bits. Since e4m3 is a floating format its relative precision does not depend on the scale as
// long as values are normal, so a power of two costs nothing against a scale of 448 / m, multiplying by
// it is exact, and it is stored as its exponent byte.
//
// Both are bound by memory traffic: every row is read once and written once. A row is handled by D / 8
// lanes with 8 elements each, so that every load and store of a wave covers whole rows, and a lane takes
// the K and the V row of its token and head (two loads in flight). 8,192 tokens of 8 KV heads at head_dim 128
// go from bf16 into an e4m3 pool in 14.7 us (3.4 TB/s, read and written; the rows come out of the caches in
// part) and come back in 11.1 (4.5); 32,768 come out of the pool in 32.4 (6.2; a large copy moves 5.1). A step of 24
// sequences takes 3.3 and 3.1 us, the latency of a launch and two dependent loads.
#include "cache.hpp"

namespace fl {
namespace cache {
namespace {

constexpr int kThreads = 256;
// Rows are held to 1.875 times the largest power of two of their type (61,440 in fp16): rounded to e4m3's
// four significant bits, the values beyond could become twice that power, which the type does not hold.
template <typename Tag>
constexpr float kMost = std::is_same_v<Tag, f16_tag> ? 61440.f : 0x1.ep127f;
constexpr uint32_t kNan = 0x7f;

// A lane's 8 elements of a row, as they lie in memory.
template <typename Tag>
struct Eight {
  static constexpr int kWords = sizeof(typename Elem<Tag>::storage) / 2;
  u32x4 w[kWords];
};
template <typename Tag>
__device__ __forceinline__ Eight<Tag> load8(const char* p) {
  Eight<Tag> r;
#pragma unroll
  for (int i = 0; i < Eight<Tag>::kWords; ++i) r.w[i] = load16(p + 16 * i);
  return r;
}
template <typename Tag>
__device__ __forceinline__ void store8(char* p, const Eight<Tag>& r) {
#pragma unroll
  for (int i = 0; i < Eight<Tag>::kWords; ++i) *reinterpret_cast<u32x4*>(p + 16 * i) = r.w[i];
}
template <typename Tag>
__device__ __forceinline__ float element(const Eight<Tag>& r, int i) {
  if constexpr (std::is_same_v<Tag, f32_tag>) {
    return __uint_as_float(r.w[i / 4][i % 4]);
  } else {
    return Elem<Tag>::to_float(static_cast<uint16_t>(r.w[0][i / 2] >> 16 * (i % 2)));
  }
}

// 8 codes times their row's scale.
template <typename Tag>
__device__ __forceinline__ Eight<Tag> decode8(u32x2 codes, float scale) {
  Eight<Tag> r;
  if constexpr (std::is_same_v<Tag, f32_tag>) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[h], scale, false);
      const f32x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[h], scale, true);
      r.w[h] = u32x4{__float_as_uint(lo[0]), __float_as_uint(lo[1]), __float_as_uint(hi[0]), __float_as_uint(hi[1])};
    }
  } else {
    const u32x2 lo = values4<Tag>(codes[0], scale), hi = values4<Tag>(codes[1], scale);
    r.w[0] = u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
  return r;
}

// Codes and scale byte of a row, 8 elements in each of kLanes lanes.
struct Quantised {
  u32x2 codes;
  uint32_t byte;
};
template <typename Tag, int kLanes>
__device__ __forceinline__ Quantised quantise(const Eight<Tag>& row) {
  float v[8];
  bool finite[8];
  uint32_t top = 0;  // bits of the largest magnitude: non-negative floats order as their bits do
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = element<Tag>(row, i);
    finite[i] = (__float_as_uint(v[i]) & 0x7f800000u) != 0x7f800000u;
    v[i] = fminf(fmaxf(v[i], -kMost<Tag>), kMost<Tag>);
    const uint32_t mag = __float_as_uint(v[i]) & 0x7fffffffu;
    top = max(top, finite[i] ? mag : 0u);
  }
  auto step = [&](uint32_t other) { top = max(top, other); };
  auto move = [&](auto ctrl) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(top), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  step(move(std::integral_constant<int, kDppQuadSwap1>{}));
  step(move(std::integral_constant<int, kDppQuadSwap2>{}));
  step(move(std::integral_constant<int, kDppRowHalfMirror>{}));
  if constexpr (kLanes == 16) step(move(std::integral_constant<int, kDppRowMirror>{}));
  static_assert(kLanes == 8 || kLanes == 16, "lanes of a row");
  // top = f 2^x with f in [1, 2): e = x - 8 for f <= 1.75, else x - 7. (A subnormal top is below 2^-126,
  // where e is held to -126 anyway.)
  const int x = static_cast<int>(top >> 23) - 127;
  int e = x - ((top & 0x7fffffu) <= 0x600000u ? 8 : 7);
  e = top == 0 ? 0 : min(max(e, -126), 120);
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  Quantised q;
  q.byte = static_cast<uint32_t>(e + 127);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float* y = v + 4 * h;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, w, true);
    uint32_t u = static_cast<uint32_t>(w);
#pragma unroll
    for (int i = 0; i < 4; ++i) u = finite[4 * h + i] ? u : (u & ~(0xffu << 8 * i)) | kNan << 8 * i;
    q.codes[h] = u;
  }
  return q;
}

// The row of this lane: token, head, the lane's chunk of 8 elements.
template <int D>
struct Lane {
  static constexpr int kLanes = D / 8;
  int token, head, chunk;
  bool in;
  Token t;
  int position;  // of the token in its sequence; meaningless for b < 0
};
template <int D>
__device__ __forceinline__ Lane<D> this_lane(const CacheArgs& c) {
  Lane<D> l;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / Lane<D>::kLanes;
  const int64_t rows = static_cast<int64_t>(c.tokens) * c.heads_kv;
  l.in = at < rows;
  const uint32_t row = static_cast<uint32_t>(l.in ? at : rows - 1);
  l.token = static_cast<int>(row / static_cast<uint32_t>(c.heads_kv));
  l.head = static_cast<int>(row) - l.token * c.heads_kv;
  l.chunk = threadIdx.x % Lane<D>::kLanes;
  l.t = find_token<Lane<D>::kLanes>(c, l.token);
  l.position = static_cast<int>(max(min(static_cast<int64_t>(l.t.len) - l.t.count + l.t.index, int64_t{INT32_MAX}),
                                    int64_t{-1}));
  return l;
}

// Element offset of this lane's 8 elements in the token rows.
template <int D>
__device__ __forceinline__ int64_t row_offset(const CacheArgs& c, const Lane<D>& l, int64_t bs, int64_t ss,
                                              int64_t hs) {
  const bool ragged = c.cu_seqlens != nullptr;
  return (ragged ? 0 : l.t.b * bs) + (ragged ? l.token : l.t.index) * ss + l.head * hs + 8 * l.chunk;
}

template <typename Tag, int D, bool kE4M3>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const CacheArgs c, const TokenRows r) {
  constexpr int kElem = sizeof(typename Elem<Tag>::storage);
  const Lane<D> l = this_lane<D>(c);
  const int64_t ko = row_offset(c, l, r.k_bs, r.k_ss, r.k_hs);
  const int64_t vo = row_offset(c, l, r.v_bs, r.v_ss, r.v_hs);
  // (The loads go out before the place is known; a token of no sequence has a row too.)
  const Eight<Tag> k = load8<Tag>(r.k + ko * kElem);
  const Eight<Tag> v = load8<Tag>(r.v + vo * kElem);
  bool keep = l.in && l.t.b >= 0 && l.position >= 0 && l.position < c.capacity;
  const Place at = place(c, keep ? l.t.b : 0, keep ? l.position : 0);
  keep = keep && at.outer >= 0 && at.outer < c.outer;
  const int64_t kc = at.outer * c.k_bs + at.row * c.k_ss + l.head * c.k_hs + 8 * l.chunk;
  const int64_t vc = at.outer * c.v_bs + at.row * c.v_ss + l.head * c.v_hs + 8 * l.chunk;
  if constexpr (kE4M3) {
    const Quantised qk = quantise<Tag, Lane<D>::kLanes>(k);
    const Quantised qv = quantise<Tag, Lane<D>::kLanes>(v);
    if (!keep) return;
    *reinterpret_cast<u32x2*>(c.k + kc) = qk.codes;
    *reinterpret_cast<u32x2*>(c.v + vc) = qv.codes;
    if (l.chunk == 0) {
      c.k_scales[at.outer * c.ks_bs + at.row * c.ks_ss + l.head * c.ks_hs] = static_cast<uint8_t>(qk.byte);
      c.v_scales[at.outer * c.vs_bs + at.row * c.vs_ss + l.head * c.vs_hs] = static_cast<uint8_t>(qv.byte);
    }
  } else {
    if (!keep) return;
    store8<Tag>(c.k + kc * kElem, k);
    store8<Tag>(c.v + vc * kElem, v);
  }
}

template <typename Tag, int D, bool kE4M3>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const CacheArgs c, const TokenRows r) {
  constexpr int kElem = sizeof(typename Elem<Tag>::storage);
  const Lane<D> l = this_lane<D>(c);
  const bool held = l.t.b >= 0 && l.position >= 0 && l.position < c.capacity;
  Place at = place(c, held ? l.t.b : 0, held ? l.position : 0);
  at.outer = min(max(at.outer, 0), c.outer - 1);
  const int64_t kc = at.outer * c.k_bs + at.row * c.k_ss + l.head * c.k_hs + 8 * l.chunk;
  const int64_t vc = at.outer * c.v_bs + at.row * c.v_ss + l.head * c.v_hs + 8 * l.chunk;
  Eight<Tag> k, v;
  if constexpr (kE4M3) {
    const u32x2 kq = *reinterpret_cast<const u32x2*>(c.k + kc);
    const u32x2 vq = *reinterpret_cast<const u32x2*>(c.v + vc);
    const float ks = scale_of(c.k_scales[at.outer * c.ks_bs + at.row * c.ks_ss + l.head * c.ks_hs]);
    const float vs = scale_of(c.v_scales[at.outer * c.vs_bs + at.row * c.vs_ss + l.head * c.vs_hs]);
    k = decode8<Tag>(kq, ks);
    v = decode8<Tag>(vq, vs);
  } else {
    k = load8<Tag>(c.k + kc * kElem);
    v = load8<Tag>(c.v + vc * kElem);
  }
  if (!l.in) return;
  if (!held) {
    k = Eight<Tag>{};
    v = Eight<Tag>{};
  }
  store8<Tag>(r.k + row_offset(c, l, r.k_bs, r.k_ss, r.k_hs) * kElem, k);
  store8<Tag>(r.v + row_offset(c, l, r.v_bs, r.v_ss, r.v_hs) * kElem, v);
}

template <typename Tag, int D, bool kE4M3>
hipError_t launch(const CacheArgs& args, const TokenRows& rows, bool write, hipStream_t stream) {
  const int64_t lanes = static_cast<int64_t>(args.tokens) * args.heads_kv * Lane<D>::kLanes;
  const dim3 grid(static_cast<uint32_t>((lanes + kThreads - 1) / kThreads));
  if (write) {
    hipLaunchKernelGGL((cache_write_kernel<Tag, D, kE4M3>), grid, dim3(kThreads), 0, stream, args, rows);
  } else {
    hipLaunchKernelGGL((cache_read_kernel<Tag, D, kE4M3>), grid, dim3(kThreads), 0, stream, args, rows);
  }
  return hipGetLastError();
}

template <typename Tag, int D>
hipError_t launch_format(const CacheArgs& args, const TokenRows& rows, bool e4m3, bool write, hipStream_t stream) {
  return e4m3 ? launch<Tag, D, true>(args, rows, write, stream) : launch<Tag, D, false>(args, rows, write, stream);
}

template <typename Tag>
hipError_t launch_dim(const CacheArgs& args, const TokenRows& rows, bool e4m3, int head_dim, bool write,
                      hipStream_t stream) {
  return head_dim == 64 ? launch_format<Tag, 64>(args, rows, e4m3, write, stream)
                        : launch_format<Tag, 128>(args, rows, e4m3, write, stream);
}

hipError_t launch_rows(const CacheArgs& args, const TokenRows& rows, DType dtype, bool e4m3, int head_dim, bool write,
                       hipStream_t stream) {
  switch (dtype) {
    case DType::bf16: return launch_dim<bf16_tag>(args, rows, e4m3, head_dim, write, stream);
    case DType::f16: return launch_dim<f16_tag>(args, rows, e4m3, head_dim, write, stream);
    default: return launch_dim<f32_tag>(args, rows, e4m3, head_dim, write, stream);
  }
}

}  // namespace
}  // namespace cache

hipError_t launch_cache_write(const CacheArgs& args, const TokenRows& rows, DType rows_dtype, bool e4m3,
                              int head_dim, hipStream_t stream) {
  return cache::launch_rows(args, rows, rows_dtype, e4m3, head_dim, true, stream);
}

hipError_t launch_cache_read(const CacheArgs& args, const TokenRows& rows, DType rows_dtype, bool e4m3,
                             int head_dim, hipStream_t stream) {
  return cache::launch_rows(args, rows, rows_dtype, e4m3, head_dim, false, stream);
}

}  // namespace fl

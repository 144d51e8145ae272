// The attention and decode ops as torch's dispatcher sees them, over the C ABI of
// include/flash_lab_hip.h (the reference registers its ops the same way, csrc/bindings.cpp:7-42).
//
// Each op checks its tensors (csrc/common/attn_host.h:18-57, csrc/decode/decode_host.h:18-53 of the
// reference), allocates the outputs and the workspace with torch's caching allocator on the inputs'
// device, and calls the library on the current stream. Nothing here synchronizes or reads seq_lens,
// so the ops can be captured in a HIP graph.
//
// Native because the call is what bounds a short decode: the same steps in Python, with the ctypes
// structures and the dispatcher's Python kernels, took 20 us for a decode of 9 us on the GPU.
//
// The library's functions are bound by address (fl_torch_bind), so that this file links against torch
// only and serves whichever build of the kernels was loaded.
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>
#include <utility>

#include "flash_lab_hip.h"

namespace {

using at::Tensor;
using Pair = std::tuple<Tensor, Tensor>;

struct Library {
  decltype(&fl_attention_plan) attention_plan;
  decltype(&fl_attention_fwd_split) attention_fwd_split;
  decltype(&fl_decode_plan) decode_plan;
  decltype(&fl_decode_schedule) decode_schedule;
  decltype(&fl_decode) decode;
  decltype(&fl_decode_balanced) decode_balanced;
  decltype(&fl_cache_write) cache_write;
  decltype(&fl_cache_read) cache_read;
  decltype(&fl_cached_attention_plan) cached_attention_plan;
  decltype(&fl_cached_attention) cached_attention;
  decltype(&fl_last_error) last_error;
};
Library lib{};

void check(int rc) { TORCH_CHECK(rc == FL_OK, lib.last_error()); }

const char* dtype_name(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    default: return c10::toString(x.scalar_type());
  }
}

int32_t dtype_code(const Tensor& x) {
  return x.scalar_type() == at::kBFloat16 ? FL_DTYPE_BF16 : x.scalar_type() == at::kHalf ? FL_DTYPE_F16 : FL_DTYPE_F32;
}

void check_cuda(const Tensor& x, const char* name) { TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor"); }

void check_rows(const Tensor& x, const char* name) {
  TORCH_CHECK(x.stride(-1) == 1, name, " must be contiguous in its last dimension");
}

int32_t cu_count(const Tensor& x) {
  return at::cuda::getDeviceProperties(x.device().index())->multiProcessorCount;
}

fl_stream_t current_stream(const Tensor& x) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
}

// A size that the library's int32 fields hold.
int32_t size32(int64_t n) {
  TORCH_CHECK(n <= INT32_MAX, "tensor dimension ", n, " is too large");
  return static_cast<int32_t>(n);
}

Pair attention(const Tensor& q, const Tensor& k_in, const Tensor& v_in, bool causal, double softmax_scale) {
  check_cuda(q, "q");
  check_cuda(k_in, "k");
  check_cuda(v_in, "v");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
              "attention_mma_pipelined takes bf16 or fp16");
  TORCH_CHECK(k_in.scalar_type() == q.scalar_type() && v_in.scalar_type() == q.scalar_type(),
              "k and v must have dtype ", dtype_name(q));
  TORCH_CHECK(q.dim() == 4 && k_in.dim() == 4 && v_in.dim() == 4, "q, k, v must be [B, S, H, D]");
  TORCH_CHECK(k_in.sizes() == v_in.sizes(), "k and v must have the same shape");
  TORCH_CHECK(q.size(0) == k_in.size(0) && q.size(3) == k_in.size(3),
              "q and k must agree on batch size and head_dim");
  TORCH_CHECK(q.device() == k_in.device() && q.device() == v_in.device(), "q, k, v on different devices");
  check_rows(q, "q");
  check_rows(k_in, "k");
  check_rows(v_in, "v");
  // The kernels need non-overlapping K and V rows (sequence stride >= head_dim); broadcast or
  // overlapping views, which the reference also accepts, are passed as contiguous copies.
  auto rows = [&](const Tensor& x) { return x.size(1) > 1 && x.stride(1) < x.size(3) ? x.contiguous() : x; };
  const Tensor k = rows(k_in);
  const Tensor v = rows(v_in);
  const c10::DeviceGuard guard(q.device());
  Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));

  fl_attn_params p{};
  p.q = q.const_data_ptr();
  p.k = k.const_data_ptr();
  p.v = v.const_data_ptr();
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.q_batch_stride = q.stride(0), p.q_seq_stride = q.stride(1), p.q_head_stride = q.stride(2);
  p.k_batch_stride = k.stride(0), p.k_seq_stride = k.stride(1), p.k_head_stride = k.stride(2);
  p.v_batch_stride = v.stride(0), p.v_seq_stride = v.stride(1), p.v_head_stride = v.stride(2);
  p.o_batch_stride = o.stride(0), p.o_seq_stride = o.stride(1), p.o_head_stride = o.stride(2);
  p.batch = size32(q.size(0));
  p.seqlen_q = size32(q.size(1));
  p.seqlen_k = size32(k.size(1));
  p.heads = size32(q.size(2));
  p.heads_kv = size32(k.size(2));
  p.head_dim = size32(q.size(3));
  p.causal = causal;
  p.dtype = dtype_code(q);
  p.softmax_scale = softmax_scale;
  const fl_stream_t stream = current_stream(q);
  const int32_t cus = cu_count(q);
  const int rc = lib.attention_fwd_split(&p, 0, cus, nullptr, 0, stream);
  if (rc != FL_ERR_WORKSPACE) {
    check(rc);
    return {o, lse};
  }
  int32_t splits = 0;
  size_t bytes = 0;
  check(lib.attention_plan(&p, 0, cus, &splits, &bytes));
  Tensor workspace = at::empty({static_cast<int64_t>(bytes / sizeof(float))}, lse.options());
  check(lib.attention_fwd_split(&p, splits, cus, workspace.data_ptr<float>(), bytes, stream));
  return {o, lse};
}

Pair decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& seq_lens,
            const Tensor* block_tables, double softmax_scale, int64_t num_splits, bool allow_splits) {
  check_cuda(q, "q");
  check_cuda(k_cache, "k_cache");
  check_cuda(v_cache, "v_cache");
  check_cuda(seq_lens, "seq_lens");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat,
              "decode takes bf16, fp16, or fp32");
  TORCH_CHECK(k_cache.scalar_type() == q.scalar_type() && v_cache.scalar_type() == q.scalar_type(),
              "k_cache and v_cache must have dtype ", dtype_name(q));
  TORCH_CHECK(seq_lens.scalar_type() == at::kInt, "seq_lens must have dtype int32");
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4, "q must be [B, H, D], caches [B, S_max, H_kv, D]");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
  if (block_tables == nullptr) {
    TORCH_CHECK(k_cache.size(0) == q.size(0) && k_cache.size(3) == q.size(2),
                "q and the caches must agree on batch size and head_dim");
  } else {
    check_cuda(*block_tables, "block_tables");
    TORCH_CHECK(block_tables->scalar_type() == at::kInt, "block_tables must have dtype int32");
    TORCH_CHECK(block_tables->dim() == 2 && block_tables->size(0) == q.size(0) && block_tables->size(1) >= 1 &&
                    block_tables->stride(1) == 1,
                "block_tables must be [B, max_blocks] with unit stride in its last dimension");
    TORCH_CHECK(k_cache.size(3) == q.size(2), "q and the caches must agree on head_dim");
    TORCH_CHECK(block_tables->size(1) * k_cache.size(1) <= INT32_MAX,
                "paged cache too long (max_blocks * page_size must fit in int32)");
  }
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == q.size(0), "seq_lens must be [B]");
  TORCH_CHECK(seq_lens.is_contiguous(), "seq_lens must be contiguous");
  check_rows(q, "q");
  check_rows(k_cache, "k_cache");
  check_rows(v_cache, "v_cache");
  TORCH_CHECK(0 <= num_splits && num_splits <= 128, "num_splits must be in [0, 128]");

  const c10::DeviceGuard guard(q.device());
  Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  fl_decode_params p{};
  p.q = q.const_data_ptr();
  p.k_cache = k_cache.const_data_ptr();
  p.v_cache = v_cache.const_data_ptr();
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.seq_lens = seq_lens.const_data_ptr<int32_t>();
  p.q_batch_stride = q.stride(0), p.q_head_stride = q.stride(1);
  p.k_batch_stride = k_cache.stride(0), p.k_seq_stride = k_cache.stride(1), p.k_head_stride = k_cache.stride(2);
  p.v_batch_stride = v_cache.stride(0), p.v_seq_stride = v_cache.stride(1), p.v_head_stride = v_cache.stride(2);
  p.o_batch_stride = o.stride(0), p.o_head_stride = o.stride(1);
  p.batch = size32(q.size(0));
  p.heads = size32(q.size(1));
  p.heads_kv = size32(k_cache.size(2));
  p.head_dim = size32(q.size(2));
  p.max_seqlen = size32(k_cache.size(1));
  p.num_splits = 1;
  p.dtype = dtype_code(q);
  p.softmax_scale = softmax_scale;
  if (block_tables != nullptr) {
    // [num_blocks, page_size, H_kv, D] caches: the batch strides are block strides.
    p.max_seqlen = size32(block_tables->size(1) * k_cache.size(1));
    p.block_tables = block_tables->const_data_ptr<int32_t>();
    p.block_tables_stride = block_tables->stride(0);
    p.page_size = size32(k_cache.size(1));
    p.num_blocks = size32(k_cache.size(0));
  }
  int32_t splits = 0;
  int32_t workgroups = 0;
  if (allow_splits && num_splits == 0) {
    check(lib.decode_schedule(&p, cu_count(q), &splits, &workgroups, &p.workspace_bytes));
  } else {
    check(lib.decode_plan(&p, static_cast<int32_t>(num_splits), allow_splits, cu_count(q), &splits, &p.workspace_bytes));
  }
  p.num_splits = splits;
  Tensor workspace;
  if (p.workspace_bytes > 0) {
    workspace = at::empty({static_cast<int64_t>(p.workspace_bytes / sizeof(float))}, lse.options());
    p.workspace = workspace.data_ptr<float>();
  }
  const fl_stream_t stream = current_stream(q);
  check(workgroups > 0 ? lib.decode_balanced(&p, workgroups, stream) : lib.decode(&p, stream));
  return {o, lse};
}

template <bool kSplits>
Pair decode_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& seq_lens, double scale,
               int64_t num_splits) {
  return decode(q, k, v, seq_lens, nullptr, scale, num_splits, kSplits);
}

template <bool kSplits>
Pair paged_decode_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& seq_lens,
                     const Tensor& block_tables, double scale, int64_t num_splits) {
  return decode(q, k, v, seq_lens, &block_tables, scale, num_splits, kSplits);
}

// ---------------------------------------------------------------------------------------------
// The cache operators: a cache is slabs [B, S_max, H_kv, D] or, with block_tables, a pool of blocks, in the
// tokens' type or in e4m3 codes with scales. No counterpart in the reference.

using OptTensor = std::optional<Tensor>;

int32_t cache_dtype_code(const Tensor& x) {
  return x.scalar_type() == at::kFloat8_e4m3fn ? int32_t{FL_DTYPE_E4M3} : dtype_code(x);
}

// The cache and the call's tokens: `tokens` of them, of B sequences that cu_seqlens parts, or per_seq each
// without it.
fl_kv_cache kv_cache(const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_scales,
                     const OptTensor& v_scales, const Tensor& seq_lens, const OptTensor& cu_seqlens,
                     const OptTensor& block_tables, at::ScalarType dtype, int64_t tokens, int64_t per_seq) {
  check_cuda(k_cache, "k_cache");
  check_cuda(v_cache, "v_cache");
  check_cuda(seq_lens, "seq_lens");
  auto same_device = [&](const Tensor& x, const char* name) {
    TORCH_CHECK(x.device() == k_cache.device(), name, " is on ", x.device(), ", k_cache on ", k_cache.device());
  };
  same_device(v_cache, "v_cache");
  same_device(seq_lens, "seq_lens");
  TORCH_CHECK(k_cache.dim() == 4, "caches must be [B, S_max, H_kv, D] or [num_blocks, page_size, H_kv, D]");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
  TORCH_CHECK(k_cache.scalar_type() == v_cache.scalar_type(), "k_cache and v_cache must have the same dtype");
  check_rows(k_cache, "k_cache");
  check_rows(v_cache, "v_cache");
  const bool e4m3 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(e4m3 || k_cache.scalar_type() == dtype, "the caches must have the tokens' dtype, or float8_e4m3fn");
  TORCH_CHECK(e4m3 == k_scales.has_value() && e4m3 == v_scales.has_value(),
              "k_scales and v_scales go with float8_e4m3fn caches, and with no other");
  TORCH_CHECK(seq_lens.scalar_type() == at::kInt && seq_lens.dim() == 1 && seq_lens.is_contiguous() &&
                  seq_lens.size(0) >= 1,
              "seq_lens must be a contiguous int32 [B]");
  fl_kv_cache c{};
  c.k = k_cache.data_ptr();
  c.v = v_cache.data_ptr();
  c.seq_lens = seq_lens.const_data_ptr<int32_t>();
  c.k_batch_stride = k_cache.stride(0), c.k_seq_stride = k_cache.stride(1), c.k_head_stride = k_cache.stride(2);
  c.v_batch_stride = v_cache.stride(0), c.v_seq_stride = v_cache.stride(1), c.v_head_stride = v_cache.stride(2);
  c.batch = size32(seq_lens.size(0));
  c.outer = size32(k_cache.size(0));
  c.rows = size32(k_cache.size(1));
  c.heads_kv = size32(k_cache.size(2));
  c.head_dim = size32(k_cache.size(3));
  c.dtype = cache_dtype_code(k_cache);
  c.tokens = size32(tokens);
  c.tokens_per_seq = size32(per_seq);
  if (e4m3) {
    for (const Tensor* s : {&*k_scales, &*v_scales}) {
      check_cuda(*s, "k_scales and v_scales");
      same_device(*s, "a scale tensor");
      TORCH_CHECK(s->scalar_type() == at::kByte && s->sizes() == k_cache.sizes().slice(0, 3),
                  "k_scales and v_scales must be uint8 of the caches' shape without D");
    }
    c.k_scales = static_cast<uint8_t*>(k_scales->data_ptr());
    c.v_scales = static_cast<uint8_t*>(v_scales->data_ptr());
    c.ks_batch_stride = k_scales->stride(0), c.ks_seq_stride = k_scales->stride(1);
    c.vs_batch_stride = v_scales->stride(0), c.vs_seq_stride = v_scales->stride(1);
    c.ks_head_stride = k_scales->stride(2), c.vs_head_stride = v_scales->stride(2);
  }
  if (cu_seqlens) {
    check_cuda(*cu_seqlens, "cu_seqlens");
    same_device(*cu_seqlens, "cu_seqlens");
    TORCH_CHECK(cu_seqlens->scalar_type() == at::kInt && cu_seqlens->dim() == 1 && cu_seqlens->is_contiguous() &&
                    cu_seqlens->size(0) == seq_lens.size(0) + 1,
                "cu_seqlens must be a contiguous int32 [B + 1]");
    c.cu_seqlens = cu_seqlens->const_data_ptr<int32_t>();
  }
  if (block_tables) {
    check_cuda(*block_tables, "block_tables");
    same_device(*block_tables, "block_tables");
    TORCH_CHECK(block_tables->scalar_type() == at::kInt && block_tables->dim() == 2 &&
                    block_tables->size(0) == seq_lens.size(0) && block_tables->size(1) >= 1 &&
                    block_tables->stride(1) == 1,
                "block_tables must be int32 [B, max_blocks] with unit stride in its last dimension");
    c.block_tables = block_tables->const_data_ptr<int32_t>();
    c.block_tables_stride = block_tables->stride(0);
    c.max_blocks = size32(block_tables->size(1));
  } else {
    TORCH_CHECK(k_cache.size(0) == seq_lens.size(0), "batch size mismatch: the cache has ", k_cache.size(0),
                ", seq_lens ", seq_lens.size(0));
  }
  return c;
}

// Tokens in all and per sequence of a tensor [tokens, H, D], or [B, S, H, D] without cu_seqlens.
std::pair<int64_t, int64_t> token_counts(const Tensor& x, const char* name, const Tensor& seq_lens,
                                         const OptTensor& cu_seqlens) {
  check_cuda(x, name);
  check_rows(x, name);
  if (cu_seqlens) {
    TORCH_CHECK(x.dim() == 3, name, " must be [tokens, H, D] with cu_seqlens");
    return {x.size(0), 0};
  }
  TORCH_CHECK(x.dim() == 4 && seq_lens.dim() == 1 && x.size(0) == seq_lens.size(0), name,
              " must be [B, S, H, D] without cu_seqlens");
  return {x.size(0) * x.size(1), x.size(1)};
}

// (Ragged tensors have no batch stride.)
int64_t batch_stride(const Tensor& x) { return x.dim() == 4 ? x.stride(0) : 0; }

fl_token_rows token_rows(const Tensor& k, const Tensor& v, const Tensor& k_cache) {
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == v.device(),
              "k and v must have the same shape, dtype and device");
  TORCH_CHECK(k.device() == k_cache.device(), "k is on ", k.device(), ", k_cache on ", k_cache.device());
  TORCH_CHECK(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf || k.scalar_type() == at::kFloat,
              "token rows are bf16, fp16, or fp32");
  TORCH_CHECK(k_cache.dim() == 4 && k.size(-2) == k_cache.size(2) && k.size(-1) == k_cache.size(3),
              "token rows and caches must agree on KV heads and head_dim");
  fl_token_rows r{};
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  r.k_batch_stride = batch_stride(k), r.k_seq_stride = k.stride(-3), r.k_head_stride = k.stride(-2);
  r.v_batch_stride = batch_stride(v), r.v_seq_stride = v.stride(-3), r.v_head_stride = v.stride(-2);
  r.dtype = dtype_code(k);
  return r;
}

void write_cache(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache,
                 const OptTensor& k_scales, const OptTensor& v_scales, const Tensor& seq_lens,
                 const OptTensor& cu_seqlens, const OptTensor& block_tables) {
  const auto [tokens, per_seq] = token_counts(k, "k", seq_lens, cu_seqlens);
  token_counts(v, "v", seq_lens, cu_seqlens);
  const fl_token_rows rows = token_rows(k, v, k_cache);
  const fl_kv_cache c = kv_cache(k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables,
                                 k.scalar_type(), tokens, per_seq);
  const c10::DeviceGuard guard(k_cache.device());
  check(lib.cache_write(&c, &rows, current_stream(k_cache)));
}

Pair read_cache(const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_scales, const OptTensor& v_scales,
                const Tensor& seq_lens, const Tensor& cu_seqlens, const OptTensor& block_tables, int64_t num_tokens,
                at::ScalarType dtype) {
  TORCH_CHECK(num_tokens >= 0, "num_tokens must not be negative");
  const fl_kv_cache c = kv_cache(k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables, dtype,
                                 num_tokens, 0);
  const c10::DeviceGuard guard(k_cache.device());
  const auto options = k_cache.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous);
  Tensor k = at::empty({num_tokens, k_cache.size(2), k_cache.size(3)}, options);
  Tensor v = at::empty_like(k);
  const fl_token_rows rows = token_rows(k, v, k_cache);
  check(lib.cache_read(&c, &rows, current_stream(k_cache)));
  return {k, v};
}

Pair attention_cached(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_scales,
                      const OptTensor& v_scales, const Tensor& seq_lens, const OptTensor& cu_seqlens,
                      const OptTensor& block_tables, bool causal, double softmax_scale, int64_t num_splits) {
  const auto [tokens, per_seq] = token_counts(q, "q", seq_lens, cu_seqlens);
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "attention_cached takes bf16 or fp16");
  TORCH_CHECK(q.device() == k_cache.device(), "q is on ", q.device(), ", k_cache on ", k_cache.device());
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(3) == q.size(-1), "q and the caches must agree on head_dim");
  TORCH_CHECK(0 <= num_splits && num_splits <= 128, "num_splits must be in [0, 128]");
  const c10::DeviceGuard guard(q.device());
  Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor lse = at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
  fl_cached_attn_params p{};
  p.cache = kv_cache(k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables, q.scalar_type(), tokens,
                     per_seq);
  p.q = q.const_data_ptr();
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.q_batch_stride = batch_stride(q), p.q_seq_stride = q.stride(-3), p.q_head_stride = q.stride(-2);
  p.o_batch_stride = batch_stride(o), p.o_seq_stride = o.stride(-3), p.o_head_stride = o.stride(-2);
  p.heads = size32(q.size(-2));
  p.causal = causal;
  p.dtype = dtype_code(q);
  p.num_splits = static_cast<int32_t>(num_splits);
  p.softmax_scale = softmax_scale;
  const int32_t cus = cu_count(q);
  check(lib.cached_attention_plan(&p, cus, &p.workspace_bytes));
  Tensor workspace;
  if (p.workspace_bytes > 0) {
    workspace = at::empty({static_cast<int64_t>(p.workspace_bytes / sizeof(float))}, lse.options());
    p.workspace = workspace.data_ptr<float>();
  }
  check(lib.cached_attention(&p, cus, current_stream(q)));
  return {o, lse};
}

// The ops have no gradient. With inputs that require one, the outputs are part of the graph and a
// backward through them raises; otherwise the call goes straight on below autograd.
template <typename... Args>
struct NoGradient {
  using Op = c10::TypedOperatorHandle<Pair(Args...)>;
  struct Node : torch::autograd::Function<Node> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Op& op,
                                                  const std::string& name, Args... args) {
      ctx->saved_data["op"] = name;
      at::AutoDispatchBelowADInplaceOrView below;
      auto [o, lse] = op.call(args...);
      return {o, lse};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list) {
      TORCH_CHECK(false, "Trying to backward through flash_lab.", ctx->saved_data["op"].toStringRef(),
                  ".default but no autograd formula was registered. Please use register_autograd to add one.");
    }
  };
  static bool requires_grad(const Tensor& x) { return x.requires_grad(); }
  static bool requires_grad(const OptTensor& x) { return x && x->requires_grad(); }
  template <typename T>
  static bool requires_grad(const T&) {
    return false;
  }
  static Pair call(const char* name, const Op& op, Args... args) {
    if (at::GradMode::is_enabled() && (requires_grad(args) || ...)) {
      auto outputs = Node::apply(op, std::string(name), args...);
      return {outputs[0], outputs[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(args...);
  }
};

using Prefill = NoGradient<const Tensor&, const Tensor&, const Tensor&, bool, double>;
using Decode = NoGradient<const Tensor&, const Tensor&, const Tensor&, const Tensor&, double, int64_t>;
using PagedDecode =
    NoGradient<const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, double, int64_t>;

#define FL_AUTOGRAD(kind, op_name, params, args)                                                        \
  Pair op_name##_autograd params {                                                                       \
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("flash_lab::" #op_name, "")    \
                               .typed<Pair params>();                                                    \
    return kind::call args;                                                                              \
  }
FL_AUTOGRAD(Prefill, attention_mma_pipelined,
            (const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale),
            ("attention_mma_pipelined", op, q, k, v, causal, scale))
FL_AUTOGRAD(Prefill, attention_mma, (const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale),
            ("attention_mma", op, q, k, v, causal, scale))
#define FL_DECODE_AUTOGRAD(name)                                                                         \
  FL_AUTOGRAD(Decode, name,                                                                              \
              (const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens, double scale, int64_t n), \
              (#name, op, q, k, v, lens, scale, n))
#define FL_PAGED_AUTOGRAD(name)                                                                          \
  FL_AUTOGRAD(PagedDecode, name,                                                                         \
              (const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens, const Tensor& tables, \
               double scale, int64_t n),                                                                 \
              (#name, op, q, k, v, lens, tables, scale, n))
FL_DECODE_AUTOGRAD(decode_splitkv)
FL_DECODE_AUTOGRAD(decode_inplace)
FL_PAGED_AUTOGRAD(decode_splitkv_paged)
FL_PAGED_AUTOGRAD(decode_inplace_paged)

using CachedAttention = NoGradient<const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                   const Tensor&, const OptTensor&, const OptTensor&, bool, double, int64_t>;
FL_AUTOGRAD(CachedAttention, attention_cached,
            (const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs,
             const Tensor& lens, const OptTensor& cu, const OptTensor& tables, bool causal, double scale, int64_t n),
            ("attention_cached", op, q, k, v, ks, vs, lens, cu, tables, causal, scale, n))
using ReadCache = NoGradient<const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&,
                             const Tensor&, const OptTensor&, int64_t, at::ScalarType>;
FL_AUTOGRAD(ReadCache, read_cache,
            (const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs, const Tensor& lens,
             const Tensor& cu, const OptTensor& tables, int64_t n, at::ScalarType dtype),
            ("read_cache", op, k, v, ks, vs, lens, cu, tables, n, dtype))

// A write gives nothing that a backward could start from, so rows that require a gradient would lose it
// without a word: they are refused.
void write_cache_autograd(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache,
                          const OptTensor& k_scales, const OptTensor& v_scales, const Tensor& seq_lens,
                          const OptTensor& cu_seqlens, const OptTensor& block_tables) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("flash_lab::write_cache", "")
                             .typed<decltype(write_cache)>();
  TORCH_CHECK(!at::GradMode::is_enabled() || !(k.requires_grad() || v.requires_grad() || k_cache.requires_grad() ||
                                               v_cache.requires_grad()),
              "write_cache has no gradient: pass detached rows and caches, or call it under torch.no_grad()");
  {
    at::AutoDispatchBelowADInplaceOrView below;
    op.call(k, v, k_cache, v_cache, k_scales, v_scales, seq_lens, cu_seqlens, block_tables);
  }
  // A graph that saved one of these for its backward then says that it was changed.
  auto changed = [](const Tensor& x) {
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
  };
  changed(k_cache);
  changed(v_cache);
  if (k_scales) changed(*k_scales);
  if (v_scales) changed(*v_scales);
}

}  // namespace

// The reference's schemas, verbatim (csrc/bindings.cpp:9-41); the paged forms, which the reference
// lacks (its kernels reject paged caches), take the block tables after seq_lens.
TORCH_LIBRARY_FRAGMENT(flash_lab, m) {
  const char* prefill = "(Tensor q, Tensor k, Tensor v, bool causal, float softmax_scale) -> (Tensor, Tensor)";
  const char* decode = "(Tensor q, Tensor k_cache, Tensor v_cache, Tensor seq_lens, float softmax_scale,"
                       " int num_splits) -> (Tensor, Tensor)";
  const char* paged = "(Tensor q, Tensor k_cache, Tensor v_cache, Tensor seq_lens, Tensor block_tables,"
                      " float softmax_scale, int num_splits) -> (Tensor, Tensor)";
  auto def = [&](const char* name, const char* schema) {
    m.def(torch::schema((std::string(name) + schema).c_str()), {at::Tag::pt2_compliant_tag});
  };
  def("attention_mma_pipelined", prefill);
  def("attention_mma", prefill);
  def("decode_splitkv", decode);
  def("decode_inplace", decode);
  def("decode_splitkv_paged", paged);
  def("decode_inplace_paged", paged);
  def("attention_cached",
      "(Tensor q, Tensor k_cache, Tensor v_cache, Tensor? k_scales, Tensor? v_scales, Tensor seq_lens,"
      " Tensor? cu_seqlens, Tensor? block_tables, bool causal, float softmax_scale, int num_splits)"
      " -> (Tensor, Tensor)");
  def("write_cache",
      "(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scales, Tensor(d!)? v_scales,"
      " Tensor seq_lens, Tensor? cu_seqlens, Tensor? block_tables) -> ()");
  def("read_cache",
      "(Tensor k_cache, Tensor v_cache, Tensor? k_scales, Tensor? v_scales, Tensor seq_lens, Tensor cu_seqlens,"
      " Tensor? block_tables, int num_tokens, ScalarType dtype) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(flash_lab, CUDA, m) {
  m.impl("attention_mma_pipelined", &attention);
  m.impl("attention_mma", &attention);
  m.impl("decode_splitkv", &decode_op<true>);
  m.impl("decode_inplace", &decode_op<false>);
  m.impl("decode_splitkv_paged", &paged_decode_op<true>);
  m.impl("decode_inplace_paged", &paged_decode_op<false>);
  m.impl("attention_cached", &attention_cached);
  m.impl("write_cache", &write_cache);
  m.impl("read_cache", &read_cache);
}

TORCH_LIBRARY_IMPL(flash_lab, Autograd, m) {
  m.impl("attention_mma_pipelined", &attention_mma_pipelined_autograd);
  m.impl("attention_mma", &attention_mma_autograd);
  m.impl("decode_splitkv", &decode_splitkv_autograd);
  m.impl("decode_inplace", &decode_inplace_autograd);
  m.impl("decode_splitkv_paged", &decode_splitkv_paged_autograd);
  m.impl("decode_inplace_paged", &decode_inplace_paged_autograd);
  m.impl("attention_cached", &attention_cached_autograd);
  m.impl("write_cache", &write_cache_autograd);
  m.impl("read_cache", &read_cache_autograd);
}

// The addresses of the library's functions, in this order; once, before the first call of an op.
extern "C" void fl_torch_bind(void* attention_plan, void* attention_fwd_split, void* decode_plan,
                              void* decode_schedule, void* decode, void* decode_balanced, void* cache_write,
                              void* cache_read, void* cached_attention_plan, void* cached_attention,
                              void* last_error) {
  lib.attention_plan = reinterpret_cast<decltype(lib.attention_plan)>(attention_plan);
  lib.attention_fwd_split = reinterpret_cast<decltype(lib.attention_fwd_split)>(attention_fwd_split);
  lib.decode_plan = reinterpret_cast<decltype(lib.decode_plan)>(decode_plan);
  lib.decode_schedule = reinterpret_cast<decltype(lib.decode_schedule)>(decode_schedule);
  lib.decode = reinterpret_cast<decltype(lib.decode)>(decode);
  lib.decode_balanced = reinterpret_cast<decltype(lib.decode_balanced)>(decode_balanced);
  lib.cache_write = reinterpret_cast<decltype(lib.cache_write)>(cache_write);
  lib.cache_read = reinterpret_cast<decltype(lib.cache_read)>(cache_read);
  lib.cached_attention_plan = reinterpret_cast<decltype(lib.cached_attention_plan)>(cached_attention_plan);
  lib.cached_attention = reinterpret_cast<decltype(lib.cached_attention)>(cached_attention);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(last_error);
}

// torch_op.cpp — the attention operator and the paged-cache operators as torch
// custom ops over the C ABI.
//
// torch.ops.b200.fused_attention keeps the argument meaning, checks and
// exception types of the reference operator triton_fused_attention
// (model/triton_fused_attention.py:1877-1891; _validate_inputs :1217-1253):
// contract violations raise ValueError / TypeError (TORCH_CHECK_VALUE /
// TORCH_CHECK_TYPE), inputs outside the kernel envelope raise ValueError
// (there is no fallback), a launch refused because the error word holds an
// earlier launch's report raises RuntimeError with the "b200 device error"
// prefix.  It validates, allocates the output and launches b200_attn_fwd on the
// current stream in one C++ call, so a call costs no Python-side argument
// packing; the kernel, its tensor maps and its checks are the C library's.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cmath>
#include <map>
#include <mutex>
#include <optional>
#include <utility>

#include "b200_attn.h"
#include "b200_paged.h"

namespace {

const char* dtype_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "bfloat16";
    case at::kHalf: return "float16";
    case at::kFloat: return "float32";
    default: return c10::toString(t);
  }
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return B200_ATTN_DTYPE_BF16;
    case at::kHalf: return B200_ATTN_DTYPE_FP16;
    case at::kFloat: return B200_ATTN_DTYPE_FP32;
    default: return -1;
  }
}

void fill_strides(int64_t dst[3], const at::Tensor& t) {
  dst[0] = t.stride(0);
  dst[1] = t.stride(1);
  dst[2] = t.stride(2);
}

at::Tensor fused_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                           const std::optional<at::Tensor>& valid_token_mask, bool causal,
                           std::optional<double> scale, bool output_bshd,
                           bool zero_masked_queries, const std::optional<at::Tensor>& out,
                           int64_t error_word) {
  // the reference's _validate_inputs (model/triton_fused_attention.py:1217-1253)
  TORCH_CHECK_VALUE(q.dim() == 4, "q must have shape [B, H, S, D], got ", q.sizes());
  TORCH_CHECK_VALUE(k.sizes() == q.sizes() && v.sizes() == q.sizes(),
                    "q, k, and v must have the same [B, H, S, D] shape; got q=", q.sizes(),
                    ", k=", k.sizes(), ", v=", v.sizes());
  TORCH_CHECK_VALUE(q.device() == k.device() && q.device() == v.device(),
                    "q, k, and v must be on the same device");
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                   "q, k, and v must have the same dtype");
  TORCH_CHECK_TYPE(at::isFloatingType(q.scalar_type()),
                   "q/k/v must use a floating-point dtype, got ", q.scalar_type());
  const int64_t B = q.size(0), H = q.size(1), S = q.size(2), D = q.size(3);
  TORCH_CHECK_VALUE(S > 0 && D > 0, "sequence length and head dimension must be positive");
  const at::Tensor* mask = valid_token_mask.has_value() ? &valid_token_mask.value() : nullptr;
  if (mask) {
    TORCH_CHECK_VALUE(mask->dim() == 2 && mask->size(0) == B && mask->size(1) == S,
                      "valid_token_mask must have shape (", B, ", ", S, "), got ", mask->sizes());
    TORCH_CHECK_TYPE(mask->scalar_type() == at::kBool, "valid_token_mask must have dtype torch.bool");
    TORCH_CHECK_VALUE(mask->device() == q.device(),
                      "valid_token_mask and q must be on the same device");
  }
  const double sc = scale.has_value() ? scale.value() : std::pow(static_cast<double>(D), -0.5);
  TORCH_CHECK_VALUE(sc > 0.0, "scale must be positive");
  // the kernel envelope: no fallback, unsupported inputs raise
  TORCH_CHECK_VALUE(q.is_cuda(), "unsupported sm_100a attention invocation: inputs must be CUDA tensors");
  const int32_t dt = dtype_code(q.scalar_type());
  TORCH_CHECK_VALUE(dt >= 0, "unsupported sm_100a attention invocation: dtype ",
                    dtype_name(q.scalar_type()),
                    " is outside the kernel envelope (bfloat16, float16, float32)");
  TORCH_CHECK_VALUE(b200_attn_query(dt, D, causal ? 1 : 0, mask ? 1 : 0) == 1,
                    "unsupported sm_100a attention invocation: head_dim ", D,
                    " is outside the kernel envelope for ", dtype_name(q.scalar_type()),
                    " (multiples of 8 up to ", dt == B200_ATTN_DTYPE_FP32 ? 64 : 128, ")");
  TORCH_CHECK_VALUE(q.stride(3) == 1 && k.stride(3) == 1 && v.stride(3) == 1,
                    "unsupported sm_100a attention invocation: q/k/v must have a contiguous last "
                    "dimension");
  TORCH_CHECK_VALUE(!(c10::GradMode::is_enabled() &&
                      (q.requires_grad() || k.requires_grad() || v.requires_grad())),
                    "unsupported sm_100a attention invocation: the kernel is inference-only "
                    "(autograd requested)");
  TORCH_CHECK_VALUE(!zero_masked_queries || mask, "zero_masked_queries requires valid_token_mask");

  const std::vector<int64_t> shape = output_bshd ? std::vector<int64_t>{B, S, H, D}
                                                 : std::vector<int64_t>{B, H, S, D};
  at::Tensor result;
  if (out.has_value()) {
    result = out.value();
    TORCH_CHECK_VALUE(result.sizes() == at::IntArrayRef(shape), "out must have shape ", shape);
  } else {
    result = at::empty(shape, q.options());
  }
  const at::Tensor o = output_bshd ? result.transpose(1, 2) : result;
  TORCH_CHECK_VALUE(result.scalar_type() == q.scalar_type() && result.device() == q.device() &&
                        o.stride(3) == 1,
                    "out must match q's dtype and device with a contiguous last dim");

  b200_attn_fwd_params p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.o = o.data_ptr();
  p.batch = B;
  p.heads = H;
  p.seq_len = S;
  p.head_dim = D;
  fill_strides(p.q_stride, q);
  fill_strides(p.k_stride, k);
  fill_strides(p.v_stride, v);
  fill_strides(p.o_stride, o);
  if (mask) {
    p.key_mask = static_cast<const uint8_t*>(mask->data_ptr());
    p.mask_stride[0] = mask->stride(0);
    p.mask_stride[1] = mask->stride(1);
  }
  p.scale = static_cast<float>(sc);
  p.dtype = dt;
  p.causal = causal ? 1 : 0;
  p.zero_masked_queries = zero_masked_queries ? 1 : 0;
  p.error_word = reinterpret_cast<int32_t*>(static_cast<intptr_t>(error_word));

  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(q.device().index()).stream();
  const int32_t rc = b200_attn_fwd(&p, stream);
  if (rc == B200_ATTN_OK) return result;
  const char* text = b200_attn_error_string(rc);
  TORCH_CHECK_VALUE(rc != B200_ATTN_ERR_INVALID_ARGUMENT && rc != B200_ATTN_ERR_ALIGNMENT,
                    "b200_attn_fwd: ", text);
  TORCH_CHECK_VALUE(rc != B200_ATTN_ERR_UNSUPPORTED, "unsupported sm_100a attention invocation: ",
                    text);
  TORCH_CHECK(rc != B200_ATTN_ERR_TIMEOUT && rc != B200_ATTN_ERR_DEVICE_BOUNDS,
              "b200 device error: b200_attn_fwd refused to launch: ", text);
  TORCH_CHECK(false, "b200_attn_fwd: ", text, " (", b200_attn_last_error_detail(), ")");
}

// ------------------------------------------------------------- paged cache
using OptTensor = std::optional<at::Tensor>;

void raise_code(const char* entry, int32_t rc) {
  if (rc == B200_ATTN_OK) return;
  const char* text = b200_attn_error_string(rc);
  TORCH_CHECK_VALUE(rc != B200_ATTN_ERR_INVALID_ARGUMENT && rc != B200_ATTN_ERR_ALIGNMENT, entry,
                    ": ", text);
  TORCH_CHECK_VALUE(rc != B200_ATTN_ERR_UNSUPPORTED, "unsupported sm_100a invocation (", entry,
                    "): ", text);
  TORCH_CHECK(rc != B200_ATTN_ERR_TIMEOUT && rc != B200_ATTN_ERR_DEVICE_BOUNDS,
              "b200 device error: ", entry, " refused to launch: ", text);
  TORCH_CHECK(false, entry, ": ", text, " (", b200_attn_last_error_detail(), ")");
}

// An int32 tensor of the shape given, contiguous, on `device`.
int32_t* ints(const at::Tensor& t, const char* name, at::IntArrayRef shape, c10::Device device) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must have dtype torch.int32, got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == device, name, " must be on the cache's device");
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
  return static_cast<int32_t*>(t.data_ptr());
}

// The page table, lengths and counts.
b200_cache table_view(const at::Tensor& table, const OptTensor& lens, const OptTensor& refs,
                      int64_t page_size, int64_t error_word) {
  TORCH_CHECK_VALUE(table.dim() == 2, "page_table must have shape [batch, slots], got ",
                    table.sizes());
  TORCH_CHECK_TYPE(table.scalar_type() == at::kInt, "page_table must have dtype torch.int32, got ",
                   table.scalar_type());
  TORCH_CHECK_VALUE(table.is_cuda(), "the paged cache runs on CUDA tensors only");
  TORCH_CHECK_VALUE(table.size(1) <= 1 || table.stride(1) == 1,
                    "page_table must have a contiguous last dimension");
  TORCH_CHECK_VALUE(table.size(0) >= 1 && table.size(0) <= B200_CACHE_MAX_BATCH &&
                        table.size(1) >= 1,
                    "page_table must have 1 to ", B200_CACHE_MAX_BATCH,
                    " sequences and at least one slot, got ", table.sizes());
  TORCH_CHECK_VALUE(page_size >= 1, "page_size must be positive");
  b200_cache c{};
  c.page_table = static_cast<int32_t*>(table.data_ptr());
  c.batch = table.size(0);
  c.slots = table.size(1);
  c.table_stride = table.stride(0);
  if (lens.has_value()) c.seq_lens = ints(*lens, "seq_lens", {c.batch}, table.device());
  c.page_size = page_size;
  if (refs.has_value()) {
    TORCH_CHECK_VALUE(refs->dim() == 1 && refs->size(0) >= 1,
                      "page_refs must have shape [pages], got ", refs->sizes());
    c.pages = refs->size(0);
    c.page_refs = ints(*refs, "page_refs", {c.pages}, table.device());
  }
  c.error_word = reinterpret_cast<int32_t*>(static_cast<intptr_t>(error_word));
  return c;
}

// The whole cache; pools are [layers, pages, kv_heads, page_size, head_dim] or,
// of one layer, [pages, kv_heads, page_size, head_dim].
b200_cache cache_view(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                      const OptTensor& lens, const OptTensor& refs, int64_t error_word) {
  TORCH_CHECK_VALUE(k.dim() == 4 || k.dim() == 5,
                    "k_pages must have shape [(layers,) pages, kv_heads, page_size, head_dim], "
                    "got ", k.sizes());
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "k_pages and v_pages must have the same shape; got ",
                    k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type(),
                   "k_pages and v_pages must have the same dtype");
  const int32_t dt = dtype_code(k.scalar_type());
  TORCH_CHECK_TYPE(dt >= 0, "k_pages must be bfloat16, float16 or float32, got ", k.scalar_type());
  const int64_t d = k.dim() - 4;  // of the page dimension
  b200_cache c = table_view(table, lens, refs, k.size(d + 2), error_word);
  TORCH_CHECK_VALUE(k.device() == table.device() && v.device() == table.device(),
                    "the pools and the page table must be on the same device");
  TORCH_CHECK_VALUE(k.stride(d + 3) == 1 && v.stride(d + 3) == 1,
                    "the pools must have a contiguous last dimension");
  TORCH_CHECK_VALUE(k.numel() > 0, "the pools must not be empty");
  TORCH_CHECK_VALUE(!(c10::GradMode::is_enabled() && (k.requires_grad() || v.requires_grad())),
                    "the paged cache is inference-only (autograd requested)");
  TORCH_CHECK_VALUE(!refs.has_value() || c.pages == k.size(d), "page_refs must have one count for "
                    "each of the ", k.size(d), " pages, got ", c.pages);
  TORCH_CHECK_VALUE(k.size(d + 3) % 8 == 0 && k.size(d + 3) <= 128, "head_dim ", k.size(d + 3),
                    " is outside the kernel envelope (multiples of 8 up to 128)");
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.layers = d ? k.size(0) : 1;
  c.pages = k.size(d);
  c.kv_heads = k.size(d + 1);
  c.head_dim = k.size(d + 3);
  for (int64_t i = 0; i < 4; ++i) {
    c.k_stride[i] = i == 0 && !d ? 0 : k.stride(d + i - 1);
    c.v_stride[i] = i == 0 && !d ? 0 : v.stride(d + i - 1);
  }
  c.dtype = dt;
  return c;
}

cudaStream_t stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

at::Tensor scratch(int64_t bytes, const at::Tensor& like) {
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

void cache_append(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& k,
                  const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens,
                  const OptTensor& counts, int64_t error_word) {
  const b200_cache c = cache_view(k, v, table, lens, std::nullopt, error_word);
  const int64_t d = k.dim() - 4;
  TORCH_CHECK_VALUE(k_new.dim() == k.dim() && v_new.sizes() == k_new.sizes(),
                    "k_new and v_new must have shape [(layers,) batch, kv_heads, tokens, "
                    "head_dim] like the pools; got ", k_new.sizes(), " and ", v_new.sizes());
  TORCH_CHECK_VALUE((!d || k_new.size(0) == c.layers) && k_new.size(d) == c.batch &&
                        k_new.size(d + 1) == c.kv_heads && k_new.size(d + 3) == c.head_dim,
                    "k_new must have shape [(", c.layers, ",) ", c.batch, ", ", c.kv_heads,
                    ", tokens, ", c.head_dim, "], got ", k_new.sizes());
  TORCH_CHECK_TYPE(k_new.scalar_type() == k.scalar_type() && v_new.scalar_type() == k.scalar_type(),
                   "k_new and v_new must have the pools' dtype ", k.scalar_type());
  TORCH_CHECK_VALUE(k_new.device() == k.device() && v_new.device() == k.device(),
                    "k_new and v_new must be on the cache's device");
  TORCH_CHECK_VALUE(k_new.stride(d + 3) == 1 && v_new.stride(d + 3) == 1,
                    "k_new and v_new must have a contiguous last dimension");
  TORCH_CHECK_VALUE(!(c10::GradMode::is_enabled() &&
                      (k_new.requires_grad() || v_new.requires_grad())),
                    "the paged cache is inference-only (autograd requested)");
  b200_cache_rows r{};
  r.k = k_new.data_ptr();
  r.v = v_new.data_ptr();
  r.tokens = k_new.size(d + 2);
  for (int64_t i = 0; i < 4; ++i) {
    r.k_stride[i] = i == 0 && !d ? 0 : k_new.stride(d + i - 1);
    r.v_stride[i] = i == 0 && !d ? 0 : v_new.stride(d + i - 1);
  }
  if (counts.has_value()) r.counts = ints(*counts, "draft_lens", {c.batch}, k.device());
  if (r.tokens == 0) return;
  raise_code("b200_cache_append", b200_cache_append(&c, &r, stream_of(k)));
}

at::Tensor cache_accept(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                        const at::Tensor& lens, const at::Tensor& paths, const at::Tensor& counts,
                        int64_t error_word) {
  const b200_cache c = cache_view(k, v, table, lens, std::nullopt, error_word);
  TORCH_CHECK_VALUE(paths.dim() == 2 && paths.size(0) == c.batch && paths.size(1) >= 1,
                    "paths must have shape [", c.batch, ", width], got ", paths.sizes());
  const int32_t* p = ints(paths, "paths", paths.sizes(), k.device());
  const int32_t* n = ints(counts, "counts", {c.batch}, k.device());
  at::Tensor out = at::empty_like(lens);
  raise_code("b200_cache_accept",
             b200_cache_accept(&c, p, paths.size(1), paths.size(1), n,
                               static_cast<int32_t*>(out.data_ptr()), stream_of(k)));
  return out;
}

at::Tensor cache_reserve(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                         const at::Tensor& lens, const at::Tensor& refs, const OptTensor& tokens,
                         int64_t uniform, int64_t error_word) {
  const b200_cache c = cache_view(k, v, table, lens, refs, error_word);
  TORCH_CHECK_VALUE(tokens.has_value() || (uniform >= 0 && uniform <= 0x3fffffff),
                    "tokens must not be negative");
  const int32_t* n = tokens.has_value() ? ints(*tokens, "tokens", {c.batch}, k.device()) : nullptr;
  at::Tensor status = at::empty({1}, lens.options());
  const int64_t bytes = b200_cache_workspace_bytes(&c);
  at::Tensor ws = scratch(bytes, k);
  raise_code("b200_cache_reserve",
             b200_cache_reserve(&c, n, uniform, static_cast<int32_t*>(status.data_ptr()),
                                ws.data_ptr(), bytes, stream_of(k)));
  return status;
}

void cache_fork(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& refs,
                const at::Tensor& src, const at::Tensor& dst, int64_t page_size,
                int64_t error_word) {
  const b200_cache c = table_view(table, lens, refs, page_size, error_word);
  TORCH_CHECK_VALUE(src.dim() == 1 && src.size(0) <= c.batch,
                    "src must name at most one sequence for each of the batch, got ", src.sizes());
  const int32_t* s = ints(src, "src", src.sizes(), table.device());
  const int32_t* d = ints(dst, "dst", src.sizes(), table.device());
  raise_code("b200_cache_fork", b200_cache_fork(&c, s, d, src.size(0), stream_of(table)));
}

void cache_free(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& refs,
                const at::Tensor& rows, int64_t error_word) {
  const b200_cache c = table_view(table, lens, refs, 1, error_word);
  TORCH_CHECK_VALUE(rows.dim() == 1, "rows must be one-dimensional, got ", rows.sizes());
  const int32_t* r = ints(rows, "rows", rows.sizes(), table.device());
  raise_code("b200_cache_free", b200_cache_free(&c, r, rows.size(0), stream_of(table)));
}

at::Tensor cache_compact(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                         const at::Tensor& refs, int64_t error_word) {
  const b200_cache c = cache_view(k, v, table, std::nullopt, refs, error_word);
  at::Tensor live = at::empty({1}, refs.options());
  const int64_t bytes = b200_cache_workspace_bytes(&c);
  at::Tensor ws = scratch(bytes, k);
  raise_code("b200_cache_compact",
             b200_cache_compact(&c, static_cast<int32_t*>(live.data_ptr()), ws.data_ptr(), bytes,
                                stream_of(k)));
  return live;
}

// Zeroed counters of a stream's calls (b200_tree_attn_params::counters), kept for the
// process.  None while a graph is captured: a replay may run beside calls on the stream
// that captured it.
int32_t* counters_of(cudaStream_t stream, const at::Tensor& like) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &status) != cudaSuccess ||
      status != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    return nullptr;
  }
  static std::mutex mu;
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();
  std::lock_guard<std::mutex> lock(mu);
  at::Tensor& t = (*kept)[{like.device().index(), stream}];
  if (!t.defined()) {
    const c10::InferenceMode off(false);
    t = at::zeros({B200_TREE_ATTN_COUNTERS}, like.options().dtype(at::kInt));
  }
  return static_cast<int32_t*>(t.data_ptr());
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                          const at::Tensor& table, const at::Tensor& lens, const OptTensor& mask,
                          const OptTensor& draft_lens, std::optional<double> scale,
                          bool output_bshd, const OptTensor& out, int64_t error_word) {
  TORCH_CHECK_VALUE(q.dim() == 4, "q must have shape [B, H, T, D], got ", q.sizes());
  TORCH_CHECK_VALUE(k.dim() == 4, "k_pages must be one layer's pool [pages, kv_heads, page_size, "
                    "head_dim], got ", k.sizes());
  b200_tree_attn_params p{};
  p.cache = cache_view(k, v, table, lens, std::nullopt, error_word);
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  TORCH_CHECK_VALUE(B == p.cache.batch, "q has ", B, " sequences, page_table ", p.cache.batch);
  TORCH_CHECK_VALUE(D == p.cache.head_dim, "q has head_dim ", D, ", the pools ", p.cache.head_dim);
  TORCH_CHECK_VALUE(H >= 1 && H % p.cache.kv_heads == 0, "q's heads (", H,
                    ") must be a multiple of the pools' (", p.cache.kv_heads, ")");
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type(), "q must have the pools' dtype ",
                   k.scalar_type(), ", got ", q.scalar_type());
  TORCH_CHECK_VALUE(q.device() == k.device(), "q must be on the cache's device");
  TORCH_CHECK_VALUE(q.stride(3) == 1, "q must have a contiguous last dimension");
  TORCH_CHECK_VALUE(!(c10::GradMode::is_enabled() && q.requires_grad()),
                    "b200_tree_attention is inference-only (autograd requested)");
  const double sc = scale.has_value() ? scale.value() : std::pow(static_cast<double>(D), -0.5);
  TORCH_CHECK_VALUE(sc > 0.0, "scale must be positive");
  if (mask.has_value()) {
    TORCH_CHECK_TYPE(mask->scalar_type() == at::kBool, "tree_mask must have dtype torch.bool");
    TORCH_CHECK_VALUE(mask->device() == q.device(), "tree_mask must be on q's device");
    const bool shared = mask->dim() == 2;
    TORCH_CHECK_VALUE((shared || (mask->dim() == 3 && mask->size(0) == B)) &&
                          mask->size(-2) == T && mask->size(-1) == T,
                      "tree_mask must have shape [", T, ", ", T, "] or [", B, ", ", T, ", ", T,
                      "], got ", mask->sizes());
    p.mask = static_cast<const uint8_t*>(mask->data_ptr());
    p.mask_stride[0] = shared ? 0 : mask->stride(0);
    p.mask_stride[1] = mask->stride(-2);
    p.mask_stride[2] = mask->stride(-1);
  }
  if (draft_lens.has_value())
    p.draft_lens = ints(*draft_lens, "draft_lens", {B}, q.device());
  const std::vector<int64_t> shape = output_bshd ? std::vector<int64_t>{B, T, H, D}
                                                 : std::vector<int64_t>{B, H, T, D};
  at::Tensor result;
  if (out.has_value()) {
    result = out.value();
    TORCH_CHECK_VALUE(result.sizes() == at::IntArrayRef(shape), "out must have shape ", shape);
    TORCH_CHECK_VALUE(result.scalar_type() == q.scalar_type() && result.device() == q.device() &&
                          result.stride(3) == 1,
                      "out must match q's dtype and device with a contiguous last dim");
  } else {
    result = at::empty(shape, q.options());
  }
  if (T == 0) return result;
  const at::Tensor o = output_bshd ? result.transpose(1, 2) : result;
  p.q = q.data_ptr();
  p.o = o.data_ptr();
  p.heads = H;
  p.tokens = T;
  fill_strides(p.q_stride, q);
  fill_strides(p.o_stride, o);
  p.scale = static_cast<float>(sc);
  p.workspace_bytes = b200_tree_attn_workspace_bytes(&p);
  at::Tensor ws;
  if (p.workspace_bytes > 0) {
    ws = scratch(p.workspace_bytes, q);
    p.workspace = ws.data_ptr();
  }
  const cudaStream_t stream = stream_of(q);
  p.counters = counters_of(stream, q);
  raise_code("b200_tree_attn_fwd", b200_tree_attn_fwd(&p, stream));
  return result;
}

}  // namespace

TORCH_LIBRARY(b200, m) {
  m.def(
      "cache_append(Tensor k_new, Tensor v_new, Tensor(a!) k_pages, Tensor(b!) v_pages, "
      "Tensor page_table, Tensor seq_lens, Tensor? draft_lens, int error_word) -> ()",
      &cache_append);
  m.def(
      "cache_accept(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor seq_lens, "
      "Tensor paths, Tensor counts, int error_word) -> Tensor",
      &cache_accept);
  m.def(
      "cache_reserve(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!) page_table, "
      "Tensor seq_lens, Tensor(d!) page_refs, Tensor? tokens, int uniform, int error_word) -> "
      "Tensor",
      &cache_reserve);
  m.def(
      "cache_fork(Tensor(a!) page_table, Tensor(b!) seq_lens, Tensor(c!) page_refs, Tensor src, "
      "Tensor dst, int page_size, int error_word) -> ()",
      &cache_fork);
  m.def(
      "cache_free(Tensor(a!) page_table, Tensor(b!) seq_lens, Tensor(c!) page_refs, Tensor rows, "
      "int error_word) -> ()",
      &cache_free);
  m.def(
      "cache_compact(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!) page_table, "
      "Tensor(d!) page_refs, int error_word) -> Tensor",
      &cache_compact);
  m.def(
      "tree_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, "
      "Tensor seq_lens, Tensor? tree_mask, Tensor? draft_lens, float? scale, bool output_bshd, "
      "Tensor(a!)? out, int error_word) -> Tensor",
      &tree_attention);
  m.def(
      "fused_attention(Tensor q, Tensor k, Tensor v, Tensor? valid_token_mask, bool causal, "
      "float? scale, bool output_bshd, bool zero_masked_queries, Tensor? out, int error_word) "
      "-> Tensor",
      &fused_attention);
}

// torch_op.cpp — the attention operator, the paged-cache operators and the check of
// drafted tokens as torch custom ops over the C ABI.
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
#include <tuple>
#include <utility>
#include <vector>

#include "b200_attn.h"
#include "b200_cache4.h"
#include "b200_paged.h"
#include "b200_verify.h"

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
// of one layer, [pages, kv_heads, page_size, head_dim].  Pools of uint8 hold rows of 4-bit numbers
// (b200_cache4.h) and are described as 16-bit ones of half as many elements.
b200_cache cache_view(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                      const OptTensor& lens, const OptTensor& refs, int64_t error_word) {
  TORCH_CHECK_VALUE(k.dim() == 4 || k.dim() == 5,
                    "k_pages must have shape [(layers,) pages, kv_heads, page_size, head_dim], "
                    "got ", k.sizes());
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "k_pages and v_pages must have the same shape; got ",
                    k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type(),
                   "k_pages and v_pages must have the same dtype");
  const bool coded = k.scalar_type() == at::kByte;
  const int32_t dt = coded ? B200_ATTN_DTYPE_BF16 : dtype_code(k.scalar_type());
  TORCH_CHECK_TYPE(dt >= 0, "k_pages must be bfloat16, float16 or float32, or uint8 for a 4-bit "
                   "cache, got ", k.scalar_type());
  const int64_t d = k.dim() - 4;  // of the page dimension
  const int64_t each = coded ? 2 : 1;  // elements of the pools to one of the description
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
  if (coded) {
    TORCH_CHECK_VALUE(k.size(d + 3) == b200_cache4_row_bytes(64) ||
                          k.size(d + 3) == b200_cache4_row_bytes(128),
                      "rows of a 4-bit cache have ", b200_cache4_row_bytes(64), " bytes (head_dim up "
                      "to 64) or ", b200_cache4_row_bytes(128), " (up to 128), got ", k.size(d + 3));
    for (int64_t i = 0; i < d + 3; ++i)
      TORCH_CHECK_VALUE(k.size(i) == 1 || (k.stride(i) % 16 == 0 && v.stride(i) % 16 == 0),
                        "the strides of a 4-bit cache must be multiples of 16 bytes");
  } else {
    TORCH_CHECK_VALUE(k.size(d + 3) % 8 == 0 && k.size(d + 3) <= 128, "head_dim ", k.size(d + 3),
                      " is outside the kernel envelope (multiples of 8 up to 128)");
  }
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.layers = d ? k.size(0) : 1;
  c.pages = k.size(d);
  c.kv_heads = k.size(d + 1);
  c.head_dim = k.size(d + 3) / each;
  for (int64_t i = 0; i < 4; ++i) {
    c.k_stride[i] = i == 0 && !d ? 0 : k.stride(d + i - 1) / each;
    c.v_stride[i] = i == 0 && !d ? 0 : v.stride(d + i - 1) / each;
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

// The head dim of vectors that go into rows of a 4-bit cache, checked against them.
void check_coded(const b200_cache& c, int64_t head_dim, const char* whose) {
  const int64_t bytes = b200_cache4_row_bytes(head_dim);
  TORCH_CHECK_VALUE(bytes > 0, "head_dim ", head_dim,
                    " is outside the kernel envelope (multiples of 8 up to 128)");
  TORCH_CHECK_VALUE(bytes == 2 * c.head_dim, whose, " has head_dim ", head_dim, ", whose rows have ",
                    bytes, " bytes in a 4-bit cache; the pools' have ", 2 * c.head_dim);
}

void fill_rows(b200_cache_rows* r, const at::Tensor& k, const at::Tensor& v, int64_t d) {
  r->k = k.data_ptr();
  r->v = v.data_ptr();
  r->tokens = k.size(d + 2);
  for (int64_t i = 0; i < 4; ++i) {
    r->k_stride[i] = i == 0 && !d ? 0 : k.stride(d + i - 1);
    r->v_stride[i] = i == 0 && !d ? 0 : v.stride(d + i - 1);
  }
}

void cache_append(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& k,
                  const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens,
                  const OptTensor& counts, int64_t error_word) {
  const b200_cache c = cache_view(k, v, table, lens, std::nullopt, error_word);
  const int64_t d = k.dim() - 4;
  TORCH_CHECK_VALUE(k_new.dim() == k.dim() && v_new.sizes() == k_new.sizes(),
                    "k_new and v_new must have shape [(layers,) batch, kv_heads, tokens, "
                    "head_dim] like the pools; got ", k_new.sizes(), " and ", v_new.sizes());
  const bool coded = k.scalar_type() == at::kByte;
  const int64_t head_dim = k_new.size(d + 3);
  if (coded) check_coded(c, head_dim, "k_new");
  TORCH_CHECK_VALUE((!d || k_new.size(0) == c.layers) && k_new.size(d) == c.batch &&
                        k_new.size(d + 1) == c.kv_heads && (coded || head_dim == c.head_dim),
                    "k_new must have shape [(", c.layers, ",) ", c.batch, ", ", c.kv_heads,
                    ", tokens, ", coded ? head_dim : c.head_dim, "], got ", k_new.sizes());
  const int32_t dt = dtype_code(k_new.scalar_type());
  if (coded) {
    TORCH_CHECK_TYPE(dt >= 0 && v_new.scalar_type() == k_new.scalar_type(),
                     "k_new and v_new must both be bfloat16, float16 or float32, got ",
                     k_new.scalar_type(), " and ", v_new.scalar_type());
  } else {
    TORCH_CHECK_TYPE(k_new.scalar_type() == k.scalar_type() && v_new.scalar_type() == k.scalar_type(),
                     "k_new and v_new must have the pools' dtype ", k.scalar_type());
  }
  TORCH_CHECK_VALUE(k_new.device() == k.device() && v_new.device() == k.device(),
                    "k_new and v_new must be on the cache's device");
  TORCH_CHECK_VALUE(k_new.stride(d + 3) == 1 && v_new.stride(d + 3) == 1,
                    "k_new and v_new must have a contiguous last dimension");
  TORCH_CHECK_VALUE(!(c10::GradMode::is_enabled() &&
                      (k_new.requires_grad() || v_new.requires_grad())),
                    "the paged cache is inference-only (autograd requested)");
  b200_cache_rows r{};
  fill_rows(&r, k_new, v_new, d);
  if (counts.has_value()) r.counts = ints(*counts, "draft_lens", {c.batch}, k.device());
  if (r.tokens == 0) return;
  if (coded)
    raise_code("b200_cache4_append", b200_cache4_append(&c, head_dim, dt, &r, stream_of(k)));
  else
    raise_code("b200_cache_append", b200_cache_append(&c, &r, stream_of(k)));
}

std::tuple<at::Tensor, at::Tensor> cache_read(const at::Tensor& k, const at::Tensor& v,
                                              const at::Tensor& table, const at::Tensor& starts,
                                              int64_t tokens, int64_t head_dim, at::ScalarType dtype,
                                              const OptTensor& counts, int64_t error_word) {
  TORCH_CHECK_TYPE(k.scalar_type() == at::kByte, "b200_cache_read reads 4-bit caches (uint8 pools), "
                   "got ", k.scalar_type());
  const b200_cache c = cache_view(k, v, table, starts, std::nullopt, error_word);
  check_coded(c, head_dim, "the call");
  const int32_t dt = dtype_code(dtype);
  TORCH_CHECK_TYPE(dt >= 0, "dtype must be bfloat16, float16 or float32, got ", dtype);
  TORCH_CHECK_VALUE(tokens >= 0, "tokens must not be negative");
  const int64_t d = k.dim() - 4;
  std::vector<int64_t> shape{c.batch, c.kv_heads, tokens, head_dim};
  if (d) shape.insert(shape.begin(), c.layers);
  at::Tensor k_out = at::empty(shape, k.options().dtype(dtype)), v_out = at::empty_like(k_out);
  b200_cache_rows r{};
  fill_rows(&r, k_out, v_out, d);
  if (counts.has_value()) r.counts = ints(*counts, "counts", {c.batch}, k.device());
  if (tokens > 0)
    raise_code("b200_cache4_read", b200_cache4_read(&c, head_dim, dt, &r, stream_of(k)));
  return {k_out, v_out};
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
  const bool coded = k.scalar_type() == at::kByte;
  if (coded) {
    check_coded(p.cache, D, "q");
  } else {
    TORCH_CHECK_VALUE(D == p.cache.head_dim, "q has head_dim ", D, ", the pools ", p.cache.head_dim);
  }
  TORCH_CHECK_VALUE(H >= 1 && H % p.cache.kv_heads == 0, "q's heads (", H,
                    ") must be a multiple of the pools' (", p.cache.kv_heads, ")");
  if (coded) {
    TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
                     "q must be bfloat16 or float16 over a 4-bit cache, got ", q.scalar_type());
  } else {
    TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type(), "q must have the pools' dtype ",
                     k.scalar_type(), ", got ", q.scalar_type());
  }
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
  const int32_t dt = dtype_code(q.scalar_type());
  p.workspace_bytes = coded ? b200_cache4_attn_workspace_bytes(&p, D, dt)
                            : b200_tree_attn_workspace_bytes(&p);
  at::Tensor ws;
  if (p.workspace_bytes > 0) {
    ws = scratch(p.workspace_bytes, q);
    p.workspace = ws.data_ptr();
  }
  const cudaStream_t stream = stream_of(q);
  p.counters = counters_of(stream, q);
  if (coded)
    raise_code("b200_cache4_attn_fwd", b200_cache4_attn_fwd(&p, D, dt, stream));
  else
    raise_code("b200_tree_attn_fwd", b200_tree_attn_fwd(&p, stream));
  return result;
}

// ------------------------------------------------------------ drafted tokens
std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_drafts(
    const at::Tensor& logits, const at::Tensor& tokens, const at::Tensor& uniforms,
    const OptTensor& draft_probs, const OptTensor& parents, const OptTensor& draft_lens,
    double temperature, int64_t error_word) {
  TORCH_CHECK_VALUE(logits.dim() == 3, "logits must have shape [B, T, V], got ", logits.sizes());
  TORCH_CHECK_VALUE(logits.is_cuda(), "b200_verify_drafts runs on CUDA tensors only");
  const int64_t B = logits.size(0), T = logits.size(1), V = logits.size(2);
  TORCH_CHECK_VALUE(B >= 1 && B <= 65535, "logits must have 1 to 65535 sequences, got ", B);
  TORCH_CHECK_VALUE(T >= 1 && T <= B200_VERIFY_MAX_NODES, "logits must have 1 to ",
                    B200_VERIFY_MAX_NODES, " nodes, got ", T);
  TORCH_CHECK_VALUE(V >= 1 && V <= B200_VERIFY_MAX_VOCAB, "logits must have 1 to ",
                    B200_VERIFY_MAX_VOCAB, " tokens, got ", V);
  b200_verify_params p{};
  p.dtype = dtype_code(logits.scalar_type());
  TORCH_CHECK_TYPE(p.dtype >= 0, "logits must be bfloat16, float16 or float32, got ",
                   logits.scalar_type());
  TORCH_CHECK_VALUE(V == 1 || logits.stride(2) == 1, "logits must have a contiguous last dimension");
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
                   "tokens must have dtype torch.int64 or torch.int32, got ", tokens.scalar_type());
  TORCH_CHECK_TYPE(uniforms.scalar_type() == at::kFloat, "uniforms must have dtype torch.float32, "
                   "got ", uniforms.scalar_type());
  for (const at::Tensor* t : {&tokens, &uniforms}) {
    const char* name = t == &tokens ? "tokens" : "uniforms";
    TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == B && t->size(1) == T, name,
                      " must have shape [", B, ", ", T, "], got ", t->sizes());
    TORCH_CHECK_VALUE(T == 1 || t->stride(1) == 1, name, " must have a contiguous last dimension");
    TORCH_CHECK_VALUE(t->device() == logits.device(), name, " must be on the logits' device");
  }
  TORCH_CHECK_VALUE(temperature >= 0.0 && std::isfinite(temperature),
                    "temperature must be a finite number of 0 or more, got ", temperature);
  TORCH_CHECK_VALUE(temperature == 0.0 || std::isfinite(1.0 / temperature),
                    "temperature must be 0 or have a finite reciprocal, got ", temperature);
  TORCH_CHECK_VALUE(!(c10::GradMode::is_enabled() &&
                      (logits.requires_grad() || uniforms.requires_grad() ||
                       (draft_probs.has_value() && draft_probs->requires_grad()))),
                    "b200_verify_drafts is inference-only (autograd requested)");
  if (draft_probs.has_value()) {
    const at::Tensor& q = *draft_probs;
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == B && q.size(1) == T - 1 && q.size(2) == V,
                      "draft_probs must have shape [", B, ", ", T - 1, ", ", V, "], got ", q.sizes());
    p.draft_dtype = dtype_code(q.scalar_type());
    TORCH_CHECK_TYPE(p.draft_dtype >= 0, "draft_probs must be bfloat16, float16 or float32, got ",
                     q.scalar_type());
    TORCH_CHECK_VALUE(V == 1 || q.stride(2) == 1,
                      "draft_probs must have a contiguous last dimension");
    TORCH_CHECK_VALUE(q.device() == logits.device(), "draft_probs must be on the logits' device");
    if (T > 1) p.draft_probs = q.data_ptr();
    p.draft_stride[0] = q.stride(0);
    p.draft_stride[1] = q.stride(1);
  }
  if (parents.has_value()) {
    const at::Tensor& t = *parents;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, "parents must have dtype torch.int32, got ",
                     t.scalar_type());
    const bool shared = t.dim() == 1;
    TORCH_CHECK_VALUE((shared || (t.dim() == 2 && t.size(0) == B)) && t.size(-1) == T,
                      "parents must have shape [", T, "] or [", B, ", ", T, "], got ", t.sizes());
    TORCH_CHECK_VALUE(T == 1 || t.stride(-1) == 1, "parents must have a contiguous last dimension");
    TORCH_CHECK_VALUE(t.device() == logits.device(), "parents must be on the logits' device");
    p.parents = static_cast<const int32_t*>(t.data_ptr());
    p.parent_stride = shared ? 0 : t.stride(0);
  }
  if (draft_lens.has_value()) p.draft_lens = ints(*draft_lens, "draft_lens", {B}, logits.device());
  at::Tensor paths = at::empty({B, T}, logits.options().dtype(at::kInt));
  at::Tensor counts = at::empty({B}, logits.options().dtype(at::kInt));
  at::Tensor next = at::empty({B}, logits.options().dtype(at::kLong));
  p.logits = logits.data_ptr();
  p.logits_stride[0] = logits.stride(0);
  p.logits_stride[1] = logits.stride(1);
  p.tokens = tokens.data_ptr();
  p.token_stride = tokens.stride(0);
  p.wide_tokens = tokens.scalar_type() == at::kLong;
  p.uniforms = static_cast<const float*>(uniforms.data_ptr());
  p.uniform_stride = uniforms.stride(0);
  p.paths = static_cast<int32_t*>(paths.data_ptr());
  p.counts = static_cast<int32_t*>(counts.data_ptr());
  p.next = static_cast<int64_t*>(next.data_ptr());
  p.batch = B;
  p.nodes = T;
  p.vocab = V;
  p.temperature = temperature;
  p.error_word = reinterpret_cast<int32_t*>(static_cast<intptr_t>(error_word));
  raise_code("b200_verify_drafts", b200_verify_drafts(&p, stream_of(logits)));
  return {paths, counts, next};
}

}  // namespace

TORCH_LIBRARY(b200, m) {
  m.def(
      "cache_append(Tensor k_new, Tensor v_new, Tensor(a!) k_pages, Tensor(b!) v_pages, "
      "Tensor page_table, Tensor seq_lens, Tensor? draft_lens, int error_word) -> ()",
      &cache_append);
  m.def(
      "cache_read(Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor starts, int tokens, "
      "int head_dim, ScalarType dtype, Tensor? counts, int error_word) -> (Tensor, Tensor)",
      &cache_read);
  m.def(
      "verify_drafts(Tensor logits, Tensor tokens, Tensor uniforms, Tensor? draft_probs, "
      "Tensor? parents, Tensor? draft_lens, float temperature, int error_word) -> "
      "(Tensor, Tensor, Tensor)",
      &verify_drafts);
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

// q3s_torch_decode.cpp -- torch.ops.q3s.*: the decode step's operators beside
// the sampler (include/q3s_decode.h) as PyTorch operators.  Each checks its
// tensors, allocates outputs and workspace from torch's allocator, fills the C
// descriptor and calls the C ABI on the current CUDA stream; a bad argument
// raises before anything is launched.
//
//   cache_tables(context_lengths, new_lengths, block_table!, free_blocks!, free_state, block_size, max_tokens,
//                released=None, whole_rows=False) -> (query_offsets, slot_map, positions, lengths, free_state, error_word)
//   cache_append(k, v, k_cache!, v_cache!, slot_map, error_word!=None) -> ()
//   prefix_attention(q, k_cache, v_cache, query_offsets, block_table, lengths, prefix_blocks=None, prefix_length=0,
//                    scale=None, error_word!=None, slot_map=None) -> (out, lse)
//   quantize_rows(x) -> (values, scales)
//   int8_matmul(values, scales, weight, weight_scales, dtype, bias=None, error_word!=None) -> y
//   int8_linear(x, weight, weight_scales, bias=None, error_word!=None) -> (y, values, scales)
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cmath>
#include <cstring>
#include <tuple>

#include "q3s_decode.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_status(q3s_status s, const char* what) {
  TORCH_CHECK(s == Q3S_OK, what, " failed (status ", static_cast<int>(s), "): ", q3s_last_error_string());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void need_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "q3s: ", name, " must be a CUDA tensor (there is no CPU fallback)");
}
void need(const Tensor& t, const Tensor& ref, at::ScalarType dt, int64_t dims, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == ref.device(), "q3s: ", name, " must be on ", ref.device());
  TORCH_CHECK(t.scalar_type() == dt, "q3s: ", name, " must be ", dt, ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dims, "q3s: ", name, " must have ", dims, " dimensions, got ", t.sizes());
}
void need_vector(const Tensor& t, const Tensor& ref, at::ScalarType dt, int64_t n, const char* name) {
  need(t, ref, dt, 1, name);
  TORCH_CHECK(t.size(0) == n, "q3s: ", name, " must have ", n, " entries, got ", t.size(0));
  TORCH_CHECK(t.is_contiguous(), "q3s: ", name, " must be contiguous");
}
int32_t elem_of(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return Q3S_ELEM_F32;
  if (t.scalar_type() == at::kBFloat16) return Q3S_ELEM_BF16;
  if (t.scalar_type() == at::kHalf) return Q3S_ELEM_F16;
  TORCH_CHECK(false, "q3s: ", name, " must be bf16, f16 or fp32, got ", t.scalar_type());
}
int32_t* error_of(const OptTensor& e, const Tensor& ref) {
  if (!e.has_value()) return nullptr;
  need_vector(*e, ref, at::kInt, 1, "error_word");
  return e->data_ptr<int32_t>();
}
int32_t i32(int64_t x, const char* name) {
  TORCH_CHECK(x >= 0 && x <= INT32_MAX, "q3s: ", name, " is ", x, ", not in [0, 2^31)");
  return static_cast<int32_t>(x);
}
// A new contiguous tensor like at::empty's, straight from the CUDA allocator: at a decode step's sizes the dispatcher
// costs more than the kernels.
Tensor make(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& ref) {
  return at::detail::empty_cuda(sizes, dt, ref.device(), c10::nullopt);
}
// Two tensors that a call reads and writes must not share memory.
void apart(const Tensor& out, const Tensor& in, const char* what) {
  TORCH_CHECK(!out.is_alias_of(in) || out.data_ptr() != in.data_ptr(), "q3s: ", what, " must not be the same tensor");
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> cache_tables(
    const Tensor& context, const Tensor& fresh, Tensor block_table, Tensor free_blocks, const Tensor& free_state,
    int64_t block_size, int64_t max_tokens, const OptTensor& released, bool whole_rows) {
  need_cuda(context, "context_lengths");
  c10::cuda::CUDAGuard guard(context.device());
  need(context, context, at::kInt, 1, "context_lengths");
  const int64_t B = context.size(0);
  need_vector(context, context, at::kInt, B, "context_lengths");
  need_vector(fresh, context, at::kInt, B, "new_lengths");
  need(block_table, context, at::kInt, 2, "block_table");
  TORCH_CHECK(block_table.size(0) == B && (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "q3s: block_table must be [", B, ", max_blocks] with unit column stride, got ", block_table.sizes());
  need(free_blocks, context, at::kInt, 1, "free_blocks");
  need_vector(free_blocks, context, at::kInt, free_blocks.size(0), "free_blocks");
  need_vector(free_state, context, at::kInt, 2, "free_state");
  apart(block_table, free_blocks, "block_table and free_blocks");
  apart(block_table, context, "block_table and context_lengths");
  q3s_cache_tables_desc d;
  std::memset(&d, 0, sizeof(d));
  d.struct_size = sizeof(d);
  d.batch = i32(B, "batch");
  d.block_size = i32(block_size, "block_size");
  d.max_blocks = i32(block_table.size(1), "max_blocks");
  d.context_lengths = context.data_ptr<int32_t>();
  d.new_lengths = fresh.data_ptr<int32_t>();
  if (released.has_value()) {
    TORCH_CHECK(released->scalar_type() == at::kBool || released->scalar_type() == at::kByte,
                "q3s: released must be bool or uint8, got ", released->scalar_type());
    need_vector(*released, context, released->scalar_type(), B, "released");
    d.released = static_cast<const uint8_t*>(released->data_ptr());
  }
  d.block_table = block_table.data_ptr<int32_t>();
  d.block_table_stride = B > 1 ? block_table.stride(0) : block_table.size(1);
  TORCH_CHECK(d.block_table_stride >= block_table.size(1), "q3s: rows of block_table overlap");
  d.free_blocks = free_blocks.data_ptr<int32_t>();
  d.ring_size = i32(free_blocks.size(0), "free_blocks");
  d.free_state = free_state.data_ptr<int32_t>();
  d.max_tokens = i32(max_tokens, "max_tokens");
  d.flags = whole_rows ? Q3S_TABLES_WHOLE_ROWS : 0;
  Tensor slots = make({max_tokens}, at::kLong, context), positions = make({max_tokens}, at::kInt, context);
  Tensor offsets = make({B + 1}, at::kInt, context), lengths = make({B}, at::kInt, context);
  Tensor state = make({2}, at::kInt, context), error = make({1}, at::kInt, context);
  d.query_offsets = offsets.data_ptr<int32_t>();
  d.slot_map = slots.data_ptr<int64_t>();
  d.positions = positions.data_ptr<int32_t>();
  d.lengths_out = lengths.data_ptr<int32_t>();
  d.free_state_out = state.data_ptr<int32_t>();
  d.error_word = error.data_ptr<int32_t>();
  check_status(q3s_cache_tables(&d, stream_of(context)), "q3s_cache_tables");
  return {offsets, slots, positions, lengths, state, error};
}

// [blocks, kv_heads, block_size, dim] with unit last stride, and like `ref`.
void need_cache(const Tensor& c, const Tensor& ref, const char* name) {
  need(c, ref, ref.scalar_type(), 4, name);
  TORCH_CHECK(c.size(3) <= 1 || c.stride(3) == 1, "q3s: ", name, " must have unit last stride");
}

void cache_append(const Tensor& k, const Tensor& v, Tensor k_cache, Tensor v_cache, const Tensor& slot_map,
                  OptTensor error_word) {
  need_cuda(k, "k");
  c10::cuda::CUDAGuard guard(k.device());
  need(k, k, k.scalar_type(), 3, "k");
  need(v, k, k.scalar_type(), 3, "v");
  need_cache(k_cache, k, "k_cache");
  need_cache(v_cache, k, "v_cache");
  TORCH_CHECK(k.sizes() == v.sizes() && k_cache.sizes() == v_cache.sizes() && k_cache.size(1) == k.size(1) &&
                  k_cache.size(3) == k.size(2),
              "q3s: k and v must be [T, kv_heads, dim] and the caches [blocks, kv_heads, block_size, dim], got ",
              k.sizes(), v.sizes(), k_cache.sizes(), v_cache.sizes());
  TORCH_CHECK((k.size(2) <= 1 || k.stride(2) == 1) && (v.size(2) <= 1 || v.stride(2) == 1),
              "q3s: k and v must have unit last stride");
  need_vector(slot_map, k, at::kLong, k.size(0), "slot_map");
  q3s_cache_append_desc d;
  std::memset(&d, 0, sizeof(d));
  d.struct_size = sizeof(d);
  d.tokens = i32(k.size(0), "tokens");
  d.kv_heads = i32(k.size(1), "kv_heads");
  d.dim = i32(k.size(2), "dim");
  d.block_size = i32(k_cache.size(2), "block_size");
  d.blocks = i32(k_cache.size(0), "blocks");
  d.elem = elem_of(k, "k");
  d.k = k.data_ptr();
  d.v = v.data_ptr();
  d.k_token_stride = k.stride(0);
  d.k_head_stride = k.stride(1);
  d.v_token_stride = v.stride(0);
  d.v_head_stride = v.stride(1);
  d.slot_map = slot_map.data_ptr<int64_t>();
  d.k_cache = k_cache.data_ptr();
  d.v_cache = v_cache.data_ptr();
  d.k_block_stride = k_cache.stride(0);
  d.k_cache_head_stride = k_cache.stride(1);
  d.k_place_stride = k_cache.stride(2);
  d.v_block_stride = v_cache.stride(0);
  d.v_cache_head_stride = v_cache.stride(1);
  d.v_place_stride = v_cache.stride(2);
  d.error_word = error_of(error_word, k);
  check_status(q3s_cache_append(&d, stream_of(k)), "q3s_cache_append");
}

std::tuple<Tensor, Tensor> prefix_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                            const Tensor& query_offsets, const Tensor& block_table,
                                            const Tensor& lengths, const OptTensor& prefix_blocks,
                                            int64_t prefix_length, c10::optional<double> scale,
                                            OptTensor error_word, const OptTensor& slot_map) {
  need_cuda(q, "q");
  c10::cuda::CUDAGuard guard(q.device());
  need(q, q, q.scalar_type(), 3, "q");
  need_cache(k_cache, q, "k_cache");
  need_cache(v_cache, q, "v_cache");
  TORCH_CHECK(q.stride(2) == 1 || q.size(2) <= 1, "q3s: q must have unit last stride");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.size(3) == q.size(2),
              "q3s: the caches must be [blocks, kv_heads, block_size, ", q.size(2), "], got ", k_cache.sizes(), " and ",
              v_cache.sizes());
  need(lengths, q, at::kInt, 1, "lengths");
  const int64_t B = lengths.size(0), T = q.size(0);
  need_vector(lengths, q, at::kInt, B, "lengths");
  need_vector(query_offsets, q, at::kInt, B + 1, "query_offsets");
  need(block_table, q, at::kInt, 2, "block_table");
  TORCH_CHECK(block_table.size(0) == B && (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "q3s: block_table must be [", B, ", max_blocks] with unit column stride, got ", block_table.sizes());
  q3s_prefix_attention_desc d;
  std::memset(&d, 0, sizeof(d));
  d.struct_size = sizeof(d);
  d.batch = i32(B, "batch");
  d.tokens = i32(T, "tokens");
  d.q_heads = i32(q.size(1), "q_heads");
  d.kv_heads = i32(k_cache.size(1), "kv_heads");
  d.dim = i32(q.size(2), "dim");
  d.block_size = i32(k_cache.size(2), "block_size");
  d.blocks = i32(k_cache.size(0), "blocks");
  d.elem = elem_of(q, "q");
  d.max_blocks = i32(block_table.size(1), "max_blocks");
  d.prefix_length = i32(prefix_length, "prefix_length");
  if (prefix_length > 0) {
    TORCH_CHECK(prefix_blocks.has_value(), "q3s: a prefix needs prefix_blocks");
    need(*prefix_blocks, q, at::kInt, 1, "prefix_blocks");
    need_vector(*prefix_blocks, q, at::kInt, prefix_blocks->size(0), "prefix_blocks");
    TORCH_CHECK(prefix_blocks->size(0) * k_cache.size(2) >= prefix_length, "q3s: prefix_blocks holds ",
                prefix_blocks->size(0), " blocks of ", k_cache.size(2), " for a prefix of ", prefix_length);
    d.prefix_blocks = prefix_blocks->data_ptr<int32_t>();
  }
  d.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2))));
  d.q = q.data_ptr();
  d.q_token_stride = T > 1 ? q.stride(0) : q.size(1) * q.size(2);
  d.q_head_stride = q.stride(1);
  d.k_cache = k_cache.data_ptr();
  d.v_cache = v_cache.data_ptr();
  d.k_block_stride = k_cache.stride(0);
  d.k_head_stride = k_cache.stride(1);
  d.k_place_stride = k_cache.stride(2);
  d.v_block_stride = v_cache.stride(0);
  d.v_head_stride = v_cache.stride(1);
  d.v_place_stride = v_cache.stride(2);
  d.query_offsets = query_offsets.data_ptr<int32_t>();
  d.block_table = block_table.data_ptr<int32_t>();
  d.block_table_stride = B > 1 ? block_table.stride(0) : block_table.size(1);
  d.lengths = lengths.data_ptr<int32_t>();
  Tensor out = make({T, q.size(1), q.size(2)}, q.scalar_type(), q), lse = make({T, q.size(1)}, at::kFloat, q);
  d.out = out.data_ptr();
  d.out_token_stride = q.size(1) * q.size(2);
  d.out_head_stride = q.size(2);
  d.lse = lse.data_ptr<float>();
  d.error_word = error_of(error_word, q);
  if (slot_map.has_value()) {
    need_vector(*slot_map, q, at::kLong, T, "slot_map");
    d.slot_map = slot_map->data_ptr<int64_t>();
  }
  int64_t bytes = 0;
  check_status(q3s_prefix_attention_workspace(&d, &bytes), "q3s_prefix_attention");
  const Tensor ws = make({bytes}, at::kByte, q);
  d.workspace = ws.data_ptr();
  d.workspace_bytes = bytes;
  check_status(q3s_prefix_attention(&d, stream_of(q)), "q3s_prefix_attention");
  return {out, lse};
}

// Rows of x as [M, K] (a view where the strides allow it).
Tensor rows_of(const Tensor& x) {
  need_cuda(x, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "q3s: x must be [..., K], got ", x.sizes());
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) r = r.contiguous();
  return r;
}

q3s_quantize_rows_desc quantize_desc(const Tensor& r, const Tensor& values, const Tensor& scales) {
  q3s_quantize_rows_desc d;
  std::memset(&d, 0, sizeof(d));
  d.struct_size = sizeof(d);
  d.rows = i32(r.size(0), "rows");
  d.cols = i32(r.size(1), "cols");
  d.elem = elem_of(r, "x");
  d.x = r.data_ptr();
  d.x_row_stride = r.size(0) > 1 ? r.stride(0) : r.size(1);
  d.values = values.data_ptr<int8_t>();
  d.values_row_stride = r.size(1);
  d.scales = scales.data_ptr<float>();
  return d;
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  const Tensor r = rows_of(x);
  c10::cuda::CUDAGuard guard(r.device());
  Tensor values = make({r.size(0), r.size(1)}, at::kChar, r), scales = make({r.size(0)}, at::kFloat, r);
  const q3s_quantize_rows_desc d = quantize_desc(r, values, scales);
  check_status(q3s_quantize_rows(&d, stream_of(r)), "q3s_quantize_rows");
  if (x.dim() == 2) return {values, scales};
  return {values.view(x.sizes()), scales.view(x.sizes().slice(0, x.dim() - 1))};
}

q3s_int8_matmul_desc matmul_desc(const Tensor& a, const Tensor& a_scales, const Tensor& w, const Tensor& w_scales,
                                 const OptTensor& bias, const OptTensor& error_word, const Tensor& y) {
  const int64_t M = a.size(0), K = a.size(1), N = w.size(0);
  need(w, a, at::kChar, 2, "weight");
  TORCH_CHECK(w.size(1) == K && w.stride(1) == 1, "q3s: weight must be [N, ", K, "] with unit column stride, got ", w.sizes());
  need_vector(a_scales, a, at::kFloat, M, "scales");
  need_vector(w_scales, a, at::kFloat, N, "weight_scales");
  q3s_int8_matmul_desc d;
  std::memset(&d, 0, sizeof(d));
  d.struct_size = sizeof(d);
  d.rows = i32(M, "rows");
  d.inputs = i32(K, "inputs");
  d.outputs = i32(N, "outputs");
  d.elem = elem_of(y, "y");
  d.a = a.data_ptr<int8_t>();
  d.a_row_stride = M > 1 ? a.stride(0) : K;
  d.a_scales = a_scales.data_ptr<float>();
  d.w = w.data_ptr<int8_t>();
  d.w_row_stride = N > 1 ? w.stride(0) : K;
  d.w_scales = w_scales.data_ptr<float>();
  if (bias.has_value()) {
    need_vector(*bias, a, at::kFloat, N, "bias");
    d.bias = bias->data_ptr<float>();
  }
  d.y = y.data_ptr();
  d.y_row_stride = N;
  d.error_word = error_of(error_word, a);
  return d;
}

Tensor int8_matmul(const Tensor& values, const Tensor& scales, const Tensor& weight, const Tensor& weight_scales,
                   at::ScalarType dtype, const OptTensor& bias, OptTensor error_word) {
  need_cuda(values, "values");
  c10::cuda::CUDAGuard guard(values.device());
  need(values, values, at::kChar, 2, "values");
  TORCH_CHECK(values.size(1) <= 1 || values.stride(1) == 1, "q3s: values must have unit column stride");
  TORCH_CHECK(weight.dim() == 2, "q3s: weight must be [N, K], got ", weight.sizes());
  Tensor y = make({values.size(0), weight.size(0)}, dtype, values);
  const q3s_int8_matmul_desc d = matmul_desc(values, scales, weight, weight_scales, bias, error_word, y);
  check_status(q3s_int8_matmul(&d, stream_of(values)), "q3s_int8_matmul");
  return y;
}

std::tuple<Tensor, Tensor, Tensor> int8_linear(const Tensor& x, const Tensor& weight, const Tensor& weight_scales,
                                               const OptTensor& bias, OptTensor error_word) {
  const Tensor r = rows_of(x);
  c10::cuda::CUDAGuard guard(r.device());
  TORCH_CHECK(weight.dim() == 2, "q3s: weight must be [N, K], got ", weight.sizes());
  const int64_t M = r.size(0), K = r.size(1), N = weight.size(0);
  Tensor values = make({M, K}, at::kChar, r), scales = make({M}, at::kFloat, r), y = make({M, N}, r.scalar_type(), r);
  const q3s_quantize_rows_desc q = quantize_desc(r, values, scales);
  const q3s_int8_matmul_desc d = matmul_desc(values, scales, weight, weight_scales, bias, error_word, y);
  check_status(q3s_int8_linear(&q, &d, stream_of(r)), "q3s_int8_linear");
  if (x.dim() == 2) return {y, values, scales};
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  return {y.view(shape), values.view(x.sizes()), scales.view(x.sizes().slice(0, x.dim() - 1))};
}

// ---- Meta kernels: shapes and dtypes only ------------------------------------
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> cache_tables_meta(const Tensor& context, const Tensor&,
                                                                             Tensor, Tensor, const Tensor&, int64_t,
                                                                             int64_t max_tokens, const OptTensor&, bool) {
  const auto o = context.options();
  const int64_t B = context.size(0);
  return {at::empty({B + 1}, o), at::empty({max_tokens}, o.dtype(at::kLong)), at::empty({max_tokens}, o),
          at::empty({B}, o), at::empty({2}, o), at::empty({1}, o)};
}
void cache_append_meta(const Tensor&, const Tensor&, Tensor, Tensor, const Tensor&, OptTensor) {}
std::tuple<Tensor, Tensor> prefix_attention_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&,
                                                 const Tensor&, const Tensor&, const OptTensor&, int64_t,
                                                 c10::optional<double>, OptTensor, const OptTensor&) {
  return {at::empty(q.sizes(), q.options()), at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor> quantize_rows_meta(const Tensor& x) {
  return {at::empty(x.sizes(), x.options().dtype(at::kChar)),
          at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat))};
}
Tensor int8_matmul_meta(const Tensor& values, const Tensor&, const Tensor& weight, const Tensor&, at::ScalarType dtype,
                        const OptTensor&, OptTensor) {
  return at::empty({values.size(0), weight.size(0)}, values.options().dtype(dtype));
}
std::tuple<Tensor, Tensor, Tensor> int8_linear_meta(const Tensor& x, const Tensor& weight, const Tensor&,
                                                    const OptTensor&, OptTensor) {
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = weight.size(0);
  const auto q = quantize_rows_meta(x);
  return {at::empty(shape, x.options()), std::get<0>(q), std::get<1>(q)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(q3s, m) {
  m.def("cache_tables(Tensor context_lengths, Tensor new_lengths, Tensor(a!) block_table, Tensor(b!) free_blocks, "
        "Tensor free_state, int block_size, int max_tokens, Tensor? released=None, bool whole_rows=False) -> (Tensor, "
        "Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("cache_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slot_map, "
        "Tensor(c!)? error_word=None) -> ()");
  m.def("prefix_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor query_offsets, Tensor block_table, "
        "Tensor lengths, Tensor? prefix_blocks=None, int prefix_length=0, float? scale=None, "
        "Tensor(a!)? error_word=None, Tensor? slot_map=None) -> (Tensor, Tensor)");
  m.def("quantize_rows(Tensor x) -> (Tensor, Tensor)");
  m.def("int8_matmul(Tensor values, Tensor scales, Tensor weight, Tensor weight_scales, ScalarType dtype, "
        "Tensor? bias=None, Tensor(a!)? error_word=None) -> Tensor");
  m.def("int8_linear(Tensor x, Tensor weight, Tensor weight_scales, Tensor? bias=None, Tensor(a!)? error_word=None) -> "
        "(Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(q3s, CUDA, m) {
  m.impl("cache_tables", &cache_tables);
  m.impl("cache_append", &cache_append);
  m.impl("prefix_attention", &prefix_attention);
  m.impl("quantize_rows", &quantize_rows);
  m.impl("int8_matmul", &int8_matmul);
  m.impl("int8_linear", &int8_linear);
}

TORCH_LIBRARY_IMPL(q3s, Meta, m) {
  m.impl("cache_tables", &cache_tables_meta);
  m.impl("cache_append", &cache_append_meta);
  m.impl("prefix_attention", &prefix_attention_meta);
  m.impl("quantize_rows", &quantize_rows_meta);
  m.impl("int8_matmul", &int8_matmul_meta);
  m.impl("int8_linear", &int8_linear_meta);
}

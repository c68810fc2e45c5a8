// q3s_int8.cu -- host side of the 8-bit projections: q3s_quantize_rows and
// q3s_int8_matmul.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "q3s_int8.cuh"
#include "q3s_tma.cuh"

namespace {

// 2-D tensor of bytes [rows, cols] (row stride `ld`), boxes of [box_rows, 128]
// in the 128-byte swizzle; what lies outside reads as zeros.
bool byte_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  const q3s::EncodeTiled enc = q3s::encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(q3s::I8_BK), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int ELEM>
cudaError_t launch_quantize(const q3s::QuantArgs& a, bool vec, cudaStream_t st) {
  // A warp a row once there are 8 rows a SM; below that a CTA a row has the
  // shorter chain.  CTA against warp: 592 rows of 2048 1.9 against 2.1 us, 1184
  // rows 2.5 against 2.3 (of 64: 2.1 against 1.7), 4096 rows 5.6 against 4.4.
  if (vec && a.M >= 8 * q3s::sm_count() && a.K <= 32 * q3s::QW_KEEP * q3s::Elem<ELEM>::N)
    return q3s::launch_maybe_pdl(q3s::quantize_warps_kernel<ELEM>, dim3((a.M + q3s::QW_WARPS - 1) / q3s::QW_WARPS),
                                 dim3(q3s::QW_WARPS * 32), 0, st, true, a);
  return vec ? q3s::launch_maybe_pdl(q3s::quantize_rows_kernel<ELEM, true>, dim3(a.M), dim3(128), 0, st, true, a)
             : q3s::launch_maybe_pdl(q3s::quantize_rows_kernel<ELEM, false>, dim3(a.M), dim3(128), 0, st, true, a);
}

// -- few rows --
template <bool QUANT, int ELEM, int MB, int RW>
cudaError_t launch_gemv_rw(const q3s::Int8Args& a, const q3s::QuantArgs& q, cudaStream_t st) {
  auto kern = q3s::int8_gemv_kernel<QUANT, ELEM, MB, RW>;
  const int smem = MB * a.K;
  const int per = q3s::GV_WARPS * RW;
  return q3s::launch_maybe_pdl(kern, dim3((a.N + per - 1) / per), dim3(q3s::GV_NT), smem, st, true, a, q);
}
template <bool QUANT, int ELEM, int MB>
cudaError_t launch_gemv_mb(const q3s::Int8Args& a, const q3s::QuantArgs& q, cudaStream_t st) {
  // Outputs of a warp: the fewest with which the CTAs are one a SM.  One against
  // two, 1 row: 1184 outputs 2.3 against 2.5 us, 2048 outputs 2.7 against 2.5; two
  // against four, 8 rows: 2048 outputs 4.6 against 5.4, 8000 outputs 10.2 against 7.6.
  const int warps = q3s::sm_count() * q3s::GV_WARPS;
  if (a.N <= warps) return launch_gemv_rw<QUANT, ELEM, MB, 1>(a, q, st);
  if (a.N <= 2 * warps) return launch_gemv_rw<QUANT, ELEM, MB, 2>(a, q, st);
  return launch_gemv_rw<QUANT, ELEM, MB, 4>(a, q, st);
}
template <bool QUANT, int ELEM>
cudaError_t launch_gemv(const q3s::Int8Args& a, const q3s::QuantArgs& q, cudaStream_t st) {
  if (a.M == 1) return launch_gemv_mb<QUANT, ELEM, 1>(a, q, st);
  if (a.M == 2) return launch_gemv_mb<QUANT, ELEM, 2>(a, q, st);
  if (a.M <= 4) return launch_gemv_mb<QUANT, ELEM, 4>(a, q, st);
  return launch_gemv_mb<QUANT, ELEM, 8>(a, q, st);
}
// The vector kernel up to 8 rows of 24 KB in all: every CTA quantises all of
// them.  Vector kernel against tensor cores with the quantisation: 1 row of 2048,
// 2048 outputs 2.5 against 7.2 us; 8 rows of 2048, 8000 outputs 7.6 against 7.6,
// of 4096 13.0 against 10.7; 4 rows of 6144, 8000 outputs 11.9 against 14.2, of
// 8192 16.7 against 13.8.
bool few_rows(int M, int K) { return M <= q3s::GV_MAX_M && static_cast<int64_t>(K) * (M <= 2 ? M : M <= 4 ? 4 : 8) <= q3s::GV_SMEM; }

// -- tensor cores --
template <int ELEM, int KS>
cudaError_t launch_split_ks(const q3s::Int8Args& a, const q3s::I8Cut& cut, const CUtensorMap& tw, const CUtensorMap& ta,
                            cudaStream_t st) {
  auto kern = q3s::int8_split_kernel<ELEM, KS>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = q3s::allow_smem(kern, 220 * 1024, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((a.N + 127) / 128, KS, (a.M + cut.bt - 1) / cut.bt);
  lc.blockDim = dim3(q3s::I8C_NT);
  lc.dynamicSmemBytes = cut.smem;
  lc.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1;
  at[0].val.clusterDim.y = KS;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = at;
  lc.numAttrs = 2;
  e = cudaLaunchKernelEx(&lc, kern, tw, ta, a, cut);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <int ELEM>
cudaError_t launch_split(const q3s::Int8Args& a, cudaStream_t st) {
  const q3s::I8Cut cut = q3s::int8_cut(a.M, a.N, a.K, q3s::sm_count());
  CUtensorMap tw, ta;
  if (!byte_map(&tw, a.w, a.N, a.K, a.ldw, 128) || !byte_map(&ta, a.a, a.M, a.K, a.lda, cut.bt)) return cudaErrorInvalidValue;
  if (cut.ks == 1) return launch_split_ks<ELEM, 1>(a, cut, tw, ta, st);
  if (cut.ks == 2) return launch_split_ks<ELEM, 2>(a, cut, tw, ta, st);
  if (cut.ks == 4) return launch_split_ks<ELEM, 4>(a, cut, tw, ta, st);
  return launch_split_ks<ELEM, 8>(a, cut, tw, ta, st);
}

template <int ELEM>
bool out_map(CUtensorMap* m, const q3s::Int8Args& a) {
  const q3s::EncodeTiled enc = q3s::encode_tiled();
  if (!enc) return false;
  constexpr int size = ELEM == Q3S_ELEM_F32 ? 4 : 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.N), static_cast<cuuint64_t>(a.M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.ldy) * size};
  const cuuint32_t box[2] = {128 / size, 32}, estr[2] = {1, 1};
  return enc(m, ELEM == Q3S_ELEM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.y, dims,
             strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <int ELEM>
cudaError_t launch_pair(const q3s::Int8Args& a, cudaStream_t st) {
  auto kern = q3s::int8_pair_kernel<ELEM>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = q3s::allow_smem(kern, q3s::I8P_SMEM, done);
  if (e != cudaSuccess) return e;
  CUtensorMap ta, tw, ty = {};
  if (!byte_map(&ta, a.a, a.M, a.K, a.lda, 128) || !byte_map(&tw, a.w, a.N, a.K, a.ldw, 128) || (a.vec_y && !out_map<ELEM>(&ty, a)))
    return cudaErrorInvalidValue;
  const int64_t tiles = static_cast<int64_t>((a.M + 255) / 256) * ((a.N + q3s::I8P_N - 1) / q3s::I8P_N);
  const int grid = 2 * static_cast<int>(std::min<int64_t>(tiles, q3s::sm_count() / 2));
  return q3s::launch_maybe_pdl(kern, dim3(grid), dim3(q3s::I8P_NT), q3s::I8P_SMEM, st, true, ta, tw, ty, a);
}

template <int ELEM>
cudaError_t launch_matmul(const q3s::Int8Args& a, cudaStream_t st) {
  if (few_rows(a.M, a.K)) return launch_gemv<false, ELEM>(a, q3s::QuantArgs{}, st);
  // Pairs of CTAs where their 256 x 256 tiles fill half of the SMs.  Both sides
  // measured, clusters against pairs, inputs 2048: 800 x 2048 outputs (32 tiles)
  // 11.9 against 13.4 us, 1500 x 2048 (48) 16.3 against 15.1, 2048 x 4096 (128)
  // 36.5 against 21.5.
  const int64_t tiles = static_cast<int64_t>((a.M + 255) / 256) * ((a.N + q3s::I8P_N - 1) / q3s::I8P_N);
  if (tiles * 4 >= q3s::sm_count()) return launch_pair<ELEM>(a, st);
  return launch_split<ELEM>(a, st);
}

bool known_elem(int e) { return e == Q3S_ELEM_F32 || e == Q3S_ELEM_BF16 || e == Q3S_ELEM_F16; }

}  // namespace

namespace {

// Checks of the two descriptors; `go`: there is something to do.
q3s_status quant_args(const q3s_quantize_rows_desc* d, const char* who, q3s::QuantArgs* a, bool* vec, bool* go) {
  using q3s::report;
  *go = false;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "%s: desc is NULL", who);
  if (d->struct_size != sizeof(q3s_quantize_rows_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: struct_size %u != %u (ABI mismatch)", who, d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_quantize_rows_desc)));
  if (d->rows < 0 || d->cols < 1)
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: rows must not be negative and cols must be positive", who);
  if (!known_elem(d->elem)) return report(Q3S_ERR_INVALID_ARGUMENT, "%s: unknown elem %d", who, d->elem);
  if (d->rows == 0) return report(Q3S_OK, "");
  if (!d->x || !d->values || !d->scales)
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: x, values and scales are required", who);
  if (d->rows > 1 && (d->x_row_stride < d->cols || d->values_row_stride < d->cols))
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: row strides are below cols", who);
  a->M = d->rows;
  a->K = d->cols;
  a->x = d->x;
  a->ldx = d->x_row_stride;
  a->values = d->values;
  a->ldv = d->values_row_stride;
  a->scales = d->scales;
  const int n = d->elem == Q3S_ELEM_F32 ? 4 : 8;  // elements in 16 bytes
  *vec = a->K % n == 0 && q3s::aligned16(a->x) && reinterpret_cast<uintptr_t>(a->values) % n == 0 &&
         (a->M == 1 || (a->ldx % n == 0 && a->ldv % n == 0));
  *go = true;
  return Q3S_OK;
}

q3s_status matmul_args(const q3s_int8_matmul_desc* d, const char* who, q3s::Int8Args* a, bool* go) {
  using q3s::report;
  *go = false;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "%s: desc is NULL", who);
  if (d->struct_size != sizeof(q3s_int8_matmul_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: struct_size %u != %u (ABI mismatch)", who, d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_int8_matmul_desc)));
  if (d->rows < 0 || d->outputs < 1)
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: rows must not be negative and outputs must be positive", who);
  if (d->inputs < 16 || d->inputs % 16 || d->inputs > 131056)
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: inputs %d is not a multiple of 16 in [16, 131056]", who, d->inputs);
  if (!known_elem(d->elem)) return report(Q3S_ERR_INVALID_ARGUMENT, "%s: unknown elem %d", who, d->elem);
  if (d->rows == 0) return report(Q3S_OK, "");
  if (!d->a || !d->a_scales || !d->w || !d->w_scales || !d->y)
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: a, a_scales, w, w_scales and y are required", who);
  a->lda = d->rows > 1 ? d->a_row_stride : d->inputs;
  a->ldw = d->outputs > 1 ? d->w_row_stride : d->inputs;
  if (!q3s::aligned16(d->a) || !q3s::aligned16(d->w) || a->lda < d->inputs || a->lda % 16 || a->ldw < d->inputs || a->ldw % 16)
    return report(Q3S_ERR_INVALID_ARGUMENT, "%s: rows of a and w must start on 16 bytes, with strides of at least inputs", who);
  a->ldy = d->rows > 1 ? d->y_row_stride : d->outputs;
  if (a->ldy < d->outputs) return report(Q3S_ERR_INVALID_ARGUMENT, "%s: y_row_stride is below outputs", who);
  if (static_cast<int64_t>(d->rows) + 256 > 0x7fffffffll || static_cast<int64_t>(d->outputs) + 256 > 0x7fffffffll ||
      static_cast<int64_t>((d->rows + 255) / 256) * ((d->outputs + 127) / 128) > 0x7fffffffll)
    return report(Q3S_ERR_UNSUPPORTED, "%s: %d x %d outputs are too many", who, d->rows, d->outputs);
  a->M = d->rows;
  a->N = d->outputs;
  a->K = d->inputs;
  a->a = d->a;
  a->a_scales = d->a_scales;
  a->w = d->w;
  a->w_scales = d->w_scales;
  a->bias = d->bias;
  a->y = d->y;
  const int size = d->elem == Q3S_ELEM_F32 ? 4 : 2;
  // rows of y on 16 bytes; one row is read as if the next began on the next 16
  a->vec_y = q3s::aligned16(a->y) && (a->ldy * size % 16 == 0 || a->M == 1);
  if (a->M == 1) a->ldy = (a->ldy * size + 15) / 16 * 16 / size;
  a->error_word = d->error_word;
  *go = true;
  return Q3S_OK;
}

q3s_status cuda_status(cudaError_t e, const char* who) {
  if (e != cudaSuccess) return q3s::report(Q3S_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
  return q3s::report(Q3S_OK, "");
}
cudaError_t quantize(const q3s::QuantArgs& a, int elem, bool vec, cudaStream_t st) {
  return elem == Q3S_ELEM_F32    ? launch_quantize<Q3S_ELEM_F32>(a, vec, st)
         : elem == Q3S_ELEM_BF16 ? launch_quantize<Q3S_ELEM_BF16>(a, vec, st)
                                 : launch_quantize<Q3S_ELEM_F16>(a, vec, st);
}
cudaError_t matmul(const q3s::Int8Args& a, int elem, cudaStream_t st) {
  return elem == Q3S_ELEM_F32    ? launch_matmul<Q3S_ELEM_F32>(a, st)
         : elem == Q3S_ELEM_BF16 ? launch_matmul<Q3S_ELEM_BF16>(a, st)
                                 : launch_matmul<Q3S_ELEM_F16>(a, st);
}

}  // namespace

extern "C" q3s_status q3s_quantize_rows(const q3s_quantize_rows_desc* d, void* stream) {
  q3s::QuantArgs a;
  bool vec, go;
  const q3s_status s = quant_args(d, "q3s_quantize_rows", &a, &vec, &go);
  if (!go) return s;
  return cuda_status(quantize(a, d->elem, vec, static_cast<cudaStream_t>(stream)), "q3s_quantize_rows");
}

extern "C" q3s_status q3s_int8_matmul(const q3s_int8_matmul_desc* d, void* stream) {
  q3s::Int8Args a;
  bool go;
  const q3s_status s = matmul_args(d, "q3s_int8_matmul", &a, &go);
  if (!go) return s;
  return cuda_status(matmul(a, d->elem, static_cast<cudaStream_t>(stream)), "q3s_int8_matmul");
}

extern "C" q3s_status q3s_int8_linear(const q3s_quantize_rows_desc* q, const q3s_int8_matmul_desc* d, void* stream) {
  const char* who = "q3s_int8_linear";
  q3s::QuantArgs qa;
  q3s::Int8Args a;
  bool vec, go, product;
  q3s_status s = quant_args(q, who, &qa, &vec, &go);
  if (s != Q3S_OK) return s;
  s = matmul_args(d, who, &a, &product);
  if (s != Q3S_OK) return s;
  if (q->rows != d->rows || q->cols != d->inputs || q->elem != d->elem || q->values != d->a || q->scales != d->a_scales ||
      (q->rows > 1 && q->values_row_stride != d->a_row_stride))
    return q3s::report(Q3S_ERR_INVALID_ARGUMENT, "%s: the product's left operand must be the quantised rows, of y's type", who);
  if (!go) return q3s::report(Q3S_OK, "");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vec && few_rows(a.M, a.K))  // one launch
    return cuda_status(d->elem == Q3S_ELEM_F32    ? launch_gemv<true, Q3S_ELEM_F32>(a, qa, st)
                       : d->elem == Q3S_ELEM_BF16 ? launch_gemv<true, Q3S_ELEM_BF16>(a, qa, st)
                                                  : launch_gemv<true, Q3S_ELEM_F16>(a, qa, st),
                       who);
  const cudaError_t e = quantize(qa, q->elem, vec, st);
  if (e != cudaSuccess) return cuda_status(e, who);
  return cuda_status(matmul(a, d->elem, st), who);
}

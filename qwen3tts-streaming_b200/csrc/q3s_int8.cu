// q3s_int8.cu -- host side of the 8-bit projections: q3s_quantize_rows and
// q3s_int8_matmul.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
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
  if (vec)
    q3s::quantize_rows_kernel<ELEM, true><<<a.M, 128, 0, st>>>(a);
  else
    q3s::quantize_rows_kernel<ELEM, false><<<a.M, 128, 0, st>>>(a);
  return cudaGetLastError();
}

template <int BN, int ELEM>
cudaError_t launch_matmul(const CUtensorMap& ta, const CUtensorMap& tw, const q3s::Int8Args& a, cudaStream_t st) {
  using Tile = q3s::I8Tile<BN>;
  auto kern = q3s::int8_matmul_kernel<BN, ELEM>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = q3s::allow_smem(kern, Tile::SMEM, done);
  if (e != cudaSuccess) return e;
  const int grid = std::min(a.mtiles * a.ntiles, q3s::sm_count());
  return q3s::launch_maybe_pdl(kern, dim3(grid), dim3(q3s::I8_NT), Tile::SMEM, st, true, ta, tw, a);
}

template <int BN>
cudaError_t launch_matmul_elem(int elem, const CUtensorMap& ta, const CUtensorMap& tw, const q3s::Int8Args& a,
                               cudaStream_t st) {
  if (elem == Q3S_ELEM_F32) return launch_matmul<BN, Q3S_ELEM_F32>(ta, tw, a, st);
  if (elem == Q3S_ELEM_BF16) return launch_matmul<BN, Q3S_ELEM_BF16>(ta, tw, a, st);
  return launch_matmul<BN, Q3S_ELEM_F16>(ta, tw, a, st);
}

bool known_elem(int e) { return e == Q3S_ELEM_F32 || e == Q3S_ELEM_BF16 || e == Q3S_ELEM_F16; }

}  // namespace

extern "C" q3s_status q3s_quantize_rows(const q3s_quantize_rows_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_quantize_rows: desc is NULL");
  if (d->struct_size != sizeof(q3s_quantize_rows_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_quantize_rows: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_quantize_rows_desc)));
  if (d->rows < 0 || d->cols < 1)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_quantize_rows: rows must not be negative and cols must be positive");
  if (!known_elem(d->elem)) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_quantize_rows: unknown elem %d", d->elem);
  if (d->rows == 0) return report(Q3S_OK, "");
  if (!d->x || !d->values || !d->scales)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_quantize_rows: x, values and scales are required");
  if (d->rows > 1 && (d->x_row_stride < d->cols || d->values_row_stride < d->cols))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_quantize_rows: row strides are below cols");
  q3s::QuantArgs a;
  a.M = d->rows;
  a.K = d->cols;
  a.x = d->x;
  a.ldx = d->x_row_stride;
  a.values = d->values;
  a.ldv = d->values_row_stride;
  a.scales = d->scales;
  const int n = d->elem == Q3S_ELEM_F32 ? 4 : 8;  // elements in 16 bytes
  const bool vec = a.K % n == 0 && q3s::aligned16(a.x) && reinterpret_cast<uintptr_t>(a.values) % n == 0 &&
                   (a.M == 1 || (a.ldx % n == 0 && a.ldv % n == 0));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->elem == Q3S_ELEM_F32    ? launch_quantize<Q3S_ELEM_F32>(a, vec, st)
                        : d->elem == Q3S_ELEM_BF16 ? launch_quantize<Q3S_ELEM_BF16>(a, vec, st)
                                                   : launch_quantize<Q3S_ELEM_F16>(a, vec, st);
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_quantize_rows: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}

extern "C" q3s_status q3s_int8_matmul(const q3s_int8_matmul_desc* d, void* stream) {
  using q3s::report;
  if (!d) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: desc is NULL");
  if (d->struct_size != sizeof(q3s_int8_matmul_desc))
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: struct_size %u != %u (ABI mismatch)", d->struct_size,
                  static_cast<unsigned>(sizeof(q3s_int8_matmul_desc)));
  if (d->rows < 0 || d->outputs < 1)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: rows must not be negative and outputs must be positive");
  if (d->inputs < 16 || d->inputs % 16 || d->inputs > 131072)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: inputs %d is not a multiple of 16 in [16, 131072]", d->inputs);
  if (!known_elem(d->elem)) return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: unknown elem %d", d->elem);
  if (d->rows == 0) return report(Q3S_OK, "");
  if (!d->a || !d->a_scales || !d->w || !d->w_scales || !d->y)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: a, a_scales, w, w_scales and y are required");
  const int64_t lda = d->rows > 1 ? d->a_row_stride : d->inputs, ldw = d->outputs > 1 ? d->w_row_stride : d->inputs;
  if (!q3s::aligned16(d->a) || !q3s::aligned16(d->w) || lda < d->inputs || lda % 16 || ldw < d->inputs || ldw % 16)
    return report(Q3S_ERR_INVALID_ARGUMENT,
                  "q3s_int8_matmul: rows of a and w must start on 16 bytes, with strides of at least inputs");
  if (d->rows > 1 && d->y_row_stride < d->outputs)
    return report(Q3S_ERR_INVALID_ARGUMENT, "q3s_int8_matmul: y_row_stride is below outputs");
  q3s::Int8Args a;
  a.M = d->rows;
  a.N = d->outputs;
  a.K = d->inputs;
  a.a_scales = d->a_scales;
  a.w_scales = d->w_scales;
  a.bias = d->bias;
  a.y = d->y;
  a.ldy = d->y_row_stride;
  a.error_word = d->error_word;
  const int per16 = d->elem == Q3S_ELEM_F32 ? 4 : 8;
  a.vec_y = q3s::aligned16(a.y) && (a.M == 1 || a.ldy % per16 == 0);
  a.mtiles = (a.M + q3s::I8_BM - 1) / q3s::I8_BM;
  a.kchunks = (a.K + q3s::I8_BK - 1) / q3s::I8_BK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int bn = 128;
  a.ntiles = (a.N + bn - 1) / bn;
  if (static_cast<int64_t>(a.mtiles) * a.ntiles > 0x7fffffffll)
    return report(Q3S_ERR_UNSUPPORTED, "q3s_int8_matmul: %d x %d outputs are too many", a.M, a.N);
  CUtensorMap ta, tw;
  if (!byte_map(&ta, d->a, a.M, a.K, lda, q3s::I8_BM) || !byte_map(&tw, d->w, a.N, a.K, ldw, bn))
    return report(Q3S_ERR_CUDA, "q3s_int8_matmul: cuTensorMapEncodeTiled failed or is unavailable");
  const cudaError_t e = launch_matmul_elem<128>(d->elem, ta, tw, a, st);
  if (e != cudaSuccess) return report(Q3S_ERR_CUDA, "q3s_int8_matmul: launch failed: %s", cudaGetErrorString(e));
  return report(Q3S_OK, "");
}

// Shared by the kernels of the 8-bit integer product (gemm_i8_sm100.cu: entry point and many tokens, gemm_i8_stream_sm100.cu: few tokens,
// gemm_i8_split_sm100.cu: in between):
//   out[t, f] = act(sx[t] sw[f] sum_k x[t, k] w[f, k] + bias[f]) + residual[t, f]
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention_sm100.cuh"
#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

constexpr int I8_BK = 128;   // columns of a box: 128-byte swizzled rows
constexpr int I8_GATED = 5;  // act: 16 gate rows of the weight, then their 16 up rows

struct I8Gemm {
  const int8_t *x, *w;
  const float *sx, *sw;
  __nv_bfloat16* out;
  const __nv_bfloat16 *bias, *residual;
  long long ldx, ldw, ld_out, ld_res;
  int tokens, features, k, act, early;
  uint32_t* status;
};

// One rounding each for the sum, the scale, their product and the bias (no contraction: every kernel gives the same bits).
__device__ __forceinline__ float i8_value(int sum, float sx, float sw, float bias) {
  return __fadd_rn(__fmul_rn(__int2float_rn(sum), __fmul_rn(sx, sw)), bias);
}
// x sigmoid(u).  The hardware's exponential and quotient are off by about 2^-21 (|u| 2^-24 more for large |u|), far below the rounding to bf16 that follows;
// expf and the IEEE division made the epilogue of a 256 x 256 tile longer than its products (8192 x 22016 x 4096, gated: 732 us).
__device__ __forceinline__ float i8_gate(float x, float u) { return __fdividef(x, 1.f + __expf(-u)); }
// v Phi(v).  Half of erfc(v / sqrt 2), v >= 0, as a polynomial in t = 1 / (1 + 0.245 v) times exp(-v^2 / 2): coefficients of the least greatest error in units of
// (value + 0.001), found by reweighted least squares over 0 .. 14.  With the coefficients as they stand half of erfc is off by 3.0e-8 (5.3e-6 of it up to v = 5, 1.5e-4 up
// to 8, 1.2e-3 up to 13), v times it by 6.6e-9; fp32 adds a few 2^-24 of the terms.  With erff, whose two branches a warp walks
// one after the other, the epilogue of 2820 x 11648 x 1088 took longer than its products.
__device__ __forceinline__ float i8_gelu(float v) {
  const float t = __fdividef(1.f, __fmaf_rn(0.245f, fabsf(v), 1.f));
  float s = -0.109306395f;
  s = __fmaf_rn(s, t, 0.447354406f);
  s = __fmaf_rn(s, t, -0.449595600f);
  s = __fmaf_rn(s, t, 0.443083793f);
  s = __fmaf_rn(s, t, -0.0574047603f);
  s = __fmaf_rn(s, t, 0.131341979f);
  s = __fmaf_rn(s, t, 0.0945266038f);
  const float q = s * t * __expf(-0.5f * v * v);
  return v * (v < 0.f ? q : 1.f - q);
}
// act = 1 relu, 2 gelu, 3 gelu (tanh form: 0.5 x (1 + tanh(u)) = x sigmoid(2u)), 4 silu
template <int N>
__device__ __forceinline__ void i8_activate(float (&v)[N], int act) {
  switch (act) {
    case 1:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];  // (NaN stays)
      break;
    case 2:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = i8_gelu(v[j]);
      break;
    case 3:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = i8_gate(v[j], 1.5957691216057308f * (v[j] + 0.044715f * v[j] * v[j] * v[j]));
      break;
    case 4:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = i8_gate(v[j], v[j]);
      break;
  }
}

// Tokens t0 .. t0 + N of feature m, for the kernels whose lanes are features: neighbouring lanes of a warp have neighbouring features, m_ok says whether this lane's
// exists, sx points to the scales of the tokens, res are the residual's values.  Called by whole warps.
template <int N>
__device__ __forceinline__ void i8_finish(const I8Gemm& g, const int (&sum)[N], const float* sx, int t0, int m, bool m_ok, float sw, float bias, const float* res) {
  float v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = i8_value(sum[j], sx[j], sw, bias);
  int col = m;
  if (g.act == I8_GATED) {  // lanes 0-15 hold gate rows, lanes 16-31 the matching up rows
    col = (m >> 5) * 16 + (m & 15);
    m_ok = m_ok && !(m & 16);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float up = __shfl_xor_sync(0xffffffffu, v[j], 16);
      v[j] = i8_gate(v[j], v[j]) * up;
    }
  } else {
    i8_activate(v, g.act);
    if (g.residual) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += res[j];
    }
  }
  if (!m_ok) return;
  __nv_bfloat16* out = g.out + t0 * g.ld_out + col;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (t0 + j < g.tokens) out[j * g.ld_out] = __float2bfloat16(v[j]);
}
// The residual of those tokens (zeros without one).  Addresses past the end are drawn back into the matrix: loads that no branch keeps apart are in flight together.
template <int N>
__device__ __forceinline__ void i8_residual(const I8Gemm& g, float (&res)[N], int t0, int m) {
  if (!g.residual) {
#pragma unroll
    for (int j = 0; j < N; ++j) res[j] = 0.f;
    return;
  }
  const uint16_t* at = reinterpret_cast<const uint16_t*>(g.residual) + min(m, g.features - 1);
  uint16_t raw[N];
#pragma unroll
  for (int j = 0; j < N; ++j) raw[j] = at[min(t0 + j, g.tokens - 1) * g.ld_res];
#pragma unroll
  for (int j = 0; j < N; ++j) res[j] = bf16_bits_to_float(raw[j]);
}

// [rows, k] bytes, row pitch ld; box = [box_rows][128 columns], 128-byte swizzle.  What lies past k is not read: it arrives as zeros.
inline int i8_tmap(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t k, uint64_t ld, uint32_t box_rows) {
  EncodeTiledFn fn = fa_encode_fn();
  if (!fn) return TPB_ERR_DRIVER;
  cuuint64_t dims[2] = {k, rows}, strides[1] = {ld};
  cuuint32_t box[2] = {I8_BK, box_rows}, estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? TPB_OK
             : TPB_ERR_TMAP;
}

int gemm_i8_stream_launch(const I8Gemm& g, int sms, cudaStream_t stream);  // at most 64 tokens
// bn tokens of a tile (32, 64, 128), CTAs that share its contraction (1, 2, 4, 8; at most one per k-block of 128 columns; bn / splits at least 8)
bool gemm_i8_split_pick(int tokens, int features, int k, int sms, int* bn, int* splits);  // false: another kernel is faster
int gemm_i8_split_launch(const I8Gemm& g, int bn, int splits, cudaStream_t stream);

cudaError_t gemm_i8_stream_preload();
cudaError_t gemm_i8_split_preload();
cudaError_t rows_int8_preload();

}  // namespace tpb

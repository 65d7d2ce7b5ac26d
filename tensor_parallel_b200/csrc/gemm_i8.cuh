// Shared by the kernels of the 8-bit integer product (gemm_i8_sm100.cu: entry point and many tokens, gemm_i8_stream_sm100.cu: few tokens):
//   out[t, f] = act(sx[t] sw[f] sum_k x[t, k] w[f, k] + bias[f]) + residual[t, f]
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention_sm100.cuh"
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
__device__ __forceinline__ float i8_silu(float x) { return x / (1.f + expf(-x)); }
__device__ __forceinline__ float i8_act(float x, int act) {
  switch (act) {
    case 1: return fmaxf(x, 0.f);
    case 2: return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    case 3: return 0.5f * x * (1.f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x)));
    case 4: return i8_silu(x);
    default: return x;
  }
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

}  // namespace tpb

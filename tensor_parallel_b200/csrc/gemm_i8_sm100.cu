// Matrix product of 8-bit integers with a scale per token and per output channel:
//   out[t, f] = act(sx[t] sw[f] sum_k x[t, k] w[f, k] + bias[f]) + residual[t, f]
// The sum is exact (32-bit integers; k <= 131071, so that even rows of -128 stay below 2^31), the rest is fp32, rounded once to bf16.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

constexpr int I8_MAX_K = 131071;
constexpr int I8_GATED = 5;  // act: 16 gate rows of the weight, then their 16 up rows

struct I8Gemm {
  const int8_t *x, *w;
  const float *sx, *sw;
  __nv_bfloat16* out;
  const __nv_bfloat16 *bias, *residual;
  long long ldx, ldw, ld_out, ld_res;
  int tokens, features, k, act;
};

__device__ __forceinline__ float i8_act(float x, int act) {
  switch (act) {
    case 1: return fmaxf(x, 0.f);
    case 2: return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    case 3: return 0.5f * x * (1.f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x)));
    case 4: return x / (1.f + expf(-x));
    default: return x;
  }
}

// 64 x 64 outputs per CTA on the integer dot products of the CUDA cores, 4 x 4 per thread: columns ty, ty + 16, .. of the tokens and tx,
// tx + 16, .. of the features, so that a gate column and its up column are one thread's.
constexpr int I8_TILE = 64, I8_STEP = 64;
__global__ void __launch_bounds__(256)
gemm_i8_kernel(const I8Gemm p) {
  __shared__ int xs[I8_TILE][I8_STEP / 4 + 1], ws[I8_TILE][I8_STEP / 4 + 1];
  pdl_wait();
  pdl_trigger();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int t0 = blockIdx.y * I8_TILE, f0 = blockIdx.x * I8_TILE;
  int acc[4][4] = {};
  auto word = [&](const int8_t* rows, long long ld, int row, int count, int k0) {  // 4 bytes of a row, zero where it has ended
    uint32_t v = 0;
    if (row < count) {
      const int8_t* at = rows + row * ld + k0;
      for (int i = 0; i < 4; ++i)
        if (k0 + i < p.k) v |= uint32_t(uint8_t(at[i])) << (8 * i);
    }
    return int(v);
  };
  for (int k0 = 0; k0 < p.k; k0 += I8_STEP) {
    for (int i = threadIdx.x; i < I8_TILE * I8_STEP / 4; i += 256) {
      const int r = i / (I8_STEP / 4), c = i % (I8_STEP / 4);
      xs[r][c] = word(p.x, p.ldx, t0 + r, p.tokens, k0 + 4 * c);
      ws[r][c] = word(p.w, p.ldw, f0 + r, p.features, k0 + 4 * c);
    }
    __syncthreads();
    for (int c = 0; c < I8_STEP / 4; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xs[ty + 16 * i][c], ws[tx + 16 * j][c], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + ty + 16 * i;
    if (t >= p.tokens) continue;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int f = f0 + tx + 16 * j;
      v[j] = f < p.features ? float(acc[i][j]) * (p.sx[t] * p.sw[f]) + (p.bias ? __bfloat162float(p.bias[f]) : 0.f) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int f = f0 + tx + 16 * j;
      if (f >= p.features || (p.act == I8_GATED && (j & 1))) continue;
      const int c = p.act == I8_GATED ? (f >> 5) * 16 + (f & 15) : f;
      float r = p.act == I8_GATED ? i8_act(v[j], 4) * v[(j + 1) & 3] : i8_act(v[j], p.act);
      if (p.residual) r += __bfloat162float(p.residual[t * p.ld_res + c]);
      p.out[t * p.ld_out + c] = __float2bfloat16(r);
    }
  }
}

}  // namespace tpb

extern "C" int tpb_gemm_int8(const int8_t* x, const float* sx, const int8_t* w, const float* sw, void* out, const void* bias, const void* residual,
                             int tokens, int features, int k, long long ldx, long long ldw, long long ld_out, long long ld_res, int act, int early, void* status,
                             void* stream) {
  using bf16 = __nv_bfloat16;
  if (!x || !sx || !w || !sw || !out || !status || tokens <= 0 || features <= 0 || k <= 0 || act < 0 || act > tpb::I8_GATED) return TPB_ERR_ARG;
  if (k > tpb::I8_MAX_K) return TPB_ERR_SIZE;
  const int cols = act == tpb::I8_GATED ? features / 2 : features;
  if (act == tpb::I8_GATED && (features % 32 || residual)) return TPB_ERR_ARG;
  if (ldx < k || ldw < k || ld_out < cols || (residual && ld_res < cols)) return TPB_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) || ldx % 16 || ldw % 16) return TPB_ERR_ALIGN;
  tpb::I8Gemm p = {x, w, sx, sw, static_cast<bf16*>(out), static_cast<const bf16*>(bias), static_cast<const bf16*>(residual), ldx, ldw, ld_out, ld_res,
                   tokens, features, k, act};
  const dim3 grid((features + tpb::I8_TILE - 1) / tpb::I8_TILE, (tokens + tpb::I8_TILE - 1) / tpb::I8_TILE);
  if (grid.y > 65535) return TPB_ERR_SIZE;
  return tpb::launch_dependent(tpb::gemm_i8_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), early != 0, p) == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

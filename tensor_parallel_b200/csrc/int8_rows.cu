// Rows in 8-bit integers with a scale each: as they are (activations, weights), or RMSNorm / LayerNorm of x (+ residual).
//   v = h                             scale = amax / 127
//   v = h w                (RMSNorm)  scale = amax rstd / 127
//   v = (h - mean) rstd w + b         scale = amax / 127
// with amax = max(max |v|, 1e-30) over the row and q = rint(v (127 / amax)).  An RMSNorm's rstd is common to the row, so it only enters
// the scale: the integers depend on no order of summation, and a row needs one exchange (sum of squares and maximum together) instead of two.
// A row with a value that is not finite gets integers 0 and the scale NaN, so that everything computed from it is NaN.
//
// Memory-bound: x and the residual are read once, h and the integers written once; a row waits in registers, in its own type, for its
// statistics.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

typedef __nv_bfloat16 bf16;

constexpr int RI_ROWS = 0, RI_RMS = 1, RI_LAYER = 2;
constexpr int RI_MAX_THREADS = 1024;
constexpr float RI_LEAST = 1e-30f;  // 127 / 1e-30 is finite, and half a step of such a row is 4e-33

struct RiParams {
  const void *x, *residual, *weight, *bias;
  void* sum_out;
  int8_t* q;
  float* scales;
  long long ldx, ldr, lds, ldq;  // row pitches in elements
  int rows, cols;
  float eps;
};

__device__ __forceinline__ float ri_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float ri_float(float x) { return x; }
template <typename T> __device__ __forceinline__ T ri_round(float x);
template <> __device__ __forceinline__ bf16 ri_round<bf16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ float ri_round<float>(float x) { return x; }

template <typename T> struct __align__(16) Ri8 { T e[8]; };  // 8 elements of a thread

// Columns of a thread: V groups of 8.  VEC: 8 consecutive columns each, rows on 16-byte boundaries; else the lanes of a warp own consecutive
// columns, so that rows of any width and alignment are read and written in whole sectors.
template <bool VEC>
__device__ __forceinline__ int ri_col(int base, int i, int j) {
  return VEC ? base + (int(threadIdx.x) + i * int(blockDim.x)) * 8 + j : base + int(threadIdx.x) + (i * 8 + j) * int(blockDim.x);
}
template <typename T, bool VEC>
__device__ __forceinline__ Ri8<T> ri_load(const T* row, int base, int i, int cols) {
  Ri8<T> r;
  if constexpr (VEC) {
    const int c = ri_col<true>(base, i, 0);
#pragma unroll
    for (int u = 0; u < int(sizeof(T) / 2); ++u)
      reinterpret_cast<uint4*>(&r)[u] = c < cols ? reinterpret_cast<const uint4*>(row + c)[u] : make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = ri_col<false>(base, i, j);
      r.e[j] = c < cols ? row[c] : ri_round<T>(0.f);
    }
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void ri_store(T* row, int base, int i, int cols, const Ri8<T>& r) {
  if constexpr (VEC) {
    const int c = ri_col<true>(base, i, 0);
    if (c < cols) {
#pragma unroll
      for (int u = 0; u < int(sizeof(T) / 2); ++u) reinterpret_cast<uint4*>(row + c)[u] = reinterpret_cast<const uint4*>(&r)[u];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = ri_col<false>(base, i, j);
      if (c < cols) row[c] = r.e[j];
    }
  }
}

// Over the threads of a row: the sum of a, and the maximum of b (non-negative floats order as their bits do, with NaN above infinity).
template <bool SUM, bool MAX>
__device__ __forceinline__ void ri_reduce(float& a, uint32_t& b, float* sums, uint32_t* maxima) {
  if (SUM) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  if (MAX) b = __reduce_max_sync(0xffffffffu, b);
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return;
  sums += threadIdx.y * warps;
  maxima += threadIdx.y * warps;
  __syncthreads();
  if (lane == 0) {
    if (SUM) sums[warp] = a;
    if (MAX) maxima[warp] = b;
  }
  __syncthreads();
  if (SUM) {
    a = lane < warps ? sums[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  if (MAX) b = __reduce_max_sync(0xffffffffu, lane < warps ? maxima[lane] : 0u);
}

// A block of blockDim.y rows, blockDim.x threads each.  WIDE: rows of more than 8 V blockDim.x columns, read again from memory for every pass.
template <typename T, int MODE, int V, bool VEC, bool WIDE>
__global__ void __launch_bounds__(RI_MAX_THREADS)
rows_int8_kernel(const RiParams p) {
  __shared__ float sums[32];
  __shared__ uint32_t maxima[32];
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const int cols = row < p.rows ? p.cols : 0;  // (a row past the end still takes part in the block's barriers)
  const int chunk = 8 * V * int(blockDim.x);
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* residual = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
  T* sum_out = p.sum_out ? static_cast<T*>(p.sum_out) + row * p.lds : nullptr;
  const T* weight = static_cast<const T*>(p.weight);
  const T* bias = static_cast<const T*>(p.bias);

  Ri8<T> h[V];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = ri_load<T, VEC>(x, base, i, cols);
    if (MODE != RI_ROWS && residual) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const Ri8<T> r = ri_load<T, VEC>(residual, base, i, cols);
        // rounded to the type it is stored in: the norm is taken of what later kernels read
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i].e[j] = ri_round<T>(ri_float(h[i].e[j]) + ri_float(r.e[j]));
        if (sum_out) ri_store<T, VEC>(sum_out, base, i, cols, h[i]);
      }
    }
  };
  auto fetch_again = [&](int base) {
    if (!WIDE) return;  // (still in registers)
    if (MODE != RI_ROWS && residual && sum_out) {  // (x may have been overwritten by the sum: what this thread stored)
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = ri_load<T, VEC>(sum_out, base, i, cols);
    } else {
      fetch(base);
    }
  };
  const int end = WIDE ? cols : 1;

  float mean = 0.f, rstd = 0.f, sum = 0.f;
  uint32_t most = 0;
  auto values = [&](int base, int i, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ri_float(h[i].e[j]);
    if (MODE == RI_RMS && weight) {
      const Ri8<T> w = ri_load<T, VEC>(weight, base, i, cols);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], ri_float(w.e[j]));
    }
    if (MODE == RI_LAYER) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (v[j] - mean) * rstd;
      if (weight) {
        const Ri8<T> w = ri_load<T, VEC>(weight, base, i, cols);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= ri_float(w.e[j]);
      }
      if (bias) {
        const Ri8<T> b = ri_load<T, VEC>(bias, base, i, cols);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += ri_float(b.e[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (ri_col<VEC>(base, i, j) >= cols) v[j] = 0.f;
    }
  };
  auto raise = [&](const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(fabsf(v[j])));
  };

  pdl_wait();
  pdl_trigger();
  for (int base = 0; base < end; base += chunk) {
    fetch(base);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (MODE == RI_RMS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { const float f = ri_float(h[i].e[j]); sum += f * f; }
      }
      if (MODE == RI_LAYER) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += ri_float(h[i].e[j]);
      } else {
        float v[8];
        values(base, i, v);
        raise(v);
      }
    }
  }
  if (MODE == RI_ROWS) {
    ri_reduce<false, true>(sum, most, sums, maxima);
  } else if (MODE == RI_RMS) {
    ri_reduce<true, true>(sum, most, sums, maxima);
    rstd = rsqrtf(sum / float(p.cols) + p.eps);
  } else {
    // (the deviations are summed up around the mean: a difference of two sums would lose the digits that they share)
    ri_reduce<true, false>(sum, most, sums, maxima);
    mean = sum / float(p.cols);
    float squares = 0.f;
    for (int base = 0; base < end; base += chunk) {
      fetch_again(base);
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = ri_float(h[i].e[j]) - mean;
          if (ri_col<VEC>(base, i, j) < cols) squares += d * d;
        }
      }
    }
    ri_reduce<true, false>(squares, most, sums, maxima);
    rstd = rsqrtf(squares / float(p.cols) + p.eps);
    for (int base = 0; base < end; base += chunk) {
      fetch_again(base);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v[8];
        values(base, i, v);
        raise(v);
      }
    }
    ri_reduce<false, true>(sum, most, sums, maxima);
  }

  const bool finite = most < 0x7F800000u;
  const float amax = fmaxf(__uint_as_float(most), RI_LEAST);
  const float inv = __fdiv_rn(127.f, amax);
  if (threadIdx.x == 0 && row < p.rows) p.scales[row] = finite ? amax / 127.f * (MODE == RI_RMS ? rstd : 1.f) : __int_as_float(0x7FC00000);
  int8_t* q = p.q + row * p.ldq;
  for (int base = 0; base < end; base += chunk) {
    fetch_again(base);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v[8];
      values(base, i, v);
      uint32_t b[8];
      // v inv is rounded to fp32, then, by the addition of 1.5 2^23, to the nearest integer (ties to even), whose two's complement the low bits are
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = finite ? __float_as_uint(__fadd_rn(__fmul_rn(v[j], inv), 12582912.f)) : 0u;
      if constexpr (VEC) {
        const int c = ri_col<true>(base, i, 0);
        if (c < cols) {
          uint2 w;
          w.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
          w.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
          *reinterpret_cast<uint2*>(q + c) = w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = ri_col<false>(base, i, j);
          if (c < cols) q[c] = int8_t(b[j] & 0xFFu);
        }
      }
    }
  }
}

template <typename T, int MODE, bool VEC>
static cudaError_t ri_launch(const RiParams& p, bool early, cudaStream_t stream) {
  const int groups = (p.cols + 7) / 8;
  const int v = groups <= 256 ? 1 : groups <= 2048 ? 2 : 4;
  int threads = ((groups + v - 1) / v + 31) / 32 * 32;
  const bool wide = threads > RI_MAX_THREADS;
  if (wide) threads = RI_MAX_THREADS;
  const int rows_per_block = threads >= 256 ? 1 : 256 / threads;
  const dim3 block(threads, rows_per_block), grid((unsigned(p.rows) + rows_per_block - 1) / rows_per_block);
  auto go = [&](auto kernel) { return launch_dependent(kernel, grid, block, 0, stream, early, p); };
  if (wide) return go(rows_int8_kernel<T, MODE, 4, VEC, true>);
  if (v == 1) return go(rows_int8_kernel<T, MODE, 1, VEC, false>);
  if (v == 2) return go(rows_int8_kernel<T, MODE, 2, VEC, false>);
  return go(rows_int8_kernel<T, MODE, 4, VEC, false>);
}

template <typename T>
static cudaError_t ri_dispatch(const RiParams& p, int mode, bool early, cudaStream_t stream) {
  auto rows_aligned = [](const void* base, long long ld) { return !(reinterpret_cast<uintptr_t>(base) & 15) && (ld * sizeof(T)) % 16 == 0; };
  const bool vec = p.cols % 8 == 0 && rows_aligned(p.x, p.ldx) && rows_aligned(p.residual, p.ldr) && rows_aligned(p.sum_out, p.lds) &&
                   rows_aligned(p.weight, 0) && rows_aligned(p.bias, 0) && !(reinterpret_cast<uintptr_t>(p.q) & 7) && p.ldq % 8 == 0;
#define RI_GO(MODE) (vec ? ri_launch<T, MODE, true>(p, early, stream) : ri_launch<T, MODE, false>(p, early, stream))
  return mode == RI_ROWS ? RI_GO(RI_ROWS) : mode == RI_RMS ? RI_GO(RI_RMS) : RI_GO(RI_LAYER);
#undef RI_GO
}

}  // namespace tpb

extern "C" int tpb_rows_int8(const void* x, const void* residual, const void* weight, const void* bias, void* sum_out, int8_t* q, float* scales, int rows,
                             int cols, long long ldx, long long ldr, long long lds, long long ldq, float eps, int mode, int dtype, int early, void* stream) {
  if (!x || !q || !scales || rows <= 0 || cols <= 0 || mode < 0 || mode > 2 || dtype < 0 || dtype > 1) return TPB_ERR_ARG;
  if (mode == tpb::RI_ROWS && (residual || weight || bias || sum_out)) return TPB_ERR_ARG;
  if ((bias && mode != tpb::RI_LAYER) || (sum_out && !residual)) return TPB_ERR_ARG;
  if (ldx < cols || ldq < cols || (residual && ldr < cols) || (sum_out && lds < cols)) return TPB_ERR_ARG;
  tpb::RiParams p = {x, residual, weight, bias, sum_out, q, scales, ldx, residual ? ldr : 0, sum_out ? lds : 0, ldq, rows, cols, eps};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == 0 ? tpb::ri_dispatch<tpb::bf16>(p, mode, early != 0, s) : tpb::ri_dispatch<float>(p, mode, early != 0, s);
  return e == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

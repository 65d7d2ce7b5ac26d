// Rows in 8-bit integers with a scale each: as they are (activations, weights), or RMSNorm / LayerNorm of x (+ residual).
//   v = h                             scale = amax / 127
//   v = h w                (RMSNorm)  scale = amax rstd / 127
//   v = (h - mean) rstd w + b         scale = amax / 127
// with amax = max(max |v|, 1e-30) over the row and q = rint(v (127 / amax)).  An RMSNorm's rstd is common to the row, so it only enters
// the scale: the integers depend on no order of summation, and a row needs one exchange (sum of squares and maximum together) instead of two.
// A row with a value that is not finite gets integers 0 and the scale NaN, so that everything computed from it is NaN.  So does the scale of a finite row whose sum of
// squares passes the range of fp32 (a value above 2^64 is enough), instead of the zero that 1 / rms would be.  (Done again with a scaled sum, in the same kernel, such a
// row cost the ordinary ones 2 to 27 % of their time: registers, or a branch per warp.)
//
// Memory-bound: x and the residual are read once, h and the integers written once.  A row waits for its statistics in registers as fp32: in a block of its own, in
// a persistent block that has the next row on its way (norms of many rows), or, where many wide rows need more of them in flight than registers hold, in shared
// memory.  Measured (us, and of the floor at 6549 GB/s), 8192 x 4096 bf16: rows 17.8 (0.86), RMSNorm 20.6 (0.75), with a residual 37.3 (0.96), LayerNorm 27.8 (0.55),
// with a residual 39.0 (0.92); 8192 x 11008 rows 46.8 (0.88).  What is above is instructions (unpacking, maxima, the integers, most of them on the half-rate
// pipe; a LayerNorm meets three times), and 2 us of launch and first latency.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention_sm100.cuh"
#include "gemm_i8.cuh"
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
  int ahead;
  uint32_t* status;
};

// Waits for the kernel in front, and lets the one behind come in: as every kernel does (launch.cuh), or with `ahead` before the wait.  A product behind may then fetch
// its weights while the kernel in front drains (decode step of four 7B layers, batch 8 x 2048, 484 -> 463 us, batch 8 x 64 291 -> 267); its CTAs leave no room for a third,
// so no chain piles up.  What it reads early must then be older than the kernel in front of this one too, which only a caller that knows the chain can vouch for.
__device__ __forceinline__ void ri_begin(int ahead) {
  if (ahead) pdl_trigger();
  pdl_wait();
  pdl_trigger();
}

__device__ __forceinline__ float ri_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float ri_float(float x) { return x; }
template <typename T> __device__ __forceinline__ T ri_round(float x);
template <> __device__ __forceinline__ bf16 ri_round<bf16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ float ri_round<float>(float x) { return x; }

// 8 elements of a thread as they lie in memory (in words: one instruction takes an element out of its word).
template <typename T> struct Ri8 {};
template <> struct Ri8<bf16> {
  static constexpr int WORDS = 4;
  uint32_t w[4];
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(j & 1 ? w[j >> 1] & 0xFFFF0000u : w[j >> 1] << 16); }
  __device__ __forceinline__ void set2(int j, float a, float b) { w[j >> 1] = pack_bf16x2(a, b); }
  __device__ __forceinline__ void clear(int j) { w[j >> 1] &= j & 1 ? 0x0000FFFFu : 0xFFFF0000u; }
};
template <> struct Ri8<float> {
  static constexpr int WORDS = 8;
  uint32_t w[8];
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(w[j]); }
  __device__ __forceinline__ void set2(int j, float a, float b) { w[j] = __float_as_uint(a); w[j + 1] = __float_as_uint(b); }
  __device__ __forceinline__ void clear(int j) { w[j] = 0; }
};
template <typename T>
__device__ __forceinline__ Ri8<T> ri_load8(const T* at, bool ok) {  // 16-byte aligned
  Ri8<T> r;
#pragma unroll
  for (int u = 0; u < Ri8<T>::WORDS / 4; ++u) {
    const uint4 q = ok ? reinterpret_cast<const uint4*>(at)[u] : make_uint4(0, 0, 0, 0);
    r.w[4 * u] = q.x;
    r.w[4 * u + 1] = q.y;
    r.w[4 * u + 2] = q.z;
    r.w[4 * u + 3] = q.w;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void ri_store8(T* at, const Ri8<T>& r) {
#pragma unroll
  for (int u = 0; u < Ri8<T>::WORDS / 4; ++u) reinterpret_cast<uint4*>(at)[u] = make_uint4(r.w[4 * u], r.w[4 * u + 1], r.w[4 * u + 2], r.w[4 * u + 3]);
}

// Columns of a thread: V groups of 8 consecutive ones.
__device__ __forceinline__ int ri_col(int base, int i) { return base + (int(threadIdx.x) + i * int(blockDim.x)) * 8; }

// 8 columns of a row from column c on, zeros past its end.  VEC: rows begin on 16 bytes and have a multiple of 8 columns.  Else the columns are taken out of the
// aligned 16-byte blocks that hold them (and a few bytes of their neighbours, which lie in the same blocks), which costs two instructions per element.
template <typename T, bool VEC>
__device__ __forceinline__ Ri8<T> ri_load(const T* row, int c, int cols) {
  if constexpr (VEC) return ri_load8(row + c, c < cols);
  constexpr int BLOCKS = sizeof(T) / 2 + 1, WORDS = Ri8<T>::WORDS;
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c), end = reinterpret_cast<uintptr_t>(row + cols);
  const uint32_t skip = uint32_t(at) & 15;  // (the same for all groups of a row)
  uint32_t w[4 * BLOCKS];
#pragma unroll
  for (int u = 0; u < BLOCKS; ++u) {
    const uintptr_t block = at - skip + 16 * u;
    const uint4 q = c < cols && block < end ? *reinterpret_cast<const uint4*>(block) : make_uint4(0, 0, 0, 0);
    w[4 * u] = q.x;
    w[4 * u + 1] = q.y;
    w[4 * u + 2] = q.z;
    w[4 * u + 3] = q.w;
  }
  if (skip & 4) {
#pragma unroll
    for (int i = 0; i + 1 < 4 * BLOCKS; ++i) w[i] = w[i + 1];
  }
  if (skip & 8) {
#pragma unroll
    for (int i = 0; i + 2 < 4 * BLOCKS; ++i) w[i] = w[i + 2];
  }
  Ri8<T> r;
#pragma unroll
  for (int i = 0; i < WORDS; ++i) r.w[i] = sizeof(T) == 4 ? w[i] : __funnelshift_r(w[i], w[i + 1], (skip & 2) * 8);
  if (c + 8 > cols) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j >= cols) r.clear(j);
  }
  return r;
}
// The same 8 columns back.  Rows of any alignment are turned in the warp's part of shared memory, so that neighbouring lanes store neighbouring columns.
template <typename T, bool VEC>
__device__ __forceinline__ void ri_store(T* row, int c, int cols, const Ri8<T>& r, T* stage) {
  if constexpr (VEC) {
    if (c < cols) ri_store8(row + c, r);
  } else {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    ri_store8(stage + lane * 8, r);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = c - lane * 8 + 32 * j + lane;
      if (d < cols) row[d] = stage[32 * j + lane];
    }
  }
}

// Over the threads of a row: the sum of a, and the maximum of b (non-negative floats order as their bits do, with NaN above infinity).  `sums` and `maxima`
// have not been used yet, or not since the last barrier.  With both, only the row's first warp gets the sum.
template <bool SUM, bool MAX>
__device__ __forceinline__ void ri_reduce(float& a, uint32_t& b, float* sums, uint32_t* maxima) {
  if (MAX) b = __reduce_max_sync(0xffffffffu, b);
  if (SUM) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return;
  sums += threadIdx.y * warps;
  maxima += threadIdx.y * warps;
  if (lane == 0) {
    if (SUM) sums[warp] = a;
    if (MAX) maxima[warp] = b;
  }
  __syncthreads();
  if (MAX) b = __reduce_max_sync(0xffffffffu, lane < warps ? maxima[lane] : 0u);
  if (SUM && (!MAX || warp == 0)) {
    a = lane < warps ? sums[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  }
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// An integer in [-127, 127] stands in the low bits of x + 1.5 2^23, in two's complement, where that sum is rounded to nearest (ties to even).  The four integers
// of v * inv.  `one` is 1, which the compiler does not know: y * one + 1.5 2^23 rounds like the sum, which it would contract with the product in front of it.
constexpr float RI_MAGIC = 12582912.f;
__device__ __forceinline__ uint32_t ri_integers(float2 v0, float2 v1, float inv, float one) {
  const float2 a = __ffma2_rn(__fmul2_rn(v0, both(inv)), both(one), both(RI_MAGIC));
  const float2 b = __ffma2_rn(__fmul2_rn(v1, both(inv)), both(one), both(RI_MAGIC));
  return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

// The scale of a row, by its first thread: of an RMSNorm from the sum of squares, of a LayerNorm with 1 / deviation as it was used.
template <int MODE>
__device__ __forceinline__ float ri_scale(float amax, bool finite, float squares, float rstd, const RiParams& p) {
  const bool in_range = MODE == RI_RMS ? squares <= 3.402823466e38f : MODE == RI_LAYER ? rstd > 0.f : true;
  const float scale = amax / 127.f * (MODE == RI_RMS ? rsqrtf(squares / float(p.cols) + p.eps) : 1.f);
  return finite && in_range ? scale : __int_as_float(0x7FC00000);
}

// Blocks that an SM is to hold: as many registers as the row and its raw words take, without spills to speak of (8192 x 4096, RMSNorm with 8 blocks 28.6 us
// instead of 24.8; with 32 columns a thread, 11008 wide, two blocks of 512 instead of one 76 us instead of 116).
template <typename T, int MODE, int V, bool VEC>
constexpr int ri_blocks(int threads) {
  if (V == 4) return threads > 256 ? 1024 / threads : 3;
  return threads != 256 || !VEC ? 1 : MODE == RI_LAYER ? 4 : V == 1 ? 6 : sizeof(T) == 4 ? 4 : MODE == RI_ROWS ? 8 : 6;
}

// A block of blockDim.y rows, blockDim.x threads each.  WIDE: rows of more than 8 V blockDim.x columns, read again from memory for every pass.
template <typename T, int MODE, int V, bool VEC, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS, ri_blocks<T, MODE, V, VEC>(THREADS))
rows_int8_kernel(const RiParams p, float one) {
  __shared__ float sums[2][32];
  __shared__ uint32_t maxima[32];
  __shared__ __align__(16) T turned[VEC || MODE == RI_ROWS ? 1 : THREADS * 8];
  T* stage = turned + (VEC || MODE == RI_ROWS ? 0 : (threadIdx.y * blockDim.x + threadIdx.x) / 32 * 256);
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const int cols = row < p.rows ? p.cols : 0;  // (a row past the end still takes part in the block's barriers)
  const int chunk = 8 * V * int(blockDim.x);
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* residual = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
  T* sum_out = p.sum_out ? static_cast<T*>(p.sum_out) + row * p.lds : nullptr;
  const T* weight = static_cast<const T*>(p.weight);
  const T* bias = static_cast<const T*>(p.bias);

  Ri8<T> w[V];
  float2 v[V][4];  // the row: h, then the values to be rounded
  auto fetch = [&](int base, bool again) {
    Ri8<T> raw[V];
    // (x may be overwritten by the sum: a second pass reads what its warp stored)
    const bool summed = again && residual && sum_out;
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = ri_load<T, VEC>(summed ? sum_out : x, ri_col(base, i), cols);
    if (MODE != RI_ROWS && residual && !summed) {
      Ri8<T> add[V];
#pragma unroll
      for (int i = 0; i < V; ++i) add[i] = ri_load<T, VEC>(residual, ri_col(base, i), cols);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // rounded to the type it is stored in: the norm is taken of what later kernels read
#pragma unroll
        for (int j = 0; j < 8; j += 2) raw[i].set2(j, raw[i].get(j) + add[i].get(j), raw[i].get(j + 1) + add[i].get(j + 1));
        if (sum_out) ri_store<T, VEC>(sum_out, ri_col(base, i), cols, raw[i], stage);
      }
    }
    if (MODE != RI_ROWS && weight) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = ri_load<T, VEC>(weight, ri_col(base, i), cols);
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = make_float2(raw[i].get(2 * j), raw[i].get(2 * j + 1));
  };
  const int end = WIDE ? cols : 1;

  auto clear_past = [&](int c, float2 (&g)[4]) {  // the columns past the end, of a group at column c
    if (VEC ? c < cols : c + 8 <= cols) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (VEC || c + 2 * j >= cols) g[j].x = 0.f;
      if (VEC || c + 2 * j + 1 >= cols) g[j].y = 0.f;
    }
  };
  // v times the weight (and plus the bias, of a LayerNorm's (h - mean) rstd), and the largest |v|
  float most0 = 0.f, most1 = 0.f;
  auto finish_values = [&](int base, float mean, float rstd) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (MODE == RI_LAYER) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = __fmul2_rn(WIDE ? __fadd2_rn(v[i][j], both(-mean)) : v[i][j], both(rstd));
      }
      if (MODE != RI_ROWS && weight) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = __fmul2_rn(v[i][j], make_float2(w[i].get(2 * j), w[i].get(2 * j + 1)));
      }
      if (MODE == RI_LAYER) {
        if (bias) {
          const Ri8<T> b = ri_load<T, VEC>(bias, ri_col(base, i), cols);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[i][j] = __fadd2_rn(v[i][j], make_float2(b.get(2 * j), b.get(2 * j + 1)));
        }
        if (WIDE) clear_past(ri_col(base, i), v[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        most0 = fmax3_abs_nan(most0, v[i][j].x, v[i][j].y);
        most1 = fmax3_abs_nan(most1, v[i][j + 1].x, v[i][j + 1].y);
      }
    }
  };

  ri_begin(p.ahead);
  float sum = 0.f, rstd = 1.f, mean = 0.f;
  for (int base = 0; base < end; base += chunk) {
    fetch(base, false);
    if (MODE == RI_RMS) {
      float2 squares = both(0.f);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) squares = __ffma2_rn(v[i][j], v[i][j], squares);
      sum += squares.x + squares.y;
    }
    if (MODE == RI_LAYER) {
      float2 total = both(0.f);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) total = __fadd2_rn(total, v[i][j]);
      sum += total.x + total.y;
    } else {
      finish_values(base, 0.f, 1.f);
    }
  }
  uint32_t most = 0;
  if (MODE == RI_LAYER) {
    // (the deviations are summed up around the mean: a difference of two sums would lose the digits that they share)
    ri_reduce<true, false>(sum, most, sums[0], maxima);
    mean = sum / float(p.cols);
    float2 around = both(0.f);
    for (int base = 0; base < end; base += chunk) {
      if (WIDE) fetch(base, true);
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = __fadd2_rn(v[i][j], both(-mean));
        clear_past(ri_col(base, i), v[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) around = __ffma2_rn(v[i][j], v[i][j], around);
      }
    }
    float squares = around.x + around.y;
    ri_reduce<true, false>(squares, most, sums[1], maxima);
    rstd = rsqrtf(squares / float(p.cols) + p.eps);
    for (int base = 0; base < end; base += chunk) {
      if (WIDE) fetch(base, true);
      finish_values(base, mean, rstd);
    }
  }
  most = __float_as_uint(fmax3_abs_nan(most0, most1, 0.f));
  ri_reduce<MODE == RI_RMS, true>(sum, most, sums[0], maxima);

  const bool finite = most < 0x7F800000u;
  const float amax = fmaxf(__uint_as_float(most), RI_LEAST);
  const float inv = __fdiv_rn(127.f, amax);
  if (threadIdx.x == 0 && row < p.rows) {
    p.scales[row] = ri_scale<MODE>(amax, finite, sum, rstd, p);
  }
  int8_t* q = p.q + row * p.ldq;
  const bool whole = VEC || !((reinterpret_cast<uintptr_t>(p.q) | uintptr_t(p.ldq)) & 7);  // 8 integers may be stored at once
  for (int base = 0; base < end; base += chunk) {
    if (WIDE) {
      fetch(base, true);
      finish_values(base, mean, rstd);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      uint2 u = make_uint2(ri_integers(v[i][0], v[i][1], inv, one), ri_integers(v[i][2], v[i][3], inv, one));
      if (!finite) u = make_uint2(0, 0);
      const int c = ri_col(base, i);
      if (VEC || (whole && c + 8 <= cols)) {
        if (c < cols) *reinterpret_cast<uint2*>(q + c) = u;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < cols) q[c + j] = int8_t((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
      }
    }
  }
}

// Norms of many aligned bf16 rows: persistent blocks that keep the weights in registers and have the next row (TWO: and its residual) on its way while they work on
// one.  The exchanges alternate between two sets of shared memory, so that a row of an RMSNorm has one barrier.  At most as many blocks as rows.
constexpr int ri_walk_threads(int v, int threads, bool two) {  // of an SM, by what a thread needs in registers
  return v == 2 ? (two ? 768 : 1024) : threads <= 128 && !two ? 640 : 512;
}
template <int MODE, int V, int THREADS, bool TWO>
__global__ void __launch_bounds__(THREADS, ri_walk_threads(V, THREADS, TWO) / THREADS)
rows_int8_walk_kernel(const RiParams p, float one) {
  __shared__ float sums[2][2][32];
  __shared__ uint32_t maxima[2][32];
  const bf16* weight = static_cast<const bf16*>(p.weight);
  const bf16* bias = static_cast<const bf16*>(p.bias);
  ri_begin(p.ahead);
  Ri8<bf16> next[V], next2[TWO ? V : 1], w[V];
  const bf16* x = static_cast<const bf16*>(p.x) + blockIdx.x * p.ldx;  // (of the row on its way)
  const long long step_x = (long long)gridDim.x * p.ldx, step_q = (long long)gridDim.x * p.ldq;
  int8_t* q = p.q + blockIdx.x * p.ldq;
  const bf16* r = TWO ? static_cast<const bf16*>(p.residual) + blockIdx.x * p.ldr : nullptr;
  bf16* h = TWO && p.sum_out ? static_cast<bf16*>(p.sum_out) + blockIdx.x * p.lds : nullptr;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    next[i] = ri_load<bf16, true>(x, ri_col(0, i), p.cols);
    if (TWO) next2[i] = ri_load<bf16, true>(r, ri_col(0, i), p.cols);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (weight) {
      w[i] = ri_load<bf16, true>(weight, ri_col(0, i), p.cols);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i].w[j] = 0x3F803F80u;  // ones
    }
  }
  int buffer = 0;
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x, q += step_q, buffer ^= 1) {
    float2 v[V][4];
    if (TWO) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // rounded to the type it is stored in: the norm is taken of what later kernels read
#pragma unroll
        for (int j = 0; j < 8; j += 2) next[i].set2(j, next[i].get(j) + next2[i].get(j), next[i].get(j + 1) + next2[i].get(j + 1));
        if (h) ri_store<bf16, true>(h, ri_col(0, i), p.cols, next[i], nullptr);
      }
      if (h) h += (long long)gridDim.x * p.lds;
      r += (long long)gridDim.x * p.ldr;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = make_float2(next[i].get(2 * j), next[i].get(2 * j + 1));
    x += step_x;
    if (row + int(gridDim.x) < p.rows) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        next[i] = ri_load<bf16, true>(x, ri_col(0, i), p.cols);
        if (TWO) next2[i] = ri_load<bf16, true>(r, ri_col(0, i), p.cols);
      }
    }
    float sum = 0.f, rstd = 1.f;
    uint32_t most = 0;
    if (MODE == RI_RMS) {
      float2 squares = both(0.f);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) squares = __ffma2_rn(v[i][j], v[i][j], squares);
      sum = squares.x + squares.y;
    }
    if (MODE == RI_LAYER) {
      float2 total = both(0.f);
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) total = __fadd2_rn(total, v[i][j]);
      sum = total.x + total.y;
      // (the deviations are summed up around the mean: a difference of two sums would lose the digits that they share)
      ri_reduce<true, false>(sum, most, sums[0][buffer], maxima[buffer]);
      const float mean = sum / float(p.cols);
      float2 around = both(0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool in = ri_col(0, i) < p.cols;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[i][j] = in ? __fadd2_rn(v[i][j], both(-mean)) : both(0.f);
          around = __ffma2_rn(v[i][j], v[i][j], around);
        }
      }
      float squares = around.x + around.y;
      ri_reduce<true, false>(squares, most, sums[1][buffer], maxima[buffer]);
      rstd = rsqrtf(squares / float(p.cols) + p.eps);
    }
    float most0 = 0.f, most1 = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Ri8<bf16> b;
      if (MODE == RI_LAYER && bias) b = ri_load<bf16, true>(bias, ri_col(0, i), p.cols);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (MODE == RI_LAYER) v[i][j] = __fmul2_rn(v[i][j], both(rstd));
        v[i][j] = __fmul2_rn(v[i][j], make_float2(w[i].get(2 * j), w[i].get(2 * j + 1)));
        if (MODE == RI_LAYER && bias) v[i][j] = __fadd2_rn(v[i][j], make_float2(b.get(2 * j), b.get(2 * j + 1)));
      }
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        most0 = fmax3_abs_nan(most0, v[i][j].x, v[i][j].y);
        most1 = fmax3_abs_nan(most1, v[i][j + 1].x, v[i][j + 1].y);
      }
    }
    most = __float_as_uint(fmax3_abs_nan(most0, most1, 0.f));
    ri_reduce<MODE == RI_RMS, true>(sum, most, sums[0][buffer], maxima[buffer]);
    const bool finite = most < 0x7F800000u;
    const float amax = fmaxf(__uint_as_float(most), RI_LEAST);
    const float inv = __fdiv_rn(127.f, amax);
    if (threadIdx.x == 0) {
      p.scales[row] = ri_scale<MODE>(amax, finite, sum, rstd, p);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      uint2 u = make_uint2(ri_integers(v[i][0], v[i][1], inv, one), ri_integers(v[i][2], v[i][3], inv, one));
      if (!finite) u = make_uint2(0, 0);
      const int c = ri_col(0, i);
      if (c < p.cols) *reinterpret_cast<uint2*>(q + c) = u;
    }
  }
}

// ---- many wide rows: persistent groups of threads, rows arriving by bulk copies several ahead -------------------------------------------------------

__device__ __forceinline__ void ri_bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// The whole 16-byte blocks that hold `cols` elements at `row` (at most 15 bytes more on either side, in the same blocks as the row's own): first
// byte, and how far behind it the row begins.
template <typename T>
__device__ __forceinline__ uint32_t ri_span(const T* row, int cols, const void** first, uint32_t* bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(row), begin = at & ~uintptr_t(15);
  *first = reinterpret_cast<const void*>(begin);
  *bytes = uint32_t(((at + size_t(cols) * sizeof(T) + 15) & ~uintptr_t(15)) - begin);
  return uint32_t(at - begin) / uint32_t(sizeof(T));
}

constexpr int RI_RING_BARS = 64;                 // slots of all groups
constexpr size_t RI_RING_BYTES = 222 * 1024;     // dynamic shared memory of the one block of an SM

// A quad: 4 consecutive columns.  Its integers are a word, its fp32 weights 16 bytes; neighbouring threads have neighbouring quads.
template <typename T> struct Ri4 {};
template <> struct Ri4<bf16> {
  uint2 w;
  __device__ __forceinline__ float2 low() const { return make_float2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u)); }
  __device__ __forceinline__ float2 high() const { return make_float2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u)); }
  __device__ __forceinline__ void set(float2 a, float2 b) { w = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y)); }
};
template <> struct Ri4<float> {
  float4 w;
  __device__ __forceinline__ float2 low() const { return make_float2(w.x, w.y); }
  __device__ __forceinline__ float2 high() const { return make_float2(w.z, w.w); }
  __device__ __forceinline__ void set(float2 a, float2 b) { w = make_float4(a.x, a.y, b.x, b.y); }
};
// blockDim.y groups of blockDim.x threads; a group walks rows and has a ring of `stages` slots (x, and the residual behind it) of its own, which one thread
// fills by bulk copies.  A row is read from its slot once for its statistics and once for its integers, so that registers limit neither its width nor the
// rows in flight.  What bounds the kernel beside the bytes is instructions, a third of which are a row's and not an element's: few threads per row (one warp,
// without barriers, where the slots of a block suffice for a dozen), fp32 arithmetic on two values at a time, weights as fp32 in shared memory.
template <typename T, int MODE>
__global__ void __launch_bounds__(RI_MAX_THREADS, 1)
rows_int8_ring_kernel(const RiParams p, int stages, int slot_bytes, float one) {
  extern __shared__ __align__(128) uint8_t ri_smem[];
  __shared__ uint64_t full_bars[RI_RING_BARS];
  __shared__ float sums[3][32];
  __shared__ uint32_t maxima[32];
  __shared__ uint32_t abort_word;
  volatile uint32_t* abort_flag = &abort_word;
  const int group = threadIdx.y, groups = blockDim.y, tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const int quads = p.cols / 4;
  uint64_t* full = full_bars + group * stages;
  const bool two = MODE != RI_ROWS && p.residual;
  const int stage_bytes = slot_bytes * (two ? 2 : 1);
  float* weights = reinterpret_cast<float*>(ri_smem);
  float* biases = weights + 4 * quads;
  uint8_t* ring = ri_smem + size_t(MODE == RI_ROWS ? 0 : MODE == RI_RMS ? 16 : 32) * quads + size_t(group) * stages * stage_bytes;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    if (group == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  ri_begin(p.ahead);
  const long long step = (long long)gridDim.x * groups;
  auto load = [&](long long row, int s) {
    const uint32_t dst = smem_u32(ring + s * stage_bytes);
    const void *from, *from2 = nullptr;
    uint32_t bytes, bytes2 = 0;
    ri_span(static_cast<const T*>(p.x) + row * p.ldx, p.cols, &from, &bytes);
    if (two) ri_span(static_cast<const T*>(p.residual) + row * p.ldr, p.cols, &from2, &bytes2);
    mbar_expect_tx(&full[s], bytes + bytes2);
    ri_bulk_load(dst, from, bytes, &full[s]);
    if (two) ri_bulk_load(dst + slot_bytes, from2, bytes2, &full[s]);
  };
  auto meet = [&]() {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
  };
  auto total = [&](float a, int which) {  // over the group
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (warps == 1) return a;
    float* at = sums[which] + group * warps;
    if (lane == 0) at[warp] = a;
    meet();
    a = lane < warps ? at[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
  };
  // f(quad) for the thread's quads, four at a time
  auto each = [&](auto f) {
    int q = tid;
    for (; q + 3 * threads < quads; q += 4 * threads) {
#pragma unroll
      for (int k = 0; k < 4; ++k) f(q + k * threads);
    }
    for (; q < quads; q += threads) f(q);
  };

  long long row = (long long)blockIdx.x * groups + group;
  long long issued = 0;
  if (tid == 0)
    for (; issued < stages && row + issued * step < p.rows; ++issued) load(row + issued * step, int(issued));
  if (MODE != RI_ROWS) {
    const T* weight = static_cast<const T*>(p.weight);
    const T* bias = static_cast<const T*>(p.bias);
    for (int c = group * threads + tid; c < 4 * quads; c += groups * threads) {
      weights[c] = weight ? ri_float(weight[c]) : 1.f;
      if (MODE == RI_LAYER) biases[c] = bias ? ri_float(bias[c]) : 0.f;
    }
  }
  __syncthreads();
  int s = 0;
  uint32_t parity = 0;
  for (; row < p.rows; row += step) {
    if (!*abort_flag && !mbar_wait(&full[s], parity)) {  // (the row's results are not valid then; the group stays together)
      atomicMax(p.status, STATUS_TIMEOUT_MBAR);
      *abort_flag = 1;
    }
    uint8_t* slot = ring + s * stage_bytes;
    const void* unused;
    uint32_t n;
    T* xs = reinterpret_cast<T*>(slot) + ri_span(static_cast<const T*>(p.x) + row * p.ldx, p.cols, &unused, &n);
    const T* rs = two ? reinterpret_cast<const T*>(slot + slot_bytes) + ri_span(static_cast<const T*>(p.residual) + row * p.ldr, p.cols, &unused, &n) : nullptr;
    T* sum_out = two && p.sum_out ? static_cast<T*>(p.sum_out) + row * p.lds : nullptr;
    struct Quad { float2 a, b; };
    auto get = [&](int q) -> Quad {
      const Ri4<T> x = *reinterpret_cast<const Ri4<T>*>(xs + 4 * q);
      return {x.low(), x.high()};
    };
    auto get_sum = [&](int q) -> Quad {  // h, which takes the place of x
      Ri4<T> x = *reinterpret_cast<const Ri4<T>*>(xs + 4 * q);
      const Ri4<T> r = *reinterpret_cast<const Ri4<T>*>(rs + 4 * q);
      // rounded to the type it is stored in: the norm is taken of what later kernels read
      x.set(__fadd2_rn(x.low(), r.low()), __fadd2_rn(x.high(), r.high()));
      *reinterpret_cast<Ri4<T>*>(xs + 4 * q) = x;
      if (sum_out) *reinterpret_cast<Ri4<T>*>(sum_out + 4 * q) = x;
      return {x.low(), x.high()};
    };
    float mean = 0.f, rstd = 1.f;
    auto value = [&](int q, Quad h) -> Quad {  // what is rounded
      if (MODE == RI_LAYER) {
        h.a = __fmul2_rn(__fadd2_rn(h.a, both(-mean)), both(rstd));
        h.b = __fmul2_rn(__fadd2_rn(h.b, both(-mean)), both(rstd));
      }
      if (MODE != RI_ROWS) {
        const float4 w = *reinterpret_cast<const float4*>(weights + 4 * q);
        h.a = __fmul2_rn(h.a, make_float2(w.x, w.y));
        h.b = __fmul2_rn(h.b, make_float2(w.z, w.w));
      }
      if (MODE == RI_LAYER) {
        const float4 b = *reinterpret_cast<const float4*>(biases + 4 * q);
        h.a = __fadd2_rn(h.a, make_float2(b.x, b.y));
        h.b = __fadd2_rn(h.b, make_float2(b.z, b.w));
      }
      return h;
    };
    float most0 = 0.f, most1 = 0.f;
    float2 squares = both(0.f);
    auto raise = [&](const Quad& v) {
      most0 = fmax3_abs_nan(most0, v.a.x, v.a.y);
      most1 = fmax3_abs_nan(most1, v.b.x, v.b.y);
    };
    auto statistics = [&](int q, const Quad& h) {
      if (MODE == RI_RMS) squares = __ffma2_rn(h.b, h.b, __ffma2_rn(h.a, h.a, squares));
      if (MODE == RI_LAYER) squares = __fadd2_rn(squares, __fadd2_rn(h.a, h.b));
      else raise(value(q, h));
    };
    if (two) each([&](int q) { statistics(q, get_sum(q)); });
    else each([&](int q) { statistics(q, get(q)); });
    float sum = squares.x + squares.y;
    if (MODE == RI_LAYER) {
      // (the deviations are summed up around the mean: a difference of two sums would lose the digits that they share)
      mean = total(sum, 0) / float(p.cols);
      squares = both(0.f);
      each([&](int q) {
        Quad h = get(q);
        h.a = __fadd2_rn(h.a, both(-mean));
        h.b = __fadd2_rn(h.b, both(-mean));
        squares = __ffma2_rn(h.b, h.b, __ffma2_rn(h.a, h.a, squares));
      });
      rstd = rsqrtf(total(squares.x + squares.y, 1) / float(p.cols) + p.eps);
      each([&](int q) { raise(value(q, get(q))); });
    }
    uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(fmax3_abs_nan(most0, most1, 0.f)));
    if (warps > 1 && lane == 0) maxima[group * warps + warp] = most;
    if (MODE == RI_RMS) sum = total(sum, 2);
    else meet();
    if (warps > 1) most = __reduce_max_sync(0xffffffffu, lane < warps ? maxima[group * warps + lane] : 0u);
    const bool finite = most < 0x7F800000u;
    const float amax = fmaxf(__uint_as_float(most), RI_LEAST);
    const float inv = __fdiv_rn(127.f, amax);
    if (tid == 0) {
      p.scales[row] = ri_scale<MODE>(amax, finite, sum, rstd, p);
    }
    int8_t* out = p.q + row * p.ldq;
    each([&](int q) {
      const Quad v = value(q, get(q));
      uint32_t four = ri_integers(v.a, v.b, inv, one);
      if (!finite) four = 0;
      *reinterpret_cast<uint32_t*>(out + 4 * q) = four;
    });
    if (two) fence_proxy_async_smem();  // (h was written to the slot that a bulk copy fills next)
    meet();
    if (tid == 0 && row + stages * step < p.rows && !*abort_flag) {
      load(row + stages * step, s);
      ++issued;
    }
    if (++s == stages) { s = 0; parity ^= 1; }
  }
  if (tid == 0 && *abort_flag) {  // copies that are still on their way arrive before the block's memory goes
    for (int i = 0; i < stages && i < issued; ++i) mbar_wait(&full[(issued - 1 - i) % stages], uint32_t((issued - 1 - i) / stages) & 1);
  }
}

// True if the ring kernel was launched (or its launch failed: *e): rows that begin and end on a quad's boundary, and room for two.
template <typename T, int MODE>
static bool ri_ring_launch(const RiParams& p, int sms, cudaStream_t stream, cudaError_t* e) {
  const size_t slot = (size_t(p.cols) * sizeof(T) + 15) / 16 * 16 + 16;  // (a row may begin in the middle of 16 bytes)
  const size_t stage = slot * (p.residual ? 2 : 1);
  const size_t params = size_t(MODE == RI_ROWS ? 0 : MODE == RI_RMS ? 1 : 2) * size_t((p.cols + 3) / 4) * 16;
  auto whole = [](const void* base, long long ld) { return reinterpret_cast<uintptr_t>(base) % (4 * sizeof(T)) == 0 && ld % 4 == 0; };
  if (params + 2 * stage > RI_RING_BYTES || p.cols % 4 || !whole(p.x, p.ldx) || !whole(p.residual, p.ldr) || !whole(p.sum_out, p.lds) ||
      (reinterpret_cast<uintptr_t>(p.q) & 3) || p.ldq % 4)
    return false;
  size_t slots = (RI_RING_BYTES - params) / stage;
  if (slots > RI_RING_BARS) slots = RI_RING_BARS;
  int groups = int(slots / 2);
  if (groups < 1) groups = 1;
  if (groups > (p.rows + sms - 1) / sms) groups = (p.rows + sms - 1) / sms;
  int warps = 1;
  while (warps < 8 && warps * groups < 16) warps *= 2;
  if (groups * warps > 32) groups = 32 / warps;
  if (warps > 1 && groups > 15) groups = 15;  // (named barriers)
  int stages = int(slots / groups);
  if (stages > 4) stages = 4;
  auto go = [&](auto kernel) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(RI_RING_BYTES));
    return err != cudaSuccess ? err
                              : launch_dependent(kernel, dim3(sms), dim3(32 * warps, groups), params + groups * stages * stage, stream, true, p, stages, int(slot), 1.f);
  };
  *e = go(rows_int8_ring_kernel<T, MODE>);
  return true;
}

// Which rows go by the ring, and which by 32 columns a thread instead of 16 (bf16 rows of at most 32768 columns: the fp32 ones do not fit the registers).
// Fewer threads a row cost latency, which few rows do not hide, and save the row's own share of the instructions.  us, 16 columns / 32 columns / ring:
//   rows       8192 x 5120 - / 22.1 / 24.9     1024 x 8192 - / 6.1 / 9.0      8192 x 11008 - / 56 / 46.8    2048 x 11008 - / 16.2 / 15.0   1024 x 11008 - / 9.3 / 10.5
//              592 x 20000 - / 10.5 / 9.6      2048 x 20000 - / 31.0 / 23.2
//   RMSNorm    8192 x 4096 24.8 / 25.2 / 26.1  8192 x 5120 - / 34.6 / 31.4    8192 x 8192 - / 50.1 / 46.9   2048 x 8192 - / 14.8 / 16.8    2048 x 16384 - / 26.2 / 28.7
//   + residual 8192 x 4096 37.4 / 37.8 / -     8192 x 8192 81 / 72 / -        8192 x 11008 - / 109 / 112    300 x 5120 4.0 / 4.5 / -       300 x 8192 6.0 / 5.4 / -
//              8192 x 16392 - / 205 / 163      8192 x 20000 - / 222 / 312     8 x 16392 5.0 / 3.6 / -
//   LayerNorm  8192 x 2560 22.5 / 22.9 / -     8192 x 3584 31.6 / 29.6 / -    8192 x 4096 37.2 / 30.3 / -   8192 x 8192 78 / 60 / -        8192 x 11008 - / 94 / 107
// Norms of many rows, a block a row / persistent blocks with 16 columns a thread / with 32 (rows_int8_walk_kernel; the better of both in the last two lines):
//   RMSNorm    16384 x 512 7.2 / 7.7 / 8.5     16384 x 1024 13.7 / 12.3 / 10.5   2400 x 1024 3.8 / 4.0 / 4.0    8192 x 2048 13.6 / 11.2 / 11.8   8192 x 4096 25.0 / 20.6 / 21.0
//              8192 x 5120 31.4 / 25.3 / 25.8  8192 x 8192 46.7 / 38.2 / 38.6    8192 x 11008 60 / 75 / 58      8192 x 16384 87 / 90 / 74
//   LayerNorm  16384 x 1024 20.0 / 15.7 / 12.1 8192 x 2560 22.5 / 19.8 / 22.3    8192 x 4096 30.6 / 29.8 / 27.8 8192 x 8192 61 / 60 / 47         8192 x 16384 122 / 122 / 98
//   fewer rows 1200 x 2048 3.8 / 3.4 / -       1200 x 5120 7.4 / - / 5.5         600 x 11008 8.4 / - / 6.5
//   + residual 600 x 2048 4.2 / 3.5, 1200 x 8192 14.1 / 13.0, 8192 x 4096 37.5 / 37.9, 8192 x 8192 72.6 / 77.5; LayerNorm 8192 x 1024 14.3 / 11.7, 8192 x 5120 55 / 49,
//              16384 x 4096 76.7 / 80.1, 2400 x 16384 60 / 48
// Rows of any alignment, bf16, 16 columns a thread / 32: rows 8192 x 5255 40.1 / 32.8, 300 x 5255 3.1 / 3.9, 2000 x 11007 29.9 / 19.9, 8 x 16610 5.2 / 2.5; RMSNorm 8192 x 4490
// 41.1 / 46.2, 2000 x 11007 38.7 / 28.9, with a residual 59.2 / 55.2, 300 rows of it 12.6 / 14.0, 8192 x 16610 640 / 391; LayerNorm 8192 x 5255 92 / 70, 2000 x 16610 241 / 72.
// Other rows (fp32, or of any alignment), 16 columns / ring: RMSNorm with a residual 4096 x 8192 42.7 / 45.2; 4096 x 11008 30.7 / 25.9, RMSNorm 58 / 35.
template <typename T, int MODE, bool VEC>
static bool ri_ring(const RiParams& p, int sms) {
  if (!VEC || sizeof(T) != 2 || p.cols > 32768) return p.rows >= 2 * sms && p.cols > (p.residual || MODE == RI_LAYER ? 8192 : 4096);
  if (MODE == RI_ROWS) return p.cols > 8192 && p.rows >= (p.cols > 16384 ? 4 : 12) * sms;
  return MODE == RI_RMS && !p.residual && p.cols > 16384 && p.rows >= 16 * sms;
}
template <typename T, int MODE, bool VEC>
static bool ri_four(const RiParams& p, int sms) {
  if (sizeof(T) != 2 || p.cols > 32768) return false;
  if (!VEC) return p.cols > 16384 || (p.cols > 6144 ? p.rows >= (p.residual ? 8 : 2) * sms : p.cols > 4096 && MODE != RI_RMS && p.rows >= 4 * sms);
  return p.cols > 16384 || (p.rows >= (p.cols > 6144 ? 2 : 4) * sms && p.cols > 4096);
}

template <int MODE>
static bool ri_walk(const RiParams& p, int sms) {
  if (p.cols < 768 || p.cols > 16384 || p.rows < (p.cols > 1024 ? 4 : 32) * sms) return false;
  return MODE == RI_LAYER || !p.residual || p.cols <= 1024 || p.rows <= 32 * sms;
}

template <typename T, int MODE, bool VEC>
static cudaError_t ri_launch(const RiParams& p, int sms, cudaStream_t stream) {
  cudaError_t e;
  if (ri_ring<T, MODE, VEC>(p, sms) && ri_ring_launch<T, MODE>(p, sms, stream, &e)) return e;
  const int groups = (p.cols + 7) / 8;
  if constexpr (VEC && sizeof(T) == 2 && MODE != RI_ROWS) {
    if (ri_walk<MODE>(p, sms)) {
      auto walk = [&](auto kernel, int v, int most) {
        const int threads = ((groups + v - 1) / v + 31) / 32 * 32, blocks = ri_walk_threads(v, most, p.residual) / threads * sms;
        return launch_dependent(kernel, dim3(blocks < p.rows ? blocks : p.rows), dim3(threads), 0, stream, true, p, 1.f);
      };
#define WALK(V, N) (p.residual ? walk(rows_int8_walk_kernel<MODE, V, N, true>, V, N) : walk(rows_int8_walk_kernel<MODE, V, N, false>, V, N))
      if (p.cols <= 1024) return WALK(4, 32);
      if (p.cols <= 2048) return WALK(2, 128);
      if constexpr (MODE == RI_LAYER) {
        if (p.cols > 3584 && p.cols <= 4096) return WALK(4, 128);
      }
      if (p.cols <= 4096) return WALK(2, 256);
      return p.cols <= 8192 ? WALK(4, 256) : WALK(4, 512);
#undef WALK
    }
  }
  const int v = groups <= 32 ? 1 : ri_four<T, MODE, VEC>(p, sms) ? 4 : 2;
  int threads = ((groups + v - 1) / v + 31) / 32 * 32;
  const bool wide = threads > RI_MAX_THREADS;
  if (wide) threads = RI_MAX_THREADS;
  const int rows_per_block = threads >= 256 || v == 4 ? 1 : 256 / threads;
  const dim3 block(threads, rows_per_block), grid((unsigned(p.rows) + rows_per_block - 1) / rows_per_block);
  auto go = [&](auto kernel) { return launch_dependent(kernel, grid, block, 0, stream, true, p, 1.f); };
  if constexpr (sizeof(T) == 2) {
    if (v == 4)
      return threads <= 256   ? go(rows_int8_kernel<T, MODE, 4, VEC, false, 256>)
             : threads <= 512 ? go(rows_int8_kernel<T, MODE, 4, VEC, false, 512>)
                              : go(rows_int8_kernel<T, MODE, 4, VEC, false, 1024>);
  }
  if (wide) return go(rows_int8_kernel<T, MODE, 2, VEC, true, 1024>);
  if (v == 1) return go(rows_int8_kernel<T, MODE, 1, VEC, false, 256>);
  return threads <= 256 ? go(rows_int8_kernel<T, MODE, 2, VEC, false, 256>) : go(rows_int8_kernel<T, MODE, 2, VEC, false, 1024>);
}

template <typename T>
static cudaError_t ri_dispatch(const RiParams& p, int sms, int mode, cudaStream_t stream) {
  auto rows_aligned = [](const void* base, long long ld) { return !(reinterpret_cast<uintptr_t>(base) & 15) && (ld * sizeof(T)) % 16 == 0; };
  const bool vec = p.cols % 8 == 0 && rows_aligned(p.x, p.ldx) && rows_aligned(p.residual, p.ldr) && rows_aligned(p.sum_out, p.lds) &&
                   rows_aligned(p.weight, 0) && rows_aligned(p.bias, 0) && !(reinterpret_cast<uintptr_t>(p.q) & 7) && p.ldq % 8 == 0;
#define RI_GO(MODE) (vec ? ri_launch<T, MODE, true>(p, sms, stream) : ri_launch<T, MODE, false>(p, sms, stream))
  return mode == RI_ROWS ? RI_GO(RI_ROWS) : mode == RI_RMS ? RI_GO(RI_RMS) : RI_GO(RI_LAYER);
#undef RI_GO
}

template <typename T, int MODE>
static cudaError_t ri_preload() {
  cudaFuncAttributes attr;
  cudaError_t e = cudaSuccess;
#define LOAD(...) if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, __VA_ARGS__)
  LOAD(rows_int8_ring_kernel<T, MODE>);
  LOAD(rows_int8_kernel<T, MODE, 2, true, true, 1024>);
  LOAD(rows_int8_kernel<T, MODE, 2, false, true, 1024>);
  LOAD(rows_int8_kernel<T, MODE, 1, true, false, 256>);
  LOAD(rows_int8_kernel<T, MODE, 1, false, false, 256>);
  LOAD(rows_int8_kernel<T, MODE, 2, true, false, 256>);
  LOAD(rows_int8_kernel<T, MODE, 2, false, false, 256>);
  LOAD(rows_int8_kernel<T, MODE, 2, true, false, 1024>);
  LOAD(rows_int8_kernel<T, MODE, 2, false, false, 1024>);
  if constexpr (sizeof(T) == 2) {
    LOAD(rows_int8_kernel<T, MODE, 4, true, false, 256>);
    LOAD(rows_int8_kernel<T, MODE, 4, true, false, 512>);
    LOAD(rows_int8_kernel<T, MODE, 4, true, false, 1024>);
    LOAD(rows_int8_kernel<T, MODE, 4, false, false, 256>);
    LOAD(rows_int8_kernel<T, MODE, 4, false, false, 512>);
    LOAD(rows_int8_kernel<T, MODE, 4, false, false, 1024>);
    if constexpr (MODE != RI_ROWS) {
#define LOAD_WALK(V, N) LOAD(rows_int8_walk_kernel<MODE, V, N, false>); LOAD(rows_int8_walk_kernel<MODE, V, N, true>)
      LOAD_WALK(4, 32);
      LOAD_WALK(2, 128);
      LOAD_WALK(2, 256);
      LOAD_WALK(4, 256);
      LOAD_WALK(4, 512);
      if constexpr (MODE == RI_LAYER) {
        LOAD_WALK(4, 128);
      }
#undef LOAD_WALK
    }
  }
#undef LOAD
  return e;
}
cudaError_t rows_int8_preload() {
  const cudaError_t all[6] = {ri_preload<bf16, RI_ROWS>(), ri_preload<bf16, RI_RMS>(), ri_preload<bf16, RI_LAYER>(),
                              ri_preload<float, RI_ROWS>(), ri_preload<float, RI_RMS>(), ri_preload<float, RI_LAYER>()};
  for (const cudaError_t e : all)
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace tpb

extern "C" int tpb_rows_int8(const void* x, const void* residual, const void* weight, const void* bias, void* sum_out, int8_t* q, float* scales, int rows,
                             int cols, long long ldx, long long ldr, long long lds, long long ldq, float eps, int mode, int dtype, int ahead, void* status, void* stream) {
  if (!x || !q || !scales || !status || rows <= 0 || cols <= 0 || mode < 0 || mode > 2 || dtype < 0 || dtype > 1) return TPB_ERR_ARG;
  if (cols > 1 << 30) return TPB_ERR_SIZE;
  if (mode == tpb::RI_ROWS && (residual || weight || bias || sum_out)) return TPB_ERR_ARG;
  if ((bias && mode != tpb::RI_LAYER) || (sum_out && !residual)) return TPB_ERR_ARG;
  if (ldx < cols || ldq < cols || (residual && ldr < cols) || (sum_out && lds < cols)) return TPB_ERR_ARG;
  tpb::RiParams p = {x, residual, weight, bias, sum_out, q, scales, ldx, residual ? ldr : 0, sum_out ? lds : 0, ldq, rows, cols, eps, ahead, static_cast<uint32_t*>(status)};
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return TPB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == 0 ? tpb::ri_dispatch<tpb::bf16>(p, sms, mode, s) : tpb::ri_dispatch<float>(p, sms, mode, s);
  return e == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

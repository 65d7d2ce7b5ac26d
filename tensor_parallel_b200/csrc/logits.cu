// Logits in front of the pick of a token: penalties for tokens that a sequence has had, biases, and the tokens that its grammar allows.
//
//   seen:  x = x > 0 ? x / repetition : x * repetition;   x -= frequency * count + presence * (count > 0);   x += bias;   not allowed: -inf
//
// Bound by memory: each logit is read once and written once.  A block has a slice of one row's vocabulary; it counts the tokens of that slice in shared memory
// (a 32-bit word per entry: the top bit for a token that was seen at all, the rest for how often it was said) by walking the row's whole history, which
// the other slices of the row find in L2, and then passes over its logits.  Integer atomics: the counts do not depend on their order.  Long slices walk
// the history less often, short ones fill the GPU when there are few rows.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

typedef __nv_bfloat16 bf16;

constexpr int LG_THREADS = 256;

struct LogitsParams {
  const void* logits;
  void* out;
  const long long* tokens;
  const int *lengths, *prompts;
  const float *repetition, *frequency, *presence;
  const void* bias;
  const uint32_t* allowed;
  uint32_t* status;
  long long logits_ld, out_ld, tokens_ld, bias_ld, allowed_ld;
  int vocab, width, slice, bias_fp32;
  float repetition_all, frequency_all, presence_all;
};

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
};
template <> struct Vec<bf16> {
  static constexpr int N = 8;
};
__device__ __forceinline__ float lg_load(const float* p) { return *p; }
__device__ __forceinline__ float lg_load(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void lg_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void lg_store(bf16* p, float v) { *p = __float2bfloat16(v); }

// WIDE: logits and results of a row lie alike to a 16-byte boundary, and go in 16-byte vectors; else one by one.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(LG_THREADS)
adjust_logits_kernel(const LogitsParams p) {
  extern __shared__ uint32_t counts[];
  constexpr int N = WIDE ? Vec<T>::N : 1;
  const long long row = blockIdx.x;
  const int begin = blockIdx.y * p.slice, end = min(p.vocab, begin + p.slice);
  const T* x = static_cast<const T*>(p.logits) + row * p.logits_ld;
  T* y = static_cast<T*>(p.out) + row * p.out_ld;
  const bool history = p.tokens != nullptr;
  if (history) {
    for (int i = threadIdx.x; i < end - begin; i += LG_THREADS) counts[i] = 0;
    int length = p.lengths ? __ldg(p.lengths + row) : p.width;
    const int prompt = p.prompts ? __ldg(p.prompts + row) : 0;
    if (length < 0 || length > p.width || prompt < 0) {
      if (threadIdx.x == 0) atomicMax(p.status, uint32_t(STATUS_BAD_ARG));
      length = min(max(length, 0), p.width);
    }
    __syncthreads();
    const long long* said = p.tokens + row * p.tokens_ld;
    for (int i = threadIdx.x; i < length; i += LG_THREADS) {
      const long long token = __ldg(said + i);
      if (token >= begin && token < end) {
        if (i < prompt)
          atomicOr(&counts[token - begin], 0x80000000u);
        else
          atomicAdd(&counts[token - begin], 1u);
      }
    }
    __syncthreads();
  }
  const float repetition = p.repetition ? __ldg(p.repetition + row) : p.repetition_all;
  const float frequency = p.frequency ? __ldg(p.frequency + row) : p.frequency_all;
  const float presence = p.presence ? __ldg(p.presence + row) : p.presence_all;
  const uint32_t* allowed = p.allowed ? p.allowed + row * p.allowed_ld : nullptr;

  auto adjust = [&](float v, int i) {
    if (history) {
      const uint32_t seen = counts[i - begin];
      if (seen) {
        v = v > 0.f ? v / repetition : v * repetition;
        const uint32_t count = seen & 0x7fffffffu;
        if (count) v -= frequency * float(count) + presence;
      }
    }
    if (p.bias) v += p.bias_fp32 ? __ldg(static_cast<const float*>(p.bias) + row * p.bias_ld + i) : __bfloat162float(static_cast<const bf16*>(p.bias)[row * p.bias_ld + i]);
    if (allowed && !(__ldg(allowed + (i >> 5)) >> (i & 31) & 1u)) v = -INFINITY;
    return v;
  };
  if (!WIDE) {
    for (int i = begin + threadIdx.x; i < end; i += LG_THREADS) lg_store(y + i, adjust(lg_load(x + i), i));
    return;
  }
  // vectors of the row's own 16-byte grid: the first may begin in front of the slice, the last end behind it
  const int skew = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % N);
  for (int at = (begin + skew) / N * N - skew + int(threadIdx.x) * N; at < end; at += LG_THREADS * N) {
    if (at >= begin && at + N <= end) {
      uint4 u = *reinterpret_cast<const uint4*>(x + at);
      T* v = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) lg_store(v + i, adjust(lg_load(v + i), at + i));
      *reinterpret_cast<uint4*>(y + at) = u;
    } else {
      for (int i = max(at, begin); i < min(at + N, end); ++i) lg_store(y + i, adjust(lg_load(x + i), i));
    }
  }
}

template <typename T>
static int lg_launch(LogitsParams& p, int rows, cudaStream_t stream) {
  auto grid_place = [](const void* t) { return reinterpret_cast<uintptr_t>(t) / sizeof(T) % Vec<T>::N; };
  const bool wide = grid_place(p.logits) == grid_place(p.out) && (rows == 1 || p.logits_ld % Vec<T>::N == p.out_ld % Vec<T>::N) && p.logits_ld >= 0;
  // slices: short enough for a few blocks per SM, long enough that walking the history (one read per 256 tokens and thread) stays below the logits' own
  p.slice = 8192;
  while (p.slice > 1024 && (long long)rows * ((p.vocab + p.slice - 1) / p.slice) < 148 * 4) p.slice /= 2;
  const dim3 grid(rows, (p.vocab + p.slice - 1) / p.slice);
  if (grid.y > 65535) return TPB_ERR_SIZE;
  const size_t smem = p.tokens ? p.slice * 4 : 0;
  if (wide)
    adjust_logits_kernel<T, true><<<grid, LG_THREADS, smem, stream>>>(p);
  else
    adjust_logits_kernel<T, false><<<grid, LG_THREADS, smem, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb_adjust_logits(const tpb_adjust_logits_t* a, void* stream_) {
  if (!a || !a->logits || !a->out || !a->status || a->rows <= 0 || a->vocab <= 0 || a->width < 0 || a->dtype < 0 || a->dtype > 1) return TPB_ERR_ARG;
  LogitsParams p = {a->logits, a->out, a->tokens, a->lengths, a->prompts, a->repetition, a->frequency, a->presence, a->bias, reinterpret_cast<const uint32_t*>(a->allowed),
                    static_cast<uint32_t*>(a->status), a->logits_ld, a->out_ld, a->tokens_ld, a->bias_ld, a->allowed_ld, a->vocab, a->width, 0, a->bias_dtype,
                    a->repetition_all, a->frequency_all, a->presence_all};
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  return a->dtype ? lg_launch<float>(p, a->rows, s) : lg_launch<bf16>(p, a->rows, s);
}

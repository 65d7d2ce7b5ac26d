// Logits in front of the pick of a token: penalties for tokens that a sequence has had, biases, and the tokens that its grammar allows.
//
//   seen:  x = x > 0 ? x / repetition : x * repetition;   x -= frequency * count + presence * (count > 0);   x += bias;   not allowed: -inf
//
// Bound by memory: each logit is read once and written once.  A block has a part of one row's vocabulary.  It counts the tokens of that part in shared memory (a
// 32-bit word per entry: the top bit for a token that was seen at all, the rest for how often it was said) by walking the row's whole history, which the other
// blocks of the row find in L2, and then streams its logits, four 16-byte vectors per thread on their way at a time, the first of them during the count.  Integer
// atomics: the counts do not depend on their order.  Parts are as long as leaves three blocks to an SM: the walk, a chain of loads that nothing hides, is then
// paid once (128 x 65024 fp32, 1000 tokens: parts of 1024 to 8192 entries in registers 28 to 33 us, 12 us without the walk).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

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
  int vocab, width, bias_fp32, part;
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

// Elements at, at + 1, ... of a row of numbers, `n` of them in [0, limit); one vector where the address allows.
template <int N>
__device__ __forceinline__ void lg_numbers(const float* row, int at, int limit, float (&v)[N]) {
  if (N > 1 && at >= 0 && at + N <= limit && !(reinterpret_cast<uintptr_t>(row + at) & 15)) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(row + at + i));
      v[i] = f.x;
      if (N > 1) v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = at + i >= 0 && at + i < limit ? __ldg(row + at + i) : 0.f;
}

constexpr int LG_DEPTH = 4;         // vectors of a thread on their way
constexpr int LG_MOST_ENTRIES = 16384;  // of a part: 64 KB of counts, three blocks per SM

// WIDE: logits and results of a row lie alike to a 16-byte boundary, and go in 16-byte vectors of the row's own grid, of which the first may begin in front of the
// row and the last end behind it; else one by one.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(LG_THREADS)
adjust_logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t counts[];
  constexpr int N = WIDE ? Vec<T>::N : 1, ROUND = LG_THREADS * N;
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.logits_ld;
  T* y = static_cast<T*>(p.out) + row * p.out_ld;
  const int skew = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % N);
  const int begin = blockIdx.y * p.part - skew, end = int(min((long long)p.vocab, (long long)begin + p.part));  // (the first part begins up to N - 1 in front of the row)
  const int mine = begin + int(threadIdx.x) * N;
  uint4 raw[LG_DEPTH];
  auto fetch = [&](uint4& u, int at) {
    T* v = reinterpret_cast<T*>(&u);
    if (WIDE && at >= 0 && at + N <= p.vocab) {
      u = __ldcs(reinterpret_cast<const uint4*>(x + at));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i >= 0 && at + i < p.vocab) v[i] = x[at + i];
    }
  };
#pragma unroll
  for (int j = 0; j < LG_DEPTH; ++j)
    if (mine + j * ROUND < end) fetch(raw[j], mine + j * ROUND);
  const bool history = p.tokens != nullptr;
  if (history) {
    for (int i = threadIdx.x * 4; i < p.part; i += LG_THREADS * 4) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
    int length = p.lengths ? __ldg(p.lengths + row) : p.width;
    const int prompt = p.prompts ? __ldg(p.prompts + row) : 0;
    if (length < 0 || length > p.width || prompt < 0) {
      if (threadIdx.x == 0) atomicMax(p.status, uint32_t(STATUS_BAD_ARG));
      length = min(max(length, 0), p.width);
    }
    __syncthreads();
    const long long* said = p.tokens + row * p.tokens_ld;
#pragma unroll 4
    for (int i = threadIdx.x; i < p.width; i += LG_THREADS) {
      const long long token = __ldg(said + i);
      if (i < length && token >= max(begin, 0) && token < end) {
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
  const int words = (p.vocab + 31) / 32;

  auto adjust = [&](uint4 taken, int at) {
    T* packed = reinterpret_cast<T*>(&taken);
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lg_load(packed + i);
    if (history) {
      uint32_t seen[N], any = 0;
#pragma unroll
      for (int i = 0; i < N; i += N < 4 ? 1 : 4) {
        const uint32_t* from = counts + (at - begin) + i;
        if (N < 4) {
          seen[i] = *from;
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(from);
          seen[i] = u.x, seen[i + (N > 1)] = u.y, seen[i + 2 * (N > 2)] = u.z, seen[i + 3 * (N > 3)] = u.w;
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) any |= seen[i];
      if (any) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (seen[i]) {
            v[i] = v[i] > 0.f ? v[i] / repetition : v[i] * repetition;
            const uint32_t count = seen[i] & 0x7fffffffu;
            if (count) v[i] -= frequency * float(count) + presence;
          }
      }
    }
    if (p.bias) {
      if (p.bias_fp32) {
        float b[N];
        lg_numbers<N>(static_cast<const float*>(p.bias) + row * p.bias_ld, at, p.vocab, b);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += b[i];
      } else {
        const bf16* b = static_cast<const bf16*>(p.bias) + row * p.bias_ld;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i >= 0 && at + i < p.vocab) v[i] += __bfloat162float(b[at + i]);
      }
    }
    if (allowed) {
      // bits of tokens at, at + 1, ...: from two words (the vector may cross their border, and begin in front of the first)
      const int word = at >> 5;
      const uint32_t low = word >= 0 ? __ldg(allowed + word) : 0u, high = word + 1 < words ? __ldg(allowed + word + 1) : 0u;
      const uint32_t bits = __funnelshift_r(low, high, at & 31);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!(bits >> i & 1u)) v[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) lg_store(packed + i, v[i]);
    if (WIDE && at >= 0 && at + N <= p.vocab) {
      __stcs(reinterpret_cast<uint4*>(y + at), taken);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i >= 0 && at + i < p.vocab) y[at + i] = packed[i];
    }
  };
  for (int at = mine; at < end; at += LG_DEPTH * ROUND) {
#pragma unroll
    for (int j = 0; j < LG_DEPTH; ++j) {
      const int now = at + j * ROUND, next = now + LG_DEPTH * ROUND;
      if (now >= end) break;
      const uint4 taken = raw[j];
      if (next < end) fetch(raw[j], next);
      adjust(taken, now);
    }
  }
}

template <typename T, bool WIDE>
static int lg_go(LogitsParams p, int rows, cudaStream_t stream) {
  constexpr int N = WIDE ? Vec<T>::N : 1, ROUND = LG_THREADS * (N < 4 ? 4 : N);
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(adjust_logits_kernel<T, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_MOST_ENTRIES * 4) != cudaSuccess) return TPB_ERR_CUDA;
    ready[dev].store(true, std::memory_order_release);
  }
  // entries of a part: a row's over as many blocks as make three per SM of all rows, whole rounds of the block
  const long long entries = (long long)p.vocab + N - 1, blocks = max(1LL, 148LL * 3 / rows);
  const long long part = min((long long)LG_MOST_ENTRIES, ((entries + blocks - 1) / blocks + ROUND - 1) / ROUND * ROUND);
  const long long parts = (entries + part - 1) / part;
  if (parts > 65535) return TPB_ERR_SIZE;
  p.part = int(part);
  adjust_logits_kernel<T, WIDE><<<dim3(rows, unsigned(parts)), LG_THREADS, p.tokens ? size_t(part) * 4 : 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

template <typename T>
static int lg_launch(const LogitsParams& p, int rows, cudaStream_t stream) {
  constexpr int N = Vec<T>::N;
  auto place = [](const void* t) { return reinterpret_cast<uintptr_t>(t) / sizeof(T) % N; };
  const bool wide = place(p.logits) == place(p.out) && (rows == 1 || (p.logits_ld - p.out_ld) % N == 0);
  return wide ? lg_go<T, true>(p, rows, stream) : lg_go<T, false>(p, rows, stream);
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb_adjust_logits(const tpb_adjust_logits_t* a, void* stream_) {
  if (!a || !a->logits || !a->out || !a->status || a->rows <= 0 || a->vocab <= 0 || a->width < 0 || a->dtype < 0 || a->dtype > 1) return TPB_ERR_ARG;
  LogitsParams p = {a->logits, a->out, a->tokens, a->lengths, a->prompts, a->repetition, a->frequency, a->presence, a->bias, reinterpret_cast<const uint32_t*>(a->allowed),
                    static_cast<uint32_t*>(a->status), a->logits_ld, a->out_ld, a->tokens_ld, a->bias_ld, a->allowed_ld, a->vocab, a->width, a->bias_dtype, 0,
                    a->repetition_all, a->frequency_all, a->presence_all};
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  return a->dtype ? lg_launch<float>(p, a->rows, s) : lg_launch<bf16>(p, a->rows, s);
}

// Logits in front of the pick of a token: penalties for tokens that a sequence has had, biases, and the tokens that its grammar allows.
//
//   seen:  x = x > 0 ? x / repetition : x * repetition;   x -= frequency * count + presence * (count > 0);   x += bias;   not allowed: -inf
//
// Bound by memory: each logit is read once and written once.  Two kernels.  The first streams the logits with bias and mask, four 16-byte vectors per thread
// on their way at a time with their biases.  The second deals with the few entries that a row has had; it is launched ahead and does all but its stores while the first one runs:
// a block has a part of one row's vocabulary, counts the row's tokens of that part in shared memory (a 32-bit word per entry: the top bit for a token
// that was seen at all, the rest for how often it was said), and whoever takes an entry's count computes its logit anew and stores it when the first kernel
// has ended.  Integer atomics: the counts do not depend on their order.  In one kernel the walk over the history, a chain of loads, stood in front of every
// block's stream, or its penalties in it (128 x 65024 fp32, 1000 tokens: 28 to 40 us; the stream alone takes 12).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "launch.cuh"
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
  int vocab, width, bias_fp32;
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

__device__ __forceinline__ void lg_wait_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void lg_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

constexpr int LG_DEPTH = 4;           // vectors of 16 bytes of fp32 of a thread on their way, half as many of bf16
constexpr int LG_ENTRIES = 24576;     // of a part of the vocabulary at most: 96 KB of counts, two blocks per SM
constexpr int LG_SEEN_THREADS = 512;  // of a block behind the first kernel: 4096 tokens at once
constexpr int LG_ALONE = 4096;        // entries of a part where one kernel does both
constexpr int LG_HELD = 8;            // tokens of a thread at a time; the first of them wait for the first kernel with their results

// WIDE: logits and results of a row lie alike to a 16-byte boundary, and go in 16-byte vectors of the row's own grid, of which the first may begin in front of the
// row and the last end behind it; else one by one.
// Bias and mask of the entries [begin, end) of a row; begin may lie up to N - 1 in front of it, on its grid.
template <typename T, bool WIDE>
__device__ __forceinline__ void stream_part(const LogitsParams& p, long long row, int begin, int end) {
  constexpr int N = WIDE ? Vec<T>::N : 1, ROUND = LG_THREADS * N, DEPTH = LG_DEPTH * 4 / (N < 4 ? 4 : N);
  const T* x = static_cast<const T*>(p.logits) + row * p.logits_ld;
  T* y = static_cast<T*>(p.out) + row * p.out_ld;
  const int skew = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % N);
  const uint32_t* allowed = p.allowed ? p.allowed + row * p.allowed_ld : nullptr;
  const float* wide_bias = p.bias && p.bias_fp32 ? static_cast<const float*>(p.bias) + row * p.bias_ld : nullptr;
  const bf16* narrow_bias = p.bias && !p.bias_fp32 ? static_cast<const bf16*>(p.bias) + row * p.bias_ld : nullptr;
  const bool bias_vectors = N % 4 == 0 && !(reinterpret_cast<uintptr_t>(wide_bias - skew) & 15);
  const int words = (p.vocab + 31) / 32;
  for (int base = begin + int(threadIdx.x) * N; base < end; base += DEPTH * ROUND) {
    uint4 raw[DEPTH];
    float bias[DEPTH][N];
    uint32_t low[DEPTH], high[DEPTH];
    // all loads of a round in front of the first use
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      const int at = base + j * ROUND;
      if (at >= end) break;
      T* v = reinterpret_cast<T*>(&raw[j]);
      const bool inner = at >= 0 && at + N <= p.vocab;
      if (WIDE && inner) {
        raw[j] = *reinterpret_cast<const uint4*>(x + at);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i >= 0 && at + i < p.vocab) v[i] = x[at + i];
      }
      if (wide_bias) {
        if (bias_vectors && inner) {
#pragma unroll
          for (int i = 0; i + 3 < N; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(wide_bias + at + i));
            bias[j][i] = f.x, bias[j][i + 1] = f.y, bias[j][i + 2] = f.z, bias[j][i + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (at + i >= 0 && at + i < p.vocab) bias[j][i] = __ldg(wide_bias + at + i);
        }
      } else if (narrow_bias) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i >= 0 && at + i < p.vocab) bias[j][i] = __bfloat162float(narrow_bias[at + i]);
      }
      if (allowed) {
        // bits of tokens at, at + 1, ...: from two words (the vector may cross their border, and begin in front of the first)
        const int word = at >> 5;
        low[j] = word >= 0 ? __ldg(allowed + word) : 0u;
        high[j] = word + 1 < words ? __ldg(allowed + word + 1) : 0u;
      }
    }
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      const int at = base + j * ROUND;
      if (at >= end) break;
      T* v = reinterpret_cast<T*>(&raw[j]);
      const uint32_t bits = allowed ? __funnelshift_r(low[j], high[j], at & 31) : ~0u;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float f = p.bias ? lg_load(v + i) + bias[j][i] : lg_load(v + i);
        lg_store(v + i, bits >> i & 1u ? f : -INFINITY);
      }
      if (WIDE && at >= 0 && at + N <= p.vocab) {
        *reinterpret_cast<uint4*>(y + at) = raw[j];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i >= 0 && at + i < p.vocab) y[at + i] = v[i];
      }
    }
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(LG_THREADS, 4)
adjust_stream_kernel(const LogitsParams p, int part) {
  constexpr int N = WIDE ? Vec<T>::N : 1;
  lg_wait_prior();  // (launched ahead of the previous kernel's end: nothing is read or written before that)
  lg_launch_next();
  const long long row = blockIdx.x;
  const int skew = int((reinterpret_cast<uintptr_t>(static_cast<const T*>(p.logits) + row * p.logits_ld) / sizeof(T)) % N);
  const int begin = blockIdx.y * part - skew;
  stream_part<T, WIDE>(p, row, begin, int(min((long long)p.vocab, (long long)begin + part)));
}

// FORM 0: behind the first kernel.  1 and 2: alone, with the stream of its own part in front (in vectors, one by one).
template <typename T, int FORM>
__global__ void __launch_bounds__(FORM ? LG_THREADS : LG_SEEN_THREADS, FORM ? 4 : 2)
adjust_seen_kernel(const LogitsParams p, int part) {
  constexpr int THREADS = FORM ? LG_THREADS : LG_SEEN_THREADS;
  extern __shared__ __align__(16) uint32_t counts[];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.logits_ld;
  T* y = static_cast<T*>(p.out) + row * p.out_ld;
  // (alone, parts lie on the row's grid of vectors)
  const long long begin = (long long)blockIdx.y * part - (FORM == 1 ? int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % Vec<T>::N) : 0);
  const long long end = min((long long)p.vocab, begin + part);
  for (int i = threadIdx.x * 4; i < part; i += THREADS * 4) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
  if (FORM) {
    lg_wait_prior();
    lg_launch_next();
  }
  int length = p.lengths ? __ldg(p.lengths + row) : p.width;
  const int prompt = p.prompts ? __ldg(p.prompts + row) : 0;
  if (length < 0 || length > p.width || prompt < 0) {
    if (threadIdx.x == 0 && blockIdx.y == 0) atomicMax(p.status, uint32_t(STATUS_BAD_ARG));
    length = min(max(length, 0), p.width);
  }
  const float repetition = p.repetition ? __ldg(p.repetition + row) : p.repetition_all;
  const float frequency = p.frequency ? __ldg(p.frequency + row) : p.frequency_all;
  const float presence = p.presence ? __ldg(p.presence + row) : p.presence_all;
  const uint32_t* allowed = p.allowed ? p.allowed + row * p.allowed_ld : nullptr;
  const long long* said = p.tokens + row * p.tokens_ld;
  auto entry = [&](int i) {  // of token i in the counts, -1: not of this part
    const long long token = __ldg(said + i);
    return token >= max(begin, 0LL) && token < end ? int(token - begin) : -1;
  };
  auto count = [&](int at, int i) {
    if (at < 0) return;
    if (i < prompt)
      atomicOr(&counts[at], 0x80000000u);
    else
      atomicAdd(&counts[at], 1u);
  };
  int at[LG_HELD];
  float value[LG_HELD];
  auto entries = [&](int from) {
#pragma unroll
    for (int j = 0; j < LG_HELD; ++j) at[j] = from + j * THREADS < length ? entry(from + j * THREADS) : -1;
  };
  // the logits of entries that nobody has taken yet; the others' places become -1.  (All loads of one kind behind one another, not a token's.)
  auto take = [&]() {
    uint32_t seen[LG_HELD];
    float bias[LG_HELD];
    uint32_t word[LG_HELD];
#pragma unroll
    for (int j = 0; j < LG_HELD; ++j) {
      seen[j] = at[j] < 0 ? 0u : atomicExch(&counts[at[j]], 0u);
      if (!seen[j]) at[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < LG_HELD; ++j) {
      const long long token = begin + at[j];
      value[j] = at[j] < 0 ? 0.f : lg_load(x + token);
      bias[j] = at[j] < 0 || !p.bias ? 0.f
                : p.bias_fp32        ? __ldg(static_cast<const float*>(p.bias) + row * p.bias_ld + token)
                                     : __bfloat162float(static_cast<const bf16*>(p.bias)[row * p.bias_ld + token]);
      word[j] = at[j] < 0 || !allowed ? ~0u : __ldg(allowed + (token >> 5));
    }
#pragma unroll
    for (int j = 0; j < LG_HELD; ++j) {
      float v = value[j];
      if (at[j] >= 0) v = v > 0.f ? v / repetition : v * repetition;
      const uint32_t often = seen[j] & 0x7fffffffu;
      if (often) v -= frequency * float(often) + presence;
      if (p.bias) v += bias[j];
      value[j] = word[j] >> ((begin + at[j]) & 31) & 1u ? v : -INFINITY;
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int j = 0; j < LG_HELD; ++j)
      if (at[j] >= 0) lg_store(y + begin + at[j], value[j]);
  };
  entries(threadIdx.x);
  if (FORM) stream_part<T, FORM == 1>(p, row, int(begin), int(end));
  __syncthreads();
#pragma unroll
  for (int j = 0; j < LG_HELD; ++j) count(at[j], threadIdx.x + j * THREADS);
#pragma unroll 4
  for (int i = threadIdx.x + LG_HELD * THREADS; i < length; i += THREADS) count(entry(i), i);
  __syncthreads();
  take();
  if (!FORM) {
    lg_wait_prior();
    lg_launch_next();
  }
  store();
  for (int i = threadIdx.x + LG_HELD * THREADS; i < length; i += LG_HELD * THREADS) {
    entries(i);
    take();
    store();
  }
}

template <typename T, bool WIDE>
static int lg_stream(const LogitsParams& p, int rows, cudaStream_t stream) {
  constexpr int N = WIDE ? Vec<T>::N : 1, ROUND = LG_THREADS * N;
  // entries of a block: a row's over as many as make four blocks per SM of all rows, whole rounds
  const long long entries = (long long)p.vocab + N - 1, blocks = max(1LL, 148LL * 4 / rows);
  const long long part = min((1LL << 30) / ROUND * ROUND, ((entries + blocks - 1) / blocks + ROUND - 1) / ROUND * ROUND);
  return launch_dependent(adjust_stream_kernel<T, WIDE>, dim3(rows, unsigned((entries + part - 1) / part)), dim3(LG_THREADS), 0, stream, true, p, int(part)) == cudaSuccess ? TPB_OK
                                                                                                                                                                    : TPB_ERR_CUDA;
}

template <typename T, int FORM>
static int lg_seen(const LogitsParams& p, int rows, int part, int parts, cudaStream_t stream) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(adjust_seen_kernel<T, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_ENTRIES * 4) != cudaSuccess) return TPB_ERR_CUDA;
    ready[dev].store(true, std::memory_order_release);
  }
  if (parts > 65535) return TPB_ERR_SIZE;
  return launch_dependent(adjust_seen_kernel<T, FORM>, dim3(rows, unsigned(parts)), dim3(FORM ? LG_THREADS : LG_SEEN_THREADS), size_t(part) * 4, stream, true, p, part) == cudaSuccess ? TPB_OK
                                                                                                                                                               : TPB_ERR_CUDA;
}

template <typename T>
static int lg_launch(const LogitsParams& p, int rows, cudaStream_t stream, int& launches) {
  constexpr int N = Vec<T>::N;
  auto place = [](const void* t) { return reinterpret_cast<uintptr_t>(t) / sizeof(T) % N; };
  const bool wide = place(p.logits) == place(p.out) && (rows == 1 || (p.logits_ld - p.out_ld) % N == 0);
  const bool history = p.tokens && p.width;
  const long long entries = (long long)p.vocab + N - 1;
  launches = 1;
  if (history && rows * entries <= 148LL * 4 * LG_ALONE) {
    // short parts for each SM to have one, in whole vectors
    const long long blocks = max(1LL, 148LL * 2 / rows);
    const int part = int(min((long long)LG_ALONE, max(1024LL, ((entries + blocks - 1) / blocks + 31) / 32 * 32)));
    const int parts = int((entries + part - 1) / part);
    return wide ? lg_seen<T, 1>(p, rows, part, parts, stream) : lg_seen<T, 2>(p, rows, part, parts, stream);
  }
  const int rc = wide ? lg_stream<T, true>(p, rows, stream) : lg_stream<T, false>(p, rows, stream);
  if (rc != TPB_OK || !history) return rc;
  launches = 2;
  // as few parts as fit where there are blocks enough for the SMs, shorter ones else
  const long long parts = max((p.vocab + (long long)LG_ENTRIES - 1) / LG_ENTRIES, min(148LL / rows, (p.vocab + 4095LL) / 4096));
  const int part = int((((p.vocab + parts - 1) / parts) + 3) / 4 * 4);
  return lg_seen<T, 0>(p, rows, part, int((p.vocab + (long long)part - 1) / part), stream);
}

// Whether results may be written where they are: the logits of tokens that a row has had are read once more behind the stream's stores of their neighbours, or (two kernels) while
// they are under way, so that nothing of the two may lie in one place.  Without a history a thread stores what it has read itself.
static bool lg_places(const tpb_adjust_logits_t& a) {
  const long long size = a.dtype ? 4 : 2, row = a.vocab * size, x_pitch = a.logits_ld * size, y_pitch = a.out_ld * size;
  const intptr_t x = reinterpret_cast<intptr_t>(a.logits), y = reinterpret_cast<intptr_t>(a.out);
  const bool one_pitch = a.rows == 1 || x_pitch == y_pitch;
  if (x == y && one_pitch) return !(a.tokens && a.width);
  const long long x_rest = (a.rows - 1) * x_pitch, y_rest = (a.rows - 1) * y_pitch;
  const intptr_t x0 = x + min(0LL, x_rest), x1 = x + max(0LL, x_rest) + row, y0 = y + min(0LL, y_rest), y1 = y + max(0LL, y_rest) + row;
  if (x1 <= y0 || y1 <= x0) return true;
  // rows of one in the gaps of the other's
  if (a.rows == 1 || !one_pitch || x_pitch <= 0) return false;
  const long long apart = ((y - x) % x_pitch + x_pitch) % x_pitch;
  return apart >= row && apart + row <= x_pitch;
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb_adjust_logits(tpb_adjust_logits_t* a, void* stream_) {
  if (!a || !a->logits || !a->out || !a->status || a->rows <= 0 || a->vocab <= 0 || a->width < 0 || a->dtype < 0 || a->dtype > 1) return TPB_ERR_ARG;
  if (a->vocab > 1 << 30) return TPB_ERR_SIZE;
  if (!lg_places(*a)) return TPB_ERR_ARG;
  LogitsParams p = {a->logits, a->out, a->tokens, a->lengths, a->prompts, a->repetition, a->frequency, a->presence, a->bias, reinterpret_cast<const uint32_t*>(a->allowed),
                    static_cast<uint32_t*>(a->status), a->logits_ld, a->out_ld, a->tokens_ld, a->bias_ld, a->allowed_ld, a->vocab, a->width, a->bias_dtype,
                    a->repetition_all, a->frequency_all, a->presence_all};
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  return a->dtype ? lg_launch<float>(p, a->rows, s, a->launches) : lg_launch<bf16>(p, a->rows, s, a->launches);
}

// New tokens into a paged cache, with the norms of their query and key heads and the rotation of their positions on the way.
//
//   n = x * w / sqrt(mean(x^2) + eps)  (heads with a norm);   (a, b) -> (a cos - b sin, b cos + a sin) * factor  over the pairs of the first rotary_dim elements
//
// Bound by memory: every row is read once and written once, 4 bytes per element in all.  A row is a group of head_dim / 8 lanes (a power of two of them) with
// eight elements each, so that the sum of squares and the partner of a pair come by shuffles; the rows of a token (query, key and value heads)
// are dealt out to the groups of one block, or of several blocks where there are few tokens.  The angles are common to a token's heads: one thread per
// frequency evaluates them into shared memory while the rows are on their way.  They are taken modulo a turn in 64 bits (position * frequency in
// 32 bits is off by position * 2^-24 radians, 0.06 at a million), then by sincospif.  Rounded to bf16 once, at the end.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "launch.cuh"
#include "paged.cuh"

namespace tpb {

typedef __nv_bfloat16 bf16;

constexpr int AP_THREADS = 256;
constexpr int AP_MAX_HALF = 128;  // rotary_dim / 2 at head_dim 256

struct AppendParams {
  PagedBatch b;
  const bf16 *q, *k, *v, *q_norm, *k_norm;
  bf16 *q_out, *keys, *values;
  const float* frequencies;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh, k_sp, k_shead, k_ss, v_sp, v_shead, v_ss;
  int q_heads, kv_heads, head_dim, half, interleaved, fill_rest;  // q_heads 0: q is left alone
  float factor, eps;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// The sequence of a row: the last one with starts[s] <= t, by 32-way steps of the warp.  -1: in front of all; n: behind the last.  (Starts that are not in
// order give some sequence, and the caller sees that the row is not one of its.)
__device__ __forceinline__ int sequence_of(const PagedBatch& b, int t, int lane) {
  int low = 0, high = b.n + 1;  // low starts are known to be <= t, those from high on to lie behind
  while (low < high) {
    const int step = (high - low + 31) / 32, i = low + (lane + 1) * step - 1;
    low += step * __popc(__ballot_sync(0xffffffffu, i < high && __ldg(b.starts + min(i, b.n)) <= t));
    high = min(high, low + step - 1);
  }
  return low - 1;
}

template <int LANES>
__global__ void __launch_bounds__(AP_THREADS)
paged_append_kernel(const AppendParams p) {
  __shared__ float cos_s[AP_MAX_HALF], sin_s[AP_MAX_HALF];
  constexpr int GROUPS = AP_THREADS / LANES;  // rows at a time
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x;
  const int c = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int e0 = c * 8;
  const bool on = e0 < p.head_dim;
  const int rows = p.q_heads + 2 * p.kv_heads;

  auto source = [&](int r) {
    return r < p.q_heads ? p.q + t * p.q_st + r * p.q_sh
                         : r < p.q_heads + p.kv_heads ? p.k + t * p.k_st + (r - p.q_heads) * p.k_sh : p.v + t * p.v_st + (r - p.q_heads - p.kv_heads) * p.v_sh;
  };
  // the rows of the first rounds are on their way while the token's place is looked up
  constexpr int AHEAD = 4;
  const int stride = gridDim.y * GROUPS, r0 = blockIdx.y * GROUPS + group;
  uint4 raw[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (on && r0 + i * stride < rows) raw[i] = *reinterpret_cast<const uint4*>(source(r0 + i * stride) + e0);

  const int seq = sequence_of(p.b, t, lane);
  const bool outside = seq < 0 || seq >= p.b.n;
  int position = 0;
  long long k_at = -1, v_at = -1;
  if (!outside) {
    const PagedSequence s = paged_sequence(p.b, seq);
    position = s.past + (t - s.token0);
    int page = -1;
    if (!s.bad && t >= s.token0 && t < s.token0 + s.fresh) page = __ldg(p.b.table + seq * p.b.table_ld + (position >> p.b.page_shift));
    if (page >= 0 && page < p.b.pages) {
      const int at = position & ((1 << p.b.page_shift) - 1);
      k_at = page * p.k_sp + at * p.k_ss;
      v_at = page * p.v_sp + at * p.v_ss;
    } else if (threadIdx.x == 0 && blockIdx.y == 0) {
      atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
    }
  }
  if (outside && !p.fill_rest) return;  // (of the whole block: the token is)
  for (int i = threadIdx.x; i < p.half; i += AP_THREADS) {
    // turns = position * f / (2 pi), less whole turns
    double turns = double(position) * (double(p.frequencies[i]) * 0.15915494309189533577);
    turns -= rint(turns);
    float sn, cs;
    sincospif(float(2.0 * turns), &sn, &cs);
    cos_s[i] = cs * p.factor;
    sin_s[i] = sn * p.factor;
  }
  __syncthreads();

  auto finish = [&](int r, const uint4& u, const bf16* src) {
    const bool is_q = r < p.q_heads, is_v = r >= p.q_heads + p.kv_heads;
    bf16* dst = nullptr;
    if (r < rows) {
      if (is_q)
        dst = p.q_out + t * p.o_st + r * p.o_sh;
      else if (!is_v && k_at >= 0)
        dst = p.keys + k_at + (r - p.q_heads) * p.k_shead;
      else if (is_v && v_at >= 0)
        dst = p.values + v_at + (r - p.q_heads - p.kv_heads) * p.v_shead;
    }
    if (outside) {
      if (is_q && dst && on) *reinterpret_cast<uint4*>(dst + e0) = make_uint4(0, 0, 0, 0);
      return;
    }
    float x[8] = {};
    if (on && r < rows) unpack8(u, x);
    const bf16* weight = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
    float rstd = 1.f;
    if (p.q_norm || p.k_norm) {  // (all lanes of the warp take part)
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (weight) {
        rstd = rsqrtf(sum / p.head_dim + p.eps);
        if (on) {
          float w[8];
          unpack8(__ldg(reinterpret_cast<const uint4*>(weight + e0)), w);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= rstd * w[i];
        }
      }
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
    if (p.half && p.interleaved) {
      if (!is_v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = e0 / 2 + i;
          if (f < p.half) {
            const float cs = cos_s[f], sn = sin_s[f];
            y[2 * i] = x[2 * i] * cs - x[2 * i + 1] * sn;
            y[2 * i + 1] = x[2 * i + 1] * cs + x[2 * i] * sn;
          }
        }
      }
    } else if (p.half && p.half % 8 == 0) {
      const int step = p.half / 8;  // lanes between the elements of a pair
      const bool second = e0 >= p.half;
      const int from = second ? lane - step : lane + step;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl_sync(0xffffffffu, x[i], from & 31);
        if (!is_v && e0 < 2 * p.half) {
          const int f = second ? e0 - p.half + i : e0 + i;
          y[i] = second ? x[i] * cos_s[f] + other * sin_s[f] : x[i] * cos_s[f] - other * sin_s[f];
        }
      }
    } else if (p.half) {
      // pairs that do not lie a multiple of eight elements apart: the partners come from memory once more, before any lane of the warp stores
      if (!is_v && on && r < rows) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = e0 + i;
          if (e < 2 * p.half) {
            const bool second = e >= p.half;
            const int other = second ? e - p.half : e + p.half, f = second ? other : e;
            float o = __bfloat162float(src[other]);
            if (weight) o *= rstd * __bfloat162float(weight[other]);
            y[i] = second ? x[i] * cos_s[f] + o * sin_s[f] : x[i] * cos_s[f] - o * sin_s[f];
          }
        }
      }
      __syncwarp();
    }
    if (dst && on) *reinterpret_cast<uint4*>(dst + e0) = pack8(y);
  };

  // (every lane makes the same rounds: the shuffles are the whole warp's)
  const int first = blockIdx.y * GROUPS + (threadIdx.x & ~31) / LANES;  // row of the warp's first group
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (first + i * stride < rows) finish(r0 + i * stride, raw[i], r0 + i * stride < rows ? source(r0 + i * stride) : nullptr);
  for (int i = AHEAD; first + i * stride < rows; ++i) {
    const int r = r0 + i * stride;
    uint4 u = make_uint4(0, 0, 0, 0);
    const bf16* src = r < rows ? source(r) : nullptr;
    if (on && src) u = *reinterpret_cast<const uint4*>(src + e0);
    finish(r, u, src);
  }
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb_paged_append(const tpb_paged_append_t* a, void* stream_) {
  if (!a || !a->k || !a->v || !a->keys || !a->values || !a->table || !a->starts || !a->past || !a->status || !a->q != !a->q_out) return TPB_ERR_ARG;
  if (a->n <= 0 || a->tokens <= 0 || a->heads < 0 || a->kv_heads <= 0 || a->pages <= 0 || a->table_width <= 0 || (a->q && a->heads <= 0)) return TPB_ERR_ARG;
  if (a->head_dim <= 0 || a->head_dim > 256 || a->head_dim % 8 || a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return TPB_ERR_ARG;
  if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 2 || (a->rotary_dim && !a->frequencies)) return TPB_ERR_ARG;
  uintptr_t addresses = 0;
  for (const void* t : {a->q, a->k, a->v, (const void*)a->q_out, (const void*)a->keys, (const void*)a->values, a->q_norm, a->k_norm}) addresses |= reinterpret_cast<uintptr_t>(t);
  const long long strides = (a->q ? a->q_st | a->q_sh | a->o_st | a->o_sh : 0) | a->k_st | a->k_sh | a->v_st | a->v_sh | a->k_sp | a->k_shead | a->k_ss | a->v_sp |
                            a->v_shead | a->v_ss;
  if ((addresses & 15) || (strides & 7)) return TPB_ERR_ALIGN;
  AppendParams p = {};
  int shift = 0;
  while ((1 << shift) < a->page_size) ++shift;
  p.b = {a->starts, a->past, a->table, a->table_ld, a->n, a->tokens, a->table_width, a->pages, shift, INT_MAX, static_cast<uint32_t*>(a->status)};
  p.q = static_cast<const bf16*>(a->q), p.k = static_cast<const bf16*>(a->k), p.v = static_cast<const bf16*>(a->v);
  p.q_norm = static_cast<const bf16*>(a->q_norm), p.k_norm = static_cast<const bf16*>(a->k_norm);
  p.q_out = static_cast<bf16*>(a->q_out), p.keys = static_cast<bf16*>(a->keys), p.values = static_cast<bf16*>(a->values);
  p.frequencies = a->frequencies;
  p.q_st = a->q_st, p.q_sh = a->q_sh, p.k_st = a->k_st, p.k_sh = a->k_sh, p.v_st = a->v_st, p.v_sh = a->v_sh, p.o_st = a->o_st, p.o_sh = a->o_sh;
  p.k_sp = a->k_sp, p.k_shead = a->k_shead, p.k_ss = a->k_ss, p.v_sp = a->v_sp, p.v_shead = a->v_shead, p.v_ss = a->v_ss;
  p.q_heads = a->q ? a->heads : 0;
  p.kv_heads = a->kv_heads, p.head_dim = a->head_dim, p.half = a->rotary_dim / 2, p.interleaved = a->interleaved, p.fill_rest = a->fill_rest;
  p.factor = a->factor, p.eps = a->eps;
  const int lanes = a->head_dim <= 64 ? 8 : a->head_dim <= 128 ? 16 : 32;
  const int rows = p.q_heads + 2 * p.kv_heads, groups = AP_THREADS / lanes;
  const int rounds = (rows + groups - 1) / groups;
  // few tokens: a token's rows over several blocks
  const int split = a->tokens >= 148 * 4 ? 1 : rounds;
  const dim3 grid(a->tokens, split);
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  if (lanes == 8)
    paged_append_kernel<8><<<grid, AP_THREADS, 0, s>>>(p);
  else if (lanes == 16)
    paged_append_kernel<16><<<grid, AP_THREADS, 0, s>>>(p);
  else
    paged_append_kernel<32><<<grid, AP_THREADS, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

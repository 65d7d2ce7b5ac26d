// New tokens into a paged cache, with the norms of their query and key heads and the rotation of their positions on the way.
//
//   n = x * w / sqrt(mean(x^2) + eps)  (heads with a norm);   (a, b) -> (a cos - b sin, b cos + a sin) * factor  over the pairs of the first rotary_dim elements
//
// Bound by memory: every row is read once and written once, 4 bytes per element in all.  A row is a group of head_dim / 8 lanes (a power of two of them) with
// eight elements each, so that the sum of squares and the partner of a pair come by shuffles; the rows (query, key and value heads) of a block's tokens are
// dealt out to its groups.  A token's place (a search for its sequence, its lengths, its page: four loads behind one another) and its angles are common to its
// heads: a warp per token looks the place up and a thread per frequency evaluates the angle, while the first rows are on their way.  Many tokens go eight to a
// block, so that this chain is paid once for 8 x 48 rows; few tokens have several blocks each.  Angles are taken modulo a turn in 64 bits (position *
// frequency in 32 bits is off by position * 2^-24 radians, 0.06 at a million), then by sincospif.  Rounded to bf16 once, at the end.
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
constexpr int AP_TOKENS = 8;      // of a block, at most: one per warp

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

struct AppendPlace {  // of a token
  int position;
  int inside;           // of a sequence
  long long k_at, v_at; // -1: not stored
};

template <int LANES>
__global__ void __launch_bounds__(AP_THREADS, 4)
paged_append_kernel(const AppendParams p, int tokens_of_block) {
  __shared__ float cos_s[AP_TOKENS * AP_MAX_HALF], sin_s[AP_TOKENS * AP_MAX_HALF];
  __shared__ AppendPlace places[AP_TOKENS];
  constexpr int GROUPS = AP_THREADS / LANES;  // rows at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * tokens_of_block, tokens = min(tokens_of_block, p.b.tokens - t0);
  const int e0 = threadIdx.x % LANES * 8;
  const bool on = e0 < p.head_dim;
  const int rows = p.q_heads + 2 * p.kv_heads;
  // rows of the block: (token, head), heads fastest, one to a group and round; every lane makes its warp's rounds (the shuffles are the whole warp's)
  const int all = tokens * rows, stride = gridDim.y * GROUPS;
  const int i0 = blockIdx.y * GROUPS + threadIdx.x / LANES, first = blockIdx.y * GROUPS + (threadIdx.x & ~31) / LANES;

  auto source = [&](int i) {
    const long long t = t0 + i / rows;
    const int r = i % rows;
    return r < p.q_heads ? p.q + t * p.q_st + r * p.q_sh
                         : r < p.q_heads + p.kv_heads ? p.k + t * p.k_st + (r - p.q_heads) * p.k_sh : p.v + t * p.v_st + (r - p.q_heads - p.kv_heads) * p.v_sh;
  };
  constexpr int AHEAD = 4;
  uint4 raw[AHEAD];
  auto fetch = [&](int from) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = from + j * stride;
      if (on && i < all) raw[j] = *reinterpret_cast<const uint4*>(source(i) + e0);
    }
  };
  fetch(i0);

  if (warp < tokens) {
    const int t = t0 + warp, seq = sequence_of(p.b, t, lane);
    AppendPlace at = {0, seq >= 0 && seq < p.b.n, -1, -1};
    if (at.inside) {
      const PagedSequence s = paged_sequence(p.b, seq);
      at.position = s.past + (t - s.token0);
      int page = -1;
      if (!s.bad && t >= s.token0 && t < s.token0 + s.fresh) page = __ldg(p.b.table + seq * p.b.table_ld + (at.position >> p.b.page_shift));
      if (page >= 0 && page < p.b.pages) {
        const int slot = at.position & ((1 << p.b.page_shift) - 1);
        at.k_at = page * p.k_sp + slot * p.k_ss;
        at.v_at = page * p.v_sp + slot * p.v_ss;
      } else if (lane == 0 && blockIdx.y == 0) {
        atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
      }
    }
    if (lane == 0) places[warp] = at;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * p.half; i += AP_THREADS) {
    const int t = i / p.half, f = i % p.half;
    // turns = position * f / (2 pi), less whole turns
    double turns = double(places[t].position) * (double(__ldg(p.frequencies + f)) * 0.15915494309189533577);
    turns -= rint(turns);
    float sn, cs;
    sincospif(float(2.0 * turns), &sn, &cs);
    cos_s[t * AP_MAX_HALF + f] = cs * p.factor;
    sin_s[t * AP_MAX_HALF + f] = sn * p.factor;
  }
  __syncthreads();

  auto finish = [&](int i, const uint4& u) {
    const bool there = i < all;
    const int t = there ? i / rows : 0, r = there ? i % rows : 0;
    const bool is_q = r < p.q_heads, is_v = r >= p.q_heads + p.kv_heads;
    const AppendPlace at = places[t];
    bf16* dst = nullptr;
    if (there && on) {
      if (is_q)
        dst = at.inside || p.fill_rest ? p.q_out + (t0 + t) * p.o_st + r * p.o_sh : nullptr;
      else if (!is_v && at.k_at >= 0)
        dst = p.keys + at.k_at + (r - p.q_heads) * p.k_shead;
      else if (is_v && at.v_at >= 0)
        dst = p.values + at.v_at + (r - p.q_heads - p.kv_heads) * p.v_shead;
    }
    const float *cs = cos_s + t * AP_MAX_HALF, *sn = sin_s + t * AP_MAX_HALF;
    float x[8] = {};
    if (on && there) unpack8(u, x);
    const bf16* weight = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
    float rstd = 1.f;
    if (p.q_norm || p.k_norm) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (weight) {
        rstd = rsqrtf(sum / p.head_dim + p.eps);
        if (on) {
          float w[8];
          unpack8(__ldg(reinterpret_cast<const uint4*>(weight + e0)), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= rstd * w[j];
        }
      }
    }
    if (p.half && p.interleaved) {
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int f = e0 / 2 + j;
          if (f < p.half) {
            const float a = x[2 * j], b = x[2 * j + 1];
            x[2 * j] = a * cs[f] - b * sn[f];
            x[2 * j + 1] = b * cs[f] + a * sn[f];
          }
        }
      }
    } else if (p.half && p.half % 8 == 0) {
      const int step = p.half / 8;  // lanes between the elements of a pair
      const bool second = e0 >= p.half, turns = !is_v && e0 < 2 * p.half;
      const int from = (second ? lane - step : lane + step) & 31, f0 = second ? e0 - p.half : e0;
      // (a, b) -> (a cos - b sin, b cos + a sin): the second of a pair adds what the first subtracts
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 c = turns ? *reinterpret_cast<const float4*>(cs + f0 + j) : make_float4(1.f, 1.f, 1.f, 1.f);
        const float4 s = turns ? *reinterpret_cast<const float4*>(sn + f0 + j) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float cj[4] = {c.x, c.y, c.z, c.w}, sj[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float other = __shfl_sync(0xffffffffu, x[j + k], from);
          if (turns) x[j + k] = x[j + k] * cj[k] + (second ? other : -other) * sj[k];
        }
      }
    } else if (p.half) {
      // pairs that do not lie a multiple of eight elements apart: the partners come from memory once more, before any lane of the warp stores
      if (!is_v && on && there) {
        const bf16* src = source(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = e0 + j;
          if (e < 2 * p.half) {
            const bool second = e >= p.half;
            const int other = second ? e - p.half : e + p.half, f = second ? other : e;
            float o = __bfloat162float(src[other]);
            if (weight) o *= rstd * __bfloat162float(weight[other]);
            x[j] = second ? x[j] * cs[f] + o * sn[f] : x[j] * cs[f] - o * sn[f];
          }
        }
      }
      __syncwarp();
    }
    if (dst) *reinterpret_cast<uint4*>(dst + e0) = at.inside ? pack8(x) : make_uint4(0, 0, 0, 0);
  };

  for (int base = 0; first + base < all; base += AHEAD * stride) {
    if (base) fetch(i0 + base);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (first + base + j * stride < all) finish(i0 + base + j * stride, raw[j]);
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
  // tokens to a block where that leaves four blocks to an SM and more, else a token's rows over several blocks
  const int per_block = a->tokens >= 148 * 4 * AP_TOKENS ? AP_TOKENS : a->tokens >= 148 * 4 * 2 ? 2 : 1;
  const dim3 grid((a->tokens + per_block - 1) / per_block, a->tokens >= 148 * 4 ? 1 : (rows + groups - 1) / groups);
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  if (lanes == 8)
    paged_append_kernel<8><<<grid, AP_THREADS, 0, s>>>(p, per_block);
  else if (lanes == 16)
    paged_append_kernel<16><<<grid, AP_THREADS, 0, s>>>(p, per_block);
  else
    paged_append_kernel<32><<<grid, AP_THREADS, 0, s>>>(p, per_block);
  return cudaGetLastError() == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

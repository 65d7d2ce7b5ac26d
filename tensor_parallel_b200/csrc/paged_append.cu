// New tokens into a paged cache, with the norms of their query and key heads and the rotation of their positions on the way.
//
//   n = x * w / sqrt(mean(x^2) + eps)  (heads with a norm);   (a, b) -> (a cos - b sin, b cos + a sin) * factor  over the pairs of the first rotary_dim elements
//
// Bound by memory: every row is read once and written once, 4 bytes per element in all; next to it by instructions (65 % of the issue slots at 16.4 k tokens: 313 for the 16 elements
// of each lane, angles and weights from shared memory for every row, as consecutive rows of a group are of different tokens, and 52 bytes that do not fit 64 registers), so a lane has both elements of its pairs and
// needs no exchange for them: a row is a group of head_dim / 16 lanes (a power of two of them) with two chunks of eight elements each, rotary_dim / 2 apart
// (with one chunk per lane and shuffles, 16 k tokens of 48 heads of 128 took 168 us).  The rows (query, key and value heads) of a block's tokens are dealt out to its
// groups.  A token's place (a search for its sequence, its lengths, its page: four loads behind one another) and its angles are common to its heads: a
// warp per token looks the place up and a thread per frequency evaluates the angle, while the first rows are on their way.  Many tokens go eight to a block, so
// that this chain is paid once for 8 x 48 rows; few tokens have several blocks each.  Angles are taken modulo a turn in 64 bits (position * frequency
// in 32 bits is off by position * 2^-24 radians, 0.06 at a million), then by sincospif.  Rounded to bf16 once, at the end.
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
  long long k_sp, k_ss, v_sp, v_ss;
  int q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;  // (pointers then are one 32 x 32 + 64 bit product away)
  unsigned k_shead, v_shead;                           // in 16 bytes, so that 64 GB between heads are within reach (those of the rows as well: 89 us for 87, more spills)
  int q_heads, kv_heads, head_dim, half, interleaved, fill_rest;  // q_heads 0: q is left alone
  float factor, eps, inv_dim;
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

// How the elements of a pair lie: none are turned; a multiple of eight apart; side by side; any other distance apart.
enum { TURN_NONE, TURN_HALVES, TURN_PAIRS, TURN_ODD };

template <int LANES, int TURN>
__global__ void __launch_bounds__(AP_THREADS, 4)
paged_append_kernel(const AppendParams p, int tokens_of_block) {
  __shared__ __align__(16) float cos_s[AP_TOKENS * AP_MAX_HALF], sin_s[AP_TOKENS * AP_MAX_HALF];
  __shared__ __align__(16) float norm_s[2][2 * AP_MAX_HALF];  // weights of queries and keys
  __shared__ AppendPlace places[AP_TOKENS];
  constexpr int GROUPS = AP_THREADS / LANES;  // rows at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * tokens_of_block, tokens = min(tokens_of_block, p.b.tokens - t0);
  const int rows = p.q_heads + 2 * p.kv_heads, chunks = p.head_dim / 8;
  // this lane's chunks: pairs of the turned part, then those that stay
  const int l = threadIdx.x % LANES, turned = TURN == TURN_HALVES ? p.half / 8 : 0;
  const bool pair = l < turned;
  const int c0 = pair ? l : TURN == TURN_HALVES ? 2 * turned + 2 * (l - turned) : l, c1 = pair ? l + turned : TURN == TURN_HALVES ? c0 + 1 : l + LANES;
  const bool on0 = c0 < chunks, on1 = c1 < chunks;
  // rows of the block: (token, head), heads fastest, one to a group and round; every lane makes its warp's rounds (the shuffles are the whole warp's)
  const int all = tokens * rows, stride = gridDim.y * GROUPS, step_tokens = stride / rows, step_rows = stride % rows;
  const int i0 = blockIdx.y * GROUPS + threadIdx.x / LANES, first = blockIdx.y * GROUPS + (threadIdx.x & ~31) / LANES;
  struct Cursor {
    int t, r;
  };
  auto step = [&](Cursor& c) {
    c.t += step_tokens;
    c.r += step_rows;
    if (c.r >= rows) {
      c.r -= rows;
      ++c.t;
    }
  };
  auto source = [&](const Cursor& c) {
    const bool is_q = c.r < p.q_heads, is_k = c.r < p.q_heads + p.kv_heads;
    const bf16* base = is_q ? p.q : is_k ? p.k : p.v;
    const int st = is_q ? p.q_st : is_k ? p.k_st : p.v_st, sh = is_q ? p.q_sh : is_k ? p.k_sh : p.v_sh, r = is_q ? c.r : is_k ? c.r - p.q_heads : c.r - p.q_heads - p.kv_heads;
    return base + (long long)(t0 + c.t) * st + (long long)r * sh;
  };
  constexpr int AHEAD = 2;  // rows on their way (three, in three blocks per SM: 88 -> 90 us, 32 KV heads 151 -> 157)
  uint4 raw[AHEAD][2];
  Cursor next = {i0 / rows, i0 % rows}, at = next;
  auto fetch = [&](uint4 (&u)[2]) {
    if (next.t < tokens) {
      const bf16* src = source(next);
      if (on0) u[0] = *reinterpret_cast<const uint4*>(src + c0 * 8);
      if (on1) u[1] = *reinterpret_cast<const uint4*>(src + c1 * 8);
    }
    step(next);
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched ahead of the previous kernel's end: nothing is read or written before that)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) fetch(raw[j]);

  if (warp < tokens) {
    const int t = t0 + warp, seq = sequence_of(p.b, t, lane);
    AppendPlace place = {0, seq >= 0 && seq < p.b.n, -1, -1};
    if (place.inside) {
      const PagedSequence s = paged_sequence(p.b, seq);
      place.position = s.past + (t - s.token0);
      int page = -1;
      if (!s.bad && t >= s.token0 && t < s.token0 + s.fresh) page = __ldg(p.b.table + seq * p.b.table_ld + (place.position >> p.b.page_shift));
      if (page >= 0 && page < p.b.pages) {
        const int slot = place.position & ((1 << p.b.page_shift) - 1);
        place.k_at = page * p.k_sp + slot * p.k_ss;
        place.v_at = page * p.v_sp + slot * p.v_ss;
      } else if (lane == 0 && blockIdx.y == 0) {
        atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
      }
    }
    if (lane == 0) places[warp] = place;
  }
  const bool norms = p.q_norm || p.k_norm;
  if (norms)
    for (int i = threadIdx.x; i < p.head_dim; i += AP_THREADS) {
      norm_s[0][i] = p.q_norm ? __bfloat162float(p.q_norm[i]) : 1.f;
      norm_s[1][i] = p.k_norm ? __bfloat162float(p.k_norm[i]) : 1.f;
    }
  __syncthreads();
  if (TURN != TURN_NONE) {
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
  }

  auto times = [](float (&x)[8], const float* w) {  // x *= w, eight of them from shared memory
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const float4 f = *reinterpret_cast<const float4*>(w + j);
      ffma2(x[j], x[j + 1], x[j], x[j + 1], f.x, f.y, 0.f, 0.f);
      ffma2(x[j + 2], x[j + 3], x[j + 2], x[j + 3], f.z, f.w, 0.f, 0.f);
    }
  };
  auto finish = [&](const Cursor& c, const uint4 (&u)[2]) {
    const bool there = c.t < tokens, is_q = c.r < p.q_heads, is_v = c.r >= p.q_heads + p.kv_heads;
    const AppendPlace place = places[there ? c.t : 0];
    bf16* dst = nullptr;
    if (is_q) {
      if (there && (place.inside || p.fill_rest)) dst = p.q_out + (long long)(t0 + c.t) * p.o_st + (long long)c.r * p.o_sh;
    } else {
      const long long into = is_v ? place.v_at : place.k_at;
      const int r = c.r - p.q_heads - (is_v ? p.kv_heads : 0);
      if (there && into >= 0) dst = (is_v ? p.values : p.keys) + into + (static_cast<unsigned long long>(unsigned(r)) * (is_v ? p.v_shead : p.k_shead) << 3);
    }
    uint4 y0 = u[0], y1 = u[1];
    if (__any_sync(0xffffffffu, there && !is_v)) {
      float x0[8] = {}, x1[8] = {};
      if (on0 && there) unpack8(u[0], x0);
      if (on1 && there) unpack8(u[1], x1);
      const bool normed = !is_v && (is_q ? p.q_norm : p.k_norm);
      float rstd = 1.f;
      if (norms) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          ffma2(s0, s1, x0[j], x0[j + 1], x0[j], x0[j + 1], s0, s1);
          ffma2(s0, s1, x1[j], x1[j + 1], x1[j], x1[j + 1], s0, s1);
        }
        s0 += s1;
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, d);
        if (normed) {
          rstd = rsqrtf(s0 * p.inv_dim + p.eps);
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            ffma2(x0[j], x0[j + 1], x0[j], x0[j + 1], rstd, rstd, 0.f, 0.f);
            ffma2(x1[j], x1[j + 1], x1[j], x1[j + 1], rstd, rstd, 0.f, 0.f);
          }
          const float* w = norm_s[is_q ? 0 : 1];
          if (on0) times(x0, w + c0 * 8);
          if (on1) times(x1, w + c1 * 8);
        }
      }
      const float *cs = cos_s + (there ? c.t : 0) * AP_MAX_HALF, *sn = sin_s + (there ? c.t : 0) * AP_MAX_HALF;
      if (TURN == TURN_HALVES && pair) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 cv = *reinterpret_cast<const float4*>(cs + c0 * 8 + j), sv = *reinterpret_cast<const float4*>(sn + c0 * 8 + j);
          const float cj[4] = {cv.x, cv.y, cv.z, cv.w}, sj[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            float &a0 = x0[j + k], &a1 = x0[j + k + 1], &b0 = x1[j + k], &b1 = x1[j + k + 1];
            float m0, m1, n0, n1;
            ffma2(m0, m1, b0, b1, -sj[k], -sj[k + 1], 0.f, 0.f);
            ffma2(n0, n1, a0, a1, sj[k], sj[k + 1], 0.f, 0.f);
            ffma2(a0, a1, a0, a1, cj[k], cj[k + 1], m0, m1);
            ffma2(b0, b1, b0, b1, cj[k], cj[k + 1], n0, n1);
          }
        }
      } else if (TURN == TURN_PAIRS) {
        auto turn = [&](float (&x)[8], int chunk) {
          const int f0 = chunk * 4;
          if (f0 >= p.half) return;
          const float4 cv = *reinterpret_cast<const float4*>(cs + f0), sv = *reinterpret_cast<const float4*>(sn + f0);  // (those beyond the turned part are not used)
          const float cj[4] = {cv.x, cv.y, cv.z, cv.w}, sj[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (f0 + j < p.half) {
              const float a = x[2 * j], b = x[2 * j + 1];
              x[2 * j] = a * cj[j] - b * sj[j];
              x[2 * j + 1] = b * cj[j] + a * sj[j];
            }
        };
        turn(x0, c0);
        turn(x1, c1);
      } else if (TURN == TURN_ODD) {
        // the partners come from memory once more, before any lane of the warp stores
        auto turn = [&](float (&x)[8], int chunk, bool on) {
          if (!on || !there || is_v) return;
          const bf16* src = source(c);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = chunk * 8 + j;
            if (e >= 2 * p.half) continue;
            const bool second = e >= p.half;
            const int other = second ? e - p.half : e + p.half, f = second ? other : e;
            float o = __bfloat162float(src[other]);
            if (normed) o = o * rstd * norm_s[is_q ? 0 : 1][other];
            x[j] = second ? x[j] * cs[f] + o * sn[f] : x[j] * cs[f] - o * sn[f];
          }
        };
        turn(x0, c0, on0);
        turn(x1, c1, on1);
        __syncwarp();
      }
      if (!is_v) {
        y0 = pack8(x0);
        y1 = pack8(x1);
      }
    }
    if (dst) {
      if (!place.inside) y0 = y1 = make_uint4(0, 0, 0, 0);
      if (on0) *reinterpret_cast<uint4*>(dst + c0 * 8) = y0;
      if (on1) *reinterpret_cast<uint4*>(dst + c1 * 8) = y1;
    }
  };

  for (int base = 0; first + base < all; base += AHEAD * stride) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (first + base + j * stride >= all) break;
      const uint4 taken[2] = {raw[j][0], raw[j][1]};
      fetch(raw[j]);
      finish(at, taken);
      step(at);
    }
  }
}

template <int LANES>
static cudaError_t ap_launch(const AppendParams& p, dim3 grid, int per_block, cudaStream_t stream) {
  auto kernel = !p.half            ? paged_append_kernel<LANES, TURN_NONE>
                : p.interleaved     ? paged_append_kernel<LANES, TURN_PAIRS>
                : p.half % 8 == 0   ? paged_append_kernel<LANES, TURN_HALVES>
                                    : paged_append_kernel<LANES, TURN_ODD>;
  return launch_dependent(kernel, grid, dim3(AP_THREADS), 0, stream, true, p, per_block);
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
  for (const long long t : {a->q_st, a->q_sh, a->k_st, a->k_sh, a->v_st, a->v_sh, a->o_st, a->o_sh})
    if (t >= TPB_APPEND_ROW_STRIDE || t < 0) return TPB_ERR_SIZE;
  for (const long long t : {a->k_shead, a->v_shead})
    if (t >= TPB_APPEND_HEAD_STRIDE || t < 0) return TPB_ERR_SIZE;
  p.q_st = int(a->q_st), p.q_sh = int(a->q_sh), p.k_st = int(a->k_st), p.k_sh = int(a->k_sh), p.v_st = int(a->v_st), p.v_sh = int(a->v_sh);
  p.o_st = int(a->o_st), p.o_sh = int(a->o_sh), p.k_shead = unsigned(a->k_shead / 8), p.v_shead = unsigned(a->v_shead / 8);
  p.k_sp = a->k_sp, p.k_ss = a->k_ss, p.v_sp = a->v_sp, p.v_ss = a->v_ss;
  p.inv_dim = 1.f / float(a->head_dim);
  p.q_heads = a->q ? a->heads : 0;
  p.kv_heads = a->kv_heads, p.head_dim = a->head_dim, p.half = a->rotary_dim / 2, p.interleaved = a->interleaved, p.fill_rest = a->fill_rest;
  p.factor = a->factor, p.eps = a->eps;
  const int lanes = a->head_dim <= 64 ? 4 : a->head_dim <= 128 ? 8 : 16;
  const int rows = p.q_heads + 2 * p.kv_heads, groups = AP_THREADS / lanes;
  // tokens to a block where that leaves four blocks to an SM and more, else a token's rows over several blocks
  const int per_block = a->tokens >= 148 * 4 * AP_TOKENS ? AP_TOKENS : a->tokens >= 148 * 4 * 2 ? 2 : 1;
  const dim3 grid((a->tokens + per_block - 1) / per_block, a->tokens >= 148 * 4 ? 1 : (rows + groups - 1) / groups);
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  const cudaError_t launched = lanes == 4 ? ap_launch<4>(p, grid, per_block, s) : lanes == 8 ? ap_launch<8>(p, grid, per_block, s) : ap_launch<16>(p, grid, per_block, s);
  return launched == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

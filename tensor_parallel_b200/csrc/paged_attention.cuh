// Shared by the two kernels that attend to a paged cache (paged_attention.cu, paged_attention_sm100.cu).
#pragma once
#include <atomic>

#include "paged.cuh"

namespace tpb {

inline int pa_sms() {
  static std::atomic<int> sms[64];
  int dev = 0, count = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return count;
  count = sms[dev].load(std::memory_order_relaxed);
  if (!count) {
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || count <= 0) return 148;
    sms[dev].store(count, std::memory_order_relaxed);
  }
  return count;
}

typedef __nv_bfloat16 bf16;

// Results of a row tile whose keys lie in several CTAs' ranges: piece by piece in a workspace, joined by a kernel of its own.  The first piece is in
// slot 2c + 1 of the CTA c in whose range the keys begin, those of the CTAs behind it in their slots 2c'.
struct PagedParts {
  float* o;    // [2 per CTA][rows of a tile][head_dim], not divided by the sum
  float2* ml;  // [2 per CTA][rows of a tile] maximum (of scaled scores, in powers of two; -inf: the piece adds nothing) and sum
  int4* joins; // [2 per CTA]: (first row of the queries, first row of the tile, rows, KV head) and (last CTA); first -1: nothing to join
  int rows;    // of a tile
};

struct PagedAttnParams {
  PagedBatch b;
  const bf16* q;
  bf16* out;
  long long q_st, q_sh, o_st, o_sh;
  int heads, kv_heads, group, window;
  int rows_low, rows_high;  // sequences with rows (new tokens x group) in [rows_low, rows_high] are this launch's
  int takes_bad;            // and those whose lengths are not possible
  int fill_rest;            // rows outside all sequences become zeros
  int whole;                // ranges end where row tiles do: nothing is cut, and nothing to join
  float scale_log2e;
  PagedParts parts;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pa_wait_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pa_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Number of the sequence and its place on the line of costs at which a CTA's range begins.
template <int THREADS>
struct RangeSearch {
  long long scan[THREADS / 32];
  long long begin;
  int seq;
};
// A CTA's equal share [from, to) of the line on which all sequences' costs lie one behind the other; `at` receives where it begins.  Called by all threads.
template <int THREADS, typename Cost>
__device__ __forceinline__ void share_out(int n, int least, RangeSearch<THREADS>& at, Cost cost_of, long long& share, long long& from, long long& to) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto scan = [&](long long v, long long& before, long long& total) {
    long long inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 31) at.scan[warp] = inc;
    __syncthreads();
    before = inc - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += at.scan[w];
      total += at.scan[w];
    }
  };
  if (threadIdx.x == 0) {
    at.seq = n;
    at.begin = 0;
  }
  long long all = 0, mine_before = 0, mine = 0;
  for (int base = 0; base < n; base += THREADS) {
    const int s = base + threadIdx.x;
    long long before, total;
    mine = s < n ? cost_of(s) : 0;
    scan(mine, before, total);
    mine_before = all + before;
    all += total;
  }
  // (64-bit divisions are long)
  share = max((long long)least, all < INT_MAX / 2 ? (long long)((unsigned(all) + gridDim.x - 1) / gridDim.x) : (all + gridDim.x - 1) / gridDim.x);
  from = min(all, share * blockIdx.x);
  to = min(all, from + share);
  if (n <= THREADS) {
    if (mine > 0 && from >= mine_before && from < mine_before + mine) {
      at.seq = threadIdx.x;
      at.begin = mine_before;
    }
  } else {
    long long so_far = 0;
    for (int base = 0; base < n && so_far <= from; base += THREADS) {
      const int s = base + threadIdx.x;
      long long before, total;
      const long long cost = s < n ? cost_of(s) : 0;
      scan(cost, before, total);
      before += so_far;
      if (cost > 0 && from >= before && from < before + cost) {
        at.seq = s;
        at.begin = before;
      }
      so_far += total;
    }
  }
  __syncthreads();
}

// Rows of the result outside all sequences (zeros), or of one whose lengths are not possible (NaN).
template <int D, int THREADS>
__device__ __forceinline__ void fill_rows(const PagedAttnParams& p, long long t0, int count, uint32_t bits) {
  const int chunks = p.heads * (D / 8);
  for (int i = blockIdx.x; i < count; i += gridDim.x)
    for (int c = threadIdx.x; c < chunks; c += THREADS)
      *reinterpret_cast<uint4*>(p.out + (t0 + i) * p.o_st + (c / (D / 8)) * p.o_sh + (c % (D / 8)) * 8) = make_uint4(bits, bits, bits, bits);
}
template <int D, int THREADS>
__device__ __forceinline__ void fill_around(const PagedAttnParams& p) {
  const int used0 = min(max(__ldg(p.b.starts), 0), p.b.tokens);
  const int used1 = min(max(__ldg(p.b.starts + p.b.n), used0), p.b.tokens);
  fill_rows<D, THREADS>(p, 0, used0, 0u);
  fill_rows<D, THREADS>(p, used1, p.b.tokens - used1, 0u);
}

// The launch for sequences with many query rows (paged_attention_sm100.cu).  ahead: of the kernel in front of it in the stream, whose results it does not
// read; it ends after it.
constexpr int PW_ROWS = 256;  // of its tiles
int pw_grid(int head_dim);
int pw_launch(int head_dim, const PagedAttnParams& p, const CUtensorMap& k, const CUtensorMap& v, int grid, bool ahead, cudaStream_t stream);
int pw_tile(int head_dim);  // keys of a tile: the rows of a box at most

}  // namespace tpb

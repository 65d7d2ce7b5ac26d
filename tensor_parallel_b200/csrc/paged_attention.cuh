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

// Results of a row tile whose keys lie in several ranges: piece by piece in a workspace, joined by a kernel of its own.  The first piece is in
// slot 2c + 1 of the range c in which the keys begin, those of the ranges behind it in their slots 2c'.
struct PagedParts {
  float* o;    // [2 per range][rows of a tile][head_dim], not divided by the sum
  float2* ml;  // [2 per range][rows of a tile] maximum (of scaled scores, in powers of two) and sum; -inf and 0: the piece adds nothing
  int4* joins; // [2 per range]: (first row of the queries, first row of the tile, rows, KV head) and (last range); first -1: nothing to join
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
  int ranges;               // of the line, where the SMs are not shared with another launch
  int few_high, split_sms;  // a second launch beside this one (sequences with up to few_high rows are the first's), the two on so many SMs; 0: on all of them, one by one
  float scale_log2e;
  PagedParts parts;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pa_wait_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pa_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The two launches of a batch with both kinds of sequences share out the SMs, so that one loads while the other multiplies: an SM alone reads about twice what
// its part is when all of them read.  Both launches estimate from the lengths what either has to do, in the time that an SM needs for a tile of 64 keys
// and up to 16 rows of the first; in whole numbers, whose sums are the same in both.  (In a graph, one after the other on all SMs / side by side, us: 31 decoding, 777 tokens behind 3396, 32 / 8 heads of 128 143 / 119; 64 x 2001 keys
// and 512 behind 4000 145 / 121, of 64 99 / 80, 64 query heads per KV head 232 / 218; 64 x 2001 keys and four prompts of 512 128 / 110; 128 x 4001 keys and 100 334 / 331.)
constexpr float PA_FEW_PIECE = 3.f, PA_WIDE_PIECE = 5.f;                // beside the tiles of a row tile
constexpr float PA_FEW_32_ROWS = 2.f, PA_FEW_64_ROWS = 3.5f;           // a tile of as many rows
constexpr float PA_WIDE_TILE_64 = 4.5f, PA_WIDE_TILE_128 = 5.5f;        // a tile of the second launch: 256 rows, as many keys as elements
__device__ __forceinline__ void pa_load(const PagedAttnParams& p, const PagedSequence& s, int head_dim, long long& few, long long& wide) {
  if (s.bad || s.fresh == 0) return;
  const int rows = s.fresh * p.group;
  const float keys = s.past + 0.5f * s.fresh, seen = p.window ? fminf(keys, p.window) : keys;  // of a row in the middle
  if (rows <= p.few_high)
    few += llrintf(p.kv_heads * (seen / 64.f + PA_FEW_PIECE) * (p.few_high > 32 ? PA_FEW_64_ROWS : p.few_high > 16 ? PA_FEW_32_ROWS : 1.f));
  else
    wide += llrintf(p.kv_heads * float((rows + 255) / 256) * (seen / head_dim + PA_WIDE_PIECE) * (head_dim == 64 ? PA_WIDE_TILE_64 : PA_WIDE_TILE_128));
}
// SMs of the first launch.  The smaller part is rounded up, and then by half an SM more: one too few would weigh most there.
__device__ __forceinline__ int pa_few_sms(long long few, long long wide, int sms) {
  if (few == 0) return 0;
  if (wide == 0) return sms;
  const float want = float(sms) * float(few) / float(few + wide);
  return max(1, min(sms - 1, int(2.f * want < sms ? ceilf(want + 0.5f) : floorf(want - 0.5f))));
}

// Number of the sequence and its place on the line of costs at which a range begins.
template <int THREADS>
struct RangeSearch {
  long long scan[THREADS / 32];
  long long load[2][THREADS / 32];
  long long begin;
  int seq;
};
// The sums of two numbers over THREADS threads.
template <int THREADS, typename Meet>
__device__ __forceinline__ void sum_loads(RangeSearch<THREADS>& at, int thread, Meet meet, long long& a, long long& b) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, d);
    b += __shfl_xor_sync(0xffffffffu, b, d);
  }
  if ((thread & 31) == 0) at.load[0][thread >> 5] = a, at.load[1][thread >> 5] = b;
  meet();
  a = b = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) a += at.load[0][w], b += at.load[1][w];
}
// The equal share [from, to) that is number `block` of `blocks_of()`, of the line on which all sequences' costs lie one behind the other; `at` receives where it
// begins.  Called by THREADS threads, which meet in `meet`; blocks_of is asked after cost_of has been for every sequence.
template <int THREADS, typename Cost, typename Blocks, typename Meet>
__device__ __forceinline__ void share_out(int n, int least, int thread, int block, RangeSearch<THREADS>& at, Cost cost_of, Blocks blocks_of, Meet meet, long long& share,
                                          long long& from, long long& to) {
  const int warp = thread >> 5, lane = thread & 31;
  auto scan = [&](long long v, long long& before, long long& total) {
    long long inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    meet();
    if (lane == 31) at.scan[warp] = inc;
    meet();
    before = inc - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += at.scan[w];
      total += at.scan[w];
    }
  };
  if (thread == 0) {
    at.seq = n;
    at.begin = 0;
  }
  long long all = 0, mine_before = 0, mine = 0;
  for (int base = 0; base < n; base += THREADS) {
    const int s = base + thread;
    long long before, total;
    mine = s < n ? cost_of(s) : 0;
    scan(mine, before, total);
    mine_before = all + before;
    all += total;
  }
  // (64-bit divisions are long)
  const unsigned blocks = blocks_of();
  share = max((long long)least, all < INT_MAX / 2 ? (long long)((unsigned(all) + blocks - 1) / blocks) : (all + blocks - 1) / blocks);
  from = min(all, share * block);
  to = min(all, from + share);
  if (n <= THREADS) {
    if (mine > 0 && from >= mine_before && from < mine_before + mine) {
      at.seq = thread;
      at.begin = mine_before;
    }
  } else {
    long long so_far = 0;
    for (int base = 0; base < n && so_far <= from; base += THREADS) {
      const int s = base + thread;
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
  meet();
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

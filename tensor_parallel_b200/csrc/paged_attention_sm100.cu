// Attention of new tokens over a paged cache for sequences with many query rows (chunks of prompts, whole prompts), on tcgen05 tensor cores.
//
// Bound by the tensor cores and the softmax between their two products, as the dense kernel (attention_sm100.cu), whose two query tiles per CTA it has:
// while the softmax warps of one tile of 128 rows work, the tensor cores multiply for the other.  The rows of a tile are (token, query head) pairs
// of one KV head, heads fastest, so that the heads of a group read their keys once and short chunks fill their tiles.  What differs:
//
//   work      : (sequence, row tile of 256, KV head, tile of keys) on one line, cut into equal ranges of the resident CTAs (share_out); what is cut goes by the
//               workspace and the joining kernel.  Ranges balance ragged and causal work, and split long contexts with few rows.
//   warp 3    : walks the range and announces its pieces in a ring of four (64-bit divisions and lengths from memory: 2 us each in front of the loads)
//   warp 0    : keys and values by TMA boxes of a page, table entries 32 at a time and 32 ahead
//   warp 1    : issues the MMAs, and writes zeros over values of no key in reach
//   warp 2    : query rows, into the room of rows whose last scores are done: a TMA box of (64 elements, the heads of a group, tokens) where 128 rows are
//               whole tokens, else (7, 12 or 71 heads to a group; rows that repeat) by cp.async.  (Fetched by the softmax warps themselves they were 3 us of theirs per piece)
//   warps 4-11: softmax, as there; results leave through shared memory in whole lines
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "launch.cuh"
#include "paged_attention.cuh"

namespace tpb {

constexpr int PW_M = 128;
constexpr int PW_THREADS = 384;
// In tiles: a piece's fill, drain and result (whole calls at 1 / 2 / 3 / 5, in us: the prompts of 16.4 k tokens, 32 heads of 128 474 / 445 / 456 / 476, 16 x 1000, 32 / 8
// heads 315 / 275 / 296 / 301, 8 x 2048, 32 heads of 64 319 / 317 / 303 / 305).
template <int N>
__device__ __forceinline__ constexpr int piece_cost() { return N == 64 ? 3 : 2; }
constexpr int PW_MIN_SHARE = 6;   // a piece and four tiles
constexpr float PW_RESCALE_LOG2 = 8.f;  // (see attention_sm100.cu: beyond the first 128 keys of a piece, the maximum follows large rises only)
constexpr int PW_EXACT_KEYS = 128;
constexpr int PW_PIECES = 4;  // announced at a time
constexpr int PW_LOST = 8;    // (the loads are three pieces ahead of the results at most: two stages of one tile each)

// D and keys per tile: 128 x 128, one CTA per SM; 64 x 64, two.
template <int D, int N>
struct Wide {
  static constexpr int CTAS = N == 64 ? 2 : 1;
  static constexpr int W = N == 64 ? 16 : 32;  // columns per TMEM access beside a row of scores in registers
  static constexpr int REGS_OTHER = N == 64 ? 32 : 56, REGS_SOFTMAX = N == 64 ? 104 : 224;
  static constexpr int DB = D / 64;
  static constexpr int Q_BYTES = DB * PW_M * 128, T_BYTES = DB * N * 128;
  static constexpr int STAGE_BYTES = 4096;  // of a softmax warp: 32 rows of 128 bytes on their way to memory
  static constexpr int SMEM = 1024 + 2 * Q_BYTES + 4 * T_BYTES + 8 * STAGE_BYTES + 1024;
  static_assert(4 * 32 * REGS_OTHER + 8 * 32 * REGS_SOFTMAX <= (N == 64 ? 80 : 168) * PW_THREADS, "registers of a CTA at its launch");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory of an SM");
};

struct WidePiece {
  int token0, row0, rows, past, total, low, kvh, slot;
  int seq;
  int tile0, n[2];  // first tile of keys, and how many each query tile takes of them; n both 0: no further piece
};

// Of a row tile: its first and last tile of keys, and the first key that its first row sees.
template <int N>
__device__ __forceinline__ void wide_span(const PagedAttnParams& p, const PagedSequence& s, int rows, int rt, int& first, int& end, int& low) {
  const int row0 = rt * PW_ROWS;
  low = p.window ? max(0, s.past + row0 / p.group - p.window + 1) : 0;
  first = low / N;
  end = (s.past + (min(rows, row0 + PW_ROWS) - 1) / p.group) / N + 1;
}

__device__ __forceinline__ void tm_load(uint32_t at, uint32_t (&r)[16]) { tmem_ld_x16(at, r); }
__device__ __forceinline__ void tm_load(uint32_t at, uint32_t (&r)[32]) { tmem_ld_x32(at, r); }
__device__ __forceinline__ void tm_store(uint32_t at, const uint32_t (&r)[16]) { tmem_st_x16(at, r); }
__device__ __forceinline__ void tm_store(uint32_t at, const uint32_t (&r)[32]) { tmem_st_x32(at, r); }

// From shared memory: rows of 128 bytes, swizzled.
__device__ __forceinline__ void tma_store_3d(const void* tmap, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n\tcp.async.bulk.commit_group;"
               ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int D, int N>
__global__ void __launch_bounds__(PW_THREADS, Wide<D, N>::CTAS)
paged_attn_wide_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                       const __grid_constant__ CUtensorMap tmap_o, const PagedAttnParams p, const int boxed, const int boxed_out, const int ahead) {
  using C = Wide<D, N>;
  constexpr int DB = C::DB, W = C::W;
  constexpr uint32_t Q_BYTES = C::Q_BYTES, T_BYTES = C::T_BYTES;
  constexpr uint32_t TMEM_COLS = 512 / C::CTAS, O_COL0 = 2 * N;
  static_assert(O_COL0 + 2 * D <= TMEM_COLS, "tensor memory columns");
  constexpr uint32_t IDESC_QK = make_idesc_bf16(PW_M, N, false, false);
  constexpr uint32_t IDESC_PV = make_idesc_bf16(PW_M, D, false, true);

  extern __shared__ uint8_t pw_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pw_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                 // [2 tiles]
  uint8_t* k_s = q_s + 2 * Q_BYTES;    // [2 stages]
  uint8_t* v_s = k_s + 2 * T_BYTES;    // [2 stages]
  uint8_t* out_s = v_s + 2 * T_BYTES;  // [8 softmax warps]
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_s + 8 * C::STAGE_BYTES);
  uint64_t* q_full = bars;             // [2 tiles]
  uint64_t* k_full = bars + 2;         // [2 stages]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 8;
  uint64_t* s_full = bars + 10;        // [2 tiles]
  uint64_t* p_full = bars + 12;
  uint64_t* o_full = bars + 14;
  uint64_t* q_empty = bars + 16;
  uint64_t* piece_full = bars + 18;    // [PW_PIECES]
  uint64_t* piece_empty = bars + 18 + PW_PIECES;
  WidePiece* pieces = reinterpret_cast<WidePiece*>(bars + 18 + 2 * PW_PIECES);  // [PW_PIECES]
  // [PW_LOST] (number (from 1) of a piece of which a page is not there) << 32 | its first tile with such a page.  A query tile that ends in front of that tile of keys
  // may look while the producer writes: in one word, which it finds wrong either way
  unsigned long long* lost = reinterpret_cast<unsigned long long*>(pieces + PW_PIECES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(lost + PW_LOST);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  __shared__ RangeSearch<PW_THREADS> range;
  __shared__ int any_bad;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    if (boxed) prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);  // one arrival per softmax warp of the tile
      mbar_init(&o_full[s], 1);
    }
    for (int s = 0; s < PW_PIECES; ++s) {
      mbar_init(&piece_full[s], 1);
      mbar_init(&piece_empty[s], 11);  // warps 0 to 2, softmax warps
    }
    for (int s = 0; s < PW_LOST; ++s) lost[s] = 0;
    *abort_flag = 0;
    any_bad = 0;
    fence_mbar_init();
  }
  __syncthreads();
  // beside the launch for few rows, which has waited for what is in front of it, before this one was let in: its end is awaited at this one's
  if (!ahead) pa_wait_prior();
  if (threadIdx.x < 2) p.parts.joins[2 * blockIdx.x + threadIdx.x] = make_int4(-1, 0, 0, 0);
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  __syncthreads();
  pa_launch_next();  // (not before this CTA has its tensor memory: whoever comes next may want some while it waits)
  auto units_of = [&](int i, PagedSequence& s, int& rows) {  // row tiles of a sequence that is this launch's
    s = paged_sequence(p.b, i);
    rows = s.fresh * p.group;
    return s.bad || rows < p.rows_low || rows > p.rows_high ? 0 : (rows + PW_ROWS - 1) / PW_ROWS;
  };
  long long share, w0, w1;
  long long few = 0, wide = 0;
  auto meet = [&]() { __syncthreads(); };
  share_out<PW_THREADS>(p.b.n, PW_MIN_SHARE, threadIdx.x, blockIdx.x, range, [&](int i) {
    PagedSequence s;
    int rows, first, end, low;
    const int row_tiles = units_of(i, s, rows);
    if (p.split_sms) pa_load(p, s, D, few, wide);
    if (s.bad && p.takes_bad) {
      any_bad = 1;
      if (blockIdx.x == 0) atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
    }
    long long cost = 0;
    for (int rt = 0; rt < row_tiles; ++rt) {
      wide_span<N>(p, s, rows, rt, first, end, low);
      cost += end - first + piece_cost<N>();
    }
    return cost * p.kv_heads;
  }, [&]() {
    if (!p.split_sms) return gridDim.x;
    sum_loads<PW_THREADS>(range, threadIdx.x, meet, few, wide);
    return unsigned(max(1, p.split_sms - pa_few_sms(few, wide, p.split_sms)) * C::CTAS);
  }, meet, share, w0, w1);
  if (any_bad)
    for (int i = 0; i < p.b.n; ++i) {
      const PagedSequence s = paged_sequence(p.b, i);
      if (s.bad) fill_rows<D, PW_THREADS>(p, s.token0, s.fresh, 0x7fc07fc0u);
    }
  if (p.fill_rest) fill_around<D, PW_THREADS>(p);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  auto give_up = [&](uint32_t code) {
    atomicMax(p.b.status, code);
    *abort_flag = 1;
  };
  // (of a whole warp)
  auto wait_all = [&](uint64_t* bar, uint32_t parity) {
    const bool there = __all_sync(0xffffffffu, !*abort_flag && mbar_wait(bar, parity));
    if (!there && lane == 0 && !*abort_flag) give_up(STATUS_TIMEOUT_MBAR);
    return there;
  };

  if (warp < 4) {
    setmaxnreg_dec<C::REGS_OTHER>();
    if (warp == 3) {
      // ---------------- planner: the pieces of the range, up to PW_PIECES ahead ----------------
      int seq = range.seq, rt = 0;
      long long at = w0, unit_begin = range.begin;  // of the row tile rt of sequence seq
      bool more = true;
      for (int i = 0; more; ++i) {
        WidePiece o = {};
        while (at < w1 && seq < p.b.n) {
          PagedSequence s;
          int rows, first, end, low;
          if (rt >= units_of(seq, s, rows)) {
            ++seq;
            rt = 0;
            continue;
          }
          wide_span<N>(p, s, rows, rt, first, end, low);
          const int length = end - first + piece_cost<N>();
          if (at >= unit_begin + (long long)length * p.kv_heads) {
            unit_begin += (long long)length * p.kv_heads;
            ++rt;
            continue;
          }
          const int into = int(at - unit_begin), kvh = into / length, from = into % length, to = int(min((long long)length, from + (w1 - at)));
          const int t0 = max(0, from - piece_cost<N>()), t1 = max(0, to - piece_cost<N>());
          const long long unit_end = unit_begin + (long long)(kvh + 1) * length;
          at += to - from;
          if (t0 == t1) continue;
          o.seq = seq, o.token0 = s.token0, o.row0 = rt * PW_ROWS, o.rows = min(PW_ROWS, rows - o.row0), o.past = s.past, o.total = s.past + s.fresh, o.low = low;
          o.kvh = kvh, o.tile0 = first + t0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int last = min(o.rows, (t + 1) * PW_M) - 1;  // row of the piece
            o.n[t] = last < t * PW_M ? 0 : max(0, min(first + t1, (s.past + (o.row0 + last) / p.group) / N + 1) - o.tile0);
          }
          o.slot = t0 == 0 && t1 == end - first ? -1 : 2 * int(blockIdx.x) + (t0 == 0 ? 1 : 0);
          if (t0 == 0 && o.slot >= 0 && lane == 0) {
            p.parts.joins[2 * blockIdx.x] = make_int4(o.token0, o.row0, o.rows, kvh);
            p.parts.joins[2 * blockIdx.x + 1] = make_int4(int((unit_end - 1) / share), 0, 0, 0);
          }
          break;
        }
        more = max(o.n[0], o.n[1]) > 0;
        if (!wait_all(&piece_empty[i % PW_PIECES], ((i / PW_PIECES) & 1) ^ 1)) break;
        if (lane == 0) {
          pieces[i % PW_PIECES] = o;
          mbar_arrive(&piece_full[i % PW_PIECES]);
        }
        __syncwarp();
      }
    } else if (warp == 0) {
      // ---------------- producer ----------------
      const int page_size = 1 << p.b.page_shift;
      const int per_tile = max(1, N >> p.b.page_shift), box_rows = min(page_size, N);
      const int my_page = lane / DB, my_block = lane % DB;
      int kt = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        ok = wait_all(&piece_full[i % PW_PIECES], (i / PW_PIECES) & 1);
        if (!ok) break;
        const WidePiece& pc = pieces[i % PW_PIECES];
        const int n = max(pc.n[0], pc.n[1]), tile0 = pc.tile0, total = pc.total, low = pc.low, kvh = pc.kvh;
        const int* row = p.b.table + (long long)pc.seq * p.b.table_ld;
        __syncwarp();
        if (lane == 0) mbar_arrive(&piece_empty[i % PW_PIECES]);
        if (n == 0) break;
        const int entries = ((total - 1) >> p.b.page_shift) + 1;
        int entry0 = tile0 * N >> p.b.page_shift;
        auto fetch = [&](int e) { return e < entries ? __ldg(row + e) : -1; };
        int now = fetch(entry0 + lane), next = fetch(entry0 + 32 + lane);
        for (int j = 0; ok && j < n; ++j, ++kt) {
          const int s = kt & 1, key0 = (tile0 + j) * N;
          const uint32_t par = ((kt >> 1) & 1) ^ 1;
          int e = (key0 >> p.b.page_shift) - entry0;
          if (e >= 32) {
            entry0 += 32;
            e -= 32;
            now = next;
            next = fetch(entry0 + 32 + lane);
          }
          const int page = __shfl_sync(0xffffffffu, now, (e + my_page) & 31);
          const int first = key0 + my_page * page_size;
          const bool wanted = lane < per_tile * DB && (per_tile == 1 || (first < total && first + page_size > low));
          const bool good = wanted && page >= 0 && page < p.b.pages;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, good)) * box_rows * 128;
          if (__any_sync(0xffffffffu, wanted && !good) && lane == 0) {
            atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
            volatile unsigned long long* record = lost + i % PW_LOST;
            if (int(*record >> 32) != i + 1) *record = static_cast<unsigned long long>(i + 1) << 32 | unsigned(j);
          }
          const uint32_t to = my_block * (N * 128) + my_page * box_rows * 128;
          const int slot = per_tile == 1 ? key0 & (page_size - 1) : 0;
          ok = wait_all(&k_empty[s], par);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&k_full[s], bytes);
          __syncwarp();
          if (good) tma_load_4d(k_s + s * T_BYTES + to, &tmap_k, &k_full[s], my_block * 64, slot, kvh, page);
          ok = wait_all(&v_empty[s], par);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&v_full[s], bytes);
          __syncwarp();
          if (good) tma_load_4d(v_s + s * T_BYTES + to, &tmap_v, &v_full[s], my_block * 64, slot, kvh, page);
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer (the warp stays together, one lane issues: see umma_bf16_lead) ----------------
      const uint32_t leader = elect_one();
      const uint32_t q_lo = desc_kmajor_lo(smem_u32(q_s));
      auto issue_qk = [&](int t, int kt) {  // S_t = Q_t K^T
        const uint32_t k_lo = desc_kmajor_lo(smem_u32(k_s + (kt & 1) * T_BYTES));
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_bf16_lead(leader, tmem_base + t * N, q_lo + (t * Q_BYTES + d * (PW_M * 128)) / 16 + kk * 2, k_lo + d * (N * 128 / 16) + kk * 2, IDESC_QK,
                           (d | kk) ? 1u : 0u);
        umma_commit_lead(leader, &s_full[t]);
      };
      auto issue_pv = [&](int t, int kt, int j) {  // O_t (+)= P_t V
        const uint32_t v_lo = desc_mnmajor_lo(smem_u32(v_s + (kt & 1) * T_BYTES), N * 128);
#pragma unroll
        for (int kk = 0; kk < N / 16; ++kk)
          umma_bf16_tmem_a_lead(leader, tmem_base + O_COL0 + t * D, tmem_base + t * N + kk * 8, v_lo + kk * (16 * 128 / 16), IDESC_PV, (j | kk) ? 1u : 0u);
      };
      auto arrived = [&](uint64_t* bar, uint32_t parity) {
        const bool there = wait_all(bar, parity);
        tc_fence_after();
        return there;
      };
      int kt = 0, q_count[2] = {0, 0}, p_count[2] = {0, 0};
      bool ok = true;
      for (int i = 0; ok; ++i) {
        ok = arrived(&piece_full[i % PW_PIECES], (i / PW_PIECES) & 1);
        if (!ok) break;
        const WidePiece pc = pieces[i % PW_PIECES];
        __syncwarp();
        if (lane == 0) mbar_arrive(&piece_empty[i % PW_PIECES]);
        const int n = max(pc.n[0], pc.n[1]);
        if (n == 0) break;
        ok = arrived(&k_full[kt & 1], (kt >> 1) & 1);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && pc.n[t] > 0) {
            ok = arrived(&q_full[t], q_count[t]++ & 1);
            if (ok) {
              issue_qk(t, kt);
              if (pc.n[t] == 1) umma_commit_lead(leader, &q_empty[t]);
            }
          }
        if (!ok) break;
        umma_commit_lead(leader, &k_empty[kt & 1]);
        for (int j = 0; ok && j < n; ++j, ++kt) {
          const bool next = j + 1 < n;
          const int key0 = (pc.tile0 + j) * N;
          if (next) ok = arrived(&k_full[(kt + 1) & 1], ((kt + 1) >> 1) & 1);
          ok = ok && arrived(&v_full[kt & 1], (kt >> 1) & 1);
          if (!ok) break;
          if (key0 < pc.low || key0 + N > pc.total) {
            // slots of no key in reach (the end of the last page, in front of the window): zeros, since a probability of zero times a NaN is not zero
            const int before = max(0, pc.low - key0), from = min(N, pc.total - key0), gone = before + N - from;
            for (int c = lane; c < gone * DB * 8; c += 32) {
              const int r = c / (DB * 8), e = c % (DB * 8), at = r < before ? r : from + r - before;
              *reinterpret_cast<uint4*>(v_s + (kt & 1) * T_BYTES + (e >> 3) * (N * 128) + at * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (ok && j < pc.n[t]) {
              ok = arrived(&p_full[t], p_count[t]++ & 1);
              if (ok) {
                issue_pv(t, kt, j);
                if (j == pc.n[t] - 1)
                  umma_commit_lead(leader, &o_full[t]);
                else
                  issue_qk(t, kt + 1);
                if (j == pc.n[t] - 2) umma_commit_lead(leader, &q_empty[t]);  // (those were its last scores)
              }
            }
          if (!ok) break;
          umma_commit_lead(leader, &v_empty[kt & 1]);                 // the values may be overwritten once these MMAs retire
          if (next) umma_commit_lead(leader, &k_empty[(kt + 1) & 1]);  // and the next keys
        }
      }
    } else if (warp == 2) {
      // ---------------- query rows of the next piece, as soon as the last scores of this one are done ----------------
      int count[2] = {0, 0};
      bool ok = true;
      for (int i = 0; ok; ++i) {
        ok = wait_all(&piece_full[i % PW_PIECES], (i / PW_PIECES) & 1);
        if (!ok) break;
        const WidePiece& in_ring = pieces[i % PW_PIECES];
        const int token0 = in_ring.token0, row0 = in_ring.row0, rows = in_ring.rows, kvh = in_ring.kvh, n[2] = {in_ring.n[0], in_ring.n[1]};
        __syncwarp();
        if (lane == 0) mbar_arrive(&piece_empty[i % PW_PIECES]);
        if (max(n[0], n[1]) == 0) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || n[t] == 0) continue;
          ok = wait_all(&q_empty[t], (count[t]++ & 1) ^ 1);
          if (!ok) continue;
          if (boxed) {  // (rows of a box: the heads of a group, tokens)
            if (lane == 0) {
              mbar_expect_tx(&q_full[t], Q_BYTES);
#pragma unroll
              for (int d = 0; d < DB; ++d)
                tma_load_3d(q_s + t * Q_BYTES + d * (PW_M * 128), &tmap_q, &q_full[t], d * 64, kvh * p.group, token0 + (row0 + t * PW_M) / p.group);
            }
            __syncwarp();
            continue;
          }
          constexpr int STEP = 32 / (D / 8);  // rows at a time
          const int e = lane % (D / 8), r0 = lane / (D / 8);
          const int step_tokens = STEP / p.group, step_heads = STEP % p.group;
          int token = (row0 + t * PW_M + r0) / p.group, head = (row0 + t * PW_M + r0) % p.group;
          const bf16* base = p.q + (long long)token0 * p.q_st + (long long)kvh * p.group * p.q_sh + e * 8;
          const uint32_t to = smem_u32(q_s + t * Q_BYTES + (e >> 3) * (PW_M * 128));
#pragma unroll 4
          for (int r = r0; r < PW_M; r += STEP) {
            if (t * PW_M + r < rows) cp_async16(to + r * 128 + (((e & 7) ^ (r & 7)) << 4), base + token * p.q_st + head * p.q_sh, 16);  // (other rows' results go nowhere)
            token += step_tokens;
            head += step_heads;
            if (head >= p.group) {
              head -= p.group;
              ++token;
            }
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[t]);
        }
      }
    }
  } else {
    // ---------------- softmax warps ----------------
    setmaxnreg_inc<C::REGS_SOFTMAX>();
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;  // TMEM lane quarter this warp may access
    const int row = quarter * 32 + lane;
    const uint32_t s_addr = tmem_base + (uint32_t(quarter * 32) << 16) + t * N;  // scores, and in their first half the probabilities
    const uint32_t o_addr = tmem_base + (uint32_t(quarter * 32) << 16) + O_COL0 + t * D;
    int s_count = 0, o_count = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      ok = wait_all(&piece_full[i % PW_PIECES], (i / PW_PIECES) & 1);
      if (!ok) break;
      const WidePiece pc = pieces[i % PW_PIECES];
      if (max(pc.n[0], pc.n[1]) == 0) break;
      const int n = pc.n[t];
      const int here = pc.row0 + t * PW_M + row;  // row of the sequence
      const int pos = pc.past + here / p.group;
      const int least_pos = pc.past + (pc.row0 + t * PW_M) / p.group, most_pos = pc.past + (pc.row0 + t * PW_M + PW_M - 1) / p.group;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < n; ++j) {
        const int key0 = (pc.tile0 + j) * N;
        const int visible = pos + 1 - key0, hidden = p.window ? pos - p.window + 1 - key0 : 0;  // keys [hidden, visible) of this tile count
        const bool plain = key0 + N - 1 <= least_pos && (!p.window || key0 > most_pos - p.window);
        ok = wait_all(&s_full[t], s_count++ & 1);
        if (!ok) break;
        tc_fence_after();
        uint32_t r[N];
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < N; c += 32) tmem_ld_x32(s_addr + c, *reinterpret_cast<uint32_t(*)[32]>(r + c));
        tmem_ld_wait();
        if (!plain) {
#pragma unroll
          for (int c = 0; c < N; c += 32) {
            // a bit for each of 32 keys: below `visible`, from `hidden` on
            const int up = min(max(visible - c, 0), 32), down = min(max(hidden - c, 0), 32);
            const uint32_t seen = (up == 32 ? 0xffffffffu : (1u << up) - 1u) & (down == 32 ? 0u : 0xffffffffu << down);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!(seen >> x & 1u)) r[c + x] = 0xff800000u;
          }
        }
#pragma unroll
        for (int c = 0; c < N; c += 4) {
          m0 = fmax3_nan(m0, __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
          m1 = fmax3_nan(m1, __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
        }
        // (the scale is positive: the maximum commutes with it.  A score that is NaN makes the maximum NaN, and with it all that follows of the row: the
        // exponentials on the FMA pipe would drop it)
        const float m_tile = fmax3_nan(m0, m1, m1) * p.scale_log2e;
        float factor = 1.f;
        bool rescale = false;
        if (m_run == -INFINITY) {
          m_run = m_tile;  // nothing accumulated for this row yet
          factor = 0.f;    // (but 2^-140 in the sum for some keys of a tile in which it saw none)
          rescale = j > 0;
        } else if (m_run == m_run && !(m_tile <= m_run + (j * N < PW_EXACT_KEYS ? 0.f : PW_RESCALE_LOG2))) {  // (a row that is NaN stays it, and calls for no more rescaling)
          factor = ex2_approx(m_run - m_tile);
          m_run = m_tile;
          rescale = true;
        }
        if (j > 0 && __any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int c = 0; c < D; c += W) {  // (rolled, as the result below: code that is not in the instruction cache costs more than its instructions)
            uint32_t o[W];
            tm_load(o_addr + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < W; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
            tm_store(o_addr + c, o);
          }
        }
        l_run *= factor;
        const float nbase = m_run == -INFINITY ? 0.f : -m_run;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int c = 0; c < N / 2; c += W) {
          // The sum is of the probabilities in 32 bits.  That of the rounded ones, as the few-row kernel has it, cancels part of their error where few keys have most of a row, but
          // up to 128 keys the heaviest one has the probability 1, which is not rounded (the maximum is exact there), and behind them ordinary rows gain little (error of
          // 512 keys 2.25e-3 -> 2.20e-3, of one key with most of the row 2.1e-3 -> 1.8e-3) for 3 to 8 % of the time (prompts of 16.4 k tokens 435 -> 470 us).
          uint32_t packed[W];
#pragma unroll
          for (int x = 0; x < W; ++x) {
            float t0, t1;
            ffma2(t0, t1, __uint_as_float(r[2 * (c + x)]), __uint_as_float(r[2 * (c + x) + 1]), p.scale_log2e, p.scale_log2e, nbase, nbase);
            float p0, p1;
            if ((x & 3) == 0) {  // (a quarter of the exponentials on the FMA pipe)
              ex2_poly2(t0, t1, EX2_NOTHING);  // (2^-126 of a value that a row does not see yet is not nothing: values go up to 2^128)
              p0 = t0;
              p1 = t1;
            } else {
              p0 = ex2_approx(t0);
              p1 = ex2_approx(t1);
            }
            fadd2(sum0, sum1, sum0, sum1, p0, p1);
            packed[x] = pack_bf16x2(p0, p1);
          }
          tm_store(s_addr + c, packed);
        }
        l_run += sum0 + sum1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      // ---- the result, or this piece of it ----
      if (n > 0) {
        ok = wait_all(&o_full[t], o_count++ & 1);
        if (!ok) break;
        tc_fence_after();
      }
      const unsigned long long gone = *reinterpret_cast<volatile unsigned long long*>(lost + i % PW_LOST);
      const bool poisoned = int(gone >> 32) == i + 1 && int(unsigned(gone)) < n;
      if (m_run == -INFINITY) l_run = 0.f;
      if (poisoned || !(m_run < INFINITY)) l_run = __uint_as_float(0x7fc00000u);  // (scores that are NaN or infinite)
      const int left = pc.rows - t * PW_M - quarter * 32;  // of this warp's rows
      uint8_t* stage = out_s + (warp - 4) * C::STAGE_BYTES;
      if (lane == 0) tma_stores_read();  // (of the piece in front)
      __syncwarp();
      if (boxed_out && left >= 32 && n > 0 && pc.slot < 0) {
        // whole tokens: 64 elements of 32 rows at a time by a box of their own (by loads and stores, as below, a piece's results hold both of its tiles up for 2.9 us:
        // us without / with boxes, 64 prompts of 256 tokens, 32 heads of 128 155 / 135, 16 of 1000, 32 / 8 heads 227 / 217, of 16.4 k tokens 453 / 441)
        const float inv = 1.f / l_run;  // (a row sees its own key at least: a sum of zero is of scores that are all -inf, and its result NaN)
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
          uint32_t o[64];
#pragma unroll
          for (int w0 = 0; w0 < 64; w0 += W) tm_load(o_addr + c + w0, *reinterpret_cast<uint32_t(*)[W]>(o + w0));
          tmem_ld_wait();
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = pack_bf16x2(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv);
          if (c) {
            if (lane == 0) tma_stores_read();
            __syncwarp();
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(stage + lane * 128 + ((x ^ (lane & 7)) << 4)) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_3d(&tmap_o, stage, c, pc.kvh * p.group, pc.token0 + (pc.row0 + t * PW_M + quarter * 32) / p.group);
        }
      } else if (left > 0) {
        // through shared memory, 128 bytes of each row at a time in swizzled chunks of 16: a thread has a row, and eight threads store a line of one
        const bool whole = pc.slot < 0;
        const float inv = whole ? 1.f / l_run : 1.f;
        if (!whole && lane < left) p.parts.ml[(long long)pc.slot * PW_ROWS + t * PW_M + quarter * 32 + lane] = make_float2(poisoned ? 0.f : m_run, l_run);
        const int step_tokens = 4 / p.group, step_heads = 4 % p.group;
        const int first_token = (pc.row0 + t * PW_M + quarter * 32 + (lane >> 3)) / p.group, first_head = (pc.row0 + t * PW_M + quarter * 32 + (lane >> 3)) % p.group;
        char* base = whole ? reinterpret_cast<char*>(p.out + (long long)pc.token0 * p.o_st + (long long)pc.kvh * p.group * p.o_sh)
                           : reinterpret_cast<char*>(p.parts.o + ((long long)pc.slot * PW_ROWS + t * PW_M + quarter * 32 + (lane >> 3)) * D);
        base += (lane & 7) * 16;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (n > 0) {
#pragma unroll
            for (int w0 = 0; w0 < 32; w0 += W) tm_load(o_addr + c + w0, *reinterpret_cast<uint32_t(*)[W]>(o + w0));
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0u;
          }
          const int k0 = whole ? (c >> 3) & 4 : 0;  // 32 columns are half of 128 bytes in bf16, all of them in fp32
          if (whole) {
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = pack_bf16x2(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (x < 4 || !whole)
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((k0 + x) ^ (lane & 7)) << 4)) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          if (whole && !(c & 32)) continue;
          __syncwarp();
          int token = first_token, head = first_head;
#pragma unroll 2
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
            char* to = whole ? base + (token * p.o_st + head * p.o_sh + (c & ~63)) * 2 : base + (i * 4 * D + c) * 4;
            if (r < left) *reinterpret_cast<uint4*>(to) = v;
            token += step_tokens;
            head += step_heads;
            if (head >= p.group) {
              head -= p.group;
              ++token;
            }
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[i % PW_PIECES]);
    }
    if (lane == 0) tma_stores_done();
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
  if (ahead) pa_wait_prior();  // (whoever waits for this launch waits for both)
}

template <int D, int N>
static int pw_go(const PagedAttnParams& p, const CUtensorMap& k, const CUtensorMap& v, int grid, bool ahead, cudaStream_t stream) {
  using C = Wide<D, N>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(paged_attn_wide_kernel<D, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return TPB_ERR_CUDA;
    ready[dev].store(true, std::memory_order_release);
  }
  // query rows by boxes: whole tokens in 128 rows, and strides that TMA takes
  CUtensorMap q = k;
  bool boxed = PW_M % p.group == 0 && (p.b.tokens == 1 || p.q_st > 0) && (p.heads == 1 || p.q_sh > 0);
  if (boxed) boxed = paged_rows_tmap(&q, p.q, D, p.heads, p.b.tokens, p.q_sh, p.q_st, p.group, PW_M / p.group) == TPB_OK;
  // and 32 rows of results
  CUtensorMap o = k;
  bool boxed_out = 32 % p.group == 0 && (p.b.tokens == 1 || p.o_st > 0) && (p.heads == 1 || p.o_sh > 0);
  if (boxed_out) boxed_out = paged_rows_tmap(&o, p.out, D, p.heads, p.b.tokens, p.o_sh, p.o_st, p.group, 32 / p.group) == TPB_OK;
  return launch_dependent(paged_attn_wide_kernel<D, N>, dim3(grid), dim3(PW_THREADS), C::SMEM, stream, true, q, k, v, o, p, int(boxed), int(boxed_out), int(ahead)) == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

int pw_tile(int head_dim) { return head_dim; }

int pw_grid(int head_dim) { return pa_sms() * (head_dim == 64 ? 2 : 1); }

int pw_launch(int head_dim, const PagedAttnParams& p, const CUtensorMap& k, const CUtensorMap& v, int grid, bool ahead, cudaStream_t stream) {
  return head_dim == 64 ? pw_go<64, 64>(p, k, v, grid, ahead, stream) : pw_go<128, 128>(p, k, v, grid, ahead, stream);
}

}  // namespace tpb

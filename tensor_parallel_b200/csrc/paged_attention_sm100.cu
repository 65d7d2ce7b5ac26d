// Attention of new tokens over a paged cache for sequences with many query rows (chunks of prompts, whole prompts), on tcgen05 tensor cores.
//
// Bound by the tensor cores and the softmax between their two products, as the dense kernel (attention_sm100.cu), whose two query tiles per CTA it has:
// while the softmax warps of one tile of 128 rows work, the tensor cores multiply for the other.  The rows of a tile are (token, query head) pairs
// of one KV head, heads fastest, so that the heads of a group read their keys once and short chunks fill their tiles.  What differs:
//
//   work      : (sequence, row tile of 256, KV head, tile of keys) on one line, cut into equal ranges of the resident CTAs (share_out); what is cut goes by the
//               workspace and the joining kernel.  Ranges balance ragged and causal work, and split long contexts with few rows.
//   warp 0    : walks the range, one piece ahead of its own loads; announces pieces in a ring of four; keys and values by TMA boxes of a page
//   warp 1    : issues the MMAs, and writes zeros over values of no key in reach
//   warps 4-11: softmax, as there; they fetch the rows of the next piece themselves (cp.async, into the room of rows whose last scores are done), so that any
//               strides and any number of heads in a group will do
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
constexpr int PW_PIECE_COST = 1;  // in tiles: a piece's fill, drain and result
constexpr int PW_MIN_SHARE = 5;   // a piece and four tiles
constexpr float PW_RESCALE_LOG2 = 8.f;  // (see attention_sm100.cu: beyond the first 128 keys of a piece, the maximum follows large rises only)
constexpr int PW_EXACT_KEYS = 128;
constexpr int PW_PIECES = 4;

// D and keys per tile: 128 x 128, one CTA per SM; 64 x 64, two.
template <int D, int N>
struct Wide {
  static constexpr int CTAS = N == 64 ? 2 : 1;
  static constexpr int W = N == 64 ? 16 : 32;  // columns per TMEM access beside a row of scores in registers
  static constexpr int REGS_OTHER = N == 64 ? 32 : 56, REGS_SOFTMAX = N == 64 ? 104 : 224;
  static constexpr int DB = D / 64;
  static constexpr int Q_BYTES = DB * PW_M * 128, T_BYTES = DB * N * 128;
  static constexpr int SMEM = 1024 + 2 * Q_BYTES + 4 * T_BYTES + 1024;
  static_assert(4 * 32 * REGS_OTHER + 8 * 32 * REGS_SOFTMAX <= (N == 64 ? 80 : 168) * PW_THREADS, "registers of a CTA at its launch");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory of an SM");
};

struct WidePiece {
  int token0, row0, rows, past, total, low, kvh, slot;
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

template <int D, int N>
__global__ void __launch_bounds__(PW_THREADS, Wide<D, N>::CTAS)
paged_attn_wide_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const PagedAttnParams p) {
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
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + 2 * T_BYTES);
  uint64_t* q_full = bars;             // [2 tiles]
  uint64_t* k_full = bars + 2;         // [2 stages]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 8;
  uint64_t* s_full = bars + 10;        // [2 tiles]
  uint64_t* p_full = bars + 12;
  uint64_t* o_full = bars + 14;
  uint64_t* piece_full = bars + 16;    // [PW_PIECES]
  uint64_t* piece_empty = bars + 16 + PW_PIECES;
  WidePiece* pieces = reinterpret_cast<WidePiece*>(bars + 16 + 2 * PW_PIECES);  // [PW_PIECES]
  int* lost = reinterpret_cast<int*>(pieces + PW_PIECES);                       // [PW_PIECES] number (from 1) of a piece of which a page is not there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(lost + PW_PIECES);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  __shared__ RangeSearch<PW_THREADS> range;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 4);  // one arrival per softmax warp of the tile
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_full[s], 1);
    }
    for (int s = 0; s < PW_PIECES; ++s) {
      mbar_init(&piece_full[s], 1);
      mbar_init(&piece_empty[s], 9);  // MMA warp, softmax warps
      lost[s] = 0;
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < 2) p.parts.joins[2 * blockIdx.x + threadIdx.x] = make_int4(-1, 0, 0, 0);
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  pa_launch_next();
  auto units_of = [&](int i, PagedSequence& s, int& rows) {  // row tiles of a sequence that is this launch's
    s = paged_sequence(p.b, i);
    rows = s.fresh * p.group;
    return s.bad || rows < p.rows_low || rows > p.rows_high ? 0 : (rows + PW_ROWS - 1) / PW_ROWS;
  };
  long long share, w0, w1;
  share_out<PW_THREADS>(p.b.n, PW_MIN_SHARE, range, [&](int i) {
    PagedSequence s;
    int rows, first, end, low;
    const int row_tiles = units_of(i, s, rows);
    if (s.bad && p.takes_bad && blockIdx.x == 0) atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
    long long cost = 0;
    for (int rt = 0; rt < row_tiles; ++rt) {
      wide_span<N>(p, s, rows, rt, first, end, low);
      cost += end - first + PW_PIECE_COST;
    }
    return cost * p.kv_heads;
  }, share, w0, w1);
  if (p.takes_bad)
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
    if (warp == 0) {
      // ---------------- producer ----------------
      const int page_size = 1 << p.b.page_shift;
      const int per_tile = max(1, N >> p.b.page_shift), box_rows = min(page_size, N);
      const int my_page = lane / DB, my_block = lane % DB;
      int seq = range.seq, rt = 0, announced = 0, kt = 0;
      long long at = w0, unit_begin = range.begin;  // of the row tile rt of sequence seq
      bool ok = true;
      // the next piece of the range into the ring; its sequence, for the table
      auto announce = [&]() {
        int of = 0;
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
          const int length = end - first + PW_PIECE_COST;
          if (at >= unit_begin + (long long)length * p.kv_heads) {
            unit_begin += (long long)length * p.kv_heads;
            ++rt;
            continue;
          }
          const int kvh = int((at - unit_begin) / length), from = int((at - unit_begin) % length), to = int(min((long long)length, from + (w1 - at)));
          const int t0 = max(0, from - PW_PIECE_COST), t1 = max(0, to - PW_PIECE_COST);
          const long long unit_end = unit_begin + (long long)(kvh + 1) * length;
          at += to - from;
          if (t0 == t1) continue;
          of = seq;
          o.token0 = s.token0, o.row0 = rt * PW_ROWS, o.rows = min(PW_ROWS, rows - o.row0), o.past = s.past, o.total = s.past + s.fresh, o.low = low, o.kvh = kvh;
          o.tile0 = first + t0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int last = min(o.rows, (t + 1) * PW_M) - 1;  // row of the piece
            o.n[t] = last < t * PW_M ? 0 : max(0, min(first + t1, (s.past + (o.row0 + last) / p.group) / N + 1) - o.tile0);
          }
          o.slot = t0 == 0 && t1 == end - first ? -1 : 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
          if (t0 == 0 && o.slot >= 0 && lane == 0) {
            p.parts.joins[2 * blockIdx.x] = make_int4(o.token0, o.row0, o.rows, kvh);
            p.parts.joins[2 * blockIdx.x + 1] = make_int4(int((unit_end - 1) / share), 0, 0, 0);
          }
          break;
        }
        const int slot = announced % PW_PIECES;
        ok = wait_all(&piece_empty[slot], ((announced / PW_PIECES) & 1) ^ 1);
        if (ok && lane == 0) {
          pieces[slot] = o;
          mbar_arrive(&piece_full[slot]);
        }
        __syncwarp();
        ++announced;
        return of;
      };
      int of = announce(), of_next = 0;
      for (int i = 0; ok; ++i) {
        const WidePiece pc = pieces[i % PW_PIECES];
        const int n = max(pc.n[0], pc.n[1]);
        if (n == 0) break;
        of_next = announce();  // (before this piece's loads: the softmax warps want to know)
        const int* row = p.b.table + (long long)of * p.b.table_ld;
        of = of_next;
        const int entries = ((pc.total - 1) >> p.b.page_shift) + 1;
        int entry0 = pc.tile0 * N >> p.b.page_shift;
        auto fetch = [&](int e) { return e < entries ? __ldg(row + e) : -1; };
        int now = fetch(entry0 + lane), next = fetch(entry0 + 32 + lane);
        for (int j = 0; ok && j < n; ++j, ++kt) {
          const int s = kt & 1, key0 = (pc.tile0 + j) * N;
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
          const bool wanted = lane < per_tile * DB && (per_tile == 1 || (first < pc.total && first + page_size > pc.low));
          const bool good = wanted && page >= 0 && page < p.b.pages;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, good)) * box_rows * 128;
          if (__any_sync(0xffffffffu, wanted && !good) && lane == 0) {
            atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
            lost[i % PW_PIECES] = i + 1;
          }
          const uint32_t to = my_block * (N * 128) + my_page * box_rows * 128;
          const int slot = per_tile == 1 ? key0 & (page_size - 1) : 0;
          ok = wait_all(&k_empty[s], par);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&k_full[s], bytes);
          __syncwarp();
          if (good) tma_load_4d(k_s + s * T_BYTES + to, &tmap_k, &k_full[s], my_block * 64, slot, pc.kvh, page);
          ok = wait_all(&v_empty[s], par);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&v_full[s], bytes);
          __syncwarp();
          if (good) tma_load_4d(v_s + s * T_BYTES + to, &tmap_v, &v_full[s], my_block * 64, slot, pc.kvh, page);
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
            if (ok) issue_qk(t, kt);
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
              }
            }
          if (!ok) break;
          umma_commit_lead(leader, &v_empty[kt & 1]);                 // the values may be overwritten once these MMAs retire
          if (next) umma_commit_lead(leader, &k_empty[(kt + 1) & 1]);  // and the next keys
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
    // this warp's 32 query rows of a piece on their way to shared memory
    auto fetch_rows = [&](const WidePiece& pc) {
#pragma unroll 4
      for (int c = lane; c < 32 * (D / 8); c += 32) {
        const int r = quarter * 32 + c / (D / 8), e = c % (D / 8), in = min(t * PW_M + r, pc.rows - 1);
        const int token = (pc.row0 + in) / p.group, head = (pc.row0 + in) % p.group;
        const bf16* src = p.q + (long long)(pc.token0 + token) * p.q_st + (long long)(pc.kvh * p.group + head) * p.q_sh + e * 8;
        cp_async16(smem_u32(q_s + t * Q_BYTES + (e >> 3) * (PW_M * 128) + r * 128 + (((e & 7) ^ (r & 7)) << 4)), src, 16);
      }
    };
    auto announce_rows = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    };
    int s_count = 0, o_count = 0;
    bool announced = false, ok = true;
    for (int i = 0; ok; ++i) {
      ok = wait_all(&piece_full[i % PW_PIECES], (i / PW_PIECES) & 1);
      if (!ok) break;
      const WidePiece pc = pieces[i % PW_PIECES];
      if (max(pc.n[0], pc.n[1]) == 0) break;
      const int n = pc.n[t];
      if (n > 0 && !announced) {
        fetch_rows(pc);
        announce_rows();
      }
      announced = false;
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
          for (int c = 0; c < N; ++c)
            if (c >= visible || c < hidden) r[c] = 0xff800000u;
        }
#pragma unroll
        for (int c = 0; c < N; c += 4) {
          m0 = fmax3(m0, __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
          m1 = fmax3(m1, __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
        }
        const float m_tile = fmaxf(m0, m1) * p.scale_log2e;  // (the scale is positive: the maximum commutes with it)
        float factor = 1.f;
        bool rescale = false;
        if (m_run == -INFINITY) {
          m_run = m_tile;  // nothing accumulated for this row yet
          factor = 0.f;    // (but 2^-126 for each key of a tile in which it saw none)
          rescale = j > 0;
        } else if (m_tile > m_run + (j * N < PW_EXACT_KEYS ? 0.f : PW_RESCALE_LOG2)) {
          factor = ex2_approx(m_run - m_tile);
          m_run = m_tile;
          rescale = true;
        }
        if (j > 0 && __any_sync(0xffffffffu, rescale)) {
#pragma unroll
          for (int c = 0; c < D; c += W) {
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
          uint32_t packed[W];
#pragma unroll
          for (int x = 0; x < W; ++x) {
            float t0, t1;
            ffma2(t0, t1, __uint_as_float(r[2 * (c + x)]), __uint_as_float(r[2 * (c + x) + 1]), p.scale_log2e, p.scale_log2e, nbase, nbase);
            float p0, p1;
            if ((x & 3) == 0) {  // (a quarter of the exponentials on the FMA pipe)
              ex2_poly2(t0, t1);
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
      // the rows of the next piece, in the room of this one's: their last scores are done
      const int ni = i + 1;
      if (__all_sync(0xffffffffu, mbar_try_wait(&piece_full[ni % PW_PIECES], (ni / PW_PIECES) & 1))) {
        const WidePiece& next = pieces[ni % PW_PIECES];
        if (next.n[t] > 0) {
          fetch_rows(next);
          announced = true;
        }
      }
      // ---- the result, or this piece of it ----
      if (n > 0) {
        ok = wait_all(&o_full[t], o_count++ & 1);
        if (!ok) break;
        tc_fence_after();
      }
      if (announced) announce_rows();  // (their scores may come while the results leave: the products with them wait for the probabilities)
      const bool poisoned = reinterpret_cast<volatile int*>(lost)[i % PW_PIECES] == i + 1;
      if (m_run == -INFINITY) l_run = 0.f;
      if (poisoned) l_run = __uint_as_float(0x7fc00000u);
      if (t * PW_M < pc.rows) {  // (warp-uniform: the loads from tensor memory are the whole warp's)
        const bool mine = t * PW_M + row < pc.rows;
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        const int token = here / p.group, head = here % p.group;
        bf16* to = p.out + (long long)(pc.token0 + token) * p.o_st + (long long)(pc.kvh * p.group + head) * p.o_sh;
        const bool sectors = (reinterpret_cast<uintptr_t>(to) & 31) == 0;  // (whole sectors leave at once)
        float* part = p.parts.o + ((long long)max(pc.slot, 0) * PW_ROWS + t * PW_M + row) * D;
#pragma unroll
        for (int c = 0; c < D; c += W) {
          uint32_t o[W];
          if (n > 0) {
            tm_load(o_addr + c, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int x = 0; x < W; ++x) o[x] = 0u;
          }
          if (mine && pc.slot >= 0) {
#pragma unroll
            for (int x = 0; x < W; x += 8) st_global_v8(part + c + x, o + x);
          } else if (mine && sectors) {
            uint32_t w[W / 2];
#pragma unroll
            for (int x = 0; x < W / 2; ++x) w[x] = pack_bf16x2(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv);
#pragma unroll
            for (int x = 0; x < W / 2; x += 8) st_global_v8(to + c + 2 * x, w + x);
          } else if (mine) {
#pragma unroll
            for (int x = 0; x < W; x += 8)
              *reinterpret_cast<uint4*>(to + c + x) =
                  make_uint4(pack_bf16x2(__uint_as_float(o[x]) * inv, __uint_as_float(o[x + 1]) * inv), pack_bf16x2(__uint_as_float(o[x + 2]) * inv, __uint_as_float(o[x + 3]) * inv),
                             pack_bf16x2(__uint_as_float(o[x + 4]) * inv, __uint_as_float(o[x + 5]) * inv), pack_bf16x2(__uint_as_float(o[x + 6]) * inv, __uint_as_float(o[x + 7]) * inv));
          }
        }
        if (mine && pc.slot >= 0) p.parts.ml[(long long)pc.slot * PW_ROWS + t * PW_M + row] = make_float2(poisoned ? 0.f : m_run, l_run);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[i % PW_PIECES]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
  pa_wait_prior();  // (launched ahead of the kernel in front: whoever waits for this one waits for both)
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
  return launch_dependent(paged_attn_wide_kernel<D, N>, dim3(grid), dim3(PW_THREADS), C::SMEM, stream, ahead, k, v, p) == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

int pw_tile(int head_dim) { return head_dim; }

int pw_grid(int head_dim) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms = 148;
  return sms * (head_dim == 64 ? 2 : 1);
}

int pw_launch(int head_dim, const PagedAttnParams& p, const CUtensorMap& k, const CUtensorMap& v, int grid, bool ahead, cudaStream_t stream) {
  return head_dim == 64 ? pw_go<64, 64>(p, k, v, grid, ahead, stream) : pw_go<128, 128>(p, k, v, grid, ahead, stream);
}

}  // namespace tpb

// Attention of new tokens over a paged cache, for sequences with few query rows (a new token or a few of them, times the query heads of a KV head).
//
//   o[t, h] = sum_j softmax_j(scale * q[t, h] . k[j]) v[j],   j in (p - window, p],   p = past + t the token's own position
//
// What bounds it is reading the pages once: 4 * head_dim bytes per key and KV head, and two products of 16 rows with each.  One launch deals with every
// sequence of the batch, whatever their lengths: the work (sequence, row tile, KV head, tile of 64 keys) lies on one line, cut into as many equal
// ranges as there are teams of warps (one to three in a CTA, a CTA per SM).  A range may begin and end inside a row tile's keys; such pieces leave unnormalised sums with their maximum in a workspace, and a
// second kernel, launched ahead, joins them in the order of the keys (no counters, no atomics: the result does not depend on timing, and calls on
// other streams or captured graphs share nothing).
//
// A team:
//   producer warp : walks the range; TMA boxes of up to 64 slots per page into a ring of stages (keys and values of 64 keys), up to 32 table entries
//                   fetched at a time and 32 ahead; query rows by cp.async into one of two buffers, so that the next piece's are there when its first keys are
//   compute warps : a warp holds 16 query rows and a part of the stage's keys (ROW_GROUPS x key groups): mma.sync m16n8k16 (what there is to multiply
//                   here leaves the tensor cores idle; tcgen05 would fill 128 rows for 1 to 64), its own running maximum and sum; key groups meet at the end of a piece
//
// Keys outside a sequence (the rest of its last page, slots that left the window) may hold anything: their scores are replaced, not added to, and
// their values are cut out of the fragments, so that neither NaN nor infinities get through.  Scores of a row's own keys that are not finite make it NaN.
//
// Probabilities are rounded to bf16 for their product (a relative error of 1.6e-3 of ordinary rows beside the 1.65e-3 of the result's own rounding: 2.1 to 2.3e-3 in all), which one product of
// two bf16 operands asks for.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "launch.cuh"
#include "paged_attention.cuh"

namespace tpb {

constexpr int PA_TILE = 64;                 // keys of a stage
constexpr int PA_BLOCK = PA_TILE * 128;     // bytes of a swizzled block of 64 keys x 64 elements
constexpr int PA_MIN_SHARE = 3;             // of a team's range, at least: a piece and two tiles
// What a row tile costs beside its key tiles, in tiles: its query rows, the meeting of the key groups, its result.  It stands in front of them on the line.
constexpr int PA_PIECE_COST = 1;
constexpr float PA_RESCALE_LOG2 = 8.f;
// Tables with room for so few keys do without cut row tiles, and so without the second kernel (in a graph, both ways, us: one sequence of 256 keys, 32 heads of 128 8.8 / 10.5, 16
// of 256, 32 / 8 heads 10.3 / 13.1, 16 of 512 13.9 / 16.0; one of 512 11.1 / 10.6, of 1024 18.9 / 13.6).
constexpr int PA_WHOLE_TILES = 8;

// A sequence as this launch deals with it.
struct PagedUnits {
  PagedSequence s;
  int rows, row_tiles, first_tile, tiles;  // tiles of keys, from first_tile on
  long long cost;                          // row_tiles * kv_heads * (tiles + PA_PIECE_COST), 0: not this launch's
};

template <int ROWS>
__device__ __forceinline__ PagedUnits paged_units(const PagedAttnParams& p, int s) {
  PagedUnits u;
  u.s = paged_sequence(p.b, s);
  u.rows = u.s.fresh * p.group;
  u.row_tiles = (u.rows + ROWS - 1) / ROWS;
  const bool mine = u.rows > 0 && (u.s.bad ? p.takes_bad : u.rows >= p.rows_low && u.rows <= p.rows_high);
  u.first_tile = 0;
  u.tiles = 1;  // (a bad sequence: one tile without keys)
  if (!u.s.bad) {
    u.first_tile = p.window ? max(0, u.s.past - p.window + 1) / PA_TILE : 0;
    u.tiles = (u.s.past + u.s.fresh + PA_TILE - 1) / PA_TILE - u.first_tile;
  }
  u.cost = mine ? (long long)u.row_tiles * p.kv_heads * (u.tiles + PA_PIECE_COST) : 0;
  return u;
}

enum { PIECE_FIRST = 1, PIECE_LAST = 2, PIECE_POISON = 4, RANGE_END = 8 };

struct PagedPiece {  // of a row tile's keys, as the producer hands it to the compute warps
  int token0, row0, rows, past, total, low, kvh;  // low: first key that any row of the sequence sees
  int slot;                                       // of the workspace, -1: the piece is the whole
  int bad;
};

__device__ __forceinline__ void tma_load_5d(void* smem_dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w, int v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
      : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// R groups of 16 rows.  Teams of four warps, several per SM, fill each other's gaps where their registers fit; 64 rows of 128 elements take eight warps and the
// SM (32 x 2049 keys, us, with 2 teams of 4 warps / one of 8: 32 rows, 8 heads of 64 35.0 / 47.7, of 128 60.3 / 64.0; 64 rows, of 64 50.9 / 63.6, of 128 one
// team each 95.3 / 90.4; 16 rows of 64 by 2 / 3 / 4 teams, 48 ragged sequences 72.5 / 61.2 / 60.6).  Teams know nothing of each other; that they are one CTA and not
// several costs nothing (within 2 % of those) and leaves the other launch whole SMs.
template <int D, int R>
struct Few {
  static constexpr int ROWS = 16 * R;
  static constexpr int WARPS = R == 4 && D == 128 ? 8 : 4;
  static constexpr int KEY_GROUPS = WARPS / R;
  static constexpr int KEYS = PA_TILE / KEY_GROUPS;  // of a warp
  static constexpr int TEAMS = WARPS == 8 ? 1 : R == 1 && D == 64 ? 3 : 2;  // of a CTA, each with a range of its own
  static constexpr int DB = D / 64;
  static constexpr int STAGE_BYTES = 2 * DB * PA_BLOCK;
  static constexpr int STAGES = (WARPS == 8 ? 160 : R == 1 && D == 128 ? 96 : 64) * 1024 / STAGE_BYTES;
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int MERGE_COLS = STAGE_BYTES / (WARPS * 16 * 4) < D ? STAGE_BYTES / (WARPS * 16 * 4) : D;  // that the partial results of all warps fill a stage with
  static constexpr int THREADS = WARPS * 32 + 32;
  static_assert(PA_TILE % (16 * KEY_GROUPS) == 0 && MERGE_COLS >= 32, "a warp has whole groups of 16 keys");
  static constexpr int TEAM_SMEM = (STAGES * STAGE_BYTES + 2 * Q_BYTES + WARPS * 16 * 8 + STAGES * 8 + 2 * int(sizeof(PagedPiece)) + (2 * STAGES + 6) * 8 + 1279) / 1024 * 1024;
  static constexpr int SMEM = 1024 + TEAMS * TEAM_SMEM;
  static_assert(SMEM + 1024 <= 228 * 1024, "shared memory of an SM");
};

template <int D, int R>
__global__ void __launch_bounds__(Few<D, R>::THREADS* Few<D, R>::TEAMS, 1)
paged_attn_few_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const PagedAttnParams p) {
  using C = Few<D, R>;
  constexpr int DB = C::DB, STAGES = C::STAGES, WARPS = C::WARPS, ROWS = C::ROWS;

  extern __shared__ uint8_t pa_smem_raw[];
  const int team = __shfl_sync(0xffffffffu, threadIdx.x / C::THREADS, 0), thread = threadIdx.x - team * C::THREADS;
  // ranges that lie side by side on an SM when another launch has the SMs behind, else on all SMs first
  const int range_no = p.split_sms ? int(blockIdx.x) * C::TEAMS + team : int(blockIdx.x) + team * int(gridDim.x);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pa_smem_raw) + 1023) & ~uintptr_t(1023)) + team * C::TEAM_SMEM;
  uint8_t* ring = smem;                                    // [STAGES][keys | values][DB][64 keys][128 bytes]
  uint8_t* q_s = ring + STAGES * C::STAGE_BYTES;           // [2][DB][ROWS][128 bytes], swizzled like the ring
  float2* stats = reinterpret_cast<float2*>(q_s + 2 * C::Q_BYTES);       // [WARPS][16 rows]
  int2* stage_info = reinterpret_cast<int2*>(stats + WARPS * 16);        // [STAGES] first key, flags
  PagedPiece* pieces = reinterpret_cast<PagedPiece*>(stage_info + STAGES);  // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(pieces + 2) + 7) & ~uintptr_t(7));
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* q_full = bars + 2 * STAGES;       // [2]
  uint64_t* q_empty = bars + 2 * STAGES + 2;  // [2]
  uint64_t* meet = bars + 2 * STAGES + 4;     // the compute warps, phase by phase
  volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
  __shared__ RangeSearch<C::THREADS> ranges[C::TEAMS];
  RangeSearch<C::THREADS>& range = ranges[team];

  const int warp = __shfl_sync(0xffffffffu, thread >> 5, 0), lane = threadIdx.x & 31;
  if (thread == 0) {
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], WARPS);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 33);  // the lanes' copies and the piece
      mbar_init(&q_empty[s], WARPS);
    }
    mbar_init(meet, WARPS);
    *abort_flag = 0;
    fence_mbar_init();
  }
  pa_wait_prior();  // (launched ahead of the previous kernel's end: nothing is read or written before that)
  pa_launch_next();
  if (thread < 2) p.parts.joins[2 * range_no + thread] = make_int4(-1, 0, 0, 0);

  long long share, w0, w1;
  long long few = 0, wide = 0;
  auto meet_team = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(C::THREADS) : "memory"); };
  share_out<C::THREADS>(p.b.n, p.whole ? 1 : PA_MIN_SHARE, thread, range_no, range, [&](int i) {
    const PagedUnits u = paged_units<ROWS>(p, i);
    if (u.s.bad && p.takes_bad && range_no == 0) atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
    if (p.split_sms) pa_load(p, u.s, D, few, wide);
    return u.cost;
  }, [&]() {
    if (!p.split_sms) return unsigned(p.ranges);
    sum_loads<C::THREADS>(range, thread, meet_team, few, wide);
    return unsigned(max(1, pa_few_sms(few, wide, p.split_sms)) * C::TEAMS);
  }, meet_team, share, w0, w1);
  if (p.fill_rest) fill_around<D, C::THREADS * C::TEAMS>(p);

  auto give_up = [&]() {
    atomicMax(p.b.status, uint32_t(STATUS_TIMEOUT_MBAR));
    *abort_flag = 1;
  };

  if (warp == WARPS) {
    // ---------------- producer ----------------
    const int page_size = 1 << p.b.page_shift;
    const int per_tile = max(1, PA_TILE >> p.b.page_shift);  // pages of a tile
    const int box_rows = min(page_size, PA_TILE);
    const int my_page = lane / 2, box_bytes = box_rows * 128 * DB;  // the box of this lane: keys or values of a page
    int seq = range.seq, it = 0, piece = 0;
    long long at = w0, seq_begin = range.begin;
    bool ok = true;
    while (ok && at < w1) {
      ok = seq < p.b.n;  // (the costs add up to w1, unless somebody writes the lengths meanwhile)
      if (!ok) break;
      const PagedUnits u = paged_units<ROWS>(p, seq);
      if (at >= seq_begin + u.cost) {
        seq_begin += u.cost;
        ++seq;
        continue;
      }
      const int length = u.tiles + PA_PIECE_COST;
      const long long into = at - seq_begin;
      const long long unit = into < INT_MAX ? int(into) / length : into / length;  // (64-bit divisions are long)
      const int from = int(into - unit * length), to = p.whole ? length : int(min((long long)length, from + (w1 - at)));
      if (p.whole && from) {  // (whoever has the beginning of the row tile in its range takes all of it)
        at += length - from;
        continue;
      }
      const int t0 = max(0, from - PA_PIECE_COST), t1 = max(0, to - PA_PIECE_COST);
      at += to - from;
      if (t0 == t1) continue;  // (the range ends in front of the first tile)
      const int kvh = int(unit) % p.kv_heads, row0 = int(unit) / p.kv_heads * ROWS;
      const int total = u.s.bad ? 0 : u.s.past + u.s.fresh;
      const int low = p.window && !u.s.bad ? max(0, u.s.past - p.window + 1) : 0;
      const int qb = piece & 1;
      // table entries, 32 at a time and 32 ahead
      const int* row = p.b.table + (long long)seq * p.b.table_ld;
      int entry0 = (u.first_tile + t0) * PA_TILE >> p.b.page_shift;
      const int entries = total > 0 ? ((total - 1) >> p.b.page_shift) + 1 : 0;
      auto fetch = [&](int e) { return e < entries ? __ldg(row + e) : -1; };
      int now = fetch(entry0 + lane), next = fetch(entry0 + 32 + lane);
      // ---- query rows ----
      ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[qb], ((piece >> 1) & 1) ^ 1));
      if (!ok) break;
      if (lane == 0) {
        PagedPiece& o = pieces[qb];
        o.token0 = u.s.token0;
        o.row0 = row0;
        o.rows = min(ROWS, u.rows - row0);
        o.past = u.s.past;
        o.total = total;
        o.low = low;
        o.kvh = kvh;
        o.bad = u.s.bad;
        // keys that begin in this range and end in another's are joined by the blocks of this range; its other piece continues the range in front
        o.slot = t0 == 0 && t1 == u.tiles ? -1 : 2 * range_no + (t0 == 0 ? 1 : 0);
      }
      {
        constexpr int STEP = 32 / (D / 8);  // rows at a time
        const int e = lane % (D / 8), left = u.rows - row0;
        const int step_tokens = STEP / p.group, step_heads = STEP % p.group;
        int r = lane / (D / 8), t = (row0 + r) / p.group, g = (row0 + r) % p.group;
        const bf16* base = p.q + (long long)u.s.token0 * p.q_st + (long long)kvh * p.group * p.q_sh + e * 8;
        const uint32_t to = smem_u32(q_s + qb * C::Q_BYTES + (e >> 3) * (ROWS * 128));
#pragma unroll
        for (int i = 0; i < ROWS / STEP; ++i, r += STEP) {
          cp_async16(to + r * 128 + (((e & 7) ^ (r & 7)) << 4), r < left ? base + t * p.q_st + g * p.q_sh : base, r < left ? 16 : 0);
          t += step_tokens;
          g += step_heads;
          if (g >= p.group) {
            g -= p.group;
            ++t;
          }
        }
        cp_async_arrive(&q_full[qb]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[qb]);
      }
      // ---- keys and values ----
      for (int t = t0; t < t1; ++t, ++it) {
        const int stage = it % STAGES;
        const int key0 = (u.first_tile + t) * PA_TILE;
        int e = (key0 >> p.b.page_shift) - entry0;
        if (e >= 32) {
          entry0 += 32;
          e -= 32;
          now = next;
          next = fetch(entry0 + 32 + lane);
        }
        const int page = __shfl_sync(0xffffffffu, now, (e + my_page) & 31);
        const int first = key0 + my_page * page_size;  // (of pages shorter than a tile; longer ones have one box, with keys of use in it)
        const bool wanted = lane < per_tile * 2 && (per_tile == 1 || (first < total && first + page_size > low)) && total > 0;
        const bool good = wanted && page >= 0 && page < p.b.pages;
        const uint32_t boxes = __ballot_sync(0xffffffffu, good), lost = __ballot_sync(0xffffffffu, wanted && !good);
        ok = __all_sync(0xffffffffu, !*abort_flag && mbar_wait(&empty[stage], ((it / STAGES) & 1) ^ 1));
        if (!ok) break;
        if (lane == 0) {
          if (lost) atomicMax(p.b.status, uint32_t(STATUS_BAD_ARG));
          stage_info[stage] = make_int2(key0, (t == t0 ? PIECE_FIRST : 0) | (t == t1 - 1 ? PIECE_LAST : 0) | (lost ? PIECE_POISON : 0));
          mbar_expect_tx(&full[stage], __popc(boxes) * box_bytes);
        }
        __syncwarp();
        if (good)
          tma_load_5d(ring + stage * C::STAGE_BYTES + (lane & 1) * (DB * PA_BLOCK) + my_page * box_bytes, lane & 1 ? &tmap_v : &tmap_k, &full[stage], 0,
                      per_tile == 1 ? key0 & (page_size - 1) : 0, 0, kvh, page);
      }
      if (!ok) break;
      ++piece;
      if (t0 == 0 && t1 < u.tiles && lane == 0) {
        const long long unit_end = seq_begin + (unit + 1) * length;
        p.parts.joins[2 * range_no] = make_int4(u.s.token0, row0, min(ROWS, u.rows - row0), kvh);
        p.parts.joins[2 * range_no + 1] = make_int4(int((unit_end - 1) / share), 0, 0, 0);
      }
    }
    if (ok) {
      const int stage = it % STAGES;
      ok = __all_sync(0xffffffffu, !*abort_flag && mbar_wait(&empty[stage], ((it / STAGES) & 1) ^ 1));
      if (ok && lane == 0) {
        stage_info[stage] = make_int2(0, RANGE_END);
        mbar_arrive(&full[stage]);
      }
    }
    if (!ok && lane == 0 && !*abort_flag) give_up();
    return;
  }

  // ---------------- compute warps ----------------
  constexpr int NT = C::KEYS / 8;  // blocks of 8 keys
  const int rg = warp % R, kg = warp / R;
  const int key_off = kg * C::KEYS;
  const int g8 = lane >> 2, t4 = lane & 3, mi = lane >> 3, mr = lane & 7;
  const uint32_t ring_a = smem_u32(ring), q_a = smem_u32(q_s);
  // a stage holds page by page, in each its blocks of 64 elements; 16 keys are always of one page
  const int box_shift = min(p.b.page_shift, 6), block_step = 128 << box_shift;
  uint32_t group_a[NT / 2];
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) {
    const int key = key_off + i * 16;
    group_a[i] = (key >> box_shift) * (block_step * DB) + (key & ((1 << box_shift) - 1)) * 128;
  }
  float o[D / 8][4];
  float m[2], l[2];
  uint32_t qf[R == 1 ? D / 16 : 1][4];
  PagedPiece pc = {};
  int pos[2] = {0, 0}, piece = 0, plain_from = 0, plain_to = 0;
  uint32_t meet_phase = 0;
  bool poisoned = false;
  bool ok = true;
  auto meet_all = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(meet);
    ok = __all_sync(0xffffffffu, mbar_wait(meet, meet_phase));
    meet_phase ^= 1;
    return ok;
  };
  for (int stage = 0, phase = 0;; phase ^= stage == STAGES - 1, stage = stage == STAGES - 1 ? 0 : stage + 1) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase));
    if (!ok) break;
    const int2 info = stage_info[stage];
    if (info.y & RANGE_END) break;
    const int key0 = info.x + key_off;
    if (info.y & PIECE_FIRST) {
      ok = __all_sync(0xffffffffu, mbar_wait(&q_full[piece & 1], (piece >> 1) & 1));
      if (!ok) break;
      pc = pieces[piece & 1];
      poisoned = pc.bad;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        pos[i] = pc.past + (pc.row0 + rg * 16 + g8 + 8 * i) / p.group;
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      // the warp's keys of a tile need no mask if they begin in [plain_from, plain_to]
      plain_from = p.window ? pc.past + (pc.row0 + pc.rows - 1) / p.group - p.window + 1 : 0;
      plain_to = pc.past + pc.row0 / p.group + 1 - C::KEYS;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      if (R == 1) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int r = (mi & 1) * 8 + mr, c = kk * 2 + (mi >> 1);
          ldsm4(qf[R == 1 ? kk : 0], q_a + (piece & 1) * C::Q_BYTES + (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
        }
      }
    }
    poisoned |= (info.y & PIECE_POISON) != 0;
    // ---- scores: all fragments of 16 keys in front of the products, which go in two chains (what bounds a tile is the length of its chain) ----
    float sc[NT][4];
    const uint32_t k_a = ring_a + stage * C::STAGE_BYTES, v_a = k_a + DB * PA_BLOCK;
#pragma unroll
    for (int np = 0; np < NT / 2; ++np) {
      uint32_t kf[D / 16][4];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int c = kk * 2 + (mi & 1);
        ldsm4(kf[kk], k_a + group_a[np] + (kk >> 2) * block_step + ((mi >> 1) * 8 + mr) * 128 + (((c & 7) ^ mr) << 4));
      }
      float odd[2][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[2 * np][j] = sc[2 * np + 1][j] = odd[0][j] = odd[1][j] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t a[4];
        if (R == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) a[j] = qf[R == 1 ? kk : 0][j];
        } else {
          const int r = rg * 16 + (mi & 1) * 8 + mr, c = kk * 2 + (mi >> 1);
          ldsm4(a, q_a + (piece & 1) * C::Q_BYTES + (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
        }
        mma16816(kk & 1 ? odd[0] : sc[2 * np], a, kf[kk][0], kf[kk][1]);
        mma16816(kk & 1 ? odd[1] : sc[2 * np + 1], a, kf[kk][2], kf[kk][3]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[2 * np][j] += odd[0][j];
        sc[2 * np + 1][j] += odd[1][j];
      }
    }
    // the values of the first 16 keys come while the probabilities are made
    uint32_t vf[D / 16][4];
    auto load_values = [&](int ks) {
#pragma unroll
      for (int dn = 0; dn < D / 16; ++dn) {
        const int c = dn * 2 + (mi >> 1);
        ldsm4_t(vf[dn], v_a + group_a[ks] + (dn >> 2) * block_step + ((mi & 1) * 8 + mr) * 128 + (((c & 7) ^ mr) << 4));
      }
    };
    load_values(0);
    // ---- mask, maximum, probabilities (2^(score - m), scores in powers of two) ----
    if (key0 < plain_from || key0 > plain_to) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + i * 8 + t4 * 2 + (j & 1), at = pos[j >> 1];
          if (key > at || (p.window && key <= at - p.window)) sc[i][j] = -INFINITY;
        }
    }
    float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; j += 2) mt[j >> 1] = fmax3(mt[j >> 1], sc[i][j], sc[i][j + 1]);
    // the maximum is followed when it rises by more than 2^8, which is rare behind the first tiles (it cancels in the quotient; the scale is positive);
    // only then do the four lanes of a row need to know each other's
    if (__any_sync(0xffffffffu, mt[0] * p.scale_log2e > m[0] + PA_RESCALE_LOG2 || mt[1] * p.scale_log2e > m[1] + PA_RESCALE_LOG2)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mt[i] = fmaxf(mt[i], __shfl_xor_sync(0xffffffffu, mt[i], 1));
        mt[i] = fmaxf(mt[i], __shfl_xor_sync(0xffffffffu, mt[i], 2));
        const float mn = fmaxf(m[i], mt[i] * p.scale_log2e);
        const float f = m[i] == -INFINITY ? 0.f : ex2_approx(m[i] - mn);
        m[i] = mn;
        l[i] *= f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][2 * i] *= f;
          o[d][2 * i + 1] *= f;
        }
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[i][j] = ex2_approx(fmaf(sc[i][j], p.scale_log2e, base[j >> 1]));
    // the sum is of the probabilities as the product takes them: where one key has nearly all of a row, its rounding cancels in the quotient (mean error of
    // results of 256 keys 2.5e-3 -> 2.0e-3, 1.4e-3 of it their own rounding)
    uint32_t pr[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        pr[i][j] = pack_bf16x2(sc[i][2 * j], sc[i][2 * j + 1]);
        l[j] += __uint_as_float(pr[i][j] << 16) + __uint_as_float(pr[i][j] & 0xFFFF0000u);
      }
    // ---- values ----
    const bool cut = key0 < pc.low || key0 + C::KEYS > pc.total;
#pragma unroll
    for (int ks = 0; ks < NT / 2; ++ks) {
      const uint32_t a[4] = {pr[2 * ks][0], pr[2 * ks][1], pr[2 * ks + 1][0], pr[2 * ks + 1][1]};
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (cut) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = key0 + ks * 16 + i * 8 + t4 * 2;
          keep[i] = (key >= pc.low && key < pc.total ? 0xffffu : 0u) | (key + 1 >= pc.low && key + 1 < pc.total ? 0xffff0000u : 0u);
        }
      }
      if (ks) load_values(ks);
#pragma unroll
      for (int dn = 0; dn < D / 16; ++dn) {
        if (cut) {
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[dn][j] &= keep[j & 1];
        }
        mma16816(o[2 * dn], a, vf[dn][0], vf[dn][1]);
        mma16816(o[2 * dn + 1], a, vf[dn][2], vf[dn][3]);
      }
    }
    if (!(info.y & PIECE_LAST)) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      continue;
    }
    // ---- the key groups meet, in the room of the stage that all of them have read: [warp][16 rows][COLS], blocks of eight columns swizzled by row ----
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if (t4 == 0) stats[warp * 16 + g8 + 8 * i] = make_float2(m[i], l[i]);
    }
    if (!meet_all()) break;
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < C::KEY_GROUPS; ++k) top = fmaxf(top, stats[(k * R + rg) * 16 + g8 + 8 * i].x);
      const float b0 = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < C::KEY_GROUPS; ++k) {
        const float2 st = stats[(k * R + rg) * 16 + g8 + 8 * i];
        sum += st.y * ex2_approx(st.x - b0);
      }
      f[i] = ex2_approx(m[i] - b0);
      if (poisoned) {
        top = 0.f;
        sum = __uint_as_float(0x7fc00000u);
      }
      // a row sees its own key at least: a sum of zero is of scores that are all -inf, and its result NaN (written as the plain quotient, decoding beside a chunk takes
      // 124 us for 120)
      if (pc.slot < 0) f[i] = sum == 0.f ? __uint_as_float(0x7fc00000u) : f[i] / sum;
      if (pc.slot >= 0 && kg == 0 && t4 == 0) p.parts.ml[(long long)pc.slot * ROWS + rg * 16 + g8 + 8 * i] = make_float2(top, sum);
    }
    float* merge = reinterpret_cast<float*>(ring + stage * C::STAGE_BYTES);
    constexpr int COLS = C::MERGE_COLS;
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += COLS) {
      if (c0 && !meet_all()) break;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int d = 0; d < COLS / 8; ++d)
          *reinterpret_cast<float2*>(merge + (warp * 16 + g8 + 8 * i) * COLS + ((d ^ (g8 & (COLS / 8 - 1))) * 8) + t4 * 2) =
              make_float2(o[c0 / 8 + d][2 * i] * f[i], o[c0 / 8 + d][2 * i + 1] * f[i]);
      if (!meet_all()) break;
      for (int c = thread; c < pc.rows * (COLS / 4); c += WARPS * 32) {
        const int r = c / (COLS / 4), col = (c % (COLS / 4)) * 4;
        const float* from = merge + ((r >> 4) * 16 + (r & 15)) * COLS + (((col >> 3) ^ (r & 7 & (COLS / 8 - 1))) * 8) + (col & 7);
        float4 v = *reinterpret_cast<const float4*>(from);
#pragma unroll
        for (int k = 1; k < C::KEY_GROUPS; ++k) {
          const float4 w = *reinterpret_cast<const float4*>(from + k * R * 16 * COLS);
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        if (pc.slot >= 0) {
          *reinterpret_cast<float4*>(p.parts.o + ((long long)pc.slot * ROWS + r) * D + c0 + col) = v;
        } else {
          const int t = (pc.row0 + r) / p.group, h = (pc.row0 + r) % p.group;
          *reinterpret_cast<uint2*>(p.out + (long long)(pc.token0 + t) * p.o_st + (long long)(pc.kvh * p.group + h) * p.o_sh + c0 + col) =
              make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        }
      }
    }
    if (!ok) break;
    fence_proxy_async_smem();  // (the next bulk copies come behind these writes)
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&empty[stage]);
      mbar_arrive(&q_empty[piece & 1]);
    }
    ++piece;
  }
  if (!ok && lane == 0 && !*abort_flag) give_up();
}

// Joins the pieces of the row tile whose keys begin in one range and end in another: blocks for each range, of which most have nothing to do, and a
// thread for every four columns of a row or of several.  Behind those of the launch for few rows come those of the one for many.
constexpr int PA_JOIN_THREADS = 128;

template <int D>
__global__ void __launch_bounds__(PA_JOIN_THREADS)
paged_attn_join_kernel(const PagedAttnParams p, const PagedParts few, const int few_blocks, const int blocks_of_few, const PagedParts wide, const int blocks_of_wide) {
  const bool is_wide = int(blockIdx.x) >= few_blocks;
  const PagedParts parts = is_wide ? wide : few;
  const int at = blockIdx.x - (is_wide ? few_blocks : 0), blocks = is_wide ? blocks_of_wide : blocks_of_few, c = at / blocks;
  pa_wait_prior();
  pa_launch_next();
  const int4 unit = parts.joins[2 * c];
  const int last = parts.joins[2 * c + 1].x;
  if (unit.x < 0) return;
  auto slot = [&](int i) { return (long long)(i == c ? 2 * c + 1 : 2 * i) * parts.rows; };
  for (int item = at % blocks * PA_JOIN_THREADS + threadIdx.x; item < unit.z * (D / 4); item += blocks * PA_JOIN_THREADS) {
    const int r = item / (D / 4), col = item % (D / 4) * 4;
    const float2* ml = parts.ml + r;
    const float* part = parts.o + (long long)r * D + col;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    // (several pieces at a time, all their loads in front of the first use; the sums so far are brought to a new maximum)
    constexpr int AT_ONCE = 4;
    for (int i0 = c; i0 <= last; i0 += AT_ONCE) {
      float2 s[AT_ONCE];
      float4 w[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        s[j] = make_float2(-INFINITY, 0.f);
        if (i0 + j <= last) {
          s[j] = ml[slot(i0 + j)];
          w[j] = *reinterpret_cast<const float4*>(part + slot(i0 + j) * D);
        }
      }
      float next = top;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) next = fmaxf(next, s[j].x);
      const float down = top == -INFINITY ? 0.f : ex2_approx(top - next);
      sum *= down;
      v.x *= down, v.y *= down, v.z *= down, v.w *= down;
      top = next;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        if (s[j].x == -INFINITY && s[j].y == 0.f) continue;  // (no key of the piece is the row's; scores that are all NaN leave the sum NaN)
        const float f = ex2_approx(s[j].x - top);
        sum += s[j].y * f;
        v.x += w[j].x * f, v.y += w[j].y * f, v.z += w[j].z * f, v.w += w[j].w * f;
      }
    }
    const float inv = 1.f / sum;
    const int t = (unit.y + r) / p.group, h = (unit.y + r) % p.group;
    *reinterpret_cast<uint2*>(p.out + (long long)(unit.x + t) * p.o_st + (long long)(unit.w * p.group + h) * p.o_sh + col) =
        make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
  }
}

template <int D, int R>
static int pa_few_launch(const PagedAttnParams& p, const CUtensorMap& k, const CUtensorMap& v, int grid, cudaStream_t stream) {
  using C = Few<D, R>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(paged_attn_few_kernel<D, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return TPB_ERR_CUDA;
    ready[dev].store(true, std::memory_order_release);
  }
  return launch_dependent(paged_attn_few_kernel<D, R>, dim3(grid), dim3(C::THREADS * C::TEAMS), C::SMEM, stream, true, k, v, p) == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

static int pa_few_teams(int head_dim, int row_groups) {
  if (head_dim == 64) return row_groups == 1 ? Few<64, 1>::TEAMS : row_groups == 2 ? Few<64, 2>::TEAMS : Few<64, 4>::TEAMS;
  return row_groups == 1 ? Few<128, 1>::TEAMS : row_groups == 2 ? Few<128, 2>::TEAMS : Few<128, 4>::TEAMS;
}

// What a call launches.  Sequences with few query rows (new tokens x query heads of a KV head) go by the kernel above, bound by memory; those with more by the one
// on the tensor cores of paged_attention_sm100.cu.  The host knows the rows of a sequence at most; where both kinds may be in the batch, both are launched.
struct PagedPlan {
  int row_groups, few_grid, few_slots, few_ranges, few_high, wide_grid;  // grid 0: not launched; sequences up to few_high rows are the first's
  bool joins;
  long long few_floats, wide_floats;
};
static PagedPlan pa_plan(int n, int tokens, int table_width, int page_shift, int most_new, int kv_heads, int group, int head_dim) {
  PagedPlan plan = {};
  const long long most_rows = (long long)min(most_new, tokens) * group, keys = (long long)table_width << page_shift;
  const bool wide = most_rows > 64, few = !wide || (n > 1 && group <= 64);
  plan.joins = wide || keys > PA_WHOLE_TILES * PA_TILE;
  // Rows of a tile of the first: all of a sequence's where there are no more than 64, else those of one token, since most sequences of such a batch decode and larger tiles cost
  // them (32 x 2049 keys, 8 KV heads, 16 rows in tiles of 16 / 20 in tiles of 32, us: 30.8 / 35.7 at 64, 53.8 / 56.9 at 128).  Sequences with a few tokens more pay for it, in a batch with a chunk or
  // without most_new: 20 rows, 32 x 2049 keys by this kernel / by the other 35.7 / 67.3 at 64, 56.9 / 90.0 at 128 (64 rows 52.4 / 68.6, 92.2 / 90.9); beside 777 tokens
  // behind 3396 16 rows 83.8 and 110, 20 rows 109 and 144.
  const long long usual = wide ? group : most_rows;
  plan.row_groups = usual <= 16 ? 1 : usual <= 32 ? 2 : 4;
  const int rows = 16 * plan.row_groups;
  plan.few_high = !few ? 0 : wide ? rows : INT_MAX;
  if (few) {
    const long long tiles = min((long long)tokens * group / rows + n, (long long)n * ((min(most_rows, (long long)plan.few_high) + rows - 1) / rows)) * kv_heads;
    const long long most = tiles * ((keys + PA_TILE - 1) / PA_TILE + PA_PIECE_COST), ranges = plan.joins ? (most + PA_MIN_SHARE - 1) / PA_MIN_SHARE : tiles;
    plan.few_grid = wide ? pa_sms() : int(max(1LL, min((long long)pa_sms(), ranges)));
    plan.few_slots = plan.few_grid * pa_few_teams(head_dim, plan.row_groups);
    plan.few_ranges = wide ? plan.few_slots : int(max(1LL, min((long long)plan.few_slots, ranges)));
    plan.few_floats = (long long)plan.few_slots * 2 * (rows * (head_dim + 2) + 4);
  }
  if (wide) {
    plan.wide_grid = pw_grid(head_dim);
    plan.wide_floats = (long long)plan.wide_grid * 2 * (PW_ROWS * (head_dim + 2) + 4);
  }
  return plan;
}
static PagedParts pa_parts(float*& room, int grid, int rows, int head_dim) {
  PagedParts parts;
  parts.o = room;
  parts.ml = reinterpret_cast<float2*>(room + (long long)grid * 2 * rows * head_dim);
  parts.joins = reinterpret_cast<int4*>(parts.ml + (long long)grid * 2 * rows);
  parts.rows = rows;
  room += (long long)grid * 2 * (rows * (head_dim + 2) + 4);
  return parts;
}

}  // namespace tpb

using namespace tpb;

extern "C" long long tpb_paged_attention_workspace(int n, int tokens, int table_width, int page_size, int most_new, int kv_heads, int group, int head_dim) {
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  const PagedPlan plan = pa_plan(n, tokens, table_width, shift, most_new, kv_heads, group, head_dim);
  return (plan.few_floats + plan.wide_floats) * 4;
}

extern "C" int tpb_paged_attention(tpb_paged_attn_t* a, void* stream_) {
  if (!a || !a->q || !a->out || !a->keys || !a->values || !a->table || !a->starts || !a->past || !a->status || !a->workspace) return TPB_ERR_ARG;
  if (a->n <= 0 || a->tokens <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || a->pages <= 0 || a->table_width <= 0 || a->window < 0 ||
      a->most_new < 0)
    return TPB_ERR_ARG;
  if ((a->head_dim != 64 && a->head_dim != 128) || a->page_size < 16 || (a->page_size & (a->page_size - 1))) return TPB_ERR_ARG;
  if ((long long)a->tokens * a->heads >= 1 << 30) return TPB_ERR_SIZE;
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(a->keys) |
                              reinterpret_cast<uintptr_t>(a->values) | reinterpret_cast<uintptr_t>(a->workspace);
  if ((addresses & 15) || ((a->q_st | a->q_sh | a->o_st | a->o_sh | a->k_sp | a->k_sh | a->k_ss | a->v_sp | a->v_sh | a->v_ss) & 7)) return TPB_ERR_ALIGN;
  int rc = fa_bind_thread();
  if (rc != TPB_OK) return rc;
  int shift = 0;
  while ((1 << shift) < a->page_size) ++shift;
  const int group = a->heads / a->kv_heads;
  const PagedPlan plan = pa_plan(a->n, a->tokens, a->table_width, shift, a->most_new, a->kv_heads, group, a->head_dim);
  if (a->workspace_bytes < (plan.few_floats + plan.wide_floats) * 4) return TPB_ERR_WORKSPACE;
  a->launches = (plan.few_grid != 0) + (plan.wide_grid != 0) + plan.joins;
  PagedAttnParams p = {};
  p.b = {a->starts, a->past, a->table, a->table_ld, a->n, a->tokens, a->table_width, a->pages, shift, a->most_new, static_cast<uint32_t*>(a->status)};
  p.q = static_cast<const bf16*>(a->q);
  p.out = static_cast<bf16*>(a->out);
  p.q_st = a->q_st, p.q_sh = a->q_sh, p.o_st = a->o_st, p.o_sh = a->o_sh;
  p.heads = a->heads, p.kv_heads = a->kv_heads, p.group = group, p.window = a->window;
  p.scale_log2e = a->scale * 1.4426950408889634f;
  p.whole = !plan.joins;
  p.few_high = plan.few_high;
  p.split_sms = plan.few_grid && plan.wide_grid ? pa_sms() : 0;
  float* room = static_cast<float*>(a->workspace);
  const PagedParts few = pa_parts(room, plan.few_slots, 16 * plan.row_groups, a->head_dim), wide = pa_parts(room, plan.wide_grid, PW_ROWS, a->head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  auto maps = [&](auto paged_map, CUtensorMap& k, CUtensorMap& v, int tile) {
    const int box = min(a->page_size, tile);
    const int r = paged_map(&k, a->keys, a->head_dim, a->page_size, a->kv_heads, a->pages, a->k_ss, a->k_sh, a->k_sp, box);
    return r != TPB_OK ? r : paged_map(&v, a->values, a->head_dim, a->page_size, a->kv_heads, a->pages, a->v_ss, a->v_sh, a->v_sp, box);
  };
  CUtensorMap k, v;
  if (plan.few_grid) {
    rc = maps(paged_blocks_tmap, k, v, PA_TILE);
    if (rc != TPB_OK) return rc;
    p.parts = few;
    p.ranges = plan.few_ranges;
    p.rows_low = 1, p.rows_high = plan.few_high;
    p.takes_bad = 1;
    p.fill_rest = a->fill_rest;
#define PA_LAUNCH(D) \
  (plan.row_groups == 1 ? pa_few_launch<D, 1>(p, k, v, plan.few_grid, s) : plan.row_groups == 2 ? pa_few_launch<D, 2>(p, k, v, plan.few_grid, s) : pa_few_launch<D, 4>(p, k, v, plan.few_grid, s))
    rc = a->head_dim == 64 ? PA_LAUNCH(64) : PA_LAUNCH(128);
#undef PA_LAUNCH
    if (rc != TPB_OK) return rc;
  }
  if (plan.wide_grid) {
    rc = maps(paged_tmap, k, v, pw_tile(a->head_dim));
    if (rc != TPB_OK) return rc;
    p.parts = wide;
    p.rows_low = plan.few_high + 1, p.rows_high = INT_MAX;
    p.takes_bad = plan.few_grid == 0;
    p.fill_rest = a->fill_rest && !plan.few_grid;
    rc = pw_launch(a->head_dim, p, k, v, plan.wide_grid, plan.few_grid != 0, s);
    if (rc != TPB_OK) return rc;
  }
  if (!plan.joins) return TPB_OK;
  // a thread for each four columns of the first launch's tiles, for each eight of the second's
  auto blocks = [&](int rows, int of_thread) { return (rows * (a->head_dim / 4) + of_thread * PA_JOIN_THREADS - 1) / (of_thread * PA_JOIN_THREADS); };
  const int of_few = blocks(int(min((long long)few.rows, max(1LL, (long long)min(a->most_new, a->tokens) * group))), 1), of_wide = blocks(PW_ROWS, 2);
  const int few_blocks = plan.few_ranges * of_few;
  const dim3 grid(few_blocks + plan.wide_grid * of_wide);
  auto join = a->head_dim == 64 ? paged_attn_join_kernel<64> : paged_attn_join_kernel<128>;
  const cudaError_t launched = launch_dependent(join, grid, dim3(PA_JOIN_THREADS), 0, s, true, p, few, few_blocks, of_few, wide, of_wide);
  return launched == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

// Few-token product of 8-bit integers (decode), at most 64 tokens: see gemm_i8.cuh.
//
// Bound by the stream of weights, every byte of which is read from HBM once.  The decomposition is that of the bf16 kernel
// (gemm_stream_sm100.cu): rows dealt out in units of 32, one contiguous range per CTA, walked in passes of up to 128 rows (the lanes of TMEM);
// tokens are the N side; with `early` the ring fills with weights before griddepcontrol.wait.  A box is 128 bytes wide there and here, so that
// what differs is the number of columns in it (128), the MMA (kind::i8, 32 columns a step, exact 32-bit sums) and the epilogue, which scales.
//
// One CTA: warp 0 = TMA producer, warp 1 = MMA issuer, then 4 epilogue warps (8 from 64 tokens on, each with half of them).  Rows of the MMA past the pass multiply whatever lies
// behind it in shared memory; their results are never read.  Every mbarrier wait is bounded; on expiry the CTA records a status code and drains.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>

#include "gemm_i8.cuh"
#include "gemm_stream.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

constexpr int IS_UNIT = StreamRows::UNIT;
__host__ __device__ constexpr int IS_EPI(int bn, int ks) { return bn >= 64 && ks == 1 ? 256 : 128; }  // epilogue threads
constexpr int IS_CONTROL = 2048;  // barriers, scales of the tokens
constexpr int IS_MAX_STAGES = 16;
constexpr size_t IS_RING_BYTES = 204 * 1024;
__host__ __device__ constexpr size_t IS_SLICE_BYTES(int ks) { return ks > 1 ? 9 * 1024 : 0; }

struct IsParams {
  I8Gemm g;
  StreamRows rows;  // (a stage's layout follows its pass_units; tmap_w loads boxes of its box_units, tmap_w1 of one unit)
  int k_stages;
  int slice_cols;   // KS > 1: columns of a slice
  int stages;
};

// NACC accumulators per pass: consecutive MMAs into the same TMEM columns serialise, so k-steps are dealt round-robin and the epilogue adds the
// accumulators up.  KBOX boxes of 128 columns per stage and unit.
// KS > 1 (every CTA has one unit): the contraction is cut into KS slices that run side by side: weight slice s fills rows 32 s .. of the tile, token
// slice s columns TOK s .., the diagonal blocks of the product are the slices' sums (the other blocks are never read), added up through shared memory.
template <int BN, int NACC, int KBOX, int KS>
__global__ void __launch_bounds__(64 + IS_EPI(BN, KS), 1)
gemm_i8_stream_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w1, const __grid_constant__ CUtensorMap tmap_x,
                      const IsParams p) {
  constexpr uint32_t X_BOX = BN * I8_BK, X_BYTES = KBOX * X_BOX;
  constexpr uint32_t ACC_COLS = NACC * BN, TMEM_COLS = 2 * ACC_COLS;  // two accumulator sets: a pass's epilogue runs under the next
  constexpr int STEPS = KBOX * (I8_BK / 32);  // MMAs of a stage; step n of the pass goes to accumulator n % NACC
  static_assert(TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0 && TMEM_COLS >= 32, "TMEM allocation");
  constexpr int TOK = BN / KS;  // token columns of a slice
  constexpr int EPI = IS_EPI(BN, KS);
  const I8Gemm& g = p.g;
  const uint32_t w_box = uint32_t(KS > 1 ? KS : p.rows.pass_units) * IS_UNIT * 128;  // [rows of a pass, or of all slices][128 columns]
  const uint32_t w_bytes = KBOX * w_box, stage_bytes = w_bytes + X_BYTES;

  extern __shared__ uint8_t is_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(is_smem_raw) + 1023) & ~uintptr_t(1023));
  // control block first; the ring (and the rows that an MMA reads past its pass) behind it
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty_bar = full_bar + IS_MAX_STAGES;
  uint64_t* acc_full = empty_bar + IS_MAX_STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;              // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float* sx = reinterpret_cast<float*>(tmem_slot + 4);    // [BN] scales of the tokens
  int* slices = reinterpret_cast<int*>(smem + IS_CONTROL);     // KS > 1: [KS][32 rows][TOK + 1] partial sums
  uint8_t* ring = smem + IS_CONTROL + IS_SLICE_BYTES(KS);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (known to be uniform)
  const int unit0 = p.rows.first(blockIdx.x), my_units = p.rows.first(blockIdx.x + 1) - unit0, passes = p.rows.passes;
  auto pass_start = [&](int i) { return p.rows.pass_start(unit0, my_units, i); };
  auto pass_units = [&](int i) { return pass_start(i + 1) - pass_start(i); };

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_w1);
    prefetch_tmap(&tmap_x);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], EPI / 32);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (!g.early) pdl_wait();

  auto give_up = [&]() {
    atomicMax(g.status, STATUS_TIMEOUT_MBAR);
    *abort_flag = 1;
  };

  if (warp == 0) {
    // ---------------- TMA producer (the warp stays together, one lane issues) ----------------
    const uint32_t leader = elect_one();
    struct Stage { int pass, ks, s; uint32_t parity; };
    auto advance = [&](Stage& i) {
      if (++i.ks == p.k_stages) { i.ks = 0; ++i.pass; }
      if (++i.s == p.stages) { i.s = 0; i.parity ^= 1; }
    };
    auto load_w = [&](const Stage& i) {
      const int u = pass_units(i.pass), row0 = pass_start(i.pass) * IS_UNIT, col0 = i.ks * KBOX * I8_BK;
      const uint32_t dst = smem_u32(ring + size_t(i.s) * stage_bytes);
      uint64_t* bar = &full_bar[i.s];
      mbar_expect_tx_lead(leader, bar, KBOX * uint32_t(KS > 1 ? KS : u) * IS_UNIT * 128 + X_BYTES);
      if (KS > 1) {
#pragma unroll
        for (int j = 0; j < KBOX; ++j)
#pragma unroll
          for (int sl = 0; sl < KS; ++sl)
            tma_load_2d_lead(leader, dst + j * w_box + sl * IS_UNIT * 128, &tmap_w1, bar, sl * p.slice_cols + col0 + j * I8_BK, row0);
        return;
      }
      int done = 0;
      for (; done + p.rows.box_units <= u; done += p.rows.box_units) {
#pragma unroll
        for (int j = 0; j < KBOX; ++j)  // (columns and rows past the end arrive as zeros)
          tma_load_2d_lead(leader, dst + j * w_box + done * IS_UNIT * 128, &tmap_w, bar, col0 + j * I8_BK, row0 + done * IS_UNIT);
      }
      for (; done < u; ++done) {
#pragma unroll
        for (int j = 0; j < KBOX; ++j)
          tma_load_2d_lead(leader, dst + j * w_box + done * IS_UNIT * 128, &tmap_w1, bar, col0 + j * I8_BK, row0 + done * IS_UNIT);
      }
    };
    auto load_x = [&](const Stage& i) {
      const uint32_t dst = smem_u32(ring + size_t(i.s) * stage_bytes + w_bytes);
#pragma unroll
      for (int j = 0; j < KBOX; ++j)
#pragma unroll
        for (int sl = 0; sl < KS; ++sl)
          tma_load_2d_lead(leader, dst + j * X_BOX + sl * TOK * 128, &tmap_x, &full_bar[i.s], sl * p.slice_cols + (i.ks * KBOX + j) * I8_BK, 0);
    };
    const int total = passes * p.k_stages, ahead = min(total, p.stages);
    Stage w = {0, 0, 0, 0}, x = w;  // (parity: round of the ring, a stage is free again after the round before)
    for (int n = 0; n < ahead; ++n, advance(w)) load_w(w);
    pdl_wait();
    pdl_trigger();
    for (int n = 0; n < ahead; ++n, advance(x)) load_x(x);
    for (int n = ahead; n < total; ++n, advance(w)) {
      const bool free_stage = !*abort_flag && mbar_wait(&empty_bar[w.s], w.parity ^ 1);
      if (!__all_sync(0xffffffffu, free_stage)) {
        if (leader) give_up();
        break;
      }
      load_w(w);
      load_x(w);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the warp stays together, one lane issues: see umma_bf16_lead) ----------------
    const uint32_t leader = elect_one();
    int s = 0;
    uint32_t parity = 0;
    for (int pass = 0; pass < passes; ++pass) {
      const int acc = pass & 1;
      const bool free_acc = !*abort_flag && mbar_wait(&acc_empty[acc], ((pass >> 1) & 1) ^ 1);
      if (!__all_sync(0xffffffffu, free_acc)) {
        if (leader) give_up();
        break;
      }
      tc_fence_after();
      const int u = pass_units(pass);
      const uint32_t idesc = make_idesc_i8((KS == 1 && u * IS_UNIT <= 64 && g.act != I8_GATED) ? 64 : 128, BN);
      const uint32_t d_tmem = tmem_base + acc * ACC_COLS;
      bool ok = true;
      for (int ks = 0; ks < p.k_stages; ++ks) {
        const bool full = mbar_wait(&full_bar[s], parity);
        if (!__all_sync(0xffffffffu, full)) {
          if (leader) give_up();
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w_addr = smem_u32(ring + size_t(s) * stage_bytes);
        const uint32_t w_lo = desc_kmajor_lo(w_addr), x_lo = desc_kmajor_lo(w_addr + w_bytes);
#pragma unroll
        for (int j = 0; j < KBOX; ++j) {
#pragma unroll
          for (int kk = 0; kk < I8_BK / 32; ++kk) {
            const int n = j * (I8_BK / 32) + kk;
            const uint32_t d = STEPS % NACC == 0 ? (n % NACC) * BN : ((ks * STEPS + n) % NACC) * BN;
            umma_i8_lead(leader, d_tmem + d, w_lo + j * (w_box >> 4) + kk * 2, x_lo + j * (X_BOX >> 4) + kk * 2, idesc,
                         ks * STEPS + n >= NACC ? 1u : 0u);
          }
        }
        umma_commit_lead(leader, &empty_bar[s]);
        if (++s == p.stages) { s = 0; parity ^= 1; }
      }
      if (!ok) break;
      umma_commit_lead(leader, &acc_full[acc]);
    }
  } else {
    // ---------------- epilogue warps ----------------
    const int quarter = warp & 3;
    const bool gated = g.act == I8_GATED;
    pdl_wait();
    for (int t = int(threadIdx.x) - 64; t < BN; t += EPI) sx[t] = t < g.tokens ? g.sx[t] : 0.f;
    asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
    const int n_acc = min(NACC, p.k_stages * STEPS);
    if constexpr (KS > 1) {
      constexpr int MINE = TOK / KS;  // tokens this warp finishes: the slices' sums are exchanged, then each warp takes a share
      const int m = unit0 * IS_UNIT + lane;
      const bool m_ok = m < g.features;
      const float sw = m_ok ? g.sw[m] : 0.f;
      const float bias = (g.bias && m_ok) ? __bfloat162float(g.bias[m]) : 0.f;
      float res[MINE];
      i8_residual(g, res, quarter * MINE, m);
      const bool ready = !*abort_flag && mbar_wait(&acc_full[0], 0);
      if (!ready) give_up();
      tc_fence_after();
      if (__all_sync(0xffffffffu, ready)) {
        // this warp's TMEM lanes are the 32 rows of slice `quarter`; its columns of the product are [TOK quarter, TOK quarter + TOK)
        int v[TOK];
#pragma unroll
        for (int j = 0; j < TOK; ++j) v[j] = 0;
        for (int a = 0; a < n_acc; ++a) {
          uint32_t r[16];  // (TOK = 8: the upper half belongs to the next slice, or to the next accumulator; it is not used)
          tmem_ld_x16(tmem_base + (uint32_t(quarter * 32) << 16) + a * BN + quarter * TOK, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < TOK; ++j) v[j] += int(r[j]);
        }
#pragma unroll
        for (int j = 0; j < TOK; ++j) slices[(quarter * 32 + lane) * (TOK + 1) + j] = v[j];
      }
      asm volatile("bar.sync 1, %0;" ::"n"(EPI) : "memory");
      if (!*abort_flag) {
        int sum[MINE];
#pragma unroll
        for (int j = 0; j < MINE; ++j) {
          sum[j] = 0;
#pragma unroll
          for (int sl = 0; sl < KS; ++sl) sum[j] += slices[(sl * 32 + lane) * (TOK + 1) + quarter * MINE + j];
        }
        i8_finish(g, sum, sx + quarter * MINE, quarter * MINE, m, m_ok, sw, bias, res);
      }
    } else {
      constexpr int SHARE = BN / (EPI / 128);  // tokens of this warp
      const int first = (warp - 2) / 4 * SHARE;
      for (int pass = 0; pass < passes; ++pass) {
        const int acc = pass & 1, rows = pass_units(pass) * IS_UNIT;
        const bool m64 = rows <= 64 && !gated;
        // TMEM lane -> row of the pass: lane for M = 128; with M = 64 the first 16 lanes of each quarter hold 16 rows
        const int local_row = m64 ? quarter * 16 + lane : quarter * 32 + lane;
        const int m = pass_start(pass) * IS_UNIT + local_row;
        const bool m_ok = local_row < rows && (!m64 || lane < 16) && m < g.features;
        // fetched while the weights are still streaming: a load behind the accumulators would add a full round trip
        const float sw = m_ok ? g.sw[m] : 0.f;
        const float bias = (g.bias && m_ok) ? __bfloat162float(g.bias[m]) : 0.f;
        float res[SHARE];
        i8_residual(g, res, first, m);
        const bool ready = !*abort_flag && mbar_wait(&acc_full[acc], (pass >> 1) & 1);
        if (!__all_sync(0xffffffffu, ready)) {
          if (lane == 0) give_up();
          break;
        }
        tc_fence_after();
        const uint32_t t_lane = tmem_base + (uint32_t(quarter * 32) << 16) + acc * ACC_COLS;
#pragma unroll
        for (int n0 = first; n0 < first + SHARE; n0 += 16) {
          if (n0 >= g.tokens) break;
          int v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0;
          __syncwarp();
#pragma unroll 1
          for (int a = 0; a < n_acc; ++a) {
            uint32_t r[16];
            tmem_ld_x16(t_lane + a * BN + n0, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += int(r[j]);
          }
          i8_finish(g, v, sx + n0, n0, m, m_ok, sw, bias, res + (n0 - first));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

template <int BN, int NACC, int KBOX, int KS>
static int is_launch(const I8Gemm& g, int sms, cudaStream_t stream) {
  IsParams p;
  memset(&p, 0, sizeof(p));
  p.g = g;
  p.k_stages = ((g.k + KS - 1) / KS + KBOX * I8_BK - 1) / (KBOX * I8_BK);  // (of a slice)
  p.slice_cols = p.k_stages * KBOX * I8_BK;
  p.rows = gemm_stream_rows(g.features, sms);
  const size_t w_box = size_t(KS > 1 ? KS : p.rows.pass_units) * IS_UNIT * 128;
  const size_t stage_bytes = size_t(KBOX) * (w_box + BN * I8_BK);
  // an MMA of M = 64 / 128 rows reads that many rows from the last weight box of the ring: what lies behind the last token box
  const size_t need = size_t(128) * 128, have = w_box + size_t(KBOX) * BN * I8_BK;
  const size_t over = need > have ? need - have : 0;
  int stages = int(IS_RING_BYTES / stage_bytes);
  if (stages > IS_MAX_STAGES) stages = IS_MAX_STAGES;
  p.stages = stages;
  const size_t smem = 1024 + IS_CONTROL + IS_SLICE_BYTES(KS) + stages * stage_bytes + over;
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(gemm_i8_stream_kernel<BN, NACC, KBOX, KS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return TPB_ERR_CUDA;
    configured[dev].store(true, std::memory_order_release);
  }
  CUtensorMap tw, tw1, tx;
  int rc = i8_tmap(&tw, g.w, g.features, g.k, g.ldw, p.rows.box_units * IS_UNIT);
  if (rc == TPB_OK) rc = i8_tmap(&tw1, g.w, g.features, g.k, g.ldw, IS_UNIT);
  if (rc == TPB_OK) rc = i8_tmap(&tx, g.x, g.tokens, g.k, g.ldx, BN / KS);
  if (rc != TPB_OK) return rc;
  return launch_dependent(gemm_i8_stream_kernel<BN, NACC, KBOX, KS>, dim3(p.rows.grid), dim3(64 + IS_EPI(BN, KS)), smem, stream, true, tw, tw1, tx, p) == cudaSuccess
             ? TPB_OK
             : TPB_ERR_CUDA;
}

static int is_pick(const I8Gemm& g, int sms, cudaStream_t stream) {
  // one unit per CTA: slices of the contraction side by side, as long as each has a few stages
  const bool one_unit = (g.features + IS_UNIT - 1) / IS_UNIT <= sms && g.k >= 2048;
  if (one_unit && g.tokens <= 8) return is_launch<32, 4, 2, 4>(g, sms, stream);
  if (one_unit && g.tokens <= 16) return is_launch<64, 2, 2, 4>(g, sms, stream);
  if (g.tokens <= 16) return is_launch<16, 8, 2, 1>(g, sms, stream);
  if (g.tokens <= 32) return is_launch<32, 8, 2, 1>(g, sms, stream);
  if (g.tokens <= 64) return is_launch<64, 2, 2, 1>(g, sms, stream);
  return TPB_ERR_ARG;
}

// More rows than a launch counts (310 million on 148 SMs) go by several.
int gemm_i8_stream_launch(const I8Gemm& g, int sms, cudaStream_t stream) {
  const long long most = StreamRows::most_rows(sms);
  int rc = TPB_OK;
  for (long long f = 0; f < g.features && rc == TPB_OK; f += most) {
    I8Gemm part = g;
    part.features = int(g.features - f < most ? g.features - f : most);
    part.w += f * g.ldw;
    part.sw += f;
    part.out += g.act == I8_GATED ? f / 2 : f;
    if (g.bias) part.bias += f;
    if (g.residual) part.residual += f;
    rc = is_pick(part, sms, stream);
  }
  return rc;
}

cudaError_t gemm_i8_stream_preload() {
  cudaFuncAttributes attr;
  cudaError_t e = cudaSuccess;
#define LOAD(BN, NACC, KBOX, KS) if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, gemm_i8_stream_kernel<BN, NACC, KBOX, KS>)
  LOAD(32, 4, 2, 4); LOAD(64, 2, 2, 4); LOAD(16, 8, 2, 1); LOAD(32, 8, 2, 1); LOAD(64, 2, 2, 1);
#undef LOAD
  return e;
}

}  // namespace tpb

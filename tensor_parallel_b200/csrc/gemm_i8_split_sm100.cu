// Product of 8-bit integers for a middling number of tokens, up to about a thousand, or a small weight: see gemm_i8.cuh.
//
// A tile is 128 features (the lanes of TMEM) x BN tokens, and the CTAs of a cluster of S share its contraction: there are too few tiles to occupy
// the SMs, and each SM can only bring in so many bytes per clock.  Every CTA accumulates its range of k-blocks, then hands the partial sums of each
// S-th of the tokens to the CTA that finishes them, through distributed shared memory.  The sums are integers: their order does not matter, and
// no workspace in global memory is needed that calls or captured graphs would share.
//
// One CTA (320 threads): warp 0 = TMA producer, warp 1 = MMA issuer, warps 2-9 = epilogue (two per quarter of the lanes, each with half of the tokens).
// Every mbarrier wait is bounded; on expiry the CTA records a status code and goes on through the barriers of the cluster, which every thread reaches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>

#include "gemm_i8.cuh"
#include "launch.cuh"
#include "ptx_sm100.cuh"
#include "tpb_api.h"

namespace tpb {

constexpr int IX_THREADS = 320;
constexpr int IX_MAX_STAGES = 10;
constexpr size_t IX_RING_BYTES = 204 * 1024;

struct IxParams {
  I8Gemm g;
  int k_blocks, m_tiles, stages;
};

__device__ __forceinline__ void ix_store_remote(uint32_t cluster_addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <int N> __device__ __forceinline__ void ix_tmem_ld(uint32_t taddr, uint32_t (&r)[N]);
template <> __device__ __forceinline__ void ix_tmem_ld<16>(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_x16(taddr, r); }
template <> __device__ __forceinline__ void ix_tmem_ld<8>(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
template <> __device__ __forceinline__ void ix_tmem_ld<4>(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
}

template <int BN, int S>
__global__ void __launch_bounds__(IX_THREADS, 1)
gemm_i8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const IxParams p) {
  constexpr uint32_t W_BYTES = 128 * I8_BK, X_BYTES = BN * I8_BK, STAGE_BYTES = W_BYTES + X_BYTES;
  constexpr uint32_t TMEM_COLS = BN;
  constexpr int TS = BN / S;                        // tokens that a CTA finishes
  constexpr int HALF = TS / 2;                      // of which one of the two warps of a quarter takes
  constexpr int C = HALF < 16 ? HALF : 16;          // at a time
  static_assert(C >= 4 && (C & (C - 1)) == 0, "tokens of a step");
  const I8Gemm& g = p.g;
  extern __shared__ uint8_t ix_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ix_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty_bar = full_bar + IX_MAX_STAGES;
  uint64_t* acc_full = empty_bar + IX_MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float* sx = reinterpret_cast<float*>(smem + 256);  // [TS] scales of the tokens that this CTA finishes
  uint8_t* ring = smem + 1024;                       // later: [S sources][TS / 4][128 features][4 tokens] partial sums

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = S > 1 ? int(cluster_rank()) : 0;
  const int tile = blockIdx.x / S, m0 = (tile % p.m_tiles) * 128, t0 = (tile / p.m_tiles) * BN;
  const int kb0 = int((long long)p.k_blocks * rank / S), kbs = int((long long)p.k_blocks * (rank + 1) / S) - kb0;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(acc_full, 1);
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

  bool ready = false;
  const int quarter = warp & 3, half = warp >= 2 ? (warp - 2) >> 2 : 0;
  const int m = m0 + quarter * 32 + lane, mine = rank * TS + half * HALF;  // this thread's feature; first column of its tokens
  const bool m_ok = m < g.features;
  constexpr int AHEAD = HALF <= 32 ? HALF : C;      // tokens whose residual is fetched while the weights stream
  float sw = 0.f, bias = 0.f, res[AHEAD];
  if (warp == 0) {
    // ---------------- TMA producer (the warp stays together, one lane issues) ----------------
    const uint32_t leader = elect_one();
    auto load_w = [&](int n, int s) {
      mbar_expect_tx_lead(leader, &full_bar[s], STAGE_BYTES);
      tma_load_2d_lead(leader, smem_u32(ring + size_t(s) * STAGE_BYTES), &tmap_w, &full_bar[s], (kb0 + n) * I8_BK, m0);
    };
    auto load_x = [&](int n, int s) {
      tma_load_2d_lead(leader, smem_u32(ring + size_t(s) * STAGE_BYTES) + W_BYTES, &tmap_x, &full_bar[s], (kb0 + n) * I8_BK, t0);
    };
    const int ahead = min(kbs, p.stages);
    for (int n = 0; n < ahead; ++n) load_w(n, n);
    pdl_wait();
    pdl_trigger();
    for (int n = 0; n < ahead; ++n) load_x(n, n);
    int s = 0;
    uint32_t parity = 0;
    for (int n = ahead; n < kbs; ++n) {
      const bool free_stage = !*abort_flag && mbar_wait(&empty_bar[s], parity);
      if (!__all_sync(0xffffffffu, free_stage)) {
        if (leader) give_up();
        break;
      }
      load_w(n, s);
      load_x(n, s);
      if (++s == p.stages) { s = 0; parity ^= 1; }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the warp stays together, one lane issues) ----------------
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc = make_idesc_i8(128, BN);
    int s = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (int n = 0; n < kbs; ++n) {
      const bool full = !*abort_flag && mbar_wait(&full_bar[s], parity);
      if (!__all_sync(0xffffffffu, full)) {
        if (leader) give_up();
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t w_addr = smem_u32(ring + size_t(s) * STAGE_BYTES);
      const uint32_t w_lo = desc_kmajor_lo(w_addr), x_lo = desc_kmajor_lo(w_addr + W_BYTES);
#pragma unroll
      for (int kk = 0; kk < I8_BK / 32; ++kk) umma_i8_lead(leader, tmem_base, w_lo + kk * 2, x_lo + kk * 2, idesc, (n | kk) ? 1u : 0u);
      umma_commit_lead(leader, &empty_bar[s]);
      if (++s == p.stages) { s = 0; parity ^= 1; }
    }
    if (ok) umma_commit_lead(leader, acc_full);
  } else {
    // ---------------- epilogue warps ----------------
    pdl_wait();
    const int i = int(threadIdx.x) - 64;
    if (i < TS) sx[i] = t0 + rank * TS + i < g.tokens ? g.sx[t0 + rank * TS + i] : 0.f;
    if (m_ok) {
      sw = g.sw[m];
      if (g.bias) bias = __bfloat162float(g.bias[m]);
    }
    i8_residual(g, res, t0 + mine, m);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    ready = !*abort_flag && mbar_wait(acc_full, 0);
    ready = __all_sync(0xffffffffu, ready);
    if (!ready && lane == 0) give_up();
    tc_fence_after();
  }
  const uint32_t t_lane = tmem_base + (uint32_t(quarter * 32) << 16);
  const int* part = reinterpret_cast<const int*>(ring);
  auto sums = [&](int col, int (&sum)[C]) {  // of this CTA's k-blocks, for C tokens
    uint32_t r[C];
    ix_tmem_ld<C>(t_lane + col, r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < C; ++j) sum[j] = int(r[j]);
  };
  if constexpr (S > 1) {
    __syncwarp();
    cluster_sync_all();  // the products of every CTA are complete: the rings may take the partial sums
    if (ready) {
      const uint32_t at = smem_u32(ring) + ((rank * (TS / 4) + half * (HALF / 4)) * 128 + quarter * 32 + lane) * 16;
#pragma unroll 1
      for (int d = 1; d < S; ++d) {
        const int to = (rank + d) % S;
        const uint32_t remote = mapa_u32(at, to);
#pragma unroll 1
        for (int c = 0; c < HALF; c += C) {
          int r[C];
          sums(to * TS + half * HALF + c, r);
#pragma unroll
          for (int j = 0; j < C; j += 4) ix_store_remote(remote + (c + j) / 4 * 128 * 16, r[j], r[j + 1], r[j + 2], r[j + 3]);
        }
      }
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (ready && !*abort_flag) {
#pragma unroll
    for (int c = 0; c < HALF; c += C) {
      if (t0 + mine + c >= g.tokens) break;
      if (AHEAD < HALF && c > 0) i8_residual(g, res, t0 + mine + c, m);
      int sum[C];
      sums(mine + c, sum);
      if constexpr (S > 1) {
#pragma unroll
        for (int d = 1; d < S; ++d) {
          const int from = (rank + d) % S;
#pragma unroll
          for (int j = 0; j < C; j += 4) {
            const int4 q = *reinterpret_cast<const int4*>(part + ((from * (TS / 4) + (half * HALF + c + j) / 4) * 128 + quarter * 32 + lane) * 4);
            sum[j] += q.x;
            sum[j + 1] += q.y;
            sum[j + 2] += q.z;
            sum[j + 3] += q.w;
          }
        }
      }
      i8_finish(g, sum, sx + half * HALF + c, t0 + mine + c, m, m_ok, sw, bias, AHEAD < HALF ? res : res + c);
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

template <int BN, int S>
static int ix_launch(const I8Gemm& g, cudaStream_t stream) {
  constexpr size_t STAGE_BYTES = (128 + BN) * I8_BK;
  static_assert(size_t(BN) * 512 <= 4 * STAGE_BYTES, "room for partial sums");
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(gemm_i8_split_kernel<BN, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return TPB_ERR_CUDA;
    configured[dev].store(true, std::memory_order_release);
  }
  IxParams p;
  memset(&p, 0, sizeof(p));
  p.g = g;
  p.k_blocks = (g.k + I8_BK - 1) / I8_BK;
  p.m_tiles = (g.features + 127) / 128;
  p.stages = int(IX_RING_BYTES / STAGE_BYTES);
  if (p.stages > IX_MAX_STAGES) p.stages = IX_MAX_STAGES;
  CUtensorMap tw, tx;
  int rc = i8_tmap(&tw, g.w, g.features, g.k, g.ldw, 128);
  if (rc == TPB_OK) rc = i8_tmap(&tx, g.x, g.tokens, g.k, g.ldx, BN);
  if (rc != TPB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.m_tiles) * ((g.tokens + BN - 1) / BN) * S);
  cfg.blockDim = dim3(IX_THREADS);
  cfg.dynamicSmemBytes = 2048 + p.stages * STAGE_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, gemm_i8_split_kernel<BN, S>, tw, tx, p) == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

// Where this kernel pays, from sweeps over 1 to 1024 tokens and sizes from 256 x 1024 to 22016 x 4096 (us; stream / pair / this):
//   1 x 4096 x 1024     4.5 / - / 3.9         1 x 2048 x 512     3.0 / - / 2.8         1 x 5120 x 8192     14.6 / - / 11.5     8 x 4096 x 4096   5.5 / - / 6.9
//   1 x 8192 x 4096     10.3 / - / 9.6        16 x 12288 x 4096  12.2 / - / 12.4       17 x 4096 x 4096    11.4 / 13.1 / 8.3   17 x 768 x 4096   10.7 / 10.5 / 5.9
//   64 x 4096 x 4096    11.1 / 11.7 / 9.0     64 x 4096 x 11008  19.8 / 20.9 / 13.8    64 x 22016 x 4096   21.9 / 26.7 / 28.1
//   100 x 4096 x 11008  - / 21.7 / 15.3       100 x 2999 x 1001  - / 10.8 / 6.5        100 x 12288 x 4096  - / 15.9 / 15.0
//   257 x 2999 x 1001   - / 11.1 / 8.0        256 x 4096 x 1024  - / 7.9 / 7.7         1024 x 1024 x 1024  - / 7.2 / 7.0
//   256 x 4096 x 11008  - / 22.1 / 18.6       256 x 4096 x 4096  - / 12.4 / 12.1       300 x 12288 x 4096  - / 22.6 / 30.2
// A tile takes as many CTAs as there are idle SMs, two k-blocks each at least (clusters of 8 find room in a GPU's groups of SMs up to about 96 CTAs, of 4 up to
// 128).  Up to 16 tokens the streaming kernel is ahead where it can cut long rows into slices itself, one unit of rows per CTA.
bool gemm_i8_split_pick(int tokens, int features, int k, int sms, int* bn, int* splits) {
  const int k_blocks = (k + I8_BK - 1) / I8_BK;
  auto tiles = [&](int n) { return (long long)((features + 127) / 128) * ((tokens + n - 1) / n); };
  auto most = [&](int n) {
    int s = 1;
    for (int c = 2; c <= 8; c *= 2)
      if (tiles(n) * c <= (c == 8 ? sms * 96 / 148 : c == 4 ? sms * 128 / 148 : sms) && 2 * c <= k_blocks && n / c >= 8) s = c;
    return s;
  };
  *bn = tokens <= 32 ? 32 : 64;
  *splits = most(*bn);
  if (tokens <= 16) return k_blocks < 16 ? tiles(32) * (k_blocks <= 4 ? 1 : 2) <= sms : (features + 31) / 32 > sms && tiles(32) * 2 <= sms;
  if (tokens <= 64) return tiles(*bn) <= sms;
  if (*splits > 1 || (k_blocks < 16 && tiles(64) <= sms)) return true;
  *bn = 128;
  *splits = most(128);
  return *splits > 1 ? k_blocks >= 16 : tokens <= 128 && tiles(128) <= sms;
}

#define IX_FORMS(GO) GO(32, 1) GO(32, 2) GO(32, 4) GO(64, 1) GO(64, 2) GO(64, 4) GO(64, 8) GO(128, 1) GO(128, 2)
int gemm_i8_split_launch(const I8Gemm& g, int bn, int splits, cudaStream_t stream) {
#define GO(BN, S) if (bn == BN && splits == S) return ix_launch<BN, S>(g, stream);
  IX_FORMS(GO)
#undef GO
  return TPB_ERR_ARG;
}

cudaError_t gemm_i8_split_preload() {
  cudaFuncAttributes attr;
  cudaError_t e = cudaSuccess;
#define LOAD(BN, S) if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, gemm_i8_split_kernel<BN, S>);
  IX_FORMS(LOAD)
#undef LOAD
  return e;
}

}  // namespace tpb

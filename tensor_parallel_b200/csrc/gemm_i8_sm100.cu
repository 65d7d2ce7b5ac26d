// Product of 8-bit integers: the entry point, and the kernel for many tokens on CTA pairs (see gemm_i8.cuh; few tokens: gemm_i8_stream_sm100.cu).
//
// The decomposition is that of the bf16 kernel (gemm_pair_sm100.cu): two CTAs on neighbouring SMs work on one tile of 256 tokens x BN features with
// tcgen05.mma.cta_group::2, each loads 128 token rows and BN / 2 feature rows, the leader issues for both.  A k-block is 128 bytes of every row there
// and here: 128 columns, 512 clocks of the tensor core at BN = 256.  Sums are 32-bit integers, the epilogue scales them.
//
// Measured (us, of twice the bf16 rate of a library product in short runs, 1647 TFLOP/s): 2048 x 11008 x 4096 63.0 (0.89, tensor pipe busy for 0.81 at
// 1.64 GHz), 4000 x 12288 x 4096 136 (0.90), 8192 x 22016 x 4096 gated 440 (1.02); in long runs the power limit bounds them.  About 5 to 7 us of a call
// are prologue, first bytes and the last epilogue.
//
// One CTA (320 threads), persistent over the pair's tiles:
//   warp 0    : TMA producer of this CTA's operand rows; completion is counted on the LEADER's barrier (no multicast)
//   warp 1    : leader only: one thread issues the MMAs; the commits signal the barriers of both CTAs
//   warps 2-9 : epilogue of this CTA's 128 rows, two TMEM accumulators so that it runs under the next tile's MMAs
// Every mbarrier wait is bounded; on expiry the CTA records a status code and drains.
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

constexpr int I8_MAX_K = 131071;  // rows of -128 that long sum up to 2^31 - 2^14
constexpr int I8_MAX_ROWS = 0x7fffffff - 511;  // (rows of the last tile are counted in 32 bits)
constexpr int IP_BM = 256;        // tokens of a pair tile (128 per CTA = TMEM lanes)
constexpr int IP_EPI_WARPS = 8;   // two per quarter of the TMEM lanes: one for each half of the columns
constexpr int IP_THREADS = 64 + 32 * IP_EPI_WARPS;
constexpr int IP_MAX_STAGES = 8;
constexpr int IP_BAND = 8;        // tiles are walked in bands of 8 token tiles x all feature tiles

constexpr int IP_TURN_PITCH = 17; // 16 columns of a chunk, turned in shared memory

struct IpParams {
  I8Gemm g;
  int k_blocks, m_tiles, n_tiles;
};

template <int BN>
struct IpShape {
  static constexpr int STAGES = BN > 192 ? 6 : BN > 128 ? 7 : 8;
  static constexpr int ACC_COLS = BN > 128 ? 256 : 128;  // TMEM columns of an accumulator
  static constexpr int SPLIT = (BN / 2 + 31) / 32 * 32;  // columns that the first epilogue warp of a quarter takes
  static constexpr uint32_t A_BYTES = 128 * I8_BK;
  static constexpr uint32_t B_BYTES = BN / 2 * I8_BK;
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr size_t PARAM_BYTES = 2 * 2 * BN * sizeof(float);                         // scales and biases of the features of two tiles
  static constexpr size_t TURN_BYTES = size_t(IP_EPI_WARPS) * 32 * IP_TURN_PITCH * sizeof(float);  // where rows of `out` are not aligned
  static constexpr size_t SMEM = size_t(STAGES) * STAGE_BYTES + 1024 /*align*/ + PARAM_BYTES + TURN_BYTES + (2 * IP_MAX_STAGES + 4) * 8 + 16;
};

template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(IP_THREADS, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const IpParams p) {
  using S = IpShape<BN>;
  constexpr uint32_t TMEM_COLS = 2 * S::ACC_COLS;
  const I8Gemm& g = p.g;
  extern __shared__ uint8_t ip_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ip_smem_raw) + 1023) & ~uintptr_t(1023));
  float* params = reinterpret_cast<float*>(smem + size_t(S::STAGES) * S::STAGE_BYTES);  // [2 tiles][scales, biases][BN]
  float* turn = params + S::PARAM_BYTES / sizeof(float);                               // [epilogue warp][32 tokens][IP_TURN_PITCH]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(turn + S::TURN_BYTES / sizeof(float));  // used in the leader
  uint64_t* empty_bar = full_bar + IP_MAX_STAGES;
  uint64_t* acc_full = empty_bar + IP_MAX_STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;              // [2], used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();  // 0 = leader
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.m_tiles * p.n_tiles;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * IP_EPI_WARPS);  // one arrival per epilogue warp of either CTA
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  auto tile_at = [&](int t, int& mt, int& nt) {
    const int band = t / (IP_BAND * p.n_tiles), r = t - band * IP_BAND * p.n_tiles;
    const int rows = min(IP_BAND, p.m_tiles - band * IP_BAND);
    mt = band * IP_BAND + r % rows;
    nt = r / rows;
  };
  auto give_up = [&]() {
    atomicMax(g.status, STATUS_TIMEOUT_MBAR);
    *abort_flag = 1;
  };

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        int mt, nt;
        tile_at(t, mt, nt);
        const int m0 = mt * IP_BM + int(rank) * 128, n0 = nt * BN + int(rank) * (BN / 2);
        for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
          const int s = it % S::STAGES;
          if (*abort_flag || !mbar_wait(&empty_bar[s], ((it / S::STAGES) & 1) ^ 1)) {
            give_up();
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + size_t(s) * S::STAGE_BYTES;
          const uint32_t bar = mapa_u32(smem_u32(&full_bar[s]), 0);
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * S::STAGE_BYTES);  // both CTAs' bytes
          tma_load_2d_pair(a_dst, &tmap_a, bar, kb * I8_BK, m0);
          tma_load_2d_pair(a_dst + S::A_BYTES, &tmap_b, bar, kb * I8_BK, n0);
        }
      }
      // the leader's last commits still arrive on this CTA's barriers: stay until each used stage has been released
      for (uint32_t i = it > uint32_t(S::STAGES) ? it - S::STAGES : 0; ok && i < it; ++i) {
        if (!mbar_wait(&empty_bar[i % S::STAGES], (i / S::STAGES) & 1)) {
          give_up();
          ok = false;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = make_idesc_i8(IP_BM, BN);
      uint32_t it = 0, local = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs, ++local) {
        const int acc = local & 1;
        if (*abort_flag || !mbar_wait(&acc_empty[acc], ((local >> 1) & 1) ^ 1)) {
          give_up();
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * S::ACC_COLS;
        for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
          const int s = it % S::STAGES;
          if (!mbar_wait(&full_bar[s], (it / S::STAGES) & 1)) {
            give_up();
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + size_t(s) * S::STAGE_BYTES), b_addr = a_addr + S::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < I8_BK / 32; ++kk)
            umma_i8_pair(d_tmem, make_desc_kmajor_sw128(a_addr + kk * 32), make_desc_kmajor_sw128(b_addr + kk * 32), idesc, (kb | kk) ? 1u : 0u);
          umma_commit_pair(&empty_bar[s]);
        }
        if (ok) umma_commit_pair(&acc_full[acc]);
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lane quarter this warp may access
    const int half = (warp - 2) >> 2, col0 = half * S::SPLIT, col1 = half ? BN : S::SPLIT;
    const uint32_t acc_empty_leader[2] = {mapa_u32(smem_u32(&acc_empty[0]), 0), mapa_u32(smem_u32(&acc_empty[1]), 0)};
    const bool gated = g.act == I8_GATED;
    auto aligned = [](const void* ptr, long long ld) { return !(reinterpret_cast<uintptr_t>(ptr) & 15) && (ld & 7) == 0; };
    const bool vec = aligned(g.out, g.ld_out) && (!g.residual || aligned(g.residual, g.ld_res));
    const bool sectors = vec && (g.ld_out & 15) == 0 && !(reinterpret_cast<uintptr_t>(g.out) & 31);
    float* mine = turn + (warp - 2) * 32 * IP_TURN_PITCH;
    bool gone = false;  // given up: on to the end without waits, through the barriers that the epilogue warps share
    uint32_t local = 0;
    for (int t = pair; t < tiles; t += pairs, ++local) {
      int mt, nt;
      tile_at(t, mt, nt);
      const int m0 = mt * IP_BM + int(rank) * 128 + quarter * 32, m = m0 + lane;
      const int acc = local & 1;
      float* sws = params + acc * 2 * BN;
      const float* biases = sws + BN;
      // (every warp has read what the tile before the last left there: it has passed the last tile's barrier)
      for (int c = int(threadIdx.x) - 64; c < 2 * BN; c += 32 * IP_EPI_WARPS) {
        const int f = nt * BN + (c < BN ? c : c - BN);
        sws[c] = f >= g.features ? 0.f : c < BN ? g.sw[f] : g.bias ? __bfloat162float(g.bias[f]) : 0.f;
      }
      const float sx = m < g.tokens ? g.sx[m] : 0.f;
      // the residual of a chunk, a chunk ahead
      uint4 res[4];
      auto fetch = [&](int c0) {
        const int n0 = nt * BN + c0;
        if (!g.residual || !vec || c0 >= col1 || n0 + 32 > g.features || m >= g.tokens) return;
        const uint4* rp = reinterpret_cast<const uint4*>(g.residual + m * g.ld_res + n0);
#pragma unroll
        for (int q = 0; q < 4; ++q) res[q] = rp[q];
      };
      // of half a chunk, where it leaves through shared memory: rows lane / 16, + 2, .. of one column (addresses past the end are drawn back, see i8_residual)
      uint16_t turned[16];
      auto fetch_turned = [&](int c) {
        if (!g.residual || nt * BN + c >= g.features) return;
        const uint16_t* rp = reinterpret_cast<const uint16_t*>(g.residual) + min(nt * BN + c + (lane & 15), g.features - 1);
#pragma unroll
        for (int i = 0; i < 16; ++i) turned[i] = rp[min(m0 + (lane >> 4) + 2 * i, g.tokens - 1) * g.ld_res];
      };
      if (vec) fetch(col0);
      else fetch_turned(col0);
      asm volatile("bar.sync 1, %0;" ::"n"(32 * IP_EPI_WARPS) : "memory");
      const bool ready = !*abort_flag && mbar_wait(&acc_full[acc], (local >> 1) & 1);
      if (!__all_sync(0xffffffffu, ready)) {
        if (lane == 0) give_up();
        gone = true;
      }
      tc_fence_after();
      const uint32_t t_lane = tmem_base + (uint32_t(quarter * 32) << 16) + acc * S::ACC_COLS;
      // Both accumulator halves may be overwritten after all of these.  Nothing but the tcgen05 loads, which have completed, has to come before (a release would
      // wait for the stores, about 1 us), and only a tile that waits for it is told, so that no arrival is on its way to a CTA that has left.
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && t + 2 * pairs < tiles) mbar_arrive_cluster_relaxed(acc_empty_leader[acc]);
      };
#pragma unroll 1
      for (int c0 = col0; c0 < col1; c0 += 32) {
        const int n0 = nt * BN + c0;
        if (gone || n0 >= g.features) break;
        uint32_t r[32];
        __syncwarp();
        tmem_ld_x32(t_lane + c0, r);
        tmem_ld_wait();
        if (c0 + 32 >= col1 || n0 + 32 >= g.features) release();
        float v[32];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float4 s = *reinterpret_cast<const float4*>(sws + c0 + 4 * q), b = *reinterpret_cast<const float4*>(biases + c0 + 4 * q);
          v[4 * q] = i8_value(int(r[4 * q]), sx, s.x, b.x);
          v[4 * q + 1] = i8_value(int(r[4 * q + 1]), sx, s.y, b.y);
          v[4 * q + 2] = i8_value(int(r[4 * q + 2]), sx, s.z, b.z);
          v[4 * q + 3] = i8_value(int(r[4 * q + 3]), sx, s.w, b.w);
        }
        if (gated) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = i8_gate(v[j], v[j]) * v[16 + j];
        } else {
          i8_activate(v, g.act);
        }
        const int cols = gated ? 16 : 32, at = gated ? n0 >> 1 : n0;  // output columns of the chunk
        if (vec && n0 + 32 <= g.features) {
          if (m >= g.tokens) continue;
          __nv_bfloat16* out = g.out + m * g.ld_out + at;
          if (g.residual) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t rw[4] = {res[q].x, res[q].y, res[q].z, res[q].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                v[8 * q + 2 * j] += bf16_bits_to_float(rw[j] & 0xFFFF);
                v[8 * q + 2 * j + 1] += bf16_bits_to_float(rw[j] >> 16);
              }
            }
          }
          fetch(c0 + 32);
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
          if (sectors) {  // whole 32-byte sectors
            st_global_v8(out, w);
            if (!gated) st_global_v8(out + 16, w + 8);
          } else {
            uint4* op = reinterpret_cast<uint4*>(out);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (q < 2 || !gated) op[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
          }
        } else {
          // 16 columns at a time through shared memory, so that neighbouring lanes store neighbouring columns
          const int last = gated ? g.features >> 1 : g.features;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (16 * h >= cols) break;
            if (vec) fetch_turned(c0 + 16 * h);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) mine[lane * IP_TURN_PITCH + j] = v[16 * h + j];
            __syncwarp();
            const int c = at + 16 * h + (lane & 15);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int row = (lane >> 4) + 2 * i;
              float x = mine[row * IP_TURN_PITCH + (lane & 15)];
              if (g.residual) x += bf16_bits_to_float(turned[i]);
              if (m0 + row < g.tokens && c < last) g.out[(m0 + row) * g.ld_out + c] = __float2bfloat16(x);
            }
            if (!vec && c0 + 16 * h + 16 < col1) fetch_turned(c0 + 16 * h + 16);
          }
        }
      }
      if (!gone && nt * BN + col0 >= g.features) release();  // (nothing of the tile is this warp's)
    }
  }

  // both CTAs stay until nobody can touch the other's barriers or TMEM any more
  __syncwarp();
  tc_fence_before();
  cluster_meet();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem_base, TMEM_COLS);
}

template <int BN>
static int ip_launch(const I8Gemm& g, int sms, cudaStream_t stream) {
  using S = IpShape<BN>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TPB_ERR_CUDA;
  if (!configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(gemm_i8_pair_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::SMEM)) != cudaSuccess) return TPB_ERR_CUDA;
    configured[dev].store(true, std::memory_order_release);
  }
  CUtensorMap ta, tb;
  int rc = i8_tmap(&ta, g.x, g.tokens, g.k, g.ldx, 128);
  if (rc == TPB_OK) rc = i8_tmap(&tb, g.w, g.features, g.k, g.ldw, BN / 2);
  if (rc != TPB_OK) return rc;
  IpParams p;
  memset(&p, 0, sizeof(p));
  p.g = g;
  p.k_blocks = (g.k + I8_BK - 1) / I8_BK;
  p.m_tiles = (g.tokens + IP_BM - 1) / IP_BM;
  p.n_tiles = (g.features + BN - 1) / BN;
  const long long tiles = (long long)p.m_tiles * p.n_tiles;
  if (tiles > 0x7fffffffLL - sms) return TPB_ERR_SIZE;
  const int pairs = int(tiles < sms / 2 ? tiles : sms / 2);
  return launch_dependent(gemm_i8_pair_kernel<BN>, dim3(2 * pairs), dim3(IP_THREADS), S::SMEM, stream, true, ta, tb, p) == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

// Columns of the pair tile: the least rounds of tiles x clocks of a k-block, which is bound by the products at 256 columns and by what an SM gets from L2 at 128.
// A narrower tile has to win 4.5 %: it moves more bytes per product, which costs where the card is at its power limit.  us with 256 / 224 / 192 / 160 / 128 columns:
//   256 x 12288 x 4096 18.3 17.6 16.2 21.8 19.7    300 x 12288 x 4096 26.5 24.4 22.3 26.8 24.3     512 x 4096 x 4096 17.2 15.5 14.2 12.9 11.8
//   300 x 11008 x 4096 26.7 24.6 22.3 20.7 24.1    300 x 22016 x 4096 38.6 36.0 39.0 37.2 39.5     768 x 12288 x 4096 30.5 34.8 33.0 36.1 35.0
//   2048 x 12288 x 4096 74 71 74 80 86             2048 x 4096 x 11008 63 74 70 66 74              8192 x 22016 x 4096 (gated) 443 468 615 607 653
static int ip_tile(int tokens, int features, int sms) {
  struct Shape { int bn, clocks; };
  constexpr Shape SHAPES[] = {{256, 512}, {224, 450}, {192, 412}, {160, 365}, {128, 325}};
  int bn = 0;
  double least = 0;
  for (const Shape& shape : SHAPES) {
    const long long tiles = (long long)((tokens + IP_BM - 1) / IP_BM) * ((features + shape.bn - 1) / shape.bn);
    const double clocks = double((tiles + sms / 2 - 1) / (sms / 2)) * shape.clocks;
    if (bn && clocks * 1.045 >= least) continue;
    bn = shape.bn;
    least = clocks;
  }
  return bn;
}

// Results (or residuals) whose rows are not aligned leave a pair's tile 2 bytes at a time through shared memory, which costs about as much as 20 k-blocks: the shared
// contraction's kernel stores as fast as ever, tiles of 128 x 128, but brings in more per product (looked at up to three rounds of tiles).  us, pairs / 128 x 128: 150 x 6370 x 512 9.5 / 6.2, x 2048
// 11.2 / 8.7, x 6000 22.4 / 22.9; 600 x 6370 x 2048 (2 rounds of either) 22.9 / 17.8; 1000 x 3043 x 512 (1 / 2 rounds) 12.1 / 11.7, x 2048 14.9 / 17.0.
static bool ip_yields(int tokens, int features, int k, int sms) {
  const int bn = ip_tile(tokens, features, sms), k_blocks = (k + I8_BK - 1) / I8_BK;
  const long long pairs = (long long)((tokens + IP_BM - 1) / IP_BM) * ((features + bn - 1) / bn), tiles = (long long)((tokens + 127) / 128) * ((features + 127) / 128);
  const long long pair_rounds = (pairs + sms / 2 - 1) / (sms / 2), rounds = (tiles + sms - 1) / sms;
  return k_blocks < 32 && rounds <= 3 && rounds <= (k_blocks <= 4 ? 2 : 1) * pair_rounds;
}

#define IP_FORMS(GO) GO(128) GO(160) GO(192) GO(224) GO(256)

}  // namespace tpb

extern "C" int tpb_gemm_int8(const int8_t* x, const float* sx, const int8_t* w, const float* sw, void* out, const void* bias, const void* residual,
                             int tokens, int features, int k, long long ldx, long long ldw, long long ld_out, long long ld_res, int act, int early, void* status,
                             void* stream) {
  using bf16 = __nv_bfloat16;
  if (!x || !sx || !w || !sw || !out || !status || tokens <= 0 || features <= 0 || k <= 0 || act < 0 || act > tpb::I8_GATED) return TPB_ERR_ARG;
  if (k > tpb::I8_MAX_K || tokens > tpb::I8_MAX_ROWS || features > tpb::I8_MAX_ROWS) return TPB_ERR_SIZE;
  const int cols = act == tpb::I8_GATED ? features / 2 : features;
  if (act == tpb::I8_GATED && (features % 32 || residual)) return TPB_ERR_ARG;
  if (ldx < k || ldw < k || ld_out < cols || (residual && ld_res < cols)) return TPB_ERR_ARG;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) || ldx % 16 || ldw % 16) return TPB_ERR_ALIGN;
  if (((reinterpret_cast<uintptr_t>(sx) | reinterpret_cast<uintptr_t>(sw)) & 3) ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(residual)) & 1))
    return TPB_ERR_ALIGN;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return TPB_ERR_CUDA;
  const tpb::I8Gemm g = {x, w, sx, sw, static_cast<bf16*>(out), static_cast<const bf16*>(bias), static_cast<const bf16*>(residual), ldx, ldw, ld_out, ld_res,
                         tokens, features, k, act, early, static_cast<uint32_t*>(status)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int bn = 0, splits = 0;
  if (tpb::gemm_i8_split_pick(tokens, features, k, sms, &bn, &splits)) return tpb::gemm_i8_split_launch(g, bn, splits, s);
  if (tokens <= 64) return tpb::gemm_i8_stream_launch(g, sms, s);
  auto aligned = [](const void* p, long long ld) { return !(reinterpret_cast<uintptr_t>(p) & 15) && ld % 8 == 0; };
  if (!(aligned(out, ld_out) && (!residual || aligned(residual, ld_res))) && tpb::ip_yields(tokens, features, k, sms))
    return tpb::gemm_i8_split_launch(g, 128, 1, s);
  bn = tpb::ip_tile(tokens, features, sms);
#define GO(BN) if (bn == BN) return tpb::ip_launch<BN>(g, sms, s);
  IP_FORMS(GO)
#undef GO
  return TPB_ERR_ARG;
}

// The kernel that takes a product of these sizes (contiguous results, no activation that changes their number), for tests: 0 streaming, 1 shared contraction (form: tokens of a tile, CTAs that share it), 2 CTA pairs (columns
// of a tile).
extern "C" int tpb_gemm_int8_form(int tokens, int features, int k, int sms, int* form) {
  if (tokens <= 0 || features <= 0 || k <= 0 || k > tpb::I8_MAX_K || tokens > tpb::I8_MAX_ROWS || features > tpb::I8_MAX_ROWS || sms < 2 || !form) return -1;
  form[0] = form[1] = 0;
  if (tpb::gemm_i8_split_pick(tokens, features, k, sms, &form[0], &form[1])) return 1;
  if (tokens > 64 && features % 8 && tpb::ip_yields(tokens, features, k, sms)) {
    form[0] = 128;
    form[1] = 1;
    return 1;
  }
  form[1] = 0;
  form[0] = tokens <= 64 ? 0 : tpb::ip_tile(tokens, features, sms);
  return tokens <= 64 ? 0 : 2;
}

// Loads every kernel of the 8-bit operators on the current device: a single host thread that drives several GPUs does so before the first of them waits for a peer.
extern "C" int tpb_int8_preload(void) {
  cudaFuncAttributes attr;
  cudaError_t e = cudaSuccess;
#define LOAD(BN) if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, tpb::gemm_i8_pair_kernel<BN>);
  IP_FORMS(LOAD)
#undef LOAD
  if (e == cudaSuccess) e = tpb::gemm_i8_stream_preload();
  if (e == cudaSuccess) e = tpb::gemm_i8_split_preload();
  if (e == cudaSuccess) e = tpb::rows_int8_preload();
  return e == cudaSuccess ? TPB_OK : TPB_ERR_CUDA;
}

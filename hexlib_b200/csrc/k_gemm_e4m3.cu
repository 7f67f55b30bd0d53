// k_gemm_e4m3.cu -- out = act(a @ w + bias) (+ resid) for operands in their e4m3
// form (hb_e4m3.cuh), fp32 sums, one rounding to fp16.
//
// Codes and scales go to the tensor cores as they are: tcgen05.mma kind::mxf8f6f4
// multiplies 32 of K at a time and scales each product by the two rows' powers of
// two, so nothing is dequantized and no partial sum is rescaled on the CUDA cores.
// The hardware's scale granularity is 32; a block of 128 uses its byte four times.
//
// Scale bytes: a word of the form holds the bytes of four consecutive blocks (512 of
// K) of a row. The 128 words of a tile's rows are laid out as 32 rows of 16 bytes
// (row r at r % 32, word r / 32), which one tcgen05.cp brings to tensor memory where
// the MMA wants them; the instruction descriptor then picks the byte of the block.
#include <cuda.h>
#include <cuda_runtime.h>

#include "hb_device.cuh"
#include "hb_e4m3.cuh"
#include "hb_kernels.h"
#include "hb_tma.h"

namespace hb {
namespace {

constexpr int kBlockK = 128;          // bytes of K in a stage: one scale block
constexpr int kThreads = 256;

struct E4m3Params {
  const uint32_t* a_scales;   // [groups, M]
  const uint32_t* w_scales;   // [groups, N]
  const float* bias;
  const __half* resid;
  __half* out;
  int M, N, num_kb, act;
  int tiles_n;                // tiles of 128 features
  int* err;
};

__device__ __forceinline__ float finish(float v, int act) {
  if (act == 1) return gelu_tanh_f(v);
  if (act == 2) return gelu_erf_f(v);
  return v;
}

// ---- one tile per CTA, features by tokens --------------------------------------
//
// The tile is 128 FEATURES (rows of w, the MMA's M) by BN TOKENS (rows of a, its N):
// a few tokens then cost a narrow MMA and no padding to 128 rows, and in tensor
// memory a lane is a feature, so a warp stores 32 consecutive features of a token at
// any alignment of the output.
//
// A cluster of S CTAs shares a tile and splits K: with few tokens the time is that
// of reading w once, which takes all SMs. Each CTA leaves its partial tile in its
// shared memory, and CTA r adds up its BN / S tokens from all of them, in rank order.
template <int BN>
struct TileCfg {
  static constexpr int W_BYTES = 128 * kBlockK;
  static constexpr int A_BYTES = BN * kBlockK;
  static constexpr int STAGE_BYTES = W_BYTES + A_BYTES;
  static constexpr int STAGES = BN == 128 ? 3 : 4;
  static constexpr int SF_BYTES = 2 * 2 * 512;                    // two buffers of w and a
  static constexpr int TMEM_COLS = BN == 16 ? 32 : 2 * BN;        // accumulator + 16 of scales
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + SF_BYTES + 1024 + 256;
};

template <int BN>
__global__ void __launch_bounds__(kThreads)
    gemm_e4m3_tile(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                   const E4m3Params p, const int split) {
  using Cfg = TileCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sA = smem + Cfg::STAGES * Cfg::W_BYTES;
  uint8_t* sSF = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sSF + Cfg::SF_BYTES);
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* sf_full = empty + Cfg::STAGES;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* done = sf_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sf_full[b], 1);
      mbar_init(&sf_empty[b], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / split;
  const int n0 = (tile % p.tiles_n) * 128, m0 = (tile / p.tiles_n) * BN;
  // the blocks of K of this CTA (at least one: split <= num_kb)
  const int kb0 = (int)((int64_t)p.num_kb * rank / split);
  const int kb1 = (int)((int64_t)p.num_kb * (rank + 1) / split);

  if (warp == 0 && lane == 0) {
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, s = i % Cfg::STAGES;
      if (!mbar_wait(&empty[s], ((i / Cfg::STAGES) & 1) ^ 1, abort_flag, p.err)) break;
      mbar_arrive_expect_tx(&full[s], Cfg::STAGE_BYTES);
      tma_load_2d(&tmW, &full[s], sW + s * Cfg::W_BYTES, kb * kBlockK, n0);
      tma_load_2d(&tmA, &full[s], sA + s * Cfg::A_BYTES, kb * kBlockK, m0);
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_e4m3_scaled(128, BN);
    int u = 0;                                        // scale words used so far
    bool ok = true;
    for (int kb = kb0; kb < kb1 && ok; ++kb) {
      const int i = kb - kb0, s = i % Cfg::STAGES;
      const uint32_t sf = tmem + BN + (u & 1) * 8;
      if (i == 0 || (kb & 3) == 0) {
        ok = mbar_wait(&sf_full[u & 1], (u >> 1) & 1, abort_flag, p.err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t src = smem_u32(sSF + (u & 1) * 1024);
        tmem_copy_scales(sf, sdesc_rows16(src));
        tmem_copy_scales(sf + 4, sdesc_rows16(src + 512));
      }
      ok = mbar_wait(&full[s], (i / Cfg::STAGES) & 1, abort_flag, p.err);
      if (!ok) break;
      tc_fence_after();
      const uint32_t w0 = smem_u32(sW + s * Cfg::W_BYTES), a0 = smem_u32(sA + s * Cfg::A_BYTES);
      const uint32_t id = idesc_with_scale_byte(idesc, kb & 3);
#pragma unroll
      for (int kk = 0; kk < kBlockK / 32; ++kk)
        umma_e4m3_scaled(tmem, sdesc_sw128(w0 + kk * 32, 16, 1024),
                         sdesc_sw128(a0 + kk * 32, 16, 1024), id, sf, sf + 4, (i | kk) ? 1u : 0u);
      umma_commit(&empty[s]);
      if ((kb & 3) == 3 || kb + 1 == kb1) {
        umma_commit(&sf_empty[u & 1]);
        ++u;
      }
    }
    if (ok) umma_commit(done);
  } else if (warp == 2) {
    // scale words of 512 of K: row lane + 32 j of the tile to word j of row `lane`
    int u = 0;
    for (int g = kb0 >> 2; g <= (kb1 - 1) >> 2; ++g, ++u) {
      uint32_t w[4], a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = lane + 32 * j, n = n0 + r, m = m0 + r;
        w[j] = n < p.N ? __ldg(p.w_scales + (int64_t)g * p.N + n) : 0x7f7f7f7fu;
        a[j] = r < BN && m < p.M ? __ldg(p.a_scales + (int64_t)g * p.M + m) : 0x7f7f7f7fu;
      }
      const bool ok = mbar_wait(&sf_empty[u & 1], ((u >> 1) & 1) ^ 1, abort_flag, p.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      uint4* dst = reinterpret_cast<uint4*>(sSF + (u & 1) * 1024);
      dst[lane] = make_uint4(w[0], w[1], w[2], w[3]);
      dst[32 + lane] = make_uint4(a[0], a[1], a[2], a[3]);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[u & 1]);
    }
  }
  __syncwarp();

  // The finished tile: warp (quarter, half) has features n0 + 32 quarter + lane and
  // half of the tokens.
  bool ok = mbar_wait(done, 0, abort_flag, p.err);
  ok = __all_sync(0xffffffffu, ok);
  tc_fence_after();
  const int quarter = warp & 3, half = warp >> 2;
  constexpr int COLS = BN / 2;                       // tokens of a warp
  constexpr int CH = COLS < 32 ? COLS : 32;          // of them at a time
  const uint32_t tacc = tmem + ((uint32_t)(quarter * 32) << 16) + half * COLS;
  const int n = n0 + quarter * 32 + lane;
#pragma unroll
  for (int c0 = 0; c0 < COLS; c0 += CH) {
    if (!ok) break;
    uint32_t v[CH];
    if constexpr (CH == 8) tmem_ld_32x32b_x8(tacc + c0, v);
    else if constexpr (CH == 16) tmem_ld_32x32b_x16(tacc + c0, v);
    else tmem_ld_32x32b_x32(tacc + c0, v);
    tmem_ld_wait();
    if (split > 1) {
      float* part = reinterpret_cast<float*>(smem);  // [BN][128]; every load has been used
#pragma unroll
      for (int c = 0; c < CH; ++c)
        part[(half * COLS + c0 + c) * 128 + quarter * 32 + lane] = __uint_as_float(v[c]);
    } else if (n < p.N) {
      const float bias = p.bias ? __ldg(p.bias + n) : 0.f;
      const int m = m0 + half * COLS + c0;
      const int64_t o = (int64_t)m * p.N + n;
      float r[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c)
        r[c] = p.resid && m + c < p.M ? __half2float(p.resid[o + (int64_t)c * p.N]) : 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (m + c < p.M)
          p.out[o + (int64_t)c * p.N] =
              __float2half_rn(finish(__uint_as_float(v[c]) + bias, p.act) + r[c]);
    }
  }
  if (split > 1) {
    tc_fence_before();
    cluster_sync();
    const int cols = BN / split;                     // tokens this CTA finishes
    const int f = threadIdx.x & 127;
    const bool in_n = n0 + f < p.N;
    const float bias = p.bias && in_n ? __ldg(p.bias + n0 + f) : 0.f;
    for (int c = rank * cols + (threadIdx.x >> 7); c < (rank + 1) * cols; c += kThreads / 128) {
      const int m = m0 + c;
      if (m >= p.M || !in_n) continue;
      const int64_t o = (int64_t)m * p.N + n0 + f;
      const float r = p.resid ? __half2float(p.resid[o]) : 0.f;
      const float* mine = reinterpret_cast<const float*>(smem) + c * 128 + f;
      float v = 0.f;
      for (int q = 0; q < split; ++q) v += ld_cluster_f32(cluster_addr(mine, q));
      p.out[o] = __float2half_rn(finish(v + bias, p.act) + r);
    }
    cluster_sync();                                  // until the others have read this CTA's part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

template <int BN>
int launch_tile(const GemmE4m3Desc& g, int split, int* err, cudaStream_t s) {
  using Cfg = TileCfg<BN>;
  const uint64_t pitch = (uint64_t)e4m3_pitch(g.K);
  CUtensorMap tw, ta;
  if (!make_tmap_2d_u8(&tw, g.w, pitch, (uint64_t)g.N, 128) ||
      !make_tmap_2d_u8(&ta, g.a, pitch, (uint64_t)g.M, BN))
    return HEXLIB_B200_ERR_CUDA;
  E4m3Params p;
  p.a_scales = g.a_scales;
  p.w_scales = g.w_scales;
  p.bias = g.bias;
  p.resid = (const __half*)g.resid;
  p.out = (__half*)g.out;
  p.M = g.M;
  p.N = g.N;
  p.num_kb = (int)(pitch / kBlockK);
  p.act = g.act;
  p.tiles_n = (g.N + 127) / 128;
  p.err = err;
  const int64_t tiles = (int64_t)p.tiles_n * ((g.M + BN - 1) / BN);
  if (tiles * split > 0x7fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, gemm_e4m3_tile<BN>, tw, ta, p, split) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

}  // namespace

int gemm_e4m3_kernels_init() {
  if (cudaFuncSetAttribute(gemm_e4m3_tile<16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<16>::SMEM_BYTES) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_e4m3_tile<32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<32>::SMEM_BYTES) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_e4m3_tile<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<64>::SMEM_BYTES) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_e4m3_tile<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<128>::SMEM_BYTES) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

int launch_gemm_e4m3(const GemmE4m3Desc& g, int* err, cudaStream_t s) {
  const int num_kb = (int)(e4m3_pitch(g.K) / kBlockK);
  const int bn = g.M <= 16 ? 16 : g.M <= 32 ? 32 : g.M <= 64 ? 64 : 128;
  const int64_t tiles = (int64_t)((g.N + 127) / 128) * ((g.M + bn - 1) / bn);
  int split = 1;
  while (split < 8 && tiles * split * 2 <= 296 && num_kb >= split * 4) split *= 2;
  switch (bn) {
    case 16: return launch_tile<16>(g, split, err, s);
    case 32: return launch_tile<32>(g, split, err, s);
    case 64: return launch_tile<64>(g, split, err, s);
  }
  return launch_tile<128>(g, split, err, s);
}

}  // namespace hb

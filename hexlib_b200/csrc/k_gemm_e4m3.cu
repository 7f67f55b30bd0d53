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

#include <math.h>

#include <atomic>

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
  int tiles_n;                // tiles along N
  int wide;                   // rows of out and resid are whole 16-byte vectors
  int ahead;                  // fetch the residual to L2 a tile ahead
  int* err;
};

// The next 1024-byte boundary, reached by an offset: rounding the pointer as an integer
// would lose that it is shared memory, and every access through it would be a generic
// one, ordered with the stores of the output (16384 x 128 x 2304: 27.5 us then, 24.9 so).
__device__ __forceinline__ uint8_t* aligned_1024(uint8_t* p) {
  return p + ((0u - smem_u32(p)) & 1023u);
}

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
// of reading w once, which takes all SMs. Each CTA sends the partial sums of BN / S
// tokens to each of the others' shared memory, and adds up what it was sent in rank
// order, so the result does not depend on who was first.
//
// Launched with programmatic serialization: a CTA may start while the kernel before
// (the quantization of a, which lets it) is still running. Until that has finished it
// only sets up and brings its part of w to L2, which is right whoever wrote w last; after
// it, plain loads: the read-only path is for data that nothing writes while the kernel lives.
template <int BN>
struct TileCfg {
  static constexpr int W_BYTES = 128 * kBlockK;
  static constexpr int A_BYTES = BN * kBlockK;
  static constexpr int STAGE_BYTES = W_BYTES + A_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int SF_BYTES = 2 * 2 * 512;                    // two buffers of w and a
  static constexpr int PART_BYTES = BN * 128 * 4;                 // sums from the other ranks
  static constexpr int TMEM_COLS = 2 * BN;                        // accumulator + 16 of scales
  static constexpr int smem(int split) {
    return STAGES * STAGE_BYTES + SF_BYTES + (split > 1 ? PART_BYTES : 0) + 1024 + 256;
  }
};

template <int BN>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_e4m3_tile(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                   const E4m3Params p, const int split_log2) {
  const int split = 1 << split_log2;
  using Cfg = TileCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_1024(smem_raw);
  uint8_t* sW = smem;
  uint8_t* sA = smem + Cfg::STAGES * Cfg::W_BYTES;
  uint8_t* sSF = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  float* part = reinterpret_cast<float*>(sSF + Cfg::SF_BYTES);   // [split][BN / split][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(sSF + Cfg::SF_BYTES +
                                               (split > 1 ? Cfg::PART_BYTES : 0));
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* sf_full = empty + Cfg::STAGES;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* done = sf_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int tile = blockIdx.x / split;
  const int n0 = (tile % p.tiles_n) * 128, m0 = (tile / p.tiles_n) * BN;
  // the blocks of K of this CTA (at least one: split <= num_kb)
  const int kb0 = (int)((int64_t)p.num_kb * rank / split);
  const int kb1 = (int)((int64_t)p.num_kb * (rank + 1) / split);
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmA);
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
  } else if (warp == 3 && lane == 0) {
    for (int kb = kb0; kb < kb1 && kb < kb0 + 8; ++kb) tma_prefetch_l2_2d(&tmW, kb * kBlockK, n0);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (split > 1) cluster_arrive();                   // waited for before the parts are sent
  grid_dependency_wait();

  // A role's whole warp runs its loop and an elected lane issues, which keeps addresses
  // and descriptors in uniform registers: with one lane forming them anew a block took
  // 400 ns to issue, more than its loads. The loops are not unrolled over the stages: the
  // roles share the instruction cache (unrolled: 16384 x 768 x 2304 33.6 against 31.9 us on
  // the pairs below; with the epilogue unrolled too 43).
  if (warp == 0) {
    int kb = kb0;
    for (uint32_t ph = 1; kb < kb1; ph ^= 1u) {
#pragma unroll 1
      for (int s = 0; s < Cfg::STAGES; ++s) {
        if (kb >= kb1) break;
        if (!mbar_wait_warp(&empty[s], ph, abort_flag, p.err)) {
          kb = kb1;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(&full[s], Cfg::STAGE_BYTES);
          tma_load_2d(&tmW, &full[s], sW + s * Cfg::W_BYTES, kb * kBlockK, n0);
          tma_load_2d(&tmA, &full[s], sA + s * Cfg::A_BYTES, kb * kBlockK, m0);
        }
        ++kb;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_e4m3_scaled(128, BN);
    const uint64_t dw = sdesc_sw128(smem_u32(sW), 16, 1024);
    const uint64_t da = sdesc_sw128(smem_u32(sA), 16, 1024);
    const uint64_t dsf = sdesc_rows16(smem_u32(sSF));
    uint32_t u = 0;                                   // scale words used so far
    int kb = kb0;
    bool ok = true;
    for (uint32_t ph = 0; kb < kb1; ph ^= 1u) {
#pragma unroll 1
      for (int s = 0; s < Cfg::STAGES; ++s) {
        if (kb >= kb1) break;
        const uint32_t b = u & 1, sf = tmem + BN + b * 8;
        const bool fresh = kb == kb0 || (kb & 3) == 0;
        if (fresh) ok = mbar_wait_warp(&sf_full[b], (u >> 1) & 1, abort_flag, p.err);
        ok = ok && mbar_wait_warp(&full[s], ph, abort_flag, p.err);
        if (!ok) {
          kb = kb1;
          break;
        }
        tc_fence_after();
        const bool last_of_word = (kb & 3) == 3 || kb + 1 == kb1;
        if (elect_one()) {
          if (fresh) {
            tmem_copy_scales(sf, dsf + b * (1024 >> 4));
            tmem_copy_scales(sf + 4, dsf + b * (1024 >> 4) + (512 >> 4));
          }
          const uint32_t id = idesc_with_scale_byte(idesc, kb & 3);
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            umma_e4m3_scaled(tmem, dw + (s * Cfg::W_BYTES + kk * 32 >> 4),
                             da + (s * Cfg::A_BYTES + kk * 32 >> 4), id, sf, sf + 4,
                             kk > 0 || kb > kb0 ? 1u : 0u);
          umma_commit(&empty[s]);
          if (last_of_word) umma_commit(&sf_empty[b]);
        }
        u += last_of_word;
        ++kb;
      }
    }
    if (ok && elect_one()) umma_commit(done);
  } else if (warp == 2) {
    // scale words of 512 of K: row lane + 32 j of the tile to word j of row `lane`
    int u = 0;
    for (int g = kb0 >> 2; g <= (kb1 - 1) >> 2; ++g, ++u) {
      uint32_t w[4], a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = lane + 32 * j, n = n0 + r, m = m0 + r;
        w[j] = n < p.N ? p.w_scales[(int64_t)g * p.N + n] : 0x7f7f7f7fu;
        a[j] = r < BN && m < p.M ? p.a_scales[(int64_t)g * p.M + m] : 0x7f7f7f7fu;
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
  if (split > 1) cluster_wait();                     // every rank has started
#pragma unroll
  for (int c0 = 0; c0 < COLS; c0 += CH) {
    if (!ok) break;
    uint32_t v[CH];
    if constexpr (CH == 8) tmem_ld_32x32b_x8(tacc + c0, v);
    else if constexpr (CH == 16) tmem_ld_32x32b_x16(tacc + c0, v);
    else tmem_ld_32x32b_x32(tacc + c0, v);
    tmem_ld_wait();
    if (split > 1) {
      // token c goes to rank c / cols, at [this rank][c % cols][feature] there
      constexpr int BN_LOG2 = BN == 16 ? 4 : BN == 32 ? 5 : 6;
      const int cols_log2 = BN_LOG2 - split_log2, cols = 1 << cols_log2;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int tok = half * COLS + c0 + c;
        float* to = part + ((rank << cols_log2) + (tok & (cols - 1))) * 128 + quarter * 32 + lane;
        st_cluster_u32(cluster_addr(to, tok >> cols_log2), v[c]);
      }
    } else if (n < p.N) {
      const float bias = p.bias ? p.bias[n] : 0.f;
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
    cluster_sync();                                  // every rank's part has arrived
    const int cols = BN >> split_log2;               // tokens this CTA finishes
    const int f = threadIdx.x & 127;
    const bool in_n = n0 + f < p.N;
    const float bias = p.bias && in_n ? p.bias[n0 + f] : 0.f;
    for (int c = threadIdx.x >> 7; c < cols; c += kThreads / 128) {
      const int m = m0 + rank * cols + c;
      if (m >= p.M || !in_n) continue;
      const int64_t o = (int64_t)m * p.N + n0 + f;
      const float r = p.resid ? __half2float(p.resid[o]) : 0.f;
      float v = 0.f;
      for (int q = 0; q < split; ++q) v += part[(q * cols + c) * 128 + f];
      p.out[o] = __float2half_rn(finish(v + bias, p.act) + r);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

constexpr int64_t kHalfL2 = 64ll << 20;    // bytes

E4m3Params params_of(const GemmE4m3Desc& g, int* err) {
  E4m3Params p = {};
  p.a_scales = g.a_scales;
  p.w_scales = g.w_scales;
  p.bias = g.bias;
  p.resid = (const __half*)g.resid;
  p.out = (__half*)g.out;
  p.M = g.M;
  p.N = g.N;
  p.num_kb = (int)(e4m3_pitch(g.K) / kBlockK);
  p.act = g.act;
  p.wide = ((reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.resid) |
             static_cast<uintptr_t>(2) * g.N) & 15u) == 0;
  // Fetching the residual to L2 a tile ahead pays where it is not there yet and K is too short
  // to hide its way. By vectors, without and with, at K = 128, 1024, 2048: 4750 x 6800 49.0 and
  // 40.2 us, 54.1 and 49.2, 65.0 and 65.0 (1536: 57.9 and 56.3; 4096: 105.5 and 108.9);
  // 7680 x 4096 43.3 and 39.9, 48.7 and 48.0, 60.7 and 62.3; 2600 x 6800, 71 MB of residual
  // and output, 33.9 and 29.1, 38.2 and 34.3, 42.3 and 42.1; 4096 x 4096, 67 MB, 26.3 and
  // 25.9, 30.9 and 31.1, 35.9 and 37.1; 16384 x 768, 50 MB, 20.7 and 21.3, 25.4 and 25.6,
  // 30.1 and 30.6. By words, where every row is waited for, it costs nothing at any K:
  // 4750 x 6795 112 and 108 at 128, 105 and 103 at 1024, 134 and 134 at 4096.
  p.ahead = !p.wide || (g.K <= 1024 && static_cast<int64_t>(4) * g.M * g.N > kHalfL2);
  p.err = err;
  return p;
}

cudaLaunchAttribute* cluster_of(cudaLaunchAttribute* attr, int n) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)n;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  return attr;
}

template <int BN>
int launch_tile(const GemmE4m3Desc& g, int split_log2, int* err, cudaStream_t s) {
  const int split = 1 << split_log2;
  using Cfg = TileCfg<BN>;
  const uint64_t pitch = (uint64_t)e4m3_pitch(g.K);
  CUtensorMap tw, ta;
  if (!make_tmap_2d_u8(&tw, g.w, pitch, (uint64_t)g.N, 128) ||
      !make_tmap_2d_u8(&ta, g.a, pitch, (uint64_t)g.M, BN))
    return HEXLIB_B200_ERR_CUDA;
  E4m3Params p = params_of(g, err);
  p.tiles_n = (g.N + 127) / 128;
  const int64_t tiles = (int64_t)p.tiles_n * ((g.M + BN - 1) / BN);
  if (tiles * split > 0x7fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::smem(split);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = cluster_of(attr, split);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, gemm_e4m3_tile<BN>, tw, ta, p, split_log2) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

// ---- CTA pairs, 256 tokens by 256 features ---------------------------------------
//
// A persistent kernel on clusters of two SMs. Per block of 128 of K each CTA lands its
// own 128 rows of a and of w (32 KiB), and the leader's MMA thread multiplies the
// 256 x 256 x 128 block across both SMs: half the fill traffic of one-CTA tiles. What
// bounds the mainloop is shared memory: at the tensor cores' full rate (512 cycles a
// block) reading the operands and landing the next ones takes all of its 128 bytes a
// cycle. Measured, the four MMAs of a block take 528 cycles with a quarter of the loads
// beside them, 571 with half, about 640 with all.
//
// Tensor memory holds 512 columns: two 256-column accumulators would leave none for
// the scales. The accumulators therefore OVERLAP by 24 columns, [0, 256) and
// [232, 488), and the scales take [488, 512). The epilogue reads the overlap first and
// tells the MMA thread as soon as it has; the next tile's MMAs start then, while the
// rest of the tile is finished. That arrival also says that the warp is done with
// every earlier tile, so one arrival covers both uses. A warp may arrive for the next tile
// before another has for this one -- the half without the overlap arrives as it begins
// the tile -- so tiles take turns at two barriers; further ahead no warp comes, since it
// waits for its tile's accumulator in between. (Tiles of 192 columns with two
// whole accumulators: 16384 x 768 x 2304 in 42.5 us against 37.6, 8192 x 4096 x 4096 in
// 134 against 108; narrower MMAs re-read the tokens' rows more often.)
//
//   full[s]     leader: both CTAs' loads of stage s
//   empty[s]    both: the stage has been read
//   sf_full[b]  leader: both CTAs have written scale buffer b
//   sf_empty[b] both: the MMAs that use scale buffer b are done
//   tfull[a]    both: accumulator a is complete
//   tempty[a]   leader: the pair's 16 epilogue warps have read accumulator a's overlap
//               and the whole of the other
//
// Epilogue: 8 warps, each 32 rows by 128 columns, 32 columns at a time: from tensor
// memory through registers and a 2 KiB box in shared memory to rows of 64 bytes, stored
// by the LSU at any alignment. One kernel for each activation, with and without a
// residual: shorter code leaves the instruction cache to the other roles (16384 x 768 x
// 2304 with GELU: 41.8 us as one kernel, 37.8 as six; without 32.0 and 31.6).
constexpr int kPairThreads = 384;   // loads, MMAs, 2 warps of scales, 8 of epilogue

struct PairCfg {
  static constexpr int BN = 256;
  static constexpr int STAGES = 5;
  static constexpr int A_BYTES = 128 * kBlockK;           // of each CTA
  static constexpr int W_BYTES = BN / 2 * kBlockK;
  static constexpr int STAGE_BYTES = A_BYTES + W_BYTES;
  static constexpr int SF_BYTES = 512 + 1024;             // own rows of a, all rows of w
  static constexpr int BOX_BYTES = 2048;                  // 32 rows of 32 fp16 per warp
  static constexpr int BIAS_BYTES = BN / 2 * 4;           // the columns of each warp
  static constexpr int SMEM_BYTES =
      STAGES * STAGE_BYTES + 8 * (BOX_BYTES + BIAS_BYTES) + 2 * SF_BYTES + 1024 + 256;
  static constexpr uint32_t ACC1 = 232, SF = 488;
};

// 32 columns of a row: bias (its 32 values in shared memory), activation.
template <int ACT>
__device__ __forceinline__ void activate32(const E4m3Params& p, const uint32_t (&r)[32],
                                           const float* bias, float2 (&v)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    v[j] = make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float4 b = *reinterpret_cast<const float4*>(bias + 2 * j);
      v[j] = __fadd2_rn(v[j], make_float2(b.x, b.y));
      v[j + 1] = __fadd2_rn(v[j + 1], make_float2(b.z, b.w));
    }
  }
  if (ACT == 1) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = gelu_tanh_f2(v[j]);
  } else if (ACT == 2) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = make_float2(gelu_erf_f(v[j].x), gelu_erf_f(v[j].y));
  }
}

// A box of 32 rows of 64 bytes, the 16-byte slot q of row r at q ^ (r / 2 % 4): a lane
// that writes its own row and a quarter warp that reads two rows both touch every bank
// once.
__device__ __forceinline__ uint32_t box_at(int r, int q) {
  return r * 64 + ((q ^ ((r >> 1) & 3)) * 16);
}

// The box between shared and global memory, rows [row0, row0 + 32) clipped to M and
// columns [n, n + 32) to N: 16 bytes to a lane where all rows allow it, else two values,
// as one word where the row allows it (with an odd N every other row does).
__device__ __forceinline__ void box_store(const E4m3Params& p, const uint8_t* box, int64_t row0,
                                          int n, int lane) {
  if (p.wide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2), q = lane & 3;
      if (row0 + r < p.M && n + q * 8 < p.N)
        *reinterpret_cast<uint4*>(p.out + (row0 + r) * p.N + n + q * 8) =
            *reinterpret_cast<const uint4*>(box + box_at(r, q));
    }
  } else {
    const int k = lane & 15, left = p.N - n - 2 * k;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int r = i * 2 + (lane >> 4);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(box + box_at(r, k >> 2) + (k & 3) * 4);
      if (row0 + r >= p.M || left <= 0) continue;
      __half* to = p.out + (row0 + r) * p.N + n + 2 * k;
      if (left > 1 && (reinterpret_cast<uintptr_t>(to) & 3u) == 0) {
        *reinterpret_cast<uint32_t*>(to) = w;
      } else {
        to[0] = __ushort_as_half((unsigned short)w);
        if (left > 1) to[1] = __ushort_as_half((unsigned short)(w >> 16));
      }
    }
  }
}
__device__ __forceinline__ void box_load(const E4m3Params& p, uint8_t* box, int64_t row0, int n,
                                         int lane) {
  if (p.wide) {
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2), q = lane & 3;
      u[i] = row0 + r < p.M && n + q * 8 < p.N
                 ? *reinterpret_cast<const uint4*>(p.resid + (row0 + r) * p.N + n + q * 8)
                 : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(box + box_at(i * 8 + (lane >> 2), lane & 3)) = u[i];
  } else {
    // Aligned pairs: a row that starts between two words takes each word from its second
    // element on, and the element before from the lane before (a row's first one is the lane
    // of its number's). All 32 rows are loaded at once (4750 x 260 x 6795: 105 us with single
    // elements, sixteen rows at once, 98 so).
    const int k = lane & 15, left = p.N - n - 2 * k;
    const unsigned short* base =
        reinterpret_cast<const unsigned short*>(p.resid) + row0 * p.N + n;
    const uint32_t first = row0 + lane < p.M && n < p.N ? base[(int64_t)lane * p.N] : 0;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = i * 2 + (lane >> 4);
      const unsigned short* from = base + (int64_t)r * p.N + 2 * k;
      const int odd = (int)(reinterpret_cast<uintptr_t>(from) >> 1) & 1;
      w[i] = 0;
      if (row0 + r < p.M && left > odd + 1)
        w[i] = *reinterpret_cast<const uint32_t*>(from + odd);
      else if (row0 + r < p.M && left == odd + 1)
        w[i] = from[odd];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = i * 2 + (lane >> 4);
      const bool odd = (reinterpret_cast<uintptr_t>(base + (int64_t)r * p.N) & 2u) != 0;
      const uint32_t before = __shfl_up_sync(0xffffffffu, w[i], 1, 16) >> 16;
      const uint32_t own = __shfl_sync(0xffffffffu, first, r);
      *reinterpret_cast<uint32_t*>(box + box_at(r, k >> 2) + (k & 3) * 4) =
          odd ? (k ? before : own) | (w[i] << 16) : w[i];
    }
  }
}

// The tiles of a CTA pair, `step` apart in row-major order, without a division between
// them (the 64-bit ones of the direct form took a tenth of a short tile's time).
struct TileWalk {
  uint32_t m, n, left;                               // tile coordinates, tiles still to do
  uint32_t dm, dn, tiles_n;
  __device__ TileWalk(uint32_t tiles_m, uint32_t tiles_n_, uint32_t first, uint32_t step)
      : tiles_n(tiles_n_) {
    const uint32_t total = tiles_m * tiles_n;
    m = first / tiles_n;
    n = first - m * tiles_n;
    dm = step / tiles_n;
    dn = step - dm * tiles_n;
    left = first < total ? (total - first + step - 1) / step : 0;
  }
  __device__ void next() {
    --left;
    m += dm;
    n += dn;
    if (n >= tiles_n) {
      n -= tiles_n;
      ++m;
    }
  }
};

template <int ACT, bool RESID>
__global__ void __launch_bounds__(kPairThreads, 1)
    gemm_e4m3_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                   const E4m3Params p) {
  using Cfg = PairCfg;
  constexpr int BN = Cfg::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_1024(smem_raw);
  uint8_t* sA = smem;
  uint8_t* sW = smem + Cfg::STAGES * Cfg::A_BYTES;
  uint8_t* sBox = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  uint8_t* sSF = sBox + 8 * Cfg::BOX_BYTES;
  uint8_t* sBias = sSF + 2 * Cfg::SF_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sBias + 8 * Cfg::BIAS_BYTES);
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* sf_full = empty + Cfg::STAGES;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* tfull = sf_empty + 2;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sf_full[b], 2);
      mbar_init(&sf_empty[b], 1);
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t peer_abort = cluster_addr(tmem_slot + 1, rank ^ 1u);
  grid_dependency_wait();

  TileWalk t((p.M + 255u) / 256u, p.tiles_n, blockIdx.x >> 1, gridDim.x >> 1);

  // (loops round the ring of stages, as in the tile kernel, through all tiles)
  if (warp == 0) {
    const uint32_t full_lead = cluster_addr(full, 0);
    int kb = 0;
    for (uint32_t ph = 1; t.left; ph ^= 1u) {
#pragma unroll 1
      for (int s = 0; s < Cfg::STAGES; ++s) {
        if (!t.left) break;
        if (!mbar_wait_cluster_warp(&empty[s], ph, abort_flag, p.err)) {
          if (lane == 0) st_cluster_u32(peer_abort, 1);
          t.left = 0;
          break;
        }
        const int row = t.m * 256 + rank * 128, col = t.n * BN + rank * (BN / 2);
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * Cfg::STAGE_BYTES);
          tma_load_2d_pair(&tmA, full_lead + s * 8, sA + s * Cfg::A_BYTES, kb * kBlockK, row);
          tma_load_2d_pair(&tmW, full_lead + s * 8, sW + s * Cfg::W_BYTES, kb * kBlockK, col);
        }
        if (++kb == p.num_kb) {
          kb = 0;
          t.next();
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_e4m3_scaled(256, BN);
      const uint64_t da = sdesc_sw128(smem_u32(sA), 16, 1024);
      const uint64_t dw = sdesc_sw128(smem_u32(sW), 16, 1024);
      const uint64_t dsf = sdesc_rows16(smem_u32(sSF));
      uint32_t u = 0, i = 0;                         // scale words, tiles so far
      int kb = 0;
      for (uint32_t ph = 0; t.left; ph ^= 1u) {
#pragma unroll 1
        for (int s = 0; s < Cfg::STAGES; ++s) {
          if (!t.left) break;
          const uint32_t b = u & 1, sf = tmem + Cfg::SF + b * 12;
          const uint32_t acc = tmem + ((i & 1) ? Cfg::ACC1 : 0u);
          const bool fresh = (kb & 3) == 0;
          bool ok = true;
          if (kb == 0 && i > 0)
            ok = mbar_wait_cluster_warp(&tempty[(i - 1) & 1], ((i - 1) >> 1) & 1, abort_flag,
                                        p.err);
          if (fresh)
            ok = ok && mbar_wait_cluster_warp(&sf_full[b], (u >> 1) & 1, abort_flag, p.err);
          ok = ok && mbar_wait_cluster_warp(&full[s], ph, abort_flag, p.err);
          if (!ok) {
            if (lane == 0) st_cluster_u32(peer_abort, 1);
            t.left = 0;
            break;
          }
          tc_fence_after();
          const bool last = kb + 1 == p.num_kb;
          const bool last_of_word = last || (kb & 3) == 3;
          if (elect_one()) {
            if (fresh) {
              tmem_copy_scales_pair(sf, dsf + b * (Cfg::SF_BYTES >> 4));
              tmem_copy_scales_pair(sf + 4, dsf + b * (Cfg::SF_BYTES >> 4) + (512 >> 4));
              tmem_copy_scales_pair(sf + 8, dsf + b * (Cfg::SF_BYTES >> 4) + (1024 >> 4));
            }
            const uint32_t id = idesc_with_scale_byte(idesc, kb & 3);
#pragma unroll
            for (int kk = 0; kk < kBlockK / 32; ++kk)
              umma_e4m3_scaled_pair(acc, da + (s * Cfg::A_BYTES + kk * 32 >> 4),
                                    dw + (s * Cfg::W_BYTES + kk * 32 >> 4), id, sf, sf + 4,
                                    kk > 0 || kb > 0 ? 1u : 0u);
            umma_commit_pair(&empty[s], 0x3);
            if (last_of_word) umma_commit_pair(&sf_empty[b], 0x3);
            if (last) umma_commit_pair(&tfull[i & 1], 0x3);
          }
          u += last_of_word;
          ++kb;
          if (last) {
            kb = 0;
            t.next();
            ++i;
          }
        }
      }
    }
  } else if (warp <= 3) {
    // Scale words of 512 of K: row lane + 32 j of the tile to word j of row `lane`. A word
    // takes its loads, the fence and the arrival one after the other, longer than its
    // MMAs at two words a tile; so two warps take turns, each with a buffer of its own.
    const uint32_t b = warp - 2, sf_full_lead = cluster_addr(sf_full + b, 0);
    const int groups = (p.num_kb + 3) >> 2;
    uint32_t ph = 1, mine = b;                       // words until this warp's next
    for (; t.left; t.next()) {
      const int m0 = t.m * 256 + rank * 128 + lane, n0 = t.n * BN + lane;
      for (int g = 0; g < groups; ++g) {
        if (mine-- != 0) continue;
        mine = 1;
        uint32_t a[4], w[8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = m0 + 32 * j < p.M ? p.a_scales[(int64_t)g * p.M + m0 + 32 * j] : 0x7f7f7f7fu;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j] = n0 + 32 * j < p.N ? p.w_scales[(int64_t)g * p.N + n0 + 32 * j] : 0x7f7f7f7fu;
        const bool ok = mbar_wait_cluster(&sf_empty[b], ph, abort_flag, p.err);
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) st_cluster_u32(peer_abort, 1);
          goto out;
        }
        ph ^= 1u;
        uint4* dst = reinterpret_cast<uint4*>(sSF + b * Cfg::SF_BYTES);
        dst[lane] = make_uint4(a[0], a[1], a[2], a[3]);
        dst[32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
        dst[64 + lane] = make_uint4(w[4], w[5], w[6], w[7]);
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(sf_full_lead);
      }
    }
  } else {
    // Epilogue: TMEM lanes of `quarter`, the columns of `half` from the end that may
    // overlap the other accumulator (columns 232.. of the first, 0..23 of the second).
    constexpr int COLS = BN / 2;
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    uint8_t* box = sBox + (warp - 4) * Cfg::BOX_BYTES;
    float* bias = reinterpret_cast<float*>(sBias + (warp - 4) * Cfg::BIAS_BYTES);
    const uint32_t tempty_lead = cluster_addr(tempty, 0);
    // a tile's bias is read while the tile before is finished
    float next_bias[COLS / 32];
    auto read_bias = [&](uint32_t tn) {
#pragma unroll
      for (int j = 0; j < COLS / 32; ++j) {
        const int n = tn * BN + half * COLS + j * 32 + lane;
        next_bias[j] = p.bias && n < p.N ? p.bias[n] : 0.f;
      }
    };
    read_bias(t.n);
    // ... and its rows of the residual are fetched to L2 where that pays (p.ahead)
    auto fetch_resid = [&](uint32_t tm, uint32_t tn) {
      const int64_t row = (int64_t)tm * 256 + rank * 128 + quarter * 32 + lane;
      if (row >= p.M) return;
#pragma unroll
      for (int c = 0; c < COLS; c += 32) {
        const int n = (int)tn * BN + half * COLS + c;
        if (n < p.N)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.resid + row * p.N + n));
      }
    };
    if (RESID && p.ahead) fetch_resid(t.m, t.n);
    uint32_t i = 0;
    for (; t.left; ++i) {
      const int64_t row0 = (int64_t)t.m * 256 + rank * 128 + quarter * 32;
      const int n0 = t.n * BN + half * COLS;
      t.next();
      const bool overlaps = half != (int)(i & 1);    // this half has the overlap
      tc_fence_before();                             // (the loads of the tile before)
      if (!overlaps && lane == 0) mbar_arrive_cluster_relaxed(tempty_lead + (i & 1) * 8);
#pragma unroll
      for (int j = 0; j < COLS / 32; ++j) bias[j * 32 + lane] = next_bias[j];
      __syncwarp();
      if (t.left) read_bias(t.n);
      if (RESID && p.ahead && t.left) fetch_resid(t.m, t.n);
      if (RESID) box_load(p, box, row0, n0 + (half ? COLS - 32 : 0), lane);
      const bool ok = mbar_wait_cluster(&tfull[i & 1], (i >> 1) & 1, abort_flag, p.err);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) st_cluster_u32(peer_abort, 1);
        goto out;
      }
      tc_fence_after();
      const uint32_t tacc = tmem + ((i & 1) ? Cfg::ACC1 : 0u) + half * COLS +
                            ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int j = 0; j < COLS / 32; ++j) {
        const int c = half ? COLS - 32 - 32 * j : 32 * j;
        uint32_t r[32];
        tmem_ld_32x32b_x32(tacc + c, r);
        tmem_ld_wait();
        if (overlaps && j == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(tempty_lead + (i & 1) * 8);
        }
        float2 v[16];
        activate32<ACT>(p, r, bias + c, v);
        if (RESID) {
          if (j > 0) box_load(p, box, row0, n0 + c, lane);
          __syncwarp();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4* slot = reinterpret_cast<uint4*>(box + box_at(lane, q));
          if (RESID) {
            const uint4 u = *slot;
            const uint32_t h[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[4 * q + e] = __fadd2_rn(v[4 * q + e], unpack_half2(h[e]));
          }
          *slot = make_uint4(pack_half2(v[4 * q].x, v[4 * q].y),
                             pack_half2(v[4 * q + 1].x, v[4 * q + 1].y),
                             pack_half2(v[4 * q + 2].x, v[4 * q + 2].y),
                             pack_half2(v[4 * q + 3].x, v[4 * q + 3].y));
        }
        __syncwarp();
        box_store(p, box, row0, n0 + c, lane);
        __syncwarp();                                // read before the next chunk's writes
      }
    }
  }

out:
  tc_fence_before();
  __syncthreads();
  cluster_sync();            // no CTA leaves while the other may still use it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

using PairKernel = void (*)(CUtensorMap, CUtensorMap, E4m3Params);
PairKernel pair_kernel(int act, bool resid) {
  if (resid)
    return act == 0 ? gemm_e4m3_pair<0, true>
                    : act == 1 ? gemm_e4m3_pair<1, true> : gemm_e4m3_pair<2, true>;
  return act == 0 ? gemm_e4m3_pair<0, false>
                  : act == 1 ? gemm_e4m3_pair<1, false> : gemm_e4m3_pair<2, false>;
}

std::atomic<int> g_pairs{0};   // pairs resident at once, 0 until the kernel is loaded

int launch_pair(const GemmE4m3Desc& g, int* err, cudaStream_t s) {
  using Cfg = PairCfg;
  constexpr int BN = Cfg::BN;
  const uint64_t pitch = (uint64_t)e4m3_pitch(g.K);
  CUtensorMap ta, tw;
  if (!make_tmap_2d_u8(&ta, g.a, pitch, (uint64_t)g.M, 128) ||
      !make_tmap_2d_u8(&tw, g.w, pitch, (uint64_t)g.N, BN / 2))
    return HEXLIB_B200_ERR_CUDA;
  E4m3Params p = params_of(g, err);
  p.tiles_n = (g.N + BN - 1) / BN;
  const int64_t tiles = (int64_t)((g.M + 255) / 256) * p.tiles_n;
  if (tiles > 0x3fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  const int64_t pairs = g_pairs.load(std::memory_order_relaxed);
  if (pairs <= 0) return HEXLIB_B200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs)), 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = cluster_of(attr, 2);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, pair_kernel(g.act, g.resid != nullptr), ta, tw, p) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

bool load_pair() {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(512, 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = PairCfg::SMEM_BYTES;
  cudaLaunchAttribute attr[1];
  cfg.attrs = cluster_of(attr, 2);
  cfg.numAttrs = 1;
  int pairs = 0;
  for (int act = 0; act < 3; ++act)
    for (int resid = 0; resid < 2; ++resid)
      if (cudaFuncSetAttribute((const void*)pair_kernel(act, resid != 0),
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               PairCfg::SMEM_BYTES) != cudaSuccess ||
          cudaOccupancyMaxActiveClusters(&pairs, (const void*)pair_kernel(act, resid != 0),
                                         &cfg) != cudaSuccess)
        return false;
  g_pairs.store(pairs, std::memory_order_relaxed);
  return pairs > 0;
}

}  // namespace

int gemm_e4m3_kernels_init() {
  if (cudaFuncSetAttribute(gemm_e4m3_tile<16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<16>::smem(2)) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_e4m3_tile<32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<32>::smem(2)) != cudaSuccess ||
      cudaFuncSetAttribute(gemm_e4m3_tile<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           TileCfg<64>::smem(2)) != cudaSuccess ||
      !load_pair()) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

// The kernel and tiling with the least estimated time, in us. The estimate is a fixed
// cost, the blocks of K a CTA goes through at the rate measured for one or two CTAs on an
// SM (68 and 108 bytes a ns), its epilogue, and the joining of a split; w from memory at
// 6 TB/s bounds the loop below. It was fitted to sweeps of every choice: 4096 x 4096 for
// 1 token 8.5 us on 16-token tiles split by 4 (16.9 unsplit), for 256 tokens 16.0 on
// 64-token tiles (22.0 on pairs, 27 split); 1000 x 1000 for 2000 tokens 10.2 on pairs and
// on 64-token tiles, 2304 x 256 for 4096 tokens 11.4 on pairs.
// Its counts, 148 SMs and 74 pairs, are the GPU's this is written for; with fewer the choice
// may be slower, never wrong.
struct Choice {
  int bn, split_log2;                      // bn = 0: CTA pairs
};

Choice choose(const GemmE4m3Desc& g) {
  const double kb = (double)(e4m3_pitch(g.K) / kBlockK);
  const int64_t pair_tiles = (int64_t)((g.M + 255) / 256) * ((g.N + 255) / 256);
  const double from_memory = kb * kBlockK * g.N / 6000e3;
  Choice best = {0, 0};
  double least = 5.0 + (double)((pair_tiles + 73) / 74) * (1.8 + 0.43 * kb);
  for (int bn = 16; bn <= 64; bn *= 2) {
    const int64_t tiles = (int64_t)((g.N + 127) / 128) * ((g.M + bn - 1) / bn);
    for (int sl = 0; sl <= 3 && kb >= (2 << sl) - (sl == 0); ++sl) {
      const int64_t ctas = tiles << sl, resident = bn == 64 && sl > 0 ? 1 : 2;
      if (sl > 0 && ctas > 148 * resident) break;
      const int64_t waves = (ctas + 148 * resident - 1) / (148 * resident);
      const int64_t beside = ctas > 148 ? resident : 1;      // CTAs on an SM at once
      const double bytes = (double)(128 + bn) * kBlockK * beside;
      double loop = (double)waves * ceil(kb / (1 << sl)) * bytes / (beside == 1 ? 68e3 : 108e3);
      if (loop < from_memory) loop = from_memory;
      const double finish = (double)waves * beside * 0.02 * bn;
      const double t = 4.0 + loop + finish + (sl ? 0.5 + 0.036 * bn : 0.0);
      if (t < least) {
        least = t;
        best = {bn, sl};
      }
    }
  }
  return best;
}

int launch_gemm_e4m3(const GemmE4m3Desc& g, int* err, cudaStream_t s) {
  const Choice c = choose(g);
  switch (c.bn) {
    case 16: return launch_tile<16>(g, c.split_log2, err, s);
    case 32: return launch_tile<32>(g, c.split_log2, err, s);
    case 64: return launch_tile<64>(g, c.split_log2, err, s);
  }
  return launch_pair(g, err, s);
}

}  // namespace hb

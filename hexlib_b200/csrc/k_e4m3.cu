// k_e4m3.cu -- fp16 matrices to and from their e4m3 form (hb_e4m3.cuh): the
// activations and weights of the 8-bit matrix product (k_gemm_e4m3.cu).
#include <cuda_runtime.h>

#include "hb_device.cuh"
#include "hb_e4m3.cuh"
#include "hb_kernels.h"

namespace hb {
namespace {

constexpr int kThreads = 256;

int grid_for(int64_t items) {
  const int64_t blocks = (items + kThreads - 1) / kThreads;
  return static_cast<int>(blocks < 148 * 8 ? blocks : 148 * 8);
}

// Half a warp per scale word: 512 values of a row, a block of 128 at a time, 8 to a
// lane, so a lane has four 16-byte loads in flight and a word is stored whole. Bound
// by memory: 2 bytes read and 1 written per value (8192 x 4096: 18.7 us, 5.4 TB/s;
// 60.6 us a block to a warp and a value at a time).
template <int VEC>
__global__ void __launch_bounds__(kThreads) quantize_e4m3(const __half* __restrict__ x,
                                                          uint8_t* __restrict__ codes,
                                                          uint32_t* __restrict__ scales,
                                                          int64_t R, int K) {
  grid_dependents_may_start();         // the product that follows waits for the codes itself
  const int l = threadIdx.x & 15;
  const uint32_t half_mask = 0xffffu << (threadIdx.x & 16);
  const int blocks = (K + 127) / 128, groups = (blocks + 3) / 4;
  const int64_t t = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 4;
  if (t >= R * groups) return;
  const int64_t r = t / groups;
  const int g = (int)(t - r * groups);
  uint32_t w[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = g * 512 + j * 128 + l * 8;
    load8<VEC>(w[j], x + r * K + k, K - k);
  }
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = g * 512 + j * 128 + l * 8;
    uint32_t byte;
    const uint2 c = e4m3_encode8(w[j], half_mask, byte);
    if (g * 4 + j < blocks)
      *reinterpret_cast<uint2*>(codes + r * (int64_t)blocks * 128 + k) = c;
    word |= byte << (8 * j);           // (a block past the last is zeros: 1.0)
  }
  if (l == 0) scales[(int64_t)g * R + r] = word;
}

// The form of the transpose of w [K, N]: a CTA turns a block of 128 of K by 32 columns
// through shared memory, then a warp has a column's block, 4 values to a lane. Done
// once per weight (4096 x 4096: 44 us, bytes alone 7.7; 768 x 2304: 6.8), by two-byte loads
// and shared-memory columns.
__global__ void __launch_bounds__(kThreads) quantize_weight_e4m3(const __half* __restrict__ w,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales,
                                                                 int K, int N) {
  __shared__ __half tile[128][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = (K + 127) / 128, padded = (blocks + 3) / 4 * 4;
  const int n_tiles = (N + 31) / 32;
  const int b = blockIdx.x / n_tiles, n0 = (blockIdx.x % n_tiles) * 32;
  for (int i = warp; i < 128; i += kThreads / 32) {
    const int64_t k = (int64_t)b * 128 + i;
    tile[i][lane] = k < K && n0 + lane < N ? w[k * N + n0 + lane] : __half(0.f);
  }
  __syncthreads();
  for (int c = warp; c < 32 && n0 + c < N; c += kThreads / 32) {
    const int64_t n = n0 + c;
    uint32_t w[2], byte;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w[j] = __half_as_ushort(tile[lane * 4 + 2 * j][c]) |
             ((uint32_t)__half_as_ushort(tile[lane * 4 + 2 * j + 1][c]) << 16);
    const uint32_t q = e4m3_encode4(w[0], w[1], byte);
    *reinterpret_cast<uint32_t*>(codes + n * (int64_t)blocks * 128 + b * 128 + lane * 4) = q;
    if (lane == 0) scales[e4m3_scale_at(n, b, N)] = (uint8_t)byte;
    if (b == blocks - 1 && lane < padded - blocks)
      scales[e4m3_scale_at(n, blocks + lane, N)] = (uint8_t)kE4m3One;
  }
}

// A value to a thread, with the row's division for each: bound by those instructions and by
// one- and two-byte accesses (8192 x 4096: 151 us, bytes alone 15.4). It shows what a form
// holds; no product dequantizes.
__global__ void dequant_e4m3(const uint8_t* __restrict__ codes,
                             const uint8_t* __restrict__ scales, __half* __restrict__ out,
                             int64_t R, int K) {
  const int64_t pitch = (K + 127) / 128 * 128, total = R * K;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / K;
    const int k = (int)(i - r * K);
    out[i] = __float2half_rn(e4m3_value(codes[r * pitch + k]) *
                             e4m3_scale(scales[e4m3_scale_at(r, k >> 7, R)]));
  }
}

int launched() {
  if (cudaPeekAtLastError() != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

}  // namespace

// Load the kernels now, so that none is loaded lazily inside a graph capture.
int e4m3_kernels_init() {
  cudaFuncAttributes a;
  for (const void* f : {(const void*)quantize_e4m3<8>, (const void*)quantize_e4m3<4>,
                        (const void*)quantize_e4m3<2>, (const void*)quantize_e4m3<1>,
                        (const void*)quantize_weight_e4m3, (const void*)dequant_e4m3})
    if (cudaFuncGetAttributes(&a, f) != cudaSuccess) {
      cudaGetLastError();
      return HEXLIB_B200_ERR_CUDA;
    }
  return HEXLIB_B200_OK;
}

int launch_quantize_e4m3(const void* x, void* codes, void* scales, int64_t R, int K,
                         cudaStream_t s) {
  const int64_t ctas = (R * e4m3_scale_groups(K) * 16 + kThreads - 1) / kThreads;
  if (ctas > 0x7fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  auto go = [&](auto kernel) {
    kernel<<<(unsigned)ctas, kThreads, 0, s>>>((const __half*)x, (uint8_t*)codes,
                                               (uint32_t*)scales, R, K);
    return launched();
  };
  switch (row_vec(K, x)) {
    case 8: return go(quantize_e4m3<8>);
    case 4: return go(quantize_e4m3<4>);
    case 2: return go(quantize_e4m3<2>);
  }
  return go(quantize_e4m3<1>);
}

int launch_quantize_weight_e4m3(const void* w, void* codes, void* scales, int K, int N,
                                cudaStream_t s) {
  const int64_t ctas = e4m3_pitch(K) / 128 * ((N + 31) / 32);
  if (ctas > 0x7fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  quantize_weight_e4m3<<<(unsigned)ctas, kThreads, 0, s>>>((const __half*)w, (uint8_t*)codes,
                                                           (uint8_t*)scales, K, N);
  return launched();
}

int launch_dequant_e4m3(const void* codes, const void* scales, void* out, int64_t R, int K,
                        cudaStream_t s) {
  dequant_e4m3<<<grid_for(R * K), kThreads, 0, s>>>((const uint8_t*)codes,
                                                    (const uint8_t*)scales, (__half*)out, R, K);
  return launched();
}

}  // namespace hb

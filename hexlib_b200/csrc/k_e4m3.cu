// k_e4m3.cu -- fp16 matrices to and from their e4m3 form (hb_e4m3.cuh): the
// activations and weights of the 8-bit matrix product (k_gemm_e4m3.cu).
#include <cuda_runtime.h>

#include "hb_e4m3.cuh"
#include "hb_kernels.h"

namespace hb {
namespace {

constexpr int kThreads = 256;

int grid_for(int64_t items) {
  const int64_t blocks = (items + kThreads - 1) / kThreads;
  return static_cast<int>(blocks < 148 * 8 ? blocks : 148 * 8);
}

// One warp per block of 128 values; the value i of row r is x[r * sr + i * si], so
// the same kernel reads a matrix and its transpose. Blocks past the row's last
// (up to a whole word of scales) only get their scale byte.
__global__ void quantize_e4m3(const __half* __restrict__ x, uint8_t* __restrict__ codes,
                              uint8_t* __restrict__ scales, int64_t R, int K, int64_t sr,
                              int64_t si) {
  const int lane = threadIdx.x & 31;
  const int blocks = (K + 127) / 128, padded = (blocks + 3) / 4 * 4;
  const int64_t pitch = blocks * 128;
  const int64_t total = R * padded;
  for (int64_t t = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; t < total;
       t += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t r = t / padded;
    const int b = (int)(t - r * padded);
    uint32_t byte = kE4m3One;
    if (b < blocks) {
      float v[4], amax = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = b * 128 + lane + 32 * j;
        v[j] = k < K ? __half2float(x[r * sr + k * si]) : 0.f;
        if (isfinite(v[j])) amax = fmaxf(amax, fabsf(v[j]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      byte = e4m3_scale_byte(amax);
      const float inv = e4m3_inverse(byte);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        codes[r * pitch + b * 128 + lane + 32 * j] = (uint8_t)e4m3_code(v[j], inv);
    }
    if (lane == 0) scales[e4m3_scale_at(r, b, R)] = (uint8_t)byte;
  }
}

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
  for (const void* f : {(const void*)quantize_e4m3, (const void*)dequant_e4m3})
    if (cudaFuncGetAttributes(&a, f) != cudaSuccess) {
      cudaGetLastError();
      return HEXLIB_B200_ERR_CUDA;
    }
  return HEXLIB_B200_OK;
}

int launch_quantize_e4m3(const void* x, void* codes, void* scales, int64_t R, int K,
                         cudaStream_t s) {
  quantize_e4m3<<<grid_for(R * e4m3_scale_groups(K) * 4 * 32), kThreads, 0, s>>>(
      (const __half*)x, (uint8_t*)codes, (uint8_t*)scales, R, K, K, 1);
  return launched();
}

int launch_quantize_weight_e4m3(const void* w, void* codes, void* scales, int K, int N,
                                cudaStream_t s) {
  quantize_e4m3<<<grid_for(N * e4m3_scale_groups(K) * 4 * 32), kThreads, 0, s>>>(
      (const __half*)w, (uint8_t*)codes, (uint8_t*)scales, N, K, 1, N);
  return launched();
}

int launch_dequant_e4m3(const void* codes, const void* scales, void* out, int64_t R, int K,
                        cudaStream_t s) {
  dequant_e4m3<<<grid_for(R * K), kThreads, 0, s>>>((const uint8_t*)codes,
                                                    (const uint8_t*)scales, (__half*)out, R, K);
  return launched();
}

}  // namespace hb

// k_gemm_e4m3.cu -- out = act(a @ w + bias) (+ resid) for operands in their e4m3
// form (hb_e4m3.cuh), fp32 sums, one rounding to fp16.
#include <cuda_runtime.h>

#include "hb_device.cuh"
#include "hb_e4m3.cuh"
#include "hb_kernels.h"

namespace hb {
namespace {

// 64 x 64 outputs per CTA, 32 of K at a time through shared memory, the scale
// applied as each code is read (a product of a code and a power of two is exact).
__global__ void __launch_bounds__(256) gemm_e4m3_simt(const GemmE4m3Desc g) {
  __shared__ float sa[32][65], sw[32][65];
  const int64_t pitch = (g.K + 127) / 128 * 128;
  const uint8_t* a = (const uint8_t*)g.a;
  const uint8_t* w = (const uint8_t*)g.w;
  const int tiles_n = (g.N + 63) / 64;
  const int64_t total = (int64_t)((g.M + 63) / 64) * tiles_n;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int m0 = (int)(t / tiles_n) * 64, n0 = (int)(t % tiles_n) * 64;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < pitch; k0 += 32) {
      for (int e = threadIdx.x; e < 64 * 32; e += 256) {
        const int row = e / 32, kk = e % 32, m = m0 + row, n = n0 + row, b = k0 >> 7;
        sa[kk][row] = m < g.M ? e4m3_value(a[m * pitch + k0 + kk]) *
                                    e4m3_scale(((const uint8_t*)g.a_scales)[e4m3_scale_at(m, b, g.M)])
                              : 0.f;
        sw[kk][row] = n < g.N ? e4m3_value(w[n * pitch + k0 + kk]) *
                                    e4m3_scale(((const uint8_t*)g.w_scales)[e4m3_scale_at(n, b, g.N)])
                              : 0.f;
      }
      __syncthreads();
      for (int kk = 0; kk < 32; ++kk)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[kk][ty * 4 + i], sw[kk][tx * 4 + j], acc[i][j]);
      __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
        if (m >= g.M || n >= g.N) continue;
        float v = acc[i][j] + (g.bias ? g.bias[n] : 0.f);
        if (g.act == 1) v = gelu_tanh_f(v);
        if (g.act == 2) v = gelu_erf_f(v);
        const int64_t o = (int64_t)m * g.N + n;
        if (g.resid) v += __half2float(((const __half*)g.resid)[o]);
        ((__half*)g.out)[o] = __float2half_rn(v);
      }
  }
}

}  // namespace

int gemm_e4m3_kernels_init() {
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, gemm_e4m3_simt) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

int launch_gemm_e4m3(const GemmE4m3Desc& g, int* err, cudaStream_t s) {
  const int64_t tiles = (int64_t)((g.M + 63) / 64) * ((g.N + 63) / 64);
  gemm_e4m3_simt<<<(int)(tiles < 148 * 4 ? tiles : 148 * 4), 256, 0, s>>>(g);
  if (cudaPeekAtLastError() != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

}  // namespace hb

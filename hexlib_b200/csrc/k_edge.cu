// k_edge.cu -- the edge between two transformer blocks in one pass over the rows:
//   u  = norm(y) (or y);  x' = fp16(x_scale x + y_scale f(gate) u);
//   h  = fp16(norm(x')), or that in its e4m3 form (hb_e4m3.cuh).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "hb_e4m3.cuh"
#include "hb_kernels.h"

namespace hb {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float gate_value(float g, int act) {
  switch (act) {
    case HEXLIB_B200_GATE_SIGMOID: return 1.f / (1.f + expf(-g));
    case HEXLIB_B200_GATE_SILU: return g / (1.f + expf(-g));
    case HEXLIB_B200_GATE_TANH: return tanhf(g);
  }
  return g;
}

// One value of a norm, every rounding written out: the fp16 and the 8-bit form (and
// every row layout) then give the same bits from the same moments.
__device__ __forceinline__ float normed(float v, float2 ms, float w, const float* b, int c) {
  v = __fmul_rn(__fsub_rn(v, ms.x), ms.y);
  return b ? fmaf(v, w, b[c]) : __fmul_rn(v, w);
}
__device__ __forceinline__ __half blended(float x_scale, float x, float y_scale, float u) {
  return __float2half_rn(fmaf(x_scale, x, __fmul_rn(y_scale, u)));
}

__device__ __forceinline__ float cta_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < kThreads / 32; ++i) t += red[i];
  __syncthreads();
  return t;
}

// mean (0 for rms) and 1 / sqrt(mean of squared deviations + eps) of a row
__device__ __forceinline__ float2 moments(const __half* v, int C, bool layer, float eps,
                                          float* red) {
  float mean = 0.f;
  if (layer) {
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) s += __half2float(v[c]);
    mean = cta_sum(s, red) / C;
  }
  float ss = 0.f;
  for (int c = threadIdx.x; c < C; c += kThreads) {
    const float d = __half2float(v[c]) - mean;
    ss = fmaf(d, d, ss);
  }
  return make_float2(mean, 1.f / sqrtf(cta_sum(ss, red) / C + eps));
}

// One CTA per row, its values read again from global memory for each pass; a thread
// reads x' back only where it wrote it, and the sums between the passes order them.
template <bool E4M3>
__global__ void __launch_bounds__(kThreads) edge_rows(const EdgeDesc d) {
  __shared__ float red[kThreads / 32];
  const bool layer = d.norm == HEXLIB_B200_NORM_LAYER;
  const int per_gate = d.gate ? d.R / d.gate_rows : 1;
  for (int64_t r = blockIdx.x; r < d.R; r += gridDim.x) {
    const __half* x = (const __half*)d.x + r * d.C;
    if (d.y) {
      const __half* y = (const __half*)d.y + r * d.C;
      __half* xo = (__half*)d.x_out + r * d.C;
      float2 ms = make_float2(0.f, 1.f);
      if (d.post_w) ms = moments(y, d.C, layer, d.eps, red);
      for (int c = threadIdx.x; c < d.C; c += kThreads) {
        float u = __half2float(y[c]);
        if (d.post_w) u = normed(u, ms, d.post_w[c], d.post_b, c);
        if (d.gate)
          u = __fmul_rn(u, gate_value(__half2float(((const __half*)d.gate)[(r / per_gate) * d.C + c]),
                                      d.gate_act));
        xo[c] = blended(d.x_scale, __half2float(x[c]), d.y_scale, u);
      }
      x = xo;
    }
    if (!d.pre_w) continue;
    const float2 ms = moments(x, d.C, layer, d.eps, red);
    auto h_of = [&](int c) {
      return __float2half_rn(normed(__half2float(x[c]), ms, d.pre_w[c], d.pre_b, c));
    };
    if constexpr (!E4M3) {
      for (int c = threadIdx.x; c < d.C; c += kThreads) ((__half*)d.h)[r * d.C + c] = h_of(c);
    } else {
      // a warp per block of 128; the x' of other threads' columns is visible after
      // the barriers inside moments()
      const int blocks = (d.C + 127) / 128, padded = (blocks + 3) / 4 * 4, lane = threadIdx.x & 31;
      uint8_t* codes = (uint8_t*)d.h_codes + r * (int64_t)blocks * 128;
      for (int b = threadIdx.x >> 5; b < padded; b += kThreads / 32) {
        uint32_t byte = kE4m3One;
        if (b < blocks) {
          float v[4], amax = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = b * 128 + lane + 32 * j;
            v[j] = c < d.C ? __half2float(h_of(c)) : 0.f;
            if (isfinite(v[j])) amax = fmaxf(amax, fabsf(v[j]));
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          byte = e4m3_scale_byte(amax);
          const float inv = e4m3_inverse(byte);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            codes[b * 128 + lane + 32 * j] = (uint8_t)e4m3_code(v[j], inv);
        }
        if (lane == 0) ((uint8_t*)d.h_scales)[e4m3_scale_at(r, b, d.R)] = (uint8_t)byte;
      }
    }
  }
}

}  // namespace

int edge_kernels_init() {
  cudaFuncAttributes a;
  for (const void* f : {(const void*)edge_rows<false>, (const void*)edge_rows<true>})
    if (cudaFuncGetAttributes(&a, f) != cudaSuccess) {
      cudaGetLastError();
      return HEXLIB_B200_ERR_CUDA;
    }
  return HEXLIB_B200_OK;
}

int launch_edge(const EdgeDesc& d, cudaStream_t s) {
  const int grid = d.R < 148 * 8 ? d.R : 148 * 8;
  if (d.h_codes)
    edge_rows<true><<<grid, kThreads, 0, s>>>(d);
  else
    edge_rows<false><<<grid, kThreads, 0, s>>>(d);
  if (cudaPeekAtLastError() != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

}  // namespace hb

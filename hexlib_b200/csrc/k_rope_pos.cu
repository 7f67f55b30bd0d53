// k_rope_pos.cu -- rotary positions from integer positions and a table of
// frequencies in 64-bit fixed-point turns, and the host function that fills it.
//
// The phase of pair j at position p is p * table[j] / 2^64 turns. Angles only
// matter modulo a turn, so the 64-bit product modulo 2^64 is the phase reduced
// exactly, at any position: what is lost is the table's own rounding (2^-53
// relative) and the 24 bits an fp32 keeps of the reduced phase. fp32 radians, by
// contrast, are off by 0.06 at position 10^6.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "hb_kernels.h"

namespace hb {
namespace {

constexpr int kThreads = 256;

// One thread per pair (or pair of elements past `rot`) of every token and head.
__global__ void rope_pos_pairs(const RopePosDesc d) {
  const int half = d.rot >> 1;
  const int per_head = half + (d.D - d.rot);
  const int64_t total = (int64_t)d.T * d.H * per_head;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int j = (int)(i % per_head);
    const int64_t th = i / per_head;
    const int64_t t = th / d.H;
    const int h = (int)(th % d.H);
    const __half* x = (const __half*)d.x + t * d.x_stride + (int64_t)h * d.D;
    __half* y = (__half*)d.y + t * d.y_stride + (int64_t)h * d.D;
    if (j >= half) {
      y[d.rot + j - half] = x[d.rot + j - half];
      continue;
    }
    const int ax = d.axis ? min(max(d.axis[j], 0), d.n_axes - 1) : 0;
    const int64_t pos = d.positions[(int64_t)ax * d.T + t];
    const uint64_t phase = (uint64_t)pos * d.table[j];
    float s, c;
    sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);
    const int ia = d.layout ? 2 * j : j, ib = d.layout ? 2 * j + 1 : j + half;
    const float a = __half2float(x[ia]), b = __half2float(x[ib]);
    s *= d.mscale;
    c *= d.mscale;
    y[ia] = __float2half_rn(a * c - b * s);
    y[ib] = __float2half_rn(a * s + b * c);
  }
}

}  // namespace

int rope_pos_kernels_init() {
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, rope_pos_pairs) != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

int launch_rope_pos(const RopePosDesc& d, cudaStream_t s) {
  const int64_t total = (int64_t)d.T * d.H * (d.D - d.rot / 2);
  const int64_t blocks = (total + kThreads - 1) / kThreads;
  rope_pos_pairs<<<(int)(blocks < 148 * 8 ? blocks : 148 * 8), kThreads, 0, s>>>(d);
  if (cudaPeekAtLastError() != cudaSuccess) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

}  // namespace hb

extern "C" int hexlib_b200_rope_pos_table(int scaling, int rot, double theta, double factor,
                                          double length, double low, double high,
                                          uint64_t* table, float* mscale) {
  const bool factored = scaling != HEXLIB_B200_ROPE_SCALE_NONE;
  const bool banded = scaling == HEXLIB_B200_ROPE_SCALE_YARN ||
                      scaling == HEXLIB_B200_ROPE_SCALE_BANDED;
  auto positive = [](double v) { return isfinite(v) && v > 0; };
  if (scaling < HEXLIB_B200_ROPE_SCALE_NONE || scaling > HEXLIB_B200_ROPE_SCALE_BANDED ||
      rot <= 0 || (rot & 1) || !isfinite(theta) || !(theta > 1) || !table || !mscale ||
      (factored && !positive(factor)) ||
      (banded && (!positive(length) || !positive(low) || !positive(high) || !(low < high))) ||
      (scaling == HEXLIB_B200_ROPE_SCALE_BASE && rot < 4))
    return HEXLIB_B200_ERR_INVAL_PARAMS;
  const double turn = 2 * M_PI;
  if (scaling == HEXLIB_B200_ROPE_SCALE_BASE) theta *= pow(factor, rot / (rot - 2.0));
  if (!isfinite(theta) || !(theta > 1)) return HEXLIB_B200_ERR_INVAL_PARAMS;
  const int pairs = rot / 2;
  double first = 0, last = 0;
  if (scaling == HEXLIB_B200_ROPE_SCALE_YARN) {
    // the pair whose frequency turns n times in `length` positions
    auto pair_of = [&](double n) {
      return rot * log(length / (n * turn)) / (2 * log(theta));
    };
    first = fmax(floor(pair_of(high)), 0.0);
    last = fmin(ceil(pair_of(low)), rot - 1.0);
    if (!(last > first)) last = first + 0.001;
  }
  for (int j = 0; j < pairs; ++j) {
    double f = pow(theta, -2.0 * j / rot);
    if (scaling == HEXLIB_B200_ROPE_SCALE_LINEAR) {
      f /= factor;
    } else if (banded) {
      const double keep = scaling == HEXLIB_B200_ROPE_SCALE_YARN
                              ? 1 - fmin(fmax((j - first) / (last - first), 0.0), 1.0)
                              : fmin(fmax((length * f / turn - low) / (high - low), 0.0), 1.0);
      f = f / factor * (1 - keep) + f * keep;
    }
    double turns = f / turn;
    turns -= floor(turns);                       // positions are whole, so turns are modulo 1
    table[j] = turns >= 1 ? 0 : (uint64_t)(turns * 0x1p64);   // (a product by 2^64 is exact)
  }
  *mscale = scaling == HEXLIB_B200_ROPE_SCALE_YARN && factor > 1 ? (float)(0.1 * log(factor) + 1)
                                                                 : 1.0f;
  return HEXLIB_B200_OK;
}

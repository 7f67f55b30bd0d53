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

struct RopeShape {
  int tokens;      // of a CTA
  int pairs;       // rot / 2
  int rot_items;   // items of a head that rotate, then those that are copied
  int items;       // of a head
  int head_split;  // CTAs that share a token tile's heads
  int heads;       // of a CTA
};

// The phases of a tile of tokens are turned into cosines and sines once, in shared
// memory, for all heads; then a thread takes an item of 16 (half layout: 8 pairs) or 8
// (interleaved: 4 pairs) elements of a head at a time, in 16-byte loads and stores.
// An item's cosines lie `stride` apart, so that the threads of a warp, which take
// consecutive items, read consecutive words.
//
// VEC: D and the row strides whole 16-byte vectors, rot whole items. Otherwise an item
// is one pair, or one element copied.
template <bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_pos_tile(const RopePosDesc d, const RopeShape sh) {
  extern __shared__ float2 cs[];                       // [tokens][pairs]
  constexpr int PAIRS = VEC ? (INTERLEAVED ? 4 : 8) : 1;
  const int tile = blockIdx.x / sh.head_split;
  const int h0 = (blockIdx.x % sh.head_split) * sh.heads;
  const int heads = min(sh.heads, d.H - h0);
  const int64_t t0 = (int64_t)tile * sh.tokens;
  const int tokens = (int)min((int64_t)sh.tokens, d.T - t0);
  for (int i = threadIdx.x; i < tokens * sh.pairs; i += kThreads) {
    const int t = i / sh.pairs, j = i - t * sh.pairs;
    const int ax = d.axis ? min(max(__ldg(d.axis + j), 0), d.n_axes - 1) : 0;
    const int64_t pos = __ldg(d.positions + (int64_t)ax * d.T + t0 + t);
    const uint64_t phase = (uint64_t)pos * __ldg((const unsigned long long*)d.table + j);
    float s, c;
    sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);
    cs[t * sh.pairs + (j % PAIRS) * sh.rot_items + j / PAIRS] =
        make_float2(d.mscale * c, d.mscale * s);
  }
  __syncthreads();
  const bool in_place = d.x == d.y;
  const int per_head = in_place ? sh.rot_items : sh.items;
  const int half = d.rot >> 1;
  const int total = tokens * heads * per_head;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int th = i / per_head, item = i - th * per_head;
    const int t = th / heads, h = h0 + th - t * heads;
    const __half* x = (const __half*)d.x + (t0 + t) * d.x_stride + (int64_t)h * d.D;
    __half* y = (__half*)d.y + (t0 + t) * d.y_stride + (int64_t)h * d.D;
    if (item >= sh.rot_items) {
      const int e = d.rot + (item - sh.rot_items) * (VEC ? 8 : 1);
      if constexpr (VEC) *reinterpret_cast<uint4*>(y + e) = *reinterpret_cast<const uint4*>(x + e);
      else y[e] = x[e];
      continue;
    }
    const float2* c = cs + t * sh.pairs + item;
    if constexpr (!VEC) {
      const int ia = INTERLEAVED ? 2 * item : item, ib = INTERLEAVED ? ia + 1 : ia + half;
      const float a = __half2float(x[ia]), b = __half2float(x[ib]);
      y[ia] = __float2half_rn(a * c->x - b * c->y);
      y[ib] = __float2half_rn(a * c->y + b * c->x);
    } else if constexpr (INTERLEAVED) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + item * 8);
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[q]));
        const float2 k = c[q * sh.rot_items];
        const __half2 r = __floats2half2_rn(f.x * k.x - f.y * k.y, f.x * k.y + f.y * k.x);
        w[q] = *reinterpret_cast<const uint32_t*>(&r);
      }
      *reinterpret_cast<uint4*>(y + item * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      const uint4 ua = *reinterpret_cast<const uint4*>(x + item * 8);
      const uint4 ub = *reinterpret_cast<const uint4*>(x + half + item * 8);
      uint32_t a[4] = {ua.x, ua.y, ua.z, ua.w}, b[4] = {ub.x, ub.y, ub.z, ub.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a[q]));
        const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b[q]));
        const float2 k0 = c[2 * q * sh.rot_items], k1 = c[(2 * q + 1) * sh.rot_items];
        const __half2 ra = __floats2half2_rn(fa.x * k0.x - fb.x * k0.y, fa.y * k1.x - fb.y * k1.y);
        const __half2 rb = __floats2half2_rn(fa.x * k0.y + fb.x * k0.x, fa.y * k1.y + fb.y * k1.x);
        a[q] = *reinterpret_cast<const uint32_t*>(&ra);
        b[q] = *reinterpret_cast<const uint32_t*>(&rb);
      }
      *reinterpret_cast<uint4*>(y + item * 8) = make_uint4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<uint4*>(y + half + item * 8) = make_uint4(b[0], b[1], b[2], b[3]);
    }
  }
}

constexpr int kMaxPairBytes = 96 * 1024;   // cosines and sines of a tile

}  // namespace

int rope_pos_kernels_init() {
  for (auto k : {rope_pos_tile<true, true>, rope_pos_tile<true, false>, rope_pos_tile<false, true>,
                 rope_pos_tile<false, false>})
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPairBytes) !=
        cudaSuccess) {
      cudaGetLastError();
      return HEXLIB_B200_ERR_CUDA;
    }
  return HEXLIB_B200_OK;
}

int launch_rope_pos(const RopePosDesc& d, cudaStream_t s) {
  const bool inter = d.layout == HEXLIB_B200_ROPE_INTERLEAVED;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.y) |
                         static_cast<uintptr_t>(2 * d.x_stride) |
                         static_cast<uintptr_t>(2 * d.y_stride) | static_cast<uintptr_t>(2 * d.D);
  const bool vec = bits % 16 == 0 && d.rot % (inter ? 8 : 16) == 0;
  RopeShape sh;
  sh.pairs = d.rot / 2;
  sh.rot_items = vec ? sh.pairs / (inter ? 4 : 8) : sh.pairs;
  sh.items = sh.rot_items + (vec ? (d.D - d.rot) / 8 : d.D - d.rot);
  if ((int64_t)sh.pairs * 8 > kMaxPairBytes) return HEXLIB_B200_ERR_INVAL_PARAMS;
  // tokens of a CTA: about a cosine for each thread and a few items for each, but no
  // fewer CTAs than SMs; few tokens split their heads over CTAs instead
  const int64_t per_token = (int64_t)d.H * sh.items;
  int64_t tokens = kThreads / sh.pairs;
  if (tokens > 4 * kThreads / per_token) tokens = 4 * kThreads / per_token;
  if (tokens > d.T / 148) tokens = d.T / 148;
  if (tokens < 1) tokens = 1;
  sh.tokens = (int)tokens;
  const int64_t tiles = (d.T + tokens - 1) / tokens;
  int64_t split = 296 / tiles;
  if (split > (per_token + kThreads - 1) / kThreads) split = (per_token + kThreads - 1) / kThreads;
  if (split > d.H) split = d.H;
  if (split < 1) split = 1;
  sh.heads = (int)((d.H + split - 1) / split);
  sh.head_split = (d.H + sh.heads - 1) / sh.heads;
  if (tiles * sh.head_split > 0x7fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  const unsigned grid = (unsigned)(tiles * sh.head_split);
  const size_t smem = (size_t)sh.tokens * sh.pairs * sizeof(float2);
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, smem, s>>>(d, sh); };
  if (vec) inter ? go(rope_pos_tile<true, true>) : go(rope_pos_tile<true, false>);
  else inter ? go(rope_pos_tile<false, true>) : go(rope_pos_tile<false, false>);
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

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

#include "hb_device.cuh"
#include "hb_kernels.h"

namespace hb {
namespace {

constexpr int kThreads = 256;

struct RopeShape {
  int tokens;      // of a CTA
  int pairs;       // rot / 2
  int rot_items;   // items of a head that rotate, then those that are copied
  int copy_w;      // elements of a copied item (8, 4 or 2; 1 where nothing is a vector)
  int items;       // of a head, of them the ones to do (in place nothing is copied)
  int head_split;  // CTAs that share a token tile's heads
  int heads;       // of a CTA
  // 2^32 / items and 2^32 / heads, rounded up: for more than one, i / items is the high
  // word of the product for every i with i * items < 2^32
  uint32_t per_item, per_head;
};

// The cosine and sine of every pair of a tile of tokens, for all its heads, pair j at
// (j % P) * n + j / P: the P pairs of an item n apart, so that the threads of a warp,
// which take consecutive items, read consecutive words.
template <int P>
__device__ __forceinline__ void tile_phases(const RopePosDesc& d, const RopeShape& sh, int64_t t0,
                                            int tokens, float2* cs) {
  for (int i = threadIdx.x; i < tokens * sh.pairs; i += kThreads) {
    const int t = i / sh.pairs, j = i - t * sh.pairs;
    const int ax = d.axis ? min(max(__ldg(d.axis + j), 0), d.n_axes - 1) : 0;
    const int64_t pos = __ldg(d.positions + (int64_t)ax * d.T + t0 + t);
    const uint64_t phase = (uint64_t)pos * __ldg((const unsigned long long*)d.table + j);
    float s, c;
    sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);
    cs[t * sh.pairs + (j % P) * sh.rot_items + j / P] = make_float2(d.mscale * c, d.mscale * s);
  }
}

// Rows of whole vectors of W = 8, 4 or 2 elements: an item is W elements of either half
// of a head (half layout, W pairs), W elements (interleaved, W / 2 pairs), or one vector
// copied, as wide as its rows allow.
// Bound by memory; a thread has two items in
// flight, the first two from before the phases are formed, which hides the positions'
// way through memory behind the rows' (32768 tokens of 40 of 48 heads of 128: 112 us,
// 5.97 TB/s; 135 without, 118 with four items in flight and half the warps; 4097 tokens
// of 24 heads of 64, three axes: 8.0 us, of which 3.8 are memory's; 32768 of 40 heads of 96,
// 24 rotated by halves: 101 us on vectors of 4 and copies of 8, 145 with copies of 4, over
// 250 pair by pair).
constexpr int kBatch = 2;

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&w)[W / 2], const __half* p) {
  if constexpr (W == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (W == 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
template <int W>
__device__ __forceinline__ void store_words(__half* p, const uint32_t (&w)[W / 2]) {
  if constexpr (W == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (W == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

template <int W, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_pos_vec(const RopePosDesc d, const RopeShape sh) {
  extern __shared__ float2 cs[];                       // [tokens][pairs]
  constexpr int VECS = INTERLEAVED ? 1 : 2;            // of a rotating item
  const int tile = blockIdx.x / sh.head_split;
  const int h0 = (blockIdx.x % sh.head_split) * sh.heads;
  const int heads = min(sh.heads, d.H - h0);
  const int64_t t0 = (int64_t)tile * sh.tokens;
  const int tokens = (int)min((int64_t)sh.tokens, d.T - t0);
  // (the last CTA of a split may have fewer heads; items past them are skipped)
  const uint32_t total = tokens * sh.heads * sh.items;
  const int half = d.rot >> 1;
  struct Item {
    int t, h, item;                                    // h < 0: none
  };
  auto item_of = [&](uint32_t i) {
    const uint32_t th = sh.items == 1 ? i : __umulhi(i, sh.per_item);
    const uint32_t t = sh.heads == 1 ? th : __umulhi(th, sh.per_head);
    const int h = th - t * sh.heads;
    return Item{(int)t, i < total && h < heads ? h : -1, (int)(i - th * sh.items)};
  };
  auto first_of = [&](const Item& m) {                 // its first element within the head
    return m.item < sh.rot_items ? m.item * W : d.rot + (m.item - sh.rot_items) * sh.copy_w;
  };
  uint32_t u[kBatch][VECS][W / 2], v[kBatch][4];      // (v: copied, where wider than W)
  auto load = [&](uint32_t i0) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const Item m = item_of(i0 + b * kThreads);
      if (m.h < 0) continue;
      const __half* x = (const __half*)d.x + (t0 + m.t) * d.x_stride + (int64_t)(h0 + m.h) * d.D +
                        first_of(m);
      if (W < 8 && m.item >= sh.rot_items) {
        if (sh.copy_w == 8) load_words<8>(v[b], x);
        else if (sh.copy_w == 4) load_words<4>(reinterpret_cast<uint32_t(&)[2]>(v[b]), x);
        else load_words<2>(reinterpret_cast<uint32_t(&)[1]>(v[b]), x);
        continue;
      }
      load_words<W>(u[b][0], x);
      if (!INTERLEAVED && m.item < sh.rot_items) load_words<W>(u[b][VECS - 1], x + half);
    }
  };
  load(threadIdx.x);
  tile_phases<INTERLEAVED ? W / 2 : W>(d, sh, t0, tokens, cs);
  __syncthreads();
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += kBatch * kThreads) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const Item m = item_of(i0 + b * kThreads);
      if (m.h < 0) continue;
      __half* y = (__half*)d.y + (t0 + m.t) * d.y_stride + (int64_t)(h0 + m.h) * d.D + first_of(m);
      if (m.item < sh.rot_items) {
        const float2* c = cs + m.t * sh.pairs + m.item;
        uint32_t(&a)[W / 2] = u[b][0];
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int q = 0; q < W / 2; ++q) {
            const float2 f = unpack_half2(a[q]), k = c[q * sh.rot_items];
            a[q] = pack_half2(f.x * k.x - f.y * k.y, f.x * k.y + f.y * k.x);
          }
        } else {
          uint32_t(&e)[W / 2] = u[b][VECS - 1];
#pragma unroll
          for (int q = 0; q < W / 2; ++q) {
            const float2 fa = unpack_half2(a[q]), fb = unpack_half2(e[q]);
            const float2 k0 = c[2 * q * sh.rot_items], k1 = c[(2 * q + 1) * sh.rot_items];
            a[q] = pack_half2(fa.x * k0.x - fb.x * k0.y, fa.y * k1.x - fb.y * k1.y);
            e[q] = pack_half2(fa.x * k0.y + fb.x * k0.x, fa.y * k1.y + fb.y * k1.x);
          }
          store_words<W>(y + half, e);
        }
      }
      if (W < 8 && m.item >= sh.rot_items) {
        if (sh.copy_w == 8) store_words<8>(y, v[b]);
        else if (sh.copy_w == 4) store_words<4>(y, reinterpret_cast<uint32_t(&)[2]>(v[b]));
        else store_words<2>(y, reinterpret_cast<uint32_t(&)[1]>(v[b]));
        continue;
      }
      store_words<W>(y, u[b][0]);
    }
    load(i0 + kBatch * kThreads);
  }
}

// Any rows: an item is one pair, or one element copied (32768 tokens of 40 heads of 128 from
// an odd row pitch: 378 us interleaved, 397 in halves, 112 on vectors; four two-byte accesses
// and a division of 64 bits an item).
template <bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_pos_any(const RopePosDesc d, const RopeShape sh) {
  extern __shared__ float2 cs[];
  const int tile = blockIdx.x / sh.head_split;
  const int h0 = (blockIdx.x % sh.head_split) * sh.heads;
  const int heads = min(sh.heads, d.H - h0);
  const int64_t t0 = (int64_t)tile * sh.tokens;
  const int tokens = (int)min((int64_t)sh.tokens, d.T - t0);
  tile_phases<1>(d, sh, t0, tokens, cs);
  __syncthreads();
  const int half = d.rot >> 1;
  const int64_t total = (int64_t)tokens * heads * sh.items;
  for (int64_t i = threadIdx.x; i < total; i += kThreads) {
    const int64_t th = i / sh.items;
    const int item = (int)(i - th * sh.items);
    const int t = (int)(th / heads), h = h0 + (int)(th - (int64_t)t * heads);
    const __half* x = (const __half*)d.x + (t0 + t) * d.x_stride + (int64_t)h * d.D;
    __half* y = (__half*)d.y + (t0 + t) * d.y_stride + (int64_t)h * d.D;
    if (item >= sh.rot_items) {
      const int e = d.rot + item - sh.rot_items;
      y[e] = x[e];
      continue;
    }
    const float2 c = cs[t * sh.pairs + item];
    const int ia = INTERLEAVED ? 2 * item : item, ib = INTERLEAVED ? ia + 1 : ia + half;
    const float a = __half2float(x[ia]), b = __half2float(x[ib]);
    y[ia] = __float2half_rn(a * c.x - b * c.y);
    y[ib] = __float2half_rn(a * c.y + b * c.x);
  }
}

constexpr int kMaxPairBytes = kRopePosMostRot / 2 * sizeof(float2);   // those of a tile of one token

}  // namespace

int rope_pos_kernels_init() {
  for (auto k : {rope_pos_vec<8, true>, rope_pos_vec<8, false>, rope_pos_vec<4, true>,
                 rope_pos_vec<4, false>, rope_pos_vec<2, true>, rope_pos_vec<2, false>,
                 rope_pos_any<true>, rope_pos_any<false>})
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPairBytes) !=
        cudaSuccess) {
      cudaGetLastError();
      return HEXLIB_B200_ERR_CUDA;
    }
  return HEXLIB_B200_OK;
}

int launch_rope_pos(const RopePosDesc& desc, cudaStream_t s) {
  RopePosDesc d = desc;
  if (d.n_axes == 1) d.axis = nullptr;     // every number clamps to 0
  const bool inter = d.layout == HEXLIB_B200_ROPE_INTERLEAVED;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.y) |
                         2 * static_cast<uintptr_t>(d.x_stride) |
                         2 * static_cast<uintptr_t>(d.y_stride) | 2 * static_cast<uintptr_t>(d.D);
  // the widest vector that divides the rows and the rotated part (each half of it)
  const int part = inter ? d.rot : d.rot / 2;
  int w = 8;
  while (w > 1 && (bits % (2 * w) != 0 || part % w != 0)) w /= 2;
  if (d.D > 4096) w = 1;
  RopeShape sh;
  sh.pairs = d.rot / 2;
  sh.rot_items = w > 1 ? part / w : sh.pairs;
  sh.copy_w = w;                           // (w divides rot, D and the strides)
  while (w > 1 && sh.copy_w < 8 &&
         ((bits | static_cast<uintptr_t>(2 * d.rot)) % (4 * sh.copy_w)) == 0)
    sh.copy_w *= 2;
  sh.items = sh.rot_items + (d.x == d.y ? 0 : (d.D - d.rot) / sh.copy_w);
  // tokens of a CTA: a few cosines and about eight items to a thread, but four CTAs to
  // an SM where there are tokens for them; few tokens split their heads over CTAs
  const int64_t per_token = (int64_t)d.H * sh.items;
  int64_t tokens = 2 * kThreads / sh.pairs;
  if (tokens > 8 * kThreads / per_token) tokens = 8 * kThreads / per_token;
  if (tokens > d.T / (4 * 148)) tokens = d.T / (4 * 148);
  if (tokens < 1) tokens = 1;
  sh.tokens = (int)tokens;
  const int64_t tiles = (d.T + tokens - 1) / tokens;
  int64_t split = 296 / tiles, most = (per_token + kThreads - 1) / kThreads;
  if (split > most) split = most;
  const int64_t least = ((int64_t)d.H + 1023) / 1024;   // (items in 32 bits)
  if (split < least) split = least;
  if (split > d.H) split = d.H;
  if (split < 1) split = 1;
  sh.heads = (int)((d.H + split - 1) / split);
  sh.head_split = (int)(((int64_t)d.H + sh.heads - 1) / sh.heads);
  if (tiles * sh.head_split > 0x7fffffff) return HEXLIB_B200_ERR_INVAL_PARAMS;
  sh.per_item = (uint32_t)(((1ull << 32) + sh.items - 1) / sh.items);
  sh.per_head = (uint32_t)(((1ull << 32) + sh.heads - 1) / sh.heads);
  const unsigned grid = (unsigned)(tiles * sh.head_split);
  const size_t smem = (size_t)sh.tokens * sh.pairs * sizeof(float2);
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, smem, s>>>(d, sh); };
  switch (w) {
    case 8: inter ? go(rope_pos_vec<8, true>) : go(rope_pos_vec<8, false>); break;
    case 4: inter ? go(rope_pos_vec<4, true>) : go(rope_pos_vec<4, false>); break;
    case 2: inter ? go(rope_pos_vec<2, true>) : go(rope_pos_vec<2, false>); break;
    default: inter ? go(rope_pos_any<true>) : go(rope_pos_any<false>);
  }
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

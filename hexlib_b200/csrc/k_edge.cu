// k_edge.cu -- the edge between two transformer blocks in one pass over the rows:
//   u  = norm(y) (or y);  x' = fp16(x_scale x + y_scale f(gate) u);
//   h  = fp16(norm(x')), or that in its e4m3 form (hb_e4m3.cuh).
// Bound by memory: 4 bytes read and 4 (3 with 8-bit h) written per value, 2 more
// where the gate has a row of its own for every row.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "hb_device.cuh"
#include "hb_e4m3.cuh"
#include "hb_kernels.h"

namespace hb {
namespace {

constexpr int kThreads = 256;

// 1 / (1 + e^-g) of a pair of fp16 values. e^-g = 2^(-g L), L = log2(e): with L cut
// to its first 13 bits the product by g's 11 is exact, and what was cut enters as
// 1 + d, d = -g (L - L13) ln 2 (|d| < 2^-9 where the result is above 2^-32), so the
// error is that of 2^x and the reciprocal, a few 2^-23.
__device__ __forceinline__ float2 sigmoid2(float2 g) {
  constexpr float L13 = 1.442626953125f;
  constexpr float D = 4.719484e-5f;                   // (log2(e) - L13) ln 2
  const float2 t = __fmul2_rn(g, make_float2(-L13, -L13));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  float2 d = __fmul2_rn(g, make_float2(-D, -D));
  d = make_float2(fmaxf(d.x, -1.f), fmaxf(d.y, -1.f));   // an infinite g: 0 (1 + d) is 0
  e = __fadd2_rn(__ffma2_rn(e, d, e), make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
  return r;
}

__device__ __forceinline__ float gate_value(float g, int act) {
  if (act == HEXLIB_B200_GATE_NONE) return g;
  if (act == HEXLIB_B200_GATE_TANH) return tanhf(g);
  const float s = sigmoid2(make_float2(g, g)).x;
  return act == HEXLIB_B200_GATE_SILU ? g * s : s;
}

__device__ __forceinline__ float blended(float x_scale, float x, float y_scale, float u) {
  return fmaf(x_scale, x, __fmul_rn(y_scale, u));
}

// 1 / sqrt(a): rsqrtf (2 ulp) and one Newton step, which leaves its own rounding. Every
// value of the row carries this error, and with it one in 2^18 codes of the 8-bit form
// fell on the other side of a tie.
__device__ __forceinline__ float inverse_root(float a) {
  const float y = rsqrtf(a);
  const float e = fmaf(-__fmul_rn(a, y), y, 1.f);
  return a < INFINITY ? fmaf(0.5f * y, e, y) : y;
}

// Sum over the G threads of a row: a warp, or the CTA of G threads through shared
// memory. The slots rotate, so that one barrier a sum suffices: a slot is written
// again only three barriers after it was read.
constexpr int kSumSlot = 16;                         // two sums of 8 warps
template <int G>
struct RowSum {
  float (*red)[kSumSlot];
  int slot = 0;
  static __device__ float of_warps(const float* r) {
    const float4 a = *reinterpret_cast<const float4*>(r);
    float v = (a.x + a.y) + (a.z + a.w);
    if constexpr (G == 256) {
      const float4 b = *reinterpret_cast<const float4*>(r + 4);
      v += (b.x + b.y) + (b.z + b.w);
    }
    return v;
  }
  __device__ float operator()(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (G == 32) return v;
    float* r = red[slot];
    slot = (slot + 1) & 3;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    return of_warps(r);
  }
  // two sums at once
  __device__ float2 operator()(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      v = __fadd2_rn(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o),
                                    __shfl_xor_sync(0xffffffffu, v.y, o)));
    if constexpr (G == 32) return v;
    float* r = red[slot];
    slot = (slot + 1) & 3;
    if ((threadIdx.x & 31) == 0) {
      r[threadIdx.x >> 5] = v.x;
      r[8 + (threadIdx.x >> 5)] = v.y;
    }
    __syncthreads();
    return make_float2(of_warps(r), of_warps(r + 8));
  }
};

// A layer norm takes the mean off each value before it multiplies: the rounding of
// mean inv in v inv - mean inv would stay in every value (0.5 in a constant row of 30000 at
// eps 1e-5, whose norm is its shift alone). What rounding leaves out of the mean is held as
// `rest` and taken off after it, where the values have become small, (d - rest) inv, and its
// square off the mean square of the d = v - mean.
struct Mean {
  float mean, rest;
};
// From a sum that is exact where the mean is far larger than the deviations: up to 8192
// values of one binade, 11 bits each, add up within 24 bits. The remainder of the division
// is then all that the mean lacks; the first one corrects the quotient.
__device__ __forceinline__ Mean mean_of(float s, int C, float per_c) {
  float m = __fmul_rn(s, per_c);
  m = fmaf(fmaf(-m, (float)C, s), per_c, m);
  return Mean{m, __fmul_rn(fmaf(-m, (float)C, s), per_c)};
}
// What an inexact sum left out of a mean shows in the sum of the deviations, sums.x; with
// that of their squares, sums.y: the rest and the variance.
__device__ __forceinline__ float2 corrected(float2 sums, int C, float per_c) {
  const float rest = mean_of(sums.x, C, per_c).mean;
  return make_float2(rest, fmaxf(fmaf(-rest, rest, __fmul_rn(sums.y, per_c)), 0.f));
}

// The columns of a thread. With rows of whole 16-byte vectors (WIDE), vector j of thread
// g is columns (j G + g) 8 to + 7, so 16 threads hold a block of 128. Otherwise a WARP
// holds a block, element i of a lane 32 (i % 4) further, so that scalar accesses of a
// warp are consecutive (1001 rows of 1203, tanh gate, 8-bit h: 15.0 us with the first
// order and scalar accesses, 12.1 with this one).
template <int G, bool WIDE>
struct Columns {
  int base;                                          // of element 0 of vector 0
  __device__ Columns() {
    const int g = G == 32 ? (threadIdx.x & 31) : threadIdx.x;
    base = WIDE ? g * 8 : (G == 32 ? 0 : (g >> 5) * 128) + (g & 31);
  }
  // from its first column, a constant once the loops are unrolled; rows below start there
  static __device__ __forceinline__ int off(int j, int i) {
    return WIDE ? j * G * 8 + i : (2 * j + (i >> 2)) * (G / 32) * 128 + (i & 3) * 32;
  }
  __device__ __forceinline__ int at(int j, int i) const { return base + off(j, i); }

  __device__ __forceinline__ void load(uint32_t (&w)[4], const __half* row, int j, int C) const {
    if constexpr (WIDE) {
      load8<8>(w, row + off(j, 0), C - at(j, 0));
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = (at(j, 2 * q) < C ? (uint32_t)p[off(j, 2 * q)] : 0u) |
               (at(j, 2 * q + 1) < C ? (uint32_t)p[off(j, 2 * q + 1)] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void store(__half* row, const uint32_t (&w)[4], int j, int C) const {
    if constexpr (WIDE) {
      if (at(j, 0) < C)
        *reinterpret_cast<uint4*>(row + off(j, 0)) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      unsigned short* p = reinterpret_cast<unsigned short*>(row);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (at(j, 2 * q) < C) p[off(j, 2 * q)] = (unsigned short)w[q];
        if (at(j, 2 * q + 1) < C) p[off(j, 2 * q + 1)] = (unsigned short)(w[q] >> 16);
      }
    }
  }
  __device__ __forceinline__ void load(float2 (&f)[4], const float* row, int j, int C) const {
    if constexpr (WIDE) {
      const float4* p = reinterpret_cast<const float4*>(row + off(j, 0));
      const bool in = at(j, 0) < C;
      const float4 a = in ? __ldg(p) : make_float4(0, 0, 0, 0);
      const float4 b = in ? __ldg(p + 1) : make_float4(0, 0, 0, 0);
      f[0] = make_float2(a.x, a.y);
      f[1] = make_float2(a.z, a.w);
      f[2] = make_float2(b.x, b.y);
      f[3] = make_float2(b.z, b.w);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        f[q] = make_float2(at(j, 2 * q) < C ? __ldg(row + off(j, 2 * q)) : 0.f,
                           at(j, 2 * q + 1) < C ? __ldg(row + off(j, 2 * q + 1)) : 0.f);
    }
  }
  // a vector past C, as zeros
  __device__ __forceinline__ void zero_out(uint32_t (&w)[4], int j, int C) const {
    if (WIDE && at(j, 0) >= C) w[0] = w[1] = w[2] = w[3] = 0;
  }
  // a pair with zeros past C, where a vector may end within the row
  __device__ __forceinline__ uint32_t pack_in(float2 f, int j, int q, int C) const {
    const uint32_t w = pack_half2(f.x, f.y);
    if constexpr (WIDE) return w;                    // the vector is in or not: see zero_out
    return (at(j, 2 * q) < C ? w & 0xffffu : 0u) | (at(j, 2 * q + 1) < C ? w & 0xffff0000u : 0u);
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A row in the registers of the G threads that share it, as floats, zeros past C. Each step runs over all V vectors
// between two branches, so that their chains overlap, in two-wide instructions with
// every rounding written out: the fp16 and the 8-bit form give the same bits.
template <int G, int V, bool WIDE>
struct Row {
  float2 v[V][4];
  Columns<G, WIDE> col;

  __device__ __forceinline__ void unpack(const uint32_t (&w)[V][4]) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[j][q] = unpack_half2(w[j][q]);
  }

  // norm(v) w + b, the moments taken over the whole row (the squared deviations of a
  // layer norm after its mean). Rows too long for an exact sum take what their mean
  // lacks from the sum of the deviations instead of the division's remainder.
  static constexpr bool LONG = G * V * 8 > 8192;
  __device__ __forceinline__ void norm(const float* w, const float* b, int C, float per_c,
                                       bool layer, float eps, RowSum<G>& sum) {
    float2 ss = both(0.f), ds = both(0.f);
    Mean m = {0.f, 0.f};
    if (layer) {
      float2 s = both(0.f);
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) s = __fadd2_rn(s, v[j][q]);
      m = mean_of(sum(s.x + s.y), C, per_c);
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float2 d = __fadd2_rn(v[j][q], both(-m.mean));
          if (col.at(j, WIDE ? 0 : 2 * q) >= C) d.x = 0.f;
          if (col.at(j, WIDE ? 0 : 2 * q + 1) >= C) d.y = 0.f;
          if (LONG) ds = __fadd2_rn(ds, d);
          ss = __ffma2_rn(d, d, ss);
          v[j][q] = d;
        }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) ss = __ffma2_rn(v[j][q], v[j][q], ss);
    }
    // the weights of a row by a CTA are read ahead of the sum's barrier (a warp's own row
    // has none, and registers to lose)
    constexpr bool AHEAD = G > 32;
    float2 ahead[AHEAD ? V : 1][4];
    if constexpr (AHEAD) {
#pragma unroll
      for (int j = 0; j < V; ++j) col.load(ahead[j], w + col.base, j, C);
    }
    auto weights = [&](int j, float2 (&wv)[4]) {
      if constexpr (AHEAD) {
#pragma unroll
        for (int q = 0; q < 4; ++q) wv[q] = ahead[j][q];
      } else {
        col.load(wv, w + col.base, j, C);
      }
    };
    float ms;
    if (LONG && layer) {
      const float2 t = corrected(sum(make_float2(ds.x + ds.y, ss.x + ss.y)), C, per_c);
      m.rest = t.x;
      ms = __fadd_rn(t.y, eps);
    } else {
      ms = fmaf(-m.rest, m.rest, fmaf(sum(ss.x + ss.y), per_c, eps));
    }
    const float inv = inverse_root(ms);
    const float2 shift = both(-__fmul_rn(m.rest, inv));
    if (b) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float2 wv[4], bv[4];
        weights(j, wv);
        col.load(bv, b + col.base, j, C);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          v[j][q] = __ffma2_rn(__ffma2_rn(v[j][q], both(inv), shift), wv[q], bv[q]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float2 wv[4];
        weights(j, wv);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          v[j][q] = __fmul2_rn(__ffma2_rn(v[j][q], both(inv), shift), wv[q]);
      }
    }
  }

  // v *= f(gate), vector j of the gate being gate(j, w)
  template <class Gate>
  __device__ __forceinline__ void gated(Gate gate, int act) {
    auto times = [&](auto f) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        uint32_t w[4];
        gate(j, w);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[j][q] = __fmul2_rn(v[j][q], f(unpack_half2(w[q])));
      }
    };
    if (act == HEXLIB_B200_GATE_NONE) times([](float2 x) { return x; });
    else if (act == HEXLIB_B200_GATE_SIGMOID) times([](float2 x) { return sigmoid2(x); });
    else if (act == HEXLIB_B200_GATE_SILU) times([](float2 x) { return __fmul2_rn(x, sigmoid2(x)); });
    else times([](float2 x) { return make_float2(tanhf(x.x), tanhf(x.y)); });
  }
};

// h of row r from the normed row v, in fp16 or in its e4m3 form.
template <int G, int V, bool WIDE, bool E4M3>
__device__ __forceinline__ void write_h(const EdgeDesc& d, const Row<G, V, WIDE>& v, int64_t r) {
  const Columns<G, WIDE>& col = v.col;
  const int C = d.C, blocks = (C + 127) / 128, padded = (blocks + 3) / 4 * 4;
  const int64_t at = r * C + col.base;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    uint32_t h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = col.pack_in(v.v[j][q], j, q, C);
    if constexpr (!E4M3) {
      col.store((__half*)d.h + at, h, j, C);
    } else if constexpr (WIDE) {
      // 16 consecutive threads hold a block; blocks past the last are zeros
      const int c = col.at(j, 0), b128 = c >> 7;
      col.zero_out(h, j, C);
      uint32_t byte;
      const uint2 codes = e4m3_encode8(h, 0xffffu << (threadIdx.x & 16), byte);
      if (b128 < blocks)
        *reinterpret_cast<uint2*>((uint8_t*)d.h_codes + r * (int64_t)blocks * 128 + c) = codes;
      if ((threadIdx.x & 15) == 0 && b128 < padded)
        ((uint8_t*)d.h_scales)[e4m3_scale_at(r, b128, d.R)] = (uint8_t)byte;
    } else {
      // the warp holds two blocks, four values of each to a lane
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = col.at(j, 4 * k), b128 = c >> 7;
        uint32_t byte;
        const uint32_t codes = e4m3_encode4(h[2 * k], h[2 * k + 1], byte);
        if (b128 < blocks) {
          uint8_t* to = (uint8_t*)d.h_codes + r * (int64_t)blocks * 128 + c;
#pragma unroll
          for (int i = 0; i < 4; ++i) to[i * 32] = (uint8_t)(codes >> (8 * i));
        }
        if ((threadIdx.x & 31) == 0 && b128 < padded)
          ((uint8_t*)d.h_scales)[e4m3_scale_at(r, b128, d.R)] = (uint8_t)byte;
      }
    }
  }
  if constexpr (E4M3) {
    // scale bytes of the last word that no thread's columns reach
    for (int b = G * V / 16 + (G == 32 ? threadIdx.x & 31 : threadIdx.x); b < padded; b += G)
      ((uint8_t*)d.h_scales)[e4m3_scale_at(r, b, d.R)] = (uint8_t)kE4m3One;
  }
}

// A row of up to G * V * 8 values in the registers of G threads (a warp, or the CTA),
// read once and written once; its gate is read with it, ahead of the sums.
constexpr int held_threads(int G) { return G == 32 ? 128 : G; }
constexpr int held_ctas(int G, int V) {       // of an SM: registers for V vectors of x, y, gate
  return (V == 1 ? 1024 : V == 2 ? 768 : V == 3 ? 640 : V == 4 ? 512 : 256) / held_threads(G);
}
template <int G, int V, bool WIDE, bool E4M3>
__global__ void __launch_bounds__(held_threads(G), held_ctas(G, V)) edge_held(const EdgeDesc d) {
  __shared__ __align__(16) float red[4][kSumSlot];
  if (E4M3) grid_dependents_may_start();   // the product that follows waits itself
  RowSum<G> sum{red};
  constexpr int ROWS = G == 32 ? held_threads(G) / 32 : 1;
  const bool layer = d.norm == HEXLIB_B200_NORM_LAYER;
  const int per_gate = d.gate ? d.R / d.gate_rows : 1;
  const int C = d.C;
  const float per_c = 1.f / C;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  const Columns<G, WIDE> col;
  for (int64_t r = blockIdx.x * (int64_t)ROWS + (G == 32 ? threadIdx.x >> 5 : 0); r < d.R;
       r += step) {
    Row<G, V, WIDE> v;
    const int64_t at = r * C + col.base;
    uint32_t x[V][4];
#pragma unroll
    for (int j = 0; j < V; ++j) col.load(x[j], (const __half*)d.x + at, j, C);
    if (d.y) {
      uint32_t y[V][4], gate[V][4];
#pragma unroll
      for (int j = 0; j < V; ++j) col.load(y[j], (const __half*)d.y + at, j, C);
      if (d.gate) {
        const __half* gp =
            (const __half*)d.gate + (int64_t)((int)r / per_gate) * C + col.base;
#pragma unroll
        for (int j = 0; j < V; ++j) col.load(gate[j], gp, j, C);
      }
      v.unpack(y);
      if (d.post_w) v.norm(d.post_w, d.post_b, C, per_c, layer, d.eps, sum);
      if (d.gate)
        v.gated([&](int j, uint32_t (&w)[4]) {
#pragma unroll
          for (int q = 0; q < 4; ++q) w[q] = gate[j][q];
        }, d.gate_act);
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          x[j][q] = col.pack_in(__ffma2_rn(both(d.x_scale), unpack_half2(x[j][q]),
                                           __fmul2_rn(both(d.y_scale), v.v[j][q])), j, q, C);
        col.store((__half*)d.x_out + at, x[j], j, C);
        col.zero_out(x[j], j, C);
      }
    }
    if (!d.pre_w) continue;
    v.unpack(x);
    v.norm(d.pre_w, d.pre_b, C, per_c, layer, d.eps, sum);
    write_h<G, V, WIDE, E4M3>(d, v, r);
  }
}

// Wide rows of whole vectors, one CTA of G threads to a row: the bulk copy engine brings
// x, y and the gate of the next row to shared memory while the norm before the next
// block and the codes of this one are computed, so no warp waits for memory with its
// registers full, and more of them fit (16384 x 4096 with a sigmoid gate for each element
// and 8-bit h: 124 us, 4.9 TB/s; 140 with the rows loaded to registers, 134 with 128
// threads of four vectors to a row).
constexpr int row_ctas(int G, int V) {
  return G == 128 ? (V == 2 ? 8 : 6) : V == 2 ? 4 : V <= 4 ? 3 : 1;
}
template <int G, int V, bool E4M3>
__global__ void __launch_bounds__(G, row_ctas(G, V)) edge_row(const EdgeDesc d) {
  extern __shared__ __align__(16) __half rows[];     // x, y, gate of a row
  __shared__ __align__(16) float red[4][kSumSlot];
  __shared__ uint64_t full;
  __shared__ int abort_flag;
  if (E4M3) grid_dependents_may_start();
  RowSum<G> sum{red};
  const Columns<G, true> col;
  const bool layer = d.norm == HEXLIB_B200_NORM_LAYER;
  const int per_gate = d.gate ? d.R / d.gate_rows : 1;
  const int C = d.C;
  const float per_c = 1.f / C;
  const uint32_t bytes = C * 2;
  auto bring = [&](int r) {                          // by thread 0
    mbar_arrive_expect_tx(&full, bytes * (1 + (d.y != nullptr) + (d.gate != nullptr)));
    bulk_load(rows, (const __half*)d.x + (int64_t)r * C, bytes, &full);
    if (d.y) bulk_load(rows + C, (const __half*)d.y + (int64_t)r * C, bytes, &full);
    if (d.gate)
      bulk_load(rows + 2 * C, (const __half*)d.gate + (int64_t)(r / per_gate) * C, bytes, &full);
  };
  if (threadIdx.x == 0) {
    mbar_init(&full, 1);
    abort_flag = 0;
    fence_mbar_init();
    bring(blockIdx.x);
  }
  __syncthreads();
  uint32_t phase = 0;
  for (int r = blockIdx.x; r < d.R; r += gridDim.x, phase ^= 1u) {
    if (!__syncthreads_and(mbar_wait(&full, phase, &abort_flag, d.err))) return;
    const int64_t at = (int64_t)r * C + col.base;
    Row<G, V, true> v;
    uint32_t x[V][4];
    if (d.y) {
#pragma unroll
      for (int j = 0; j < V; ++j) col.load(x[j], rows + C + col.base, j, C);
      v.unpack(x);
      if (d.post_w) v.norm(d.post_w, d.post_b, C, per_c, layer, d.eps, sum);
      if (d.gate)
        v.gated([&](int j, uint32_t (&w)[4]) { col.load(w, rows + 2 * C + col.base, j, C); },
                d.gate_act);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) col.load(x[j], rows + col.base, j, C);
    __syncthreads();                                 // the row has been read
    if (threadIdx.x == 0 && r + (int)gridDim.x < d.R) bring(r + gridDim.x);
    if (d.y) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          x[j][q] = col.pack_in(__ffma2_rn(both(d.x_scale), unpack_half2(x[j][q]),
                                           __fmul2_rn(both(d.y_scale), v.v[j][q])), j, q, C);
        col.store((__half*)d.x_out + at, x[j], j, C);
        col.zero_out(x[j], j, C);
      }
    }
    if (!d.pre_w) continue;
    v.unpack(x);
    v.norm(d.pre_w, d.pre_b, C, per_c, layer, d.eps, sum);
    write_h<G, V, true, E4M3>(d, v, r);
  }
}

// Rows wider than the registers hold: one CTA per row, read again for each pass, an
// element at a time (2000 x 20000: 229 us for an rms norm alone, 443 with one on both sides
// and 8-bit h; bytes once would take 49 and 43). A thread reads x' of other threads' columns
// only after the barriers of the sums.
struct Moments {
  float mean, inv, shift;                            // of (v - mean) inv + shift
};
__device__ __forceinline__ Moments moments_wide(const __half* v, int C, float per_c, bool layer,
                                                float eps, RowSum<kThreads>& sum) {
  float ss = 0.f;
  if (!layer) {
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float d = __half2float(v[c]);
      ss = fmaf(d, d, ss);
    }
    return Moments{0.f, inverse_root(fmaf(sum(ss), per_c, eps)), -0.f};
  }
  float s = 0.f, ds = 0.f;
  for (int c = threadIdx.x; c < C; c += kThreads) s += __half2float(v[c]);
  const float mean = mean_of(sum(s), C, per_c).mean;
  for (int c = threadIdx.x; c < C; c += kThreads) {
    const float d = __half2float(v[c]) - mean;
    ds += d;
    ss = fmaf(d, d, ss);
  }
  const float2 t = corrected(sum(make_float2(ds, ss)), C, per_c);
  const float inv = inverse_root(__fadd_rn(t.y, eps));
  return Moments{mean, inv, -__fmul_rn(t.x, inv)};
}
__device__ __forceinline__ float normed(float v, const Moments& m, float w, float b) {
  return fmaf(fmaf(__fsub_rn(v, m.mean), m.inv, m.shift), w, b);
}

template <bool E4M3>
__global__ void __launch_bounds__(kThreads) edge_wide(const EdgeDesc d) {
  __shared__ __align__(16) float red[4][kSumSlot];
  RowSum<kThreads> sum{red};
  const bool layer = d.norm == HEXLIB_B200_NORM_LAYER;
  const int per_gate = d.gate ? d.R / d.gate_rows : 1;
  const float per_c = 1.f / d.C;
  for (int64_t r = blockIdx.x; r < d.R; r += gridDim.x) {
    const __half* x = (const __half*)d.x + r * d.C;
    if (d.y) {
      const __half* y = (const __half*)d.y + r * d.C;
      const __half* gate = (const __half*)d.gate + (r / per_gate) * d.C;
      __half* xo = (__half*)d.x_out + r * d.C;
      Moments ms = {0.f, 1.f, -0.f};
      if (d.post_w) ms = moments_wide(y, d.C, per_c, layer, d.eps, sum);
      for (int c = threadIdx.x; c < d.C; c += kThreads) {
        float u = __half2float(y[c]);
        if (d.post_w) u = normed(u, ms, d.post_w[c], d.post_b ? d.post_b[c] : 0.f);
        if (d.gate) u = __fmul_rn(u, gate_value(__half2float(gate[c]), d.gate_act));
        xo[c] = __float2half_rn(blended(d.x_scale, __half2float(x[c]), d.y_scale, u));
      }
      x = xo;
    }
    if (!d.pre_w) continue;
    const Moments ms = moments_wide(x, d.C, per_c, layer, d.eps, sum);
    auto h_of = [&](int c) {
      return __float2half_rn(normed(__half2float(x[c]), ms, d.pre_w[c],
                                    d.pre_b ? d.pre_b[c] : 0.f));
    };
    if constexpr (!E4M3) {
      for (int c = threadIdx.x; c < d.C; c += kThreads) ((__half*)d.h)[r * d.C + c] = h_of(c);
    } else {
      const int blocks = (d.C + 127) / 128, padded = (blocks + 3) / 4 * 4;
      const int l = threadIdx.x & 15;
      for (int b0 = 0; b0 < padded; b0 += kThreads / 16) {
        const int b = b0 + (threadIdx.x >> 4), c = b * 128 + l * 8;
        uint32_t h[4], byte;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const __half lo = c + 2 * q < d.C ? h_of(c + 2 * q) : __half(0.f);
          const __half hi = c + 2 * q + 1 < d.C ? h_of(c + 2 * q + 1) : __half(0.f);
          h[q] = __half_as_ushort(lo) | ((uint32_t)__half_as_ushort(hi) << 16);
        }
        const uint2 codes = e4m3_encode8(h, 0xffffu << (threadIdx.x & 16), byte);
        if (b < blocks)
          *reinterpret_cast<uint2*>((uint8_t*)d.h_codes + r * (int64_t)blocks * 128 + c) = codes;
        if (l == 0 && b < padded)
          ((uint8_t*)d.h_scales)[e4m3_scale_at(r, b, d.R)] = (uint8_t)byte;
      }
    }
  }
}

// Every (threads per row, vectors per thread) a width can take: a warp to a row while its
// registers hold it (65536 x 768: 69 us, 5.8 TB/s, 740 CTAs of 96 registers a thread), then
// a CTA. (A warp to rows of 1344 with a layer norm either side measured 77 us against 84,
// but 20000 x 2048 120 against 88 and eight rows of 1344 6.2 against 4.0.)
template <class F>
int with_layout(int C, F&& f) {
  const int v = (C + 7) / 8;
#define HB_EDGE_LAYOUT(G, V) \
  if (v <= G * V) return f(std::integral_constant<int, G>{}, std::integral_constant<int, V>{});
  HB_EDGE_LAYOUT(32, 1)
  HB_EDGE_LAYOUT(32, 2)
  HB_EDGE_LAYOUT(32, 3)
  HB_EDGE_LAYOUT(32, 4)
  HB_EDGE_LAYOUT(128, 2)
  HB_EDGE_LAYOUT(128, 3)
  HB_EDGE_LAYOUT(256, 2)
  HB_EDGE_LAYOUT(256, 3)
  HB_EDGE_LAYOUT(256, 4)
  HB_EDGE_LAYOUT(256, 8)
#undef HB_EDGE_LAYOUT
  return f(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
}

// CTAs of a form that are resident on the device at once, found when it is loaded (a
// grid of more would leave a partial last wave: 65536 x 768 on 1184 CTAs, 444 of them
// resident, took 77 us against 72).
template <int G, int V, bool WIDE, bool E4M3>
std::atomic<int> g_resident{0};

constexpr bool by_row(int G, bool wide) { return wide && G > 32; }
constexpr int row_bytes(int C) { return 3 * 2 * C; }

template <bool WIDE, bool E4M3>
int launch_form(const EdgeDesc& d, cudaStream_t s) {
  return with_layout(d.C, [&](auto G, auto V) {
    if constexpr (G.value == 0) {
      edge_wide<E4M3><<<d.R < 148 * 8 ? d.R : 148 * 8, kThreads, 0, s>>>(d);
    } else {
      const int64_t rows = G.value == 32 ? held_threads(32) / 32 : 1;
      const int64_t ctas = (d.R + rows - 1) / rows;
      const int64_t most = g_resident<G.value, V.value, WIDE, E4M3>.load(std::memory_order_relaxed);
      const unsigned grid = (unsigned)(ctas < most ? ctas : most);
      if constexpr (by_row(G.value, WIDE))
        edge_row<G.value, V.value, E4M3><<<grid, G.value, row_bytes(d.C), s>>>(d);
      else
        edge_held<G.value, V.value, WIDE, E4M3><<<grid, held_threads(G.value), 0, s>>>(d);
    }
    if (cudaPeekAtLastError() != cudaSuccess) {
      cudaGetLastError();
      return HEXLIB_B200_ERR_CUDA;
    }
    return HEXLIB_B200_OK;
  });
}

template <bool WIDE, bool E4M3>
bool load_form(int sms) {
  cudaFuncAttributes a;
  bool ok = cudaFuncGetAttributes(&a, (const void*)edge_wide<E4M3>) == cudaSuccess;
  for (int C : {256, 512, 768, 1024, 2048, 3000, 4096, 6144, 8192, 16384})
    with_layout(C, [&](auto G, auto V) {
      if constexpr (G.value != 0) {
        int n = 0;
        if constexpr (by_row(G.value, WIDE)) {
          // for the layout's widest row: narrower ones leave no more than a CTA's room unused
          const int most = row_bytes(G.value * V.value * 8);
          auto* k = edge_row<G.value, V.value, E4M3>;
          ok = ok && cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most) ==
                         cudaSuccess &&
               cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, G.value, most) == cudaSuccess;
        } else {
          ok = ok && cudaOccupancyMaxActiveBlocksPerMultiprocessor(
                         &n, (const void*)edge_held<G.value, V.value, WIDE, E4M3>,
                         held_threads(G.value), 0) == cudaSuccess;
        }
        ok = ok && n > 0;
        g_resident<G.value, V.value, WIDE, E4M3>.store(n * sms, std::memory_order_relaxed);
      }
      return 0;
    });
  return ok;
}

}  // namespace

// Load the kernels now, so that none is loaded lazily inside a graph capture.
int edge_kernels_init() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      !load_form<true, false>(sms) || !load_form<true, true>(sms) || !load_form<false, false>(sms) ||
      !load_form<false, true>(sms)) {
    cudaGetLastError();
    return HEXLIB_B200_ERR_CUDA;
  }
  return HEXLIB_B200_OK;
}

int launch_edge(const EdgeDesc& d, cudaStream_t s) {
  uintptr_t bits = static_cast<uintptr_t>(2) * d.C;
  for (const void* p : {d.x, d.y, d.gate, (const void*)d.x_out, (const void*)d.h,
                        (const void*)d.pre_w, (const void*)d.pre_b, (const void*)d.post_w,
                        (const void*)d.post_b})
    bits |= reinterpret_cast<uintptr_t>(p);
  const bool wide = bits % 16 == 0;
  if (d.h_codes) return wide ? launch_form<true, true>(d, s) : launch_form<false, true>(d, s);
  return wide ? launch_form<true, false>(d, s) : launch_form<false, false>(d, s);
}

}  // namespace hb

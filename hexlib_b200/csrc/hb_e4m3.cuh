// hb_e4m3.cuh -- the e4m3 form of a row (8-bit floating point codes with a
// power-of-two scale for each block of 128), shared by the kernels that write it.
//
// A block whose largest finite |x| is m 2^k (1 <= m < 2) gets the scale 2^e with
// the smallest e for which m 2^k <= 448 * 2^e = 1.75 * 2^(e + 8): e = k - 8 for
// m <= 1.75 and k - 7 above, read off the bits of the float. x * 2^-e is then exact
// in fp32 and the conversion to e4m3 (nearest even) is the one rounding, so every
// kernel and the definition agree bit for bit.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace hb {

constexpr uint32_t kE4m3One = 127;   // the scale byte of 1.0
constexpr uint32_t kE4m3Nan = 0x7f;

// The scale byte (e + 127) of a block from its largest finite magnitude.
__device__ __forceinline__ uint32_t e4m3_scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return u == 0 ? kE4m3One : (u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
}
// 2^-e of a scale byte this form holds (e in [-32, 8], so 254 - byte is normal).
__device__ __forceinline__ float e4m3_inverse(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}
// 2^e of any scale byte (0 stands for 2^-127, 255 for NaN).
__device__ __forceinline__ float e4m3_scale(uint32_t byte) {
  return byte == 0 ? __uint_as_float(1u << 22)
                   : byte == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

// Two codes of finite, scaled values (|v| <= 448): lo in the low byte.
__device__ __forceinline__ uint32_t e4m3_pack2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// One code, with NaN for what is not finite (the conversion alone would make
// infinities 448).
__device__ __forceinline__ uint32_t e4m3_code(float x, float inv) {
  return isfinite(x) ? (e4m3_pack2(x * inv, 0.f) & 0xffu) : kE4m3Nan;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
  return __half2float(
      __half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3)));
}

// The codes of a block of 128 fp16 values held by 16 consecutive lanes (half of a
// warp, the lanes of `half_mask`), 8 to a lane as four words of two, and the block's
// scale byte. The largest magnitude is found on the bits (halves of the same sign
// order as integers), two to an instruction.
__device__ __forceinline__ uint2 e4m3_encode8(const uint32_t (&w)[4], uint32_t half_mask,
                                              uint32_t& byte) {
  uint32_t m2 = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int j = 1; j < 4; ++j) m2 = __vmaxu2(m2, w[j] & 0x7fff7fffu);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m2 = __vmaxu2(m2, __shfl_xor_sync(half_mask, m2, o));
  uint32_t m = max(m2 & 0xffffu, m2 >> 16);
  const bool finite = m < 0x7c00u;
  if (!finite) {                       // the same for all 16 lanes
    m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < 32; h += 16) {
        const uint32_t a = (w[j] >> h) & 0x7fffu;
        if (a < 0x7c00u) m = max(m, a);
      }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half_mask, m, o));
  }
  byte = e4m3_scale_byte(__half2float(__ushort_as_half((unsigned short)m)));
  const float inv = e4m3_inverse(byte);
  uint32_t c[4];
  if (finite && byte >= 112u) {
    // 2^-e fits fp16, and the product in fp16 loses only bits of values under 2^-14,
    // which e4m3 rounds to zero all the same (its smallest step is 2^-9)
    const __half2 inv2 = __half2half2(__float2half_rn(inv));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c[j] = __nv_cvt_halfraw2_to_fp8x2(
          __half2_raw(__hmul2(*reinterpret_cast<const __half2*>(&w[j]), inv2)), __NV_SATFINITE,
          __NV_E4M3);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      c[j] = finite ? e4m3_pack2(__fmul_rn(f.x, inv), __fmul_rn(f.y, inv))
                    : e4m3_code(f.x, inv) | (e4m3_code(f.y, inv) << 8);
    }
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// The same for a block held by a whole warp, four values to a lane as two words: the
// lane's four codes, low byte first.
__device__ __forceinline__ uint32_t e4m3_encode4(uint32_t w0, uint32_t w1, uint32_t& byte) {
  const uint32_t w[2] = {w0, w1};
  float f[4], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (isfinite(f[j])) amax = fmaxf(amax, fabsf(f[j]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  byte = e4m3_scale_byte(amax);
  const float inv = e4m3_inverse(byte);
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) c |= e4m3_code(f[j], inv) << (8 * j);
  return c;
}

// Eight fp16 values from p, as four words of two, in loads of VEC values (VEC = 8 for
// 16-byte aligned rows down to 1 for any); values from `left` on are zeros. With
// VEC > 1, `left` is a multiple of VEC.
template <int VEC>
__device__ __forceinline__ void load8(uint32_t (&w)[4], const __half* p, int left) {
  if constexpr (VEC == 8) {
    const uint4 u = left > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (VEC == 4) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint2 u = 2 * j < left ? *reinterpret_cast<const uint2*>(p + 2 * j) : make_uint2(0, 0);
      w[j] = u.x; w[j + 1] = u.y;
    }
  } else if constexpr (VEC == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = 2 * j < left ? *reinterpret_cast<const uint32_t*>(p + 2 * j) : 0u;
  } else {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (2 * j < left ? (uint32_t)q[2 * j] : 0u) |
             (2 * j + 1 < left ? (uint32_t)q[2 * j + 1] << 16 : 0u);
  }
}
// The widest VEC of rows of C values starting at p.
inline int row_vec(int64_t C, const void* p) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(2 * C);
  return a % 16 == 0 ? 8 : a % 8 == 0 ? 4 : a % 4 == 0 ? 2 : 1;
}

// Byte offset of the scale of block b of row r of R.
__device__ __forceinline__ int64_t e4m3_scale_at(int64_t r, int b, int64_t R) {
  return ((b >> 2) * R + r) * 4 + (b & 3);
}

}  // namespace hb

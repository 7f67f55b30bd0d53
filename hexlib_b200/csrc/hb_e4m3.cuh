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

// Byte offset of the scale of block b of row r of R.
__device__ __forceinline__ int64_t e4m3_scale_at(int64_t r, int b, int64_t R) {
  return ((b >> 2) * R + r) * 4 + (b & 3);
}

}  // namespace hb

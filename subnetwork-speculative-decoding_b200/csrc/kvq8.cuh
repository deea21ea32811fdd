// The 8-bit key/value cache's row format, shared by the kernels that write,
// read, move and attend it.
//
// A row (one slot of one KV head) is head_dim e4m3 codes and one scale byte:
// the biased exponent e + 127 of a power of two. e is the smallest exponent
// with amax <= 448 * 2^e over the row's finite elements, limited to -40 .. 119
// (below, the codes reach their subnormals; above, 448 * 2^e leaves fp32).
// Scales are powers of two so that x * 2^-e and code * 2^e are exact: the
// only rounding of a row is the one to e4m3, and a row read back as bf16 or
// fp32 is exactly what attention over the cache computes with.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace ssd {

constexpr int kQ8MinScale = 127 - 40;   // smallest scale byte written
constexpr int kQ8MaxScale = 127 + 119;  // largest
// Slots of a cache: attention rounds its slot range up to whole units of key
// blocks (2^19 slots at this length), which have to stay below 2^31 too.
constexpr int64_t kQ8MaxSlots = (1ll << 31) - (1 << 21);

// Scale byte of a row with the given amax (finite, >= 0). 448 = 1.75 * 2^8:
// with amax = 1.m * 2^x, e = x - 8 up to m = 0.75 and x - 7 above; adding
// 0x1fffff carries into the exponent exactly for mantissas above 0x600000.
__device__ __forceinline__ int q8_scale_byte(float amax) {
  const int b = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8;
  return min(max(b, kQ8MinScale), kQ8MaxScale);
}
// 2^e and 2^-e of a scale byte e + 127 (bytes 0 of slots never written: 0).
__device__ __forceinline__ float q8_scale(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }
__device__ __forceinline__ float q8_inv_scale(int byte) {
  return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
}
// Two values to two e4m3 codes (low byte: lo), nearest even, saturating at
// +-448; NaN stays NaN.
__device__ __forceinline__ uint32_t q8_pack2(float lo, float hi) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Two codes (the low 16 bits of v) to their fp32 values, exact.
__device__ __forceinline__ float2 q8_unpack2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

}  // namespace ssd

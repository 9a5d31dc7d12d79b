// Device helpers of the 8-bit cache: codes to and from floats, power-of-two scales.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "paged8.h"

namespace hcp {
namespace kv8 {

// The scale of a block is the smallest power of two s in [2^-40, 2^40] with amax <= QMAX * s,
// QMAX = 448 (e4m3) or 127 (int8). e4m3 is a floating format, so a power of two loses none of its
// precision against amax / QMAX; int8 loses up to one bit of it, and gains that rescaling an open
// block shifts its codes, and that code * scale has at most 8 significant bits: exact in bf16.
// With amax = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9 and 127 = 0.9921875 * 2^7 decide on m alone.
// The limits keep every product with a scale or its reciprocal inside float32.
constexpr int kMinExp = -40, kMaxExp = 40;

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

template <bool INT8>
__device__ __forceinline__ float block_scale(float amax) {
  const int bits = __float_as_int(amax);
  const int mant = bits & 0x7fffff;                 // m = 0.5 + mant / 2^24
  int e = ((bits >> 23) & 0xff) - 126;              // amax = m 2^e (subnormals: below kMinExp anyway)
  const int limit = INT8 ? 0x7e0000 : 0x600000;     // 127 / 128 and 0.875
  e = e - (INT8 ? 7 : 9) + (mant > limit ? 1 : 0);
  return pow2(min(max(e, kMinExp), kMaxExp));
}

// Two codes in the low and high byte of the result. e4m3: round to nearest even, saturated at
// 448, NaN stays NaN. int8: round to nearest even, saturated at 127, NaN becomes 0.
template <bool INT8>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  if (INT8) {
    // cvt.rni saturates at the integer's range and gives 0 for NaN
    const int x = min(max(__float2int_rn(a), -127), 127), y = min(max(__float2int_rn(b), -127), 127);
    return uint32_t(x & 0xff) | (uint32_t(y & 0xff) << 8);
  }
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

template <bool INT8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  return encode2<INT8>(a, b) | (encode2<INT8>(c, d) << 16);
}

// Four codes as two f16 pairs (bytes 0, 1 and bytes 2, 3), exact. int8: the byte with its sign
// bit flipped is x + 128; in the low mantissa bits of the half 1024 it reads 1024 + 128 + x.
template <bool INT8>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    const __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

__device__ __forceinline__ float2 half2_floats(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// 8 consecutive elements of a row as they are stored, and in float32.
template <int DT>
struct Raw8 {
  uint4 v[DT == kF32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* base, long i) {
  Raw8<DT> r;
  const char* p = reinterpret_cast<const char*>(base) + i * (DT == kF32 ? 4 : 2);
  r.v[0] = dev::ld_nc_v4(p);
  if (DT == kF32) r.v[DT == kF32 ? 1 : 0] = dev::ld_nc_v4(p + 16);
  return r;
}

template <int DT>
__device__ __forceinline__ void floats8(const Raw8<DT>& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < (DT == kF32 ? 2 : 1); ++k) {
    const uint32_t w[4] = {r.v[k].x, r.v[k].y, r.v[k].z, r.v[k].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == kF32) {
        f[(4 * k + j) % 8] = __uint_as_float(w[j]);
      } else if (DT == kBF16) {
        f[2 * j] = dev::bf16_lo(w[j]);
        f[2 * j + 1] = dev::bf16_hi(w[j]);
      } else {
        const float2 x = half2_floats(w[j]);
        f[2 * j] = x.x;
        f[2 * j + 1] = x.y;
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void load8(const void* base, long i, float (&f)[8]) {
  floats8<DT>(load_raw8<DT>(base, i), f);
}

__device__ __forceinline__ uint32_t pack16(int dtype, float a, float b) {
  if (dtype == kBF16) return dev::pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace kv8
}  // namespace hcp

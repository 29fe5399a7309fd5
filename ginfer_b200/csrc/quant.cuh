// Arithmetic of the 8-bit cache shared by the kernels that write, read and attend over it
// (the formulas: quant_cache.cu).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace gf {

// ---- eight channels of a row, as they lie in memory until they are used
// vec: the address is a multiple of 16 bytes.  Always past L1: a kernel shortly before this one wrote them.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, int vec) {
    if (vec) {
      a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
    } else {
      a = make_float4(__ldcg(p), __ldcg(p + 1), __ldcg(p + 2), __ldcg(p + 3));
      b = make_float4(__ldcg(p + 4), __ldcg(p + 5), __ldcg(p + 6), __ldcg(p + 7));
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
};
template <> struct Raw8<bf16> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p, int vec) {
    if (vec) {
      a = __ldcg(reinterpret_cast<const uint4*>(p));
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
      a.x = (uint32_t)__ldcg(h) | (uint32_t)__ldcg(h + 1) << 16, a.y = (uint32_t)__ldcg(h + 2) | (uint32_t)__ldcg(h + 3) << 16;
      a.z = (uint32_t)__ldcg(h + 4) | (uint32_t)__ldcg(h + 5) << 16, a.w = (uint32_t)__ldcg(h + 6) | (uint32_t)__ldcg(h + 7) << 16;
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
};
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
  uint4 a;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
  *reinterpret_cast<uint4*>(p) = a;
}

// ---- rotation of a pair (a, b) by an angle with cosine c and sine s, every operation rounded
__device__ __forceinline__ float turned_first(float a, float b, float c, float s) {
  return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}
__device__ __forceinline__ float turned_second(float a, float b, float c, float s) {
  return __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
}
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float u = turned_first(a, b, c, s), v = turned_second(a, b, c, s);
  a = u, b = v;
}

// ---- quantisation
// The largest magnitude as its bits: a NaN's are above an infinity's, and that above every number's.
__device__ __forceinline__ uint32_t max_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  return m;
}
template <int LANES> __device__ __forceinline__ uint32_t group_max_bits(uint32_t m, unsigned mask = 0xffffffffu) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(mask, m, o));
  return m;
}
struct RowScale {
  float scale, inverse;        // inverse 0: no finite codes
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits, int fp8) {
  if (top_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  const float s = fmaxf(__fmul_rn(__uint_as_float(top_bits), fp8 ? 1.0f / 448.0f : 1.0f / 127.0f),
                        1.17549435e-38f);
  return {s, __fdiv_rn(1.0f, s)};
}
// x / scale is at most Q (1 + 2^-22), which rounds to Q: nothing to saturate.  Integers: 1.5 * 2^23 added leaves the
// integer, rounded to even, in the low bits.
__device__ __forceinline__ uint32_t quantise4(const float* v, const RowScale& rs, int fp8) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(v[e], rs.inverse);
  uint32_t w;
  if (fp8) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
    w = (uint32_t)lo | (uint32_t)hi << 16;
  } else {
    uint32_t n[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) n[e] = __float_as_uint(__fadd_rn(y[e], 12582912.f));
    w = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
  }
  return rs.inverse == 0.f ? 0u : w;
}
__device__ __forceinline__ uint32_t code_of(float x, const RowScale& rs, int fp8) {
  const float v[4] = {x, 0.f, 0.f, 0.f};
  return quantise4(v, rs, fp8) & 0xffu;
}
__device__ __forceinline__ uint2 quantise8(const float (&v)[8], const RowScale& rs, int fp8) {
  return make_uint2(quantise4(v, rs, fp8), quantise4(v + 4, rs, fp8));
}

// ---- codes back to numbers
// Two e4m3 codes (the low 16 bits) as two halves, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
// What four codes stand for in units of their row's scale.
__device__ __forceinline__ void values4(uint32_t w, int fp8, float* v) {
  if (fp8) {
    const uint32_t lo = e4m3x2_to_half2(w), hi = e4m3x2_to_half2(w >> 16);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)(int8_t)(w >> (8 * e));
  }
}

}  // namespace gf

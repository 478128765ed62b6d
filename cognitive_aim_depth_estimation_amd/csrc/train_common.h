// Shared device helpers of the training kernels (train_rows.hip, train_linear.hip): run-time element types, the 8-bit
// activation format, and the activations with their derivatives.
#pragma once
#include "common.h"

namespace train {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4v __attribute__((ext_vector_type(4)));

enum { DT_BF16 = 0, DT_FP16 = 1, DT_FP32 = 2 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2 };
constexpr int GROUP = 32;                       // columns of a row that share one 8-bit step

__host__ __device__ inline long long groups_of(int D) { return (D + GROUP - 1) / GROUP; }
__host__ __device__ inline int dt_size(int dt) { return dt == DT_FP32 ? 4 : 2; }

// ---- eight consecutive elements of a run-time type -----------------------------------------------------------------
// The element type is uniform over a launch: a scalar branch picks the load, and the bits are converted later, so that
// several loads are in flight before the first conversion waits.
struct Raw8 { u32x4v a, b; };

__device__ __forceinline__ Raw8 load_raw8(const void* p, int dt, size_t off) {       // 16-byte aligned
  Raw8 r;
  if (dt == DT_FP32) {
    const u32x4v* q = reinterpret_cast<const u32x4v*>(reinterpret_cast<const float*>(p) + off);
    r.a = q[0]; r.b = q[1];
  } else {
    r.a = *reinterpret_cast<const u32x4v*>(reinterpret_cast<const unsigned short*>(p) + off);
    r.b = u32x4v{0, 0, 0, 0};
  }
  return r;
}
__device__ __forceinline__ float bf16_lo(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(unsigned w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float half_bits(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ void cvt_raw8(const Raw8& r, int dt, float (&v)[8]) {
  if (dt == DT_FP32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(r.a[i]); v[4 + i] = __uint_as_float(r.b[i]); }
  } else if (dt == DT_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(r.a[i]); v[2 * i + 1] = bf16_hi(r.a[i]); }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = half_bits((unsigned short)r.a[i]); v[2 * i + 1] = half_bits((unsigned short)(r.a[i] >> 16)); }
  }
}
__device__ __forceinline__ unsigned bits16(float y, int dt) {
  if (dt == DT_BF16) return __builtin_bit_cast(unsigned short, (__bf16)y);
  return __builtin_bit_cast(unsigned short, (_Float16)y);
}
__device__ __forceinline__ void store_vec8(void* p, int dt, size_t off, const float (&y)[8]) {   // 16-byte aligned
  if (dt == DT_FP32) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + off);
    q[0] = make_float4(y[0], y[1], y[2], y[3]); q[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
    u32x4v w;
    if (dt == DT_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bits16(y[2 * i], DT_BF16) | (bits16(y[2 * i + 1], DT_BF16) << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bits16(y[2 * i], DT_FP16) | (bits16(y[2 * i + 1], DT_FP16) << 16);
    }
    *reinterpret_cast<u32x4v*>(reinterpret_cast<unsigned short*>(p) + off) = w;
  }
}
__device__ __forceinline__ float load_one(const void* p, int dt, size_t off) {
  if (dt == DT_FP32) return reinterpret_cast<const float*>(p)[off];
  const unsigned short h = reinterpret_cast<const unsigned short*>(p)[off];
  return dt == DT_BF16 ? __uint_as_float((unsigned)h << 16) : half_bits(h);
}
__device__ __forceinline__ void store_one(void* p, int dt, size_t off, float y) {
  if (dt == DT_FP32) reinterpret_cast<float*>(p)[off] = y;
  else reinterpret_cast<unsigned short*>(p)[off] = (unsigned short)bits16(y, dt);
}

// ---- 8-bit activations -----------------------------------------------------------------------------------------------
// A group's step is 2^e, e the smallest integer >= -126 for which its largest magnitude rounds to at most 127 steps;
// byte = e + 127.  With the magnitude's bits as an integer, adding 2^16 carries a mantissa of 127.5 / 64 or more into
// the exponent, so e = exponent - 6 after that carry.  A power of two makes code * step exact in bf16 (and fp32), and
// x / step exact, so the code is one rounding of x and the decoded value none.  Byte 255 marks a group that held an
// infinity or a NaN; all of it decodes to NaN, so that an overflow is not turned into a finite gradient.  At the largest
// step, 2^122, codes end at 63: 64 steps would be 2^128, past the largest finite value.
__device__ __forceinline__ unsigned group_byte(unsigned max_bits) {
  if (max_bits >= 0x7f800000u) return 255u;
  const int b = (int)((max_bits + 0x10000u) >> 23) - 6;
  return (unsigned)(b < 1 ? 1 : b);
}
__device__ __forceinline__ float group_inverse(unsigned byte) {          // 1 / step; 0 for a group without a step
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float group_step(unsigned byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ int code_of(float x, float inverse, float most) {
  const float q = __builtin_rintf(x * inverse);
  return (int)(inverse == 0.f ? 0.f : __builtin_amdgcn_fmed3f(q, -most, most));
}
__device__ __forceinline__ float most_code(unsigned byte) { return byte == 249u ? 63.f : 127.f; }
__device__ __forceinline__ unsigned mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ u32x2 pack_codes(const float (&v)[8], unsigned byte) {
  const float inverse = group_inverse(byte), most = most_code(byte);
  u32x2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    r[h] = (code_of(v[4 * h], inverse, most) & 255) | ((code_of(v[4 * h + 1], inverse, most) & 255) << 8) |
           ((code_of(v[4 * h + 2], inverse, most) & 255) << 16) | ((unsigned)code_of(v[4 * h + 3], inverse, most) << 24);
  return r;
}
__device__ __forceinline__ void decode8(u32x2 c, float step, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)(signed char)(c[i >> 2] >> (8 * (i & 3))) * step;
}
// 127 steps of a group whose magnitudes reach the top of fp16 can exceed its largest finite value by less than one
// step: such a value is held at the largest finite one (the group's own values were finite)
__device__ __forceinline__ float hold_fp16(float y) { return y > 65504.f ? 65504.f : y < -65504.f ? -65504.f : y; }

// ---- activations -----------------------------------------------------------------------------------------------------
// Phi(-a), the normal distribution's lower tail, for a in [0, 5.5]: log2 Phi(-a) is close to a parabola, and a
// degree-8 polynomial (weighted minimax fit in Chebyshev form, weight Phi(-a) max(1, a)) followed by one exp2 is within
// 6e-8 of Phi and of a Phi in fp32.  Past 5.5 both are under 1.1e-7 and the value at 5.5 is kept.
__device__ __forceinline__ float phi_tail(float a) {
  float p = -2.275866336e-06f;
  p = __builtin_fmaf(p, a, 3.296794603e-05f);
  p = __builtin_fmaf(p, a, -1.572784386e-04f);
  p = __builtin_fmaf(p, a, -2.024798159e-04f);
  p = __builtin_fmaf(p, a, 7.142783143e-03f);
  p = __builtin_fmaf(p, a, -5.254643783e-02f);
  p = __builtin_fmaf(p, a, -4.591930509e-01f);
  p = __builtin_fmaf(p, a, -1.151106954e+00f);
  p = __builtin_fmaf(p, a, -9.999999404e-01f);
  return __builtin_amdgcn_exp2f(p);
}
__device__ __forceinline__ float relu_of(float x) { return x < 0.f ? 0.f : x; }      // a NaN stays one
// x Phi(x) = max(x, 0) - |x| Phi(-|x|)
__device__ __forceinline__ float gelu_of(float x) {
  const float a = fminf(fabsf(x), 5.5f);
  return relu_of(x) - a * phi_tail(a);
}
// value and derivative: Phi(x) + x phi(x), phi(x) = exp(-x^2 / 2) / sqrt(2 pi)
__device__ __forceinline__ void gelu_both(float x, float& value, float& slope) {
  const float ax = fabsf(x), a = fminf(ax, 5.5f), q = phi_tail(a);
  value = relu_of(x) - a * q;
  const float b = fminf(ax, 16.f);                         // phi(16) is 0 in fp32; keeps inf * 0 out
  const float bell = 0.3989422804f * __builtin_amdgcn_exp2f(-0.7213475204f * b * b);
  const float d = (x < 0.f ? q : 1.f - q) + __builtin_copysignf(b, x) * bell;
  slope = x != x ? x : d;
}
__device__ __forceinline__ float relu_slope(float x) { return x > 0.f ? 1.f : x != x ? x : 0.f; }

}  // namespace train

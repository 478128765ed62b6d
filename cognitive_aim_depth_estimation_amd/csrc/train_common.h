// Shared device helpers of the training kernels (train_rows.hip, train_linear.hip): run-time element types, the 8-bit
// activation format, and the activations with their derivatives.
#pragma once
#include "common.h"

namespace train {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4v __attribute__((ext_vector_type(4)));

// A launch counts its work-items along x in 32 bits; kernels whose grid grows with the rows take no more in one launch.
constexpr long long MAX_ITEMS = 0xffffffffLL;

enum { DT_BF16 = 0, DT_FP16 = 1, DT_FP32 = 2 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2 };
constexpr int GROUP = 32;                       // columns of a row that share one 8-bit step

__host__ __device__ inline long long groups_of(int D) { return (D + GROUP - 1) / GROUP; }
__host__ __device__ inline int dt_size(int dt) { return dt == DT_FP32 ? 4 : 2; }

// ---- eight consecutive elements of a run-time type -----------------------------------------------------------------
// The element type is uniform over a launch: a scalar branch picks the load, and the bits are converted later, so that
// several loads are in flight before the first conversion waits.
struct Raw8 { u32x4v a, b; };
// 16 bytes of any alignment that the element type has (gfx950 takes them)
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ Raw8 load_raw8(const void* p, int dt, size_t off) {
  Raw8 r;
  if (dt == DT_FP32) {
    const u32x4_any* q = reinterpret_cast<const u32x4_any*>(reinterpret_cast<const float*>(p) + off);
    r.a = q[0]; r.b = q[1];
  } else {
    r.a = *reinterpret_cast<const u32x4_any*>(reinterpret_cast<const unsigned short*>(p) + off);
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
typedef float f32x8 __attribute__((ext_vector_type(8)));
// number of 16-bit parts that hold an fp32 value: three of bf16 (24 bits), two of fp16 (22 bits, down to its least number)
constexpr int parts_of(int dt) { return dt == DT_BF16 ? 3 : 2; }
template <int V> __device__ __forceinline__ void pack_half(const float (&y)[V], int dt, void* to) {       // V 16-bit values in registers
  typedef float fv __attribute__((ext_vector_type(V)));
  typedef __bf16 bv __attribute__((ext_vector_type(V)));
  typedef _Float16 hv __attribute__((ext_vector_type(V)));
  fv v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = y[i];
  if (dt == DT_BF16) { const bv h = __builtin_convertvector(v, bv); __builtin_memcpy(to, &h, 2 * V); }
  else { const hv h = __builtin_convertvector(v, hv); __builtin_memcpy(to, &h, 2 * V); }
}
// eight values rounded to 16 bits, and what the rounding left of them (nothing of one that is not finite)
__device__ __forceinline__ void take_part(float (&v)[8], int dt, void* to) {
  pack_half<8>(v, dt, to);
  u32x4v w;
  __builtin_memcpy(&w, to, 16);
  float h[8];
  cvt_raw8(Raw8{w, w}, dt, h);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float left = v[j] - h[j];
    v[j] = fabsf(left) < __builtin_inff() ? left : 0.f;
  }
}
template <bool STREAM = false>
__device__ __forceinline__ void store_vec8(void* p, int dt, size_t off, const float (&y)[8]) {
  if (dt == DT_FP32) {
    f32x4_any* q = reinterpret_cast<f32x4_any*>(reinterpret_cast<float*>(p) + off);
    const f32x4_any a = {y[0], y[1], y[2], y[3]}, b = {y[4], y[5], y[6], y[7]};
    if constexpr (STREAM) { __builtin_nontemporal_store(a, q); __builtin_nontemporal_store(b, q + 1); }
    else { q[0] = a; q[1] = b; }
  } else {
    const f32x8 v = {y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
    u32x4v w;
    if (dt == DT_BF16) w = __builtin_bit_cast(u32x4v, __builtin_convertvector(v, bf16x8));
    else w = __builtin_bit_cast(u32x4v, __builtin_convertvector(v, f16x8));
    u32x4_any* q = reinterpret_cast<u32x4_any*>(reinterpret_cast<unsigned short*>(p) + off);
    if constexpr (STREAM) __builtin_nontemporal_store((u32x4_any)w, q);
    else *q = w;
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

// An operand times a vector of scales, rounded to fp16: a LayerScale of 1e-5 would push it into fp16's subnormals (0.02 times
// that keeps two bits).  So the scales are multiplied by a power of two that brings the largest into [0.5, 1), and the
// sums by its reciprocal, both exact.  `top`: the largest magnitude's bits; infinities, NaN and all zeros: no change.
__device__ __forceinline__ void scale_units(unsigned top, float& up, float& down) {
  const unsigned e = top >> 23;
  up = down = 1.f;
  if (top == 0 || e == 255) return;
  const unsigned c = e < 252 ? e : 252;
  up = __uint_as_float((253 - c) << 23);
  down = __uint_as_float((c + 1) << 23);
}
__device__ __forceinline__ unsigned wave_top(const float* s, int n, int from, int by) {      // largest magnitude's bits
  unsigned top = 0;
#pragma unroll 4
  for (int i = from; i < n; i += by) {
    const unsigned b = __float_as_uint(s[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const unsigned o = (unsigned)__shfl_xor((int)top, d);
    top = o > top ? o : top;
  }
  return top;
}
// Sum over the 64 lanes, result in every lane, without the LDS permute path: rotations inside rows of 16 lanes (DPP), then
// the two row-swap instructions of gfx950.
__device__ __forceinline__ float wave_sum_dpp(float v) {
#define TRAIN_ROR(ctrl_) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl_, 0xf, 0xf, false))
  v += TRAIN_ROR(0x128);   // row_ror:8
  v += TRAIN_ROR(0x124);   // row_ror:4
  v += TRAIN_ROR(0x122);   // row_ror:2
  v += TRAIN_ROR(0x121);   // row_ror:1
#undef TRAIN_ROR
  unsigned u = __float_as_uint(v);
  auto s16 = __builtin_amdgcn_permlane16_swap(u, u, false, false);      // rows (0,1) and (2,3) meet
  v = __uint_as_float(s16[0]) + __uint_as_float(s16[1]);
  u = __float_as_uint(v);
  auto s32 = __builtin_amdgcn_permlane32_swap(u, u, false, false);      // the two halves meet
  return __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
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
__device__ __forceinline__ unsigned mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
// Largest magnitude of V values as bits, NaN above all: `maximum` passes a NaN on (v_maximum3_f32, two values an
// instruction).
template <int V> __device__ __forceinline__ unsigned top_bits(const float (&v)[V]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < V; ++j) m = __builtin_elementwise_maximum(m, fabsf(v[j]));
  return mag_bits(m);
}
// x / step to the nearest integer in the low bits of a float: adding 1.5 * 2^23 leaves no fraction bits, and rounds ties
// to even as any fp32 addition
__device__ __forceinline__ unsigned code_bits(float x, float inverse) {
  return __float_as_uint(__builtin_fmaf(x, inverse, 12582912.f));
}
// the two kinds of group that code_bits does not serve: no step (all codes 0), and the largest step (codes end at 63)
__device__ __forceinline__ bool group_is_rare(unsigned byte) { return byte >= 249u; }
__device__ __forceinline__ int code_of_rare(float x, unsigned byte) {
  if (byte == 255u) return 0;
  return (int)__builtin_amdgcn_fmed3f(__builtin_rintf(x * group_inverse(byte)), -63.f, 63.f);
}
__device__ __forceinline__ unsigned pack4(const float* v, unsigned byte) {
  if (group_is_rare(byte))
    return (code_of_rare(v[0], byte) & 255) | ((code_of_rare(v[1], byte) & 255) << 8) | ((code_of_rare(v[2], byte) & 255) << 16) |
           ((unsigned)code_of_rare(v[3], byte) << 24);
  const float inverse = group_inverse(byte);
  const unsigned lo = __builtin_amdgcn_perm(code_bits(v[1], inverse), code_bits(v[0], inverse), 0x0c0c0400u);
  const unsigned hi = __builtin_amdgcn_perm(code_bits(v[3], inverse), code_bits(v[2], inverse), 0x04000c0cu);
  return lo | hi;
}
__device__ __forceinline__ u32x2 pack_codes(const float (&v)[8], unsigned byte) { return u32x2{pack4(v, byte), pack4(v + 4, byte)}; }
__device__ __forceinline__ void decode4(unsigned c, float step, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)(signed char)(c >> (8 * i)) * step;
}
__device__ __forceinline__ void decode8(u32x2 c, float step, float (&v)[8]) { decode4(c[0], step, v); decode4(c[1], step, v + 4); }
// A finite fp16 number of 65024 or more becomes 64 steps of 1024: 65536, past fp16's largest finite value, at which it is
// held.  Nothing larger comes of fp16 numbers (a code is a multiple of its step); rows of bf16 or fp32 that leave fp16's
// range become infinities, as in any conversion.
__device__ __forceinline__ float hold_fp16(float y) { return fabsf(y) == 65536.f ? __builtin_copysignf(65504.f, y) : y; }

// ---- 8-bit rows in an fp16 product ---------------------------------------------------------------------------------------
// fp16 holds a code exactly from steps of 2^-24 to steps of 2^9, fewer than rows come with.  So each group of 32 columns is
// brought to where its largest step over all rows is 2^9 (`tops`: that step's byte), by a power of two that the finished sums
// of those columns are divided by again: exact for steps down to 2^-33 of the column's largest, below that rounded to
// half of fp16's least number, under 2^-41 of the column's largest magnitude.
constexpr int UNIT_BYTE = 136;                                           // 127 steps of 2^9 = 65024
__device__ __forceinline__ unsigned unit_byte(unsigned byte, unsigned top) {      // a step in those units; 0 (no step) under 2^-126
  const int b = (int)byte - (int)top + UNIT_BYTE;
  return byte == 255u ? 255u : (unsigned)(b > 0 ? b : 0);
}
__device__ __forceinline__ float from_unit(float sum, int top) { return __builtin_ldexpf(sum, top - UNIT_BYTE); }

// ---- activations -----------------------------------------------------------------------------------------------------
// Phi(-a), the normal distribution's lower tail: log2 Phi(-a) is close to a parabola, and a degree-8 polynomial (minimax in
// Chebyshev form over [0, 10] by reweighted least squares, weight Phi(-a) max(1, a), and no less than what holds log2 to 1.3)
// followed by one exp2.  x Phi(x) is then off by 2.4e-8 rms over [-2, 2] and by 2.7e-7 at most for |x| < 12, the last
// rounding included (the fp32 erf form: 2.7e-8 and 4.5e-7), and by under 1e-10 below -6; past 10 the value at 10,
// 2e-28, is kept.  Every instruction here is issued once for each element of a product's result, beside which the matrix
// pipe stands still; degree 6 is two fewer of about fifteen and saves 3 of 120 us (forward with GELU and codes at
// 10960 x 4096 x 1024), for 9.2e-8, which is more than a step of fp16's smallest numbers.
constexpr float TAIL_END = 10.f;
__device__ __forceinline__ float phi_tail(float a) {
  float p = -1.548175071e-06f;
  p = __builtin_fmaf(p, a, 2.463692853e-05f);
  p = __builtin_fmaf(p, a, -1.197106250e-04f);
  p = __builtin_fmaf(p, a, -2.877795426e-04f);
  p = __builtin_fmaf(p, a, 7.246168278e-03f);
  p = __builtin_fmaf(p, a, -5.261169310e-02f);
  p = __builtin_fmaf(p, a, -4.591737758e-01f);
  p = __builtin_fmaf(p, a, -1.151108997e+00f);
  p = __builtin_fmaf(p, a, -9.999999251e-01f);
  return __builtin_amdgcn_exp2f(p);
}
__device__ __forceinline__ float relu_of(float x) { return __builtin_elementwise_maximum(x, 0.f); }      // a NaN stays one
// x Phi(x) = max(x, 0) - |x| Phi(-|x|)
__device__ __forceinline__ float gelu_of(float x) {
  const float a = fminf(fabsf(x), TAIL_END);
  return __builtin_fmaf(-a, phi_tail(a), relu_of(x));
}
// value and derivative for a decoded x (finite or NaN): Phi(x) + x phi(x), phi(x) = exp(-x^2 / 2) / sqrt(2 pi)
__device__ __forceinline__ void gelu_both(float x, float& value, float& slope) {
  const float a = fminf(fabsf(x), TAIL_END), q = phi_tail(a);
  value = __builtin_fmaf(-a, q, relu_of(x));
  const float bell = __builtin_amdgcn_exp2f(x * x * -0.7213475204f);       // 0 for large x, NaN for NaN
  slope = __builtin_fmaf(x * 0.3989422804f, bell, 0.5f + __builtin_copysignf(0.5f - q, x));
}
__device__ __forceinline__ float relu_slope(float x) { return x > 0.f ? 1.f : x != x ? x : 0.f; }

// codes [M, D] -> fp16 [M, width], both ends as above; tops [groups], behind it room for the rows' parts (train_rows.hip)
long long tops_bytes(int M, int D);
int unpack8_units(const void* codes, const void* exponents, unsigned char* tops, void* out, int M, int D, int width, hipStream_t st);

}  // namespace train

// Products with few rows (up to 32: single tokens, pooled features), included by train_linear.hip.  What bounds them is the
// latency of one pass over the weight, so there is no staging, no split sum with a second kernel and no padded copy: a
// block owns 32 (forward) or 64 (input gradient) columns of the result, its eight waves take the k32 steps in turn and read
// fragments straight from memory into registers, at any alignment; the partial tiles meet in LDS in wave order.
#pragma once
#include "train_common.h"

namespace {
using namespace train;

constexpr int FEW_ROWS = 32, FEW_WAVES = 8;

struct Few {
  const void* A; const void* B; const float* scale;        // scale: of A's columns (input gradient), or null
  long long lda, ldb; int M, N, K;                          // result [M, N], sum over K
  int parts;                                                // 16-bit parts that A * scale is taken in
};

// ALONG: B is [N][K] (forward), a lane's fragment is one load; otherwise B is [K][N] (input gradient): a lane loads four
// columns of eight rows and byte permutes turn them into the fragments of those four columns.  The loads of whole k32
// steps have no branch among them (a step past the last is read again and zeroed; columns past the end are shifted out
// of the last whole four), so those of STEPS steps are in flight together; the part of a step left at the end of the sum
// is one wave's, element by element.
template <class T, int DT, int MT, bool ALONG, class Epi>
__global__ __launch_bounds__(FEW_WAVES * 64) void train_few_kernel(Few g, Epi epi) {
  constexpr int COLS = ALONG ? 32 : 64, NF = COLS / 16, STEPS = MT == 1 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) float part[FEW_WAVES][MT * 16][COLS];
  using H = Half<T>;
  using v8 = typename H::v8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * COLS, whole = g.K / 32;
  const unsigned short* const A = reinterpret_cast<const unsigned short*>(g.A);
  const unsigned short* const B = reinterpret_cast<const unsigned short*>(g.B);
  // rows past the last repeat it, unused; the same for B's rows along k
  const unsigned short* pa[MT];
  const unsigned short* pb[ALONG ? NF : 1];
  int shift = 0;                                              // bits of a lane's four columns that lie past the end
#pragma unroll
  for (int i = 0; i < MT; ++i) pa[i] = A + (size_t)(16 * i + fr < g.M ? 16 * i + fr : g.M - 1) * g.lda + 8 * fq;
  if constexpr (ALONG) {
#pragma unroll
    for (int j = 0; j < NF; ++j) pb[j] = B + (size_t)(n0 + 16 * j + fr < g.N ? n0 + 16 * j + fr : g.N - 1) * g.ldb + 8 * fq;
  } else {
    const int n = n0 + 4 * fr, from = n < g.N - 4 ? n : g.N - 4;             // N >= 4
    pb[0] = B + (size_t)(8 * fq) * g.ldb + from;
    shift = n - from < 4 ? 16 * (n - from) : 64;
  }
  f32x4 acc[MT][NF];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float up = 1.f, down = 1.f;
  if (DT == DT_FP16 && g.scale) scale_units(wave_top(g.scale, g.K, lane, 64), up, down);
  auto four = [&](u32x2 w) __attribute__((always_inline)) {
    if (shift == 0) return w;
    const unsigned long long x = ((unsigned long long)w[1] << 32) | w[0];
    const unsigned long long y = shift < 64 ? x >> shift : 0ULL;
    return u32x2{(unsigned)y, (unsigned)(y >> 32)};
  };
  // one step from loaded operands: k its first element for this lane, `limit` the sum's end
  auto multiply = [&](u32x4v (&af)[MT], u32x4v (&bf)[NF], const u32x2* raw, int k, int limit) __attribute__((always_inline)) {
    if constexpr (!ALONG) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = 0; d < 4; ++d)
          bf[j][d] = __builtin_amdgcn_perm(raw[2 * d + 1][j >> 1], raw[2 * d][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
    }
    float v[MT][8];
    if (g.scale) {
      float s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = g.scale[k + j < limit ? k + j : limit - 1] * up;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        cvt_raw8(Raw8{af[i], af[i]}, DT, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = k + j < limit ? v[i][j] * s[j] : 0.f;
        take_part(v[i], DT, &af[i]);
      }
    }
    for (int p = 0;;) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = H::mfma16(__builtin_bit_cast(v8, bf[j]), __builtin_bit_cast(v8, af[i]), acc[i][j]);
      if (++p >= g.parts) break;                              // uniform over the launch
#pragma unroll
      for (int i = 0; i < MT; ++i) take_part(v[i], DT, &af[i]);
    }
  };

  for (int c0 = wave; c0 < whole; c0 += FEW_WAVES * STEPS) {
    u32x4v af[STEPS][MT], bf[STEPS][NF];
    u32x2 raw[STEPS][8];
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      const int c = c0 + FEW_WAVES * u < whole ? c0 + FEW_WAVES * u : whole - 1;
#pragma unroll
      for (int i = 0; i < MT; ++i) __builtin_memcpy(&af[u][i], pa[i] + 32 * c, 16);
      if constexpr (ALONG) {
#pragma unroll
        for (int j = 0; j < NF; ++j) __builtin_memcpy(&bf[u][j], pb[j] + 32 * c, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) __builtin_memcpy(&raw[u][e], pb[0] + (size_t)(32 * c + e) * g.ldb, 8);
      }
    }
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      const int c = c0 + FEW_WAVES * u;
      if (c >= whole) break;                                  // uniform over the wave
      if constexpr (!ALONG) {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[u][e] = four(raw[u][e]);
      }
      multiply(af[u], bf[u], raw[u], 32 * c + 8 * fq, g.K);
    }
  }
  if (whole * 32 < g.K && wave == whole % FEW_WAVES) {
    const int k = 32 * whole + 8 * fq, left = g.K - k;        // of this lane's eight, `left` exist (none if negative)
    u32x4v af[MT], bf[NF];
    u32x2 raw[8];
    // the last eight of a row in one load, moved down over those that are not this lane's (a row of fewer: one by one)
    auto some = [&](const unsigned short* p) __attribute__((always_inline)) {
      u32x4v w;
      if (g.K >= 8) {
        const int by = left < 0 ? 8 : left < 8 ? 8 - left : 0;
        __builtin_memcpy(&w, left < 8 ? p + (left - 8) : p, 16);
        if (by & 4) w = u32x4v{w[2], w[3], 0u, 0u};
        if (by & 2) w = u32x4v{w[1], w[2], w[3], 0u};
        if (by & 1) w = u32x4v{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
        return by < 8 ? w : u32x4v{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (2 * j < left ? (unsigned)p[2 * j] : 0u) | (2 * j + 1 < left ? (unsigned)p[2 * j + 1] << 16 : 0u);
      return w;
    };
#pragma unroll
    for (int i = 0; i < MT; ++i) af[i] = some(pa[i] + 32 * whole);
    if constexpr (ALONG) {
#pragma unroll
      for (int j = 0; j < NF; ++j) bf[j] = some(pb[j] + 32 * whole);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        __builtin_memcpy(&raw[e], pb[0] + ((long long)(32 * whole) + (e < left ? e : left - 1)) * g.ldb, 8);      // k + left = K
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        raw[e] = four(raw[e]);
        if (e >= left) raw[e] = u32x2{0, 0};
      }
    }
    multiply(af, bf, raw, k, g.K);
  }
  if (DT == DT_FP16 && g.scale) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[i][j] *= down;
  }
  // element e of a lane is column 16 j + 4 q + e (forward), 4 (4 q + e) + j (input gradient) of row 16 i + fr
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (ALONG) {
        if (j < NF) *reinterpret_cast<f32x4*>(&part[wave][16 * i + fr][16 * (j % NF) + 4 * fq]) = acc[i][j % NF];
      } else {
        *reinterpret_cast<f32x4*>(&part[wave][16 * i + fr][16 * fq + 4 * j]) = f32x4{acc[i][0][j], acc[i][1 % NF][j], acc[i][2 % NF][j], acc[i][3 % NF][j]};
      }
    }
  __syncthreads();
  constexpr int RUNS = COLS / 8;
  const int m = threadIdx.x / RUNS, at = (threadIdx.x % RUNS) * 8, n = n0 + at;
  if (m >= MT * 16) return;                                  // whole waves
  const int col_n = n < g.N ? n : 0;
  typename Epi::Columns col;
  epi.columns(col_n, col);
  typename Epi::Row row;
  epi.template fetch<false>(m, n, row);
  float v[8];
  epi.start(col_n, v);
#pragma unroll
  for (int w = 0; w < FEW_WAVES; ++w)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += part[w][m][at + j];
  epi.template finish<false, 1, 2>(0, m, n, v, col, row, nullptr);
}

// Whether these take a product: beyond a sum of 2048 the waves' turns outlast the tiled loop with a split sum
// (16 x 1024 with K = 4096: 13 us both ways; 32 x 4096 x 4096: 17 against 14), under it one launch is shorter
// (5 x 1024 x 1024: 5 against 8 us).
inline bool few_rows(int M, int N, int K, bool along) { return M <= FEW_ROWS && K <= 2048 && (along || N >= 4); }

template <class T, int DT, bool ALONG, class Epi> int launch_few(const Few& g, const Epi& e, hipStream_t st) {
  const dim3 grid((unsigned)((g.N + (ALONG ? 31 : 63)) / (ALONG ? 32 : 64))), block(FEW_WAVES * 64);
  if (g.M <= 16) hipLaunchKernelGGL((train_few_kernel<T, DT, 1, ALONG, Epi>), grid, block, 0, st, g, e);
  else hipLaunchKernelGGL((train_few_kernel<T, DT, 2, ALONG, Epi>), grid, block, 0, st, g, e);
  return COGAIM_LAUNCH_CHECK();
}

}  // namespace

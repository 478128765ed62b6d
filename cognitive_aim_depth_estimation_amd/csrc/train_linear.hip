// Linear layers' training products: forward with bias, activation, LayerScale, residual and an 8-bit copy of the
// pre-activation in the epilogue; gradient of the input with the derivative of the activation below in the epilogue;
// gradients of weight, bias and LayerScale.  Main loop in train_gemm.h.
//
// Every product is one launch of the main loop when its tiles fill the chip; with fewer tiles the sum is split over k,
// the parts leave fp32 partial tiles in the workspace and a join kernel adds them in order and applies the epilogue
// (no atomics: results do not depend on timing).
#include "train_gemm.h"
#include "train_few.h"
#include "../../include/cogaim.h"

namespace {

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
constexpr int MAX_M = 0x7fffffff - 511;    // rows: those of the last tile still have 32-bit numbers
constexpr long long MAX_LD = 1 << 21;      // a tile's 256 rows stay inside a buffer resource's 32-bit offsets

// ---- epilogues ---------------------------------------------------------------------------------------------------
// finish<FAST, X1, X2>: eight columns [n, n + 8) of row m; the four lanes that hold a group of 32 are X1 and X2 apart.
// Every lane of the wave calls it (the 8-bit group maximum crosses lanes); rows and columns past the matrix are dropped
// here.  FAST: the width is a multiple of eight (`fast()`), so no run is cut; stores go past the caches (2 % of a large
// launch, left to the operands' lines).  The wider tiles carry only that form, up to sixteen times unrolled, and leave
// any other result to the join kernel.
//
// fp32 rows: a lane's eight columns are 32 bytes, and a 16-byte access of every lane would touch half of each sector.  The
// row swap of lane halves turns them (lane bit 5 against the half of the eight): a lane then holds columns
// 8 (q % 2) + 4 (q / 2) .. + 3 of the first and of the last 16 of its group of 32, and an access covers 64 bytes of a row.
__device__ __forceinline__ void turn8(float (&y)[8]) {                    // its own inverse
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(y[j]), __float_as_uint(y[4 + j]), false, false);
    y[j] = __uint_as_float(t[0]); y[4 + j] = __uint_as_float(t[1]);
  }
}
__device__ __forceinline__ int turned_column(int n) {                     // of the first of the two; the other is 16 on
  const int q = (n >> 3) & 3;
  return (n & ~(GROUP - 1)) + 8 * (q & 1) + 4 * (q >> 1);
}
// FAST calls come from whole waves but for lanes past the last row
template <bool FAST, bool STREAM = true>
__device__ __forceinline__ void store_run8(void* p, int dt, long long ld, int m, int n, int N, float (&y)[8]) {
  if (FAST && dt == DT_FP32) {
    turn8(y);
    const int c = turned_column(n);
    f32x4_any* q = reinterpret_cast<f32x4_any*>(reinterpret_cast<float*>(p) + (size_t)m * ld + c);
    const f32x4_any lo = {y[0], y[1], y[2], y[3]}, hi = {y[4], y[5], y[6], y[7]};
    if constexpr (STREAM) {
      if (c < N) __builtin_nontemporal_store(lo, q);
      if (c + 16 < N) __builtin_nontemporal_store(hi, q + 4);
    } else {
      if (c < N) q[0] = lo;
      if (c + 16 < N) q[4] = hi;
    }
    return;
  }
  if (n >= N) return;
  const size_t at = (size_t)m * ld + n;
  if (FAST || n + 8 <= N) store_vec8<FAST>(p, dt, at, y);
  else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n + j < N) store_one(p, dt, at + j, y[j]);
  }
}

// largest of the four lanes X1 and X2 apart: row swaps (16, 32) or quad permutations (1, 2), not the LDS permute's round trip
template <int X1, int X2> __device__ __forceinline__ unsigned max_of_four(unsigned u) {
  static_assert((X1 == 16 && X2 == 32) || (X1 == 1 && X2 == 2), "the two layouts of a group");
  if constexpr (X1 == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    u = umax(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return umax(b[0], b[1]);
  } else {
    u = umax(u, (unsigned)__builtin_amdgcn_mov_dpp((int)u, 0xB1 /* quad_perm [1,0,3,2] */, 0xf, 0xf, true));
    return umax(u, (unsigned)__builtin_amdgcn_mov_dpp((int)u, 0x4E /* quad_perm [2,3,0,1] */, 0xf, 0xf, true));
  }
}

// PRE: with the 16-bit copy.  A form of its own: tested for at run time, its stores cost the others 10 % (10960 x 4096 x 1024 with
// GELU and codes, call with unpack: 135 -> 149 us).
template <int ACT, bool PRE>
struct EpiForward {                          // y = act(acc + bias) * scale + residual, codes and 16-bit copy of acc + bias
  const float* bias; const float* scale; const void* res; void* y; signed char* codes; unsigned char* bytes; void* pre;
  long long ldr, ldy; int M, N, res_dt, y_dt, pre_dt;
  static constexpr int TABLE = 0;            // float2 entries of LDS the epilogue wants
  __device__ __forceinline__ void fill(float2*, int, int) const {}
  bool fast() const { return (N & 7) == 0; }
  struct Columns { float s[8]; };
  struct Row { Raw8 r; };
  // where the sums of columns n .. n + 7 begin
  __device__ __forceinline__ void start(int n, float (&b)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = bias ? bias[n + j < N ? n + j : N - 1] : 0.f;
  }
  __device__ __forceinline__ void columns(int n, Columns& c) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = n + j < N ? n + j : N - 1;
      c.s[j] = ACT == ACT_NONE && scale ? scale[at] : 1.f;
    }
  }
  template <bool FAST>
  __device__ __forceinline__ void fetch(int m, int n, Row& r) const {
    if (!res || m >= M) return;
    if (FAST && res_dt == DT_FP32) {
      const int c = turned_column(n);
      const float* q = reinterpret_cast<const float*>(res) + (size_t)m * ldr + c;
      r.r.a = c < N ? (u32x4v)*reinterpret_cast<const u32x4_any*>(q) : u32x4v{0, 0, 0, 0};
      r.r.b = c + 16 < N ? (u32x4v)*reinterpret_cast<const u32x4_any*>(q + 16) : u32x4v{0, 0, 0, 0};
    } else if ((FAST || n + 8 <= N) && n < N) r.r = load_raw8(res, res_dt, (size_t)m * ldr + n);
  }
  template <bool FAST, int X1, int X2>
  __device__ __forceinline__ void finish(int, int m, int n, float (&v)[8], const Columns& c, const Row& r, const float2*) const {
    if (codes) {
      if constexpr (!FAST) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = n + j < N ? v[j] : 0.f;
      }
      unsigned top = n < N ? top_bits<8>(v) : 0u;
      top = max_of_four<X1, X2>(top);
      if (m < M && n < N) {
        const unsigned byte = group_byte(top);
        const u32x2 q = pack_codes(v, byte);
        signed char* to = codes + (size_t)m * N + n;
        if (FAST || n + 8 <= N) *reinterpret_cast<u32x2_any*>(to) = q;
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < N) to[j] = (signed char)(q[j >> 2] >> (8 * (j & 3)));
        }
        if ((n & (GROUP - 1)) == 0) bytes[(size_t)m * groups_of(N) + n / GROUP] = (unsigned char)byte;
      }
    }
    if (m >= M) return;                          // lanes of one row leave together
    if constexpr (PRE) store_run8<FAST>(pre, pre_dt, N, m, n, N, v);      // 16 bits: v stays in place
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (ACT == ACT_RELU) v[j] = relu_of(v[j]);
      else if constexpr (ACT == ACT_GELU) v[j] = gelu_of(v[j]);
      else v[j] *= c.s[j];
    }
    if (res) {
      float a[8];
      if (FAST || n + 8 <= N) {
        cvt_raw8(r.r, res_dt, a);
        if (FAST && res_dt == DT_FP32) turn8(a);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = n + j < N ? load_one(res, res_dt, (size_t)m * ldr + n + j) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += a[j];
    }
    store_run8<FAST>(y, y_dt, ldy, m, n, N, v);
  }
};

// dx = acc * act'(u), a = act(u), u from its 8-bit copy.  GELU and its derivative take about 30 instructions an element,
// during which the matrix pipe stands: two fifths of the launch at 5480 x 1024 x 4096.  But a code has 256 values and
// few steps occur, so the main loop's blocks hold both functions of every code at the eight steps 2^-9 .. 2^-2 (groups
// whose largest magnitude lies between 1/8 and 32) in 16 KB of LDS, filled while their first loads are in flight;
// other groups are computed.  Both ways give the same bits.
// 5480 x 1024 x 4096: 75 -> 70 us.
constexpr unsigned TABLE_FIRST = 118;        // exponent byte of 2^-9
constexpr int TABLE_STEPS = 8;
template <int ACT>
struct EpiInput {
  const signed char* codes; const unsigned char* bytes; void* dx; void* a; long long lddx, lda;
  int M, N, dx_dt, a_dt;
  const float* unit;                           // what the sums are multiplied by (see scale_units), or null
  static constexpr int TABLE = ACT == ACT_GELU ? TABLE_STEPS * 256 : 0;
  __device__ __forceinline__ void fill(float2* table, int tid, int threads) const {
    if constexpr (ACT == ACT_GELU)
      for (int i = tid; i < TABLE; i += threads) {
        float2 f;
        gelu_both((float)((i & 255) - 128) * group_step(TABLE_FIRST + (i >> 8)), f.x, f.y);
        table[i] = f;
      }
  }
  bool fast() const { return (N & 7) == 0; }
  struct Columns {};
  struct Row { u32x2 q; unsigned byte; };
  __device__ __forceinline__ void start(int, float (&b)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.f;
  }
  __device__ __forceinline__ void columns(int, Columns&) const {}
  template <bool FAST>
  __device__ __forceinline__ void fetch(int m, int n, Row& r) const {
    r.q = u32x2{0, 0}; r.byte = 1;
    if constexpr (ACT != ACT_NONE) {
      if (m < M && n < N) {
        const signed char* p = codes + (size_t)m * N + n;
        if (FAST || n + 8 <= N) r.q = *reinterpret_cast<const u32x2_any*>(p);
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < N) r.q[j >> 2] |= (unsigned)(unsigned char)p[j] << (8 * (j & 3));
        }
        r.byte = bytes[(size_t)m * groups_of(N) + n / GROUP];
      }
    }
  }
  template <bool FAST, int X1, int X2>
  __device__ __forceinline__ void finish(int, int m, int n, float (&v)[8], const Columns&, const Row& r, const float2* table) const {
    if (m >= M) return;                          // lanes of one row leave together
    if (unit) {
      const float f = *unit;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
    }
    if constexpr (ACT != ACT_NONE) {
      float u[8];
      const bool listed = ACT == ACT_GELU && FAST && (n >= N || r.byte - TABLE_FIRST < (unsigned)TABLE_STEPS);
      if (ACT == ACT_GELU && FAST && __all(listed)) {
        const float2* t = table + (n < N ? (r.byte - TABLE_FIRST) << 8 : 0u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = t[(r.q[j >> 2] ^ 0x80808080u) >> (8 * (j & 3)) & 255u];
          u[j] = f.x;
          v[j] *= f.y;
        }
      } else {
        decode8(r.q, group_step(r.byte), u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float value, slope;
          if constexpr (ACT == ACT_GELU) gelu_both(u[j], value, slope);
          else { value = relu_of(u[j]); slope = relu_slope(u[j]); }
          v[j] *= slope;
          u[j] = a_dt == DT_FP16 ? hold_fp16(value) : value;      // finite where the forward's was
        }
      }
      if (a) store_run8<FAST>(a, a_dt, lda, m, n, N, u);
    }
    store_run8<FAST>(dx, dx_dt, lddx, m, n, N, v);
  }
};

struct EpiPlain {                            // the product itself, brought back from its columns' units (tops, or null)
  void* out; long long ld; int M, N, dt; const unsigned char* tops;
  static constexpr int TABLE = 0;
  __device__ __forceinline__ void fill(float2*, int, int) const {}
  struct Columns { int top; };
  struct Row {};
  __device__ __forceinline__ void start(int, float (&b)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.f;
  }
  __device__ __forceinline__ void columns(int n, Columns& c) const { c.top = tops && n < N ? tops[n / GROUP] : UNIT_BYTE; }
  template <bool FAST>
  __device__ __forceinline__ void fetch(int, int, Row&) const {}
  template <bool FAST, int X1, int X2>
  __device__ __forceinline__ void finish(int, int m, int n, float (&v)[8], const Columns& c, const Row&, const float2*) const {
    if (m >= M) return;
    if (tops) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = from_unit(v[j], c.top);
    }
    store_run8<FAST>(out, dt, ld, m, n, N, v);
  }
};

struct EpiPart {                             // fp32 partial sums [split][M][Np], Np = N rounded up to 8
  float* part; int M, Np;
  static constexpr int TABLE = 0;
  __device__ __forceinline__ void fill(float2*, int, int) const {}
  struct Columns {};
  struct Row {};
  __device__ __forceinline__ void start(int, float (&b)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.f;
  }
  __device__ __forceinline__ void columns(int, Columns&) const {}
  template <bool FAST>
  __device__ __forceinline__ void fetch(int, int, Row&) const {}
  template <bool FAST, int X1, int X2>
  __device__ __forceinline__ void finish(int split, int m, int n, float (&v)[8], const Columns&, const Row&, const float2*) const {
    if (m < M) store_run8<true, false>(part + (size_t)split * M * Np, DT_FP32, Np, m, n, Np, v);      // read back at once
  }
};

// adds the parts of eight columns in split order and applies the epilogue; four neighbouring threads hold a group.  `first`:
// the first of the launch's threads among all of them.
template <class Epi>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits, int M, int N, int Np, long long first, Epi epi) {
  const int per_row = (int)groups_of(N) * 4;
  const long long i = first + blockIdx.x * 256LL + threadIdx.x;
  const long long row = i / per_row;
  const int n = (int)(i - row * per_row) * 8;
  const int m = row < M ? (int)row : M;                       // past the end: dropped by the epilogue
  typename Epi::Columns col;
  epi.columns(n < N ? n : 0, col);
  typename Epi::Row r;
  epi.template fetch<false>(m, n, r);
  float v[8];
  epi.start(n < N ? n : 0, v);
  if (m < M && n < N) {
    for (int s = 0; s < splits; ++s) {
      const float4* p = reinterpret_cast<const float4*>(part + ((size_t)s * M + m) * Np + n);
      const float4 x = p[0], y = p[1];
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
  }
  epi.template finish<false, 1, 2>(0, m, n, v, col, r, nullptr);
}

// ROWS rows n of the weight's gradient to a block (their loads in flight together):  G = sum of the parts, out of its
// columns' units (tops, or null), with
// x = xh * xs + xt put back  (sum_m dy (xh xs + xt) = (dy^T xh) xs + (sum_m dy) xt);  dW = s G, db = s sum dy,
// ds = sum_k W G + b sum dy.  Four rows where they still make 512 blocks (12 against 17 us at 4096 x 1024 in two
// parts); one row, for more blocks, below.
struct WeightFinish {
  const float* part; const float* col_sum; const float* xs; const float* xt; const float* scale; const unsigned short* W;
  const float* bias; void* dW; float* db; float* ds; const unsigned char* tops; long long ldw, lddw; int N, K, Kp, splits, dt, dw_dt;
};
template <int ROWS>
__global__ __launch_bounds__(256) void weight_finish_kernel(WeightFinish a) {
  __shared__ float red[ROWS][4];
  const int n0 = blockIdx.x * ROWS;
  int row[ROWS];
  float total[ROWS], sc[ROWS], dot[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    row[r] = n0 + r < a.N ? n0 + r : a.N - 1;
    total[r] = 0.f; dot[r] = 0.f;
    sc[r] = a.scale ? a.scale[row[r]] : 1.f;
  }
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) total[r] += a.col_sum[(size_t)s * a.N + row[r]];
  for (int k = threadIdx.x * 4; k < a.K; k += 1024) {
    f32x4 g[ROWS];
    float w[ROWS][4];
    if (a.ds) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const unsigned short* q = a.W + (size_t)row[r] * a.ldw + k;
        unsigned short h[4] = {0, 0, 0, 0};
        if (k + 4 <= a.K) __builtin_memcpy(h, q, 8);
        else {
#pragma unroll
          for (int j = 0; j < 4; ++j) if (k + j < a.K) h[j] = q[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) w[r][j] = a.dt == DT_BF16 ? __uint_as_float((unsigned)h[j] << 16) : half_bits(h[j]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) g[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const f32x4 p = *reinterpret_cast<const f32x4*>(a.part + ((size_t)s * a.N + row[r]) * a.Kp + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) g[r][j] += p[j];
      }
    float xs[4], xt[4];
    const int top = a.tops ? a.tops[k / GROUP] : UNIT_BYTE;              // four columns of one group
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = k + j < a.K ? k + j : a.K - 1;
      xs[j] = a.xs ? a.xs[at] : 1.f;
      xt[j] = a.xt ? a.xt[at] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (n0 + r >= a.N) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (a.tops) g[r][j] = from_unit(g[r][j], top);
        if (a.xs) g[r][j] *= xs[j];
        if (a.xt) g[r][j] = __builtin_fmaf(total[r], xt[j], g[r][j]);
        if (a.ds && k + j < a.K) dot[r] = __builtin_fmaf(w[r][j], g[r][j], dot[r]);
        g[r][j] *= sc[r];
      }
      const size_t at = (size_t)row[r] * a.lddw + k;
      if (k + 4 <= a.K && a.dw_dt == DT_FP32) *reinterpret_cast<f32x4_any*>(reinterpret_cast<float*>(a.dW) + at) = g[r];
      else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k + j < a.K) store_one(a.dW, a.dw_dt, at + j, g[r][j]);
      }
    }
  }
  if (a.ds) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float d = wave_sum_dpp(dot[r]);
      if ((threadIdx.x & 63) == 0) red[r][threadIdx.x >> 6] = d;
    }
    __syncthreads();
  }
  if (threadIdx.x < ROWS && n0 + (int)threadIdx.x < a.N) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if ((int)threadIdx.x == r) {
        if (a.ds) a.ds[n0 + r] = (red[r][0] + red[r][1]) + (red[r][2] + red[r][3]) + (a.bias ? a.bias[n0 + r] * total[r] : 0.f);
        a.db[n0 + r] = sc[r] * total[r];
      }
  }
}

// Copies of operands whose rows the DMA's 16-byte loads cannot address (odd widths, strides or bases), padded with zeros to
// a multiple of eight columns; with `scale`, row r times scale[r] (in fp16 times scale[r] * up, and *unit = down).  The
// matrix cores take 16 bits.  For a 16-bit result the product is rounded once: the terms' roundings are independent, together
// about one rounding of a sum of their size, as the result's own (error against 64 bits 2.4e-3 with both, 1.7e-3 with the
// result's alone, in bf16).  An fp32 result keeps its precision: the copy then holds `parts` matrices, each the 16-bit rounding
// of what the ones before it left, and the product is taken with each (5480 x 1024 x 4096 through GELU: 274 us; rounded once,
// into bf16, 73).
// Both operands of a product in one launch: blocks [0, blocks0) copy the first.
struct CopyOne { const unsigned short* src; unsigned short* dst; const float* scale; float* unit; long long ld; int rows, cols, padded, parts; };
struct CopyTwo { CopyOne one[2]; unsigned blocks0; int dt; };
__global__ __launch_bounds__(256) void copy_rows_kernel(CopyTwo a) {
  const bool second = blockIdx.x >= a.blocks0;
  const CopyOne& c = a.one[second];
  const unsigned block = second ? blockIdx.x - a.blocks0 : blockIdx.x, blocks = second ? gridDim.x - a.blocks0 : a.blocks0;
  float up = 1.f;
  if (c.unit) {                                                           // uniform over the block
    __shared__ unsigned tops[4];
    const unsigned mine = wave_top(c.scale, c.rows, threadIdx.x, 256);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = mine;
    __syncthreads();
    const unsigned t0 = tops[0] > tops[1] ? tops[0] : tops[1], t1 = tops[2] > tops[3] ? tops[2] : tops[3];
    float down;
    scale_units(t0 > t1 ? t0 : t1, up, down);
    if (block == 0 && threadIdx.x == 0) *c.unit = down;
  }
  const unsigned runs = (unsigned)c.padded / 8;
  const unsigned long long total = (unsigned long long)c.rows * runs;
  for (unsigned long long i = block * 256ULL + threadIdx.x; i < total; i += 256ULL * blocks) {
    const unsigned long long r = total < (1ULL << 32) ? (unsigned)i / runs : i / runs;
    const int k0 = (int)(i - r * runs) * 8;
    const unsigned short* src = c.src + r * c.ld + k0;
    u32x4v w;
    if (k0 + 8 <= c.cols) __builtin_memcpy(&w, src, 16);               // of any alignment
    else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (k0 + 2 * j < c.cols ? (unsigned)src[2 * j] : 0u) | (k0 + 2 * j + 1 < c.cols ? (unsigned)src[2 * j + 1] << 16 : 0u);
    }
    if (c.scale) {
      const float s = c.scale[r] * up;
      float v[8];
      cvt_raw8(Raw8{w, w}, a.dt, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k0 + j < c.cols ? v[j] * s : 0.f;   // the padding stays zero whatever the scale
      take_part(v, a.dt, &w);
      for (int p = 1; p < c.parts; ++p) {
        u32x4v low;
        take_part(v, a.dt, &low);
        *reinterpret_cast<u32x4v*>(c.dst + ((unsigned long long)p * c.rows + r) * c.padded + k0) = low;
      }
    }
    *reinterpret_cast<u32x4v*>(c.dst + r * c.padded + k0) = w;
  }
}

// ---- plans -------------------------------------------------------------------------------------------------------
using T256 = Tile<256, 256, 2, 4, 2, true>;
using T192 = Tile<192, 256, 2, 4, 2, true>;        // A contiguous along k only: its 192 columns across k have no XOR swizzle
using T128W = Tile<128, 256, 2, 4, 2, true>;
using T128 = Tile<128, 128, 2, 2, 2, true>;
using T64 = Tile<64, 64, 2, 2, 4, false>;
enum { TILE_256, TILE_192, TILE_128W, TILE_128, TILE_64, TILES };
// What a launch takes, in us, measured on MI355X over 14 shapes from 5 x 1024 x 1024 to 21920 x 768 x 768 and each of the
// three layouts: `slots` blocks run at a time and a round of them takes per_k for each K-tile of 64 and `fixed` for
// its first loads and its stores; when at most half the slots are taken, a K-tile takes alone_k (less traffic, higher
// clock).  A wide tile reads the fewest bytes per product, a small one leaves fewer compute units idle in the last
// round: 5480 x 4096 x 1024 takes 58 us in 256 x 256 tiles (352 on 256 units), 50 in 192 x 256 (464), 53 in 128 x 256,
// 54 in 128 x 128 and 99 in 64 x 64; 1370 x 768 x 768 takes 22, 18, 15, 12 and 9.5; 10960 x 4096 x 1024 takes 89, 98,
// 104, 100 and 195.  `fixed` is one number for every layout and epilogue, which it is not: a tile's epilogue with GELU and codes
// takes about 8 us, and a tile of 64 x 64 with both operands across k (1370 x 768 x 768 weight gradient, three parts) 10 us where
// the table says 6.
struct TileCost { int m, n, slots; float per_k, fixed, alone_k; };
const TileCost TILE_COST[TILES] = {{256, 256, 256, 1.50f, 4.5f, 1.20f}, {192, 256, 256, 1.33f, 4.0f, 1.00f}, {128, 256, 256, 0.87f, 4.0f, 0.75f},
                                   {128, 128, 512, 0.92f, 2.6f, 0.61f}, {64, 64, 512, 0.43f, 2.5f, 0.35f}};
// Splitting the sum over k takes another kernel: about 5 us of launch and latency, and each partial sum written and
// read back once at 5 TB/s.
constexpr float JOIN_FIXED = 5.f, JOIN_PER_BYTE = 1.f / 5.0e6f;

int tile_threads(int tile) { return tile == TILE_128 || tile == TILE_64 ? 256 : 512; }

struct Shape { int tile, tiles_m, tiles_n, splits, kt_per_split; };

// `joined`: the second kernel runs whether or not the sum is split; `ragged`: it does but for the smallest tile
Shape shape_of(int M, int N, int K, bool a_along_k, bool joined, bool ragged) {
  const int nk = (K + TK - 1) / TK;
  Shape best{};
  float least = 0.f;
  for (int t = 0; t < TILES; ++t) {
    if (t == TILE_192 && !a_along_k) continue;
    const TileCost& c = TILE_COST[t];
    const int tm = (M + c.m - 1) / c.m, tn = (N + c.n - 1) / c.n;
    for (int want = 1; want <= 64; want += want < 4 ? 1 : want / 2) {
      if (want > 1 && nk < 2 * want) break;
      const int per = (nk + want - 1) / want, splits = (nk + per - 1) / per;            // no part is empty
      const double blocks = (double)tm * tn * splits;
      if (blocks * tile_threads(t) > (double)MAX_ITEMS) continue;           // (256 rows of a narrow result to a tile: any M)
      const double rounds = blocks <= c.slots ? 1.0 : (double)((long long)((blocks + c.slots - 1) / c.slots));
      float us = (float)rounds * (c.fixed + per * (blocks * 2 <= c.slots ? c.alone_k : c.per_k));
      if (splits > 1 || joined || (ragged && t != TILE_64)) us += JOIN_FIXED + JOIN_PER_BYTE * 8.f * splits * (float)M * (float)N;
      if (best.splits == 0 || us < least) {
        least = us;
        best = Shape{t, tm, tn, splits, per};
      }
    }
  }
  return best;
}

long long round256(long long v) { return (v + 255) / 256 * 256; }
int round8(int v) { return (v + 7) & ~7; }

// an operand as the main loop takes it: `copy` when 16-byte loads cannot address it
struct Side { const void* p; long long ld; int rows, cols; bool copy; const float* scale; float* unit; int parts; };
Side side(const void* p, long long ld, int rows, int cols, const float* scale = nullptr, int parts = 1) {
  Side s{p, ld, rows, cols, scale || (cols & 7) || (ld & 7) || !aligned(p, 16), scale, nullptr, parts};
  return s;
}
long long copy_bytes(const Side& s) { return s.copy ? round256((long long)s.rows * round8(s.cols) * 2 * s.parts) : 0; }

// copies those of the two operands that need it, moves `ws` behind them
int run_copies(Side& a, Side& b, int dt, char*& ws, hipStream_t st) {
  CopyTwo c{};
  c.dt = dt;
  unsigned blocks[2] = {0, 0};
  int n = 0;
  for (Side* s : {&a, &b}) {
    if (!s->copy) continue;
    const int c8 = round8(s->cols);
    const long long bytes = copy_bytes(*s);
    c.one[n] = CopyOne{(const unsigned short*)s->p, (unsigned short*)ws, s->scale, s->unit, s->ld, s->rows, s->cols, c8, s->parts};
    const unsigned long long want = ((unsigned long long)s->rows * (c8 / 8) + 255) / 256;
    blocks[n++] = (unsigned)(want > 256 * 16 ? 256 * 16 : want);
    s->p = ws; s->ld = c8; s->cols = c8;
    ws += bytes;
  }
  if (n == 0) return COGAIM_OK;
  c.blocks0 = blocks[0];
  hipLaunchKernelGGL(copy_rows_kernel, dim3(blocks[0] + blocks[1]), dim3(256), 0, st, c);
  return COGAIM_LAUNCH_CHECK();
}

template <class T, bool AKC, bool BKC, bool FAST = true, class Epi>
int launch_gemm(const Operands& g, int tile, const Epi& e, hipStream_t st) {
  const long long blocks = (long long)g.tiles_m * g.tiles_n * g.splits;
  if (blocks <= 0 || blocks * tile_threads(FAST ? tile : TILE_64) > MAX_ITEMS) return COGAIM_EINVAL;
#define TRAIN_LAUNCH(TL_) hipLaunchKernelGGL((train_gemm_kernel<T, AKC, BKC, TL_, Epi, FAST>), dim3((unsigned)blocks), dim3(TL_::NW * 64), 0, st, g, e)
  if constexpr (!FAST) TRAIN_LAUNCH(T64);
  else if (tile == TILE_256) TRAIN_LAUNCH(T256);
  else if (tile == TILE_192) {
    if constexpr (AKC) TRAIN_LAUNCH(T192);
    else return COGAIM_EINVAL;
  } else if (tile == TILE_128W) TRAIN_LAUNCH(T128W);
  else if (tile == TILE_128) TRAIN_LAUNCH(T128);
  else TRAIN_LAUNCH(T64);
#undef TRAIN_LAUNCH
  return COGAIM_LAUNCH_CHECK();
}

// the epilogue runs in a kernel of its own: parts to add, or a result that 16-byte stores cannot reach
template <class Epi> bool joins(const Shape& s, const Epi& e) { return s.splits > 1 || (!e.fast() && s.tile != TILE_64); }

// with several parts of B (matrices behind one another) the join adds their products, too
template <class T, bool AKC, bool BKC, class Epi>
int product(const Operands& g, const Shape& s, const Epi& e, float* part, hipStream_t st, int parts = 1) {
  if (parts == 1 && !joins(s, e)) return e.fast() ? launch_gemm<T, AKC, BKC>(g, s.tile, e, st) : launch_gemm<T, AKC, BKC, false>(g, s.tile, e, st);
  const int Np = round8(g.N);
  for (int p = 0; p < parts; ++p) {
    Operands one = g;
    one.B = reinterpret_cast<const unsigned short*>(g.B) + (size_t)p * g.ldb * (BKC ? g.rows_b : g.KB);
    const int rc = launch_gemm<T, AKC, BKC>(one, s.tile, EpiPart{part + (size_t)p * s.splits * g.M * Np, g.M, Np}, st);
    if (rc) return rc;
  }
  const long long threads = (long long)g.M * groups_of(g.N) * 4, most = MAX_ITEMS & ~255LL;
  for (long long first = 0; first < threads; first += most) {
    const long long n = threads - first < most ? threads - first : most;
    hipLaunchKernelGGL((join_kernel<Epi>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, s.splits * parts, g.M, g.N, Np, first, e);
  }
  return COGAIM_LAUNCH_CHECK();
}

Operands operands(const Side& a, const Side& b, bool akc, bool bkc, int M, int N, const Shape& s) {
  Operands g{};
  g.A = a.p; g.B = b.p; g.lda = a.ld; g.ldb = b.ld;
  g.rows_a = akc ? a.rows : a.cols; g.KA = akc ? a.cols : a.rows;
  g.rows_b = bkc ? b.rows : b.cols; g.KB = bkc ? b.cols : b.rows;
  g.M = M; g.N = N; g.tiles_m = s.tiles_m; g.tiles_n = s.tiles_n; g.splits = s.splits; g.kt_per_split = s.kt_per_split;
  g.col_sum = nullptr;
  return g;
}
bool half_dt(int dt) { return dt == DT_BF16 || dt == DT_FP16; }
bool any_dt(int dt) { return dt >= 0 && dt <= 2; }
bool matrix_ok(const void* p, long long ld, int cols, int elem) { return p && ld >= cols && ld <= MAX_LD && aligned(p, elem); }

bool forward_ok(const cogaim_linear_fwd_desc* d) {
  if (!d || d->M <= 0 || d->M > MAX_M || d->N <= 0 || d->K <= 0 || !half_dt(d->dtype) || !any_dt(d->y_dtype)) return false;
  if (!matrix_ok(d->x, d->ldx, d->K, 2) || !matrix_ok(d->w, d->ldw, d->K, 2) || !matrix_ok(d->y, d->ldy, d->N, dt_size(d->y_dtype))) return false;
  if (d->residual && (!any_dt(d->residual_dtype) || !matrix_ok(d->residual, d->ldr, d->N, dt_size(d->residual_dtype)))) return false;
  if (d->activation < ACT_NONE || d->activation > ACT_GELU || (d->scale && d->activation != ACT_NONE)) return false;
  if (d->extended == 1 && d->pre && !aligned(d->pre, 2)) return false;
  return !d->codes == !d->exponents;
}
bool input_ok(const cogaim_linear_bwd_input_desc* d) {
  if (!d || d->M <= 0 || d->M > MAX_M || d->N <= 0 || d->K <= 0 || !half_dt(d->dtype) || !any_dt(d->dx_dtype)) return false;
  if (!matrix_ok(d->dy, d->lddy, d->N, 2) || !matrix_ok(d->w, d->ldw, d->K, 2) || !matrix_ok(d->dx, d->lddx, d->K, dt_size(d->dx_dtype))) return false;
  if (d->activation < ACT_NONE || d->activation > ACT_GELU) return false;
  if ((d->activation == ACT_NONE) != !d->codes || !d->codes != !d->exponents) return false;
  return !d->a || (d->activation != ACT_NONE && matrix_ok(d->a, d->lda, d->K, 2));
}
bool weight_ok(const cogaim_linear_bwd_weight_desc* d) {
  if (!d || d->M <= 0 || d->M > MAX_M || d->N <= 0 || d->K <= 0 || !half_dt(d->dtype) || !any_dt(d->dw_dtype)) return false;
  if (!matrix_ok(d->dy, d->lddy, d->N, 2) || !matrix_ok(d->dw, d->lddw, d->K, dt_size(d->dw_dtype)) || !d->db) return false;
  if (!d->codes != !d->exponents || !d->x == !d->codes) return false;
  if (d->x && !matrix_ok(d->x, d->ldx, d->K, 2)) return false;
  if ((d->x_scale || d->x_shift) && !d->codes) return false;
  if (!d->ds != !d->scale) return false;
  return !d->ds || matrix_ok(d->w, d->ldw, d->K, 2);
}
}  // namespace

// the epilogues of a descriptor
template <int ACT, bool PRE = false> EpiForward<ACT, PRE> forward_epi(const cogaim_linear_fwd_desc* d) {
  return EpiForward<ACT, PRE>{d->bias, d->scale, d->residual, d->y, (signed char*)d->codes, (unsigned char*)d->exponents, PRE ? d->pre : nullptr,
                              d->ldr, d->ldy, d->M, d->N, d->residual_dtype, d->y_dtype, d->dtype};
}
static bool has_pre(const cogaim_linear_fwd_desc* d) { return d->extended == 1 && d->pre; }
template <int ACT> EpiInput<ACT> input_epi(const cogaim_linear_bwd_input_desc* d, const float* unit = nullptr) {
  return EpiInput<ACT>{(const signed char*)d->codes, (const unsigned char*)d->exponents, d->dx, d->a, d->lddx, d->lda, d->M,
                       d->K, d->dx_dtype, d->dtype, unit};
}

extern "C" {

long long cogaim_linear_fwd_workspace_bytes(const cogaim_linear_fwd_desc* d) {
  if (!forward_ok(d)) return COGAIM_EINVAL;
  if (few_rows(d->M, d->N, d->K, true)) return 0;
  const Shape s = shape_of(d->M, d->N, d->K, true, false, !forward_epi<ACT_NONE>(d).fast());
  return copy_bytes(side(d->x, d->ldx, d->M, d->K)) + copy_bytes(side(d->w, d->ldw, d->N, d->K)) +
         (joins(s, forward_epi<ACT_NONE>(d)) ? (long long)s.splits * d->M * round8(d->N) * 4 : 0);
}

}  // extern "C"

template <class T, int DT, int ACT, bool PRE> static int forward_as(const cogaim_linear_fwd_desc* d, void* workspace, hipStream_t st) {
  const EpiForward<ACT, PRE> e = forward_epi<ACT, PRE>(d);
  if (few_rows(d->M, d->N, d->K, true))
    return launch_few<T, DT, true>(Few{d->x, d->w, nullptr, d->ldx, d->ldw, d->M, d->N, d->K, 1}, e, st);
  const Shape s = shape_of(d->M, d->N, d->K, true, false, !e.fast());
  Side a = side(d->x, d->ldx, d->M, d->K), b = side(d->w, d->ldw, d->N, d->K);
  char* ws = (char*)workspace;
  const int rc = run_copies(a, b, d->dtype, ws, st);
  if (rc) return rc;
  return product<T, true, true>(operands(a, b, true, true, d->M, d->N, s), s, e, (float*)ws, st);
}
template <class T, int DT, int ACT> static int forward_act(const cogaim_linear_fwd_desc* d, void* workspace, hipStream_t st) {
  return has_pre(d) ? forward_as<T, DT, ACT, true>(d, workspace, st) : forward_as<T, DT, ACT, false>(d, workspace, st);
}
template <class T, int DT> static int forward_of(const cogaim_linear_fwd_desc* d, void* workspace, hipStream_t st) {
  if (d->activation == ACT_RELU) return forward_act<T, DT, ACT_RELU>(d, workspace, st);
  if (d->activation == ACT_GELU) return forward_act<T, DT, ACT_GELU>(d, workspace, st);
  return forward_act<T, DT, ACT_NONE>(d, workspace, st);
}

extern "C" {

int cogaim_linear_fwd(const cogaim_linear_fwd_desc* d, void* workspace, long long workspace_bytes, void* stream) {
  const long long need = cogaim_linear_fwd_workspace_bytes(d);
  if (need < 0 || (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))) return COGAIM_EINVAL;
  return d->dtype == DT_BF16 ? forward_of<__bf16, DT_BF16>(d, workspace, (hipStream_t)stream)
                             : forward_of<_Float16, DT_FP16>(d, workspace, (hipStream_t)stream);
}

static bool input_unit(const cogaim_linear_bwd_input_desc* d) { return d->scale && d->dtype == DT_FP16; }
static int input_parts(const cogaim_linear_bwd_input_desc* d) { return d->scale && d->dx_dtype == DT_FP32 ? parts_of(d->dtype) : 1; }
static Shape input_shape(const cogaim_linear_bwd_input_desc* d) {
  return shape_of(d->M, d->K, d->N, true, input_parts(d) > 1, !input_epi<ACT_NONE>(d).fast());
}

long long cogaim_linear_bwd_input_workspace_bytes(const cogaim_linear_bwd_input_desc* d) {
  if (!input_ok(d)) return COGAIM_EINVAL;
  if (few_rows(d->M, d->K, d->N, false)) return 0;
  const Shape s = input_shape(d);
  const int parts = input_parts(d);
  return (input_unit(d) ? 256 : 0) + copy_bytes(side(d->dy, d->lddy, d->M, d->N)) + copy_bytes(side(d->w, d->ldw, d->N, d->K, d->scale, parts)) +
         (parts > 1 || joins(s, input_epi<ACT_NONE>(d)) ? (long long)parts * s.splits * d->M * round8(d->K) * 4 : 0);
}

int cogaim_linear_bwd_input(const cogaim_linear_bwd_input_desc* d, void* workspace, long long workspace_bytes, void* stream) {
  const long long need = cogaim_linear_bwd_input_workspace_bytes(d);
  if (need < 0 || (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))) return COGAIM_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  if (few_rows(d->M, d->K, d->N, false)) {
    const Few f{d->dy, d->w, d->scale, d->lddy, d->ldw, d->M, d->K, d->N, input_parts(d)};
#define FEW_RUN(T_, DT_)                                                                      \
  (d->activation == ACT_RELU ? launch_few<T_, DT_, false>(f, input_epi<ACT_RELU>(d), st)       \
   : d->activation == ACT_GELU ? launch_few<T_, DT_, false>(f, input_epi<ACT_GELU>(d), st)     \
                               : launch_few<T_, DT_, false>(f, input_epi<ACT_NONE>(d), st))
    return d->dtype == DT_BF16 ? FEW_RUN(__bf16, DT_BF16) : FEW_RUN(_Float16, DT_FP16);
#undef FEW_RUN
  }
  const Shape s = input_shape(d);
  const int parts = input_parts(d);
  Side a = side(d->dy, d->lddy, d->M, d->N), b = side(d->w, d->ldw, d->N, d->K, d->scale, parts);
  char* ws = (char*)workspace;
  if (input_unit(d)) {
    b.unit = (float*)ws;
    ws += 256;
  }
  const float* const unit = b.unit;
  const int rc = run_copies(a, b, d->dtype, ws, st);
  if (rc) return rc;
  const Operands g = operands(a, b, true, false, d->M, d->K, s);
#define IN_RUN(T_)                                                                                                     \
  (d->activation == ACT_RELU ? product<T_, true, false>(g, s, input_epi<ACT_RELU>(d, unit), (float*)ws, st, parts)                         \
   : d->activation == ACT_GELU ? product<T_, true, false>(g, s, input_epi<ACT_GELU>(d, unit), (float*)ws, st, parts)                       \
                               : product<T_, true, false>(g, s, input_epi<ACT_NONE>(d, unit), (float*)ws, st, parts))
  return d->dtype == DT_BF16 ? IN_RUN(__bf16) : IN_RUN(_Float16);
}

// something to put on the finished sums, or a ragged result: the row-wise second kernel runs
static bool weight_has_more(const cogaim_linear_bwd_weight_desc* d) {
  return d->x_scale || d->x_shift || d->scale || (d->K & 7);
}
static bool weight_needs_finish(const cogaim_linear_bwd_weight_desc* d, const Shape& s) { return s.splits > 1 || weight_has_more(d); }

static bool weight_in_units(const cogaim_linear_bwd_weight_desc* d) { return d->codes && d->dtype == DT_FP16; }

long long cogaim_linear_bwd_weight_workspace_bytes(const cogaim_linear_bwd_weight_desc* d) {
  if (!weight_ok(d)) return COGAIM_EINVAL;
  const Shape s = shape_of(d->N, d->K, d->M, false, weight_has_more(d), false);
  const long long x = d->codes ? round256((long long)d->M * round8(d->K) * 2) : copy_bytes(side(d->x, d->ldx, d->M, d->K));
  const long long part = weight_needs_finish(d, s) ? round256((long long)s.splits * d->N * round8(d->K) * 4) + (long long)s.splits * d->N * 4 : 0;
  return copy_bytes(side(d->dy, d->lddy, d->M, d->N)) + x + part + (weight_in_units(d) ? round256(tops_bytes(d->M, d->K)) : 0);
}

int cogaim_linear_bwd_weight(const cogaim_linear_bwd_weight_desc* d, void* workspace, long long workspace_bytes, void* stream) {
  const long long need = cogaim_linear_bwd_weight_workspace_bytes(d);
  if (need < 0 || (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))) return COGAIM_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  const Shape s = shape_of(d->N, d->K, d->M, false, weight_has_more(d), false);
  char* ws = (char*)workspace;
  Side a = side(d->dy, d->lddy, d->M, d->N), b{};
  if (!d->codes) b = side(d->x, d->ldx, d->M, d->K);
  int rc = run_copies(a, b, d->dtype, ws, st);
  if (rc) return rc;
  unsigned char* tops = nullptr;
  if (d->codes) {
    // the 8-bit rows as 16-bit values in front of the product (a power-of-two step makes them exact in bf16, and in fp16
    // in units of their columns)
    const int k8 = round8(d->K);
    if (weight_in_units(d)) {
      tops = (unsigned char*)ws;
      ws += round256(tops_bytes(d->M, d->K));
      rc = unpack8_units(d->codes, d->exponents, tops, ws, d->M, d->K, k8, st);
    } else rc = cogaim_unpack8(d->codes, d->exponents, ws, d->dtype, k8, d->M, d->K, k8, stream);
    b = Side{ws, k8, d->M, k8, false, nullptr, nullptr, 1};
    ws += round256((long long)d->M * k8 * 2);
    if (rc) return rc;
  }
  Operands g = operands(a, b, false, false, d->N, d->K, s);
  if (!weight_needs_finish(d, s)) {
    g.col_sum = d->db;
    const EpiPlain e{d->dw, d->lddw, d->N, d->K, d->dw_dtype, tops};
    return d->dtype == DT_BF16 ? launch_gemm<__bf16, false, false>(g, s.tile, e, st) : launch_gemm<_Float16, false, false>(g, s.tile, e, st);
  }
  const int kp = round8(d->K);
  float* part = (float*)ws;
  float* sums = (float*)(ws + round256((long long)s.splits * d->N * kp * 4));
  g.col_sum = sums;
  const EpiPart e{part, d->N, kp};
  rc = d->dtype == DT_BF16 ? launch_gemm<__bf16, false, false>(g, s.tile, e, st) : launch_gemm<_Float16, false, false>(g, s.tile, e, st);
  if (rc) return rc;
  const WeightFinish f{part, sums, d->x_scale, d->x_shift, d->scale, (const unsigned short*)d->w, d->bias, d->dw, d->db, d->ds, tops, d->ldw, d->lddw,
                       d->N, d->K, kp, s.splits, d->dtype, d->dw_dtype};
  if (d->N >= 4 * 512) hipLaunchKernelGGL(weight_finish_kernel<4>, dim3((d->N + 3) / 4), dim3(256), 0, st, f);
  else hipLaunchKernelGGL(weight_finish_kernel<1>, dim3(d->N), dim3(256), 0, st, f);
  return COGAIM_LAUNCH_CHECK();
}

}  // extern "C"

// Row-wise kernels of the training path: LayerNorm forward (with row statistics and an 8-bit copy of the normalised
// rows), its backward pass with the reduction of the weight's and the bias's gradients, the 8-bit format on its own,
// and the elementwise helpers of the linear layers' backward.  All are bound by HBM.
#include "train_common.h"
#include "../../include/cogaim.h"

#include <type_traits>

namespace {
using namespace train;

// A row lives in the registers of TPR threads, NCH runs of V consecutive columns each (runs t, t + TPR, ...; 32 / V
// neighbouring threads hold a group of 32).  Rows may begin at any element: runs are moved with accesses of whatever
// alignment the row has (gfx950 takes them).
// EVEN: the width is a multiple of the run, and no run crosses a row's end.  Otherwise one does, by at most V - 1 elements:
// with V rows or more behind this one, these lie in the matrix too, so the run is loaded whole and the columns past the end
// are zeroed where they are used; only the last V rows' runs are loaded element by element.  (With a branch around every
// load they are no longer in flight together: fp32 43840 x 767 to bf16 and 8 bits 66 us, now 40, where 768 columns take 36;
// backward from 8 bits 52, now 41, against 35.)
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum_dpp(v);
  if constexpr (TPR > 64) {
    __syncthreads();                                        // the previous sum's readers are done
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) v += red[w];
  }
  return v;
}
template <int TPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  a = wave_sum_dpp(a); b = wave_sum_dpp(b);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = a; red[16 + (threadIdx.x >> 6)] = b; }
    __syncthreads();
    a = red[0]; b = red[16];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) { a += red[w]; b += red[16 + w]; }
  }
}

// Run `c .. c + V - 1` of a row of D elements that begins at element `row`, zeros past its end.  W words hold its bits.
template <int DT, int V> struct Run { static constexpr int W = DT == DT_FP32 ? V : V / 2; unsigned w[W]; };
template <int DT, int V, bool EVEN> __device__ __forceinline__ Run<DT, V> load_run(const void* p, long long row, int c, int D) {
  Run<DT, V> r;
  if constexpr (DT == DT_FP32) {
    const unsigned* q = reinterpret_cast<const unsigned*>(p) + row + c;
    if (EVEN || c + V <= D) __builtin_memcpy(r.w, q, sizeof(r.w));
    else {
#pragma unroll
      for (int j = 0; j < V; ++j) r.w[j] = c + j < D ? q[j] : 0u;
    }
  } else {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p) + row + c;
    if (EVEN || c + V <= D) __builtin_memcpy(r.w, q, sizeof(r.w));
    else {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) r.w[j] = (c + 2 * j < D ? (unsigned)q[2 * j] : 0u) | (c + 2 * j + 1 < D ? (unsigned)q[2 * j + 1] << 16 : 0u);
    }
  }
  return r;
}
template <int V> __device__ __forceinline__ void cvt_words(const unsigned* w, int dt, float (&v)[V]) {
  if (dt == DT_FP32) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __uint_as_float(w[j]);
  } else if (dt == DT_BF16) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) { v[2 * j] = half_bits((unsigned short)w[j]); v[2 * j + 1] = half_bits((unsigned short)(w[j] >> 16)); }
  }
}
template <int DT, int V> __device__ __forceinline__ void cvt_run(const Run<DT, V>& r, float (&v)[V]) { cvt_words<V>(r.w, DT, v); }
// the same of a type known at run time (uniform over the launch)
template <int V, bool EVEN> __device__ __forceinline__ Run<DT_FP32, V> load_any(const void* p, int dt, long long row, int c, int D) {
  if (dt == DT_FP32) return load_run<DT_FP32, V, EVEN>(p, row, c, D);
  const Run<DT_BF16, V> r = load_run<DT_BF16, V, EVEN>(p, row, c, D);
  Run<DT_FP32, V> o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.w[j] = j < V / 2 ? r.w[j] : 0u;
  return o;
}
// the first n < V elements of a run: of eight in pieces of four, two and one, of four one by one (the backward kernel has no
// registers for more: 43840 x 767 from fp32 74 against 72 us)
template <int V, class E> __device__ __forceinline__ void store_end(E* q, const E (&y)[V], int n) {
  if constexpr (V == 4) {
#pragma unroll
    for (int j = 0; j < V; ++j) if (j < n) q[j] = y[j];
    return;
  }
  E v[V];
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = y[j];
#pragma unroll
  for (int p = V / 2; p; p /= 2)
    if (n & p) {
      __builtin_memcpy(q, v, p * sizeof(E));
      q += p;
#pragma unroll
      for (int j = 0; j + p < V; ++j) v[j] = v[j + p];
    }
}
template <int V, bool EVEN> __device__ __forceinline__ void store_any(void* p, int dt, long long row, int c, int D, const float (&y)[V]) {
  if (dt == DT_FP32) {
    float* q = reinterpret_cast<float*>(p) + row + c;
    if (EVEN || c + V <= D) __builtin_memcpy(q, y, 4 * V);
    else store_end<V>(q, y, D - c);
  } else {
    unsigned short* q = reinterpret_cast<unsigned short*>(p) + row + c;
    unsigned short h[V];
    pack_half<V>(y, dt, h);
    if (EVEN || c + V <= D) __builtin_memcpy(q, h, 2 * V);
    else store_end<V>(q, h, D - c);
  }
}
// whether runs of row `row` may reach into the rows behind it (the same for the wave)
template <int V> __device__ __forceinline__ bool runs_whole(long long row, int M) { return __builtin_amdgcn_readfirstlane((int)(row + V <= M)); }
template <int V> __device__ __forceinline__ void end_row(float (&v)[V], int c, int D) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = c + j < D ? v[j] : 0.f;
}
template <int V> struct Codes { unsigned w[V / 4]; };
template <int V, bool EVEN> __device__ __forceinline__ Codes<V> load_codes(const signed char* row, int c, int D) {
  Codes<V> q;
  if (EVEN || c + V <= D) __builtin_memcpy(q.w, row + c, V);
  else {
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      q.w[h] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) if (c + 4 * h + j < D) q.w[h] |= (unsigned)(unsigned char)row[c + 4 * h + j] << (8 * j);
    }
  }
  return q;
}
template <int V> __device__ __forceinline__ void decode_run(const Codes<V>& q, float step, float (&v)[V]) {
#pragma unroll
  for (int h = 0; h < V / 4; ++h) decode4(q.w[h], step, v + 4 * h);
}
template <int V, bool EVEN> __device__ __forceinline__ void load_f32(const float* p, int c, int D, float (&v)[V]) {
  cvt_run<DT_FP32, V>(load_run<DT_FP32, V, EVEN>(p, 0, c, D), v);
}
// a run of an fp32 vector of D >= V elements without a branch around the load: the one that crosses the end is read from
// D - V, and moved into place by settle() where it is used
template <int V, bool EVEN> __device__ __forceinline__ Run<DT_FP32, V> load_vec(const float* p, int c, int D) {
  return load_run<DT_FP32, V, true>(p, 0, EVEN || c + V <= D ? c : D - V, D);
}
template <int V, bool EVEN> __device__ __forceinline__ void settle(Run<DT_FP32, V>& r, int c, int D) {
  const int by = c + V - D;
  if (EVEN || by <= 0) return;
#pragma unroll
  for (int p = V / 2; p; p /= 2)
#pragma unroll
    for (int j = 0; j < V; ++j) r.w[j] = by & p ? (j + p < V ? r.w[j + p < V ? j + p : j] : 0u) : r.w[j];
}
// codes and exponent byte of a thread's run; all threads of a group call this together, with zeros past the row's end
template <int V, bool EVEN> __device__ __forceinline__ void save_run(const float (&v)[V], signed char* codes, unsigned char* bytes, long long row, int D, int c) {
  unsigned m = top_bits<V>(v);
  m = umax(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1 /* quad_perm [1,0,3,2] */, 0xf, 0xf, true));
  m = umax(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E /* quad_perm [2,3,0,1] */, 0xf, 0xf, true));
  if constexpr (V == 4) m = umax(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x141 /* row_half_mirror */, 0xf, 0xf, true));
  if (c >= D) return;
  const unsigned byte = group_byte(m);
  Codes<V> q;
#pragma unroll
  for (int h = 0; h < V / 4; ++h) q.w[h] = pack4(v + 4 * h, byte);
  signed char* to = codes + row * D + c;
  if (EVEN || c + V <= D) __builtin_memcpy(to, q.w, V);
  else {
    signed char e[V];
    __builtin_memcpy(e, q.w, V);
    store_end<V>(to, e, D - c);
  }
  if ((c & (GROUP - 1)) == 0) bytes[row * groups_of(D) + c / GROUP] = (unsigned char)byte;
}

// Forward: mean and variance in two passes over registers.  HBM: 157 MB at 21920 x 1024 (fp32 -> bf16 and 8 bits) in 29 us,
// 5.4 TB/s.  Runs of eight: 16-byte stores of 16-bit rows (with runs of four the narrower stores cost 40 us).
struct LnFwd {
  const void* x; const float* gamma; const float* beta; void* y; float* mean; float* rstd;
  signed char* codes; unsigned char* bytes; long long ldx, ldy; int M, D, y_dt; float eps;
};

template <int XDT, int V, int TPR, int NCH, bool EVEN>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ln_train_fwd_kernel(LnFwd a) {
  __shared__ float red[32];
  const int t = threadIdx.x & (TPR - 1);
  constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
  if (RPB > 1 && row >= a.M) return;                        // whole waves: a row per wave
  // runs past the row's end are read from its beginning and zeroed: no branch, so all loads are in flight together
  const bool whole = EVEN || runs_whole<V>(row, a.M);
  Run<XDT, V> raw[NCH];
  Run<DT_FP32, V> g[NCH], b[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (t + TPR * i) * V;
    if (whole) raw[i] = load_run<XDT, V, true>(a.x, row * a.ldx, c < a.D ? c : 0, a.D);
    else raw[i] = load_run<XDT, V, false>(a.x, row * a.ldx, c < a.D ? c : 0, a.D);
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (t + TPR * i) * V;
    if (EVEN || a.D >= V) {
      g[i] = load_vec<V, EVEN>(a.gamma, c < a.D ? c : 0, a.D);
      b[i] = load_vec<V, EVEN>(a.beta, c < a.D ? c : 0, a.D);
    } else {
      g[i] = load_run<DT_FP32, V, false>(a.gamma, 0, c < a.D ? c : 0, a.D);
      b[i] = load_run<DT_FP32, V, false>(a.beta, 0, c < a.D ? c : 0, a.D);
    }
  }
  float v[NCH][V];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    cvt_run<XDT, V>(raw[i], v[i]);
    const int c = (t + TPR * i) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) { v[i][j] = (EVEN ? c : c + j) < a.D ? v[i][j] : 0.f; sum += v[i][j]; }
  }
  const float mean = row_sum<TPR>(sum, red) / (float)a.D;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (t + TPR * i) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[i][j] = (EVEN ? c : c + j) < a.D ? v[i][j] - mean : 0.f;
      sq = __builtin_fmaf(v[i][j], v[i][j], sq);
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<TPR>(sq, red) / (float)a.D + a.eps);
  if (t == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (t + TPR * i) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] *= rstd;
    if (a.codes) save_run<V, EVEN>(v[i], a.codes, a.bytes, row, a.D, c);
    if (c < a.D) {
      if (EVEN || a.D >= V) {
        settle<V, EVEN>(g[i], c, a.D);
        settle<V, EVEN>(b[i], c, a.D);
      }
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = __builtin_fmaf(v[i][j], __uint_as_float(g[i].w[j]), __uint_as_float(b[i].w[j]));
      store_any<V, EVEN>(a.y, a.y_dt, row * a.ldy, c, a.D, y);
    }
  }
}

// Backward.  With h = (x - mean) rstd and g = dy * gamma:  dx = rstd (g - mean(g) - h mean(g h)) [+ add],
// dgamma = sum over rows of dy h, dbeta = sum of dy.  A block walks rows blockIdx, blockIdx + gridDim, ... and keeps its
// threads' columns of dgamma / dbeta in registers; one partial row per block, summed in block order by the second
// kernel, so the result does not depend on timing (no atomics).  HBM: 471 MB at 43840 x 768 (fp32 stream, bf16 dy) in 90 us,
// 5.2 TB/s.  Runs of four: fp32 loads of whole lines; gamma in registers (read from the cache for every row: 105 us).  768
// blocks of four waves are what is resident at 150 to 170 registers (1024 would run in two uneven rounds: 101 us).
struct LnBwd {
  const void* dy; const void* x; const signed char* codes; const unsigned char* bytes; const float* mean; const float* rstd;
  const float* gamma; const void* add; void* dx; float* part; float* dgamma; float* dbeta;
  long long lddy, ldx, ldadd, lddx; int M, D, add_dt, dx_dt;
};

constexpr int SRC_CODES = 3;               // the rows come from their 8-bit copy
template <int DYT, int SRC, int V, int TPR, int NCH, bool EVEN>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, TPR == 64 && NCH <= 3 ? 3 : 1) void ln_train_bwd_kernel(LnBwd a) {
  constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
  constexpr int XDT = SRC == SRC_CODES ? DT_BF16 : SRC;
  __shared__ float red[32];
  __shared__ float acc[RPB > 1 ? RPB * TPR * NCH * V : 1];
  const int t = threadIdx.x & (TPR - 1), sub = threadIdx.x / TPR;
  float dg[NCH][V], db[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) { dg[i][j] = 0.f; db[i][j] = 0.f; }
  const long long groups = groups_of(a.D);
  struct Loads { Run<DYT, V> dy[NCH]; Run<XDT, V> x[NCH]; Codes<V> codes[NCH]; unsigned byte[NCH]; Run<DT_FP32, V> add[NCH]; float rstd, mean; };
  auto load_as = [&](auto whole, long long row, Loads& l) __attribute__((always_inline)) {
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (t + TPR * i) * V < a.D ? (t + TPR * i) * V : 0;     // no branch around the loads
      l.dy[i] = load_run<DYT, V, W>(a.dy, row * a.lddy, c, a.D);
      if constexpr (SRC == SRC_CODES) {
        l.codes[i] = load_codes<V, W>(a.codes + row * a.D, c, a.D);
        l.byte[i] = a.bytes[row * groups + c / GROUP];
      } else l.x[i] = load_run<XDT, V, W>(a.x, row * a.ldx, c, a.D);
      if (a.add) l.add[i] = load_any<V, W>(a.add, a.add_dt, row * a.ldadd, c, a.D);
    }
  };
  auto load = [&](long long row, Loads& l) __attribute__((always_inline)) {
    // 1024 threads have no registers for both forms (2000 x 12001: 178 against 160 us)
    if constexpr (EVEN) load_as(std::true_type{}, row, l);
    else if (TPR < 1024 && runs_whole<V>(row, a.M)) load_as(std::true_type{}, row, l);
    else load_as(std::false_type{}, row, l);
    l.rstd = a.rstd[row];
    l.mean = SRC == SRC_CODES ? 0.f : a.mean[row];
  };
  // while a row is worked on, the next one's loads are in flight (not where 1024 threads leave a wave 128 registers)
  constexpr bool AHEAD = TPR < 1024;
  const long long stride = (long long)gridDim.x * RPB;
  Loads next;
  long long row = (long long)blockIdx.x * RPB + sub;
  if constexpr (AHEAD) { if (row < a.M) load(row, next); }
  float gmr[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) load_f32<V, EVEN>(a.gamma, (t + TPR * i) * V < a.D ? (t + TPR * i) * V : 0, a.D, gmr[i]);
  for (; row < a.M; row += stride) {
    Loads now;
    if constexpr (AHEAD) {
      now = next;
      if (row + stride < a.M) load(row + stride, next);
    } else load(row, now);
    const float rstd = now.rstd, mean = now.mean;
    float g[NCH][V], h[NCH][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (t + TPR * i) * V;
      if (c < a.D) {
        float dy[V];
        cvt_run<DYT, V>(now.dy[i], dy);
        if constexpr (SRC == SRC_CODES) decode_run<V>(now.codes[i], group_step(now.byte[i]), h[i]);
        else {
          cvt_run<XDT, V>(now.x[i], h[i]);
#pragma unroll
          for (int j = 0; j < V; ++j) h[i][j] = (h[i][j] - mean) * rstd;
        }
        if constexpr (!EVEN && TPR < 1024) {
          end_row<V>(dy, c, a.D);
          end_row<V>(h[i], c, a.D);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dg[i][j] = __builtin_fmaf(dy[j], h[i][j], dg[i][j]);
          db[i][j] += dy[j];
          g[i][j] = dy[j] * gmr[i][j];
          s1 += g[i][j];
          s2 = __builtin_fmaf(g[i][j], h[i][j], s2);
        }
      }
    }
    row_sum2<TPR>(s1, s2, red);
    s1 /= (float)a.D; s2 /= (float)a.D;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (t + TPR * i) * V;
      if (c < a.D) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rstd * (g[i][j] - s1 - h[i][j] * s2);
        if (a.add) {
          float ad[V];
          cvt_words<V>(now.add[i].w, a.add_dt, ad);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += ad[j];
        }
        store_any<V, EVEN>(a.dx, a.dx_dt, row * a.lddx, c, a.D, o);
      }
    }
  }
  // the block's partial row: dgamma at part[block][0][.], dbeta at part[block][1][.]; a single block's is the result
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = gridDim.x == 1 ? (which ? a.dbeta : a.dgamma) : a.part + ((size_t)blockIdx.x * 2 + which) * a.D;
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[((sub * NCH + i) * V + j) * TPR + t] = which ? db[i][j] : dg[i][j];
      __syncthreads();
      // columns dealt to all threads; value (run, j) of thread run % TPR lies at run / TPR
      for (int c = threadIdx.x; c < a.D; c += RPB * TPR) {
        const int run = c / V, at = ((run / TPR) * V + c % V) * TPR + (run & (TPR - 1));
        float s = acc[at];
#pragma unroll
        for (int w = 1; w < RPB; ++w) s += acc[w * NCH * V * TPR + at];
        out[c] = s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (t + TPR * i) * V;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j < a.D) out[c + j] = which ? db[i][j] : dg[i][j];
      }
    }
  }
}

// sums the partial rows: 32 columns per block, 32 threads down the partials of each, joined in a fixed order
__global__ __launch_bounds__(1024) void ln_train_reduce_kernel(const float* __restrict__ part, float* __restrict__ dgamma,
                                                               float* __restrict__ dbeta, int nblk, int D) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + tx;
  float v = 0.f;
  if (c < 2LL * D) {
#pragma unroll 8
    for (int b = ty; b < nblk; b += 32) v += part[(size_t)b * 2 * D + c];
  }
  s[ty][tx] = v;
  __syncthreads();
  if (ty == 0 && c < 2LL * D) {
    float o = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) o += s[k][tx];
    if (c < D) dgamma[c] = o;
    else dbeta[c - D] = o;
  }
}

// A LayerScale vector times the power of two that brings its largest magnitude into [2^-5, 2^-4), where it is smaller, and
// what undoes it.  One block; a vector has a few thousand elements.
__global__ __launch_bounds__(256) void scale_unit_kernel(const float* __restrict__ scale, float* __restrict__ scaled, float* __restrict__ unit, int N) {
  __shared__ unsigned tops[4];
  const unsigned mine = wave_top(scale, N, threadIdx.x, 256);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = mine;
  __syncthreads();
  const unsigned e = umax(umax(tops[0], tops[1]), umax(tops[2], tops[3])) >> 23;           // 2^(e - 127) or more
  constexpr unsigned E = 122;                                                              // 2^-5
  const bool small = e != 0 && e < E;                                                      // not zeros alone (subnormals stay as they are)
  const float up = small ? __uint_as_float((127 + E - e) << 23) : 1.f;
  for (int i = threadIdx.x; i < N; i += 256) scaled[i] = scale[i] * up;
  if (threadIdx.x == 0) *unit = small ? __uint_as_float((127 + e - E) << 23) : 1.f;
}

// Walks the runs of a matrix, thread by thread with the grid's stride, without a division per step.
struct Walk {
  unsigned long long i, row; unsigned run, per_row, drow, drun;
  __device__ __forceinline__ explicit Walk(unsigned per_row_) : per_row(per_row_) {
    const unsigned stride = 256u * gridDim.x;
    i = blockIdx.x * 256ULL + threadIdx.x;
    row = i / per_row; run = (unsigned)(i - row * per_row);
    drow = stride / per_row; drun = stride - drow * per_row;
  }
  __device__ __forceinline__ void step() {
    i += 256ULL * gridDim.x;
    row += drow; run += drun;
    if (run >= per_row) { run -= per_row; ++row; }
  }
};

// The format on its own.  HBM: bf16 10960 x 4096 to 8 bits in 24 us (5.6 TB/s) and back in 21 us (6.4 TB/s).
// x [M, D] -> codes [M, D], bytes [M, groups].  32 / V neighbouring threads per group, a row's last group whole;
// runs of four of fp32, of eight of 16-bit elements: 16 bytes a thread.
template <int DT, int V, bool EVEN>
__global__ __launch_bounds__(256) void pack8_kernel(const void* __restrict__ x, long long ldx, signed char* __restrict__ codes,
                                                    unsigned char* __restrict__ bytes, int M, int D) {
  for (Walk w((unsigned)groups_of(D) * (GROUP / V)); w.row < (unsigned long long)M; w.step()) {     // a group's threads leave together
    const int c = (int)w.run * V;
    float v[V];
    if (c < D) {
      if (EVEN || w.row + V <= (unsigned long long)M) {
        cvt_run<DT, V>(load_run<DT, V, true>(x, (long long)w.row * ldx, c, D), v);
        if constexpr (!EVEN) end_row<V>(v, c, D);
      } else cvt_run<DT, V>(load_run<DT, V, false>(x, (long long)w.row * ldx, c, D), v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
    }
    save_run<V, EVEN>(v, codes, bytes, (long long)w.row, D, c);
  }
}

// Largest exponent byte of each column group over a part of the rows, 255 (not finite) left out: tops[part][group].  A block
// takes four groups, a thread every 1024th row of its part; the last four groups of a row are read together, not past its end.
__global__ __launch_bounds__(1024) void column_tops_kernel(const unsigned char* __restrict__ bytes, unsigned char* __restrict__ tops, int M, int G, int rows) {
  __shared__ unsigned char s[16][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g0 = G < 4 ? 0 : (int)(4 * blockIdx.x) < G - 4 ? (int)(4 * blockIdx.x) : G - 4, n = G < 4 ? G : 4;
  const long long first = (long long)blockIdx.y * rows, last = first + rows < M ? first + rows : M;
  unsigned top[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (long long r = first + threadIdx.x; r < last; r += 1024) {
    const unsigned char* p = bytes + r * G + g0;
    unsigned w = 0;
    if (n == 4) __builtin_memcpy(&w, p, 4);
    else {
      w = p[0];
      if (n > 1) w |= (unsigned)p[1] << 8;
      if (n > 2) w |= (unsigned)p[2] << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned b = w >> (8 * j) & 255u;
      top[j] = umax(top[j], b == 255u ? 0u : b);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int d = 32; d; d >>= 1) top[j] = umax(top[j], (unsigned)__shfl_xor((int)top[j], d));
    if (lane == 0) s[wave][j] = (unsigned char)top[j];
  }
  __syncthreads();
  if ((int)threadIdx.x < n) {
    unsigned t = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) t = umax(t, s[w][threadIdx.x]);
    tops[(size_t)blockIdx.y * G + g0 + threadIdx.x] = (unsigned char)t;
  }
}
// The unpacking kernel joins the parts itself, and its first block leaves the result in memory for the sums: with few rows a
// block joins the exponents of all of them in LDS and there is no other launch, with more a thread joins the eight parts
// of its run's group.  (One part of 16384 rows: 10960 x 1024 x 1024 55 us, 7 x 768 x 768 14.5.)
constexpr int UNITS_G = 2048, UNITS_BYTES = 4096, UNITS_PARTS = 8;       // groups and exponents that a block joins; parts
struct Units { const unsigned char* part; int parts; bool rows; unsigned char* tops; };      // rows: the parts are the rows' exponents
__device__ __forceinline__ unsigned joined_top(const Units& u, int G, int g) {
  unsigned t = 0;
#pragma unroll
  for (int p = 0; p < UNITS_PARTS; ++p) t = umax(t, u.part[(size_t)(p < u.parts ? p : u.parts - 1) * G + g]);
  return t;
}

// codes [M, D] -> out [M, width >= D] (columns past D are written as zero); UNITS: in units (fp16)
template <int DT, int V, bool EVEN, bool UNITS = false>
__global__ __launch_bounds__(256) void unpack8_kernel(const signed char* __restrict__ codes,
                                                      const unsigned char* __restrict__ bytes, void* __restrict__ out,
                                                      long long ldo, int M, int D, int width, Units units) {
  const long long groups = groups_of(D);
  __shared__ unsigned top[UNITS ? UNITS_G : 1];
  if constexpr (UNITS) {
    const int G = (int)groups;
    if (units.rows) {
      int wide = 1;                                             // lanes across the groups, a power of two
      while (wide < G && wide < 256) wide *= 2;
      for (int g = threadIdx.x; g < G; g += 256) top[g] = 0;
      __syncthreads();
      for (int g = threadIdx.x & (wide - 1); g < G; g += wide) {
        unsigned t = 0;
#pragma unroll 8
        for (int p = threadIdx.x / wide; p < units.parts; p += 256 / wide) {
          const unsigned b = units.part[(size_t)p * G + g];
          t = umax(t, b == 255u ? 0u : b);
        }
        atomicMax(&top[g], t);                                  // in LDS; a maximum has no order
      }
      __syncthreads();
      if (blockIdx.x == 0)
        for (int g = threadIdx.x; g < G; g += 256) units.tops[g] = (unsigned char)top[g];
    } else if (blockIdx.x == 0) {
      for (int g = threadIdx.x; g < G; g += 256) units.tops[g] = (unsigned char)joined_top(units, G, g);
    }
  }
  for (Walk w((unsigned)(width + V - 1) / V); w.row < (unsigned long long)M; w.step()) {
    const long long row = (long long)w.row;
    const int c = (int)w.run * V;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (c < D) {
      const Codes<V> q = EVEN || row + V <= M ? load_codes<V, true>(codes + row * D, c, D) : load_codes<V, false>(codes + row * D, c, D);
      float u[V];
      unsigned byte = bytes[row * groups + c / GROUP];
      if constexpr (UNITS) byte = unit_byte(byte, units.rows ? top[c / GROUP] : joined_top(units, (int)groups, c / GROUP));
      decode_run<V>(q, group_step(byte), u);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (DT == DT_FP16) u[j] = hold_fp16(u[j]);
        v[j] = c + j < D ? u[j] : 0.f;
      }
    }
    store_any<V, EVEN>(out, DT, row * ldo, c, width, v);
  }
}

// du = dy * act'(u), u from its 8-bit copy.  HBM: 226 MB of bf16 10960 x 4096 in 38 us, 6.0 TB/s; u itself, below, 270 MB in
// 42 us, 6.5 TB/s.
template <int DT, int V, bool EVEN>
__global__ __launch_bounds__(256) void act_bwd_kernel(const void* __restrict__ dy, long long lddy,
                                                      const signed char* __restrict__ codes,
                                                      const unsigned char* __restrict__ bytes, void* __restrict__ du,
                                                      int du_dt, long long lddu, int act, int M, int D) {
  const long long groups = groups_of(D);
  for (Walk w((unsigned)(D + V - 1) / V); w.row < (unsigned long long)M; w.step()) {
    const long long row = (long long)w.row;
    const int c = (int)w.run * V;
    Run<DT, V> r;
    Codes<V> q;
    if (EVEN || row + V <= M) {
      r = load_run<DT, V, true>(dy, row * lddy, c, D);
      q = load_codes<V, true>(codes + row * D, c, D);
    } else {
      r = load_run<DT, V, false>(dy, row * lddy, c, D);
      q = load_codes<V, false>(codes + row * D, c, D);
    }
    float u[V], g[V];
    decode_run<V>(q, group_step(bytes[row * groups + c / GROUP]), u);
    cvt_run<DT, V>(r, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float value, slope;
      if (act == ACT_GELU) gelu_both(u[j], value, slope);
      else slope = relu_slope(u[j]);
      g[j] *= slope;
    }
    store_any<V, EVEN>(du, du_dt, row * lddu, c, D, g);
  }
}

// the same with u itself, of a type known at run time; an infinite one (a pre-activation past fp16's range) has the slope's
// limit, 1 or 0
template <int DT, int V, bool EVEN>
__global__ __launch_bounds__(256) void act_bwd_from_kernel(const void* __restrict__ dy, long long lddy, const void* __restrict__ u, int u_dt, long long ldu,
                                                           void* __restrict__ du, int du_dt, long long lddu, int act, int M, int D) {
  for (Walk w((unsigned)(D + V - 1) / V); w.row < (unsigned long long)M; w.step()) {
    const long long row = (long long)w.row;
    const int c = (int)w.run * V;
    Run<DT, V> r;
    Run<DT_FP32, V> q;
    if (EVEN || row + V <= M) {
      r = load_run<DT, V, true>(dy, row * lddy, c, D);
      q = load_any<V, true>(u, u_dt, row * ldu, c, D);
    } else {
      r = load_run<DT, V, false>(dy, row * lddy, c, D);
      q = load_any<V, false>(u, u_dt, row * ldu, c, D);
    }
    float v[V], g[V];
    cvt_words<V>(q.w, u_dt, v);
    cvt_run<DT, V>(r, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float value, slope;
      if (act == ACT_GELU) gelu_both(fabsf(v[j]) == __builtin_inff() ? __builtin_copysignf(100.f, v[j]) : v[j], value, slope);
      else slope = relu_slope(v[j]);
      g[j] *= slope;
    }
    store_any<V, EVEN>(du, du_dt, row * lddu, c, D, g);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool dt_ok(int dt) { return dt >= 0 && dt <= 2; }
unsigned blocks_for(unsigned long long threads) {
  const unsigned long long b = (threads + 255) / 256;
  return (unsigned)(b > 256 * 32 ? 256 * 32 : b);
}
constexpr int LN_MAX_D = 16384;
constexpr int MAX_D = 1 << 30;             // column arithmetic in 32 bits
// blocks of the backward kernel: up to 4096 columns the 768 of four waves that are resident (12 waves a CU); wider rows take
// sixteen waves a block, in whole rounds of 256 units.  Each block leaves a partial row of 2 D floats.
int ln_bwd_blocks(int M, int D) {
  const int rpb = D <= 1024 ? 4 : 1, most = D <= 8192 ? 768 : 512;
  const long long want = ((long long)M + rpb - 1) / rpb;
  return (int)(want < most ? want : most);
}
// rows of the forward kernel that one launch takes: 64 threads to 1024 threads each
int ln_fwd_rows(int D) { return (int)(MAX_ITEMS / (D <= 1024 ? 64 : D <= 4096 ? 256 : 1024)) & ~255; }
template <int XDT> void run_ln_fwd(const LnFwd& a, hipStream_t st) {
  const int most = ln_fwd_rows(a.D);
  if (a.M > most) {                             // the rows in turn
    const size_t x = dt_size(XDT), y = dt_size(a.y_dt), g = groups_of(a.D);
    for (long long m = 0; m < a.M; m += most) {
      LnFwd p = a;
      p.M = (int)(a.M - m < most ? a.M - m : most);
      p.x = (const char*)a.x + m * a.ldx * x; p.y = (char*)a.y + m * a.ldy * y; p.mean += m; p.rstd += m;
      if (a.codes) { p.codes += m * a.D; p.bytes += m * g; }
      run_ln_fwd<XDT>(p, st);
    }
    return;
  }
#define LN_LAUNCH(V_, TPR_, NCH_, RPB_, TH_)                                                                              \
  do {                                                                                                                    \
    const dim3 grid((unsigned)(((long long)a.M + RPB_ - 1) / RPB_));                                                      \
    if (a.D % V_ == 0) hipLaunchKernelGGL((ln_train_fwd_kernel<XDT, V_, TPR_, NCH_, true>), grid, dim3(TH_), 0, st, a);   \
    else hipLaunchKernelGGL((ln_train_fwd_kernel<XDT, V_, TPR_, NCH_, false>), grid, dim3(TH_), 0, st, a);                \
  } while (0)
  if (a.D <= 512) LN_LAUNCH(8, 64, 1, 4, 256);
  else if (a.D <= 1024) LN_LAUNCH(8, 64, 2, 4, 256);
  else if (a.D <= 2048) LN_LAUNCH(8, 256, 1, 1, 256);
  else if (a.D <= 4096) LN_LAUNCH(8, 256, 2, 1, 256);
  else if (a.D <= 8192) LN_LAUNCH(8, 1024, 1, 1, 1024);
  else LN_LAUNCH(8, 1024, 2, 1, 1024);
#undef LN_LAUNCH
}
template <int DYT, int SRC> void run_ln_bwd(const LnBwd& a, int blocks, hipStream_t st) {
#define LN_LAUNCH(V_, TPR_, NCH_, RPB_, TH_)                                                                                         \
  do {                                                                                                                               \
    if (a.D % V_ == 0) hipLaunchKernelGGL((ln_train_bwd_kernel<DYT, SRC, V_, TPR_, NCH_, true>), dim3(blocks), dim3(TH_), 0, st, a); \
    else hipLaunchKernelGGL((ln_train_bwd_kernel<DYT, SRC, V_, TPR_, NCH_, false>), dim3(blocks), dim3(TH_), 0, st, a);              \
  } while (0)
  if (a.D <= 256) LN_LAUNCH(4, 64, 1, 4, 256);
  else if (a.D <= 512) LN_LAUNCH(4, 64, 2, 4, 256);
  else if (a.D <= 768) LN_LAUNCH(4, 64, 3, 4, 256);
  else if (a.D <= 1024) LN_LAUNCH(4, 64, 4, 4, 256);
  else if (a.D <= 2048) LN_LAUNCH(4, 256, 2, 1, 256);
  else if (a.D <= 4096) LN_LAUNCH(4, 256, 4, 1, 256);
  else if (a.D <= 8192) LN_LAUNCH(4, 1024, 2, 1, 1024);
  else LN_LAUNCH(4, 1024, 4, 1, 1024);
#undef LN_LAUNCH
}
template <int DYT> void run_ln_bwd_from(const LnBwd& a, int x_dt, int blocks, hipStream_t st) {
  if (a.codes) run_ln_bwd<DYT, SRC_CODES>(a, blocks, st);
  else if (x_dt == DT_BF16) run_ln_bwd<DYT, DT_BF16>(a, blocks, st);
  else if (x_dt == DT_FP16) run_ln_bwd<DYT, DT_FP16>(a, blocks, st);
  else run_ln_bwd<DYT, DT_FP32>(a, blocks, st);
}
}  // namespace

// KERNEL<type, columns a thread> launched for a run-time type
#define BY_TYPE(DT_, D_, KERNEL_, ...)                                                                                          \
  do {                                                                                                                          \
    if ((DT_) == DT_FP32) BY_EVEN(DT_FP32, 4, D_, KERNEL_, __VA_ARGS__);                                                        \
    else if ((DT_) == DT_BF16) BY_EVEN(DT_BF16, 8, D_, KERNEL_, __VA_ARGS__);                                                   \
    else BY_EVEN(DT_FP16, 8, D_, KERNEL_, __VA_ARGS__);                                                                         \
  } while (0)
#define BY_EVEN(DT_, V_, D_, KERNEL_, ...)                                                                                      \
  do {                                                                                                                          \
    if ((D_) % V_ == 0) hipLaunchKernelGGL((KERNEL_<DT_, V_, true>), __VA_ARGS__);                                              \
    else hipLaunchKernelGGL((KERNEL_<DT_, V_, false>), __VA_ARGS__);                                                            \
  } while (0)

namespace train {
long long tops_bytes(int, int D) { return (UNITS_PARTS + 1LL) * groups_of(D); }

int unpack8_units(const void* codes, const void* exponents, unsigned char* tops, void* out, int M, int D, int width, hipStream_t st) {
  const int G = (int)groups_of(D);
  Units u{(const unsigned char*)exponents, M, true, tops};
  if (G > UNITS_G || (long long)M * G > UNITS_BYTES) {
    const int rows = (int)((M + UNITS_PARTS - 1LL) / UNITS_PARTS);
    u = Units{tops + G, (int)((M + rows - 1LL) / rows), false, tops};
    hipLaunchKernelGGL(column_tops_kernel, dim3((G + 3) / 4, u.parts), dim3(1024), 0, st, (const unsigned char*)exponents, tops + G, M, G, rows);
  }
  const dim3 grid(blocks_for((unsigned long long)M * (width / 8LL + 1)));
  if ((D | width) % 8 == 0) hipLaunchKernelGGL((unpack8_kernel<DT_FP16, 8, true, true>), grid, dim3(256), 0, st, (const signed char*)codes, (const unsigned char*)exponents, out, (long long)width, M, D, width, u);
  else hipLaunchKernelGGL((unpack8_kernel<DT_FP16, 8, false, true>), grid, dim3(256), 0, st, (const signed char*)codes, (const unsigned char*)exponents, out, (long long)width, M, D, width, u);
  return COGAIM_LAUNCH_CHECK();
}
}  // namespace train

extern "C" {

int cogaim_layernorm_train_fwd(const void* x, int x_dtype, long long ldx, const float* gamma, const float* beta, void* y,
                               int y_dtype, long long ldy, float* mean, float* rstd, void* codes, void* exponents, int M,
                               int D, float eps, void* stream) {
  if (M <= 0 || D <= 0 || D > LN_MAX_D || !dt_ok(x_dtype) || !dt_ok(y_dtype) || ldx < D || ldy < D || !x || !gamma ||
      !beta || !y || !mean || !rstd || !codes != !exponents || !(eps >= 0.f) || !aligned(x, dt_size(x_dtype)) ||
      !aligned(y, dt_size(y_dtype)))
    return COGAIM_EINVAL;
  const LnFwd a{x, gamma, beta, y, mean, rstd, (signed char*)codes, (unsigned char*)exponents, ldx, ldy, M, D, y_dtype, eps};
  if (x_dtype == DT_BF16) run_ln_fwd<DT_BF16>(a, (hipStream_t)stream);
  else if (x_dtype == DT_FP16) run_ln_fwd<DT_FP16>(a, (hipStream_t)stream);
  else run_ln_fwd<DT_FP32>(a, (hipStream_t)stream);
  return COGAIM_LAUNCH_CHECK();
}

long long cogaim_layernorm_bwd_workspace_bytes(int M, int D) {
  if (M <= 0 || D <= 0 || D > LN_MAX_D) return COGAIM_EINVAL;
  return (long long)ln_bwd_blocks(M, D) * 2 * D * 4;                    // partial rows
}

int cogaim_layernorm_bwd(const void* dy, int dy_dtype, long long lddy, const void* x, int x_dtype, long long ldx,
                         const void* codes, const void* exponents, const float* mean, const float* rstd,
                         const float* gamma, const void* add, int add_dtype, long long ldadd, void* dx, int dx_dtype,
                         long long lddx, float* dgamma, float* dbeta, int M, int D, void* workspace,
                         long long workspace_bytes, void* stream) {
  if (M <= 0 || D <= 0 || D > LN_MAX_D || !dt_ok(dy_dtype) || !dt_ok(dx_dtype) || lddy < D || lddx < D || !dy || !rstd ||
      !gamma || !dx || !dgamma || !dbeta || !workspace || !codes != !exponents || !x == !codes)
    return COGAIM_EINVAL;
  if (x && (!mean || !dt_ok(x_dtype) || ldx < D || !aligned(x, dt_size(x_dtype)))) return COGAIM_EINVAL;
  if (add && (!dt_ok(add_dtype) || ldadd < D || !aligned(add, dt_size(add_dtype)))) return COGAIM_EINVAL;
  if (!aligned(dy, dt_size(dy_dtype)) || !aligned(dx, dt_size(dx_dtype)) || !aligned(workspace, 4) ||
      workspace_bytes < cogaim_layernorm_bwd_workspace_bytes(M, D))
    return COGAIM_EINVAL;
  const LnBwd a{dy, x, (const signed char*)codes, (const unsigned char*)exponents, mean, rstd, gamma, add, dx,
                (float*)workspace, dgamma, dbeta, lddy, ldx, ldadd, lddx, M, D, add_dtype, dx_dtype};
  const int nblk = ln_bwd_blocks(M, D);
  if (dy_dtype == DT_BF16) run_ln_bwd_from<DT_BF16>(a, x_dtype, nblk, (hipStream_t)stream);
  else if (dy_dtype == DT_FP16) run_ln_bwd_from<DT_FP16>(a, x_dtype, nblk, (hipStream_t)stream);
  else run_ln_bwd_from<DT_FP32>(a, x_dtype, nblk, (hipStream_t)stream);
  if (nblk > 1) hipLaunchKernelGGL(ln_train_reduce_kernel, dim3((2 * D + 31) / 32), dim3(1024), 0, (hipStream_t)stream,
                     (const float*)workspace, dgamma, dbeta, nblk, D);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_scale_unit(const float* scale, float* scaled, float* unit, int N, void* stream) {
  if (!scale || !scaled || !unit || N <= 0) return COGAIM_EINVAL;
  hipLaunchKernelGGL(scale_unit_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, scale, scaled, unit, N);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_pack8(const void* x, int x_dtype, long long ldx, void* codes, void* exponents, int M, int D, void* stream) {
  if (M <= 0 || D <= 0 || D > MAX_D || !dt_ok(x_dtype) || ldx < D || !x || !codes || !exponents || !aligned(x, dt_size(x_dtype)))
    return COGAIM_EINVAL;
  BY_TYPE(x_dtype, D, pack8_kernel, dim3(blocks_for((unsigned long long)M * groups_of(D) * (x_dtype == DT_FP32 ? 8 : 4))), dim3(256), 0, (hipStream_t)stream, x, ldx,
          (signed char*)codes, (unsigned char*)exponents, M, D);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_unpack8(const void* codes, const void* exponents, void* out, int out_dtype, long long ldo, int M, int D, int width,
                   void* stream) {
  if (M <= 0 || D <= 0 || D > MAX_D || width < D || width > MAX_D || !dt_ok(out_dtype) || ldo < width || !codes || !exponents || !out ||
      !aligned(out, dt_size(out_dtype)))
    return COGAIM_EINVAL;
  BY_TYPE(out_dtype, (D | width), unpack8_kernel, dim3(blocks_for((unsigned long long)M * (width / (out_dtype == DT_FP32 ? 4LL : 8LL) + 1))), dim3(256), 0, (hipStream_t)stream,
          (const signed char*)codes, (const unsigned char*)exponents, out, ldo, M, D, width, Units{});
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_activation_bwd(const void* dy, int dy_dtype, long long lddy, const void* codes, const void* exponents, void* du,
                          int du_dtype, long long lddu, int activation, int M, int D, void* stream) {
  if (M <= 0 || D <= 0 || D > MAX_D || !dt_ok(dy_dtype) || !dt_ok(du_dtype) || lddy < D || lddu < D || !dy || !codes || !exponents ||
      !du || (activation != ACT_RELU && activation != ACT_GELU) || !aligned(dy, dt_size(dy_dtype)) ||
      !aligned(du, dt_size(du_dtype)))
    return COGAIM_EINVAL;
  BY_TYPE(dy_dtype, D, act_bwd_kernel, dim3(blocks_for((unsigned long long)M * (D / (dy_dtype == DT_FP32 ? 4LL : 8LL) + 1))), dim3(256), 0, (hipStream_t)stream, dy, lddy,
          (const signed char*)codes, (const unsigned char*)exponents, du, du_dtype, lddu, activation, M, D);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_activation_bwd_from(const void* dy, int dy_dtype, long long lddy, const void* u, int u_dtype, long long ldu, void* du,
                               int du_dtype, long long lddu, int activation, int M, int D, void* stream) {
  if (M <= 0 || D <= 0 || D > MAX_D || !dt_ok(dy_dtype) || !dt_ok(u_dtype) || !dt_ok(du_dtype) || lddy < D || ldu < D || lddu < D || !dy || !u || !du ||
      (activation != ACT_RELU && activation != ACT_GELU) || !aligned(dy, dt_size(dy_dtype)) || !aligned(u, dt_size(u_dtype)) ||
      !aligned(du, dt_size(du_dtype)))
    return COGAIM_EINVAL;
  BY_TYPE(dy_dtype, D, act_bwd_from_kernel, dim3(blocks_for((unsigned long long)M * (D / (dy_dtype == DT_FP32 ? 4LL : 8LL) + 1))), dim3(256), 0, (hipStream_t)stream,
          dy, lddy, u, u_dtype, ldu, du, du_dtype, lddu, activation, M, D);
  return COGAIM_LAUNCH_CHECK();
}

}  // extern "C"

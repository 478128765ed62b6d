// Row-wise kernels of the training path: LayerNorm forward (with row statistics and an 8-bit copy of the normalised
// rows), its backward pass with the reduction of the weight's and the bias's gradients, the 8-bit format on its own,
// and the elementwise helpers of the linear layers' backward.  All are bound by HBM.
#include "train_common.h"
#include "../../include/cogaim.h"

namespace {
using namespace train;

// A row lives in the registers of TPR threads.  V = 8: a thread owns runs of eight consecutive columns (16-byte
// accesses; four neighbouring threads hold a group of 32); V = 1: single columns, neighbouring threads neighbouring
// columns, for widths or strides that 16-byte accesses cannot serve.  NCH = runs per thread.
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
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
  a = wave_sum(a); b = wave_sum(b);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = a; red[16 + (threadIdx.x >> 6)] = b; }
    __syncthreads();
    a = red[0]; b = red[16];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) { a += red[w]; b += red[16 + w]; }
  }
}

template <int V> struct Raw { Raw8 r; };
template <> struct Raw<1> { unsigned r; };
template <int V> __device__ __forceinline__ Raw<V> load_run(const void* p, int dt, size_t off) {
  Raw<V> o;
  if constexpr (V == 8) o.r = load_raw8(p, dt, off);
  else o.r = dt == DT_FP32 ? reinterpret_cast<const unsigned*>(p)[off] : reinterpret_cast<const unsigned short*>(p)[off];
  return o;
}
template <int V> __device__ __forceinline__ void cvt_run(const Raw<V>& o, int dt, float (&v)[V]) {
  if constexpr (V == 8) cvt_raw8(o.r, dt, v);
  else v[0] = dt == DT_FP16 ? half_bits((unsigned short)o.r) : __uint_as_float(dt == DT_FP32 ? o.r : o.r << 16);
}
template <int V> __device__ __forceinline__ void store_run(void* p, int dt, size_t off, const float (&y)[V]) {
  if constexpr (V == 8) store_vec8(p, dt, off, y);
  else store_one(p, dt, off, y[0]);
}
template <int V> __device__ __forceinline__ void load_f32(const float* p, int off, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = p[off + j];
}
// largest magnitude over a group of 32 columns: 32 / V neighbouring threads
template <int V> __device__ __forceinline__ unsigned group_max(unsigned m) {
#pragma unroll
  for (int o = 1; o < 32 / V; o <<= 1) m = umax(m, (unsigned)__shfl_xor((int)m, o, 64));
  return m;
}
// codes and exponent byte of a thread's run (every thread of the wave calls this; `in` = the run lies in the row)
template <int V> __device__ __forceinline__ void save_run(const float (&v)[V], bool in, signed char* codes, unsigned char* bytes,
                                                          long long row, int D, int col) {
  unsigned m;
  if constexpr (V == 8) m = top_bits8(v);
  else m = mag_bits(v[0]);
  m = group_max<V>(in ? m : 0u);
  if (!in) return;
  const unsigned byte = group_byte(m);
  if constexpr (V == 8) *reinterpret_cast<u32x2*>(codes + row * D + col) = pack_codes(v, byte);
  else codes[row * D + col] = (signed char)code_of(v[0], byte);
  if ((col & (GROUP - 1)) == 0) bytes[row * groups_of(D) + col / GROUP] = (unsigned char)byte;
}

struct LnFwd {
  const void* x; const float* gamma; const float* beta; void* y; float* mean; float* rstd;
  signed char* codes; unsigned char* bytes; long long ldx, ldy; int M, D, x_dt, y_dt; float eps;
};

template <int V, int TPR, int NCH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ln_train_fwd_kernel(LnFwd a) {
  __shared__ float red[32];
  const int t = threadIdx.x & (TPR - 1);
  constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
  if (RPB > 1 && row >= a.M) return;                        // whole waves: a row per wave
  Raw<V> raw[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (t + TPR * i) * V;
    if (c < a.D) raw[i] = load_run<V>(a.x, a.x_dt, row * a.ldx + c);
  }
  float v[NCH][V];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const bool in = (t + TPR * i) * V < a.D;
    if (in) cvt_run<V>(raw[i], a.x_dt, v[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) { v[i][j] = in ? v[i][j] : 0.f; sum += v[i][j]; }
  }
  const float mean = row_sum<TPR>(sum, red) / (float)a.D;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const bool in = (t + TPR * i) * V < a.D;
#pragma unroll
    for (int j = 0; j < V; ++j) { v[i][j] = in ? v[i][j] - mean : 0.f; sq += v[i][j] * v[i][j]; }
  }
  const float rstd = 1.f / sqrtf(row_sum<TPR>(sq, red) / (float)a.D + a.eps);
  if (t == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (t + TPR * i) * V;
    const bool in = c < a.D;
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] *= rstd;
    if (a.codes) save_run<V>(v[i], in, a.codes, a.bytes, row, a.D, c);
    if (in) {
      float g[V], b[V], y[V];
      load_f32<V>(a.gamma, c, g); load_f32<V>(a.beta, c, b);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = __builtin_fmaf(v[i][j], g[j], b[j]);
      store_run<V>(a.y, a.y_dt, row * a.ldy + c, y);
    }
  }
}

// Backward.  With h = (x - mean) rstd and g = dy * gamma:  dx = rstd (g - mean(g) - h mean(g h)) [+ add],
// dgamma = sum over rows of dy h, dbeta = sum of dy.  A block walks rows blockIdx, blockIdx + gridDim, ... and keeps its
// threads' columns of dgamma / dbeta in registers; one partial row per block, summed in block order by the second
// kernel, so the result does not depend on timing (no atomics).
struct LnBwd {
  const void* dy; const void* x; const signed char* codes; const unsigned char* bytes; const float* mean; const float* rstd;
  const float* gamma; const void* add; void* dx; float* part;
  long long lddy, ldx, ldadd, lddx; int M, D, dy_dt, x_dt, add_dt, dx_dt;
};

template <int V, int TPR, int NCH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void ln_train_bwd_kernel(LnBwd a) {
  constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
  __shared__ float red[32];
  __shared__ float acc[RPB > 1 ? RPB * TPR * NCH * V : 1];
  const int t = threadIdx.x & (TPR - 1), sub = threadIdx.x / TPR;
  float dg[NCH][V], db[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) { dg[i][j] = 0.f; db[i][j] = 0.f; }
  const long long groups = groups_of(a.D);
  for (long long row = (long long)blockIdx.x * RPB + sub; row < a.M; row += (long long)gridDim.x * RPB) {
    Raw<V> rdy[NCH], rx[NCH];
    u32x2 rc[NCH];
    unsigned rb[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (t + TPR * i) * V;
      if (c < a.D) {
        rdy[i] = load_run<V>(a.dy, a.dy_dt, row * a.lddy + c);
        if (a.codes) {
          if constexpr (V == 8) rc[i] = *reinterpret_cast<const u32x2*>(a.codes + row * a.D + c);
          else rc[i][0] = (unsigned char)a.codes[row * a.D + c];
          rb[i] = a.bytes[row * groups + c / GROUP];
        } else rx[i] = load_run<V>(a.x, a.x_dt, row * a.ldx + c);
      }
    }
    const float rstd = a.rstd[row], mean = a.codes ? 0.f : a.mean[row];
    float g[NCH][V], h[NCH][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (t + TPR * i) * V;
      const bool in = c < a.D;
      if (in) {
        float dy[V], gm[V];
        cvt_run<V>(rdy[i], a.dy_dt, dy);
        if (a.codes) {
          const float step = group_step(rb[i]);
          if constexpr (V == 8) decode8(rc[i], step, h[i]);
          else h[i][0] = (float)(signed char)rc[i][0] * step;
        } else {
          cvt_run<V>(rx[i], a.x_dt, h[i]);
#pragma unroll
          for (int j = 0; j < V; ++j) h[i][j] = (h[i][j] - mean) * rstd;
        }
        load_f32<V>(a.gamma, c, gm);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dg[i][j] = __builtin_fmaf(dy[j], h[i][j], dg[i][j]);
          db[i][j] += dy[j];
          g[i][j] = dy[j] * gm[j];
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
          const Raw<V> ra = load_run<V>(a.add, a.add_dt, row * a.ldadd + c);
          float ad[V];
          cvt_run<V>(ra, a.add_dt, ad);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += ad[j];
        }
        store_run<V>(a.dx, a.dx_dt, row * a.lddx + c, o);
      }
    }
  }
  // the block's partial row: dgamma at part[block][0][.], dbeta at part[block][1][.]
  float* out = a.part + (size_t)blockIdx.x * 2 * a.D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[((sub * NCH + i) * V + j) * TPR + t] = which ? db[i][j] : dg[i][j];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (t + TPR * i) * V;
        if (c < a.D && sub == (i & (RPB - 1))) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float s = acc[(i * V + j) * TPR + t];
#pragma unroll
            for (int w = 1; w < RPB; ++w) s += acc[((w * NCH + i) * V + j) * TPR + t];
            out[which * a.D + c + j] = s;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (t + TPR * i) * V;
        if (c < a.D)
#pragma unroll
          for (int j = 0; j < V; ++j) out[which * a.D + c + j] = which ? db[i][j] : dg[i][j];
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

// x [M, D] -> codes [M, D], bytes [M, groups].  32 / V neighbouring threads per group.
template <int V>
__global__ __launch_bounds__(256) void pack8_kernel(const void* __restrict__ x, int dt, long long ldx,
                                                    signed char* __restrict__ codes, unsigned char* __restrict__ bytes,
                                                    int M, int D) {
  const unsigned per_row = (unsigned)groups_of(D) * (GROUP / V);
  const unsigned long long total = (unsigned long long)M * per_row;
  // rounded up to whole waves: every lane of a wave takes part in its group's maximum
  const unsigned long long rounded = (total + 63) / 64 * 64;
  for (Walk w(per_row); w.i < rounded; w.step()) {
    const unsigned long long row = w.row;
    const int c = (int)w.run * V;
    const bool in = w.i < total && c < D;
    float v[V];
    if (in) {
      const Raw<V> r = load_run<V>(x, dt, row * ldx + c);
      cvt_run<V>(r, dt, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
    }
    save_run<V>(v, in, codes, bytes, (long long)row, D, c);
  }
}

// codes [M, D] -> out [M, width >= D] (columns past D are written as zero)
template <int V>
__global__ __launch_bounds__(256) void unpack8_kernel(const signed char* __restrict__ codes,
                                                      const unsigned char* __restrict__ bytes, void* __restrict__ out,
                                                      int dt, long long ldo, int M, int D, int width) {
  const unsigned per_row = (unsigned)(width + V - 1) / V;
  const unsigned long long total = (unsigned long long)M * per_row;
  const long long groups = groups_of(D);
  for (Walk w(per_row); w.i < total; w.step()) {
    const unsigned long long row = w.row;
    const int c = (int)w.run * V;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (c < D) {
      const float step = group_step(bytes[row * groups + c / GROUP]);
      if constexpr (V == 8) decode8(*reinterpret_cast<const u32x2*>(codes + row * D + c), step, v);
      else v[0] = (float)codes[row * D + c] * step;
      if (dt == DT_FP16) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = hold_fp16(v[j]);
      }
    }
    store_run<V>(out, dt, row * ldo + c, v);
  }
}

// du = dy * act'(u), u from its 8-bit copy
template <int V>
__global__ __launch_bounds__(256) void act_bwd_kernel(const void* __restrict__ dy, int dy_dt, long long lddy,
                                                      const signed char* __restrict__ codes,
                                                      const unsigned char* __restrict__ bytes, void* __restrict__ du,
                                                      int du_dt, long long lddu, int act, int M, int D) {
  const unsigned per_row = (unsigned)(D + V - 1) / V;
  const unsigned long long total = (unsigned long long)M * per_row;
  const long long groups = groups_of(D);
  for (Walk w(per_row); w.i < total; w.step()) {
    const unsigned long long row = w.row;
    const int c = (int)w.run * V;
    const Raw<V> r = load_run<V>(dy, dy_dt, row * lddy + c);
    const float step = group_step(bytes[row * groups + c / GROUP]);
    float u[V], g[V];
    if constexpr (V == 8) decode8(*reinterpret_cast<const u32x2*>(codes + row * D + c), step, u);
    else u[0] = (float)codes[row * D + c] * step;
    cvt_run<V>(r, dy_dt, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float value, slope;
      if (act == ACT_GELU) gelu_both(u[j], value, slope);
      else slope = relu_slope(u[j]);
      g[j] *= slope;
    }
    store_run<V>(du, du_dt, row * lddu + c, g);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool dt_ok(int dt) { return dt >= 0 && dt <= 2; }
// may eight elements at a time be moved with 16-byte accesses?
bool vec_rows(const void* p, long long ld) { return aligned(p, 16) && (ld & 7) == 0; }
unsigned blocks_for(unsigned long long threads) {
  const unsigned long long b = (threads + 255) / 256;
  return (unsigned)(b > 256 * 32 ? 256 * 32 : b);
}
constexpr int LN_MAX_D = 16384;
// blocks of the backward kernel: 16 waves a CU keep enough rows in flight; each leaves a partial row of 2 D floats
int ln_bwd_blocks(int M, int D, bool vec) {
  const int rpb = (vec ? D <= 2048 : D <= 1024) ? 4 : 1;
  const long long want = ((long long)M + rpb - 1) / rpb;
  return (int)(want < 1024 ? want : 1024);
}
}  // namespace

#define LN_BY_WIDTH(KERNEL, LAUNCH)                                                                     \
  if (vec) {                                                                                            \
    if (D <= 512) LAUNCH((KERNEL<8, 64, 1>), 4, 256)                                                    \
    else if (D <= 1024) LAUNCH((KERNEL<8, 64, 2>), 4, 256)                                              \
    else if (D <= 2048) LAUNCH((KERNEL<8, 64, 4>), 4, 256)                                              \
    else if (D <= 4096) LAUNCH((KERNEL<8, 256, 2>), 1, 256)                                             \
    else if (D <= 8192) LAUNCH((KERNEL<8, 256, 4>), 1, 256)                                             \
    else LAUNCH((KERNEL<8, 1024, 2>), 1, 1024)                                                          \
  } else {                                                                                              \
    if (D <= 256) LAUNCH((KERNEL<1, 64, 4>), 4, 256)                                                    \
    else if (D <= 1024) LAUNCH((KERNEL<1, 64, 16>), 4, 256)                                             \
    else if (D <= 4096) LAUNCH((KERNEL<1, 256, 16>), 1, 256)                                            \
    else LAUNCH((KERNEL<1, 1024, 16>), 1, 1024)                                                         \
  }

extern "C" {

int cogaim_layernorm_train_fwd(const void* x, int x_dtype, long long ldx, const float* gamma, const float* beta, void* y,
                               int y_dtype, long long ldy, float* mean, float* rstd, void* codes, void* exponents, int M,
                               int D, float eps, void* stream) {
  if (M <= 0 || D <= 0 || D > LN_MAX_D || !dt_ok(x_dtype) || !dt_ok(y_dtype) || ldx < D || ldy < D || !x || !gamma ||
      !beta || !y || !mean || !rstd || !codes != !exponents || !(eps >= 0.f) || !aligned(x, dt_size(x_dtype)) ||
      !aligned(y, dt_size(y_dtype)))
    return COGAIM_EINVAL;
  const bool vec = (D & 7) == 0 && vec_rows(x, ldx) && vec_rows(y, ldy) && aligned(codes, 8);
  const LnFwd a{x, gamma, beta, y, mean, rstd, (signed char*)codes, (unsigned char*)exponents, ldx, ldy, M, D, x_dtype, y_dtype, eps};
#define LN_LAUNCH(K_, RPB_, TH_) hipLaunchKernelGGL(K_, dim3((unsigned)(((long long)M + RPB_ - 1) / RPB_)), dim3(TH_), 0, (hipStream_t)stream, a);
  LN_BY_WIDTH(ln_train_fwd_kernel, LN_LAUNCH)
#undef LN_LAUNCH
  return COGAIM_LAUNCH_CHECK();
}

long long cogaim_layernorm_bwd_workspace_bytes(int M, int D) {
  if (M <= 0 || D <= 0 || D > LN_MAX_D) return COGAIM_EINVAL;
  return (long long)1024 * 2 * D * 4 < (long long)M * 2 * D * 4 ? (long long)1024 * 2 * D * 4 : (long long)M * 2 * D * 4;
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
  const bool vec = (D & 7) == 0 && vec_rows(dy, lddy) && vec_rows(dx, lddx) && (x ? vec_rows(x, ldx) : aligned(codes, 8)) &&
                   (!add || vec_rows(add, ldadd));
  const LnBwd a{dy, x, (const signed char*)codes, (const unsigned char*)exponents, mean, rstd, gamma, add, dx,
                (float*)workspace, lddy, ldx, ldadd, lddx, M, D, dy_dtype, x_dtype, add_dtype, dx_dtype};
  const int nblk = ln_bwd_blocks(M, D, vec);
#define LN_LAUNCH(K_, RPB_, TH_) hipLaunchKernelGGL(K_, dim3(nblk), dim3(TH_), 0, (hipStream_t)stream, a);
  LN_BY_WIDTH(ln_train_bwd_kernel, LN_LAUNCH)
#undef LN_LAUNCH
  hipLaunchKernelGGL(ln_train_reduce_kernel, dim3((2 * D + 31) / 32), dim3(1024), 0, (hipStream_t)stream,
                     (const float*)workspace, dgamma, dbeta, nblk, D);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_pack8(const void* x, int x_dtype, long long ldx, void* codes, void* exponents, int M, int D, void* stream) {
  if (M <= 0 || D <= 0 || !dt_ok(x_dtype) || ldx < D || !x || !codes || !exponents || !aligned(x, dt_size(x_dtype)))
    return COGAIM_EINVAL;
  const bool vec = (D & 7) == 0 && vec_rows(x, ldx) && aligned(codes, 8);
  const unsigned long long threads = (unsigned long long)M * groups_of(D) * (vec ? 4 : 32);
  if (vec) hipLaunchKernelGGL(pack8_kernel<8>, dim3(blocks_for(threads)), dim3(256), 0, (hipStream_t)stream, x, x_dtype, ldx, (signed char*)codes, (unsigned char*)exponents, M, D);
  else hipLaunchKernelGGL(pack8_kernel<1>, dim3(blocks_for(threads)), dim3(256), 0, (hipStream_t)stream, x, x_dtype, ldx, (signed char*)codes, (unsigned char*)exponents, M, D);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_unpack8(const void* codes, const void* exponents, void* out, int out_dtype, long long ldo, int M, int D, int width,
                   void* stream) {
  if (M <= 0 || D <= 0 || width < D || !dt_ok(out_dtype) || ldo < width || !codes || !exponents || !out ||
      !aligned(out, dt_size(out_dtype)))
    return COGAIM_EINVAL;
  const bool vec = (D & 7) == 0 && (width & 7) == 0 && vec_rows(out, ldo) && aligned(codes, 8);
  const unsigned long long threads = (unsigned long long)M * (vec ? width / 8 : width);
  if (vec) hipLaunchKernelGGL(unpack8_kernel<8>, dim3(blocks_for(threads)), dim3(256), 0, (hipStream_t)stream, (const signed char*)codes, (const unsigned char*)exponents, out, out_dtype, ldo, M, D, width);
  else hipLaunchKernelGGL(unpack8_kernel<1>, dim3(blocks_for(threads)), dim3(256), 0, (hipStream_t)stream, (const signed char*)codes, (const unsigned char*)exponents, out, out_dtype, ldo, M, D, width);
  return COGAIM_LAUNCH_CHECK();
}

int cogaim_activation_bwd(const void* dy, int dy_dtype, long long lddy, const void* codes, const void* exponents, void* du,
                          int du_dtype, long long lddu, int activation, int M, int D, void* stream) {
  if (M <= 0 || D <= 0 || !dt_ok(dy_dtype) || !dt_ok(du_dtype) || lddy < D || lddu < D || !dy || !codes || !exponents ||
      !du || (activation != ACT_RELU && activation != ACT_GELU) || !aligned(dy, dt_size(dy_dtype)) ||
      !aligned(du, dt_size(du_dtype)))
    return COGAIM_EINVAL;
  const bool vec = (D & 7) == 0 && vec_rows(dy, lddy) && vec_rows(du, lddu) && aligned(codes, 8);
  const unsigned long long threads = (unsigned long long)M * (vec ? D / 8 : D);
  if (vec) hipLaunchKernelGGL(act_bwd_kernel<8>, dim3(blocks_for(threads)), dim3(256), 0, (hipStream_t)stream, dy, dy_dtype, lddy, (const signed char*)codes, (const unsigned char*)exponents, du, du_dtype, lddu, activation, M, D);
  else hipLaunchKernelGGL(act_bwd_kernel<1>, dim3(blocks_for(threads)), dim3(256), 0, (hipStream_t)stream, dy, dy_dtype, lddy, (const signed char*)codes, (const unsigned char*)exponents, du, du_dtype, lddu, activation, M, D);
  return COGAIM_LAUNCH_CHECK();
}

}  // extern "C"

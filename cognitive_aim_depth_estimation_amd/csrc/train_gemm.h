// MFMA main loop of the linear layers' training products (included by train_linear.hip):
//   C[m][n] = sum_k A(m, k) B(n, k),  16-bit operands, fp32 accumulation,
// for every combination of operand layouts that a linear layer's three products need:
//   forward          y = x W^T       A = x  [m][k],  B = W  [n][k]     both contiguous along k
//   input gradient   dx = dy W       A = dy [m][k],  B = W  [k][n]     B contiguous along n
//   weight gradient  dW = dy^T x     A = dy [k][m],  B = x  [k][n]     both contiguous across k
// An operand contiguous along k is staged [row][64 k] and read with ds_read_b128; one contiguous across k is staged as
// it lies, [64 k][columns], and read with the transposing ds_read_b64_tr_b16, which hands a lane four consecutive k of
// its column: no operand is ever transposed in memory.  Staging is 16-byte LDS-DMA (buffer_load ... lds) into a ring
// of STAGES K-tiles of 64; the XOR swizzles below are applied to the DMA's source address (its destination is
// lane-linear) and again to the fragment reads, and spread the rows a read touches over all LDS banks.  Rows past the
// matrix read as zero through the buffer resource's size; a last K-tile that is not whole is masked by moving lanes
// past its end out of the resource.
//
// Accumulators hold C^T fragments (B is the MFMA's row operand), so a lane owns one row m and, with the column order
// below, runs of eight consecutive n: fragment j of a wave's strip covers columns 32 (j / 2) + 8 q + 4 (j % 2) + e for
// accumulator element e of the lanes with lane / 16 = q.  16-bit results leave as 16-byte stores and the 32 columns of
// an 8-bit group lie in four lanes.
#pragma once
#include "train_common.h"
#include <type_traits>

namespace {
using namespace train;

constexpr int TK = 64;                     // k per tile

struct Operands {
  const void* A; const void* B; long long lda, ldb;
  int rows_a, rows_b;                      // rows of A and B as stored along m and n: the matrix, with a copied operand's padding
  int KA, KB;                              // k of A and B as stored: KA may hold zero columns past KB
  int M, N;                                // the result
  int tiles_m, tiles_n, splits, kt_per_split;
  float* col_sum;                          // weight gradient: [splits][M] sums of A over k (the bias' gradient), or null
};

__device__ __forceinline__ int swz_k_plain(int r) { return (r >> 1) & 7; }                               // rows r, r + 1, ...
__device__ __forceinline__ int swz_k_wide(int r) { return ((r >> 1) & 1) | (((r >> 3) & 3) << 1); }      // rows of the column order
template <int R> __device__ __forceinline__ int swz_x_plain(int k) {                                    // in 32-byte units
  return R >= 128 ? (k & 3) | (((k >> 3) & 1) << 2) : ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
}
template <int R> __device__ __forceinline__ int swz_x_wide(int k) { return R >= 128 ? k & 3 : (k >> 1) & 1; }   // in 64-byte units

// 64 lanes bring 1 KiB into LDS.  Written as asm because the compiler answers the builtin with a wait for all DMA in
// flight before every transposing read (it cannot tell the ring's stages apart); the kernel counts its own waits.  No
// register is written.
__device__ __forceinline__ void dma16(unsigned lane_offset, u32x4v rsrc, unsigned lds_offset) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(lane_offset), "s"(rsrc), "s"(lds_offset) : "m0");
}

// One operand's side of the DMA: R rows (or columns), NW waves; KC: contiguous along k; WIDE: column order of B.  A wave
// brings PIECES KiB of every K-tile, the first half of them into the part of the stage that the eight-step loop below
// releases first: contiguous along k, the later-read rows of every wave's strip (SPLIT / 2 .. SPLIT - 1 of each SPLIT of
// A, the others of B); contiguous across k, the first 32 k.
template <int R, int NW, bool KC, bool WIDE, int SPLIT> struct Stager {
  static constexpr int PIECES = R / 8 / NW;
  unsigned off[PIECES], chunk[KC ? PIECES : 1];
  unsigned dst[PIECES];
  unsigned long long base; long long left, step;      // next K-tile's first byte, bytes of the operand from there
  int k_left;                                         // k from there to the operand's end
  u32x4v rsrc;
  // piece i of a wave: the first-released half of the K-tile is dealt to the waves ahead of the second.  Where the count is
  // odd, the middle piece of the lower half of the waves still belongs to the first half, of the others to the second.
  static constexpr int EARLY = PIECES / 2;            // pieces that lie in the first half for every wave
  __device__ __forceinline__ static int piece_of(int wave, int i) {
    constexpr int ALL = R / 8, HALF = ALL / 2;
    int second, e;                                    // half, and place among its pieces
    if constexpr (PIECES == 1) { second = wave >= NW / 2; e = second ? wave - NW / 2 : wave; }
    else if constexpr (PIECES % 2 == 0) { second = i >= EARLY; e = wave * EARLY + (second ? i - EARLY : i); }
    else {
      second = i > EARLY || (i == EARLY && wave >= NW / 2);
      if (i < EARLY) e = wave * EARLY + i;
      else if (i == EARLY) e = second ? NW * EARLY + wave - NW / 2 : NW * EARLY + wave;
      else e = wave * EARLY + i - EARLY - 1;
    }
    if constexpr (KC) {
      constexpr int P = SPLIT / 16;                   // pieces (8 rows) in half a strip
      const int in_strip = e / P * (2 * P) + e % P;   // the lower halves of the strips
      return in_strip + ((second ^ (WIDE ? 0 : 1)) ? P : 0);
    } else {
      return e + second * HALF;
    }
  }
  __device__ __forceinline__ void init(const void* p, long long ld, int first, int count, int K, int k0, int wave, int lane, unsigned lds) {
    k_left = K - k0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int piece = piece_of(wave, i);
      dst[i] = __builtin_amdgcn_readfirstlane(lds + piece * 1024);
      if constexpr (KC) {
        const int r = piece * 8 + (lane >> 3);
        const int c = (lane & 7) ^ (WIDE ? swz_k_wide(r) : swz_k_plain(r));
        off[i] = (unsigned)r * (unsigned)(ld * 2) + (unsigned)c * 16;
        chunk[i] = (unsigned)c * 8;
      } else {
        constexpr int CR = R / 8, RP = 64 / CR;       // 16-byte chunks per k, k per piece
        const int k = piece * RP + lane / CR;
        const int c = (lane % CR) ^ (WIDE ? swz_x_wide<R>(k) << 2 : swz_x_plain<R>(k) << 1);
        off[i] = (unsigned)k * (unsigned)(ld * 2) + (unsigned)c * 16;
      }
    }
    if constexpr (KC) {
      base = reinterpret_cast<unsigned long long>(p) + ((unsigned long long)first * ld + k0) * 2;
      left = (((long long)count - first - 1) * ld + K - k0) * 2;
      step = TK * 2;
    } else {
      base = reinterpret_cast<unsigned long long>(p) + ((unsigned long long)k0 * ld + first) * 2;
      left = (((long long)K - k0 - 1) * ld + count - first) * 2;
      step = TK * ld * 2;
    }
  }
  // the resource of the next K-tile; without `live` its loads are dropped (and still counted by the waits)
  __device__ __forceinline__ void aim(bool live) {
    const unsigned n = live && left > 0 ? (unsigned)(left < 0x7ffffff0LL ? left : 0x7ffffff0LL) : 0u;
    rsrc[0] = __builtin_amdgcn_readfirstlane((unsigned)base);
    rsrc[1] = __builtin_amdgcn_readfirstlane((unsigned)(base >> 32) & 0xffffu);
    rsrc[2] = __builtin_amdgcn_readfirstlane(n);
    rsrc[3] = 0x00020000u;
  }
  __device__ __forceinline__ void piece(int i, unsigned stage) {
    unsigned o = off[i];
    if (KC && k_left < TK) o = (int)chunk[KC ? i : 0] < k_left ? o : 0xffffff00u;
    dma16(o, rsrc, __builtin_amdgcn_readfirstlane(dst[i] + stage));
  }
  __device__ __forceinline__ void advance() { base += step; left -= step; k_left -= TK; }
};

// eight 16-bit values of fragment data through two transposing reads (k 0-3 and 4-7 of the lane's eight)
template <class T> struct TrRead;
typedef __bf16 bf16x4t __attribute__((ext_vector_type(4)));
typedef __fp16 f16x4t __attribute__((__vector_size__(8)));
template <> struct TrRead<__bf16> {
  static __device__ __forceinline__ bf16x8 read(const char* p, int second) {
    typedef __attribute__((address_space(3))) bf16x4t* lp;
    const bf16x4t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lp)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lp)(p + second));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};
template <> struct TrRead<_Float16> {
  static __device__ __forceinline__ f16x8 read(const char* p, int second) {
    typedef __attribute__((address_space(3))) f16x4t* lp;
    const f16x4t lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lp)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lp)(p + second));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// the fragment reads of one operand: `i` a fragment of the wave's strip, `s` the k32 half
template <class T, int R, bool KC, bool WIDE> struct Reader {
  using v8 = typename Half<T>::v8;
  int at, flip;
  __device__ __forceinline__ void init(int strip, int lane) {         // strip: the wave's first row (column) in the tile
    const int fr = lane & 15, fq = lane >> 4;
    if constexpr (KC) {
      const int r = strip + (WIDE ? 8 * (fr >> 2) + (fr & 3) : fr);
      at = r * 128; flip = (fq ^ (WIDE ? swz_k_wide(r) : swz_k_plain(r))) << 4;      // fragments move r by multiples the swizzles ignore
    } else {
      const int k = 8 * fq + (fr >> 2);
      if constexpr (WIDE) at = k * (R * 2) + (((strip / 32) ^ swz_x_wide<R>(k)) << 6) + (fr & 3) * 16;
      else at = k * (R * 2) + (((strip / 16) ^ swz_x_plain<R>(k)) << 5) + (fr & 3) * 8;
      flip = 0;
    }
  }
  __device__ __forceinline__ v8 read(const char* stage, int i, int s) const {
    if constexpr (KC) {
      const int row = WIDE ? 4 * (i & 1) + 32 * (i >> 1) : 16 * i;
      return *reinterpret_cast<const v8*>(stage + at + row * 128 + (flip ^ (s << 6)));
    } else if constexpr (WIDE) {
      return TrRead<T>::read(stage + (at ^ ((i >> 1) << 6)) + (i & 1) * 8 + s * (32 * R * 2), 4 * R * 2);
    } else {
      return TrRead<T>::read(stage + (at ^ (i << 5)) + s * (32 * R * 2), 4 * R * 2);
    }
  }
};

// bijective XCD-aware remap: blocks of one XCD (bid % 8) get a contiguous range
__device__ __forceinline__ int xcd_range(int bid, int n) {
  const int q = n >> 3, r = n & 7, x = bid & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
}

template <int BM_, int BN_, int WM_, int WN_, int ST_, bool STEPS_> struct Tile {
  static constexpr bool STEPS = STEPS_;                     // the eight-step loop
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = ST_, NW = WM_ * WN_;
  static constexpr int MI = BM_ / WM_ / 16, NJ = BN_ / WN_ / 16;
  static constexpr int STAGE = (BM_ + BN_) * TK * 2;
};

// FAST: the result's width is a multiple of eight (Epi::fast()); the other form only in the smallest tile, whose epilogue is short
template <class T, bool AKC, bool BKC, class TL, class Epi, bool FAST>
__global__ __launch_bounds__(TL::NW * 64, 2) void train_gemm_kernel(Operands g, Epi epi) {
  constexpr int BM = TL::BM, BN = TL::BN, MI = TL::MI, NJ = TL::NJ, ST = TL::STAGES;
  constexpr int PER_STAGE = (BM + BN) / 8 / TL::NW;                   // DMA instructions a wave issues per K-tile
  __shared__ __attribute__((aligned(1024))) char smem[ST * TL::STAGE + Epi::TABLE * sizeof(float2)];
  float2* const table = reinterpret_cast<float2*>(smem + ST * TL::STAGE);      // the epilogue's own, complete behind the first barrier below
  using H = Half<T>;
  using v8 = typename H::v8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / TL::WN, wn = wave % TL::WN;
  const int tiles = g.tiles_m * g.tiles_n;
  const int id = xcd_range(blockIdx.x, gridDim.x);
  const int split = id / tiles, tile = id - split * tiles;
  // bands of 8 tile rows: the 32 tiles an XCD works on at a time share 8 row panels and 4 column panels
  constexpr int BAND = 8;
  const int band = tile / (BAND * g.tiles_n), in_band = tile - band * BAND * g.tiles_n;
  const int rows = g.tiles_m - band * BAND < BAND ? g.tiles_m - band * BAND : BAND;
  const int tn = in_band / rows, tm = band * BAND + in_band - tn * rows;
  const int m0 = tm * BM, n0 = tn * BN;
  const int nk_all = (g.KA + TK - 1) / TK;
  const int kt0 = split * g.kt_per_split;
  int nk = nk_all - kt0; nk = nk < g.kt_per_split ? nk : g.kt_per_split;        // K-tiles of this block (at least 1)

  const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  Stager<BM, TL::NW, AKC, false, BM / TL::WM> sa;
  Stager<BN, TL::NW, BKC, true, BN / TL::WN> sb;
  sa.init(g.A, g.lda, m0, g.rows_a, g.KA, kt0 * TK, wave, lane, lds);
  sb.init(g.B, g.ldb, n0, g.rows_b, g.KB, kt0 * TK, wave, lane, lds + BM * TK * 2);
  int issued = 0;
  sa.aim(true); sb.aim(true);
  auto advance = [&]() {
    ++issued;
    sa.advance(); sb.advance();
    sa.aim(issued < nk); sb.aim(issued < nk);
  };
  Reader<T, BM, AKC, false> ra;
  Reader<T, BN, BKC, true> rb;
  ra.init(wm * (BM / TL::WM), lane);
  rb.init(wn * (BN / TL::WN), lane);

  // sums begin at the bias (a lane's columns are the same for all its rows)
  const int fr = lane & 15, fq = lane >> 4;
  const int mw = m0 + wm * (BM / TL::WM) + fr, nw = n0 + wn * (BN / TL::WN) + 8 * fq;
  f32x4 acc[MI][NJ];
#pragma unroll
  for (int h = 0; h < NJ / 2; ++h) {
    float b[8];
    epi.start(nw + 32 * h, b);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      acc[i][2 * h] = f32x4{b[0], b[1], b[2], b[3]};
      acc[i][2 * h + 1] = f32x4{b[4], b[5], b[6], b[7]};
    }
  }
  // what the epilogue reads (residual, 8-bit codes), requested here where the registers allow: its latency lies under the
  // main loop then
  constexpr bool FETCH_AHEAD = MI * NJ * 4 <= 64;
  typename Epi::Row row[NJ / 2][FETCH_AHEAD ? MI : 2];
  if constexpr (FETCH_AHEAD) {
#pragma unroll
    for (int h = 0; h < NJ / 2; ++h)
#pragma unroll
      for (int i = 0; i < MI; ++i) epi.template fetch<FAST>(mw + 16 * i, nw + 32 * h, row[h][i]);
  }
  // sums of A over k for the bias' gradient: products with a fragment of ones, the row fragments dealt to the WN waves
  // that share them; only the blocks of the first tile column
  constexpr bool SUMS = !AKC;
  constexpr int NS = SUMS ? MI / TL::WN : 1;
  static_assert(!SUMS || (MI % TL::WN == 0 && (BM & (BM - 1)) == 0), "row fragments are dealt evenly; rows across k in powers of two");
  f32x4 sums[NS];
  const bool with_sums = SUMS && g.col_sum && tn == 0;
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < NS; ++i) sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto add_sums = [&](const char* stage, int s) __attribute__((always_inline)) {
    if constexpr (SUMS) {
      if (with_sums) {
        v8 ones;
#pragma unroll
        for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;
#pragma unroll
        for (int q = 0; q < NS; ++q) sums[q] = H::mfma16(ones, ra.read(stage, wn * NS + q, s), sums[q]);
      }
    }
  };

  if constexpr (TL::STEPS) {
    // Two stages.  A K-tile is eight steps of 8 MFMAs, a quarter of the wave's tile at one k32 half each, ordered so that
    // a step changes one operand; the fragments of a step are read between the MFMAs of the one before it, and the
    // six to eight DMA pieces that a wave owes the K-tile after the next go out one per step, in the order in which the stage's
    // halves fall free: the first half behind the barrier in mid-tile, the second behind the one at its end.
    static_assert(NJ == 4 && ST == 2 && MI % 2 == 0, "written for strips of 64 columns");
    constexpr int MH = MI / 2, PA = decltype(sa)::PIECES, EA = decltype(sa)::EARLY, LATE = PA - EA;
    static_assert(decltype(sb)::PIECES == 4 && PA >= 2 && PA <= 4, "six to eight pieces a wave and K-tile");
    v8 ax[MH], ay[MH], wa[2], wb[2];
    unsigned fill = 0;                                       // stage the DMA fills
    // order: A's early pieces, B's two early ones | the late ones.  At most four early: three go out in steps 5 to 7
    auto piece = [&](int q) __attribute__((always_inline)) {
      if (q < EA) sa.piece(q, fill);
      else if (q < EA + 2) sb.piece(q - EA, fill);
      else if (q < EA + 2 + LATE) sa.piece(q - 2, fill);
      else if (q < PA + 4) sb.piece(q - PA, fill);
      if (q == PA + 3) { advance(); fill ^= TL::STAGE; }
    };
    constexpr int NP = PA + 4;
#pragma unroll
    for (int q = 0; q < NP; ++q) piece(q);
#pragma unroll
    for (int q = 0; q < 4; ++q) piece(q);
    epi.fill(table, threadIdx.x, TL::NW * 64);
    asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < MH; ++i) ax[i] = ra.read(smem, i, 0);
#pragma unroll
    for (int j = 0; j < 2; ++j) wa[j] = rb.read(smem + BM * TK * 2, j, 0);
// one step: MFMAs of rows MH mh_.., columns 2 nh_..; reads `load_(k)` behind the first nl_ of them, piece q_ ahead of the last
#define TRAIN_STEP(af_, wf_, mh_, nh_, nl_, load_, q_)                                                                  \
  _Pragma("unroll") for (int k_ = 0; k_ < 2 * MH; ++k_) {                                                               \
    acc[(mh_) * MH + (k_ >> 1)][(nh_) * 2 + (k_ & 1)] =                                                                 \
        H::mfma16(wf_[k_ & 1], af_[k_ >> 1], acc[(mh_) * MH + (k_ >> 1)][(nh_) * 2 + (k_ & 1)]);                        \
    if (k_ < (nl_)) { load_; }                                                                                          \
    if (k_ == 2 * MH - 2 && (q_) < NP) piece(q_);                                                                       \
    __builtin_amdgcn_sched_barrier(0);                                                                                  \
  }
    auto ktile = [&](auto stage_c) __attribute__((always_inline)) {
      constexpr int S0 = decltype(stage_c)::value * TL::STAGE, S1 = TL::STAGE - S0;
      const char* const as = smem + S0;
      const char* const bs = as + BM * TK * 2;
      const char* const an = smem + S1;
      const char* const bn = an + BM * TK * 2;
      __builtin_amdgcn_sched_barrier(0);
      TRAIN_STEP(ax, wa, 0, 0, 2, wb[k_] = rb.read(bs, 2 + k_, 0), 4)
      add_sums(as, 0);
      TRAIN_STEP(ax, wb, 0, 1, MH, ay[k_] = ra.read(as, MH + k_, 0), 5)
      TRAIN_STEP(ay, wb, 1, 1, MH, ax[k_] = ra.read(as, MH + k_, 1), 6)
      TRAIN_STEP(ay, wa, 1, 0, 2, wb[k_] = rb.read(bs, k_, 1), 7)
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      TRAIN_STEP(ax, wb, 1, 0, 2, wa[k_] = rb.read(bs, 2 + k_, 1), 0)
      add_sums(as, 1);
      TRAIN_STEP(ax, wa, 1, 1, MH, ay[k_] = ra.read(as, k_, 1), 1)
      TRAIN_STEP(ay, wa, 0, 1, 0, , 2)
      asm volatile("s_waitcnt vmcnt(3) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      TRAIN_STEP(ay, wb, 0, 0, 4, if (k_ < MH) ax[k_ < MH ? k_ : 0] = ra.read(an, k_, 0); if (k_ < 2) wa[k_ & 1] = rb.read(bn, k_ & 1, 0), 3)
    };
    for (int kt = 0; kt < nk; kt += 2) {
      ktile(std::integral_constant<int, 0>{});
      if (kt + 1 < nk) ktile(std::integral_constant<int, 1>{});
    }
#undef TRAIN_STEP
  } else {
    auto stage_all = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < decltype(sa)::PIECES; ++i) sa.piece(i, slot * TL::STAGE);
#pragma unroll
      for (int i = 0; i < decltype(sb)::PIECES; ++i) sb.piece(i, slot * TL::STAGE);
      advance();
    };
#pragma unroll
    for (int p = 0; p < ST - 1; ++p) stage_all(p);
    epi.fill(table, threadIdx.x, TL::NW * 64);
    int slot = 0;
    for (int kt = 0; kt < nk; ++kt) {
      // this K-tile has landed (the ST - 2 younger ones may still be in flight) and this wave's reads of the slot that is
      // refilled next are done; behind the barrier that holds for every wave
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"((ST - 2) * PER_STAGE) : "memory");
      stage_all(slot == 0 ? ST - 1 : slot - 1);
      const char* as = smem + slot * TL::STAGE;
      const char* bs = as + BM * TK * 2;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v8 bf[NJ], af[MI];
#pragma unroll
        for (int j = 0; j < NJ; ++j) bf[j] = rb.read(bs, j, s);
#pragma unroll
        for (int i = 0; i < MI; ++i) af[i] = ra.read(as, i, s);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = H::mfma16(bf[j], af[i], acc[i][j]);
        add_sums(as, s);
      }
      slot = slot == ST - 1 ? 0 : slot + 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the dropped loads past the end
  if constexpr (SUMS) {
    if (with_sums && fq == 0) {
#pragma unroll
      for (int q = 0; q < NS; ++q) {
        const int m = mw + 16 * (wn * NS + q);
        if (m < g.M) g.col_sum[(size_t)split * g.M + m] = sums[q][0];
      }
    }
  }
  typename Epi::Columns col[NJ / 2];
#pragma unroll
  for (int h = 0; h < NJ / 2; ++h) epi.columns(nw + 32 * h, col[h]);
  auto fetch_row = [&](int i) __attribute__((always_inline)) {
    if constexpr (!FETCH_AHEAD)
#pragma unroll
      for (int h = 0; h < NJ / 2; ++h) epi.template fetch<FAST>(mw + 16 * i, nw + 32 * h, row[h][i & 1]);
  };
  fetch_row(0);
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    if (i + 1 < MI) fetch_row(i + 1);                          // ahead of this row's stores
#pragma unroll
    for (int h = 0; h < NJ / 2; ++h) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = acc[i][2 * h][e]; v[4 + e] = acc[i][2 * h + 1][e]; }
      epi.template finish<FAST, 16, 32>(split, mw + 16 * i, nw + 32 * h, v, col[h], row[h][FETCH_AHEAD ? i : i & 1], table);
    }
  }
}

}  // namespace

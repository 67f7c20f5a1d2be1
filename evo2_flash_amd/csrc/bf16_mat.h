// bf16 matrix products on v_mfma_f32_32x32x16_bf16 with fp32 sums, in the three
// orientations a linear layer and its gradients need, and with the epilogues of
// the gated product and of the head's cross entropy:
//   MAT_NT  out[m, n] = sum_k x[m, k] w[n, k]   (x (M, K), w (N, K))
//   MAT_NN  out[m, n] = sum_k x[m, k] w[k, n]   (x (M, K), w (K, N))
//   MAT_TN  out[m, n] = sum_k x[k, m] w[k, n]   (x (K, M), w (K, N))
//
// A workgroup of four waves owns 256 columns by 64 TM rows of the output, a wave
// 128 by 32 TM of them, with w as MFMA operand A so that a lane ends up with
// four consecutive columns of one row.  K moves in slices of 64: 32 KB of w and
// 8 TM KB of x per stage, HBM -> LDS by direct-to-LDS loads; slice k + NST is
// loaded into the stage of slice k as soon as every wave has read it, and the
// workgroup meets at one barrier per slice.  Workgroups are persistent (one per
// CU walks its tiles) and the loads run on across tile boundaries, so a tile's
// first slices land while the one before finishes.
//
// An operand whose rows run along K ("K-contiguous") is staged as rows of 128
// bytes, 16-byte chunk c of row r at c ^ ((r >> 1) & 7), and read 16 bytes a
// lane.  One whose rows run along M or N is staged as 64 rows of the tile's
// width as they lie in memory and transposed on the way out of LDS
// (ds_read_b64_tr_b16: a group of 16 lanes reads 4 rows of 16 columns and each
// lane receives one column's four values), so no operand is ever transposed in
// memory.  Its 32-byte pairs of chunks are XORed with the row's low bits, so
// that the four rows a group reads lie on distinct banks.
//
// Loads go through buffer descriptors rebased to the wave's first row of each
// slice, so that operands may pass 4 GB; rows and columns outside the operand read
// zeros.
#pragma once

#include <algorithm>
#include <climits>

#include "attn_common.h"

namespace evo2 {

typedef __attribute__((ext_vector_type(16))) float mf32x16_t;
typedef __attribute__((ext_vector_type(4))) short ms16x4_t;
typedef __attribute__((address_space(3))) ms16x4_t mlds_s16x4_t;

enum MatForm { MAT_NT = 0, MAT_NN = 1, MAT_TN = 2 };
enum MatEpi {
  MAT_BF16 = 0,   // out as bf16
  MAT_F32 = 1,    // fp32 partial sums, one plane per split (or added to what is there)
  MAT_GATED = 2,  // (x w^T) * (x w2^T), and both factors of its gradients
  MAT_STATS = 3,  // each row's max and sum of exponentials over 128 columns
  MAT_DLOG = 4,   // the gradient of the cross entropy at the logits
  MAT_GELU = 5,   // gelu(x w^T) * (x w2^T), as MAT_GATED
};

constexpr int MAT_CUS = 256;     // workgroups a launch fills the card with
constexpr int MAT_BN = 256;      // output columns per workgroup
constexpr int MAT_BK = 64;       // K per slice
constexpr uint32_t MAT_OUT = 0x80000000u;  // an offset past every descriptor here

constexpr int mat_stages(int tm) { return tm <= 2 ? 3 : 2; }

struct MatArgs {
  const bf16_t *x; int64_t sx;            // row strides in elements
  const bf16_t *w, *w2; int64_t sw;
  int M, N, K;                            // K: contraction of w (of each half of a pair)
  int Kx;                                 // contraction columns x holds (K-contiguous x)
  int kpair;                              // MAT_NN: slices of w before w2's follow
  int mpair, xpair;                       // MAT_TN: row tiles of out before out2's, and x's
                                          // column where they start
  int kt;                                 // slices per tile, a multiple of the stages
  int tiles_m, tiles_n, splits;
  void *out, *out2; int64_t so;
  int64_t plane;                          // MAT_F32: elements between the splits' partial sums
  int add;                                // MAT_F32: add to out
  bf16_t *kept; int64_t kplane;           // MAT_GATED, MAT_GELU: what the backward pass needs, or null
  // cross entropy: rows' targets (less col0), log-sum-exp, upstream gradient
  const int64_t *targets; int64_t ignore; int64_t V; int64_t col0;
  const float *lse; const float *grad; int64_t sgrad;
  int weighted;                           // MAT_DLOG: rows times their upstream gradient
  float2 *part; float *tgt;
  const float *num, *den;                 // MAT_BF16: out times *num / *den (each may be null)
};

// Tile of the t-th work item: whole items go to the XCDs in turn (workgroup b
// runs on XCD b mod 8), each XCD taking one run of a sequence that walks panels of
// four column tiles row by row, so that the 32 tiles an XCD has in flight share
// 4 w tiles and 8 x tiles in its L2.  A bijection onto the items.
__host__ __device__ inline void mat_tile(int t, int tiles_m, int tiles_n, int splits, int &bm, int &bn,
                                         int &sp) {
  const int total = tiles_m * tiles_n * splits;
  const int xcd = t & 7, q = total >> 3, r = total & 7;
  int s = xcd * q + (xcd < r ? xcd : r) + (t >> 3);
  const int plane = tiles_m * tiles_n;
  sp = s / plane;
  s -= sp * plane;
  const int panel = s / (4 * tiles_m);
  s -= panel * 4 * tiles_m;
  const int width = tiles_n - 4 * panel < 4 ? tiles_n - 4 * panel : 4;
  bm = s / width;
  bn = 4 * panel + (s - bm * width);
}

// gelu(x) = x cdf(x), and its slope cdf(x) + x pdf(x).  The tail cdf(-|x|) is
// exp(-x^2 / 2) t Q(t) with t = 1 / (1 + |x| / 4): Q, a polynomial of degree 6 fitted to
// erfc(|x| / sqrt 2) exp(x^2 / 2) / (2 t) over |x| < 14, is off by 1.9e-8 at most (near
// 0.05, where that is 4e-8 of the cdf), the fp32 steps by up to 3e-7; the tail keeps its
// leading digits (to 1e-3 at -13), which 1 + erf loses below -5, and one exponential serves
// both results without a branch (by erff 2048 rows of 5120 x 1920, kept, took 118 us, so
// 100).
__device__ __forceinline__ void gelu_both(const float x, float &value, float &slope) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.25f, fabsf(x), 1.0f));
  const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
  float q = fmaf(-0.08913502097129822f, t, 0.3290213942527771f);
  q = fmaf(q, t, -0.24036912620067596f);
  q = fmaf(q, t, 0.2513173818588257f);
  q = fmaf(q, t, 0.043495841324329376f);
  q = fmaf(q, t, 0.10600420832633972f);
  q = fmaf(q, t, 0.0996653363108635f);
  const float tail = q * t * e, cdf = x > 0.0f ? 1.0f - tail : tail;
  slope = fmaf(x * 0.39894228040143268f, e, cdf);
  value = x * cdf;
}

// x's bits, of which the high 24 are x rounded to nearest (ties away from 0; an infinity or
// a NaN stays what it is).
__device__ __forceinline__ uint32_t round24(const float x) {
  const uint32_t u = __float_as_uint(x);
  return x == x ? u + 0x80u : u;  // (an infinity's low byte is dropped again)
}

// What a row's softmax less its target is multiplied by: its upstream gradient, 0 of an
// ignored row, NaN of a target outside the vocabulary.  Where all rows share the
// upstream gradient (a sum or a mean) it is left to the products' results: times one
// factor, the values near -1 at the targets would all be rounded the same way.
__device__ __forceinline__ float loss_weight(const MatArgs &p, int64_t m, int64_t target) {
  if (target == p.ignore) return 0.0f;
  if (target < 0 || target >= p.V) return __builtin_nanf("");
  return p.weighted ? p.grad[m * p.sgrad] : 1.0f;
}

// (a mean of no rows has no gradient)
__device__ __forceinline__ float mat_factor(const float *num, const float *den) {
  const float n = num ? *num : 1.0f;
  return !den ? n : *den == 0.0f ? 0.0f : n / *den;
}

template <int FORM, int TM, int EPI>
__global__ __launch_bounds__(256) void mat_kernel(MatArgs p) {
  static_assert(FORM != MAT_TN || TM != 3, "rows of 192 do not fill whole load blocks");
  constexpr int BM = 64 * TM, NST = mat_stages(TM);
  constexpr bool WR = FORM != MAT_NT, XR = FORM == MAT_TN;  // rows along N / M
  constexpr int WST = MAT_BN * MAT_BK, XST = BM * MAT_BK;   // elements per stage
  __shared__ __align__(16) bf16_t w0[WST], w1[WST], w2s[NST > 2 ? WST : 8];
  __shared__ __align__(16) bf16_t x0[XST], x1[XST], x2s[NST > 2 ? XST : 8];
  __shared__ __align__(16) float turned[4][32 * 32];        // a wave's 32 x 32 results, by rows
  constexpr bool PAIR = EPI == MAT_GATED || EPI == MAT_GELU;
  constexpr int DB = 8, DX = 2 * TM;  // 1 KB loads of w and x per wave and slice

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int total = p.tiles_m * p.tiles_n * p.splits;
  const int grid = static_cast<int>(gridDim.x);
  const int ntile = (total - static_cast<int>(blockIdx.x) + grid - 1) / grid;
  if (ntile <= 0) return;  // uniform; (the host launches no such workgroup)
  const int KT = p.kt;

  // Load block j of a wave: RP rows of LP lanes; lane i fills physical chunk i % LP of
  // row RP j + i / LP.  The swizzle depends on the row's low bits, hence on j's
  // parity alone.
  constexpr int LPW = WR ? 32 : 8, RPW = 64 / LPW;           // w
  constexpr int LPX = XR ? BM / 8 : 8, RPX = 64 / LPX;       // x
  auto logical = [](bool rows, int width, int row, int pc) {
    if (!rows) return pc ^ ((row >> 1) & 7);
    return pc ^ ((width == 64 ? (row >> 1) & 1 : row & 3) << 2);
  };
  int cw[2], cx[2];            // logical chunk
  uint32_t lw[DB], lx[DX];     // byte offset of block j from the wave's first row
#pragma unroll
  for (int par = 0; par < 2; ++par) {
    cw[par] = logical(WR, MAT_BN, RPW * par + lane / LPW, lane % LPW);
    cx[par] = logical(XR, BM, RPX * par + lane / LPX, lane % LPX);
  }
#pragma unroll
  for (int j = 0; j < DB; ++j)
    lw[j] = static_cast<uint32_t>(RPW * j + lane / LPW) * static_cast<uint32_t>(p.sw * 2) + 16u * cw[j & 1];
#pragma unroll
  for (int j = 0; j < DX; ++j)
    lx[j] = static_cast<uint32_t>(RPX * j + lane / LPX) * static_cast<uint32_t>(p.sx * 2) + 16u * cx[j & 1];
  auto stage_w = [&](auto st) __attribute__((always_inline)) -> bf16_t * {
    constexpr int S = decltype(st)::value;
    return S == 0 ? w0 : S == 1 ? w1 : w2s;
  };
  auto stage_x = [&](auto st) __attribute__((always_inline)) -> bf16_t * {
    constexpr int S = decltype(st)::value;
    return S == 0 ? x0 : S == 1 ? x1 : x2s;
  };

  // The next slice to load: slice ds of this workgroup's tile dj, at (bm, bn, sp).
  int dj = 0, ds = 0, dbm, dbn, dsp;
  mat_tile(static_cast<int>(blockIdx.x), p.tiles_m, p.tiles_n, p.splits, dbm, dbn, dsp);
  au32x4_t nw, nx;  // its descriptors
  int wpast, xpast;
  auto next = [&]() __attribute__((always_inline)) {
    if (ds == KT) {  // (past the last slice the loads repeat it: every step issues as many)
      if (dj + 1 < ntile) {
        ds = 0;
        ++dj;
        mat_tile(static_cast<int>(blockIdx.x) + dj * grid, p.tiles_m, p.tiles_n, p.splits, dbm, dbn, dsp);
      } else {
        ds = KT - 1;
      }
    }
    // K-contiguous rows at a power-of-two stride put all of a slice's lines on a few
    // cache channels: workgroups of different rows start up to seven slices apart
    // (gated, 8192 x 11264 x 4096: 1566 -> 1330 us; further apart they lose the L2's
    // sharing, 1890 with the starts spread over all of K)
    int s = ds + (FORM == MAT_NT && KT >= 16 ? dbm & 7 : 0);
    if (s >= KT) s -= KT;
    s += dsp * KT;
    ++ds;
    // w: this wave's rows of the slice, their first element, how many there are
    const bf16_t *wb;
    int wrows, wleft;  // valid rows; valid elements of the last one
    if constexpr (WR) {
      const bool second = s >= p.kpair;
      const int k0 = (second ? s - p.kpair : s) * MAT_BK + 16 * wave;
      wb = (second ? p.w2 : p.w) + k0 * p.sw + dbn * MAT_BN;
      wrows = max(0, min(16, p.K - k0));
      wleft = ((p.N + 7) & ~7) - dbn * MAT_BN;
    } else {
      const int k0 = s * MAT_BK;
      // a gated tile takes 64 rows of each weight for a wave's 128 columns
      const int n0 = PAIR ? dbn * (MAT_BN / 2) + 64 * (wave >> 1) : dbn * MAT_BN + 64 * wave;
      wb = (PAIR && (wave & 1) ? p.w2 : p.w) + n0 * p.sw + k0;
      wrows = max(0, min(64, p.N - n0));
      wleft = max(0, p.K - k0);
    }
    const bf16_t *xb;
    int xrows, xleft;
    if constexpr (XR) {
      const int k0 = s * MAT_BK + 16 * wave;
      const bool second = dbm >= p.mpair;
      const int m0 = (second ? dbm - p.mpair : dbm) * BM;
      xb = p.x + k0 * p.sx + (second ? p.xpair : 0) + m0;
      xrows = max(0, min(16, p.K - k0));
      xleft = ((p.M + 7) & ~7) - m0;
    } else {
      const int k0 = s * MAT_BK, m0 = dbm * BM + 16 * TM * wave;
      xb = p.x + m0 * p.sx + k0;
      xrows = max(0, min(16 * TM, p.M - m0));
      xleft = max(0, p.Kx - k0);
    }
    const uint32_t wbytes = wrows > 0 ? static_cast<uint32_t>(((wrows - 1) * p.sw + wleft) * 2) : 0u;
    const uint32_t xbytes = xrows > 0 ? static_cast<uint32_t>(((xrows - 1) * p.sx + xleft) * 2) : 0u;
    nw = lds_rsrc(wb, wbytes);
    nx = lds_rsrc(xb, xbytes);
    // chunks past the end of K read zeros (of rows along N or M the descriptor ends
    // with the last row)
    wpast = WR ? 0 : wleft;
    xpast = XR ? 0 : xleft;
  };
  // Load i of the slice that `next` found, into a stage.
  auto load = [&](auto st, int i) __attribute__((always_inline)) {
    if (i < DB) {
      const uint32_t v = WR || 8 * cw[i & 1] < wpast ? lw[i] : MAT_OUT;
      lds_load(nw, v, stage_w(st) + (wave * DB + i) * 512);
    } else {
      const int j = i - DB;
      const uint32_t v = XR || 8 * cx[j & 1] < xpast ? lx[j] : MAT_OUT;
      lds_load(nx, v, stage_x(st) + (wave * DX + j) * 512);
    }
  };
  auto issue = [&](auto st) __attribute__((always_inline)) {
    next();
#pragma unroll
    for (int i = 0; i < DB + DX; ++i) load(st, i);
  };

  const int wn = (wave & 1) * 128, wm = (wave >> 1) * (32 * TM);  // wave's columns and rows
  const int g = lane >> 5, lr = lane & 31;
  // K-contiguous reads: row base + lr, chunk 2 kk + g of 16-wide K step kk
  const int swz = (lr >> 1) & 7;
  // transposing reads: 16-lane group q reads K rows 16 kk + 8 (q >> 1) + 0..3 (then
  // + 4 .. 7) of columns 16 (q & 1) + 0..15 of a 32-column tile; lane i of it row
  // i >> 2, columns 4 (i & 3) .. + 3
  const int ti = lane & 15, tq = lane >> 4;
  const int trow = 8 * (tq >> 1) + (ti >> 2), tcol = 16 * (tq & 1) + 4 * (ti & 3);
  auto read_w = [&](auto st, int tn, int kk) __attribute__((always_inline)) -> abf16x8_t {
    const bf16_t *b = stage_w(st);
    if constexpr (WR) {
      const int T = ((wn >> 5) + tn) ^ (ti >> 2);  // 32-column tile, swizzled
      const bf16_t *a = b + (trow + 16 * kk) * MAT_BN + 32 * T + tcol;
      const ms16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mlds_s16x4_t *)(a));
      const ms16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mlds_s16x4_t *)(a + 4 * MAT_BN));
      return __builtin_bit_cast(abf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const bf16_t *a = b + (wn + 32 * tn + lr) * MAT_BK + 8 * ((2 * kk + g) ^ swz);
      return __builtin_bit_cast(abf16x8_t, *reinterpret_cast<const au32x4_t *>(a));
    }
  };
  auto read_x = [&](auto st, int tm, int kk) __attribute__((always_inline)) -> abf16x8_t {
    const bf16_t *b = stage_x(st);
    if constexpr (XR) {
      const int T = ((wm >> 5) + tm) ^ (BM == 64 ? (ti >> 3) & 1 : ti >> 2);
      const bf16_t *a = b + (trow + 16 * kk) * BM + 32 * T + tcol;
      const ms16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mlds_s16x4_t *)(a));
      const ms16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mlds_s16x4_t *)(a + 4 * BM));
      return __builtin_bit_cast(abf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const bf16_t *a = b + (wm + 32 * tm + lr) * MAT_BK + 8 * ((2 * kk + g) ^ swz);
      return __builtin_bit_cast(abf16x8_t, *reinterpret_cast<const au32x4_t *>(a));
    }
  };

  mf32x16_t acc[4][TM];
  abf16x8_t fa[2][4][2], fb[2][TM][2];  // fragments of a half slice (two 16-wide K steps)
  // fragment f of a half slice, in the order the MFMAs take them
  auto read_frag = [&](auto st, auto half, int f) __attribute__((always_inline)) {
    constexpr int H = decltype(half)::value;
    const int kk = f / (TM + 4), t = f % (TM + 4);
    if (t < TM) fb[H][t][kk] = read_x(st, t, 2 * H + kk);
    else fa[H][t - TM][kk] = read_w(st, t - TM, 2 * H + kk);
  };
  auto read_frags = [&](auto st, auto half) __attribute__((always_inline)) {
    constexpr int H = decltype(half)::value;
#pragma unroll
    for (int f = 0; f < 2 * (TM + 4); ++f) read_frag(st, half, f);
  };
  auto mma = [&](auto half) __attribute__((always_inline)) {
    constexpr int H = decltype(half)::value;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int tn = 0; tn < 4; ++tn)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
          acc[tn][tm] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[H][tn][kk], fb[H][tm][kk], acc[tn][tm], 0, 0, 0);
  };
  // every MFMA is followed by its share of the fragment reads
  auto interleave = [&]() __attribute__((always_inline)) {
    static_for<8 * TM>([&](auto i) __attribute__((always_inline)) {
      constexpr int I = decltype(i)::value, NM = 8 * TM, ND = 8 * (WR ? 2 : 1) + 2 * TM * (XR ? 2 : 1);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, (I + 1) * ND / NM - I * ND / NM, 0);  // DS read
    });
  };
  using std::integral_constant;
  using I0 = integral_constant<int, 0>;
  using I1 = integral_constant<int, 1>;
  // Step over the slice in stage S: the MFMAs of its first half while its second
  // is read; every wave's loads of the next slice have landed (its own, waited
  // for, before the barrier) and nobody reads stage S again: it is refilled; the
  // MFMAs of the second half while the next slice's first is read.
  auto step = [&](auto st) __attribute__((always_inline)) {
    constexpr int S = decltype(st)::value;
    using N = integral_constant<int, (S + 1) % NST>;
    next();
    read_frags(st, I1{});
    mma(I0{});
    interleave();
    lds_sync<(NST - 2) * (DB + DX)>();
    // the loads stand between the fragment reads, in this order
    constexpr int NF = 2 * (TM + 4), NV = DB + DX;
    static_for<NF>([&](auto f) __attribute__((always_inline)) {
      constexpr int F = decltype(f)::value;
#pragma unroll
      for (int i = F * NV / NF; i < (F + 1) * NV / NF; ++i) load(st, i);
      read_frag(N{}, I0{}, F);
    });
    mma(I1{});
    interleave();
  };

  // Lane (lr, g) holds, for row m = wm + 32 tm + lr of the tile, columns
  // wn + 32 tn + 8 q + 4 g + i in acc[tn][tm][4 q + i].  Results go to memory by way of
  // a wave's own 32 rows of 128 bytes in LDS (16-byte chunk c of row r at c ^ (r & 7)),
  // which turn them so that eight lanes store one whole 128-byte line of a row: stored
  // as they lie, each line takes four requests, and the caches' request rate bounds the
  // burst at a tile's end.
  auto epilogue = [&](int j) __attribute__((always_inline)) {
    int bm, bn, sp;
    mat_tile(static_cast<int>(blockIdx.x) + j * grid, p.tiles_m, p.tiles_n, p.splits, bm, bn, sp);
    const bool second = FORM == MAT_TN && bm >= p.mpair;
    const int m0 = (second ? bm - p.mpair : bm) * BM + wm;      // wave's first row
    const int n0 = bn * (PAIR ? MAT_BN / 2 : MAT_BN) + (PAIR ? wn / 2 : wn);
    const float factor = EPI == MAT_BF16 ? mat_factor(p.num, p.den) : 1.0f;
    float *tb = turned[wave];
    const int tr = lane >> 3, tc = lane & 7;  // turned: lane's row of eight, 16-byte chunk
    // (LDS serves a wave in order; the compiler is kept to it)
    auto fence = [] { asm volatile("" ::: "memory"); };
    // rows m .. m + 31, 64 columns from n0 + c of rows of `so` 16-bit values: v(t, i) holds
    // elements i and i + 1 of tile t (0, 1)
    auto put16 = [&](bf16_t *out, int64_t so, int m, int c, int cols, auto &&v) __attribute__((always_inline)) {
      bf16_t *b = reinterpret_cast<bf16_t *>(tb);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint2 *>(b + lr * 64 + 8 * ((4 * t + q) ^ (lr & 7)) + 4 * g) =
              make_uint2(v(t, 4 * q), v(t, 4 * q + 2));
      fence();
      bf16_t *o = out + m * so + n0 + c;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 8 * k + tr;
        const au32x4_t w = *reinterpret_cast<const au32x4_t *>(b + r * 64 + 8 * (tc ^ (r & 7)));
        if (m + r < p.M && n0 + c + 8 * tc < cols) *reinterpret_cast<au32x4_t *>(o + r * so + 8 * tc) = w;
      }
      fence();
    };
    // rows m .. m + 31, 32 columns from n0 + c of fp32 rows of `so` elements
    auto put_f32 = [&](float *out, int64_t so, int m, int c, bool add, auto &&v) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<af32x4_t *>(tb + lr * 32 + 4 * ((2 * q + g) ^ (lr & 7))) =
            af32x4_t{v(4 * q), v(4 * q + 1), v(4 * q + 2), v(4 * q + 3)};
      fence();
      float *o = out + m * so + n0 + c;
      if (so % 4 == 0 && p.N % 4 == 0) {  // uniform
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 8 * k + tr;
          af32x4_t w = *reinterpret_cast<const af32x4_t *>(tb + r * 32 + 4 * (tc ^ (r & 7)));
          if (m + r < p.M && n0 + c + 4 * tc < p.N) {
            af32x4_t *d = reinterpret_cast<af32x4_t *>(o + r * so + 4 * tc);
            if (add) w += *d;
            *d = w;
          }
        }
      } else {  // (an odd vocabulary's partial logits)
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
          const int r = 2 * k + (lane >> 5), cc = lane & 31;
          const float w = tb[r * 32 + 4 * ((cc >> 2) ^ (r & 7)) + (cc & 3)];
          if (m + r < p.M && n0 + c + cc < p.N) o[r * so + cc] = w;
        }
      }
      fence();
    };
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) {
      const int mr = m0 + 32 * tm, m = mr + lr;
      const bool live = m < p.M;
      if constexpr (EPI == MAT_BF16) {
        // (one output of half the size: as it lies, lanes l and l + 32, which hold the
        // same row, swapping halves of each pair of column groups for 16-byte stores;
        // by way of LDS 32768 x 4096 x 512 took 203 us, so 175)
        bf16_t *row = static_cast<bf16_t *>(second ? p.out2 : p.out) + m * p.so + n0;
        const int limit = live ? p.N - n0 : 0;
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
          for (int pq = 0; pq < 2; ++pq) {
            uint32_t v[4];  // columns 16 pq + 4 g + i and 16 pq + 8 + 4 g + i
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = pack_bf(acc[tn][tm][8 * pq + 2 * i] * factor, acc[tn][tm][8 * pq + 2 * i + 1] * factor);
            const auto s0 = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
            const int c = 32 * tn + 16 * pq + 8 * g;
            if (c < limit) *reinterpret_cast<au32x4_t *>(row + c) = au32x4_t{s0[0], s1[0], s0[1], s1[1]};
          }
      } else if constexpr (EPI == MAT_F32) {
        float *out = static_cast<float *>(second ? p.out2 : p.out) + sp * p.plane;
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
          put_f32(out, p.so, mr, 32 * tn, p.add != 0, [&](int i) { return acc[tn][tm][i]; });
      } else if constexpr (PAIR) {
        // h = act(z1) z2, and for the backward pass a = z2 act'(z1) and b = act(z1), in
        // place of z1 and z2, as three planes of 16 bits: the high halves of both and
        // the next eight bits of each (rounded to 24 of 32 bits, off by at most 2^-16, to
        // either side: rounded to bf16 they would put a second rounding under d1 and d2; as
        // fp32 the tile's stores and the gradient kernel's loads are a third more)
        // (gelu is a kernel of its own: its slopes held registers of the other, 777 x 11264
        // x 4096 151 us rather than 142)
        float slope[2][16];
        if constexpr (EPI == MAT_GELU) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float value;
              gelu_both(acc[t][tm][i], value, slope[t][i]);
              acc[t][tm][i] = value;
            }
        }
        put16(static_cast<bf16_t *>(p.out), p.so, mr, 0, p.N, [&](int t, int i) {
          return pack_bf(acc[t][tm][i] * acc[t + 2][tm][i], acc[t][tm][i + 1] * acc[t + 2][tm][i + 1]);
        });
        if (p.kept) {  // uniform
          auto bits = [&](int t, int i, int which) {
            const float a = EPI == MAT_GELU ? acc[t + 2][tm][i] * slope[t][i] : acc[t + 2][tm][i];
            return round24(which ? acc[t][tm][i] : a);
          };
#pragma unroll
          for (int which = 0; which < 2; ++which)
            put16(p.kept + which * p.kplane, p.N, mr, 0, p.N, [&](int t, int i) {
              return (bits(t, i, which) >> 16) | (bits(t, i + 1, which) & 0xffff0000u);
            });
          put16(p.kept + 2 * p.kplane, p.N, mr, 0, p.N, [&](int t, int i) {
            const uint32_t lo = ((bits(t, i, 0) >> 8) & 0xffu) | (bits(t, i, 1) & 0xff00u);
            const uint32_t hi = ((bits(t, i + 1, 0) >> 8) & 0xffu) | (bits(t, i + 1, 1) & 0xff00u);
            return lo | (hi << 16);
          });
        }
      } else if constexpr (EPI == MAT_STATS) {
        // max and sum of exp over the wave's 128 columns of the row, and the
        // target's logit where it lies among them
        const int limit = p.N - n0;  // columns of the vocabulary from the wave's first
        const int lim = limit - 4 * g;
        const int64_t t = live ? p.targets[m] - n0 : -1;
        // the target's place among the lane's own columns (the lane with none: past all)
        const int at = t >= 0 && t < min(128, limit) && ((t >> 2) & 1) == g ? static_cast<int>(t) - 4 * g : -1;
        float mx = -INFINITY, sum = 0.0f, zt = 0.0f;
        // EDGE: with columns past the vocabulary or a target among them.  A wave whose 128
        // columns have neither, as most, compares nothing (4096 x 131072 x 4096: 3230 ->
        // 3160 us; the same for MAT_DLOG gained nothing)
        auto stats = [&](auto edge) __attribute__((always_inline)) {
          constexpr bool EDGE = decltype(edge)::value;
          auto logit = [&](int tn, int i) {
            return !EDGE || 32 * tn + 8 * (i >> 2) + (i & 3) < lim ? acc[tn][tm][i] : -INFINITY;
          };
#pragma unroll
          for (int tn = 0; tn < 4; ++tn)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, logit(tn, i));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float sub = mx == -INFINITY ? 0.0f : mx * 1.44269504088896341f;
#pragma unroll
          for (int tn = 0; tn < 4; ++tn)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float v = logit(tn, i);
              sum += __builtin_amdgcn_exp2f(fmaf(v, 1.44269504088896341f, -sub));
              if (EDGE) zt = at == 32 * tn + 8 * (i >> 2) + (i & 3) ? v : zt;
            }
        };
        if (limit >= 128 && !__any(at >= 0)) stats(std::false_type{});
        else stats(std::true_type{});
        sum += __shfl_xor(sum, 32);
        if (live) {
          if (g == 0) p.part[static_cast<int64_t>(2 * bn + (wave & 1)) * p.M + m] = make_float2(mx, sum);
          if (at >= 0) p.tgt[m] = zt;
        }
      } else {
        // d = (exp(z - lse) - [n = target]) * weight, zeros in the columns that
        // pad the vocabulary to eights
        const int valid = p.N - n0 - 4 * g;
        const int64_t t = live ? p.targets[m] : p.ignore;
        const float wgt = live ? loss_weight(p, m, t) : 0.0f;
        const float lse2 = live ? p.lse[m] * 1.44269504088896341f : 0.0f;
        const int64_t tl = t - p.col0 - n0 - 4 * g;
        const int at = tl >= 0 && tl < 128 ? static_cast<int>(tl) : -1;
        const bool used = live && t != p.ignore;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          put16(static_cast<bf16_t *>(p.out), p.so, mr, 64 * h, (p.N + 7) & ~7, [&](int u, int i0) {
            float d[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int i = i0 + k, c = 64 * h + 32 * u + 8 * (i >> 2) + (i & 3);
              float e = __builtin_amdgcn_exp2f(fmaf(acc[2 * h + u][tm][i], 1.44269504088896341f, -lse2));
              e = at == c ? e - 1.0f : e;
              d[k] = used && c < valid ? e * wgt : 0.0f;
            }
            return pack_bf(d[0], d[1]);
          });
      }
    }
  };

  issue(I0{});
  issue(I1{});
  if constexpr (NST > 2) issue(integral_constant<int, 2>{});
  lds_sync<(NST - 1) * (DB + DX)>();  // slice 0
  read_frags(I0{}, I0{});
  for (int j = 0; j < ntile; ++j) {
#pragma unroll
    for (int tn = 0; tn < 4; ++tn)
#pragma unroll
      for (int tm = 0; tm < TM; ++tm)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[tn][tm][i] = 0.0f;
    for (int k = 0; k < KT; k += NST)
      static_for<NST>([&](auto st) __attribute__((always_inline)) { step(st); });
    epilogue(j);
  }
  // No direct-to-LDS write may still be landing when the workgroup's LDS is
  // handed to the next one.
  vmcnt_wait<0>();
}

// How a product is cut: tiles of 64 tm rows, K in `splits` runs of kt slices.
struct MatPlan {
  int tm, tiles_m, tiles_n, splits, kt;
};

// The tile height and split of least time: rounds of tiles over the CUs, times what a
// tile costs -- us per slice and us at its end, measured over 512 to 10240 of K -- and
// where few tiles let K be split, the partial sums' second launch and their bytes
// there and back.  Measured, us for tm 1 / 2 / 3 / 4:
//   NT     777 x 49999 x 1920             190 / 165 / 154 / 184
//          4096 x 131072 x 4096           4999 / 3808 / 3590 / 3341
//   gated  777 x 11264 x 4096             182 / 159 / 145 / 188
//          the same, gelu                 179 / 160 / 156 / 187
//          2048 x 5120 x 1920, kept       94 / 88 / 82 / 138
//          the same, gelu                 101 / 97 / 113 / 132
//          8192 x 11264 x 4096, kept      1740 / 1363 / 1283 / 1363
//          the same, gelu                 1815 / 1418 / 1471 / 1369
//   NN     2048 x 1920 x 10240            106 / 95 / 102 / 90 (split by 1, 2, 2, 4)
//          32768 x 4096 x 512             262 / 214 / 180 / 202
//          8192 x 4096 x 22528            1749 / 1474 / - / 1157
//   TN     512 x 4096 x 32768             208 / 163 / - / 147 (split by 2, 4, -, 8)
//          49999 x 1920 x 777             294 / 235 / - / 206
//          22528 x 4096 x 8192            1926 / 1285 / - / 1177
// M: rows of one of `pair` outputs; slices: of K; width: output columns per tile;
// gated: 0, or 1 + gelu (costs with what the backward pass needs kept; without, a tile's
// end is 2 to 19 us shorter and the choice the same or 3% behind at these sizes, but a
// plan by it would sum K in another order where a gradient is recorded).
inline MatPlan mat_plan(MatForm form, int64_t M, int64_t N, int64_t slices, int pair, int width,
                        bool may_split, int gated = 0) {
  static const double slice[4][5] = {{0, 0.60, 0.93, 1.30, 1.62},   // NT
                                     {0, 0.66, 1.00, 1.40, 1.72},   // NN
                                     {0, 0.66, 1.00, 1.30, 1.72},   // TN
                                     {0, 0.52, 0.83, 1.19, 1.54}};  // NT, gated
  static const double ends[3][5] = {{0, 4.0, 6.0, 7.0, 14.0},
                                    {0, 5.5, 10.0, 10.5, 33.0},
                                    {0, 7.5, 12.5, 24.0, 31.0}};
  const double *each = slice[gated ? 3 : form], *end = ends[gated];
  MatPlan best{};
  double least = 1e300;
  for (int tm : {4, 3, 2, 1}) {
    if (form == MAT_TN && tm == 3) continue;  // (rows of 192 do not fill whole load blocks)
    const int nst = mat_stages(tm);
    const int64_t tm_tiles = cdiv(M, 64 * tm) * pair, tn_tiles = cdiv(N, width), tiles = tm_tiles * tn_tiles;
    int64_t splits = 1;
    if (may_split && tiles < MAT_CUS) splits = std::max<int64_t>(1, std::min<int64_t>(MAT_CUS / tiles, slices / nst));
    const int64_t kt = cdiv(cdiv(slices, splits), nst) * nst;
    splits = std::max<int64_t>(1, cdiv(slices, kt));
    const double rounds = double(cdiv(tiles * splits, MAT_CUS));
    double cost = rounds * (kt * each[tm] + end[tm]);
    if (splits > 1) cost += 4.0 + double(splits) * M * pair * N * 1.0e-6;
    if (cost < least - 1e-9) {
      least = cost;
      best = MatPlan{tm, static_cast<int>(tm_tiles), static_cast<int>(tn_tiles), static_cast<int>(splits),
                     static_cast<int>(kt)};
    }
  }
  return best;
}

template <int FORM, int EPI>
inline void mat_launch(MatArgs a, const MatPlan &pl, hipStream_t st) {
  a.tiles_m = pl.tiles_m;
  a.tiles_n = pl.tiles_n;
  a.splits = pl.splits;
  a.kt = pl.kt;
  const int64_t items = static_cast<int64_t>(pl.tiles_m) * pl.tiles_n * pl.splits;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(MAT_CUS, items)));
  if (pl.tm == 4) hipLaunchKernelGGL((mat_kernel<FORM, 4, EPI>), grid, dim3(256), 0, st, a);
  else if (FORM != MAT_TN && pl.tm == 3)
    hipLaunchKernelGGL((mat_kernel<FORM, FORM == MAT_TN ? 4 : 3, EPI>), grid, dim3(256), 0, st, a);
  else if (pl.tm == 2) hipLaunchKernelGGL((mat_kernel<FORM, 2, EPI>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mat_kernel<FORM, 1, EPI>), grid, dim3(256), 0, st, a);
}

// Products compiled once (bf16_mat.hip): out as bf16, or fp32 partial sums.
void mat_nn(const MatArgs &a, const MatPlan &pl, bool f32, hipStream_t st);
void mat_tn(const MatArgs &a, const MatPlan &pl, bool f32, hipStream_t st);
void mat_nt_f32(const MatArgs &a, const MatPlan &pl, hipStream_t st);
// out (rows, cols) bf16 = the sum of `splits` fp32 planes (rows of cols, contiguous)
// times *num / *den (each may be null); cols a multiple of 8.
void mat_join(const float *part, int64_t plane, int splits, bf16_t *out, int64_t so, int64_t rows,
              int64_t cols, hipStream_t st, const float *num = nullptr, const float *den = nullptr);

// Sizes and strides the kernel's 32-bit offsets take.
inline bool mat_fits(int64_t M, int64_t N, int64_t K, int64_t s) {
  return M < (int64_t(1) << 30) && N < (int64_t(1) << 30) && K < (int64_t(1) << 30) && s < (int64_t(1) << 22) &&
         cdiv(M, 64) * cdiv(N, 128) < (int64_t(1) << 24);
}

}  // namespace evo2

// Decode attention over the 8-bit KV cache (kv_fp8.h): n query tokens per sequence (one at
// a decode step, a request's draft tokens at a verify step), heads of queries in groups
// that share a key head, token i of sequence b over positions 0 .. positions[b] + i:
//
//   out[b, i, h] = sum_l softmax_l(scale * q . k_l) v_l,   k_l, v_l = code * 2^e(page, head)
//
// as the decoder's attention layers compute it at decode (model.py:104-153).  A table entry
// outside [0, num_pages) is never dereferenced: its positions are left out of the softmax
// (a query with none left gets zeros).
//
// Split over the context: a wave takes one chunk of positions of one key head for up to 16
// query rows (a sequence's tokens x the head's group); on pages that all sequences share, a
// workgroup takes a chunk for up to 32 rows of any sequences, its waves the chunk's blocks in
// turn.  (o, max, sum) go to a workspace and a last launch joins the chunks.  Contexts of one
// chunk are written out at once; short ones, or those of as many (sequence, head)s as CUs,
// are one chunk of a workgroup (split_for).  A wave walks blocks of 64 positions with a
// running maximum and sum, on v_mfma_f32_16x16x32_bf16:
//  * scores S^T = K Q^T in four tiles; tile t's row m is position 4 t + m % 4 of page
//    m / 4, so that lane (n, g) ends with the 16 scores of page g for query row n.  A
//    lane's 16-byte load is 16 dims of one position: the A operands of two k-steps;
//  * o^T = V^T P^T; lane (m, g)'s 16-byte load is page g's 16 positions of dim 16 e + m:
//    the A operands of two k-steps, whose B operand is the lane's own probabilities.  No
//    lane exchanges anything but the maximum and, at the end, the sum.
// The codes become bf16 operands by v_cvt_scalef32_pk_bf16_fp8 with the page's scale (one
// instruction for two values, exact); the probabilities enter as bf16 high and low parts
// (~16 bits), the sums are fp32.  The next block's keys are requested when this block's
// have become scores, its values after this block's products, so loads stay in flight
// throughout.
#include "kv_fp8.h"

namespace evo2 {

struct AttnFp8Args {
  KvPages c;
  const bf16_t *q; int64_t qb, qt, qh;  // (B, n, heads, hd)
  const int64_t *pos;                   // (B,) of token 0
  float *part;                          // (B * n * heads, nchunk, hd): o of a chunk
  float2 *ml;                           // (B * n * heads, nchunk): its max (log2 units), sum
  bf16_t *out; int64_t ob, ot, oh;
  float scale;
  uint32_t B, n, heads, group, kv;      // group: query heads to a key head
  int shared, schunk, snum;             // positions of the shared pages; a chunk of them; chunks
  int chunk, nchunk;                    // a chunk of the positions behind; all chunks
};

constexpr int AF_T = 256, AF_NW = AF_T / 64;
constexpr int AF_BLK = 64;  // positions a wave takes at once

// Query row r of a key head: rows run over (sequence, token, head of the group).
struct AttnRow {
  int b, i, j;
};
__device__ __forceinline__ AttnRow attn_row(const AttnFp8Args &p, uint32_t r) {  // (B * n below 2^16: r fits)
  const uint32_t bi = r / p.group, b = p.n == 1 ? bi : bi / p.n;
  return AttnRow{static_cast<int>(b), static_cast<int>(bi - b * p.n), static_cast<int>(r - bi * p.group)};
}
__device__ __forceinline__ int row_len(const AttnFp8Args &p, const AttnRow &a) {
  const int64_t first = p.pos[a.b], all = p.c.max_pages * KV_PAGE;
  // (positions far off the table are clamped before the token is added)
  return static_cast<int>(min(max(min(first, all) + a.i + 1, int64_t(0)), all));
}

// The first k bytes of a dword; and the sign bits of the bytes that are NaN codes.
__device__ __forceinline__ uint32_t low_bytes(int k) { return k <= 0 ? 0u : k >= 4 ? 0xffffffffu : (1u << (8 * k)) - 1; }
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The value of the lane next to this one in its pair (lane ^ 1).
__device__ __forceinline__ uint32_t other_of_pair(uint32_t v) {
  return __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true);
}

// What takes a unit, a chunk of one key head of a sequence or of the shared pages:
//  * BY_WAVE: a wave; heads run fastest, so a workgroup's waves walk the same pages side by
//    side, and no wave waits for another (64 sequences of 8192 positions 664 us, with a unit
//    to a workgroup 672);
//  * BY_GROUP: a workgroup, whose eight waves take its blocks in turn and meet in LDS, for
//    contexts of one chunk;
//  * SHARED_BY_GROUP: a workgroup of four waves, on the shared pages.
// tiles: row tiles that a unit has, per sequence or (shared) in all.  The workgroups of one
// XCD (w mod 8) take the tiles of a unit one after the other, so its codes come from that
// XCD's L2 after the first.
enum AttnBy { BY_WAVE, BY_GROUP, SHARED_BY_GROUP };
template <AttnBy BY>
constexpr int AF_WAVES = BY == BY_GROUP ? 8 : AF_NW;  // of a workgroup

template <int HD, int NQT, AttnBy BY>
__global__ __launch_bounds__(64 * AF_WAVES<BY>, BY == BY_GROUP ? 1 : 2) void attn_fp8_kernel(AttnFp8Args p, uint32_t tiles) {
  constexpr bool SHARED = BY == SHARED_BY_GROUP;
  constexpr int NW = AF_WAVES<BY>;
  constexpr int KS = HD / 32;           // k-steps of a score
  constexpr int KH = HD / 64;           // 16-byte loads a position and lane
  constexpr int ET = HD / 16;           // dim tiles
  constexpr int EG = NQT == 2 ? 2 : 4;  // of them at once
  constexpr int ROWS = 16 * NQT;
  constexpr int STEP = BY == BY_WAVE ? 1 : NW;  // blocks from one of this wave's to the next
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = lane & 15, g = lane >> 4;
  // (all below 2^32, as the grid is: one 32-bit division each)
  const uint32_t w = blockIdx.x, j8 = w >> 3, tile = j8 % tiles;
  const uint32_t group = (j8 / tiles) * 8 + (w & 7), unit = BY == BY_WAVE ? group * NW + wave : group;
  const uint32_t rest = unit / p.kv;
  const int h = static_cast<int>(unit - rest * p.kv);
  const uint32_t c_count = SHARED ? p.snum : p.nchunk - p.snum;
  const int64_t seq = rest / c_count;
  if (seq >= (SHARED ? 1 : p.B)) return;  // the grid's padding
  const int ci = static_cast<int>(rest % c_count), c = SHARED ? ci : p.snum + ci;
  const uint32_t per = p.n * p.group, r0 = (SHARED ? 0 : seq * per) + ROWS * tile;
  const int nrow = static_cast<int>(min(static_cast<uint32_t>(ROWS), (SHARED ? p.B * per : (seq + 1) * per) - r0));
  const int64_t all = p.c.max_pages * KV_PAGE;
  const int l0 = SHARED ? ci * p.schunk : p.shared + ci * p.chunk;  // the chunk is [l0, l2)
  const int l2 = static_cast<int>(SHARED ? min(static_cast<int64_t>(l0) + p.schunk, static_cast<int64_t>(p.shared))
                                         : min(static_cast<int64_t>(l0) + p.chunk, all));
  // pages of a block: lane (n, g) reads keys of page n / 4 and values of page g
  const int32_t *row = p.c.table + (SHARED ? 0 : seq) * p.c.st;
  auto page_of = [&](int blk, int k) __attribute__((always_inline)) {
    const int l = l0 + AF_BLK * blk + KV_PAGE * k;
    int32_t pg = -1;
    if (l < l2) pg = row[l / KV_PAGE];
    return pg >= 0 && pg < p.c.num_pages ? pg : -1;  // -1: left out
  };
  const int first = BY == BY_WAVE ? 0 : wave;
  int32_t kpg = page_of(first, n >> 2), vpg = page_of(first, g);
  // ends of this lane's rows, of the positions any row attends to and that all do
  AttnRow rows[NQT];  // (slots past the last row repeat it, with no positions)
  int l1[NQT], l1max = l0, l1min = l2;
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    const bool live = 16 * nt + n < nrow;
    rows[nt] = attn_row(p, r0 + min(16 * nt + n, nrow - 1));
    l1[nt] = live ? min(l2, row_len(p, rows[nt])) : l0;
    l1max = max(l1max, l1[nt]);
    if (live) l1min = min(l1min, l1[nt]);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    l1max = max(l1max, __shfl_xor(l1max, o));
    l1min = min(l1min, __shfl_xor(l1min, o));
  }
  l1max = __builtin_amdgcn_readfirstlane(l1max);
  l1min = __builtin_amdgcn_readfirstlane(l1min);
  if (l0 >= l1max && p.nchunk > 1) return;  // the join does not ask for this chunk
  // Q as the B operand: k-slot (g, j) of k-step 2 hf + u is dim 64 hf + 16 g + 8 u + j
  // (SHARED: in LDS, for the registers that two row tiles need)
  __shared__ abf16x8_t qs[SHARED ? KS : 1][SHARED ? NQT : 1][64];
  abf16x8_t qop[KS][NQT];
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    const AttnRow a = rows[nt];
    const bf16_t *qr = p.q + a.b * p.qb + a.i * p.qt + (static_cast<int64_t>(h) * p.group + a.j) * p.qh + 16 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qop[ks][nt] = __builtin_bit_cast(
          abf16x8_t, *reinterpret_cast<const au32x4_t *>(qr + 64 * (ks / 2) + 8 * (ks % 2)));
  }

  if constexpr (SHARED) {
    if (wave == 0) {
#pragma unroll
      for (int nt = 0; nt < NQT; ++nt)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qs[ks][nt][lane] = qop[ks][nt];
    }
    __syncthreads();
  }

  float mrun[NQT], lrun[NQT];
  af32x4_t acc[ET][NQT];  // o^T: dims 16 e + 4 g + i in lane (n, g)
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    mrun[nt] = -INFINITY;
    lrun[nt] = 0.0f;
#pragma unroll
    for (int e = 0; e < ET; ++e) acc[e][nt] = af32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const int nblk = (l1max - l0 + AF_BLK - 1) / AF_BLK;
  // Loads of a block: its pages' scales, keys and values (a page left out reads page 0: its
  // scores are masked, its values set to zero).  Read once a launch, so with the
  // non-temporal hint (64 sequences of 8192 positions: 757 -> 714 us).  A key tile's 16 rows
  // of 128 bytes come as whole lines: eight lanes take a row, those of pair (m, m ^ 1) the
  // row of one of them in each of two loads, and exchange the halves when they read them
  // (half lines cost 3% of the stream).
  au32x4_t kr[4][KH], vr[ET];
  float ksc, vsc;
  const bool odd = n & 1;
  auto kload = [&](int32_t pg) __attribute__((always_inline)) {
    const int64_t at = max(pg, 0);
    ksc = p.c.ks[at * p.c.ksp + h * p.c.ksh];
    const uint8_t *a = p.c.k + at * p.c.kp + h * p.c.kh + 16 * g;
    if constexpr (HD == 128) a += (n & 2) * HD + 64 * (n & 1);
    else a += (n & 3) * HD;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int hf = 0; hf < KH; ++hf)
        kr[tt][hf] = __builtin_nontemporal_load(reinterpret_cast<const au32x4_t *>(a + (4 * tt + hf) * HD));
  };
  auto vload = [&](int32_t pg) __attribute__((always_inline)) {
    const int64_t at = max(pg, 0);
    vsc = p.c.vs[at * p.c.vsp + h * p.c.vsh];
    const uint8_t *a = p.c.v + at * p.c.vp + h * p.c.vh + 16 * n;
#pragma unroll
    for (int e = 0; e < ET; ++e) vr[e] = __builtin_nontemporal_load(reinterpret_cast<const au32x4_t *>(a + 256 * e));
  };
  // eight codes (two dwords) as a bf16 operand
  auto operand = [&](uint32_t a, uint32_t b, float s) __attribute__((always_inline)) {
    const au32x4_t o = {kv_decode2<false>(a, s), kv_decode2<true>(a, s), kv_decode2<false>(b, s), kv_decode2<true>(b, s)};
    return __builtin_bit_cast(abf16x8_t, o);
  };
  const float c2 = p.scale * 1.4426950408889634f;  // scores in log2 units
  int32_t knext = -1, vnext = -1;                  // the next block's pages
  if (first < nblk) {
    kload(kpg);
    vload(vpg);
    knext = page_of(first + STEP, n >> 2);
    vnext = page_of(first + STEP, g);
  }
  for (int blk = first; blk < nblk; blk += STEP) {
    const int lb = l0 + AF_BLK * blk;
    int at = lane;  // (not known to be the same in every round: the reads stay where they are)
    if constexpr (SHARED) asm volatile("" : "+v"(at));
    // whole (uniform): every row attends to all of it and its pages are in the cache
    const bool whole = lb + AF_BLK <= l1min && !__any(vpg < 0);
    const bool more = blk + STEP < nblk;  // uniform
    af32x4_t s[4][NQT];
    {
      const float sc = kv_pow2(kv_held(ksc));
#pragma unroll
      for (int t0 = 0; t0 < 4; t0 += 2) {  // two tiles at once: independent sums for the matrix cores
#pragma unroll
        for (int tt = t0; tt < t0 + 2; ++tt) {
          if constexpr (HD == 128) {  // whole rows into their lanes
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const uint32_t a = kr[tt][0][d], b = kr[tt][1][d], ao = other_of_pair(a), bo = other_of_pair(b);
              kr[tt][0][d] = odd ? bo : a;
              kr[tt][1][d] = odd ? b : ao;
            }
          }
#pragma unroll
          for (int nt = 0; nt < NQT; ++nt) s[tt][nt] = af32x4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int tt = t0; tt < t0 + 2; ++tt) {
            const au32x4_t x = kr[tt][ks / 2];
            const abf16x8_t a = operand(x[2 * (ks % 2)], x[2 * (ks % 2) + 1], sc);
#pragma unroll
            for (int nt = 0; nt < NQT; ++nt) {
              const abf16x8_t q = SHARED ? qs[SHARED ? ks : 0][SHARED ? nt : 0][at] : qop[ks][nt];
              s[tt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q, s[tt][nt], 0, 0, 0);
            }
          }
        __builtin_amdgcn_sched_barrier(0);  // (operands of all tiles at once would take their registers)
      }
    }
    if (more) {
      kload(knext);
      knext = page_of(blk + 2 * STEP, n >> 2);
    }
    // s[tt][nt][i]: position lb + 16 g + 4 tt + i (page g of the block), row 16 nt + n
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < NQT; ++nt)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (vpg < 0 || lb + 16 * g + 4 * tt + i >= l1[nt]) s[tt][nt][i] = -INFINITY;
    }
#pragma unroll
    for (int nt = 0; nt < NQT; ++nt) {
      float bm = -INFINITY;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) bm = fmaxf(bm, s[tt][nt][i]);
      bm = fmaxf(bm, __shfl_xor(bm, 16));
      bm = fmaxf(bm, __shfl_xor(bm, 32));
      const float mn = fmaxf(mrun[nt], bm * c2);  // (c2 > 0)
      const float msub = mn == -INFINITY ? 0.0f : mn;  // nothing but masks so far
      const float alpha = __builtin_amdgcn_exp2f(mrun[nt] - msub);
      float ls = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pe = __builtin_amdgcn_exp2f(fmaf(s[tt][nt][i], c2, -msub));
          s[tt][nt][i] = pe;
          ls += pe;
        }
      lrun[nt] = fmaf(lrun[nt], alpha, ls);  // this lane's positions only
      mrun[nt] = mn;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int e = 0; e < ET; ++e) acc[e][nt] *= alpha;
      }
    }
    if (!whole) {
      // bytes that no row attends to (of any content) become zeros, and so do NaN codes that
      // not all rows attend to: a weight of 0 would carry them into the others
      const int lp = lb + 16 * g;
      const int live = vpg >= 0 ? min(max(l1max - lp, 0), KV_PAGE) : 0, every = min(max(l1min - lp, 0), live);
      au32x4_t keep, some;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        keep[d] = low_bytes(live - 4 * d);
        some[d] = keep[d] & ~low_bytes(every - 4 * d);
      }
      uint32_t nans = 0;
#pragma unroll
      for (int e = 0; e < ET; ++e) {
        vr[e] &= keep;
#pragma unroll
        for (int d = 0; d < 4; ++d) nans |= nan_bytes(vr[e][d]) & some[d];
      }
      if (__any(nans)) {
        // the rows that attend to a dim's first such position get a NaN there themselves
#pragma unroll
        for (int e = 0; e < ET; ++e) {
          int nan = 0x7fffffff;  // of dim 16 e + n
#pragma unroll
          for (int d = 3; d >= 0; --d) {
            const uint32_t bad = nan_bytes(vr[e][d]) & some[d];
            if (bad) nan = lp + 4 * d + (__ffs(bad) - 1) / 8;
            vr[e][d] &= ~((bad >> 7) * 0xffu);
          }
          nan = min(nan, __shfl_xor(nan, 16));
          nan = min(nan, __shfl_xor(nan, 32));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int first = __shfl(nan, 4 * g + i);  // of acc's dim 16 e + 4 g + i
#pragma unroll
            for (int nt = 0; nt < NQT; ++nt)
              if (first < l1[nt]) acc[e][nt][i] = NAN;
          }
        }
      }
    }
    const float sc = kv_pow2(kv_held(vsc));
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // k-step u: positions 8 u .. 8 u + 7 of page g
      abf16x8_t ph[NQT], pl[NQT];
#pragma unroll
      for (int nt = 0; nt < NQT; ++nt) {
        au32x4_t hi, lo;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const float a = s[2 * u + d / 2][nt][2 * (d % 2)], b = s[2 * u + d / 2][nt][2 * (d % 2) + 1];
          hi[d] = pack_bf(a, b);
          lo[d] = pack_bf(a - lo_bf(hi[d]), b - hi_bf(hi[d]));
        }
        ph[nt] = __builtin_bit_cast(abf16x8_t, hi);
        pl[nt] = __builtin_bit_cast(abf16x8_t, lo);
      }
#pragma unroll
      for (int e0 = 0; e0 < ET; e0 += EG) {
        abf16x8_t a[EG];
#pragma unroll
        for (int e = 0; e < EG; ++e) a[e] = operand(vr[e0 + e][2 * u], vr[e0 + e][2 * u + 1], sc);
#pragma unroll
        for (int nt = 0; nt < NQT; ++nt) {
#pragma unroll
          for (int e = 0; e < EG; ++e)
            acc[e0 + e][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[e], ph[nt], acc[e0 + e][nt], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < EG; ++e)
            acc[e0 + e][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[e], pl[nt], acc[e0 + e][nt], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more) {
      vload(vnext);
      vpg = vnext;
      vnext = page_of(blk + 2 * STEP, g);
    }
  }

  // a row's max and sum, in all lanes (n, .) of it
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    lrun[nt] += __shfl_xor(lrun[nt], 16);
    lrun[nt] += __shfl_xor(lrun[nt], 32);
  }
  // where a row's dims go: the output (one chunk), or the chunk's part
  auto out_of = [&](const AttnRow &a) __attribute__((always_inline)) {
    return p.out + a.b * p.ob + a.i * p.ot + (static_cast<int64_t>(h) * p.group + a.j) * p.oh;
  };
  auto part_of = [&](const AttnRow &a) __attribute__((always_inline)) {
    const int64_t bi = static_cast<int64_t>(a.b) * p.n + a.i;
    return (bi * p.heads + static_cast<int64_t>(h) * p.group + a.j) * p.nchunk + c;
  };
  auto put = [&](bf16_t *to, af32x4_t o, float inv) __attribute__((always_inline)) {
    *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf(o[0] * inv, o[1] * inv), pack_bf(o[2] * inv, o[3] * inv));
  };
  auto inverse = [](float l) __attribute__((always_inline)) { return l != 0.0f ? 1.0f / l : 0.0f; };  // (NaN stays NaN)
  if constexpr (BY == BY_WAVE) {
#pragma unroll
    for (int nt = 0; nt < NQT; ++nt) {
      if (16 * nt + n >= nrow) continue;
      if (p.nchunk == 1) {
        bf16_t *to = out_of(rows[nt]) + 4 * g;
        const float inv = inverse(lrun[nt]);
#pragma unroll
        for (int e = 0; e < ET; ++e) put(to + 16 * e, acc[e][nt], inv);
      } else {
        const int64_t at = part_of(rows[nt]);
        float *to = p.part + at * HD + 4 * g;
#pragma unroll
        for (int e = 0; e < ET; ++e) *reinterpret_cast<af32x4_t *>(to + 16 * e) = acc[e][nt];
        if (g == 0) p.ml[at] = make_float2(mrun[nt], lrun[nt]);
      }
    }
  } else {  // the waves' (max, sum, o) meet
    __shared__ float wm[NW][ROWS], wl[NW][ROWS];
    __shared__ af32x4_t wo[NW][ROWS][HD / 4 + 1];  // (a row's padding parts the banks)
#pragma unroll
    for (int nt = 0; nt < NQT; ++nt) {
      const int r = 16 * nt + n;
      if (g == 0) {
        wm[wave][r] = mrun[nt];
        wl[wave][r] = lrun[nt];
      }
#pragma unroll
      for (int e = 0; e < ET; ++e) wo[wave][r][4 * e + g] = acc[e][nt];
    }
    __syncthreads();
    for (int x = t; x < nrow * (HD / 4); x += 64 * NW) {
      const int r = x / (HD / 4), d4 = x % (HD / 4);
      float M = wm[0][r];
#pragma unroll
      for (int k = 1; k < NW; ++k) M = fmaxf(M, wm[k][r]);
      float tot = 0.0f;
      af32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float f = wm[k][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm[k][r] - M);
        tot = fmaf(f, wl[k][r], tot);
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = fmaf(f, wo[k][r][d4][d], o[d]);
      }
      const AttnRow a = attn_row(p, r0 + r);
      if (p.nchunk == 1) {
        put(out_of(a) + 4 * d4, o, inverse(tot));
      } else {
        const int64_t at = part_of(a);
        *reinterpret_cast<af32x4_t *>(p.part + at * HD + 4 * d4) = o;
        if (d4 == 0) p.ml[at] = make_float2(M, tot);
      }
    }
  }
}

// Joins a query row's chunks, in a fixed order: weights 2^(max - all's max) of up to JN
// chunks at a time in LDS, then wave w sums chunks w, w + 4, ..
constexpr int JN = 256;

template <int HD>
__global__ __launch_bounds__(AF_T) void attn_fp8_join_kernel(AttnFp8Args p) {
  constexpr int DL = HD / 64;  // dims a lane
  __shared__ float f[JN], red[AF_NW], tots[AF_NW], os[AF_NW][HD];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, head = blockIdx.x;
  const int bi = blockIdx.y, b = bi / static_cast<int>(p.n), i = bi % static_cast<int>(p.n);
  const int len = row_len(p, AttnRow{b, i, 0});
  // chunks that reach below len: of the shared pages, and behind them
  const int nc = len <= p.shared ? (len + p.schunk - 1) / max(p.schunk, 1)
                                 : p.snum + (len - p.shared + p.chunk - 1) / p.chunk;
  const int64_t at = (static_cast<int64_t>(bi) * p.heads + head) * p.nchunk;
  float M = -INFINITY;
  for (int c = t; c < nc; c += AF_T) M = fmaxf(M, p.ml[at + c].x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
  if (lane == 0) red[wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float tot = 0.0f, o[DL] = {};
  for (int c0 = 0; c0 < nc; c0 += JN) {
    __syncthreads();
    if (c0 + t < nc) {
      const float2 ml = p.ml[at + c0 + t];
      const float x = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
      f[t] = x;
      tot = fmaf(x, ml.y, tot);
    }
    __syncthreads();
    const int n = min(JN, nc - c0);
#pragma unroll 4
    for (int c = wave; c < n; c += AF_NW) {
      const float x = f[c];
      const float *part = p.part + (at + c0 + c) * HD + DL * lane;
      if constexpr (DL == 2) {
        const float2 v = *reinterpret_cast<const float2 *>(part);
        o[0] = fmaf(x, v.x, o[0]);
        o[1] = fmaf(x, v.y, o[1]);
      } else {
        o[0] = fmaf(x, part[0], o[0]);
      }
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) tot += __shfl_xor(tot, d);
  if (lane == 0) tots[wave] = tot;
#pragma unroll
  for (int d = 0; d < DL; ++d) os[wave][DL * lane + d] = o[d];
  __syncthreads();
  if (t < HD) {
    const float sum = (tots[0] + tots[1]) + (tots[2] + tots[3]);
    const float v = (os[0][t] + os[1][t]) + (os[2][t] + os[3][t]);
    p.out[static_cast<int64_t>(b) * p.ob + i * p.ot + head * p.oh + t] = f2bf(sum != 0.0f ? v / sum : 0.0f);
  }
}

// Positions of a chunk (a multiple of `step`, at most `most`) for L positions of `units`
// (sequence, key head, row tile)s, `slots` chunks at once on the card.  Costs in positions
// of a chunk's own walk: its start and end are as long as AF_START of them, and each chunk
// costs the join AF_JOIN; the walk's time is between that of whole rounds of equal chunks
// and that of evenly spread work with half a chunk's tail, the mean is taken.  (64 sequences
// of 8192 positions, 32 heads: chunks of 4352 665 us, 2048 672, 1024 683, 512 704.)
constexpr int64_t AF_START = 128, AF_JOIN = 8;

// num chunks of a unit, `walked` positions of all units.
static int64_t cost_of(int64_t chunk, int64_t num, int64_t units, int64_t walked, int64_t slots) {
  const int64_t rounds = cdiv(units * num, slots) * (chunk + AF_START);
  const int64_t even = (walked + units * num * AF_START) / slots + chunk / 2;
  return rounds + (units * num > slots ? even : rounds);
}

static int chunk_for(int64_t L, int64_t units, int64_t slots, int64_t step, int64_t most, int64_t *least = nullptr) {
  int64_t best = 0, best_cost = 0;
  for (int64_t nc = 1, chunk = 0; chunk != step; nc += nc < 8 ? 1 : nc / 4) {
    chunk = cdiv(cdiv(L, nc), step) * step;
    if (chunk > most) continue;
    const int64_t num = cdiv(L, chunk);
    const int64_t cost = cost_of(chunk, num, units, units * L, slots) + AF_JOIN * num;
    if (!best || cost < best_cost) {
      best = chunk;
      best_cost = cost;
    }
  }
  if (least) *least = best_cost;
  return static_cast<int>(best);
}

// A workgroup alone may take this much longer (the join's launch), up to this many positions
// a wave (lengths differ: the longest sequence is the launch's tail).  Passes of a graph,
// a workgroup against chunks and their join, heads of 128: 8 sequences of 256 positions of 32
// heads 6.9 against 9.4 us, of 8192 86 against 89, one of 784 10.4 against 10.4 (by itself,
// where the host launches, 14.5 against 17.6), one of 2048 15 against 11; 8 of up to 8192,
// one as long, 70 against 66.
constexpr int64_t AF_SAVED = 64, AF_ALONE = 2048;

// The split of a call: shared positions, and chunks of them and of those behind.
//
// L is that of the table's columns: the host does not read the positions, and the workspace has
// to hold whatever they are.  A table far longer than its sequences makes chunks that few waves
// take (32 heads: 777 positions 10.4 us, in a table of 131072 positions 31; 8 sequences of 8192
// 91, there 129, in one of 2^20 324).  A caller who knows a bound passes the table's first
// columns.
struct AttnSplit {
  int shared, schunk, snum, chunk, nchunk;
  bool group;  // a workgroup takes all of a sequence's positions: no join
};
static AttnSplit split_for(int64_t B, int64_t n, int64_t heads, int64_t kv, int64_t max_pages, int64_t shared_pages) {
  const int64_t L = max_pages * KV_PAGE, shared = shared_pages * KV_PAGE, rows = n * (heads / kv);
  AttnSplit s{static_cast<int>(shared), 0, 0, AF_BLK, 0, false};
  if (shared) {  // of one length for all: as long as gives two workgroups a CU
    s.schunk = chunk_for(shared, kv * cdiv(B * rows, 32), 512, AF_BLK * AF_NW, int64_t(1) << 30);
    s.snum = static_cast<int>(cdiv(shared, s.schunk));
  }
  if (L > shared) {  // lengths differ: a long chunk would be the launch's tail
    const int64_t units = B * kv * cdiv(rows, 16);
    int64_t cost;
    s.chunk = chunk_for(L - shared, units, 2048, AF_BLK, 8192, &cost);
    // Without a join, a workgroup to all of a sequence's positions: where eight waves take
    // them as fast as chunks would be taken (short contexts, or as many workgroups as CUs).
    const int64_t c = cdiv(L, AF_BLK * AF_WAVES<BY_GROUP>) * AF_BLK;
    s.group = shared == 0 && s.chunk < L && c <= AF_ALONE && cost_of(c, 1, units, units * c, 256) <= cost + AF_SAVED;
    if (s.group) s.chunk = static_cast<int>(L);
  }
  s.nchunk = s.snum + static_cast<int>(cdiv(L - shared, s.chunk));
  return s;
}

static int64_t bytes_of(const AttnSplit &s, int64_t rows, int64_t hd) {  // parts, max and sum
  return s.nchunk == 1 ? 0 : rows * s.nchunk * (hd + 2) * static_cast<int64_t>(sizeof(float));
}

template <int HD>
static int launch_fp8(const AttnFp8Args &a, bool group, hipStream_t st) {
  const int64_t per = static_cast<int64_t>(a.n) * a.group, own = a.nchunk - a.snum;
  const int64_t tiles0 = cdiv(a.B * per, 32), tiles1 = cdiv(per, 16);
  const int64_t wgs0 = cdiv(static_cast<int64_t>(a.snum) * a.kv, 8) * 8 * tiles0;
  const int64_t wgs1 = cdiv(own * a.kv * a.B, group ? 8 : 8 * AF_NW) * 8 * tiles1;
  if (!grid_fits(wgs0, AF_T) || !grid_fits(wgs1, group ? 64 * AF_WAVES<BY_GROUP> : AF_T) || static_cast<int64_t>(a.B) * a.n > 65535)
    return fail(EVO2_ERR_UNSUPPORTED, "paged_decode_attention_fp8: more workgroups than a launch takes");
  if (wgs0) {
    hipLaunchKernelGGL((attn_fp8_kernel<HD, 2, SHARED_BY_GROUP>), dim3(static_cast<unsigned>(wgs0)), dim3(AF_T), 0, st, a,
                       static_cast<uint32_t>(tiles0));
    const int rc = check_launch("paged_decode_attention_fp8 shared chunks");
    if (rc) return rc;
  }
  if (wgs1) {
    if (group)
      hipLaunchKernelGGL((attn_fp8_kernel<HD, 1, BY_GROUP>), dim3(static_cast<unsigned>(wgs1)),
                         dim3(64 * AF_WAVES<BY_GROUP>), 0, st, a, static_cast<uint32_t>(tiles1));
    else
      hipLaunchKernelGGL((attn_fp8_kernel<HD, 1, BY_WAVE>), dim3(static_cast<unsigned>(wgs1)), dim3(AF_T), 0, st, a,
                         static_cast<uint32_t>(tiles1));
    const int rc = check_launch("paged_decode_attention_fp8 chunks");
    if (rc) return rc;
  }
  if (a.nchunk == 1) return EVO2_OK;
  hipLaunchKernelGGL(attn_fp8_join_kernel<HD>, dim3(a.heads, static_cast<unsigned>(a.B * a.n)), dim3(AF_T), 0, st, a);
  return check_launch("paged_decode_attention_fp8 join");
}

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_decode_attention_fp8_workspace_bytes(int64_t B, int64_t n, int64_t heads, int64_t kv_heads,
                                                             int64_t head_dim, int64_t max_pages,
                                                             int64_t shared_pages) {
  if (B <= 0 || n <= 0 || kv_heads <= 0 || heads < kv_heads || heads % kv_heads || head_dim <= 0 || max_pages <= 0 ||
      B > 65535 || n > 65535 || heads > 65535 || head_dim > 65535 || max_pages > (int64_t(1) << 26) ||
      shared_pages < 0 || shared_pages > max_pages)
    return 0;
  return bytes_of(split_for(B, n, heads, kv_heads, max_pages, shared_pages), B * n * heads, head_dim);
}

extern "C" int evo2_paged_decode_attention_fp8(const void *q, int64_t qb, int64_t qt, int64_t qh, const void *k_pages,
                                               int64_t kps, int64_t khs, const void *v_pages, int64_t vps, int64_t vhs,
                                               const float *k_scale, int64_t ksp, int64_t ksh, const float *v_scale,
                                               int64_t vsp, int64_t vsh, int64_t num_pages, const int32_t *table,
                                               int64_t st, int64_t max_pages, int64_t shared_pages,
                                               const int64_t *positions, void *workspace, int64_t workspace_bytes,
                                               void *out, int64_t ob, int64_t ot, int64_t oh, int64_t B, int64_t n,
                                               int64_t heads, int64_t kv_heads, int64_t head_dim, float scale,
                                               void *stream) {
  if (B < 0 || n < 0 || B > 65535 || n > 65535 || kv_heads <= 0 || heads <= 0 || heads > 65535 || heads % kv_heads ||
      shared_pages < 0 || shared_pages > max_pages)
    return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: bad sizes B=%lld n=%lld heads=%lld kv_heads=%lld "
                "shared_pages=%lld", (long long)B, (long long)n, (long long)heads, (long long)kv_heads,
                (long long)shared_pages);
  if (!(scale > 0.0f) || !(scale * 1.4426950408889634f < INFINITY))  // (the kernel's units)
    return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: the scale must be positive and finite");
  if (B == 0 || n == 0) return EVO2_OK;
  const KvPages c{static_cast<uint8_t *>(const_cast<void *>(k_pages)), kps, khs,
                  static_cast<uint8_t *>(const_cast<void *>(v_pages)), vps, vhs, const_cast<float *>(k_scale), ksp,
                  ksh, const_cast<float *>(v_scale), vsp, vsh, num_pages, table, st, max_pages};
  const int rc = kv_check(c, kv_heads, head_dim, false, "paged_decode_attention_fp8");
  if (rc) return rc;
  if (!q || !positions || !out) return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: null pointer argument");
  const AttnSplit sp = split_for(B, n, heads, kv_heads, max_pages, shared_pages);
  const int64_t need = bytes_of(sp, B * n * heads, head_dim);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: workspace too small");
  if (reinterpret_cast<uintptr_t>(q) % 16 || qb % 8 || qt % 8 || qh % 8 || reinterpret_cast<uintptr_t>(out) % 8 ||
      ob % 4 || ot % 4 || oh % 4 || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(EVO2_ERR_UNSUPPORTED, "paged_decode_attention_fp8: rows must be 16-byte aligned");
  float *part = static_cast<float *>(workspace);
  const AttnFp8Args a{c, static_cast<const bf16_t *>(q), qb, qt, qh, positions, part,
                      part ? reinterpret_cast<float2 *>(part + B * n * heads * sp.nchunk * head_dim) : nullptr,
                      static_cast<bf16_t *>(out), ob, ot, oh, scale, static_cast<uint32_t>(B), static_cast<uint32_t>(n),
                      static_cast<uint32_t>(heads), static_cast<uint32_t>(heads / kv_heads),
                      static_cast<uint32_t>(kv_heads),
                      sp.shared, sp.schunk, sp.snum, sp.chunk, sp.nchunk};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return head_dim == 64 ? launch_fp8<64>(a, sp.group, s) : launch_fp8<128>(a, sp.group, s);
}

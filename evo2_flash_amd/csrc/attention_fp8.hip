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
// Split over the context: a workgroup takes one chunk of positions of one key head for up
// to 16 query rows (a sequence's tokens x the head's group; on pages that all sequences
// share, up to 32 rows of any sequences), and writes (o, max, sum) for each; a second
// launch joins the chunks.  Contexts of one chunk are written out at once.  Each of the
// four waves takes the chunk's blocks of 64 positions in turn, with a running maximum and
// sum, on v_mfma_f32_16x16x32_bf16:
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
  float *part;                          // (B * n * heads, nchunk, hd + 2): o, max, sum
  bf16_t *out; int64_t ob, ot, oh;
  float scale;
  int B, n, heads, group, kv;           // group: query heads to a key head
  int chunk, nchunk;                    // positions a chunk; chunks of the table
};

constexpr int AF_T = 256, AF_NW = AF_T / 64;
constexpr int AF_BLK = 64;                    // positions a wave takes at once
constexpr int AF_CHUNK = 2048;                // most positions a chunk
constexpr int AF_PAGES = AF_CHUNK / KV_PAGE;

// Query row r of a key head: rows run over (sequence, token, head of the group).
struct AttnRow {
  int b, i, j;
};
__device__ __forceinline__ AttnRow attn_row(const AttnFp8Args &p, int64_t r) {
  const int per = p.n * p.group;
  const int b = static_cast<int>(r / per), in = static_cast<int>(r - static_cast<int64_t>(b) * per);
  return AttnRow{b, in / p.group, in % p.group};
}
__device__ __forceinline__ int row_len(const AttnFp8Args &p, const AttnRow &a) {
  const int64_t first = p.pos[a.b], all = p.c.max_pages * KV_PAGE;
  // (positions far off the table are clamped before the token is added)
  return static_cast<int>(min(max(min(first, all) + a.i + 1, int64_t(0)), all));
}

// Chunks c_first .. c_first + c_count - 1.  tiles: row tiles a (chunk, key head) has, per
// sequence (SHARED false) or in all (true).  Workgroups w of one XCD (w mod 8) take the
// tiles of a (chunk, head) one after the other, so its codes come from that XCD's L2.
template <int HD, int NQT, bool SHARED>
__global__ __launch_bounds__(AF_T, NQT == 2 ? 1 : 2) void attn_fp8_kernel(AttnFp8Args p, int c_first, int c_count, int tiles) {
  constexpr int KS = HD / 32;      // k-steps of a score
  constexpr int KH = HD / 64;      // 16-byte loads a position and lane
  constexpr int ET = HD / 16;      // dim tiles
  constexpr int ROWS = 16 * NQT;
  __shared__ int32_t pages[AF_PAGES];
  __shared__ float sk[AF_PAGES], sv[AF_PAGES];
  __shared__ float wm[AF_NW][ROWS], wl[AF_NW][ROWS];
  __shared__ float4 wo[AF_NW][ROWS][HD / 4 + 1];  // a wave's o (a row's padding parts the banks)
  const int w = blockIdx.x, j8 = w >> 3;
  const int64_t pair = static_cast<int64_t>(j8 / tiles) * 8 + (w & 7);
  const int tile = j8 % tiles;
  const int h = static_cast<int>(pair % p.kv);
  const int64_t rest = pair / p.kv;
  const int c = c_first + static_cast<int>(rest % c_count);
  const int64_t seq = rest / c_count;
  if (seq >= (SHARED ? 1 : p.B)) return;  // uniform: the grid's padding
  const int64_t per = static_cast<int64_t>(p.n) * p.group;
  const int64_t r0 = (SHARED ? 0 : seq * per) + static_cast<int64_t>(ROWS) * tile;
  const int nrow = static_cast<int>(min(static_cast<int64_t>(ROWS), (SHARED ? p.B * per : (seq + 1) * per) - r0));
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int l0 = c * p.chunk;
  // ends of this lane's rows, of the positions any row attends to and that all do
  int l1[NQT], l1max = l0, l1min = l0 + p.chunk;
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    const bool live = 16 * nt + n < nrow;
    l1[nt] = live ? min(l0 + p.chunk, row_len(p, attn_row(p, r0 + 16 * nt + n))) : l0;
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
  // the chunk's pages below l1max (-1: left out) and their scales
  const int32_t *row = p.c.table + (SHARED ? 0 : seq) * p.c.st;
  for (int i = t; i < p.chunk / KV_PAGE; i += AF_T) {
    int32_t pg = -1;
    float a = 0.0f, b = 0.0f;
    if (l0 + KV_PAGE * i < l1max) {
      pg = row[l0 / KV_PAGE + i];
      if (pg < 0 || pg >= p.c.num_pages) pg = -1;
    }
    if (pg >= 0) {
      a = kv_pow2(kv_held(p.c.ks[pg * p.c.ksp + h * p.c.ksh]));
      b = kv_pow2(kv_held(p.c.vs[pg * p.c.vsp + h * p.c.vsh]));
    }
    pages[i] = pg;
    sk[i] = a;
    sv[i] = b;
  }
  // Q as the B operand: k-slot (g, j) of k-step 2 hf + u is dim 64 hf + 16 g + 8 u + j
  abf16x8_t qop[KS][NQT];
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    const bool live = 16 * nt + n < nrow;
    const AttnRow a = attn_row(p, live ? r0 + 16 * nt + n : r0);
    const bf16_t *qr = p.q + a.b * p.qb + a.i * p.qt + (static_cast<int64_t>(h) * p.group + a.j) * p.qh + 16 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      au32x4_t x = *reinterpret_cast<const au32x4_t *>(qr + 64 * (ks / 2) + 8 * (ks % 2));
      if (!live) x = au32x4_t{0, 0, 0, 0};
      qop[ks][nt] = __builtin_bit_cast(abf16x8_t, x);
    }
  }
  __syncthreads();

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
  // (a page left out reads page 0: its scores are masked, its values set to zero)
  au32x4_t kr[4][KH], vr[ET];
  auto kload = [&](int blk) __attribute__((always_inline)) {
    const int64_t pg = max(pages[4 * blk + (n >> 2)], 0);
    const uint8_t *a = p.c.k + pg * p.c.kp + h * p.c.kh + (n & 3) * HD + 16 * g;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int hf = 0; hf < KH; ++hf) kr[tt][hf] = *reinterpret_cast<const au32x4_t *>(a + 4 * tt * HD + 64 * hf);
  };
  auto vload = [&](int blk) __attribute__((always_inline)) {
    const int64_t pg = max(pages[4 * blk + g], 0);
    const uint8_t *a = p.c.v + pg * p.c.vp + h * p.c.vh + 16 * n;
#pragma unroll
    for (int e = 0; e < ET; ++e) vr[e] = *reinterpret_cast<const au32x4_t *>(a + 256 * e);
  };
  // eight codes (two dwords) as a bf16 operand
  auto operand = [&](uint32_t a, uint32_t b, float s) __attribute__((always_inline)) {
    const au32x4_t o = {kv_decode2<false>(a, s), kv_decode2<true>(a, s), kv_decode2<false>(b, s), kv_decode2<true>(b, s)};
    return __builtin_bit_cast(abf16x8_t, o);
  };
  const float c2 = p.scale * 1.4426950408889634f;  // scores in log2 units
  auto block = [&](int blk, auto mask_c) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_c)::value;
    const int lb = l0 + AF_BLK * blk;
    const bool more = blk + AF_NW < nblk;  // uniform
    af32x4_t s[4][NQT];
    {
      const float ksc = sk[4 * blk + (n >> 2)];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
        for (int nt = 0; nt < NQT; ++nt) s[tt][nt] = af32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const au32x4_t x = kr[tt][ks / 2];
          const abf16x8_t a = operand(x[2 * (ks % 2)], x[2 * (ks % 2) + 1], ksc);
#pragma unroll
          for (int nt = 0; nt < NQT; ++nt)
            s[tt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qop[ks][nt], s[tt][nt], 0, 0, 0);
        }
      }
    }
    if (more) kload(blk + AF_NW);
    // s[tt][nt][i]: position lb + 16 g + 4 tt + i (page g of the block), row 16 nt + n
    const bool held = !MASK || pages[4 * blk + g] >= 0;
#pragma unroll
    for (int nt = 0; nt < NQT; ++nt) {
      float bm = -INFINITY;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = s[tt][nt][i] * c2;
          if constexpr (MASK) v = held && lb + 16 * g + 4 * tt + i < l1[nt] ? v : -INFINITY;
          s[tt][nt][i] = v;
          bm = fmaxf(bm, v);
        }
      bm = fmaxf(bm, __shfl_xor(bm, 16));
      bm = fmaxf(bm, __shfl_xor(bm, 32));
      const float mn = fmaxf(mrun[nt], bm);
      const float msub = mn == -INFINITY ? 0.0f : mn;  // nothing but masks so far
      const float alpha = __builtin_amdgcn_exp2f(mrun[nt] - msub);
      float ls = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pe = __builtin_amdgcn_exp2f(s[tt][nt][i] - msub);
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
    const float vsc = sv[4 * blk + g];
    if constexpr (MASK) {  // bytes that no query attends to (of any content) become zeros
      const int live = held ? min(max(l1max - lb - 16 * g, 0), KV_PAGE) : 0;
      au32x4_t keep;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int k = live - 4 * d;
        keep[d] = k <= 0 ? 0u : k >= 4 ? 0xffffffffu : (1u << (8 * k)) - 1;
      }
#pragma unroll
      for (int e = 0; e < ET; ++e) vr[e] &= keep;
    }
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
      for (int e = 0; e < ET; ++e) {
        const abf16x8_t a = operand(vr[e][2 * u], vr[e][2 * u + 1], vsc);
#pragma unroll
        for (int nt = 0; nt < NQT; ++nt) {
          acc[e][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, ph[nt], acc[e][nt], 0, 0, 0);
          acc[e][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pl[nt], acc[e][nt], 0, 0, 0);
        }
      }
    }
    if (more) vload(blk + AF_NW);
  };
  if (wave < nblk) {
    kload(wave);
    vload(wave);
  }
  for (int blk = wave; blk < nblk; blk += AF_NW) {
    // whole: every row attends to all of it and its pages are in the cache
    const int end = l0 + AF_BLK * (blk + 1);
    const bool whole = end <= l1min && !__any(pages[4 * blk + g] < 0);
    if (whole) block(blk, std::false_type{});
    else block(blk, std::true_type{});
  }

  // the waves' (max, sum, o) meet
#pragma unroll
  for (int nt = 0; nt < NQT; ++nt) {
    float l = lrun[nt];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = 16 * nt + n;
    if (g == 0) {
      wm[wave][r] = mrun[nt];
      wl[wave][r] = l;
    }
#pragma unroll
    for (int e = 0; e < ET; ++e)
      wo[wave][r][4 * e + g] = make_float4(acc[e][nt][0], acc[e][nt][1], acc[e][nt][2], acc[e][nt][3]);
  }
  __syncthreads();
  for (int x = t; x < nrow * (HD / 4); x += AF_T) {
    const int r = x / (HD / 4), d4 = x % (HD / 4);
    float M = wm[0][r];
#pragma unroll
    for (int k = 1; k < AF_NW; ++k) M = fmaxf(M, wm[k][r]);
    float tot = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < AF_NW; ++k) {
      const float f = wm[k][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm[k][r] - M);
      const float4 a = wo[k][r][d4];
      tot = fmaf(f, wl[k][r], tot);
      o.x = fmaf(f, a.x, o.x); o.y = fmaf(f, a.y, o.y); o.z = fmaf(f, a.z, o.z); o.w = fmaf(f, a.w, o.w);
    }
    const AttnRow a = attn_row(p, r0 + r);
    const int64_t head = static_cast<int64_t>(h) * p.group + a.j;
    if (p.nchunk == 1) {
      const float inv = tot != 0.0f ? 1.0f / tot : 0.0f;  // (a NaN sum stays NaN)
      uint2 y = make_uint2(pack_bf(o.x * inv, o.y * inv), pack_bf(o.z * inv, o.w * inv));
      *reinterpret_cast<uint2 *>(p.out + a.b * p.ob + a.i * p.ot + head * p.oh + 4 * d4) = y;
    } else {
      float *part = p.part + (((static_cast<int64_t>(a.b) * p.n + a.i) * p.heads + head) * p.nchunk + c) * (HD + 2);
      *reinterpret_cast<float2 *>(part + 4 * d4) = make_float2(o.x, o.y);
      *reinterpret_cast<float2 *>(part + 4 * d4 + 2) = make_float2(o.z, o.w);
      if (d4 == 0) *reinterpret_cast<float2 *>(part + HD) = make_float2(M, tot);
    }
  }
}

// Joins a query row's chunks: HD lanes, in chunk order.
template <int HD>
__global__ __launch_bounds__(HD) void attn_fp8_join_kernel(AttnFp8Args p) {
  const int d = threadIdx.x, head = blockIdx.x;
  const int bi = blockIdx.y, b = bi / p.n, i = bi % p.n;
  const int nc = (row_len(p, AttnRow{b, i, 0}) + p.chunk - 1) / p.chunk;
  const float *part = p.part + (static_cast<int64_t>(bi) * p.heads + head) * p.nchunk * (HD + 2);
  float M = -INFINITY;
#pragma unroll 8
  for (int c = 0; c < nc; ++c) M = fmaxf(M, part[c * (HD + 2) + HD]);
  float tot = 0.0f, o = 0.0f;
#pragma unroll 8
  for (int c = 0; c < nc; ++c) {
    const float mc = part[c * (HD + 2) + HD];
    const float f = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - M);
    tot = fmaf(f, part[c * (HD + 2) + HD + 1], tot);
    o = fmaf(f, part[c * (HD + 2) + d], o);
  }
  p.out[static_cast<int64_t>(b) * p.ob + i * p.ot + head * p.oh + d] = f2bf(tot != 0.0f ? o / tot : 0.0f);
}

// Positions a chunk takes: as many workgroups as keep the card's loads in flight
// (AF_GROUPS), in chunks of 256 (a block for each wave) to AF_CHUNK positions.
constexpr int64_t AF_GROUPS = 1024;

static int chunk_for(int64_t B, int64_t n, int64_t heads, int64_t kv, int64_t max_pages) {
  const int64_t L = max_pages * KV_PAGE, rows = n * (heads / kv);
  const int64_t units = B * kv * cdiv(rows, 16);
  const int64_t want = cdiv(AF_GROUPS, units);  // chunks a unit
  const int64_t chunk = cdiv(cdiv(L, want), 256) * 256;
  return static_cast<int>(chunk < AF_CHUNK ? chunk : AF_CHUNK);
}

template <int HD>
static int launch_fp8(const AttnFp8Args &a, int shared_chunks, hipStream_t st) {
  const int64_t per = static_cast<int64_t>(a.n) * a.group;
  const int64_t own = a.nchunk - shared_chunks;
  const int64_t tiles0 = cdiv(a.B * per, 32), tiles1 = cdiv(per, 16);
  const int64_t wgs0 = cdiv(static_cast<int64_t>(shared_chunks) * a.kv, 8) * 8 * tiles0;
  const int64_t wgs1 = cdiv(own * a.kv * a.B, 8) * 8 * tiles1;
  if (!grid_fits(wgs0, AF_T) || !grid_fits(wgs1, AF_T) || static_cast<int64_t>(a.B) * a.n > 65535)
    return fail(EVO2_ERR_UNSUPPORTED, "paged_decode_attention_fp8: more workgroups than a launch takes");
  if (shared_chunks > 0) {
    hipLaunchKernelGGL((attn_fp8_kernel<HD, 2, true>), dim3(static_cast<unsigned>(wgs0)), dim3(AF_T), 0, st, a, 0,
                       shared_chunks, static_cast<int>(tiles0));
    const int rc = check_launch("paged_decode_attention_fp8 shared chunks");
    if (rc) return rc;
  }
  if (own > 0) {
    hipLaunchKernelGGL((attn_fp8_kernel<HD, 1, false>), dim3(static_cast<unsigned>(wgs1)), dim3(AF_T), 0, st, a,
                       shared_chunks, static_cast<int>(own), static_cast<int>(tiles1));
    const int rc = check_launch("paged_decode_attention_fp8 chunks");
    if (rc) return rc;
  }
  if (a.nchunk == 1) return EVO2_OK;
  hipLaunchKernelGGL(attn_fp8_join_kernel<HD>, dim3(a.heads, static_cast<unsigned>(a.B * a.n)), dim3(HD), 0, st, a);
  return check_launch("paged_decode_attention_fp8 join");
}

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_decode_attention_fp8_workspace_bytes(int64_t B, int64_t n, int64_t heads, int64_t kv_heads,
                                                             int64_t head_dim, int64_t max_pages) {
  if (B <= 0 || n <= 0 || kv_heads <= 0 || heads < kv_heads || heads % kv_heads || head_dim <= 0 || max_pages <= 0 ||
      B > 65535 || n > 65535 || heads > 65535 || head_dim > 65535 || max_pages > (int64_t(1) << 26))
    return 0;
  const int64_t nchunk = cdiv(max_pages * KV_PAGE, chunk_for(B, n, heads, kv_heads, max_pages));
  return nchunk == 1 ? 0 : B * n * heads * nchunk * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
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
  if (!(scale > 0.0f) || scale > 3.0e38f)
    return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: the scale must be positive and finite");
  if (B == 0 || n == 0) return EVO2_OK;
  const KvPages c{static_cast<uint8_t *>(const_cast<void *>(k_pages)), kps, khs,
                  static_cast<uint8_t *>(const_cast<void *>(v_pages)), vps, vhs, const_cast<float *>(k_scale), ksp,
                  ksh, const_cast<float *>(v_scale), vsp, vsh, num_pages, table, st, max_pages};
  const int rc = kv_check(c, kv_heads, head_dim, "paged_decode_attention_fp8");
  if (rc) return rc;
  if (!q || !positions || !out) return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: null pointer argument");
  const int64_t need = evo2_decode_attention_fp8_workspace_bytes(B, n, heads, kv_heads, head_dim, max_pages);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(EVO2_ERR_INVALID, "paged_decode_attention_fp8: workspace too small");
  if (reinterpret_cast<uintptr_t>(q) % 16 || qb % 8 || qt % 8 || qh % 8 || reinterpret_cast<uintptr_t>(out) % 8 ||
      ob % 4 || ot % 4 || oh % 4 || reinterpret_cast<uintptr_t>(workspace) % 8)
    return fail(EVO2_ERR_UNSUPPORTED, "paged_decode_attention_fp8: rows must be 16-byte aligned");
  const int chunk = chunk_for(B, n, heads, kv_heads, max_pages);
  const AttnFp8Args a{c, static_cast<const bf16_t *>(q), qb, qt, qh, positions, static_cast<float *>(workspace),
                      static_cast<bf16_t *>(out), ob, ot, oh, scale, static_cast<int>(B), static_cast<int>(n),
                      static_cast<int>(heads), static_cast<int>(heads / kv_heads), static_cast<int>(kv_heads), chunk,
                      static_cast<int>(cdiv(max_pages * KV_PAGE, chunk))};
  const int shared_chunks = static_cast<int>(shared_pages * KV_PAGE / chunk);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return head_dim == 64 ? launch_fp8<64>(a, shared_chunks, s) : launch_fp8<128>(a, shared_chunks, s);
}

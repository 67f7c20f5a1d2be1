// Writing tokens into the 8-bit KV cache (kv_fp8.h) and reading positions back, for the
// decoder's paged cache (model.py:104-153), and the decode step's rotary with the write of
// its one token.
//
// Write: sequence b's tokens i < lengths[b] go to positions positions[b] + i.  A page's
// scale is that of its tokens; a page that holds tokens already (its first one of this
// write is not the page's first position) keeps its scale, or re-encodes what it holds
// where a new token is larger.  Codes of positions that are not written stay as they are.
//
// A wave takes one page of one key head, keys and values in workgroups of their own: it
// reads the page's new tokens once (4 KB at head_dim 128), reduces their magnitude across
// its lanes and writes the codes.  Keys: 16 bytes in, eight codes out a lane, whole rows
// of a position.  Values: a lane has two dims of every position, so the transposition is
// four byte permutes a dim pair and four positions, and a lane's codes are one 16-byte
// store a dim.  Bound by memory, each byte moving once: 32768 tokens of 32 heads of 128, 805 MB
// each way, written in 160 us and read back in 136 (together 5.4 TB/s; a plain copy 5.1).
// Non-temporal loads of the tokens moved 25 us from the write to the read after it.
#include "kv_fp8.h"

#pragma clang fp contract(off)

namespace evo2 {

struct KvTokens {
  const bf16_t *k; int64_t kb, kt, kh;  // (B, n, heads, hd); batch, token and head strides
  const bf16_t *v; int64_t vb, vt, vh;
  const int64_t *positions;             // (B,) of token 0
  const int64_t *lengths;               // (B,) tokens that count, or NULL: n
  int64_t n;
  int heads;
};

constexpr int KV_WAVES = 4;

// The page of this wave's work: column col of sequence b's table row; false where the
// write does not reach it or the table has no page there.  [lo, hi): its new positions.
struct KvSpan {
  int64_t page, first;  // page; token at the page's position 0 (negative: held before)
  int lo, hi;
};
__device__ __forceinline__ bool kv_span(const KvPages &c, const int64_t *positions, const int64_t *lengths,
                                        int64_t n, int b, int64_t step, KvSpan &s) {
  const int64_t start = positions[b];
  int64_t count = n;
  if (lengths) count = min(max(lengths[b], int64_t(0)), n);
  if (start < 0 || start >= c.max_pages * KV_PAGE) return false;
  const int64_t col = start / KV_PAGE + step;
  if (col >= c.max_pages) return false;
  s.first = col * KV_PAGE - start;
  s.lo = static_cast<int>(max(-s.first, int64_t(0)));  // (only the first column's)
  s.hi = static_cast<int>(min(max(count - s.first, int64_t(0)), int64_t(KV_PAGE)));
  if (s.hi <= s.lo) return false;
  s.page = c.table[b * c.st + col];
  return s.page >= 0 && s.page < c.num_pages;
}

template <int HD>
__global__ __launch_bounds__(64 * KV_WAVES) void kv_write_kernel(KvPages c, KvTokens t) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int groups = (t.heads + KV_WAVES - 1) / KV_WAVES;
  const int64_t step = blockIdx.x / groups;
  const int h = (blockIdx.x % groups) * KV_WAVES + wave, b = blockIdx.y;
  KvSpan s;
  if (h >= t.heads || !kv_span(c, t.positions, t.lengths, t.n, b, step, s)) return;
  if (blockIdx.z == 0) {
    // keys: round j, lane: position (64 j + lane) / (HD / 8), eight dims
    constexpr int LPR = HD / 8, ROUNDS = HD / 32;
    const bf16_t *src = t.k + b * t.kb + h * t.kh;
    uint8_t *dst = c.k + s.page * c.kp + h * c.kh;
    float *scale = c.ks + s.page * c.ksp + h * c.ksh;
    uint4 x[ROUNDS];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const int row = (64 * j + lane) / LPR, d = 8 * (lane % LPR);
      x[j] = make_uint4(0, 0, 0, 0);
      if (row >= s.lo && row < s.hi) x[j] = *reinterpret_cast<const uint4 *>(src + (s.first + row) * t.kt + d);
      amax = kv_amax2(kv_amax2(kv_amax2(kv_amax2(amax, x[j].x), x[j].y), x[j].z), x[j].w);
    }
    int e = kv_exponent(kv_wave_max(amax));
    float f = 1.0f;
    if (s.lo > 0) {
      const int held = kv_held(*scale);
      f = kv_pow2(-min(max(e - held, 0), 60));
      e = max(e, held);
    }
    const float inv = kv_pow2(-e);
    const bool top = e == KV_EMAX;
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const int row = (64 * j + lane) / LPR;
      uint2 *o = reinterpret_cast<uint2 *>(dst + 512 * j + 8 * lane);
      if (row >= s.lo && row < s.hi) {
        uint2 w;
        w.x = kv_encode2<false>(lo_bf(x[j].x), hi_bf(x[j].x), inv, top, 0);
        w.x = kv_encode2<true>(lo_bf(x[j].y), hi_bf(x[j].y), inv, top, w.x);
        w.y = kv_encode2<false>(lo_bf(x[j].z), hi_bf(x[j].z), inv, top, 0);
        w.y = kv_encode2<true>(lo_bf(x[j].w), hi_bf(x[j].w), inv, top, w.y);
        *o = w;
      } else if (row < s.lo && f != 1.0f) {
        const uint2 w = *o;
        *o = make_uint2(kv_recode4(w.x, f), kv_recode4(w.y, f));
      }
    }
    if (lane == 0) *scale = kv_pow2(e);
  } else {
    // values: a lane has dims 2 p, 2 p + 1 of TPL positions (all 16 at HD 128, half of
    // them at 64)
    constexpr int PAIRS = HD / 2, TPL = 16 * PAIRS / 64;
    const int p = lane % PAIRS, t0 = (lane / PAIRS) * TPL;
    const bf16_t *src = t.v + b * t.vb + h * t.vh + 2 * p;
    uint8_t *dst = c.v + s.page * c.vp + h * c.vh + 32 * p + t0;
    float *scale = c.vs + s.page * c.vsp + h * c.vsh;
    uint32_t x[TPL];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const int row = t0 + i;
      x[i] = 0;
      if (row >= s.lo && row < s.hi) x[i] = *reinterpret_cast<const uint32_t *>(src + (s.first + row) * t.vt);
    }
#pragma unroll
    for (int i = 0; i < TPL; ++i) amax = kv_amax2(amax, x[i]);
    int e = kv_exponent(kv_wave_max(amax));
    float f = 1.0f;
    if (s.lo > 0) {
      const int held = kv_held(*scale);
      f = kv_pow2(-min(max(e - held, 0), 60));
      e = max(e, held);
    }
    const float inv = kv_pow2(-e);
    const bool top = e == KV_EMAX, whole = s.lo == 0 && s.hi == KV_PAGE;
    // w[d][i]: codes of dim 2 p + d, positions t0 + 4 i .. + 3
    uint32_t w[2][TPL / 4];
#pragma unroll
    for (int i = 0; i < TPL / 4; ++i) {
      uint32_t a = kv_encode2<false>(lo_bf(x[4 * i]), hi_bf(x[4 * i]), inv, top, 0);
      a = kv_encode2<true>(lo_bf(x[4 * i + 1]), hi_bf(x[4 * i + 1]), inv, top, a);
      uint32_t q = kv_encode2<false>(lo_bf(x[4 * i + 2]), hi_bf(x[4 * i + 2]), inv, top, 0);
      q = kv_encode2<true>(lo_bf(x[4 * i + 3]), hi_bf(x[4 * i + 3]), inv, top, q);
      w[0][i] = __builtin_amdgcn_perm(q, a, 0x06040200u);
      w[1][i] = __builtin_amdgcn_perm(q, a, 0x07050301u);
    }
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      uint32_t *o = reinterpret_cast<uint32_t *>(dst + 16 * d);
      if (!whole) {
#pragma unroll
        for (int i = 0; i < TPL / 4; ++i) {
          // bytes of positions held before (re-encoded), new ones, and ones behind
          const uint32_t was = o[i];
          const int lo = s.lo - t0 - 4 * i, hi = s.hi - t0 - 4 * i;
          const uint32_t below = lo <= 0 ? 0u : lo >= 4 ? 0xffffffffu : (1u << (8 * lo)) - 1;
          const uint32_t upto = hi <= 0 ? 0u : hi >= 4 ? 0xffffffffu : (1u << (8 * hi)) - 1;
          const uint32_t kept = f != 1.0f ? kv_recode4(was, f) : was;
          w[d][i] = (kept & below) | (w[d][i] & upto & ~below) | (was & ~upto);
        }
      }
      if constexpr (TPL == 16)
        *reinterpret_cast<uint4 *>(o) = make_uint4(w[d][0], w[d][1], w[d][2], w[d][3]);
      else
        *reinterpret_cast<uint2 *>(o) = make_uint2(w[d][0], w[d][1]);
    }
    if (lane == 0) *scale = kv_pow2(e);
  }
}

struct KvOut {
  bf16_t *k, *v;           // (B, L, heads, hd) contiguous
  const int64_t *lengths;  // (B,) positions that are held
  int64_t L;
  int heads;
};

// Read: positions below lengths[b] as bf16, token-major; zeros from there to L and where
// the table has no page.  The mapping of lanes is the write's.
template <int HD>
__global__ __launch_bounds__(64 * KV_WAVES) void kv_read_kernel(KvPages c, KvOut r) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int groups = (r.heads + KV_WAVES - 1) / KV_WAVES;
  const int64_t col = blockIdx.x / groups;
  const int h = (blockIdx.x % groups) * KV_WAVES + wave, b = blockIdx.y;
  if (h >= r.heads) return;
  const int64_t len = min(max(r.lengths[b], int64_t(0)), r.L), p0 = col * KV_PAGE;
  const int rows = static_cast<int>(min(r.L - p0, int64_t(KV_PAGE)));
  int held = static_cast<int>(min(max(len - p0, int64_t(0)), int64_t(KV_PAGE)));
  int64_t page = held > 0 && col < c.max_pages ? c.table[b * c.st + col] : -1;
  if (page < 0 || page >= c.num_pages) {
    page = 0;
    held = 0;
  }
  const int64_t stride = static_cast<int64_t>(r.heads) * HD;  // between positions
  const int64_t at = (b * r.L + p0) * stride + static_cast<int64_t>(h) * HD;
  if (blockIdx.z == 0) {
    constexpr int LPR = HD / 8, ROUNDS = HD / 32;
    const uint8_t *src = c.k + page * c.kp + h * c.kh;
    uint2 w[ROUNDS];
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j)
      w[j] = (64 * j + lane) / LPR < held ? *reinterpret_cast<const uint2 *>(src + 512 * j + 8 * lane) : make_uint2(0, 0);
    const float scale = kv_pow2(kv_held(c.ks[page * c.ksp + h * c.ksh]));
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
      const int row = (64 * j + lane) / LPR, d = 8 * (lane % LPR);
      if (row < rows)
        *reinterpret_cast<uint4 *>(r.k + at + row * stride + d) =
            make_uint4(kv_decode2<false>(w[j].x, scale), kv_decode2<true>(w[j].x, scale),
                       kv_decode2<false>(w[j].y, scale), kv_decode2<true>(w[j].y, scale));
    }
  } else {
    constexpr int PAIRS = HD / 2, TPL = 16 * PAIRS / 64;
    const int p = lane % PAIRS, t0 = (lane / PAIRS) * TPL;
    const uint8_t *src = c.v + page * c.vp + h * c.vh + 32 * p + t0;
    const float scale = kv_pow2(kv_held(c.vs[page * c.vsp + h * c.vsh]));
    uint32_t w[2][TPL / 4];
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      if constexpr (TPL == 16)
        *reinterpret_cast<uint4 *>(w[d]) = *reinterpret_cast<const uint4 *>(src + 16 * d);
      else
        *reinterpret_cast<uint2 *>(w[d]) = *reinterpret_cast<const uint2 *>(src + 16 * d);
    }
    uint32_t *o = reinterpret_cast<uint32_t *>(r.v + at + t0 * stride + 2 * p);
#pragma unroll
    for (int i = 0; i < TPL / 4; ++i) {
      const uint32_t a = __builtin_amdgcn_perm(w[1][i], w[0][i], 0x05010400u);  // (d0, d1) of two positions
      const uint32_t q = __builtin_amdgcn_perm(w[1][i], w[0][i], 0x07030602u);
      const uint32_t y[4] = {kv_decode2<false>(a, scale), kv_decode2<true>(a, scale), kv_decode2<false>(q, scale),
                             kv_decode2<true>(q, scale)};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = t0 + 4 * i + u;
        if (row < rows) o[(4 * i + u) * (stride / 2)] = row < held ? y[u] : 0u;
      }
    }
  }
}

// The decode step between the qkv projection and the attention: neox rotary of q and k
// (each product and sum rounded by itself, the bits of rotary_decode_kernel) and the
// write of k and v.  A wave takes one head of one sequence, lane f dims f and f + HD / 2.
// Latency only: 32 heads of 128, 8 sequences 4.6-5.1 us and 64 of them 4.8-5.5 (the bytes,
// 2.6 MB, 0.5; with bf16 pages 4.5-4.8 and 6.0).
struct KvRotary {
  const bf16_t *qkv; int64_t sqkv;  // rows (q | k | v), each heads * HD
  const float *inv_freq;
  float factor;
  bf16_t *q;                        // (B, heads, HD)
  const int64_t *positions;
  int heads;
};

template <int HD>
__global__ __launch_bounds__(64 * KV_WAVES) void kv_rotary_decode_kernel(KvPages c, KvRotary t) {
  constexpr int HALF = HD / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.x * KV_WAVES + wave, b = blockIdx.y;
  if (h >= t.heads) return;
  const int f = lane % HALF;
  const bool mine = lane < HALF;  // at HD 64 the upper lanes repeat the lower ones' work
  const int64_t pos = t.positions[b], hs = static_cast<int64_t>(t.heads) * HD;
  const bf16_t *r = t.qkv + b * t.sqkv + h * HD + f;
  float sn, cs;
  sincosf((static_cast<float>(pos) / t.factor) * t.inv_freq[f], &sn, &cs);
  const float q1 = bf2f(r[0]), q2 = bf2f(r[HALF]), k1 = bf2f(r[hs]), k2 = bf2f(r[hs + HALF]);
  if (mine) {
    bf16_t *qo = t.q + b * hs + h * HD + f;
    qo[0] = f2bf(q1 * cs - q2 * sn);
    qo[HALF] = f2bf(q2 * cs + q1 * sn);
  }
  KvSpan s;
  if (!kv_span(c, t.positions, nullptr, 1, b, 0, s)) return;
  const int off = s.lo;
#pragma unroll
  for (int side = 0; side < 2; ++side) {  // keys, values
    const uint32_t x = side == 0 ? pack_bf(k1 * cs - k2 * sn, k2 * cs + k1 * sn) : pair_bf(r[2 * hs], r[2 * hs + HALF]);
    uint8_t *page = side == 0 ? c.k + s.page * c.kp + h * c.kh : c.v + s.page * c.vp + h * c.vh;
    float *scale = side == 0 ? c.ks + s.page * c.ksp + h * c.ksh : c.vs + s.page * c.vsp + h * c.vsh;
    int e = kv_exponent(kv_wave_max(kv_amax2(0, x)));
    int drop = 0;
    if (off > 0) {
      const int held = kv_held(*scale);
      drop = max(e - held, 0);
      e = max(e, held);
    }
    if (drop) {  // the page's tokens so far, in dwords of codes
      const float w = kv_pow2(-min(drop, 60));
      uint32_t *o = reinterpret_cast<uint32_t *>(page);
      if (side == 0) {
        for (int i = lane; i < off * HD / 4; i += 64) o[i] = kv_recode4(o[i], w);
      } else {
        for (int i = lane; i < HD * KV_PAGE / 4; i += 64) {
          const int lo = off - 4 * (i & 3);
          const uint32_t below = lo <= 0 ? 0u : lo >= 4 ? 0xffffffffu : (1u << (8 * lo)) - 1, was = o[i];
          o[i] = (kv_recode4(was, w) & below) | (was & ~below);
        }
      }
      // the new token's bytes lie in dwords that another lane of this wave rewrote
      __threadfence_block();
    }
    const uint32_t code = kv_encode2<false>(lo_bf(x), hi_bf(x), kv_pow2(-e), e == KV_EMAX, 0);
    if (mine) {
      const int unit = side == 0 ? 1 : KV_PAGE, at = side == 0 ? off * HD : off;
      page[at + f * unit] = static_cast<uint8_t>(code);
      page[at + (f + HALF) * unit] = static_cast<uint8_t>(code >> 8);
    }
    if (lane == 0) *scale = kv_pow2(e);
  }
}

}  // namespace evo2

using namespace evo2;

// Both grids: (columns x head groups, sequences, keys | values).
static int kv_grid(int64_t cols, int64_t heads, int64_t B, const char *what, dim3 &grid) {
  const int64_t x = cols * cdiv(heads, KV_WAVES);
  if (B > 65535 || !grid_fits(x, 64 * KV_WAVES))
    return fail(EVO2_ERR_UNSUPPORTED, "%s: more workgroups than a launch takes", what);
  grid = dim3(static_cast<unsigned>(x), static_cast<unsigned>(B), 2);
  return EVO2_OK;
}

extern "C" int evo2_kv_fp8_write(const void *k, int64_t kb, int64_t kt, int64_t kh, const void *v, int64_t vb,
                                 int64_t vt, int64_t vh, void *k_pages, int64_t kps, int64_t khs, void *v_pages,
                                 int64_t vps, int64_t vhs, float *k_scale, int64_t ksp, int64_t ksh, float *v_scale,
                                 int64_t vsp, int64_t vsh, int64_t num_pages, const int32_t *table, int64_t st,
                                 int64_t max_pages, const int64_t *positions, const int64_t *lengths, int64_t B,
                                 int64_t n, int64_t heads, int64_t head_dim, void *stream) {
  if (B < 0 || n < 0 || n > 0x7fffffff)
    return fail(EVO2_ERR_INVALID, "kv_fp8_write: bad sizes B=%lld n=%lld", (long long)B, (long long)n);
  const KvPages c{static_cast<uint8_t *>(k_pages), kps, khs, static_cast<uint8_t *>(v_pages), vps, vhs, k_scale, ksp,
                  ksh, v_scale, vsp, vsh, num_pages, table, st, max_pages};
  if (B == 0 || n == 0) return EVO2_OK;
  int rc = kv_check(c, heads, head_dim, true, "kv_fp8_write");
  if (rc) return rc;
  if (!k || !v || !positions) return fail(EVO2_ERR_INVALID, "kv_fp8_write: null pointer argument");
  const uintptr_t at = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  if (at % 16 || kb % 8 || kt % 8 || kh % 8 || vb % 8 || vt % 8 || vh % 8)
    return fail(EVO2_ERR_UNSUPPORTED, "kv_fp8_write: rows must be 16-byte aligned");
  dim3 grid;
  // n tokens reach at most this many pages, wherever the first one lies
  rc = kv_grid((n + KV_PAGE - 2) / KV_PAGE + 1, heads, B, "kv_fp8_write", grid);
  if (rc) return rc;
  const KvTokens t{static_cast<const bf16_t *>(k), kb, kt, kh, static_cast<const bf16_t *>(v), vb, vt, vh, positions,
                   lengths, n, static_cast<int>(heads)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128)
    hipLaunchKernelGGL(kv_write_kernel<128>, grid, dim3(64 * KV_WAVES), 0, s, c, t);
  else
    hipLaunchKernelGGL(kv_write_kernel<64>, grid, dim3(64 * KV_WAVES), 0, s, c, t);
  return check_launch("kv_fp8_write");
}

extern "C" int evo2_kv_fp8_read(const void *k_pages, int64_t kps, int64_t khs, const void *v_pages, int64_t vps,
                                int64_t vhs, const float *k_scale, int64_t ksp, int64_t ksh, const float *v_scale,
                                int64_t vsp, int64_t vsh, int64_t num_pages, const int32_t *table, int64_t st,
                                int64_t max_pages, const int64_t *lengths, void *k, void *v, int64_t B, int64_t L,
                                int64_t heads, int64_t head_dim, void *stream) {
  if (B < 0 || L < 0 || L > 0x7fffffff)
    return fail(EVO2_ERR_INVALID, "kv_fp8_read: bad sizes B=%lld L=%lld", (long long)B, (long long)L);
  // (the kernel only reads the pages)
  const KvPages c{static_cast<uint8_t *>(const_cast<void *>(k_pages)), kps, khs,
                  static_cast<uint8_t *>(const_cast<void *>(v_pages)), vps, vhs, const_cast<float *>(k_scale), ksp,
                  ksh, const_cast<float *>(v_scale), vsp, vsh, num_pages, table, st, max_pages};
  if (B == 0 || L == 0) return EVO2_OK;
  int rc = kv_check(c, heads, head_dim, false, "kv_fp8_read");
  if (rc) return rc;
  if (!k || !v || !lengths) return fail(EVO2_ERR_INVALID, "kv_fp8_read: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16)
    return fail(EVO2_ERR_UNSUPPORTED, "kv_fp8_read: rows must be 16-byte aligned");
  dim3 grid;
  rc = kv_grid(cdiv(L, KV_PAGE), heads, B, "kv_fp8_read", grid);
  if (rc) return rc;
  const KvOut r{static_cast<bf16_t *>(k), static_cast<bf16_t *>(v), lengths, L, static_cast<int>(heads)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128)
    hipLaunchKernelGGL(kv_read_kernel<128>, grid, dim3(64 * KV_WAVES), 0, s, c, r);
  else
    hipLaunchKernelGGL(kv_read_kernel<64>, grid, dim3(64 * KV_WAVES), 0, s, c, r);
  return check_launch("kv_fp8_read");
}

extern "C" int evo2_rotary_decode_fp8(const void *qkv, int64_t sqkv, const float *inv_freq, float factor, void *q,
                                      void *k_pages, int64_t kps, int64_t khs, void *v_pages, int64_t vps,
                                      int64_t vhs, float *k_scale, int64_t ksp, int64_t ksh, float *v_scale,
                                      int64_t vsp, int64_t vsh, int64_t num_pages, const int32_t *table, int64_t st,
                                      int64_t max_pages, const int64_t *positions, int64_t B, int64_t heads,
                                      int64_t head_dim, void *stream) {
  if (B < 0) return fail(EVO2_ERR_INVALID, "rotary_decode_fp8: bad sizes B=%lld", (long long)B);
  const KvPages c{static_cast<uint8_t *>(k_pages), kps, khs, static_cast<uint8_t *>(v_pages), vps, vhs, k_scale, ksp,
                  ksh, v_scale, vsp, vsh, num_pages, table, st, max_pages};
  if (B == 0) return EVO2_OK;
  int rc = kv_check(c, heads, head_dim, true, "rotary_decode_fp8");
  if (rc) return rc;
  if (!qkv || !inv_freq || !q || !positions)
    return fail(EVO2_ERR_INVALID, "rotary_decode_fp8: null pointer argument");
  if (B > 65535) return fail(EVO2_ERR_UNSUPPORTED, "rotary_decode_fp8: more workgroups than a launch takes");
  const KvRotary t{static_cast<const bf16_t *>(qkv), sqkv, inv_freq, factor, static_cast<bf16_t *>(q), positions,
                   static_cast<int>(heads)};
  const dim3 grid(static_cast<unsigned>(cdiv(heads, KV_WAVES)), static_cast<unsigned>(B));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128)
    hipLaunchKernelGGL(kv_rotary_decode_kernel<128>, grid, dim3(64 * KV_WAVES), 0, s, c, t);
  else
    hipLaunchKernelGGL(kv_rotary_decode_kernel<64>, grid, dim3(64 * KV_WAVES), 0, s, c, t);
  return check_launch("rotary_decode_fp8");
}

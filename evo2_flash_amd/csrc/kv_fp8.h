// The 8-bit KV cache: e4m3 codes in pages of 16 positions, one power of two a (page, key
// head) as their scale, for keys and values apart.
//
//   keys   (pages, kv_heads, 16, head_dim)   a position's row is the unit of a score
//   values (pages, kv_heads, head_dim, 16)   16 positions of a dim are one 16-byte load
//
// so that a lane's 16 bytes are an operand of the matrix cores as they lie.  The scale is
// 2^e with e the smallest integer for which no finite value of the page's tokens is over
// 448 * 2^e (448: the largest code), in [KV_EMIN, KV_EMAX].  A power of two costs a
// floating code no precision against any other scale, makes code * 2^e exact in bf16, and
// lets a page that gets a larger token later re-encode its codes exactly, all but those
// that reach the codes' subnormal range (2^-6 and below).
#pragma once

#include "attn_common.h"

namespace evo2 {

constexpr int KV_PAGE = 16;
constexpr int KV_EMIN = -110;  // zeros; every product of a code and a scale is a normal number
constexpr int KV_EMAX = 119;   // 448 * 2^119 is the largest finite value a code stands for

// e of a page whose largest finite magnitude has the bf16 bits `amax` (448 is 1.75 * 2^8).
__device__ __forceinline__ int kv_exponent(uint32_t amax) {
  const int e = static_cast<int>(amax >> 7) - 135 + ((amax & 0x7f) > 0x60);
  return min(max(e, KV_EMIN), KV_EMAX);
}

// e of a scale held in the cache (whatever stands there: a page not written yet).
__device__ __forceinline__ int kv_held(float scale) {
  return min(max(static_cast<int>((__float_as_uint(scale) >> 23) & 0xff) - 127, KV_EMIN), KV_EMAX);
}

__device__ __forceinline__ float kv_pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The larger of `m` and the bf16 magnitudes of w's two values, infinities and NaN left out.
__device__ __forceinline__ uint32_t kv_amax2(uint32_t m, uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  return max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
}

// Two values to codes (round to nearest even; NaN and infinities to NaN) in the low (HI:
// high) half of `old`.  inv = 2^-e; top: e is KV_EMAX, where values past 448 saturate.
template <bool HI>
__device__ __forceinline__ uint32_t kv_encode2(float a, float b, float inv, bool top, uint32_t old) {
  a *= inv;
  b *= inv;
  if (top) {
    if (fabsf(a) < INFINITY) a = fminf(fmaxf(a, -448.0f), 448.0f);
    if (fabsf(b) < INFINITY) b = fminf(fmaxf(b, -448.0f), 448.0f);
  }
  return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, HI);
}

// Four codes times 2^-d, d >= 0, as codes (f = 2^-min(d, 60): 2^-19 of the largest code is 0).
__device__ __forceinline__ uint32_t kv_recode4(uint32_t w, float f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, r, true);
}

// Two codes (the low, HI: the high half of w) times 2^e as two bf16 in a dword, exactly.
template <bool HI>
__device__ __forceinline__ uint32_t kv_decode2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

__device__ __forceinline__ uint32_t kv_wave_max(uint32_t m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
  return m;
}

// What both the cache's kernels and the attention over it are handed.
struct KvPages {
  uint8_t *k; int64_t kp, kh;            // key pages; page and head strides (bytes)
  uint8_t *v; int64_t vp, vh;            // value pages
  float *ks; int64_t ksp, ksh;           // scales (pages, heads); strides (elements)
  float *vs; int64_t vsp, vsh;
  int64_t num_pages;
  const int32_t *table; int64_t st;      // block table, row stride
  int64_t max_pages;                     // its columns
};

// Whether no two (page, head)s' `size` elements overlap.
inline bool kv_apart(int64_t pages, int64_t sp, int64_t heads, int64_t sh, int64_t size) {
  if (pages == 1 || heads == 1) return pages == 1 ? heads == 1 || sh >= size : sp >= size;
  return sp > sh ? sh >= size && (sp - size) / sh >= heads - 1 : sp >= size && (sh - size) / sp >= pages - 1;
}

// Whether the pages are as the kernels address them (and, for writes, lie apart); the status
// of a refusal.
inline int kv_check(const KvPages &c, int64_t heads, int64_t hd, bool writes, const char *what) {
  if (hd != 64 && hd != 128)
    return fail(EVO2_ERR_UNSUPPORTED, "%s: head_dim %lld (64 or 128)", what, (long long)hd);
  if (!c.k || !c.v || !c.ks || !c.vs || !c.table) return fail(EVO2_ERR_INVALID, "%s: null pointer argument", what);
  if (c.num_pages <= 0 || c.max_pages <= 0 || c.max_pages > (int64_t(1) << 26) || heads <= 0 || heads > 65535)
    return fail(EVO2_ERR_INVALID, "%s: bad sizes heads=%lld num_pages=%lld max_pages=%lld", what, (long long)heads,
                (long long)c.num_pages, (long long)c.max_pages);
  const uintptr_t at = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v);
  if (at % 16 || c.kp % 16 || c.kh % 16 || c.vp % 16 || c.vh % 16 || c.kh < 16 * hd || c.vh < 16 * hd)
    return fail(EVO2_ERR_UNSUPPORTED, "%s: page strides or alignment not supported", what);
  const int64_t P = c.num_pages;
  if (writes && !(kv_apart(P, c.kp, heads, c.kh, 16 * hd) && kv_apart(P, c.vp, heads, c.vh, 16 * hd) &&
                  kv_apart(P, c.ksp, heads, c.ksh, 1) && kv_apart(P, c.vsp, heads, c.vsh, 1)))
    return fail(EVO2_ERR_UNSUPPORTED, "%s: pages or scales overlap", what);
  return EVO2_OK;
}

}  // namespace evo2

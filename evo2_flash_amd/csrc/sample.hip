// The next token of each row of logits from a given uniform number, behind the decoder's
// head (model.py:343-348): temperature, then top-k, top-p of what top-k left, and min-p.
//
//   w_i = exp((z_i - max z) / T)
//   the tokens in order of (z descending, index ascending):
//     top-k keeps the first k, top-p of those the shortest front whose weights reach
//     p times theirs, min-p those with w_i >= m
//   the token is the first index i, in the vocabulary's order, with
//     sum_{j <= i, kept} w_j > u * sum_{kept} w_j
//
// Each of the three keeps a front of one order, so what they keep together is all tokens
// above some value and the first few of those that equal it: the kernels look for that
// (value, number) by counting, without sorting.  Values become whole numbers in the same
// order (-0 as 0; -inf and NaN below all, never drawn).
//
// Weights are whole numbers, round(w 2^S): sums of them are exact and the same in any
// order, also through atomics, and their steps (2^-45 of the largest at 131072 tokens)
// decide no draw that 64-bit floating point would settle.  2^y is a polynomial in 64 bits
// whose scaling and rounding to a whole number are one FMA.
//
// Rows of up to 1024 logits: a wave each, the logits in its registers, the cuts by
// bisection (sample_wave_kernel).  Longer rows: four launches over slices of 4096 logits
// (sample_slice_kernel and the ones after it), which read the logits once from memory.
#include <type_traits>

#include "common.h"

// (top c - ceil(top c) is a difference of rounded values, whatever their size)
#pragma clang fp contract(off)

namespace evo2 {

struct SampleArgs {
  const void *z; int64_t sz;  // (B, V) bf16 or fp32, row stride, unit last stride
  const float *u;             // (B,)
  const float *t; float t1;   // by row, or one for all
  const int32_t *k; int64_t k1;
  const float *p; float p1;
  const float *m; float m1;
  int64_t *out;               // (B,): the token, -1 for a row with none left
  int V;
  int shift;                  // S
};

// A row's settings.
struct SampleRow {
  double c;       // log2(e) / T: y = (z - max) c
  double ymin;    // log2(m), -inf without min-p
  float top_p;
  int64_t top_k;  // 0: all
  bool first;     // the first of the largest
};
__device__ __forceinline__ SampleRow row_of(const SampleArgs &p, int b) {
  SampleRow r;
  const float t = p.t ? p.t[b] : p.t1, m = p.m ? p.m[b] : p.m1;
  r.top_p = p.p ? p.p[b] : p.p1;
  const int64_t k = p.k ? p.k[b] : p.k1;
  r.top_k = k > 0 && k < p.V ? k : 0;
  r.first = !(t > 0.0f) || k == 1;
  r.c = 1.4426950408889634 / static_cast<double>(fminf(t, 3.0e38f));  // (any infinite T is flat)
  r.ymin = m > 0.0f ? log2(static_cast<double>(fminf(m, 1.0f))) : -INFINITY;
  return r;
}

// Whole numbers in the order of the values; 0: not a token (-inf, NaN).
__device__ __forceinline__ uint32_t key_of(float z) {
  if (!(z > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(z + 0.0f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// The value of a key (not 0); +inf as a number far above all others.
__device__ __forceinline__ double value_of(uint32_t key) {
  const float z = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
  return z < INFINITY ? static_cast<double>(z) : 1e200;
}

template <typename T>
__device__ __forceinline__ float logit(const T *z, int i) {
  if constexpr (std::is_same_v<T, float>) return z[i];
  else return bf2f(z[i]);
}

// round(2^(S + y)) for y <= 0, S <= 51: 2^f of the fraction by its series (ln 2)^k / k!
// to f^12 (|f| <= 1/2: below 2^-50 of it), times 2^(S + n) plus 2^52 in one FMA, whose
// rounding is the whole number's; its bits are the sum's low 52.
__device__ __forceinline__ uint64_t weight_of(double y, int shift) {
  const double n = rint(fmax(y, -2000.0)), f = fmax(y, -2000.0) - n;
  double p = 2.5678435993488196e-11;                // (ln 2)^12 / 12!
  p = fma(p, f, 4.44553827187081e-10);
  p = fma(p, f, 7.054911620801121e-09);
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 1.5403530393381606e-04);
  p = fma(p, f, 1.3333558146428441e-03);
  p = fma(p, f, 9.618129107628477e-03);
  p = fma(p, f, 5.5504108664821577e-02);
  p = fma(p, f, 2.402265069591007e-01);
  p = fma(p, f, 6.931471805599453e-01);
  p = fma(p, f, 1.0);
  const int e = max(static_cast<int>(n) + shift, -100);
  const double s = __longlong_as_double(static_cast<int64_t>(1023 + e) << 52);
  return __double_as_longlong(fma(p, s, 4503599627370496.0)) & 0xfffffffffffffull;
}

// ---------------------------------------------------------------- within a wave
// The value of the lane that DPP control CTRL names, 0 where there is none or the row is
// not of MASK.
template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, MASK, 0xF, false);
}
template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
  return static_cast<uint64_t>(dpp<CTRL, MASK>(static_cast<uint32_t>(v >> 32))) << 32 |
         dpp<CTRL, MASK>(static_cast<uint32_t>(v));
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
  return __builtin_amdgcn_readlane(static_cast<int>(v), lane);
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  return static_cast<uint64_t>(lane_value(static_cast<uint32_t>(v >> 32), lane)) << 32 |
         lane_value(static_cast<uint32_t>(v), lane);
}
template <typename U>
__device__ __forceinline__ U wave_scan(U v) {  // inclusive
  v += dpp<0x111>(v);        // rows of 16: from 1, 2, 4, 8 lanes before
  v += dpp<0x112>(v);
  v += dpp<0x114>(v);
  v += dpp<0x118>(v);
  v += dpp<0x142, 0xA>(v);   // row ends into the next row, then the half
  v += dpp<0x143, 0xC>(v);
  return v;
}
template <typename U>
__device__ __forceinline__ U wave_sum(U v) { return lane_value(wave_scan(v), 63); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, dpp<0x111>(v));
  v = max(v, dpp<0x112>(v));
  v = max(v, dpp<0x114>(v));
  v = max(v, dpp<0x118>(v));
  v = max(v, dpp<0x142, 0xA>(v));
  v = max(v, dpp<0x143, 0xC>(v));
  return lane_value(v, 63);
}

// f * total for 0 < f < 1, rounded down or up to a whole number, exactly (f is a whole
// number of 24 bits over a power of two): tokens of equal weight are parted where they are.
__device__ __forceinline__ uint64_t part_of(float f, uint64_t total, bool up) {
  const uint32_t bits = __float_as_uint(f), e = bits >> 23;
  const unsigned __int128 x = static_cast<unsigned __int128>(total) * (e ? (bits & 0x7fffffu) | 0x800000u : bits);
  const uint32_t sh = 150 - max(e, 1u);
  if (sh > 100) return up;  // below 2^-14 of a step
  const uint64_t q = static_cast<uint64_t>(x >> sh);
  return up && (static_cast<unsigned __int128>(q) << sh) != x ? q + 1 : q;
}
// u * total as a whole number below total (> 0): the draw's running sum has to pass it.
__device__ __forceinline__ uint64_t target_of(float u, uint64_t total) {
  return u > 0.0f ? u < 1.0f ? part_of(u, total, false) : total - 1 : 0;
}
// The least whole number that is not below p * total (> 0), p < 1, at least 1.
__device__ __forceinline__ uint64_t need_of(float p, uint64_t total) {
  return p > 0.0f ? max(part_of(p, total, true), uint64_t(1)) : 1;
}
// Tokens of one value (weight w) that a front takes whose sum before them is `above`.
__device__ __forceinline__ uint32_t ties_of(uint64_t need, uint64_t above, uint64_t w) {
  const uint64_t n = w ? (need - above + w - 1) / w : 0xffffffffull;
  return static_cast<uint32_t>(min(n, uint64_t(0xffffffff)));
}

// ---------------------------------------------------------------- rows of up to 64 E logits
// A wave takes a row, lane l logits E l .. E l + E - 1.  Top-k by bisection between the
// least and the largest key, in turn at the mean of the two values (few steps for logits
// as a head gives them) and at the middle of their keys (at most 32 for any); it ends
// where exactly k keys are not below the probe.  Top-p likewise by the weights' sums, until
// one token is left between the bounds.  8 rows of 512: see the launch below.
template <typename T, int E>
__global__ __launch_bounds__(256) void sample_wave_kernel(SampleArgs p, int B) {
  const int lane = threadIdx.x & 63;
  const int b = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (b >= B) return;
  const T *z = static_cast<const T *>(p.z) + b * p.sz;
  uint32_t key[E], top = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = E * lane + e;
    key[e] = i < p.V ? key_of(logit(z, i)) : 0;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) top = max(top, key[e]);
  const SampleRow r = row_of(p, b);
  const uint32_t kmax = wave_max(top);
  if (kmax == 0) {
    if (lane == 0) p.out[b] = -1;
    return;
  }
  if (r.first) {
    uint32_t at = E;
#pragma unroll
    for (int e = E - 1; e >= 0; --e)
      if (key[e] == kmax) at = e;
    const int l = __ffsll(static_cast<long long>(__ballot(at < E))) - 1;
    if (lane == l) p.out[b] = E * l + at;
    return;
  }
  auto count = [&](uint32_t t) __attribute__((always_inline)) {  // keys not below t
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) n += __popcll(__ballot(key[e] >= t));
    return n;
  };
  // a probe in (lo, hi), lo + 1 < hi
  auto probe = [&](uint32_t lo, uint32_t hi, int step) __attribute__((always_inline)) {
    uint32_t mid = lo + (hi - lo) / 2;
    if (step & 1) {
      const float a = static_cast<float>(0.5 * (value_of(lo) + value_of(hi - 1)));
      mid = min(max(key_of(a), lo + 1), hi - 1);
    }
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(mid));
  };
  // What is kept: keys over `cut`, and the first `tie` that equal it.
  uint32_t cut = 0, tie = 0, least = kmax;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (key[e]) least = min(least, key[e]);
  least = ~wave_max(~least);
  const uint32_t valid = count(1);
  if (r.top_k && r.top_k < valid) {
    const uint32_t k = static_cast<uint32_t>(r.top_k);
    uint32_t lo = least, hi = kmax + 1, over = 0;  // count(lo) >= k > count(hi) = over
    for (int step = 1; hi - lo > 1; ++step) {
      const uint32_t mid = probe(lo, hi, step), n = count(mid);
      if (n == k) {  // none of the next lower value
        lo = mid - 1;
        over = k;
        break;
      }
      if (n > k) lo = mid;
      else hi = mid, over = n;
    }
    cut = lo;
    tie = k - over;
  }
  const double kv = value_of(kmax);
  uint64_t w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const double y = (value_of(key[e] ? key[e] : kmax) - kv) * r.c;
    w[e] = weight_of(y, p.shift);
    if (key[e] < max(cut, 1u)) w[e] = 0;
  }
  // ranks of the tokens that equal the cut, in the vocabulary's order
  auto drop_ties = [&]() __attribute__((always_inline)) {
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) n += key[e] == cut;
    uint32_t rank = wave_scan(n) - n;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] == cut && rank++ >= tie) w[e] = 0;
  };
  if (cut) drop_ties();
  auto mass = [&](uint32_t t) __attribute__((always_inline)) {  // weight of keys not below t
    uint64_t s = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) s += key[e] >= t ? w[e] : 0;
    return wave_sum(s);
  };
  if (r.top_p < 1.0f) {
    const uint64_t need = need_of(r.top_p, mass(1));
    uint32_t lo = max(cut, least), hi = kmax + 1;  // mass(lo) >= need > mass(hi) = above
    uint32_t nlo = count(lo), nhi = 0;
    uint64_t above = 0;
    for (int step = 1; hi - lo > 1; ++step) {
      if (nlo - nhi == 1) {  // one token of [lo, hi): its key is the cut
        uint32_t at = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (key[e] >= lo && key[e] < hi) at = key[e];
        lo = wave_max(at);
        break;
      }
      const uint32_t mid = probe(lo, hi, step);
      const uint64_t s = mass(mid);
      if (s >= need) lo = mid, nlo = count(mid);
      else hi = mid, nhi = count(mid), above = s;
    }
    const uint32_t most = ties_of(need, above, weight_of((value_of(lo) - kv) * r.c, p.shift));
    tie = lo == cut ? min(tie, most) : most;
    cut = lo;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] < cut) w[e] = 0;
    drop_ties();
  }
  uint64_t sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const double y = (value_of(key[e] ? key[e] : kmax) - kv) * r.c;
    if (!(y >= r.ymin)) w[e] = 0;
    sum += w[e];
  }
  const uint64_t upto = wave_scan(sum), target = target_of(p.u[b], lane_value(upto, 63));
  const int l = __ffsll(static_cast<long long>(__ballot(upto > target))) - 1;
  if (lane == l) {
    uint64_t run = upto - sum;
    int at = 0;
    for (int e = 0; e < E; ++e) {  // the first at which the sum passes the target
      run += w[e];
      if (run > target) break;
      at = e + 1;
    }
    p.out[b] = E * l + at;
  }
}

// ---------------------------------------------------------------- longer rows
// Slices of SL logits.  sample_slice_kernel: a slice's largest logit, and a histogram of
// its tokens and weights over BINS bins of a quarter of a power of two in weight, from its
// largest down (the last bin takes all below).  Bins lie on one grid for all slices of a
// row, floor(4 z c), and weights are 2^(S + z c - R) with a whole R of the slice's own, so
// that histograms of slices add up by shifts.  sample_join_kernel: a row's histogram, the
// bins in which the cuts lie.  sample_list_kernel: the keys of the slices' tokens in those
// bins, in the vocabulary's order (top-k: all down to its cut; else the one to three bins of
// top-p's and min-p's).  sample_draw_kernel: the exact cut among them, a byte at a time
// from histograms, the slices' sums, and the token in the slice that the draw falls into.
constexpr int SL_T = 512, SL_E = 8, SL = SL_T * SL_E, SL_W = SL_T / 64;
constexpr int BINS = 256;

struct SliceInfo {
  double top;           // its largest logit
  uint64_t total;       // its weight, in its own units
  uint64_t base;        // weight in bins over the listed ones, in the row's units
  uint32_t key, at;     // largest key (0: no token) and its first index
  uint32_t listed, pad;
};
struct RowInfo {
  double top;           // the row's largest logit
  uint64_t total;       // its weight
  uint64_t over;        // of it in bins over the listed ones
  int32_t mode;         // 0: drawn already, 1: nothing is cut, 2: bins lo .. hi are listed
  int32_t lo, hi;
  uint32_t pad;
};

struct SampleWork {
  SliceInfo *slice;     // (B, S)
  RowInfo *row;         // (B,)
  uint64_t *mass;       // (B, S, BINS)
  uint32_t *count;      // (B, S, BINS)
  uint32_t *list;       // (B, S * SL)
  int S;
};

// The unit of weights for a largest logit: 2^(S + z c - R), R = ceil(top c).
struct SampleRef {
  double top, c, r, phi;  // phi = top c - R
  __device__ __forceinline__ SampleRef(double t, double cc) : top(t), c(cc), r(ceil(t * cc)) { phi = t * cc - r; }
  __device__ __forceinline__ uint64_t weight(double z, int shift) const {
    return weight_of(fma(z - top, c, phi), shift);
  }
  __device__ __forceinline__ double y(double z) const { return (z - top) * c; }  // of the largest weight
};
__device__ __forceinline__ double grid_of(double z, double c) { return floor(z * (4.0 * c)); }
__device__ __forceinline__ int bin_of(double top_grid, double z, double c) {
  return static_cast<int>(fmin(top_grid - grid_of(z, c), static_cast<double>(BINS - 1)));
}

// Thread t's keys of slice s: logits SL s + SL_E t .. + SL_E - 1.
template <typename T>
__device__ __forceinline__ void slice_keys(const SampleArgs &p, int b, int s, int t, uint32_t (&key)[SL_E]) {
  const T *z = static_cast<const T *>(p.z) + b * p.sz;
  const int i0 = SL * s + SL_E * t;
  float x[SL_E];
  if (i0 + SL_E <= p.V && reinterpret_cast<uintptr_t>(z + i0) % 16 == 0) {
    if constexpr (std::is_same_v<T, float>) {
      const float4 a = *reinterpret_cast<const float4 *>(z + i0), c = *reinterpret_cast<const float4 *>(z + i0 + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = c.x, x[5] = c.y, x[6] = c.z, x[7] = c.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4 *>(z + i0);
      const uint32_t d[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[2 * e] = lo_bf(d[e]), x[2 * e + 1] = hi_bf(d[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < SL_E; ++e) x[e] = i0 + e < p.V ? logit(z, i0 + e) : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < SL_E; ++e) key[e] = key_of(x[e]);
}

template <typename T>
__global__ __launch_bounds__(SL_T) void sample_slice_kernel(SampleArgs p, SampleWork w) {
  __shared__ unsigned long long mass[BINS];
  __shared__ uint32_t count[BINS], red[SL_W];
  const int s = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  uint32_t key[SL_E], top = 0, at = 0;
  slice_keys<T>(p, b, s, t, key);
  const SampleRow r = row_of(p, b);
#pragma unroll
  for (int e = 0; e < SL_E; ++e) top = max(top, key[e]);
  const uint32_t wtop = wave_max(top);
  if (lane == 0) red[wave] = wtop;
  for (int i = t; i < BINS; i += SL_T) mass[i] = 0, count[i] = 0;
  __syncthreads();
  uint32_t kmax = 0;
#pragma unroll
  for (int i = 0; i < SL_W; ++i) kmax = max(kmax, red[i]);
  SliceInfo &info = w.slice[static_cast<int64_t>(b) * w.S + s];
  const int64_t h = (static_cast<int64_t>(b) * w.S + s) * BINS;
  uint64_t total = 0;
  if (kmax && !r.first) {  // uniform
    const double z0 = value_of(kmax);
    const SampleRef ref(z0, r.c);
    const double g0 = grid_of(z0, r.c);
#pragma unroll
    for (int e = 0; e < SL_E; ++e) {
      if (key[e] == 0) continue;
      const double z = value_of(key[e]);
      const uint64_t x = ref.weight(z, p.shift);
      const int bin = bin_of(g0, z, r.c);
      atomicAdd(&count[bin], 1u);
      if (x) atomicAdd(&mass[bin], static_cast<unsigned long long>(x));
    }
  }
#pragma unroll
  for (int e = 0; e < SL_E; ++e)  // the first of the largest, as ~index
    if (key[e] == kmax) at = max(at, ~static_cast<uint32_t>(SL * s + SL_E * t + e));
  at = wave_max(at);
  __syncthreads();
  if (t < BINS) {
    w.mass[h + t] = total = mass[t];
    w.count[h + t] = count[t];
  }
  total = wave_sum(total);
  __syncthreads();
  if (lane == 0) {
    red[wave] = at;
    mass[wave] = total;
  }
  __syncthreads();
  if (t == 0) {
    for (int i = 0; i < SL_W; ++i) at = max(at, red[i]);
    total = 0;
    for (int i = 0; i < SL_W; ++i) total += mass[i];
    info.top = kmax ? value_of(kmax) : 0.0;
    info.total = total;
    info.key = kmax;
    info.at = ~at;
  }
}

// The bin of hist (BINS, from the top down) in which its running sum reaches `need`, and
// the sum before it; BINS where all of them do not reach it.  One wave.
__device__ __forceinline__ int bin_reaching(const unsigned long long *hist, uint64_t need, int lane, uint64_t &above) {
  uint64_t h[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += h[i] = hist[4 * lane + i];
  const uint64_t run = wave_scan(sum);
  const uint64_t hit = __ballot(run >= need);
  if (!hit) return BINS;
  const int l = __ffsll(static_cast<long long>(hit)) - 1;
  uint64_t a = run - sum;
  uint32_t bin = 4 * lane;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (bin == static_cast<uint32_t>(4 * lane + i) && a + h[i] < need) {
      a += h[i];
      ++bin;
    }
  above = lane_value(a, l);
  return lane_value(bin, l);
}

constexpr int SJ_T = 1024, SJ_G = SJ_T / BINS;  // groups of threads take slices in turn

__global__ __launch_bounds__(SJ_T) void sample_join_kernel(SampleArgs p, SampleWork w) {
  __shared__ unsigned long long mass[BINS], count[BINS];
  __shared__ uint32_t red[SJ_T / 64], red2[SJ_T / 64];
  __shared__ int by[BINS], off[BINS];
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, bin = t % BINS;
  const SliceInfo *slice = w.slice + static_cast<int64_t>(b) * w.S;
  const SampleRow r = row_of(p, b);
  RowInfo &row = w.row[b];
  if (t < BINS) mass[t] = 0, count[t] = 0;
  uint32_t km = 0, at = 0;
  for (int s = t; s < w.S; s += SJ_T) {
    const uint32_t k = slice[s].key, first = ~slice[s].at;
    at = k > km ? first : k == km ? max(at, first) : at;
    km = max(km, k);
  }
  uint32_t kmax = wave_max(km);
  at = wave_max(km == kmax ? at : 0);
  if (lane == 0) red[wave] = kmax, red2[wave] = at;
  __syncthreads();
  for (int i = 0; i < SJ_T / 64; ++i) kmax = max(kmax, red[i]);
  if (t == 0) {  // the first of the largest; the draw writes over it
    at = 0;
    for (int i = 0; i < SJ_T / 64; ++i) at = red[i] == kmax ? max(at, red2[i]) : at;
    p.out[b] = kmax ? static_cast<int64_t>(~at) : -1;
    if (kmax == 0 || r.first) row.mode = 0;
  }
  if (kmax == 0 || r.first) return;  // uniform
  const SampleRef ref(value_of(kmax), r.c);
  const double g0 = grid_of(ref.top, r.c);
  for (int s0 = 0; s0 < w.S; s0 += BINS) {
    const int n = min(w.S - s0, BINS);
    __syncthreads();
    if (t < n) {  // slice's units are 2^-by of the row's, its bins `off` below the row's
      const bool live = slice[s0 + t].key != 0;
      const double top = slice[s0 + t].top;
      by[t] = live ? static_cast<int>(fmin(ref.r - ceil(top * r.c), 63.0)) : -1;
      off[t] = static_cast<int>(fmin(g0 - grid_of(top, r.c), static_cast<double>(BINS - 1)));
    }
    __syncthreads();
    const int64_t h = (static_cast<int64_t>(b) * w.S + s0) * BINS + bin;
#pragma unroll 8
    for (int s = t / BINS; s < n; s += SJ_G) {
      const uint64_t x = w.mass[h + s * BINS];
      const uint32_t c = w.count[h + s * BINS];
      if (by[s] < 0) continue;
      if (c) atomicAdd(&count[min(bin + off[s], BINS - 1)], static_cast<unsigned long long>(c));
      if (x) atomicAdd(&mass[min(bin + off[s], BINS - 1)], static_cast<unsigned long long>(x >> by[s]));
    }
  }
  __syncthreads();
  if (wave) return;
  uint64_t total = 0, tokens = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) total += mass[4 * lane + i], tokens += count[4 * lane + i];
  total = wave_sum(total);
  tokens = wave_sum(tokens);
  int lo = BINS, hi = -1;
  uint64_t before = 0;
  if (r.top_k && static_cast<uint64_t>(r.top_k) < tokens) {
    lo = 0;
    hi = bin_reaching(count, r.top_k, lane, before);
  } else {
    if (r.top_p < 1.0f) lo = hi = bin_reaching(mass, need_of(r.top_p, total), lane, before);
    if (r.ymin > -INFINITY) {  // the value with this weight, to a bin either way
      const int at = bin_of(g0, ref.top + r.ymin / r.c, r.c);
      const int a = max(at - 1, 0), z = min(at + 1, BINS - 1);
      if (hi < 0 || z < lo) lo = a, hi = z;
      else if (a <= hi) lo = min(lo, a), hi = max(hi, z);
    }
  }
  uint64_t over = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) over += 4 * lane + i < lo ? mass[4 * lane + i] : 0;
  over = wave_sum(over);
  if (lane == 0) {
    row.top = ref.top;
    row.total = total;
    row.over = over;
    row.mode = hi < 0 ? 1 : 2;
    row.lo = lo;
    row.hi = hi;
  }
}

template <typename T>
__global__ __launch_bounds__(SL_T) void sample_list_kernel(SampleArgs p, SampleWork w) {
  __shared__ uint32_t red[SL_W];
  __shared__ uint64_t base[SL_W];
  const int s = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const RowInfo row = w.row[b];
  if (row.mode != 2) return;  // uniform
  SliceInfo &info = w.slice[static_cast<int64_t>(b) * w.S + s];
  const SampleRow r = row_of(p, b);
  uint32_t key[SL_E], n = 0;
  slice_keys<T>(p, b, s, t, key);
  const double g0 = grid_of(row.top, r.c);
#pragma unroll
  for (int e = 0; e < SL_E; ++e) {
    const int bin = key[e] ? bin_of(g0, value_of(key[e]), r.c) : BINS;
    if (bin < row.lo || bin > row.hi) key[e] = 0;  // (hi is below BINS)
    n += key[e] != 0;
  }
  // weight in bins over the listed ones
  uint64_t x = 0;
  if (t < BINS && info.key) {
    const SampleRef ref(row.top, r.c), own(info.top, r.c);
    const int by = static_cast<int>(fmin(ref.r - own.r, 63.0));
    const int off = static_cast<int>(fmin(g0 - grid_of(own.top, r.c), static_cast<double>(BINS - 1)));
    if (min(t + off, BINS - 1) < row.lo) x = w.mass[(static_cast<int64_t>(b) * w.S + s) * BINS + t] >> by;
  }
  x = wave_sum(x);
  const uint32_t run = wave_scan(n);
  if (lane == 63) red[wave] = run;
  if (lane == 0) base[wave] = x;
  __syncthreads();
  uint32_t at = run - n;
  for (int i = 0; i < wave; ++i) at += red[i];
  uint32_t *list = w.list + (static_cast<int64_t>(b) * w.S + s) * SL;
#pragma unroll
  for (int e = 0; e < SL_E; ++e)
    if (key[e]) list[at++] = key[e];
  if (t == 0) {
    uint32_t all = 0;
    uint64_t sum = 0;
    for (int i = 0; i < SL_W; ++i) all += red[i], sum += base[i];
    info.listed = all;
    info.base = sum;
  }
}

constexpr int SD_LDS = 8192;    // listed keys kept in LDS
constexpr int SD_S = 4096;      // most slices: 2^24 logits

template <typename T>
__global__ __launch_bounds__(SL_T) void sample_draw_kernel(SampleArgs p, SampleWork w) {
  __shared__ uint32_t keys[SD_LDS], start[SD_S + 1];
  __shared__ unsigned long long hist[BINS];
  __shared__ uint64_t wred[SL_W];
  __shared__ uint32_t red[SL_W], red2[SL_W];
  __shared__ uint64_t found_above, before_slice;
  __shared__ uint32_t found, tie_before;
  __shared__ int pick;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const RowInfo row = w.row[b];
  if (row.mode == 0) return;  // uniform
  SliceInfo *slice = w.slice + static_cast<int64_t>(b) * w.S;
  const SampleRow r = row_of(p, b);
  const SampleRef ref(row.top, r.c);
  const double g0 = grid_of(row.top, r.c);
  const uint32_t *list = w.list + static_cast<int64_t>(b) * w.S * SL;
  const bool cuts = row.mode == 2;
  // start[s]: listed keys before slice s
  uint32_t listed = 0;
  if (cuts) {
    if (wave == 0) {
      for (int s0 = 0; s0 < w.S; s0 += 64) {
        const uint32_t n = s0 + lane < w.S ? slice[s0 + lane].listed : 0, run = wave_scan(n) + listed;
        if (s0 + lane < w.S) start[s0 + lane + 1] = run;
        listed = lane_value(run, 63);
      }
      if (lane == 0) start[0] = 0;
    }
    __syncthreads();
    listed = start[w.S];
  }
  const bool fits = listed <= SD_LDS;
  // listed key i, wherever its slice left it
  auto fetch = [&](uint32_t i) __attribute__((always_inline)) {
    int lo = 0, hi = w.S;  // start[lo] <= i < start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (start[mid] <= i) lo = mid;
      else hi = mid;
    }
    return list[static_cast<int64_t>(lo) * SL + (i - start[lo])];
  };
  uint32_t kmin = ~0u, kmx = 0;
  for (uint32_t i = t; i < listed; i += SL_T) {
    const uint32_t k = fetch(i);
    if (fits) keys[i] = k;
    kmin = min(kmin, k), kmx = max(kmx, k);
  }
  kmx = wave_max(kmx);
  kmin = ~wave_max(~kmin);
  if (lane == 0) red[wave] = kmx, red2[wave] = kmin;
  if (t == 0) pick = 0, tie_before = 0, before_slice = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SL_W; ++i) kmx = max(kmx, red[i]), kmin = min(kmin, red2[i]);
  // f(key) for all listed keys
  auto each = [&](auto f) __attribute__((always_inline)) {
    for (uint32_t i = t; i < listed; i += SL_T) f(fits ? keys[i] : fetch(i));
  };
  auto weight = [&](uint32_t k) __attribute__((always_inline)) { return ref.weight(value_of(k), p.shift); };

  // What is kept of the listed: keys over `cut`, and the first `tie` that equal it.
  uint32_t cut = 0, tie = 0;
  // The key at which sum(of(key)) over the listed keys over the cut, from the top, reaches
  // `need`, and the sum above it; false where they do not.  `extra`: of the keys at the cut.
  auto search = [&](auto of, uint64_t need, uint64_t extra, uint32_t &key, uint64_t &above) __attribute__((always_inline)) {
    const int bits = kmx == kmin ? 0 : 32 - __clz(kmx ^ kmin);
    uint32_t prefix = bits == 32 ? 0 : kmx >> bits << bits;
    uint64_t over = 0;
    for (int sh = max(bits - 8, 0), top = bits; top > 0 || sh == 0; top = sh, sh = max(sh - 8, 0)) {
      const int width = top - sh;  // bits found now (none where all keys are equal)
      for (int i = t; i < BINS; i += SL_T) hist[i] = 0;
      __syncthreads();
      auto add = [&](uint32_t k, uint64_t x) __attribute__((always_inline)) {
        const uint32_t high = top >= 32 ? 0 : k >> top << top;
        if (high == prefix) atomicAdd(&hist[BINS - 1 - ((k >> sh) & ((1u << width) - 1))], static_cast<unsigned long long>(x));
      };
      each([&](uint32_t k) __attribute__((always_inline)) {
        if (k > cut) add(k, of(k));
      });
      if (t == 0 && extra) add(cut, extra);
      __syncthreads();
      if (wave == 0) {
        uint64_t a = 0;
        const int bin = bin_reaching(hist, need - over, lane, a);
        if (lane == 0) found = bin, found_above = a;
      }
      __syncthreads();
      const uint32_t bin = found;
      const uint64_t a = found_above;
      __syncthreads();
      if (bin == BINS) return false;  // uniform
      prefix |= (BINS - 1 - bin) << sh;
      over += a;
      if (sh == 0) break;
    }
    key = prefix;
    above = over;
    return true;
  };
  if (cuts && listed) {
    uint32_t key;
    uint64_t above;
    if (r.top_k && row.lo == 0 && search([](uint32_t) { return uint64_t(1); }, r.top_k, 0, key, above)) {
      cut = key;
      tie = static_cast<uint32_t>(r.top_k - above);
    }
    if (r.top_p < 1.0f) {
      const uint64_t extra = cut ? tie * weight(cut) : 0;
      uint64_t total = row.total;
      if (cut) {  // of what top-k kept
        uint64_t x = 0;
        each([&](uint32_t k) __attribute__((always_inline)) { x += k > cut ? weight(k) : 0; });
        x = wave_sum(x);
        if (lane == 0) wred[wave] = x;
        __syncthreads();
        total = extra;
        for (int i = 0; i < SL_W; ++i) total += wred[i];
        __syncthreads();
      }
      const uint64_t need = need_of(r.top_p, total);
      if (need > row.over &&
          search([&](uint32_t k) __attribute__((always_inline)) { return weight(k); }, need - row.over, extra, key, above)) {
        const uint32_t most = ties_of(need - row.over, above, weight(key));
        tie = key == cut ? min(tie, most) : most;
        cut = key;
      }
    }
  }
  // A token's weight in the draw, apart from ties at the cut; of tokens in bins over the
  // listed ones, and of listed ones
  const double zc = cut ? value_of(cut) : 0.0;
  const uint64_t wc = cut && ref.y(zc) >= r.ymin ? weight(cut) : 0;
  auto kept = [&](uint32_t k) __attribute__((always_inline)) -> uint64_t {
    if (k <= cut || !(ref.y(value_of(k)) >= r.ymin)) return 0;
    return weight(k);
  };
  // the slices' sums, a wave to a slice: into base (its weight apart from ties) and listed
  // (its ties)
  for (int s = wave; s < w.S; s += SL_W) {
    SliceInfo &info = slice[s];
    uint64_t x = 0;
    uint32_t n = 0;
    if (cuts) {
      const uint32_t i0 = start[s], i1 = start[s + 1];
      for (uint32_t i = i0 + lane; i < i1; i += 64) {
        const uint32_t k = fits ? keys[i] : list[static_cast<int64_t>(s) * SL + (i - i0)];
        x += kept(k);
        n += cut && k == cut;
      }
      x = wave_sum(x) + info.base;
      n = wave_sum(n);
    } else if (info.key) {
      x = info.total >> static_cast<int>(fmin(ref.r - ceil(info.top * r.c), 63.0));
    }
    if (lane == 0) info.base = x, info.listed = n;
  }
  __syncthreads();
  // the slice that the draw falls into
  if (wave == 0) {
    uint64_t total = 0;
    uint32_t nt = 0;
    for (int s0 = 0; s0 < w.S; s0 += 64) {
      const int s = s0 + lane;
      const uint32_t n = s < w.S ? slice[s].listed : 0, run = wave_scan(n) + nt;
      const uint64_t x = s < w.S ? slice[s].base + (min(run, tie) - min(run - n, tie)) * wc : 0;
      total += wave_sum(x);
      nt = lane_value(run, 63);
    }
    const uint64_t target = total ? target_of(p.u[b], total) : 0;
    uint64_t sum = 0;
    nt = 0;
    for (int s0 = 0; s0 < w.S; s0 += 64) {
      const int s = s0 + lane;
      const uint32_t n = s < w.S ? slice[s].listed : 0, run = wave_scan(n) + nt;
      const uint64_t x = s < w.S ? slice[s].base + (min(run, tie) - min(run - n, tie)) * wc : 0;
      const uint64_t upto = wave_scan(x) + sum;
      const uint64_t hit = __ballot(upto > target);
      if (hit) {
        const int l = __ffsll(static_cast<long long>(hit)) - 1;
        if (lane == l) pick = s, before_slice = target - (upto - x), tie_before = run - n;
        break;
      }
      sum = lane_value(upto, 63);
      nt = lane_value(run, 63);
    }
  }
  __syncthreads();
  // the token: thread t has logits SL_E t .. of the slice
  uint32_t key[SL_E], n = 0;
  uint64_t x[SL_E], mine = 0;
  slice_keys<T>(p, b, pick, t, key);
#pragma unroll
  for (int e = 0; e < SL_E; ++e) n += cut && key[e] == cut;
  const uint32_t trun = wave_scan(n);
  if (lane == 63) red[wave] = trun;
  __syncthreads();
  uint32_t rank = trun - n + tie_before;
  for (int i = 0; i < wave; ++i) rank += red[i];
#pragma unroll
  for (int e = 0; e < SL_E; ++e) {
    x[e] = 0;
    if (key[e] == 0) continue;
    if (cut && key[e] == cut) x[e] = rank++ < tie ? wc : 0;
    else if (!cuts || bin_of(g0, value_of(key[e]), r.c) <= row.hi) x[e] = kept(key[e]);
    mine += x[e];
  }
  const uint64_t wrun = wave_scan(mine);
  if (lane == 63) wred[wave] = wrun;
  __syncthreads();
  uint64_t run = wrun - mine, all = 0;
  for (int i = 0; i < SL_W; ++i) {
    if (i < wave) run += wred[i];
    all += wred[i];
  }
  // (sums of slices in other units were shifted: the last token's end may lie a few steps off)
  const uint64_t target = min(before_slice, all ? all - 1 : 0);
  if (mine && run <= target && target < run + mine) {
    int at = 0;
    for (int e = 0; e < SL_E; ++e) {
      run += x[e];
      if (run > target) break;
      at = e + 1;
    }
    p.out[b] = static_cast<int64_t>(SL) * pick + SL_E * t + at;
  }
}

static int64_t align16(int64_t n) { return (n + 15) & ~int64_t(15); }

// Offsets of the parts of a workspace; the last is its size.
struct SampleParts {
  int64_t slice, row, mass, count, list, bytes;
};
static SampleParts parts_of(int64_t B, int64_t V) {
  const int64_t S = cdiv(V, SL);
  SampleParts q;
  q.slice = 0;
  q.row = align16(B * S * static_cast<int64_t>(sizeof(SliceInfo)));
  q.mass = q.row + align16(B * static_cast<int64_t>(sizeof(RowInfo)));
  q.count = q.mass + B * S * BINS * 8;
  q.list = q.count + B * S * BINS * 4;
  q.bytes = q.list + B * S * SL * 4;
  return q;
}

constexpr int64_t SAMPLE_WAVE = 1024;  // logits of a row that a wave takes

template <typename T>
static int launch_sample(const SampleArgs &a, int64_t B, char *ws, bool listed, hipStream_t st) {
  if (a.V <= SAMPLE_WAVE) {
    const dim3 grid(static_cast<unsigned>(cdiv(B, 4)));
    const int n = static_cast<int>(B);
    if (a.V <= 256) hipLaunchKernelGGL((sample_wave_kernel<T, 4>), grid, dim3(256), 0, st, a, n);
    else if (a.V <= 512) hipLaunchKernelGGL((sample_wave_kernel<T, 8>), grid, dim3(256), 0, st, a, n);
    else hipLaunchKernelGGL((sample_wave_kernel<T, 16>), grid, dim3(256), 0, st, a, n);
    return check_launch("sample");
  }
  const SampleParts q = parts_of(B, a.V);
  const SampleWork w{reinterpret_cast<SliceInfo *>(ws + q.slice), reinterpret_cast<RowInfo *>(ws + q.row),
                     reinterpret_cast<uint64_t *>(ws + q.mass), reinterpret_cast<uint32_t *>(ws + q.count),
                     reinterpret_cast<uint32_t *>(ws + q.list), static_cast<int>(cdiv(a.V, SL))};
  const dim3 grid(static_cast<unsigned>(w.S), static_cast<unsigned>(B));
  hipLaunchKernelGGL(sample_slice_kernel<T>, grid, dim3(SL_T), 0, st, a, w);
  int rc = check_launch("sample slices");
  if (rc) return rc;
  hipLaunchKernelGGL(sample_join_kernel, dim3(static_cast<unsigned>(B)), dim3(SJ_T), 0, st, a, w);
  if ((rc = check_launch("sample join"))) return rc;
  if (listed) {
    hipLaunchKernelGGL(sample_list_kernel<T>, grid, dim3(SL_T), 0, st, a, w);
    if ((rc = check_launch("sample list"))) return rc;
  }
  hipLaunchKernelGGL(sample_draw_kernel<T>, dim3(static_cast<unsigned>(B)), dim3(SL_T), 0, st, a, w);
  return check_launch("sample draw");
}

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_sample_workspace_bytes(int64_t B, int64_t V) {
  if (B <= 0 || V <= SAMPLE_WAVE || V > (1 << 24) || B > 65535) return 0;
  return parts_of(B, V).bytes;
}

extern "C" int evo2_sample(const void *logits, int32_t fp32, int64_t sz, const float *u, const float *temperature,
                           float t1, const int32_t *top_k, int64_t k1, const float *top_p, float p1,
                           const float *min_p, float m1, void *workspace, int64_t workspace_bytes, int64_t *tokens,
                           int64_t B, int64_t V, void *stream) {
  if (B < 0 || V <= 0 || V > (1 << 24))
    return fail(EVO2_ERR_INVALID, "sample: bad sizes B=%lld V=%lld", (long long)B, (long long)V);
  if (B == 0) return EVO2_OK;
  if (!logits || !u || !tokens) return fail(EVO2_ERR_INVALID, "sample: null pointer argument");
  if (sz < V && B > 1) return fail(EVO2_ERR_UNSUPPORTED, "sample: rows must not overlap");
  if (V > SAMPLE_WAVE ? B > 65535 : !grid_fits(cdiv(B, 4), 256))
    return fail(EVO2_ERR_UNSUPPORTED, "sample: more workgroups than a launch takes");
  if (workspace_bytes < evo2_sample_workspace_bytes(B, V) || (V > SAMPLE_WAVE && !workspace) ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(EVO2_ERR_INVALID, "sample: workspace too small or not 16-byte aligned");
  // S: a row's weights stay below 2^62, one below 2^52
  int bits = 0;
  while ((int64_t(1) << bits) < V) ++bits;
  const SampleArgs a{logits, sz, u, temperature, t1, top_k, k1, top_p, p1, min_p, m1, tokens, static_cast<int>(V),
                     bits > 13 ? 62 - bits : 49};
  // without a setting that cuts, or with the first token asked for, there is nothing to list
  const bool listed = (temperature || t1 > 0.0f) && (top_k || k1 != 1) &&
                      (top_k || (k1 > 0 && k1 < V) || top_p || p1 < 1.0f || min_p || m1 > 0.0f);
  char *ws = static_cast<char *>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return fp32 ? launch_sample<float>(a, B, ws, listed, s) : launch_sample<bf16_t>(a, B, ws, listed, s);
}

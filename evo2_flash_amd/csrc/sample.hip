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
// order, also through atomics; tokens that are all equal are parted exactly where p and u say.
// S is 49 for rows of up to 8192 tokens.  Longer rows have 62 - ceil(log2 V) against each
// slice's own largest, and where a cut goes through their values the largest S (of at most 49)
// that leaves the row's sum at 2^62; joining the slices drops up to a step for each of a
// slice's bins.  In all a running sum is off by at most V 2^-48 of the total (2^-31 at 131072
// tokens; u has steps of 2^-24).  2^y is a polynomial in 64 bits whose scaling and rounding to
// a whole number are one FMA.
//
// Rows of up to 1024 logits: a wave each, the logits in its registers, the cuts from
// histograms of its own in LDS (sample_wave_kernel); of up to 8192: a workgroup each
// (sample_group_kernel).  Longer rows: four launches over slices of 4096 or 8192 logits
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
  int shift;                  // S; of longer rows that of a slice
};

// A row's settings.
struct SampleRow {
  double c;       // log2(e) / T: y = (z - max) c
  float c4;       // 4 c, at most the largest number
  float min_p;
  float top_p;
  int64_t top_k;  // 0: all
  bool first;     // the first of the largest
};
__device__ __forceinline__ SampleRow row_of(const SampleArgs &p, int b) {
  SampleRow r;
  const float t = p.t ? p.t[b] : p.t1;
  r.min_p = p.m ? p.m[b] : p.m1;
  r.top_p = p.p ? p.p[b] : p.p1;
  const int64_t k = p.k ? p.k[b] : p.k1;
  r.top_k = k > 0 && k < p.V ? k : 0;
  r.first = !(t > 0.0f) || k == 1;
  r.c = 1.4426950408889634 / static_cast<double>(fminf(t, 3.0e38f));  // (any infinite T is flat)
  r.c4 = static_cast<float>(fmin(4.0 * r.c, 3.0e38));
  return r;
}

// Whole numbers in the order of the values; 0: not a token (-inf, NaN).
__device__ __forceinline__ uint32_t key_of(float z) {
  if (!(z > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(z + 0.0f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t LEAST_KEY = 0x00800000u;  // of the lowest finite value

// The value of a key (not 0), and as a double with +inf a number far above all others.
__device__ __forceinline__ float float_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ double wide_of(float z) { return z < INFINITY ? static_cast<double>(z) : 1e200; }
__device__ __forceinline__ double value_of(uint32_t key) {
  return wide_of(float_of(key));
}

template <typename T>
__device__ __forceinline__ float logit(const T *z, int i) {
  if constexpr (std::is_same_v<T, float>) return z[i];
  else return bf2f(z[i]);
}

// Logits i0 .. i0 + E - 1 of a row of V (-inf past it): 16-byte loads at any alignment that
// elements have.
template <typename T, int E>
__device__ __forceinline__ void logits_of(const T *z, int i0, int V, float (&x)[E]) {
  constexpr int PER = 16 / sizeof(T);
  if (i0 + E <= V) {
#pragma unroll
    for (int g = 0; g < E; g += PER) {
      uint32_t d[4] = {};
      __builtin_memcpy(d, z + i0 + g, sizeof(T) * (E < PER ? E : PER));
#pragma unroll
      for (int e = 0; e < (E < PER ? E / (PER / 4) : 4); ++e) {
        if constexpr (std::is_same_v<T, float>) x[g + e] = __uint_as_float(d[e]);
        else x[g + 2 * e] = lo_bf(d[e]), x[g + 2 * e + 1] = hi_bf(d[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = i0 + e < V ? logit(z, i0 + e) : -INFINITY;
  }
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
// The value (4 or 8 bytes) of the lane that DPP control CTRL names, 0 where there is none or
// the row is not of MASK.
template <int CTRL, int MASK = 0xF, typename U>
__device__ __forceinline__ U dpp(U v) {
  auto word = [](uint32_t x) __attribute__((always_inline)) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, MASK, 0xF, false));
  };
  if constexpr (sizeof(U) == 4) return word(v);
  else return static_cast<U>(word(static_cast<uint32_t>(v >> 32))) << 32 | word(static_cast<uint32_t>(v));
}
template <typename U>
__device__ __forceinline__ U lane_value(U v, int lane) {
  auto word = [&](uint32_t x) __attribute__((always_inline)) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
  };
  if constexpr (sizeof(U) == 4) return word(v);
  else return static_cast<U>(word(static_cast<uint32_t>(v >> 32))) << 32 | word(static_cast<uint32_t>(v));
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
  const uint64_t a = need - above;
  if (w == 0 || a >> 31 >= w) return 0xffffffffu;
  // (the quotient, below 2^31, in 64-bit floating point: off by one at most)
  uint64_t n = static_cast<uint32_t>(static_cast<double>(a) / static_cast<double>(w));
  n -= n > 0 && n * w >= a;
  n += n * w < a;
  n += n * w < a;
  return static_cast<uint32_t>(n);
}

// LDS operations of a wave before and after it stay in order (they run in order; the
// compiler knows words and double words of one array for different memory).
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int BINS = 256;

// The bin of hist (from the top down) in which its running sum reaches `need`, and the sum
// before it; BINS where all of them do not reach it.  One wave.
template <typename U>
__device__ __forceinline__ uint32_t bin_reaching(const U *hist, U need, int lane, U &above) {
  U h[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += h[i] = hist[4 * lane + i];
  const U run = wave_scan(sum);
  const uint64_t hit = __ballot(run >= need);
  if (!hit) return BINS;
  const int l = __ffsll(static_cast<long long>(hit)) - 1;
  U a = run - sum;
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

// A key's bits that differ between keys of T: all, or the upper half of a bf16's.
template <typename T>
constexpr int LOW = std::is_same_v<T, float> ? 0 : 16;
template <typename T>
__device__ __forceinline__ uint32_t whole_key(uint32_t high) {
  if constexpr (LOW<T> == 0) return high;
  else return high << LOW<T> | (high >> (31 - LOW<T>) ? 0u : (1u << LOW<T>) - 1);
}

// A search goes a byte of the keys at a time, from the highest in which any differ: pass i
// counts the keys that share what is found so far, by their next `width` bits from `sh` up.
struct Digits {
  uint32_t prefix;  // bits found, in place (of keys without their LOW bits)
  int top, sh;      // bits below top are not found yet; this pass finds those from sh up
  __device__ __forceinline__ Digits(uint32_t kmax, uint32_t kmin) {
    top = kmax == kmin ? 0 : 32 - __clz(kmax ^ kmin);
    prefix = top == 32 ? 0 : kmax >> top << top;
    sh = max(top - 8, 0);
  }
  __device__ __forceinline__ bool has(uint32_t k) const { return (top == 32 ? 0 : k >> top << top) == prefix; }
  __device__ __forceinline__ uint32_t bin(uint32_t k) const {
    return BINS - 1 - ((k >> sh) & ((1u << (top - sh)) - 1));
  }
  // the bin of this pass is found; false after the last pass
  __device__ __forceinline__ bool next(uint32_t bin) {
    prefix |= (BINS - 1 - bin) << sh;
    if (sh == 0) return false;
    top = sh;
    sh = max(sh - 8, 0);
    return true;
  }
};

// ---------------------------------------------------------------- rows of up to 64 E logits
// A wave takes a row, lane l logits E l .. E l + E - 1.  The cuts are found from histograms
// of the wave's own in LDS (nothing but this wave's order of LDS operations parts their
// steps).  Bound by the chain of searches, not by its reads: 8 rows of 512 bf16 logits with
// top-k 4 4.7 us, 777 rows of 509 fp32 ones with all three cuts 8.9 us, a wave each.
template <typename T, int E>
__global__ __launch_bounds__(256) void sample_wave_kernel(SampleArgs p, int B) {
  __shared__ __attribute__((aligned(16))) unsigned long long hists[4][BINS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wave);
  if (b >= B) return;
  float z[E];
  logits_of<T, E>(static_cast<const T *>(p.z) + b * p.sz, E * lane, p.V, z);
  uint32_t key[E], top = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) key[e] = key_of(z[e]);
  const SampleRow r = row_of(p, b);
#pragma unroll
  for (int e = 0; e < E; ++e) top = max(top, key[e]);
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
  // What is kept: keys over `cut`, and the first `tie` that equal it.
  uint32_t cut = 0, tie = 0, least = kmax, valid = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (key[e]) least = min(least, key[e]);
    valid += __popcll(__ballot(key[e] != 0));
  }
  least = ~wave_max(~least);
  // The key at which the sum of x over the keys of [kmin, kmax] from the top reaches `need`
  // (<= all of it), and the sum above it.  First over BINS equal steps of value, `span`
  // down from the largest (the last bin takes all below): most often a token or a few are
  // left, which are taken one value after the other; else those left a byte at a time.
  auto search = [&](auto *hist, auto x, auto need, uint32_t kmin, float span, uint32_t &found, auto &above) __attribute__((always_inline)) {
    using U = std::remove_reference_t<decltype(*hist)>;
    auto clear = [&]() __attribute__((always_inline)) {
      wave_order();
#pragma unroll
      for (int i = 0; i < 4; ++i) hist[4 * lane + i] = 0;
      wave_order();
    };
    const float vmax = float_of(kmax), step = BINS / fminf(vmax - float_of(kmin), span);
    uint32_t bins[E];
    clear();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      bins[e] = static_cast<uint32_t>(fminf((vmax - float_of(key[e])) * step, BINS - 1.0f));
      if (key[e] < kmin) bins[e] = BINS;
      if (key[e] >= kmin && x(e)) atomicAdd(&hist[bins[e]], x(e));
    }
    wave_order();
    U over = 0;
    const uint32_t bin = min(bin_reaching<U>(hist, need, lane, over), static_cast<uint32_t>(BINS - 1));
    uint32_t left = 0, hi = 0, lo = ~0u;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      left += __popcll(__ballot(bins[e] == bin));
      if (bins[e] == bin) hi = max(hi, key[e]), lo = min(lo, key[e]);
    }
    hi = wave_max(hi);
    if (left <= 8) {
      for (;;) {
        U here = 0;
        uint32_t next = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          here += key[e] == hi ? x(e) : 0;
          if (bins[e] == bin && key[e] < hi) next = max(next, key[e]);
        }
        here = wave_sum(here);
        next = wave_max(next);
        if (over + here >= need || !next) break;  // (the bin's sum reaches it)
        over += here;
        hi = next;
      }
      found = hi;
      above = over;
      return;
    }
    lo = ~wave_max(~lo);
    Digits d(hi >> LOW<T>, lo >> LOW<T>);
    for (;;) {
      clear();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t k = key[e] >> LOW<T>;
        if (bins[e] == bin && x(e) && d.has(k)) atomicAdd(&hist[d.bin(k)], x(e));
      }
      wave_order();
      U a = 0;
      const uint32_t digit = min(bin_reaching<U>(hist, need - over, lane, a), static_cast<uint32_t>(BINS - 1));
      over += a;
      if (!d.next(digit)) break;
    }
    found = whole_key<T>(d.prefix);
    above = over;
  };
  // (weights below 2^-49 are 0)
  const float span = static_cast<float>(fmin(50.0 / r.c, 3.0e38));
  if (r.top_k && r.top_k < valid) {
    uint32_t over;
    search(reinterpret_cast<uint32_t *>(hists[wave]), [](int) { return 1u; }, static_cast<uint32_t>(r.top_k), least, span, cut, over);
    tie = static_cast<uint32_t>(r.top_k) - over;
  }
  const double kv = value_of(kmax);
  unsigned long long w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = key[e] && key[e] >= cut;
    w[e] = 0;
    if (__any(in)) {  // uniform
      const double y = (value_of(in ? key[e] : kmax) - kv) * r.c;
      if (in) w[e] = weight_of(y, p.shift);
    }
  }
  // of the tokens that equal the cut, those behind the first `tie` in the vocabulary's order
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
  if (r.top_p < 1.0f) {
    unsigned long long sum = 0, above;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
    const unsigned long long need = need_of(r.top_p, wave_sum(sum));
    uint32_t at;
    search(hists[wave], [&](int e) { return w[e]; }, need, max(cut, least), span, at, above);
    const uint32_t most = ties_of(need, above, weight_of((value_of(at) - kv) * r.c, p.shift));
    tie = at == cut ? min(tie, most) : most;
    cut = at;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] < cut) w[e] = 0;
    drop_ties();
  }
  const uint64_t one = uint64_t(1) << p.shift;  // the largest weight
  const uint64_t least_w = r.min_p > 0.0f ? r.min_p < 1.0f ? part_of(r.min_p, one, true) : one : 0;
  uint64_t sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (w[e] < least_w) w[e] = 0;
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

// ---------------------------------------------------------------- rows of up to 1024 E logits
// The same with a workgroup to a row, thread t logits E t .. E t + E - 1: what is left of a
// search's first pass is compared by every wave, or goes a byte at a time where it is more
// than 64 keys.  Histograms in turn, one pass clearing the next one's (whose last readers met
// before this pass).  Bound by the chain of searches (one row of 4096 bf16 logits with top-k
// and top-p 11 us), where there are many rows by the instructions of it, which every wave of a
// row runs (2048 of them 61 us, with top-p 0.95 alone 69: 1160 vector instructions a wave, some
// 100 of them the weights' 64-bit arithmetic, are 66 of the kernel's 74 us by its counters).
constexpr int SG_T = 1024, SG_W = SG_T / 64;

template <typename T, int E>
__global__ __launch_bounds__(SG_T) void sample_group_kernel(SampleArgs p) {
  __shared__ unsigned long long hist[3][BINS], few_w[64];
  __shared__ uint64_t red64[2][SG_W];
  __shared__ uint32_t red[6][SG_W], few_k[64], few[2];
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  float z[E];
  logits_of<T, E>(static_cast<const T *>(p.z) + b * p.sz, E * t, p.V, z);
  const SampleRow r = row_of(p, b);
  const float u = p.u[b];
  uint32_t key[E], top = 0, low = ~0u, valid = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    key[e] = key_of(z[e]);
    top = max(top, key[e]);
    if (key[e]) low = min(low, key[e]);
    valid += __popcll(__ballot(key[e] != 0));
  }
  top = wave_max(top);
  low = wave_max(~low);
  if (lane == 0) red[0][wave] = top, red[1][wave] = low, red[2][wave] = valid;
  if (t < BINS) hist[0][t] = 0;
  if (t < 2) few[t] = 0;
  __syncthreads();
  const uint32_t kmax = wave_max(lane < SG_W ? red[0][lane] : 0), least = ~wave_max(lane < SG_W ? red[1][lane] : 0);
  valid = wave_sum(lane < SG_W ? red[2][lane] : 0);
  if (kmax == 0) {
    if (t == 0) p.out[b] = -1;
    return;
  }
  if (r.first) {
    uint32_t at = 0;
#pragma unroll
    for (int e = E - 1; e >= 0; --e)
      if (key[e] == kmax) at = ~static_cast<uint32_t>(E * t + e);
    at = wave_max(at);
    if (lane == 0) red[3][wave] = at;
    __syncthreads();
    at = wave_max(lane < SG_W ? red[3][lane] : 0);
    if (t == 0) p.out[b] = static_cast<int64_t>(~at);
    return;
  }
  // The workgroup's inclusive sums of v, and all of it; `by`: used once.
  auto scan = [&](auto v, auto *by, auto &all) __attribute__((always_inline)) {
    const auto run = wave_scan(v);
    if (lane == 63) by[wave] = run;
    __syncthreads();
    const auto waves = wave_scan(lane < SG_W ? by[lane] : 0);
    all = lane_value(waves, SG_W - 1);
    return run + (wave ? lane_value(waves, wave - 1) : 0);
  };
  uint32_t cut = 0, tie = 0;
  int turn = 0;
  const float span = static_cast<float>(fmin(50.0 / r.c, 3.0e38));
  auto search = [&](int which, auto x, uint64_t need, uint32_t kmin, uint32_t &found, uint64_t &above) __attribute__((always_inline)) {
    const float vmax = float_of(kmax), step = BINS / fminf(vmax - float_of(kmin), span);
    uint32_t bins[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      bins[e] = key[e] >= kmin ? static_cast<uint32_t>(fminf((vmax - float_of(key[e])) * step, BINS - 1.0f)) : BINS;
    above = 0;
    auto pass = [&](auto bin_at) __attribute__((always_inline)) {
      unsigned long long *now = hist[turn], *next = hist[turn == 2 ? 0 : turn + 1];
      turn = turn == 2 ? 0 : turn + 1;
      if (t < BINS) next[t] = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t at = bin_at(e);
        if (at < BINS && x(e)) atomicAdd(&now[at], static_cast<unsigned long long>(x(e)));
      }
      __syncthreads();
      unsigned long long a = 0;
      const uint32_t bin = min(bin_reaching<unsigned long long>(now, need - above, lane, a), static_cast<uint32_t>(BINS - 1));
      above += a;
      return bin;
    };
    const uint32_t bin = pass([&](int e) __attribute__((always_inline)) { return bins[e]; });
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (bins[e] == bin) {
        const uint32_t i = atomicAdd(&few[which], 1u);
        if (i < 64) few_k[i] = key[e], few_w[i] = x(e);
      }
    __syncthreads();
    const uint32_t n = few[which];
    if (n <= 64) {  // uniform
      const bool in = static_cast<uint32_t>(lane) < n;
      const uint32_t k = in ? few_k[lane] : 0;
      const uint64_t w = in ? few_w[lane] : 0;
      uint64_t before = above, same = 0;
      for (uint32_t j = 0; j < n; ++j) {
        const uint32_t kj = lane_value(k, j);
        const uint64_t wj = lane_value(w, j);
        before += kj > k ? wj : 0;
        same += kj == k ? wj : 0;
      }
      const int l = __ffsll(static_cast<long long>(__ballot(in && before < need && need <= before + same))) - 1;
      found = lane_value(k, l);
      above = lane_value(before, l);
      return;
    }
    Digits d(kmax >> LOW<T>, kmin >> LOW<T>);
    for (;;) {
      const uint32_t digit = pass([&](int e) __attribute__((always_inline)) {
        const uint32_t k = key[e] >> LOW<T>;
        return bins[e] == bin && d.has(k) ? d.bin(k) : BINS;
      });
      if (!d.next(digit)) break;
    }
    found = whole_key<T>(d.prefix);
  };
  if (r.top_k && r.top_k < valid) {
    uint64_t over;
    search(0, [](int) { return uint64_t(1); }, r.top_k, least, cut, over);
    tie = static_cast<uint32_t>(r.top_k - over);
  }
  const double kv = value_of(kmax);
  uint64_t w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = key[e] && key[e] >= cut;
    w[e] = 0;
    if (__any(in)) {  // uniform
      const double y = (value_of(in ? key[e] : kmax) - kv) * r.c;
      if (in) w[e] = weight_of(y, p.shift);
    }
  }
  // of the tokens that equal the cut, those behind the first `tie` in the vocabulary's order
  auto drop_ties = [&](uint32_t *by) __attribute__((always_inline)) {
    uint32_t n = 0, all;
#pragma unroll
    for (int e = 0; e < E; ++e) n += key[e] == cut;
    uint32_t rank = scan(n, by, all) - n;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] == cut && rank++ >= tie) w[e] = 0;
  };
  if (cut) drop_ties(red[4]);
  if (r.top_p < 1.0f) {
    uint64_t sum = 0, all, above;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
    scan(sum, red64[0], all);
    const uint64_t need = need_of(r.top_p, all);
    uint32_t at;
    search(1, [&](int e) __attribute__((always_inline)) { return w[e]; }, need, max(cut, least), at, above);
    const uint32_t most = ties_of(need, above, weight_of((value_of(at) - kv) * r.c, p.shift));
    tie = at == cut ? min(tie, most) : most;
    cut = at;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] < cut) w[e] = 0;
    drop_ties(red[5]);
  }
  const uint64_t one = uint64_t(1) << p.shift;  // the largest weight
  const uint64_t least_w = r.min_p > 0.0f ? r.min_p < 1.0f ? part_of(r.min_p, one, true) : one : 0;
  uint64_t sum = 0, all;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (w[e] < least_w) w[e] = 0;
    sum += w[e];
  }
  const uint64_t upto = scan(sum, red64[1], all), target = target_of(u, all);
  if (upto > target && upto - sum <= target) {
    uint64_t run = upto - sum;
    int at = 0;
    for (int e = 0; e < E; ++e) {  // the first at which the sum passes the target
      run += w[e];
      if (run > target) break;
      at = e + 1;
    }
    p.out[b] = E * t + at;
  }
}

// ---------------------------------------------------------------- longer rows
// Slices of SL_T * E logits, E a thread.  sample_slice_kernel: a slice's largest logit, and a histogram over
// BINS bins of a quarter of a power of two in weight, from its largest down (the last bin
// takes all below), of its tokens in rows with top-k, else of its weights.  Bins lie on one
// grid for all slices of a row, floor(4 z c), and weights are 2^(S + z c - R) with a whole R of
// the slice's own (the row's units: its R, and an S of its own), so that histograms of slices
// add up by shifts.  A slice's sum in the row's units is that in its own, shifted once, and the
// draw looks for the token in the slice's own weights again, so that its tokens' sum reaches
// what the slice was drawn for.  Listed tokens are in the row's.  sample_join_kernel: a row's
// histogram, and the bin in which the cut lies.  sample_list_kernel: the keys of the slices'
// tokens in that bin (top-k: in all down to it), in the vocabulary's order.
// sample_draw_kernel: the exact cut among them, a byte at a time from histograms, the
// slices' sums, and the token in the slice that the draw falls into.  Bound by latency, each
// launch by the one before: one row of 131072 fp32 logits with top-p 5.0, 5.0, 4.1 and 10.8
// us; 64 rows of bf16 ones with all three cuts 14.7, 5.2, 5.4 and 12.5.  The draw's way: the
// rows' and slices' records 1.5 us, the lists 1.5, a search 2.5, the sums and
// the slice 1.5, its tokens 2.
constexpr int SL_T = 512, SL_W = SL_T / 64;
constexpr int MAX_S = 256;  // slices of the longest row, 2^20 logits
constexpr int MOST_S = 49;  // of a row (a slice's 8192 weights are then at most 2^62)

struct SliceInfo {
  double top;           // its largest logit
  uint64_t total;       // its weight, in its own units (rows without top-k)
  uint64_t base;        // of it in bins over the listed ones
  uint32_t key, at;     // largest key (0: no token) and its first index
  uint32_t listed, pad;
};
struct RowInfo {
  double top;           // the row's largest logit
  uint64_t total;       // its weight (without top-k)
  uint64_t over, bin;   // of it in bins over the listed one, and in that
  uint32_t least;       // min-p keeps keys from here on
  int32_t mode;         // 0: drawn already, 1: nothing is listed, 2: bins from lo on are
  int32_t lo;
  uint32_t from, upto;  // their keys: from .. upto - 1
  int32_t raised;       // S of the row's units is this much over the slices'
};

struct SampleWork {
  SliceInfo *slice;     // (B, S)
  RowInfo *row;         // (B,)
  uint64_t *hist;       // (B, S, BINS)
  uint32_t *list;       // (B, S * SL_T * E)
  int S;
};

// The unit of weights for a largest logit: 2^(S + z c - R), R = ceil(top c).
struct SampleRef {
  double top, c, r, phi;  // phi = top c - R
  __device__ __forceinline__ SampleRef(double t, double cc) : top(t), c(cc), r(ceil(t * cc)) { phi = t * cc - r; }
  __device__ __forceinline__ uint64_t weight(double z, int shift) const {
    return weight_of(fma(z - top, c, phi), shift);
  }
  // by: the row's units are 2^by of those of a slice with largest logit z, where S is `raised`
  // more for the row
  __device__ __forceinline__ int by(double z, int raised) const {
    return static_cast<int>(fmin(r - ceil(z * c), 4096.0)) - raised;
  }
};
// A slice's sum in the row's units (a slice of by over 62 has less than one).
__device__ __forceinline__ uint64_t in_row(uint64_t sum, int by) { return by < 0 ? sum << -by : sum >> min(by, 63); }
// floor(4 z c), where that is past 2^29 the same for all (as a whole number, so that
// differences add up).  c4: 4 c, finite.
__device__ __forceinline__ int grid_of(float z, float c4) {
  return static_cast<int>(floorf(fminf(fmaxf(z * c4, -536870912.0f), 536870912.0f)));
}
__device__ __forceinline__ int bin_of(int top_grid, float z, float c4) { return min(top_grid - grid_of(z, c4), BINS - 1); }

// Thread t's logits of slice s.
template <typename T, int E>
__device__ __forceinline__ void slice_values(const SampleArgs &p, int b, int s, int t, float (&x)[E]) {
  logits_of<T, E>(static_cast<const T *>(p.z) + b * p.sz, E * (SL_T * s + t), p.V, x);
}

template <typename T, int E>
__global__ __launch_bounds__(SL_T) void sample_slice_kernel(SampleArgs p, SampleWork w) {
  __shared__ unsigned long long hist[BINS];
  __shared__ unsigned long long sums[SL_W];
  __shared__ uint32_t red[SL_W], red2[SL_W];
  const int s = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  float z[E], top = -INFINITY;
  uint32_t at = 0;
  slice_values<T, E>(p, b, s, t, z);
  const SampleRow r = row_of(p, b);
  for (int i = t; i < BINS; i += SL_T) hist[i] = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) top = fmaxf(top, z[e]);  // (of a NaN and a number the number)
  const uint32_t wtop = wave_max(key_of(top));
  const float ztop = float_of(wtop);
#pragma unroll
  for (int e = E - 1; e >= 0; --e)  // the first of the largest, as ~index
    if (z[e] == ztop) at = ~static_cast<uint32_t>(E * (SL_T * s + t) + e);
  at = wave_max(at);
  if (lane == 0) red[wave] = wtop, red2[wave] = at;
  __syncthreads();
  uint32_t kmax = 0;
#pragma unroll
  for (int i = 0; i < SL_W; ++i) kmax = max(kmax, red[i]);
  if (kmax && !r.first) {  // uniform
    const SampleRef ref(value_of(kmax), r.c);
    const int g0 = grid_of(float_of(kmax), r.c4);
    if (r.top_k) {  // uniform: tokens; their weights are summed from the list
      uint32_t *count = reinterpret_cast<uint32_t *>(hist);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (z[e] > -INFINITY) atomicAdd(&count[bin_of(g0, z[e], r.c4)], 1u);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint64_t x = z[e] > -INFINITY ? ref.weight(wide_of(z[e]), p.shift) : 0;
        if (x) atomicAdd(&hist[bin_of(g0, z[e], r.c4)], static_cast<unsigned long long>(x));
      }
    }
  }
  __syncthreads();
  const int64_t h = (static_cast<int64_t>(b) * w.S + s) * BINS;
  unsigned long long total = 0;
  if (t < BINS) w.hist[h + t] = total = r.top_k ? reinterpret_cast<const uint32_t *>(hist)[t] : hist[t];
  total = wave_sum(total);
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  if (t == 0) {
    at = 0, total = 0;
    for (int i = 0; i < SL_W; ++i) at = red[i] == kmax ? max(at, red2[i]) : at, total += sums[i];
    SliceInfo &info = w.slice[static_cast<int64_t>(b) * w.S + s];
    info.top = kmax ? value_of(kmax) : 0.0;
    info.total = total;
    info.key = kmax;
    info.at = ~at;
  }
}

constexpr int SJ_T = 1024, SJ_G = SJ_T / BINS, SJ_E = 8;  // groups of threads take slices in turn

__global__ __launch_bounds__(SJ_T) void sample_join_kernel(SampleArgs p, SampleWork w) {
  __shared__ unsigned long long hist[BINS], totals[MAX_S / 64];
  __shared__ uint32_t red[MAX_S / 64], red2[MAX_S / 64];
  __shared__ int by[MAX_S], off[MAX_S];
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, bin = t % BINS, first = t / BINS;
  const SliceInfo *slice = w.slice + static_cast<int64_t>(b) * w.S;
  const uint64_t *h = w.hist + static_cast<int64_t>(b) * w.S * BINS + bin;
  // (all that does not depend on the row's largest is on its way at once)
  unsigned long long x[SJ_E];
#pragma unroll
  for (int i = 0; i < SJ_E; ++i) x[i] = first + SJ_G * i < w.S ? h[(first + SJ_G * i) * BINS] : 0;
  uint32_t key = 0, at = 0;
  uint64_t own = 0;
  double top = 0.0;
  if (t < w.S) key = slice[t].key, at = ~slice[t].at, top = slice[t].top, own = slice[t].total;
  const SampleRow r = row_of(p, b);
  RowInfo &row = w.row[b];
  if (t < BINS) hist[t] = 0;
  if (t < MAX_S) {
    const uint32_t k = wave_max(key), a = wave_max(key == k ? at : 0);
    if (lane == 0) red[wave] = k, red2[wave] = a;
  }
  __syncthreads();
  uint32_t kmax = 0;
#pragma unroll
  for (int i = 0; i < MAX_S / 64; ++i) kmax = max(kmax, red[i]);
  if (t == 0) {  // the first of the largest; the draw writes over it
    at = 0;
    for (int i = 0; i < MAX_S / 64; ++i) at = red[i] == kmax ? max(at, red2[i]) : at;
    p.out[b] = kmax ? static_cast<int64_t>(~at) : -1;
    if (kmax == 0 || r.first) row.mode = 0;
  }
  if (kmax == 0 || r.first) return;  // uniform
  const SampleRef ref(value_of(kmax), r.c);
  const int g0 = grid_of(float_of(kmax), r.c4);
  // The row's sum in units of the slices' S (short by less than a step a slice), which is
  // raised by the bits that leave the sum at 2^62.  A slice's bins lie `off` below the row's.
  if (t < MAX_S) {
    const int by0 = ref.by(top, 0);
    if (t < w.S) {
      by[t] = key ? r.top_k ? 0 : by0 : -1;
      off[t] = key ? min(g0 - grid_of(float_of(key), r.c4), BINS - 1) : 0;
    }
    const uint64_t sum = wave_sum(key && !r.top_k ? in_row(own, by0) : uint64_t(0));
    if (lane == 0) totals[wave] = sum;
  }
  __syncthreads();
  auto raise = [&](uint64_t sum) __attribute__((always_inline)) {
    return min(max(__clzll(static_cast<long long>(sum)) - 2, 0), MOST_S - p.shift);
  };
  uint64_t whole = MAX_S;
#pragma unroll
  for (int i = 0; i < MAX_S / 64; ++i) whole += totals[i];
  int raised = r.top_k ? 0 : raise(whole);
  auto add = [&](int s, unsigned long long v) __attribute__((always_inline)) {
    if (by[s] >= 0 && v) atomicAdd(&hist[min(bin + off[s], BINS - 1)], static_cast<unsigned long long>(in_row(v, by[s] - raised)));
  };
#pragma unroll
  for (int i = 0; i < SJ_E; ++i)
    if (first + SJ_G * i < w.S) add(first + SJ_G * i, x[i]);
#pragma unroll 4
  for (int s = first + SJ_G * SJ_E; s < w.S; s += SJ_G) add(s, h[s * BINS]);
  __syncthreads();
  if (wave) return;
  unsigned long long total = 0, before = 0, over = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) total += hist[4 * lane + i];
  total = wave_sum(total);
  // The least key of which `is` holds, as it does for all larger ones up to the largest: 64
  // probes at a time, the first ones next to each other around a guess (which is most often
  // right: one round for six).
  auto least_key = [&](float guess, auto is) __attribute__((always_inline)) {
    uint32_t below = 0, found = kmax;  // below < the key <= found
    uint32_t step = 1, first = max(key_of(guess), LEAST_KEY + 32) - 32;
    do {
      const uint32_t k = min(first + step * lane, found);
      const uint64_t yes = __ballot(k == found || (k >= LEAST_KEY && is(k)));
      const int l = __ffsll(static_cast<long long>(yes)) - 1;
      if (yes) {
        found = lane_value(k, l);
        if (l) below = lane_value(k, l - 1);
      } else {
        below = lane_value(k, 63);
      }
      step = (found - below - 1) / 64 + 1;
      first = below + step;  // (then lane 63's k is `found`)
    } while (found - below > 1);
    return found;
  };
  auto within = [&](int most) __attribute__((always_inline)) {
    return least_key(static_cast<float>((g0 - most) / static_cast<double>(r.c4)),
                     [&](uint32_t k) __attribute__((always_inline)) { return bin_of(g0, float_of(k), r.c4) <= most; });
  };
  uint32_t least = 1;
  if (r.min_p > 0.0f) {
    const double ymin = log2(static_cast<double>(fminf(r.min_p, 1.0f)));
    least = least_key(static_cast<float>(ref.top + ymin / r.c), [&](uint32_t k) __attribute__((always_inline)) {
      return (value_of(k) - ref.top) * r.c >= ymin;
    });
  }
  int lo = 0, hi = -1;
  uint64_t at_bin = 0;
  uint32_t from = 0, upto = ~0u;
  if (r.top_k) {
    hi = min(bin_reaching<unsigned long long>(hist, r.top_k, lane, before), static_cast<uint32_t>(BINS - 1));
    from = within(hi);
    // for S a bound of the listed tokens' weight: one of bin i is below 2^((1 - i) / 4) of the
    // largest, where fp32 has steps of value far below a bin's, else below the largest
    uint64_t bound = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int down = abs(g0) < (1 << 20) ? max(4 * lane + i - 2, 0) / 4 : 0;
      if (4 * lane + i <= hi) bound += hist[4 * lane + i] << max(p.shift - down, 0);
    }
    raised = raise(wave_sum(bound));
  } else {
    if (r.top_p < 1.0f) hi = bin_reaching<unsigned long long>(hist, need_of(r.top_p, total), lane, before);
    if (least > 1) {
      const int at = bin_of(g0, float_of(least), r.c4);
      hi = hi < 0 ? at : min(hi, at);
    }
    if (hi >= 0) {  // the one bin; of it what min-p keeps, where no sum of its tokens is needed
      lo = hi;
      from = r.top_p < 1.0f ? within(hi) : max(within(hi), least);
      at_bin = hist[hi];
      if (lo > 0) upto = within(lo - 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) over += 4 * lane + i < lo ? hist[4 * lane + i] : 0;
      over = wave_sum(over);
    }
  }
  if (lane == 0) {
    row.top = ref.top;
    row.total = total;
    row.over = over;
    row.bin = at_bin;
    row.least = least;
    row.mode = hi < 0 ? 1 : 2;
    row.lo = lo;
    row.from = from;
    row.upto = upto;
    row.raised = raised;
  }
}

template <typename T, int E>
__global__ __launch_bounds__(SL_T) void sample_list_kernel(SampleArgs p, SampleWork w) {
  __shared__ uint32_t red[SL_W];
  __shared__ uint64_t base[SL_W];
  const int s = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const RowInfo row = w.row[b];
  if (row.mode != 2) return;  // uniform
  SliceInfo &info = w.slice[static_cast<int64_t>(b) * w.S + s];
  float z[E];
  uint32_t n = 0, in = 0;
  slice_values<T, E>(p, b, s, t, z);
  const float from = float_of(row.from), upto = row.upto == ~0u ? NAN : float_of(row.upto);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (z[e] >= from && !(z[e] >= upto)) in |= 1u << e;  // (none of a NaN; all below no bound)
  n = __popc(in);
  // weight in bins over the listed ones, in the slice's own units (none with top-k)
  uint64_t x = 0;
  if (row.lo > 0 && t < BINS && info.key) {
    const SampleRow r = row_of(p, b);
    const int off = grid_of(static_cast<float>(row.top), r.c4) - grid_of(float_of(info.key), r.c4);
    if (min(t + min(off, BINS - 1), BINS - 1) < row.lo) x = w.hist[(static_cast<int64_t>(b) * w.S + s) * BINS + t];
  }
  x = wave_sum(x);
  const uint32_t run = wave_scan(n);
  if (lane == 63) red[wave] = run;
  if (lane == 0) base[wave] = x;
  __syncthreads();
  uint32_t at = run - n;
  for (int i = 0; i < wave; ++i) at += red[i];
  uint32_t *list = w.list + (static_cast<int64_t>(b) * w.S + s) * (SL_T * E);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (in >> e & 1) list[at++] = key_of(z[e]);
  if (t == 0) {
    uint32_t all = 0;
    uint64_t sum = 0;
    for (int i = 0; i < SL_W; ++i) all += red[i], sum += base[i];
    info.listed = all;
    info.base = sum;
  }
}

constexpr int SD_LDS = 4096;  // listed keys kept in LDS, with their weights and slices

template <typename T, int E>
__global__ __launch_bounds__(SL_T) void sample_draw_kernel(SampleArgs p, SampleWork w) {
  constexpr int SL = SL_T * E;
  __shared__ uint32_t keys[SD_LDS], start[MAX_S + 1], tied[MAX_S];
  __shared__ unsigned long long wts[SD_LDS], sums[MAX_S];
  __shared__ uint8_t of_slice[SD_LDS];
  __shared__ unsigned long long hist[3][BINS];
  __shared__ unsigned long long few_w[64];
  __shared__ uint32_t few_k[64], few[2];
  __shared__ uint64_t wred[SL_W], before_slice;
  __shared__ uint32_t red[SL_W], red2[SL_W], tie_before;
  __shared__ int pick;
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // (what does not depend on the row's state is on its way with it)
  const SliceInfo *slice = w.slice + static_cast<int64_t>(b) * w.S;
  const RowInfo row = w.row[b];
  const SampleRow r = row_of(p, b);
  const float u = p.u[b];
  SliceInfo mine{};
  if (t < w.S) mine = slice[t];
  if (row.mode == 0) return;  // uniform
  const SampleRef ref(row.top, r.c);
  const uint32_t *list = w.list + static_cast<int64_t>(b) * w.S * SL;
  const bool cuts = row.mode == 2;
  // a slice's weight apart from ties at the cut: here that in bins over the listed ones, or
  // all where nothing is listed; start[s]: listed keys before slice s
  if (t < w.S) {
    tied[t] = 0;
    sums[t] = mine.key ? in_row(cuts ? mine.base : mine.total, ref.by(mine.top, row.raised)) : 0;
  }
  uint32_t listed = 0;
  if (cuts) {
    const uint32_t run = wave_scan(t < w.S ? mine.listed : 0);
    if (lane == 63) red[wave] = run;
    if (t == 0) start[0] = 0;
    __syncthreads();
    for (int i = 0; i < wave; ++i) listed += red[i];
    if (t < w.S) start[t + 1] = listed + run;
    __syncthreads();
    listed = start[w.S];
  }
  const bool fits = listed <= SD_LDS;
  auto slice_of = [&](uint32_t i) __attribute__((always_inline)) {  // of listed key i
    int lo = 0, hi = w.S;  // start[lo] <= i < start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (start[mid] <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto fetch = [&](uint32_t i, int s) __attribute__((always_inline)) {
    return list[static_cast<int64_t>(s) * SL + (i - start[s])];
  };
  // a wave takes every SL_W-th slice, four of them at once (loads of the lists' own entries
  // behind their last as well)
  uint32_t kmin = ~0u, kmx = 0;
  if (listed) {  // uniform
#pragma unroll 1
    for (int s0 = wave; s0 < w.S; s0 += 4 * SL_W) {
      uint32_t k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = list[static_cast<int64_t>(min(s0 + SL_W * i, w.S - 1)) * SL + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = s0 + SL_W * i;
        if (s >= w.S) break;  // uniform
        const uint32_t end = start[s + 1];
        uint32_t at = start[s] + lane, key = k[i];
        while (at < end) {
          if (fits) keys[at] = key, of_slice[at] = static_cast<uint8_t>(s);
          kmin = min(kmin, key), kmx = max(kmx, key);
          at += 64;
          if (at < end) key = fetch(at, s);
        }
      }
    }
  }
  kmx = wave_max(kmx);
  kmin = ~wave_max(~kmin);
  if (lane == 0) red[wave] = kmx, red2[wave] = kmin;
  if (t == 0) pick = 0, tie_before = 0, before_slice = 0, few[0] = few[1] = 0;
  for (int i = t; i < BINS; i += SL_T) hist[0][i] = 0;
  __syncthreads();
  for (int i = 0; i < SL_W; ++i) kmx = max(kmx, red[i]), kmin = min(kmin, red2[i]);
  const int row_shift = p.shift + row.raised;
  auto weight = [&](uint32_t k) __attribute__((always_inline)) { return ref.weight(value_of(k), row_shift); };
  // f(i, key) for all listed keys
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll 1
    for (uint32_t i = t; i < listed; i += SL_T) f(i, fits ? keys[i] : fetch(i, slice_of(i)));
  };

  // What is kept of the listed: keys over `cut`, and the first `tie` that equal it, each of
  // weight `wc`.
  uint32_t cut = 0, tie = 0;
  uint64_t wc = 0;
  // Histograms in turn, one pass clearing the next one's (whose last readers met before
  // this pass), every wave reading the pass's: one meeting a pass.
  int turn = 0;
  if (cuts && listed) {
#pragma unroll 1
    for (int by_weight = r.top_k ? 0 : 1; by_weight < 2; ++by_weight) {  // top-k, top-p
      uint64_t need = r.top_k, extra = 0;  // extra: of the keys at the cut
      if (by_weight) {
        uint64_t x = 0;  // over the cut
        each([&](uint32_t i, uint32_t k) __attribute__((always_inline)) {
          const uint64_t v = k > cut ? weight(k) : 0;
          if (fits) wts[i] = v;
          x += v;
        });
        if (!(r.top_p < 1.0f)) break;
        // of what top-k kept, or of the row with its listed bin weighed as it is here: tokens
        // that are all equal then have a total of so many times their weight
        extra = tie * wc;
        x = wave_sum(x);
        if (lane == 0) wred[wave] = x;
        __syncthreads();
        uint64_t total = r.top_k ? extra : row.total - row.bin;
        for (int i = 0; i < SL_W; ++i) total += wred[i];
        need = need_of(r.top_p, total);
        if (need <= row.over) break;
        need -= row.over;
      }
      // the key at which the sum over the listed keys over the cut, from the top, reaches
      // `need`, and the sum above it.  fp32 keys of more than eight differing bits first over
      // BINS equal steps of value: few are left, which are compared with one another (10.4 ->
      // 9.9 us); many, and bf16 keys, of which most often many are equal, a byte at a time.
      Digits d(kmx >> LOW<T>, kmin >> LOW<T>);
      const float vmax = float_of(kmx), scale = BINS / (vmax - float_of(kmin));
      auto step_of = [&](uint32_t k) __attribute__((always_inline)) {
        return static_cast<uint32_t>(fminf((vmax - float_of(k)) * scale, BINS - 1.0f));  // (of a NaN the last)
      };
      unsigned long long above = 0;
      bool steps = LOW<T> == 0 && d.top > 8, found;
      uint32_t at = BINS, key = 0;  // at: the step that reaches it
      for (;;) {
        unsigned long long *now = hist[turn], *next = hist[turn == 2 ? 0 : turn + 1];
        turn = turn == 2 ? 0 : turn + 1;
        for (int i = t; i < BINS; i += SL_T) next[i] = 0;
        auto add = [&](uint32_t k, auto x) __attribute__((always_inline)) {
          if (steps) atomicAdd(&now[step_of(k)], static_cast<unsigned long long>(x()));
          else if (d.has(k >> LOW<T>) && (at == BINS || step_of(k) == at))
            atomicAdd(&now[d.bin(k >> LOW<T>)], static_cast<unsigned long long>(x()));
        };
        auto x_of = [&](uint32_t i, uint32_t k) __attribute__((always_inline)) {
          return by_weight ? fits ? static_cast<uint64_t>(wts[i]) : weight(k) : 1;
        };
        each([&](uint32_t i, uint32_t k) __attribute__((always_inline)) {
          if (k > cut) add(k, [&]() __attribute__((always_inline)) { return x_of(i, k); });
        });
        if (t == 0 && extra) add(cut, [&]() __attribute__((always_inline)) { return extra; });
        __syncthreads();
        unsigned long long a = 0;
        const uint32_t bin = bin_reaching<unsigned long long>(now, need - above, lane, a);
        found = bin < BINS;  // uniform
        above += a;
        if (!found) break;
        if (!steps) {
          if (d.next(bin)) continue;
          key = whole_key<T>(d.prefix);
          break;
        }
        steps = false;
        at = bin;
        auto put = [&](uint32_t k, uint64_t x) __attribute__((always_inline)) {
          const uint32_t i = atomicAdd(&few[by_weight], 1u);
          if (i < 64) few_k[i] = k, few_w[i] = x;
        };
        each([&](uint32_t i, uint32_t k) __attribute__((always_inline)) {
          if (k > cut && step_of(k) == at) put(k, x_of(i, k));
        });
        if (t == 0 && extra && step_of(cut) == at) put(cut, extra);
        __syncthreads();
        const uint32_t n = few[by_weight];
        if (n > 64) continue;  // uniform
        const bool in = static_cast<uint32_t>(lane) < n;
        const uint32_t k = in ? few_k[lane] : 0;
        const uint64_t x = in ? few_w[lane] : 0;
        uint64_t before = above, same = 0;
        for (uint32_t j = 0; j < n; ++j) {
          const uint32_t kj = lane_value(k, j);
          const uint64_t xj = lane_value(x, j);
          before += kj > k ? xj : 0;
          same += kj == k ? xj : 0;
        }
        const int l = __ffsll(static_cast<long long>(__ballot(in && before < need && need <= before + same))) - 1;
        key = lane_value(k, l);
        above = lane_value(before, l);
        break;
      }
      if (!found) continue;  // all of them
      const uint64_t wk = weight(key);
      const uint32_t most = ties_of(need, above, by_weight ? wk : 1);
      tie = key == cut ? min(tie, most) : most;
      cut = key;
      wc = wk;
    }
  }
  // A token's weight in the draw: over the cut and from `least` on its own, at the cut for
  // the first `tie` wc.  The slices' sums
  if (cut < row.least) wc = 0;
  each([&](uint32_t i, uint32_t k) __attribute__((always_inline)) {
    const int s = fits ? of_slice[i] : slice_of(i);
    const uint64_t x = k > cut && k >= row.least ? fits ? wts[i] : static_cast<unsigned long long>(weight(k)) : 0;
    if (x) atomicAdd(&sums[s], static_cast<unsigned long long>(x));
    if (cut && k == cut) atomicAdd(&tied[s], 1u);
  });
  __syncthreads();
  // the slice that the draw falls into
  if (wave == 0) {
    uint64_t all = 0;
    uint32_t nt = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < w.S; s0 += 64) {  // sums up to a slice's end, ties before it
      const int s = s0 + lane;
      const uint32_t n = s < w.S ? tied[s] : 0, run = wave_scan(n) + nt;
      const uint64_t upto =
          wave_scan(s < w.S ? sums[s] + (min(run, tie) - min(run - n, tie)) * wc : 0) + all;
      if (s < w.S) sums[s] = upto, tied[s] = run - n;
      nt = lane_value(run, 63);
      all = lane_value(upto, 63);
    }
    wave_order();
    const uint64_t target = all ? target_of(u, all) : 0;
#pragma unroll 1
    for (int s0 = 0; s0 < w.S; s0 += 64) {
      const int s = s0 + lane;
      const uint64_t hit = __ballot(s < w.S && sums[s] > target);
      if (hit) {
        if (lane == __ffsll(static_cast<long long>(hit)) - 1)
          pick = s, before_slice = target - (s ? sums[s - 1] : 0), tie_before = tied[s];
        break;
      }
    }
  }
  __syncthreads();
  // the token: thread t has logits E t .. of the slice, of which those that are kept
  // (most often a few hundred) go to LDS in their order, for a weight a thread
  float *vals = reinterpret_cast<float *>(wts);
  uint16_t *ids = reinterpret_cast<uint16_t *>(keys);
  static_assert(SL * sizeof(float) <= sizeof(wts) && SL * sizeof(uint16_t) <= sizeof(keys), "");
  const float at_cut = cut ? float_of(cut) : NAN, over = cut ? at_cut : -INFINITY;
  const uint32_t least = max(row.from, row.least);
  const float from = least > LEAST_KEY ? float_of(least) : -INFINITY;
  const double own_top = slice[pick].top;
  float z[E];
  slice_values<T, E>(p, b, pick, t, z);
  uint32_t n = 0;  // kept, and in the upper half those at the cut
#pragma unroll
  for (int e = 0; e < E; ++e) n += z[e] == at_cut ? 0x10001u : z[e] > over && z[e] >= from ? 1u : 0u;
  uint32_t run = wave_scan(n);
  if (lane == 63) red[wave] = run;
  __syncthreads();
  uint32_t entries = 0;
  run -= n;
  for (int i = 0; i < SL_W; ++i) {
    if (i < wave) run += red[i];
    entries += red[i] & 0xffffu;
  }
  uint32_t rank = tie_before + (run >> 16), to = run & 0xffffu;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool tied_here = z[e] == at_cut;
    if (tied_here || (z[e] > over && z[e] >= from)) {
      vals[to] = tied_here && rank >= tie ? -INFINITY : z[e];  // (no weight)
      ids[to++] = static_cast<uint16_t>(E * t + e);
      rank += tied_here;
    }
  }
  __syncthreads();
  // The slice's sum was one of its own weights, in units of which the row's are 2^by, for the
  // tokens over the listed ones, and of the row's weights for those: so it is here, in the
  // finer of the two units, and passes the target.  (8192 weights of a slice are at most 2^62;
  // a listed one that rounds to any step of the row's is at most doubled by that: 2^63.)  For
  // u >= 1 it is the slice's last token of any weight.
  const SampleRef own(own_top, r.c);
  const int by = min(ref.by(own_top, row.raised), 63), up = max(by, 0), own_up = max(-by, 0);
  const float over_listed = !cuts ? -INFINITY : row.upto == ~0u ? NAN : float_of(row.upto);
  const uint64_t target = u >= 1.0f ? ~uint64_t(0) : before_slice << up;
  uint64_t before = 0;
  uint32_t last = 0;
#pragma unroll 1
  for (uint32_t c = 0; c < entries; c += SL_T) {
    const uint32_t i = c + t;
    const float v = i < entries ? vals[i] : -INFINITY;
    uint64_t x = 0;
    if (v > -INFINITY) {
      const bool listed = !(v >= over_listed);
      x = v == at_cut ? wc : (listed ? ref : own).weight(wide_of(v), listed ? row_shift : p.shift);
      x <<= listed ? up : own_up;
    }
    if (x) last = i + 1;
    const uint64_t sum = wave_scan(x);
    if (lane == 63) wred[wave] = sum;
    __syncthreads();
    uint64_t upto = before + sum;
    for (int k = 0; k < SL_W; ++k) {
      if (k < wave) upto += wred[k];
      before += wred[k];
    }
    if (before > target) {  // uniform
      if (upto > target && upto - x <= target) p.out[b] = static_cast<int64_t>(SL) * pick + ids[i];
      return;
    }
    __syncthreads();
  }
  const uint32_t wlast = wave_max(last);
  if (lane == 0) red2[wave] = wlast;
  __syncthreads();
  uint32_t at = 0;
  for (int k = 0; k < SL_W; ++k) at = max(at, red2[k]);
  if (t == 0 && at) p.out[b] = static_cast<int64_t>(SL) * pick + ids[at - 1];
}

static int64_t align16(int64_t n) { return (n + 15) & ~int64_t(15); }

// Logits a thread: 8, where that is one round of workgroups (four a CU), else 16 (rows of
// 131072 bf16 logits with top-p 0.95: 512 of them 154 us, with 8 179; 64 of them 43.5, with 8
// 44.1, without any cut 39.1 and 34.4; 8 of them 25.3, with 16 28.8; 512 rows of 20011 51.6, with
// 8 48.5).
static int logits_a_thread(int64_t B, int64_t V) { return B * cdiv(V, SL_T * 8) <= 1024 ? 8 : 16; }

// Offsets of the parts of a workspace; the last is its size.
struct SampleParts {
  int64_t S, row, hist, list, bytes;
};
static SampleParts parts_of(int64_t B, int64_t V) {
  const int64_t size = static_cast<int64_t>(SL_T) * logits_a_thread(B, V), S = cdiv(V, size);
  SampleParts q;
  q.S = S;
  q.row = align16(B * S * static_cast<int64_t>(sizeof(SliceInfo)));
  q.hist = q.row + align16(B * static_cast<int64_t>(sizeof(RowInfo)));
  q.list = q.hist + B * S * BINS * 8;
  q.bytes = q.list + B * S * size * 4;
  return q;
}

constexpr int64_t SAMPLE_WAVE = 1024;  // logits of a row that a wave takes
// Rows that a workgroup takes by itself (us, bf16 rows with top-p 0.95: one of 4096 logits 12,
// over slices 18, 2048 of them 74, over slices 82; one of 8192 14 and 19, 512 of them 34 and
// 32), of more logits than a wave takes.
static bool by_group(int64_t B, int64_t V) { return V <= 4 * SG_T || (V <= 8 * SG_T && B <= 256); }
constexpr int64_t SAMPLE_MOST = static_cast<int64_t>(MAX_S) * SL_T * 8;

template <typename T, int E>
static int launch_slices(const SampleArgs &a, int64_t B, char *ws, bool listed, hipStream_t st) {
  const SampleParts q = parts_of(B, a.V);
  const SampleWork w{reinterpret_cast<SliceInfo *>(ws), reinterpret_cast<RowInfo *>(ws + q.row),
                     reinterpret_cast<uint64_t *>(ws + q.hist), reinterpret_cast<uint32_t *>(ws + q.list),
                     static_cast<int>(q.S)};
  const dim3 grid(static_cast<unsigned>(w.S), static_cast<unsigned>(B));
  hipLaunchKernelGGL((sample_slice_kernel<T, E>), grid, dim3(SL_T), 0, st, a, w);
  int rc = check_launch("sample slices");
  if (rc) return rc;
  hipLaunchKernelGGL(sample_join_kernel, dim3(static_cast<unsigned>(B)), dim3(SJ_T), 0, st, a, w);
  if ((rc = check_launch("sample join"))) return rc;
  if (listed) {
    hipLaunchKernelGGL((sample_list_kernel<T, E>), grid, dim3(SL_T), 0, st, a, w);
    if ((rc = check_launch("sample list"))) return rc;
  }
  hipLaunchKernelGGL((sample_draw_kernel<T, E>), dim3(static_cast<unsigned>(B)), dim3(SL_T), 0, st, a, w);
  return check_launch("sample draw");
}

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
  if (by_group(B, a.V)) {
    const dim3 grid(static_cast<unsigned>(B));
    if (a.V <= 4 * SG_T) hipLaunchKernelGGL((sample_group_kernel<T, 4>), grid, dim3(SG_T), 0, st, a);
    else hipLaunchKernelGGL((sample_group_kernel<T, 8>), grid, dim3(SG_T), 0, st, a);
    return check_launch("sample");
  }
  return logits_a_thread(B, a.V) == 8 ? launch_slices<T, 8>(a, B, ws, listed, st) : launch_slices<T, 16>(a, B, ws, listed, st);
}

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_sample_workspace_bytes(int64_t B, int64_t V) {
  if (B <= 0 || by_group(B, V) || V > SAMPLE_MOST || B > 65535) return 0;
  return parts_of(B, V).bytes;
}

extern "C" int evo2_sample(const void *logits, int32_t fp32, int64_t sz, const float *u, const float *temperature,
                           float t1, const int32_t *top_k, int64_t k1, const float *top_p, float p1,
                           const float *min_p, float m1, void *workspace, int64_t workspace_bytes, int64_t *tokens,
                           int64_t B, int64_t V, void *stream) {
  if (B < 0 || V <= 0 || V > SAMPLE_MOST)
    return fail(EVO2_ERR_INVALID, "sample: bad sizes B=%lld V=%lld", (long long)B, (long long)V);
  if (B == 0) return EVO2_OK;
  if (!logits || !u || !tokens) return fail(EVO2_ERR_INVALID, "sample: null pointer argument");
  if (sz < V && B > 1) return fail(EVO2_ERR_UNSUPPORTED, "sample: rows must not overlap");
  if (!by_group(B, V) ? B > 65535 : !grid_fits(V > SAMPLE_WAVE ? B : cdiv(B, 4), V > SAMPLE_WAVE ? SG_T : 256))
    return fail(EVO2_ERR_UNSUPPORTED, "sample: more workgroups than a launch takes");
  if (workspace_bytes < evo2_sample_workspace_bytes(B, V) || (!by_group(B, V) && !workspace) ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(EVO2_ERR_INVALID, "sample: workspace too small or not 16-byte aligned");
  // S: a row's weights stay at 2^62 or below, one below 2^52
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

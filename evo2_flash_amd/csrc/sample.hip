// The next token of each row of logits from a given uniform number, behind the decoder's
// head (model.py:343-348): temperature, then top-k, top-p of what top-k left, and min-p.
//
//   x_i = (z_i - max z) / T,  w_i = exp(x_i)
//   the tokens in order of (z descending, index ascending):
//     top-k keeps the first k, top-p of those the shortest front whose weights reach
//     p times theirs, min-p those with w_i >= m
//   the token is the first index i, in the vocabulary's order, with
//     sum_{j <= i, kept} w_j > u * sum_{kept} w_j
//
// Each of the three keeps a front of one order, so what they keep together is all tokens
// above some value and the first few of those that equal it: the kernels look for that
// (value, number) by counting, without sorting.  Values become whole numbers in the same
// order (-0 as 0; -inf and NaN below all, never drawn), and the cut is found a byte at a
// time from histograms of counts (top-k) and of weights (top-p).
//
// Weights are whole numbers, round(w_i 2^S) with 2^S V < 2^62: sums of them are exact and
// the same in any order, also through atomics, and steps of 2^-S of the largest weight
// (2^-44 at 262144 tokens) decide no draw that 64-bit floating point would settle.
#include <type_traits>

#include "common.h"

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

// Whole numbers in the order of the values; 0: not a token (-inf, NaN).
__device__ __forceinline__ uint32_t key_of(float z) {
  if (!(z > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(z + 0.0f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <typename T>
__device__ __forceinline__ float logit(const T *z, int i) {
  if constexpr (std::is_same_v<T, float>) return z[i];
  else return bf2f(z[i]);
}

struct SampleRow {
  uint32_t kmax;
  double top, rt, xmin, one;  // largest value, 1 / T, log m, 2^S
  __device__ __forceinline__ double x_of(uint32_t key) const {
    return key == kmax ? 0.0 : (static_cast<double>(value_of(key)) - top) * rt;
  }
  __device__ __forceinline__ uint64_t weight_x(double x) const {  // (an undefined x: an infinite maximum)
    return x > -50.0 ? static_cast<uint64_t>(rint(exp(x) * one)) : 0;
  }
  __device__ __forceinline__ uint64_t weight(uint32_t key) const { return weight_x(x_of(key)); }
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d), hi = __shfl_up(static_cast<uint32_t>(v >> 32), d);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  const uint32_t lo = __shfl(static_cast<uint32_t>(v), lane), hi = __shfl(static_cast<uint32_t>(v >> 32), lane);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = shfl_up64(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// The bin of hist (256) in which the sum from the top reaches `need`, and the sum above
// it; 256 if all of them do not.  One wave.
__device__ __forceinline__ int bin_reaching(const unsigned long long *hist, uint64_t need, int lane, uint64_t &above) {
  uint64_t h[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum += h[i] = hist[255 - 4 * lane - i];
  const uint64_t run = wave_scan(sum, lane);
  const uint64_t hit = __ballot(run >= need);
  if (!hit) return 256;
  const int l = __ffsll(static_cast<long long>(hit)) - 1;
  uint64_t a = run - sum;
  int bin = 255 - 4 * lane;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (a + h[i] < need && bin == 255 - 4 * lane - i) {
      a += h[i];
      --bin;
    }
  above = shfl64(a, l);
  return __shfl(bin, l);
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_row_kernel(SampleArgs p) {
  constexpr int NW = THREADS / 64;
  __shared__ unsigned long long hist[256];
  __shared__ unsigned long long seg[NW];
  __shared__ uint32_t ties[NW], red[NW];
  __shared__ uint64_t found_above;
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = p.V;
  const T *z = static_cast<const T *>(p.z) + b * p.sz;
  const float temp = p.t ? p.t[b] : p.t1, top_p = p.p ? p.p[b] : p.p1, min_p = p.m ? p.m[b] : p.m1;
  const int64_t top_k = p.k ? p.k[b] : p.k1;

  auto block_max = [&](uint32_t v) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o)));
    if (lane == 0) red[wave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v = max(v, red[w]);
    __syncthreads();
    return v;
  };
  SampleRow r;
  uint32_t km = 0;
  for (int i = tid; i < V; i += THREADS) km = max(km, key_of(logit(z, i)));
  r.kmax = block_max(km);
  if (r.kmax == 0) {  // uniform: nothing is left
    if (tid == 0) p.out[b] = -1;
    return;
  }
  if (!(temp > 0.0f) || top_k == 1) {  // uniform: the first of the largest
    uint32_t at = 0;  // (as ~index, so that the largest is the first)
    for (int i = tid; i < V; i += THREADS)
      if (key_of(logit(z, i)) == r.kmax) at = max(at, ~static_cast<uint32_t>(i));
    at = block_max(at);
    if (tid == 0) p.out[b] = static_cast<int64_t>(~at);
    return;
  }
  r.top = value_of(r.kmax);
  r.rt = 1.0 / static_cast<double>(temp);
  r.xmin = min_p > 0.0f ? log(static_cast<double>(fminf(min_p, 1.0f))) : -INFINITY;
  r.one = ldexp(1.0, p.shift);

  // What is kept: keys over `cut`, and the first `tie` that equal it.
  uint32_t cut = 0, tie = 0;
  // The key at which sum_{kept}(of(key)) from the top reaches `need`, and the sum above
  // that key; false where all of them do not reach it.  `extra`: of the keys at `cut`.
  auto search = [&](auto of, uint64_t need, uint64_t extra, uint32_t &key, uint64_t &above) __attribute__((always_inline)) {
    uint32_t prefix = 0;
    uint64_t over = 0;
    for (int sh = 24; sh >= 0; sh -= 8) {
      for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
      __syncthreads();
      const uint32_t mask = sh == 24 ? 0u : 0xffffffffu << (sh + 8);
      for (int i = tid; i < V; i += THREADS) {
        const uint32_t k = key_of(logit(z, i));
        if (k > cut && (k & mask) == prefix) atomicAdd(&hist[k >> sh & 255], static_cast<unsigned long long>(of(k)));
      }
      if (tid == 0 && extra && (cut & mask) == prefix) atomicAdd(&hist[cut >> sh & 255], static_cast<unsigned long long>(extra));
      __syncthreads();
      if (wave == 0) {
        uint64_t a = 0;
        const int bin = bin_reaching(hist, need - over, lane, a);
        if (lane == 0) {
          found = bin;
          found_above = a;
        }
      }
      __syncthreads();
      if (found == 256) return false;  // uniform
      prefix |= static_cast<uint32_t>(found) << sh;
      over += found_above;
      __syncthreads();
    }
    key = prefix;
    above = over;
    return true;
  };
  if (top_k > 0 && top_k < V) {
    uint32_t key;
    uint64_t above;
    if (search([](uint32_t) { return uint64_t(1); }, static_cast<uint64_t>(top_k), 0, key, above)) {
      cut = key;
      tie = static_cast<uint32_t>(top_k - above);
    }
  }
  if (top_p < 1.0f) {
    const uint64_t extra = cut ? tie * r.weight(cut) : 0;
    uint64_t sum = 0;
    for (int i = tid; i < V; i += THREADS) {
      const uint32_t k = key_of(logit(z, i));
      if (k > cut) sum += r.weight(k);
    }
    sum = shfl64(wave_scan(sum, lane), 63);
    if (lane == 0) seg[wave] = sum;
    __syncthreads();
    uint64_t total = extra;
#pragma unroll
    for (int w = 0; w < NW; ++w) total += seg[w];
    // the least whole number that is not below p * total
    const double want = top_p > 0.0f ? ceil(static_cast<double>(top_p) * static_cast<double>(total)) : 1.0;
    const uint64_t need = min(max(static_cast<uint64_t>(want), uint64_t(1)), total);
    uint32_t key;
    uint64_t above;
    if (search([&](uint32_t k) { return r.weight(k); }, need, extra, key, above)) {
      const uint64_t w = r.weight(key);
      const uint64_t most = w ? (need - above + w - 1) / w : 0xffffffffull;
      if (key > cut) tie = static_cast<uint32_t>(min(most, uint64_t(0xffffffff)));
      else tie = static_cast<uint32_t>(min(most, static_cast<uint64_t>(tie)));
      cut = key;
    }
  }

  // Draw: a wave sums a stretch of the vocabulary.
  const int per = ((V + NW - 1) / NW + 63) / 64 * 64, v0 = min(wave * per, V), v1 = min(v0 + per, V);
  const double xc = cut ? r.x_of(cut) : 0.0;
  const uint64_t wc = cut && xc >= r.xmin ? r.weight_x(xc) : 0;
  auto weigh = [&](uint32_t k) __attribute__((always_inline)) -> uint64_t {  // of a key over the cut
    if (k <= cut) return 0;
    const double x = r.x_of(k);
    return x >= r.xmin ? r.weight_x(x) : 0;
  };
  uint64_t sum = 0;
  uint32_t nt = 0;
  for (int i = v0 + lane; i < v1; i += 64) {
    const uint32_t k = key_of(logit(z, i));
    sum += weigh(k);
    nt += cut && k == cut;
  }
  sum = shfl64(wave_scan(sum, lane), 63);
  nt = static_cast<uint32_t>(shfl64(wave_scan(nt, lane), 63));
  __syncthreads();  // (the sums of top-p have been read)
  if (lane == 0) {
    seg[wave] = sum;
    ties[wave] = nt;
  }
  __syncthreads();
  uint64_t total = 0;
  uint32_t before = 0;  // ties in earlier stretches
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const uint32_t kept = min(ties[w], tie - min(tie, before));
    total += seg[w] + kept * wc;
    before += ties[w];
  }
  const double pick = static_cast<double>(p.u[b]) * static_cast<double>(total);
  const uint64_t target = pick > 0.0 ? min(static_cast<uint64_t>(fmin(pick, 9.0e18)), total - 1) : 0;
  uint64_t run = 0;
  before = 0;
  for (int w = 0; w < NW; ++w) {  // uniform
    const uint32_t kept = min(ties[w], tie - min(tie, before));
    const uint64_t here = seg[w] + kept * wc;
    if (run + here > target) {
      if (wave != w) return;
      for (int i0 = v0; i0 < v1; i0 += 64) {
        const int i = i0 + lane;
        const uint32_t k = i < v1 ? key_of(logit(z, i)) : 0;
        const uint64_t eq = __ballot(cut && k == cut);
        const uint32_t rank = before + __popcll(eq & ((1ull << lane) - 1));
        const uint64_t mine = cut && k == cut ? (rank < tie ? wc : 0) : weigh(k);
        const uint64_t upto = run + wave_scan(mine, lane);
        const uint64_t over = __ballot(upto > target);
        if (over) {
          if (lane == 0) p.out[b] = i0 + __ffsll(static_cast<long long>(over)) - 1;
          return;
        }
        run = shfl64(upto, 63);
        before += __popcll(eq);
      }
      return;
    }
    run += here;
    before += ties[w];
  }
}

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_sample_workspace_bytes(int64_t B, int64_t V) { return 0; }

extern "C" int evo2_sample(const void *logits, int32_t fp32, int64_t sz, const float *u, const float *temperature,
                           float t1, const int32_t *top_k, int64_t k1, const float *top_p, float p1,
                           const float *min_p, float m1, void *workspace, int64_t workspace_bytes, int64_t *tokens,
                           int64_t B, int64_t V, void *stream) {
  if (B < 0 || V <= 0 || V > (1 << 24))
    return fail(EVO2_ERR_INVALID, "sample: bad sizes B=%lld V=%lld", (long long)B, (long long)V);
  if (B == 0) return EVO2_OK;
  if (!logits || !u || !tokens) return fail(EVO2_ERR_INVALID, "sample: null pointer argument");
  if (sz < V && B > 1) return fail(EVO2_ERR_UNSUPPORTED, "sample: rows must not overlap");
  int bits = 0;
  while ((int64_t(1) << bits) < V) ++bits;
  const SampleArgs a{logits, sz, u, temperature, t1, top_k, k1, top_p, p1, min_p, m1, tokens, static_cast<int>(V),
                     bits > 12 ? 61 - bits : 49};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (!grid_fits(B, 1024)) return fail(EVO2_ERR_UNSUPPORTED, "sample: more workgroups than a launch takes");
  if (V <= 4096) {
    if (fp32) hipLaunchKernelGGL((sample_row_kernel<float, 256>), dim3(static_cast<unsigned>(B)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((sample_row_kernel<bf16_t, 256>), dim3(static_cast<unsigned>(B)), dim3(256), 0, s, a);
  } else {
    if (fp32) hipLaunchKernelGGL((sample_row_kernel<float, 1024>), dim3(static_cast<unsigned>(B)), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((sample_row_kernel<bf16_t, 1024>), dim3(static_cast<unsigned>(B)), dim3(1024), 0, s, a);
  }
  return check_launch("sample");
}

// Causal self-attention of packed sequences with its backward pass, for scoring and
// training the attention layers (evo2_flash/model.py:104-153 leaves both to its
// engine).  Rows of q, k and v are token-major views of any strides (the qkv
// projection's own rows), sequence s takes rows cu[s] .. cu[s + 1] - 1, `heads` query
// heads share `kv` key heads:
//   p_ij = softmax_{j <= i}(scale q_i . k_j), o = p v
//   dv = p^T do, dp = do v^T, ds = p (dp - delta), delta_i = sum_j p_ij dp_ij = do_i . o_i
//   dq = scale ds k, dk = scale ds^T q
//
// Three kernels of one shape, waves of 32 rows each (four; four or eight for dk and dv)
// over tiles of 64 rows that come through LDS by direct-to-LDS loads, double-buffered,
// one barrier a tile:
//   forward  32 queries a wave, sweeping keys and values:  s^T = k q^T, o^T += v^T p^T
//   dq       32 queries a wave, sweeping keys and values:  s^T, dp^T = v do^T,
//            dq^T += k^T ds^T
//   dk, dv   32 keys a wave, sweeping the queries and do of every head that shares
//            them: s = q k^T, dp = do v^T, dv^T += do^T p, dk^T += q^T ds
// all on v_mfma_f32_32x32x16_bf16 with the sweeping operand as A and the wave's rows as
// B, so that a lane (n, g) holds the products of its row n with rows 8 q + 4 g + i of a
// 32-row tile; those, as bf16, are the B operand of the second product as they stand
// (K slot (g, j) of step kp is row 16 kp + 8 (j / 4) + 4 g + j % 4), whose A operand is
// the tile read transposed out of LDS (ds_read_b64_tr_b16).  Each output is summed by
// one wave in a fixed order: no atomics, so results repeat bit for bit; the price is
// that the backward pass computes s and dp twice (seven products for five).
//
// LDS holds a tile as the load instructions' blocks of 1 KB (four rows of 128, eight of
// 64), 16 bytes apart, 16-byte chunk c of a block's row i at c ^ p_swizzle(i): the 16
// rows of a 16-byte read and the four rows of a transposing read fall on distinct
// banks, and few addresses are not constant offsets of one another.
//
// Scores, softmax statistics and sums are fp32; p and ds are rounded to bf16 as
// operands, the results once.  The forward pass keeps each row's log-sum-exp and, for
// the backward pass, what rounding took from o (as bf16): delta from the rounded o
// alone would put a second rounding under ds.  A row with a single key has p = 1
// whatever its score: its ds is exactly 0.
#include "attn_common.h"

namespace evo2 {

typedef __attribute__((ext_vector_type(16))) float pf32x16_t;
typedef __attribute__((ext_vector_type(4))) short ps16x4_t;
typedef __attribute__((address_space(3))) ps16x4_t plds_s16x4_t;

constexpr int P_NW = 4;             // waves per workgroup
constexpr int P_WR = 32;            // rows a wave owns
constexpr int P_WG = P_NW * P_WR;   // rows a workgroup owns
constexpr int P_TR = 64;            // rows per swept tile
constexpr int P_FILL = 32;          // workgroups that clear rows outside the sequences
constexpr float P_SLACK = 8.0f;     // log2 headroom of the reference max

// Keeps a wave-uniform condition a branch: the masks of the few tiles on the diagonal
// were computed for every tile otherwise, a third of the vector instructions.
#define P_BRANCH asm volatile("")

struct Rows {                       // (T, heads, HD) bf16, unit last stride
  const bf16_t *p;
  int64_t st, sh;
};

struct PackedArgs {
  Rows q, k, v, d;                  // d: do
  const int32_t *cu;
  int nseq, T, heads, kv;
  int tiles;                        // row-tile slots: T / (rows of a workgroup) + nseq
  int items;                        // workgroups that own rows; P_FILL follow
  float c2, scale;                  // scale * log2(e), scale
  bf16_t *out, *lo;                 // (T, heads, HD)
  float *lse;                       // (heads, T), log2 units
  const bf16_t *o, *olo;
  float *delta;                     // (heads, T): -delta
  bf16_t *dq, *dk, *dv;
  float *part;                      // (heads, T, 2, HD): dk and dv by query head
};

constexpr int P_BLK = 520;          // elements from one 1 KB block to the next

template <int HD>
__device__ __forceinline__ int p_swizzle(int i) {
  return HD == 128 ? (i & 3) << 2 : (((i >> 1) & 1) << 2) | (((i >> 2) & 1) << 1);
}
// Elements a tile of `rows` rows takes, and where chunk c of its row r is.
template <int HD>
constexpr int p_tile(int rows) { return rows * HD / 512 * P_BLK; }
template <int HD>
__device__ __forceinline__ int p_at(int r, int c) {
  constexpr int RPI = 512 / HD;
  return r / RPI * P_BLK + r % RPI * HD + 8 * (c ^ p_swizzle<HD>(r % RPI));
}

// Rows of sequence s, inside the tensor whatever the table holds.
__device__ __forceinline__ void p_bounds(const PackedArgs &p, int s, int &begin, int &len) {
  begin = min(max(p.cu[s], 0), p.T);
  len = min(max(p.cu[s + 1], begin), p.T) - begin;
}

// Slot t of the tiles of `rows` rows: sequence s's start at cu[s] / rows + s, which leaves
// it at least as many as it needs, so a slot finds its sequence, the last that starts at
// or before it, from the table alone (a search by 64ths, one load a step) and the host
// never reads it.  False: nothing there.
__device__ __forceinline__ bool p_slot(const PackedArgs &p, int t, int lane, int rows, int &begin, int &len,
                                      int &r0) {
  int s = 0;  // it is among s .. s + n - 1
  for (int n = p.nseq, step; n > 0; n = min(step, n)) {
    step = (n - 1) / 64 + 1;
    const int i = s + lane * step;  // (below 2^31: step is at most nseq / 64 + 1)
    const bool at = i < s + n && min(max(p.cu[i], 0), p.T) / rows + i <= t;
    const int c = __popcll(__ballot(at));
    if (c == 0) return false;  // (none starts at or before the slot: the first step's only)
    s += (c - 1) * step;
    n -= (c - 1) * step;
    if (step == 1) break;
  }
  if (p.nseq == 0) return false;
  p_bounds(p, s, begin, len);
  r0 = (t - begin / rows - s) * rows;
  return r0 >= 0 && r0 < len;
}

// Workgroup -> (head, row-tile slot).  Whole heads per XCD (workgroup b runs on XCD
// b mod 8) where they split evenly, so that an XCD's workgroups sweep the same rows
// through its L2; the longest sweeps of all its heads first (reversed: those of the last
// queries), so that what is left at the end is short: head by head, 8192 tokens of 32
// heads of 128 took 609, 812 and 1321 us forward, for dq and for dk, dv, so 588, 770 and
// 1282.
__device__ __forceinline__ void p_item(int w, int heads, int tiles, bool reversed, int &h, int &t) {
  if (heads % 8 == 0) {
    const int j = w >> 3, per = heads >> 3;
    t = j / per;
    h = (w & 7) + 8 * (j - t * per);
  } else {
    t = w / heads;
    h = w - t * heads;
  }
  if (reversed) t = tiles - 1 - t;
}

// Clears the rows of a (T, n) output that no sequence holds.
__device__ __forceinline__ void p_clear(const PackedArgs &p, bf16_t *out, int n, int part) {
  const int first = min(max(p.cu[0], 0), p.T), last = min(max(p.cu[p.nseq], first), p.T);
  const int64_t head = static_cast<int64_t>(first) * n / 8, tail = static_cast<int64_t>(p.T - last) * n / 8;
  au32x4_t *a = reinterpret_cast<au32x4_t *>(out);
  au32x4_t *b = reinterpret_cast<au32x4_t *>(out + static_cast<int64_t>(last) * n);
  const au32x4_t zero = {0, 0, 0, 0};
  for (int64_t i = part * 256 + threadIdx.x; i < head; i += P_FILL * 256) a[i] = zero;
  for (int64_t i = part * 256 + threadIdx.x; i < tail; i += P_FILL * 256) b[i] = zero;
}

// One workgroup's loads of tiles of P_TR rows: lane i of load block j fills physical
// chunk i % CH of row RPI j + i / CH; wave w takes blocks w, w + NW, .., whose rows
// share the swizzle.
template <int HD, int NW = P_NW>
struct TileLoad {
  static constexpr int CH = HD / 8, RPI = 64 / CH, PER = P_TR / RPI / NW;
  const bf16_t *p;
  int64_t st;
  uint32_t voff;
  int wave;
  __device__ __forceinline__ void init(const bf16_t *ptr, int64_t stride, int w, int lane) {
    p = ptr;
    st = stride;
    wave = w;
    const int r = lane / CH;
    voff = static_cast<uint32_t>(r) * static_cast<uint32_t>(st * 2) +
           16u * ((lane % CH) ^ p_swizzle<HD>(r));
  }
  // rows row0 .. of the sequence's `len`; the rest of the tile reads zeros
  __device__ __forceinline__ void issue(bf16_t *lds, int row0, int len) const {
    const int rows = min(P_TR, len - row0);
    const uint32_t bytes = rows > 0 ? static_cast<uint32_t>(((rows - 1) * st + HD) * 2) : 0u;
    const au32x4_t rs = lds_rsrc(p + row0 * st, bytes);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = wave + NW * i;
      lds_load(rs, voff + static_cast<uint32_t>(j * RPI) * static_cast<uint32_t>(st * 2), lds + P_BLK * j);
    }
  }
};

// A operand of the first product: rows 32 t + lr of a tile, K step kk.
template <int HD>
__device__ __forceinline__ abf16x8_t p_rows(const bf16_t *tile, int t, int kk, int lr, int g) {
  return __builtin_bit_cast(abf16x8_t, *reinterpret_cast<const au32x4_t *>(
                                           tile + t * p_tile<HD>(32) + p_at<HD>(lr, 2 * kk + g)));
}

// A operand of the second product, transposed: columns 32 e .. + 31 as its rows, K
// step kp of the tile (rows 16 kp + 8 (j / 4) + 4 g + j % 4).
template <int HD>
__device__ __forceinline__ abf16x8_t p_cols(const bf16_t *tile, int e, int kp, int lane) {
  const int ti = lane & 15, tq = lane >> 4;
  const bf16_t *a = tile + kp * p_tile<HD>(16) + 4 * (ti & 1) +
                    p_at<HD>(4 * (tq >> 1) + (ti >> 2), 4 * e + 2 * (tq & 1) + ((ti & 3) >> 1));
  const ps16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((plds_s16x4_t *)a);
  const ps16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((plds_s16x4_t *)(a + p_tile<HD>(8)));
  return __builtin_bit_cast(abf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// B operand: eight products of a lane as bf16.
__device__ __forceinline__ abf16x8_t p_pack(const pf32x16_t &s, int half) {
  au32x4_t u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = pack_bf(s[8 * half + 2 * i], s[8 * half + 2 * i + 1]);
  return __builtin_bit_cast(abf16x8_t, u);
}

// Max of lanes l and l + 32, in both (by a swap of registers: a shuffle through LDS waits
// for the fragments read before it; 8192 tokens, 32 heads of 64 on 8: 322 -> 303 us).
__device__ __forceinline__ float p_max_pair(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// A wave's own rows as B operands: row lr, K step kk.
template <int HD>
__device__ __forceinline__ void p_own(abf16x8_t (&f)[HD / 16], const Rows &r, int64_t row, int h, int g) {
  const bf16_t *p = r.p + row * r.st + h * r.sh + 8 * g;
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk)
    f[kk] = __builtin_bit_cast(abf16x8_t, *reinterpret_cast<const au32x4_t *>(p + 16 * kk));
}

// acc^T (HD x 32 rows) times f to a row of bf16: lanes l and l + 32 hold the same row
// and swap halves of each pair of column groups, so each stores 16 bytes.  lo: what
// the rounding took, as bf16.
template <int HD>
__device__ __forceinline__ void p_store(const pf32x16_t (&acc)[HD / 32], float f, bf16_t *row, bf16_t *lo, int g,
                                        bool live) {
#pragma unroll
  for (int e = 0; e < HD / 32; ++e)
#pragma unroll
    for (int pq = 0; pq < 2; ++pq) {
      float v[8], r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = acc[e][8 * pq + i] * f;
        r[i] = v[i] - rbf(v[i]);
      }
      const int c = 32 * e + 16 * pq + 8 * g;
      const auto s0 = __builtin_amdgcn_permlane32_swap(pack_bf(v[0], v[1]), pack_bf(v[4], v[5]), false, false);
      const auto s1 = __builtin_amdgcn_permlane32_swap(pack_bf(v[2], v[3]), pack_bf(v[6], v[7]), false, false);
      if (live) *reinterpret_cast<au32x4_t *>(row + c) = au32x4_t{s0[0], s1[0], s0[1], s1[1]};
      if (lo) {  // uniform
        const auto t0 = __builtin_amdgcn_permlane32_swap(pack_bf(r[0], r[1]), pack_bf(r[4], r[5]), false, false);
        const auto t1 = __builtin_amdgcn_permlane32_swap(pack_bf(r[2], r[3]), pack_bf(r[6], r[7]), false, false);
        if (live) *reinterpret_cast<au32x4_t *>(lo + c) = au32x4_t{t0[0], t1[0], t0[1], t1[1]};
      }
    }
}

template <int HD>
__global__ __launch_bounds__(256, 2) void packed_forward_kernel(PackedArgs p) {
  __shared__ __align__(16) bf16_t k0[p_tile<HD>(P_TR)], k1[p_tile<HD>(P_TR)], v0[p_tile<HD>(P_TR)], v1[p_tile<HD>(P_TR)];
  const int w = static_cast<int>(blockIdx.x);
  if (w >= p.items) {
    p_clear(p, p.out, p.heads * HD, w - p.items);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, lr = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int h, t, begin, len, q0;
  p_item(w, p.heads, p.tiles, true, h, t);
  if (!p_slot(p, t, lane, P_WG, begin, len, q0)) return;
  begin = __builtin_amdgcn_readfirstlane(begin);
  len = __builtin_amdgcn_readfirstlane(len);
  q0 = __builtin_amdgcn_readfirstlane(q0);
  const int hk = h / (p.heads / p.kv);
  const int wq0 = q0 + P_WR * wave, qi = wq0 + lr;
  const int nkb = (min(q0 + P_WG, len) + P_TR - 1) / P_TR;
  TileLoad<HD> lk, lv;
  lk.init(p.k.p + begin * p.k.st + hk * p.k.sh, p.k.st, wave, lane);
  lv.init(p.v.p + begin * p.v.st + hk * p.v.sh, p.v.st, wave, lane);
  lk.issue(k0, 0, len);
  lv.issue(v0, 0, len);
  abf16x8_t q[HD / 16];
  p_own<HD>(q, p.q, begin + min(qi, len - 1), h, g);
  pf32x16_t acc[HD / 32] = {};
  float m = -INFINITY, l = 0.0f;

  auto block = [&](int b, const bf16_t *ks, const bf16_t *vs, bf16_t *kn, bf16_t *vn)
      __attribute__((always_inline)) {
    lds_sync<0>();  // every wave's loads have landed, and it is done with the other stage
    if (b + 1 < nkb) {
      lk.issue(kn, (b + 1) * P_TR, len);
      lv.issue(vn, (b + 1) * P_TR, len);
    }
    const int kb0 = b * P_TR;
    if (kb0 > wq0 + P_WR - 1) return;  // wave-uniform: keys after all of the wave's queries
    pf32x16_t s[2] = {};
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_rows<HD>(ks, u, kk, lr, g), q[kk], s[u], 0, 0, 0);
    // the first half of the values' fragments: on their way during the softmax
    abf16x8_t vf[2][HD / 32];
#pragma unroll
    for (int kp = 0; kp < 2; ++kp)
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) vf[kp][e] = p_cols<HD>(vs, e, kp, lane);
    if (kb0 + P_TR - 1 > wq0) {  // wave-uniform: some keys come after some queries
      P_BRANCH;
      const int lim = qi - kb0 - 4 * g;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * u + 8 * (i >> 2) + (i & 3) > lim) s[u][i] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    top = p_max_pair(top) * p.c2;
    // the reference max moves only past the slack (from -inf: at the first score)
    const bool move = top > m + P_SLACK;
    const float mn = move ? top : m, sub = mn == -INFINITY ? 0.0f : mn;
    if (__any(move)) {  // wave-uniform
      const float alpha = move ? __builtin_amdgcn_exp2f(m - sub) : 1.0f;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) acc[e] *= alpha;
      m = mn;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], p.c2, -sub));
        l += s[u][i];
      }
#pragma unroll
    for (int kp = 0; kp < 4; ++kp) {
      const abf16x8_t pb = p_pack(s[kp >> 1], kp & 1);
#pragma unroll
      for (int e = 0; e < HD / 32; ++e)
        acc[e] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kp < 2 ? vf[kp][e] : p_cols<HD>(vs, e, kp, lane), pb,
                                                         acc[e], 0, 0, 0);
    }
  };
  for (int b = 0; b < nkb; b += 2) {
    block(b, k0, v0, k1, v1);
    if (b + 1 < nkb) block(b + 1, k1, v1, k0, v0);
  }

  l += __shfl_xor(l, 32);
  const bool live = qi < len;
  const int64_t row = static_cast<int64_t>(begin + qi) * p.heads + h;
  p_store<HD>(acc, 1.0f / l, p.out + row * HD, p.lo ? p.lo + row * HD : nullptr, g, live);
  if (p.lse && live && g == 0)
    p.lse[static_cast<int64_t>(h) * p.T + begin + qi] = m + __builtin_amdgcn_logf(l);
}

template <int HD>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(PackedArgs p) {
  __shared__ __align__(16) bf16_t k0[p_tile<HD>(P_TR)], k1[p_tile<HD>(P_TR)], v0[p_tile<HD>(P_TR)], v1[p_tile<HD>(P_TR)];
  const int w = static_cast<int>(blockIdx.x);
  if (w >= p.items) {
    p_clear(p, p.dq, p.heads * HD, w - p.items);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, lr = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int h, t, begin, len, q0;
  p_item(w, p.heads, p.tiles, true, h, t);
  if (!p_slot(p, t, lane, P_WG, begin, len, q0)) return;
  begin = __builtin_amdgcn_readfirstlane(begin);
  len = __builtin_amdgcn_readfirstlane(len);
  q0 = __builtin_amdgcn_readfirstlane(q0);
  const int hk = h / (p.heads / p.kv);
  const int wq0 = q0 + P_WR * wave, qi = wq0 + lr;
  const int nkb = (min(q0 + P_WG, len) + P_TR - 1) / P_TR;
  TileLoad<HD> lk, lv;
  lk.init(p.k.p + begin * p.k.st + hk * p.k.sh, p.k.st, wave, lane);
  lv.init(p.v.p + begin * p.v.st + hk * p.v.sh, p.v.st, wave, lane);
  lk.issue(k0, 0, len);
  lv.issue(v0, 0, len);
  abf16x8_t q[HD / 16], d[HD / 16];
  const int row = begin + min(qi, len - 1);
  p_own<HD>(q, p.q, row, h, g);
  p_own<HD>(d, p.d, row, h, g);
  const float lse = p.lse[static_cast<int64_t>(h) * p.T + row];
  // delta = do . o of the wave's rows, from both parts of o; the dk, dv launch reads it
  float delta = 0.0f;
  {
    abf16x8_t o[HD / 16], lo[HD / 16];
    p_own<HD>(o, Rows{p.o, static_cast<int64_t>(p.heads) * HD, HD}, row, h, g);
    p_own<HD>(lo, Rows{p.olo, static_cast<int64_t>(p.heads) * HD, HD}, row, h, g);
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        delta = fmaf(static_cast<float>(d[kk][j]), static_cast<float>(o[kk][j]) + static_cast<float>(lo[kk][j]), delta);
  }
  delta += __shfl_xor(delta, 32);
  const float less = -delta;  // (dk and dv's kernel starts its sums from it)
  if (g == 0 && qi < len) p.delta[static_cast<int64_t>(h) * p.T + row] = less;
  pf32x16_t acc[HD / 32] = {};
  // dp starts from -delta where that is the faster (8192 tokens, 32 heads of 64: 395 ->
  // 381 us; 2048 tokens, heads of 128: 72 -> 75)
  constexpr bool START = HD == 64;

  auto block = [&](int b, const bf16_t *ks, const bf16_t *vs, bf16_t *kn, bf16_t *vn)
      __attribute__((always_inline)) {
    lds_sync<0>();  // every wave's loads have landed, and it is done with the other stage
    if (b + 1 < nkb) {
      lk.issue(kn, (b + 1) * P_TR, len);
      lv.issue(vn, (b + 1) * P_TR, len);
    }
    const int kb0 = b * P_TR;
    if (kb0 > wq0 + P_WR - 1) return;  // wave-uniform
    const bool edge = kb0 + P_TR - 1 > wq0;  // wave-uniform: some keys come after some queries
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      pf32x16_t s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = START ? less : 0.0f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_rows<HD>(ks, u, kk, lr, g), q[kk], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_rows<HD>(vs, u, kk, lr, g), d[kk], dp, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c2, -lse)) * (START ? dp[i] : dp[i] - delta);
      if (edge) {  // keys after the query; a query of one key
        P_BRANCH;
        const int lim = qi == 0 ? -1 : qi - kb0 - 4 * g;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * u + 8 * (i >> 2) + (i & 3) > lim) s[i] = 0.0f;
      }
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        const abf16x8_t sb = p_pack(s, kp);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e)
          acc[e] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_cols<HD>(ks, e, 2 * u + kp, lane), sb, acc[e], 0, 0, 0);
      }
    }
  };
  for (int b = 0; b < nkb; b += 2) {
    block(b, k0, v0, k1, v1);
    if (b + 1 < nkb) block(b + 1, k1, v1, k0, v0);
  }
  p_store<HD>(acc, p.scale, p.dq + (static_cast<int64_t>(begin + qi) * p.heads + h) * HD, nullptr, g, qi < len);
}

// dk and dv of KW waves' keys.  A wave's 32 x HD sums of both take half its
// registers, its keys' B operands an eighth; its values' are read from LDS again for
// every tile, but by four waves of heads of 128, which have the registers (2048 tokens of
// 32 heads 107 -> 102 us; with eight waves they spilled, 1133 -> 1420 us for 8192 tokens).
// Heads of 64: held to what three workgroups of a CU can have (16384 tokens of 16 heads
// 1139 -> 1070 us).  SPLIT: one query head per workgroup, fp32 sums to `part`, which a
// second kernel joins over the heads that share a key head.
template <int HD, bool SPLIT, int KW>
__global__ __launch_bounds__(64 * KW, HD == 64 ? 3 : 1) void packed_dkv_kernel(PackedArgs p) {
  constexpr int KG = KW * P_WR;  // keys of the workgroup
  constexpr int TILE = p_tile<HD>(P_TR);
  constexpr bool OWN = HD == 128 && KW == 4;  // values in registers
  __shared__ __align__(16) bf16_t q0s[TILE], q1s[TILE], d0s[TILE], d1s[TILE];
  __shared__ __align__(16) bf16_t vs[OWN ? 8 : p_tile<HD>(KG)];         // the workgroup's values
  __shared__ __align__(16) float l0s[P_TR], l1s[P_TR], e0s[P_TR], e1s[P_TR];  // log-sum-exp, -delta
  const int w = static_cast<int>(blockIdx.x);
  if (w >= p.items) {
    if (!SPLIT) {
      p_clear(p, p.dk, p.kv * HD, w - p.items);
      p_clear(p, p.dv, p.kv * HD, w - p.items);
    }
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, lr = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = p.heads / p.kv;
  int hk, t, begin, len, r0;
  p_item(w, SPLIT ? p.heads : p.kv, p.tiles, false, hk, t);
  const int h0 = SPLIT ? hk : hk * group;  // first query head
  if (SPLIT) hk /= group;
  if (!p_slot(p, t, lane, KG, begin, len, r0)) return;
  begin = __builtin_amdgcn_readfirstlane(begin);
  len = __builtin_amdgcn_readfirstlane(len);
  r0 = __builtin_amdgcn_readfirstlane(r0);
  const int wk0 = r0 + P_WR * wave, ki = wk0 + lr;
  const int nqb = (len - r0 + P_TR - 1) / P_TR, total = SPLIT ? nqb : nqb * group;  // swept tiles

  TileLoad<HD, KW> lq, ld;
  lq.init(p.q.p, p.q.st, wave, lane);
  ld.init(p.d.p, p.d.st, wave, lane);
  if constexpr (!OWN) {
    TileLoad<HD, KW> lv;
    lv.init(p.v.p + begin * p.v.st + hk * p.v.sh, p.v.st, wave, lane);
    for (int i = 0; i < KG / P_TR; ++i) lv.issue(vs + i * TILE, r0 + i * P_TR, len);
  }
  int ih = 0, ib = 0;  // the next tile to load: head of the group, tile of its sweep
  auto issue = [&](bf16_t *qs, bf16_t *ds, float *ls, float *es) __attribute__((always_inline)) {
    const int h = h0 + ih, row = r0 + ib * P_TR;
    lq.p = p.q.p + begin * p.q.st + h * p.q.sh;
    ld.p = p.d.p + begin * p.d.st + h * p.d.sh;
    lq.issue(qs, row, len);
    ld.issue(ds, row, len);
    if (wave < 2) {  // 64 log-sum-exps, 64 deltas
      const float *src = (wave ? p.delta : p.lse) + static_cast<int64_t>(h) * p.T + begin + row;
      lds_load4(lds_rsrc(src, 4u * static_cast<uint32_t>(min(P_TR, len - row))), 4 * lane, wave ? es : ls);
    }
    if (++ib == nqb) {
      ib = 0;
      ++ih;
    }
  };
  issue(q0s, d0s, l0s, e0s);
  abf16x8_t k[HD / 16];
  p_own<HD>(k, p.k, begin + min(ki, len - 1), hk, g);
  abf16x8_t v[OWN ? HD / 16 : 1];
  if constexpr (OWN) p_own<HD>(v, p.v, begin + min(ki, len - 1), hk, g);
  pf32x16_t dk[HD / 32] = {}, dv[HD / 32] = {};

  int cb = 0;  // tile of the current sweep
  auto block = [&](int it, const bf16_t *qs, const bf16_t *ds, const float *ls, const float *es, bf16_t *qn,
                   bf16_t *dn, float *ln, float *en) __attribute__((always_inline)) {
    lds_sync<0>();  // every wave's loads have landed, and it is done with the other stage
    if (it + 1 < total) issue(qn, dn, ln, en);
    const int qb0 = r0 + cb * P_TR;
    if (++cb == nqb) cb = 0;
    if (wk0 >= len) return;  // wave-uniform: no keys
    // (both tiles at once where the registers allow it)
#pragma unroll HD == 64 ? 3 : 1
    for (int u = 0; u < 2; ++u) {
      const int qt0 = qb0 + 32 * u;
      if (qt0 < wk0) continue;  // wave-uniform: queries before all of the wave's keys
      pf32x16_t s = {}, dp;
#pragma unroll
      for (int b = 0; b < 4; ++b) {  // dp - delta
        const af32x4_t ee = *reinterpret_cast<const af32x4_t *>(es + 32 * u + 8 * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[4 * b + i] = ee[i];  // from LDS, no subtraction (1144 -> 1129 us)
      }
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_rows<HD>(qs, u, kk, lr, g), k[kk], s, 0, 0, 0);
        abf16x8_t vk;
        if constexpr (OWN) vk = v[kk];
        else vk = p_rows<HD>(vs, wave, kk, lr, g);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_rows<HD>(ds, u, kk, lr, g), vk, dp, 0, 0, 0);
      }
      // (queries past the sequence: zero rows of q and do, whose log-sum-exp and
      // delta read as 0, so that ds = 0 and p meets do = 0)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const af32x4_t ll = *reinterpret_cast<const af32x4_t *>(ls + 32 * u + 8 * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[4 * b + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * b + i], p.c2, -ll[i]));
          dp[4 * b + i] *= s[4 * b + i];
        }
      }
      if (qt0 == wk0) {  // wave-uniform: the diagonal tile (rows of both start on 32s)
        P_BRANCH;
        const int lim = lr - 4 * g;  // (the rows as constants: as sums they held 16 registers)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) < lim) s[i] = dp[i] = 0.0f;
        if (qt0 + 4 * g == 0) dp[0] = 0.0f;  // a query of one key
      }
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        const abf16x8_t pb = p_pack(s, kp), sb = p_pack(dp, kp);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
          dv[e] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_cols<HD>(ds, e, 2 * u + kp, lane), pb, dv[e], 0, 0, 0);
          dk[e] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p_cols<HD>(qs, e, 2 * u + kp, lane), sb, dk[e], 0, 0, 0);
        }
      }
    }
  };
  for (int it = 0; it < total; it += 2) {
    block(it, q0s, d0s, l0s, e0s, q1s, d1s, l1s, e1s);
    if (it + 1 < total) block(it + 1, q1s, d1s, l1s, e1s, q0s, d0s, l0s, e0s);
  }
  if constexpr (SPLIT) {
    if (ki >= len) return;
    // element 32 e + 8 q + 4 g + i of the row
    float *o = p.part + (static_cast<int64_t>(h0) * p.T + begin + ki) * (2 * HD) + 4 * g;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        *reinterpret_cast<af32x4_t *>(o + 32 * e + 8 * b) =
            af32x4_t{dk[e][4 * b], dk[e][4 * b + 1], dk[e][4 * b + 2], dk[e][4 * b + 3]};
        *reinterpret_cast<af32x4_t *>(o + HD + 32 * e + 8 * b) =
            af32x4_t{dv[e][4 * b], dv[e][4 * b + 1], dv[e][4 * b + 2], dv[e][4 * b + 3]};
      }
  } else {
    const int64_t at = (static_cast<int64_t>(begin + ki) * p.kv + hk) * HD;
    p_store<HD>(dk, p.scale, p.dk + at, nullptr, g, ki < len);
    p_store<HD>(dv, 1.0f, p.dv + at, nullptr, g, ki < len);
  }
}

// dk and dv rows from the sums of the heads that share them, in the heads' order; rows
// outside the sequences zero.  HD / 8 lanes per row and key head.
template <int HD>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedArgs p) {
  constexpr int CH = HD / 8;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / CH;  // row * kv + key head
  const int c = 8 * (threadIdx.x % CH);
  if (at >= static_cast<int64_t>(p.T) * p.kv) return;
  const int64_t row = at / p.kv;
  const int hk = static_cast<int>(at - row * p.kv), group = p.heads / p.kv;
  float k[8] = {}, v[8] = {};
  if (row >= p.cu[0] && row < p.cu[p.nseq])
    for (int i = 0; i < group; ++i) {
      const float *s = p.part + (static_cast<int64_t>(hk * group + i) * p.T + row) * (2 * HD) + c;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        k[j] += s[j];
        v[j] += s[HD + j];
      }
    }
#pragma unroll
  for (int j = 0; j < 8; ++j) k[j] *= p.scale;
  *reinterpret_cast<au32x4_t *>(p.dk + at * HD + c) =
      au32x4_t{pack_bf(k[0], k[1]), pack_bf(k[2], k[3]), pack_bf(k[4], k[5]), pack_bf(k[6], k[7])};
  *reinterpret_cast<au32x4_t *>(p.dv + at * HD + c) =
      au32x4_t{pack_bf(v[0], v[1]), pack_bf(v[2], v[3]), pack_bf(v[4], v[5]), pack_bf(v[6], v[7])};
}

// 16-byte aligned rows that do not overlap (a tile's rows past its sequence have to
// lie past its descriptor), a tile within 32-bit offsets.
static bool rows_ok(const void *p, int64_t st, int64_t sh, int64_t hd) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st % 8 == 0 && sh % 8 == 0 && st >= hd && sh >= 0 &&
         st < (int64_t(1) << 23) && sh < (int64_t(1) << 40);
}
static bool aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static int check_sizes(const char *what, int64_t T, int64_t nseq, int64_t heads, int64_t kv, int64_t hd, float scale) {
  if (T < 0 || nseq < 0 || heads <= 0 || kv <= 0 || heads % kv || T > 0x3fffffff || nseq > 0x3fffffff ||
      heads > 0x3fffffff)
    return fail(EVO2_ERR_INVALID, "%s: bad sizes T=%lld nseq=%lld heads=%lld kv=%lld", what, (long long)T,
                (long long)nseq, (long long)heads, (long long)kv);
  // (the dk, dv kernel's workgroups are no more; packed_wide sees to those of eight waves)
  if (!grid_fits((T / P_WG + nseq) * heads + P_FILL, 64 * P_NW))
    return fail(EVO2_ERR_UNSUPPORTED, "%s: T=%lld nseq=%lld heads=%lld are more workgroups than a launch takes",
                what, (long long)T, (long long)nseq, (long long)heads);
  if (hd != 64 && hd != 128)
    return fail(EVO2_ERR_UNSUPPORTED, "%s: head_dim %lld (64 or 128)", what, (long long)hd);
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return fail(EVO2_ERR_INVALID, "%s: scale %g (must be positive)", what, (double)scale);
  return EVO2_OK;
}

static PackedArgs packed_args(const int32_t *cu, int64_t nseq, int64_t T, int64_t heads, int64_t kv, float scale) {
  PackedArgs a{};
  a.cu = cu;
  a.nseq = static_cast<int>(nseq);
  a.T = static_cast<int>(T);
  a.heads = static_cast<int>(heads);
  a.kv = static_cast<int>(kv);
  a.tiles = static_cast<int>(T / P_WG + nseq);
  a.scale = scale;
  a.c2 = scale * 1.4426950408889634f;
  return a;
}

template <int HD>
static void launch_forward(PackedArgs a, hipStream_t st) {
  a.items = a.tiles * a.heads;
  hipLaunchKernelGGL((packed_forward_kernel<HD>), dim3(a.items + P_FILL), dim3(256), 0, st, a);
}

// Whether the dk, dv kernel's workgroups take eight waves rather than four.  Heads of
// 128: eight share a swept tile, but such a workgroup fills a CU, so that up to about one
// round of the CUs half as many keys in twice as many workgroups end sooner (us with
// eight and with four waves, by workgroups of eight: 160 of them 61 and 48, 208: 156 and
// 124, 272: 163 and 142, 288: 114 and 102, 131 and 133 or 244 and 244, 320: 62 and 60 or
// 260 and 270, 352: 147 and 166, 1056: 1085 and 1393).  Heads of 64: always four, three
// workgroups to a CU, which fill each other's waits (8192 tokens of 32 heads 754 and 625
// us, 8 x 1024 tokens 120 and 93).
static bool packed_wide(const PackedArgs &a) {
  const int64_t groups = (a.T / (8 * P_WR) + static_cast<int64_t>(a.nseq)) * (a.part ? a.heads : a.kv);
  return groups >= 304 && grid_fits(groups + P_FILL, 64 * 8);
}

template <int HD, int KW>
static void launch_dkv(PackedArgs a, hipStream_t st) {
  a.tiles = a.T / (KW * P_WR) + a.nseq;
  if (a.part) {
    a.items = a.tiles * a.heads;
    if (a.items > 0)  // (few rows and no sequences: the join clears them)
      hipLaunchKernelGGL((packed_dkv_kernel<HD, true, KW>), dim3(a.items), dim3(64 * KW), 0, st, a);
    const int64_t rows = static_cast<int64_t>(a.T) * a.kv * (HD / 8);
    hipLaunchKernelGGL((packed_join_kernel<HD>), dim3(static_cast<unsigned>(cdiv(rows, 256))), dim3(256), 0, st, a);
  } else {
    a.items = a.tiles * a.kv;
    hipLaunchKernelGGL((packed_dkv_kernel<HD, false, KW>), dim3(a.items + P_FILL), dim3(64 * KW), 0, st, a);
  }
}

template <int HD>
static void launch_backward(PackedArgs a, hipStream_t st) {
  a.items = a.tiles * a.heads;  // first: it writes delta
  hipLaunchKernelGGL((packed_dq_kernel<HD>), dim3(a.items + P_FILL), dim3(256), 0, st, a);
  if constexpr (HD == 128)
    if (packed_wide(a)) return launch_dkv<HD, 8>(a, st);
  launch_dkv<HD, 4>(a, st);
}

}  // namespace evo2

using namespace evo2;

extern "C" int evo2_packed_attention(const void *q, int64_t sqt, int64_t sqh, const void *k, int64_t skt,
                                     int64_t skh, const void *v, int64_t svt, int64_t svh, const int32_t *cu,
                                     int64_t nseq, void *out, void *out_lo, float *lse, int64_t T, int64_t heads,
                                     int64_t kv, int64_t head_dim, float scale, void *stream) {
  const int rc = check_sizes("packed_attention", T, nseq, heads, kv, head_dim, scale);
  if (rc || T == 0) return rc;
  if (!q || !k || !v || !cu || !out || !out_lo != !lse)
    return fail(EVO2_ERR_INVALID, "packed_attention: null pointer argument");
  if (!rows_ok(q, sqt, sqh, head_dim) || !rows_ok(k, skt, skh, head_dim) || !rows_ok(v, svt, svh, head_dim) ||
      !aligned(out) || !aligned(out_lo))
    return fail(EVO2_ERR_UNSUPPORTED, "packed_attention: operands must be 16-byte aligned rows");
  PackedArgs a = packed_args(cu, nseq, T, heads, kv, scale);
  a.q = Rows{static_cast<const bf16_t *>(q), sqt, sqh};
  a.k = Rows{static_cast<const bf16_t *>(k), skt, skh};
  a.v = Rows{static_cast<const bf16_t *>(v), svt, svh};
  a.out = static_cast<bf16_t *>(out);
  a.lo = static_cast<bf16_t *>(out_lo);
  a.lse = lse;
  if (head_dim == 128) launch_forward<128>(a, static_cast<hipStream_t>(stream));
  else launch_forward<64>(a, static_cast<hipStream_t>(stream));
  return check_launch("packed_attention");
}

// Whether a workgroup of the dk, dv kernel takes one query head rather than all that
// share its keys: where whole groups leave fewer workgroups than two for each CU.
static bool packed_split(int64_t T, int64_t nseq, int64_t heads, int64_t kv) {
  return heads > kv && (T / (8 * P_WR) + nseq) * kv < 512;
}

extern "C" int64_t evo2_packed_attention_workspace_bytes(int64_t T, int64_t nseq, int64_t heads, int64_t kv,
                                                         int64_t head_dim) {
  if (T <= 0 || nseq < 0 || heads <= 0 || kv <= 0 || head_dim <= 0) return 0;
  // delta, then the sums by query head
  return cdiv(heads * T * 4, 256) * 256 + (packed_split(T, nseq, heads, kv) ? heads * T * 2 * head_dim * 4 : 0);
}

extern "C" int evo2_packed_attention_backward(const void *dout, int64_t sdt, int64_t sdh, const void *q,
                                              int64_t sqt, int64_t sqh, const void *k, int64_t skt, int64_t skh,
                                              const void *v, int64_t svt, int64_t svh, const int32_t *cu,
                                              int64_t nseq, const void *out, const void *out_lo,
                                              const float *lse, void *workspace, int64_t workspace_bytes,
                                              void *dq, void *dk, void *dv, int64_t T, int64_t heads, int64_t kv,
                                              int64_t head_dim, float scale, void *stream) {
  const int rc = check_sizes("packed_attention_backward", T, nseq, heads, kv, head_dim, scale);
  if (rc || T == 0) return rc;
  if (!dout || !q || !k || !v || !cu || !out || !out_lo || !lse || !workspace || !dq || !dk || !dv)
    return fail(EVO2_ERR_INVALID, "packed_attention_backward: null pointer argument");
  if (!rows_ok(dout, sdt, sdh, head_dim) || !rows_ok(q, sqt, sqh, head_dim) || !rows_ok(k, skt, skh, head_dim) ||
      !rows_ok(v, svt, svh, head_dim) || !aligned(out) || !aligned(out_lo) || !aligned(dq) || !aligned(dk) || !aligned(dv) ||
      !aligned(workspace))
    return fail(EVO2_ERR_UNSUPPORTED, "packed_attention_backward: operands must be 16-byte aligned rows");
  if (workspace_bytes < evo2_packed_attention_workspace_bytes(T, nseq, heads, kv, head_dim))
    return fail(EVO2_ERR_INVALID, "packed_attention_backward: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes,
                (long long)evo2_packed_attention_workspace_bytes(T, nseq, heads, kv, head_dim));
  PackedArgs a = packed_args(cu, nseq, T, heads, kv, scale);
  a.q = Rows{static_cast<const bf16_t *>(q), sqt, sqh};
  a.k = Rows{static_cast<const bf16_t *>(k), skt, skh};
  a.v = Rows{static_cast<const bf16_t *>(v), svt, svh};
  a.d = Rows{static_cast<const bf16_t *>(dout), sdt, sdh};
  a.o = static_cast<const bf16_t *>(out);
  a.olo = static_cast<const bf16_t *>(out_lo);
  a.lse = const_cast<float *>(lse);
  a.delta = static_cast<float *>(workspace);
  if (packed_split(T, nseq, heads, kv))
    a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + cdiv(heads * T * 4, 256) * 256);
  a.dq = static_cast<bf16_t *>(dq);
  a.dk = static_cast<bf16_t *>(dk);
  a.dv = static_cast<bf16_t *>(dv);
  if (head_dim == 128) launch_backward<128>(a, static_cast<hipStream_t>(stream));
  else launch_backward<64>(a, static_cast<hipStream_t>(stream));
  return check_launch("packed_attention_backward");
}

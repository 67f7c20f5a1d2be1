// Softmax cross entropy at the head, from the hidden rows and the head's weight:
//   z = h w^T,  lse = log sum_n exp z_n,  nll = lse - z[target]
//   d = (exp(z - lse) - [n = target]) * g,  dh = d w,  dw = d^T h
// (evo2_flash/model.py:343-348 gives the logits; scoring and training reduce them).
// The logits are never kept.  Forward, a tile of 256 columns leaves each row's
// max and sum of exponentials over 128 columns (8 bytes for 128 logits) from its
// accumulators, and a second launch joins them.  Backward, the logits are computed
// again in pieces of the vocabulary and leave the accumulators as d, rounded to
// bf16 once as the operand of the two products that follow; the piece's dw is
// whole, dh's pieces are added in fp32.  Where rows and vocabulary together make too
// few tiles for the card (a few rows scored), K is split instead and the fp32
// partial logits of those few tiles meet in a kernel of one workgroup per row.
//
// Rows whose target is `ignore` have loss 0 and no gradient; a target outside the
// vocabulary makes the row's loss and gradient NaN.  Sums over rows are taken in
// 64 bits in a fixed order.
#include "bf16_mat.h"

namespace evo2 {

constexpr float L_LOG2E = 1.44269504088896341f, L_LN2 = 0.69314718055994531f;
constexpr int L_ROWS = 16;             // rows per workgroup of the joining kernel
constexpr int L_RUNS = 256 / L_ROWS;   // and the runs of parts it cuts each into

struct LossRows {
  const int64_t *targets;
  int64_t ignore, V;
  float *nll, *lse;
  double *sums;        // per workgroup: its rows' losses, and how many count
  int T;
};

// One row's result from its max, sum of exp2((z - max) log2 e) and target logit.
__device__ __forceinline__ float loss_row(const LossRows &p, int m, float mx, float sum, float zt) {
  const float lse = mx + L_LN2 * __builtin_amdgcn_logf(sum);
  p.lse[m] = lse;
  const int64_t t = p.targets[m];
  const float nll = t == p.ignore ? 0.0f : t < 0 || t >= p.V ? __builtin_nanf("") : lse - zt;
  p.nll[m] = nll;
  return nll;
}

// (max, sum) pairs: a joined with b; a pair of -inf has sum 0.
__device__ __forceinline__ void loss_join(float &mx, float &sum, float mx2, float sum2) {
  const float top = fmaxf(mx, mx2), sub = top == -INFINITY ? 0.0f : top;
  sum = sum * __builtin_amdgcn_exp2f((mx - sub) * L_LOG2E) + sum2 * __builtin_amdgcn_exp2f((mx2 - sub) * L_LOG2E);
  mx = top;
}

// Joins the tiles' (max, sum), 16 rows by 16 runs of the parts per workgroup: a run's
// max first, then its sum, so that the loads of neither pass wait for one another (one
// pass that rescales as it goes: 20 us for 777 rows of 392 parts, 6 so).
__global__ __launch_bounds__(256) void loss_join_kernel(LossRows p, const float2 *part, const float *tgt,
                                                        int nparts) {
  __shared__ float smx[L_RUNS][L_ROWS], ssum[L_RUNS][L_ROWS];
  const int r = threadIdx.x % L_ROWS, run = threadIdx.x / L_ROWS;
  const int m = blockIdx.x * L_ROWS + r;
  float mx = -INFINITY, sum = 0.0f;
  if (m < p.T) {
    const float2 *at = part + m;
#pragma unroll 8
    for (int i = run; i < nparts; i += L_RUNS) mx = fmaxf(mx, at[static_cast<int64_t>(i) * p.T].x);
    const float sub = mx == -INFINITY ? 0.0f : mx;
#pragma unroll 8
    for (int i = run; i < nparts; i += L_RUNS) {
      const float2 v = at[static_cast<int64_t>(i) * p.T];
      sum = fmaf(v.y, __builtin_amdgcn_exp2f((v.x - sub) * L_LOG2E), sum);
    }
  }
  smx[run][r] = mx;
  ssum[run][r] = sum;
  __syncthreads();
  if (run != 0) return;
  for (int i = 1; i < L_RUNS; ++i) loss_join(mx, sum, smx[i][r], ssum[i][r]);
  double loss = 0.0, n = 0.0;
  if (m < p.T) {
    const int64_t t = p.targets[m];
    const bool ok = t != p.ignore && t >= 0 && t < p.V;
    loss = loss_row(p, m, mx, sum, ok ? tgt[m] : 0.0f);
    n = t != p.ignore ? 1.0 : 0.0;
  }
  for (int o = L_ROWS / 2; o; o >>= 1) {
    loss += __shfl_xor(loss, o);
    n += __shfl_xor(n, o);
  }
  if (r == 0 && p.sums) {
    p.sums[2 * blockIdx.x] = loss;
    p.sums[2 * blockIdx.x + 1] = n;
  }
}

// One row's logit n from the partial sums over K.
__device__ __forceinline__ float loss_logit(const float *part, int64_t plane, int splits, int64_t at) {
  float z = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) z += part[s * plane + at];
  return z;
}

// A row per workgroup from the partial logits (splits, T, V).
__global__ __launch_bounds__(256) void loss_rows_kernel(LossRows p, const float *part, int splits) {
  __shared__ float smx[4], ssum[4];
  const int m = blockIdx.x, tid = threadIdx.x;
  const int64_t plane = static_cast<int64_t>(p.T) * p.V, row = static_cast<int64_t>(m) * p.V;
  float mx = -INFINITY, sum = 0.0f;
  for (int64_t n = tid; n < p.V; n += 256) loss_join(mx, sum, loss_logit(part, plane, splits, row + n), 1.0f);
  for (int o = 32; o; o >>= 1) loss_join(mx, sum, __shfl_xor(mx, o), __shfl_xor(sum, o));
  if ((tid & 63) == 0) {
    smx[tid >> 6] = mx;
    ssum[tid >> 6] = sum;
  }
  __syncthreads();
  if (tid != 0) return;
  for (int i = 1; i < 4; ++i) loss_join(mx, sum, smx[i], ssum[i]);
  const int64_t t = p.targets[m];
  const bool ok = t != p.ignore && t >= 0 && t < p.V;
  const float nll = loss_row(p, m, mx, sum, ok ? loss_logit(part, plane, splits, row + t) : 0.0f);
  if (p.sums) {
    p.sums[2 * m] = nll;
    p.sums[2 * m + 1] = t != p.ignore ? 1.0 : 0.0;
  }
}

// d of a row per workgroup from the partial logits, zeros in the columns that pad V.
__global__ __launch_bounds__(256) void loss_rows_grad_kernel(MatArgs p, const float *part, int splits, int Vp) {
  const int m = blockIdx.x;
  const int64_t plane = static_cast<int64_t>(p.M) * p.V, row = static_cast<int64_t>(m) * p.V;
  const int64_t t = p.targets[m];
  const float wgt = loss_weight(p, m, t);
  const float lse2 = p.lse[m] * L_LOG2E;
  bf16_t *out = static_cast<bf16_t *>(p.out) + static_cast<int64_t>(m) * p.so;
  for (int n = threadIdx.x; n < Vp; n += 256) {
    float v = 0.0f;
    if (n < p.V && t != p.ignore) {
      const float z = loss_logit(part, plane, splits, row + n);
      v = __builtin_amdgcn_exp2f(fmaf(z, L_LOG2E, -lse2));
      if (n == t) v -= 1.0f;
      v *= wgt;
    }
    out[n] = f2bf(v);
  }
}

// The rows' losses summed (or averaged over those that count) by one workgroup.
__global__ __launch_bounds__(1024) void loss_sum_kernel(const double *sums, int n, int mean, float *loss,
                                                        float *count) {
  __shared__ double sl[16], sc[16];
  const int tid = threadIdx.x;
  double l = 0.0, c = 0.0;
  for (int i = tid; i < n; i += 1024) {
    l += sums[2 * i];
    c += sums[2 * i + 1];
  }
  for (int o = 32; o; o >>= 1) {
    l += __shfl_xor(l, o);
    c += __shfl_xor(c, o);
  }
  if ((tid & 63) == 0) {
    sl[tid >> 6] = l;
    sc[tid >> 6] = c;
  }
  __syncthreads();
  if (tid != 0) return;
  for (int i = 1; i < 16; ++i) {
    l += sl[i];
    c += sc[i];
  }
  *count = static_cast<float>(c);
  *loss = static_cast<float>(mean ? l / c : l);
}

static int64_t up(int64_t n, int64_t a) { return cdiv(n, a) * a; }
static bool aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static MatPlan plan_logits(int64_t T, int64_t V, int64_t H, bool split) {
  return mat_plan(MAT_NT, T, V, cdiv(H, MAT_BK), 1, MAT_BN, split);
}

// Vocabulary columns per piece of the backward pass: d takes at most 256 MB, or
// what 8192 columns need.
static int64_t piece(int64_t T, int64_t V) {
  const int64_t most = std::max<int64_t>(8192, ((int64_t(1) << 27) / T) & ~int64_t(255));
  return V <= most ? V : up(cdiv(V, cdiv(V, most)), 256);
}

struct BackPlan {
  int64_t vp, pieces, ld;
  MatPlan z, dh, dw;      // of a whole piece
  int64_t acc, part;      // bytes behind d
};

static BackPlan plan_back(int64_t T, int64_t V, int64_t H) {
  BackPlan b{};
  b.vp = piece(T, V);
  b.pieces = cdiv(V, b.vp);
  b.ld = up(b.vp, 8);
  b.z = plan_logits(T, b.vp, H, b.pieces == 1);
  b.dh = mat_plan(MAT_NN, T, H, cdiv(b.vp, MAT_BK), 1, MAT_BN, b.pieces == 1);
  b.dw = mat_plan(MAT_TN, b.vp, H, cdiv(T, MAT_BK), 1, MAT_BN, true);
  b.acc = b.pieces > 1 ? up(T * H * 4, 256) : 0;
  b.part = std::max({b.z.splits > 1 ? b.z.splits * T * b.vp * 4 : 0, b.dh.splits > 1 ? b.dh.splits * T * H * 4 : 0,
                     b.dw.splits > 1 ? b.dw.splits * b.vp * H * 4 : 0});
  return b;
}

static int check_sizes(const char *what, int64_t T, int64_t V, int64_t H, int64_t sh, int64_t sw) {
  if (T <= 0 || V <= 0 || H <= 0)
    return fail(EVO2_ERR_INVALID, "%s: bad sizes T=%lld V=%lld H=%lld", what, (long long)T, (long long)V,
                (long long)H);
  if (H % 8) return fail(EVO2_ERR_UNSUPPORTED, "%s: H=%lld must be a multiple of 8", what, (long long)H);
  // (a piece's rows of d take V columns at most; the joining kernel a workgroup for 16 rows)
  if (V >= (int64_t(1) << 22) || !mat_fits(T, V, H, std::max(sh, sw)) || !mat_fits(V, H, T, H) ||
      !mat_fits(T, H, V, H) || !grid_fits(cdiv(T, L_ROWS), 256))
    return fail(EVO2_ERR_UNSUPPORTED, "%s: problem too large", what);
  if (sh < H || sw < H || sh % 8 || sw % 8)
    return fail(EVO2_ERR_UNSUPPORTED, "%s: operands must be 16-byte aligned rows", what);
  return EVO2_OK;
}

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_linear_loss_workspace_bytes(int64_t T, int64_t V, int64_t H, int32_t backward) {
  if (T <= 0 || V <= 0 || H <= 0) return 0;
  if (backward) {
    const BackPlan b = plan_back(T, V, H);
    return up(T * b.ld * 2, 256) + b.acc + b.part;
  }
  const MatPlan pl = plan_logits(T, V, H, true);
  // rows' sums, then the parts and the targets' logits, or the partial logits
  const int64_t sums = up(16 * (pl.splits > 1 ? T : cdiv(T, L_ROWS)), 256);
  return sums + (pl.splits > 1 ? pl.splits * T * V * 4 : up(2 * pl.tiles_n * T * 8, 256) + T * 4);
}

extern "C" int evo2_linear_loss(const void *h, int64_t sh, const void *w, int64_t sw, const int64_t *targets,
                                int64_t ignore, int32_t reduction, float *nll, float *lse, float *loss,
                                float *count, void *workspace, int64_t workspace_bytes, int64_t T, int64_t V,
                                int64_t H, void *stream) {
  int rc = check_sizes("linear_loss", T, V, H, sh, sw);
  if (rc) return rc;
  if (reduction < 0 || reduction > 2) return fail(EVO2_ERR_INVALID, "linear_loss: reduction %d", reduction);
  if (!h || !w || !targets || !nll || !lse || !workspace || (reduction && (!loss || !count)))
    return fail(EVO2_ERR_INVALID, "linear_loss: null pointer argument");
  if (!aligned(h) || !aligned(w) || !aligned(workspace))
    return fail(EVO2_ERR_UNSUPPORTED, "linear_loss: operands must be 16-byte aligned rows");
  if (workspace_bytes < evo2_linear_loss_workspace_bytes(T, V, H, 0))
    return fail(EVO2_ERR_INVALID, "linear_loss: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)evo2_linear_loss_workspace_bytes(T, V, H, 0));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const MatPlan pl = plan_logits(T, V, H, true);
  const int blocks = static_cast<int>(pl.splits > 1 ? T : cdiv(T, L_ROWS));
  char *at = static_cast<char *>(workspace);
  double *sums = reinterpret_cast<double *>(at);
  at += up(16 * static_cast<int64_t>(blocks), 256);
  MatArgs a{};
  a.x = static_cast<const bf16_t *>(h);
  a.sx = sh;
  a.w = static_cast<const bf16_t *>(w);
  a.sw = sw;
  a.M = static_cast<int>(T);
  a.N = static_cast<int>(V);
  a.K = a.Kx = static_cast<int>(H);
  a.kpair = a.mpair = INT_MAX;
  a.targets = targets;
  const LossRows r{targets, ignore, V, nll, lse, reduction ? sums : nullptr, static_cast<int>(T)};
  if (pl.splits > 1) {
    float *part = reinterpret_cast<float *>(at);
    a.out = part;
    a.so = V;
    a.plane = T * V;
    mat_nt_f32(a, pl, st);
    hipLaunchKernelGGL(loss_rows_kernel, dim3(blocks), dim3(256), 0, st, r, part, pl.splits);
  } else {
    a.part = reinterpret_cast<float2 *>(at);
    a.tgt = reinterpret_cast<float *>(at + up(2 * static_cast<int64_t>(pl.tiles_n) * T * 8, 256));
    mat_launch<MAT_NT, MAT_STATS>(a, pl, st);
    hipLaunchKernelGGL(loss_join_kernel, dim3(blocks), dim3(256), 0, st, r, a.part, a.tgt, 2 * pl.tiles_n);
  }
  if (reduction)
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, sums, blocks, reduction == 2, loss, count);
  return check_launch("linear_loss");
}

extern "C" int evo2_linear_loss_backward(const void *h, int64_t sh, const void *w, int64_t sw,
                                         const int64_t *targets, int64_t ignore, const float *lse,
                                         const float *grad, int64_t sgrad, const float *count, void *dh,
                                         void *dw, void *workspace, int64_t workspace_bytes, int64_t T,
                                         int64_t V, int64_t H, void *stream) {
  int rc = check_sizes("linear_loss_backward", T, V, H, sh, sw);
  if (rc) return rc;
  if (!h || !w || !targets || !lse || !grad || !workspace || (count && sgrad))
    return fail(EVO2_ERR_INVALID, "linear_loss_backward: null pointer argument");
  if (!aligned(h) || !aligned(w) || !aligned(dh) || !aligned(dw) || !aligned(workspace))
    return fail(EVO2_ERR_UNSUPPORTED, "linear_loss_backward: operands must be 16-byte aligned rows");
  if (workspace_bytes < evo2_linear_loss_workspace_bytes(T, V, H, 1))
    return fail(EVO2_ERR_INVALID, "linear_loss_backward: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)evo2_linear_loss_workspace_bytes(T, V, H, 1));
  if (!dh && !dw) return EVO2_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const BackPlan b = plan_back(T, V, H);
  if (b.pieces > 1 && !grid_fits(cdiv(T * (H / 8), 256), 256))  // dh's pieces are joined
    return fail(EVO2_ERR_UNSUPPORTED, "linear_loss_backward: problem too large");
  char *at = static_cast<char *>(workspace);
  bf16_t *d = reinterpret_cast<bf16_t *>(at);
  float *acc = reinterpret_cast<float *>(at + up(T * b.ld * 2, 256));
  float *part = reinterpret_cast<float *>(reinterpret_cast<char *>(acc) + b.acc);
  const bool shared = sgrad == 0;  // one upstream gradient for all rows
  const float *num = shared ? grad : nullptr, *den = shared ? count : nullptr;
  for (int64_t v0 = 0; v0 < V; v0 += b.vp) {
    const int64_t vn = std::min(b.vp, V - v0);
    const bf16_t *wp = static_cast<const bf16_t *>(w) + v0 * sw;
    MatArgs a{};
    a.kpair = a.mpair = INT_MAX;
    // d of the piece
    a.x = static_cast<const bf16_t *>(h);
    a.sx = sh;
    a.w = wp;
    a.sw = sw;
    a.M = static_cast<int>(T);
    a.N = static_cast<int>(vn);
    a.K = a.Kx = static_cast<int>(H);
    a.targets = targets;
    a.ignore = ignore;
    a.V = V;
    a.col0 = v0;
    a.lse = lse;
    a.grad = grad;
    a.sgrad = sgrad;
    a.weighted = !shared;
    if (b.z.splits > 1) {  // (one piece)
      a.out = part;
      a.so = V;
      a.plane = T * V;
      mat_nt_f32(a, b.z, st);
      a.out = d;
      a.so = b.ld;
      hipLaunchKernelGGL(loss_rows_grad_kernel, dim3(static_cast<unsigned>(T)), dim3(256), 0, st, a, part,
                         b.z.splits, static_cast<int>(b.ld));
    } else {
      a.out = d;
      a.so = b.ld;
      mat_launch<MAT_NT, MAT_DLOG>(a, plan_logits(T, vn, H, false), st);
    }
    if (dh) {
      MatArgs c{};
      c.kpair = c.mpair = INT_MAX;
      c.x = d;
      c.sx = b.ld;
      c.w = wp;
      c.sw = sw;
      c.M = static_cast<int>(T);
      c.N = static_cast<int>(H);
      c.K = static_cast<int>(vn);
      c.Kx = static_cast<int>(up(vn, 8));
      c.so = H;
      c.plane = T * H;
      c.num = num;
      c.den = den;
      if (b.pieces > 1) {
        c.out = acc;
        c.add = v0 > 0;
        mat_nn(c, mat_plan(MAT_NN, T, H, cdiv(vn, MAT_BK), 1, MAT_BN, false), true, st);
        if (v0 + vn == V) mat_join(acc, 0, 1, static_cast<bf16_t *>(dh), H, T, H, st, num, den);
      } else {
        c.out = b.dh.splits > 1 ? static_cast<void *>(part) : dh;
        mat_nn(c, b.dh, b.dh.splits > 1, st);
        if (b.dh.splits > 1) mat_join(part, T * H, b.dh.splits, static_cast<bf16_t *>(dh), H, T, H, st, num, den);
      }
    }
    if (dw) {
      MatArgs c{};
      c.kpair = c.mpair = INT_MAX;
      c.x = d;
      c.sx = b.ld;
      c.w = static_cast<const bf16_t *>(h);
      c.sw = sh;
      c.M = static_cast<int>(vn);
      c.N = static_cast<int>(H);
      c.K = static_cast<int>(T);
      c.so = H;
      // a last piece is smaller than the others: its splits are no more than theirs
      MatPlan pl = mat_plan(MAT_TN, vn, H, cdiv(T, MAT_BK), 1, MAT_BN, true);
      if (pl.splits > 1 && pl.splits * vn * H * 4 > b.part) pl = mat_plan(MAT_TN, vn, H, cdiv(T, MAT_BK), 1, MAT_BN, false);
      bf16_t *to = static_cast<bf16_t *>(dw) + v0 * H;
      c.plane = vn * H;
      c.num = num;
      c.den = den;
      c.out = pl.splits > 1 ? static_cast<void *>(part) : to;
      mat_tn(c, pl, pl.splits > 1, st);
      if (pl.splits > 1) mat_join(part, vn * H, pl.splits, to, H, vn, H, st, num, den);
    }
  }
  return check_launch("linear_loss_backward");
}

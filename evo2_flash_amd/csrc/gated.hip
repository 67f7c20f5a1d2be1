// The gated product of a feed-forward block with its backward pass:
//   z1 = x w1^T, z2 = x w2^T, h = act(z1) * z2,   act the exact GELU or the identity
//   d1 = dh * z2 * act'(z1), d2 = dh * act(z1)
//   dx = d1 w1 + d2 w2, dw1 = d1^T x, dw2 = d2^T x
// (the reference's MLP, evo2_flash/model.py:77-101, before its down projection).
// Both projections, the activation and the product are one launch whose tile takes
// 128 columns of each weight, so a lane holds z1 and z2 of the same element; h is
// rounded to bf16 once.  With a backward pass to come the launch also keeps the factors
// of d1 and d2, z2 act'(z1) and act(z1), to 24 bits.
#include "bf16_mat.h"

namespace evo2 {

// d1 | d2 as (M, 2 Ip) bf16, Ip = I rounded up to whole K slices with zeros there:
// one thread per eight columns.
__global__ __launch_bounds__(256) void gated_grad_kernel(const bf16_t *dh, int64_t sdh, const bf16_t *kept,
                                                         int64_t plane, bf16_t *dz, int64_t chunks, int I,
                                                         int Ip) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= chunks) return;
  const int per = Ip >> 3;
  const int64_t m = at / per;
  const int c = static_cast<int>(at - m * per) * 8;
  bf16_t *o = dz + m * 2 * Ip + c;
  au32x4_t d1 = {0, 0, 0, 0}, d2 = {0, 0, 0, 0};
  if (c < I) {
    const bf16_t *k = kept + m * I + c;
    const au32x4_t g = *reinterpret_cast<const au32x4_t *>(dh + m * sdh + c);
    const au32x4_t a = *reinterpret_cast<const au32x4_t *>(k);
    const au32x4_t b = *reinterpret_cast<const au32x4_t *>(k + plane);
    const au32x4_t l = *reinterpret_cast<const au32x4_t *>(k + 2 * plane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // the high half, then the next eight bits: of a the low byte, of b the high one
      const float a0 = __uint_as_float((a[j] << 16) | ((l[j] & 0xffu) << 8));
      const float a1 = __uint_as_float((a[j] & 0xffff0000u) | ((l[j] >> 8) & 0xff00u));
      const float b0 = __uint_as_float((b[j] << 16) | (l[j] & 0xff00u));
      const float b1 = __uint_as_float((b[j] & 0xffff0000u) | ((l[j] >> 16) & 0xff00u));
      d1[j] = pack_bf(lo_bf(g[j]) * a0, hi_bf(g[j]) * a1);
      d2[j] = pack_bf(lo_bf(g[j]) * b0, hi_bf(g[j]) * b1);
    }
  }
  *reinterpret_cast<au32x4_t *>(o) = d1;
  *reinterpret_cast<au32x4_t *>(o + Ip) = d2;
}

static int64_t up(int64_t n, int64_t a) { return cdiv(n, a) * a; }

// dx: K = both halves of dz; dw: K = the rows.
static MatPlan plan_dx(int64_t M, int64_t I, int64_t H) {
  return mat_plan(MAT_NN, M, H, 2 * cdiv(I, MAT_BK), 1, MAT_BN, true);
}
static MatPlan plan_dw(int64_t M, int64_t I, int64_t H) {
  return mat_plan(MAT_TN, I, H, cdiv(M, MAT_BK), 2, MAT_BN, true);
}

static int check_sizes(const char *what, int64_t M, int64_t I, int64_t H, int64_t sx, int64_t sw) {
  if (M < 0 || I <= 0 || H <= 0)
    return fail(EVO2_ERR_INVALID, "%s: bad sizes M=%lld I=%lld H=%lld", what, (long long)M, (long long)I,
                (long long)H);
  if (I % 8 || H % 8)
    return fail(EVO2_ERR_UNSUPPORTED, "%s: I=%lld and H=%lld must be multiples of 8", what, (long long)I,
                (long long)H);
  if (!mat_fits(M, up(I, 64) * 2, H, std::max({sx, sw, up(I, 64) * 2, H})) || !mat_fits(up(I, 64) * 2, H, M, H) ||
      !mat_fits(M, H, I, H))
    return fail(EVO2_ERR_UNSUPPORTED, "%s: problem too large", what);
  return EVO2_OK;
}

static bool aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace evo2

using namespace evo2;

extern "C" int64_t evo2_gated_linear_workspace_bytes(int64_t M, int64_t I, int64_t H) {
  if (M <= 0 || I <= 0 || H <= 0) return 0;
  const MatPlan a = plan_dx(M, I, H), b = plan_dw(M, I, H);
  const int64_t dz = up(M * 2 * up(I, MAT_BK) * 2, 256);
  const int64_t pa = a.splits > 1 ? a.splits * M * H * 4 : 0, pb = b.splits > 1 ? b.splits * 2 * I * H * 4 : 0;
  return dz + std::max(pa, pb);
}

extern "C" int evo2_gated_linear(const void *x, int64_t sx, const void *w1, const void *w2, int64_t sw,
                                 int32_t gelu, void *h, int64_t sh, void *kept, int64_t M, int64_t I,
                                 int64_t H, void *stream) {
  int rc = check_sizes("gated_linear", M, I, H, sx, sw);
  if (rc || M == 0) return rc;
  if (!x || !w1 || !w2 || !h) return fail(EVO2_ERR_INVALID, "gated_linear: null pointer argument");
  if (sx < H || sw < H || sh < I || sx % 8 || sw % 8 || sh % 8 || !aligned(x) || !aligned(w1) || !aligned(w2) ||
      !aligned(h) || !aligned(kept))
    return fail(EVO2_ERR_UNSUPPORTED, "gated_linear: operands must be 16-byte aligned rows");
  MatArgs a{};
  a.x = static_cast<const bf16_t *>(x);
  a.sx = sx;
  a.w = static_cast<const bf16_t *>(w1);
  a.w2 = static_cast<const bf16_t *>(w2);
  a.sw = sw;
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(I);
  a.K = a.Kx = static_cast<int>(H);
  a.kpair = a.mpair = INT_MAX;
  a.out = h;
  a.so = sh;
  a.kept = static_cast<bf16_t *>(kept);
  a.kplane = M * I;
  const MatPlan pl = mat_plan(MAT_NT, M, I, cdiv(H, MAT_BK), 1, MAT_BN / 2, false, 1 + !!gelu);
  if (gelu) mat_launch<MAT_NT, MAT_GELU>(a, pl, static_cast<hipStream_t>(stream));
  else mat_launch<MAT_NT, MAT_GATED>(a, pl, static_cast<hipStream_t>(stream));
  return check_launch("gated_linear");
}

extern "C" int evo2_gated_linear_backward(const void *dh, int64_t sdh, const void *x, int64_t sx,
                                          const void *w1, const void *w2, int64_t sw, const void *kept,
                                          void *dx, void *dw1, void *dw2, void *workspace,
                                          int64_t workspace_bytes, int64_t M, int64_t I, int64_t H, void *stream) {
  int rc = check_sizes("gated_linear_backward", M, I, H, sx, sw);
  if (rc) return rc;
  if (M == 0) return fail(EVO2_ERR_INVALID, "gated_linear_backward: no rows");
  if (!dh || !x || !w1 || !w2 || !kept || !workspace || !dw1 != !dw2)
    return fail(EVO2_ERR_INVALID, "gated_linear_backward: null pointer argument");
  if (sdh < I || sx < H || sw < H || sdh % 8 || sx % 8 || sw % 8 || !aligned(dh) || !aligned(x) || !aligned(w1) ||
      !aligned(w2) || !aligned(kept) || !aligned(dx) || !aligned(dw1) || !aligned(dw2) || !aligned(workspace))
    return fail(EVO2_ERR_UNSUPPORTED, "gated_linear_backward: operands must be 16-byte aligned rows");
  if (workspace_bytes < evo2_gated_linear_workspace_bytes(M, I, H))
    return fail(EVO2_ERR_INVALID, "gated_linear_backward: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)evo2_gated_linear_workspace_bytes(M, I, H));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t Ip = up(I, MAT_BK), chunks = M * (Ip / 8);
  if (!grid_fits(cdiv(chunks, 256), 256))
    return fail(EVO2_ERR_UNSUPPORTED, "gated_linear_backward: problem too large");
  bf16_t *dz = static_cast<bf16_t *>(workspace);
  float *part = reinterpret_cast<float *>(static_cast<char *>(workspace) + up(M * 2 * Ip * 2, 256));
  hipLaunchKernelGGL(gated_grad_kernel, dim3(static_cast<unsigned>(cdiv(chunks, 256))), dim3(256), 0, st,
                     static_cast<const bf16_t *>(dh), sdh, static_cast<const bf16_t *>(kept), M * I, dz, chunks,
                     static_cast<int>(I), static_cast<int>(Ip));
  MatArgs a{};
  a.x = dz;
  a.sx = 2 * Ip;
  a.N = static_cast<int>(H);
  a.so = H;
  if (dx) {
    const MatPlan pl = plan_dx(M, I, H);
    a.w = static_cast<const bf16_t *>(w1);
    a.w2 = static_cast<const bf16_t *>(w2);
    a.sw = sw;
    a.M = static_cast<int>(M);
    a.K = static_cast<int>(I);
    a.Kx = static_cast<int>(2 * Ip);
    a.kpair = static_cast<int>(Ip / MAT_BK);
    a.mpair = INT_MAX;
    a.plane = M * H;
    a.out = pl.splits > 1 ? static_cast<void *>(part) : dx;
    mat_nn(a, pl, pl.splits > 1, st);
    if (pl.splits > 1) mat_join(part, M * H, pl.splits, static_cast<bf16_t *>(dx), H, M, H, st);
  }
  if (dw1) {
    const MatPlan pl = plan_dw(M, I, H);
    a.w = static_cast<const bf16_t *>(x);
    a.sw = sx;
    a.M = static_cast<int>(I);
    a.K = static_cast<int>(M);
    a.kpair = INT_MAX;
    a.mpair = pl.tiles_m / 2;
    a.xpair = static_cast<int>(Ip);
    a.plane = 2 * I * H;
    a.out = pl.splits > 1 ? static_cast<void *>(part) : dw1;
    a.out2 = pl.splits > 1 ? static_cast<void *>(part + I * H) : dw2;
    mat_tn(a, pl, pl.splits > 1, st);
    if (pl.splits > 1) {
      mat_join(part, 2 * I * H, pl.splits, static_cast<bf16_t *>(dw1), H, I, H, st);
      mat_join(part + I * H, 2 * I * H, pl.splits, static_cast<bf16_t *>(dw2), H, I, H, st);
    }
  }
  return check_launch("gated_linear_backward");
}

// The orientations of bf16_mat.h that the gradients share, and the sum over the
// splits of K.
#include "bf16_mat.h"

namespace evo2 {

void mat_nn(const MatArgs &a, const MatPlan &pl, bool f32, hipStream_t st) {
  if (f32) mat_launch<MAT_NN, MAT_F32>(a, pl, st);
  else mat_launch<MAT_NN, MAT_BF16>(a, pl, st);
}

void mat_nt_f32(const MatArgs &a, const MatPlan &pl, hipStream_t st) {
  mat_launch<MAT_NT, MAT_F32>(a, pl, st);
}

// A thread sums eight columns of a row over the planes, in the planes' order.
__global__ __launch_bounds__(256) void mat_join_kernel(const float *part, int64_t plane, int splits,
                                                       bf16_t *out, int64_t so, int64_t chunks, int cols8,
                                                       const float *num, const float *den) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= chunks) return;
  const int64_t r = at / cols8;
  const int c = static_cast<int>(at - r * cols8) * 8;
  const float *src = part + at * 8;
  af32x4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll 4
  for (int s = 0; s < splits; ++s, src += plane) {
    a += *reinterpret_cast<const af32x4_t *>(src);
    b += *reinterpret_cast<const af32x4_t *>(src + 4);
  }
  const float f = mat_factor(num, den);
  a *= f;
  b *= f;
  *reinterpret_cast<au32x4_t *>(out + r * so + c) =
      au32x4_t{pack_bf(a[0], a[1]), pack_bf(a[2], a[3]), pack_bf(b[0], b[1]), pack_bf(b[2], b[3])};
}

void mat_join(const float *part, int64_t plane, int splits, bf16_t *out, int64_t so, int64_t rows,
              int64_t cols, hipStream_t st, const float *num, const float *den) {
  const int64_t chunks = rows * (cols / 8);
  hipLaunchKernelGGL(mat_join_kernel, dim3(static_cast<unsigned>(cdiv(chunks, 256))), dim3(256), 0, st, part,
                     plane, splits, out, so, chunks, static_cast<int>(cols / 8), num, den);
}

}  // namespace evo2

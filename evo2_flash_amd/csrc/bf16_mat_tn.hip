// bf16_mat.h's weight gradients: both operands' rows run across K.
#include "bf16_mat.h"

namespace evo2 {

void mat_tn(const MatArgs &a, const MatPlan &pl, bool f32, hipStream_t st) {
  if (f32) mat_launch<MAT_TN, MAT_F32>(a, pl, st);
  else mat_launch<MAT_TN, MAT_BF16>(a, pl, st);
}

}  // namespace evo2

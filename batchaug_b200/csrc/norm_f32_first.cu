// norm.cuh for fp32 tensors, channels first.
#include "norm_launch.cuh"

ba::NormKernel ba::norm_kernel_f32_first(const NormKind& k) {
  if (k.vec == 4) return norm_kernel_vec<BA_F32, false, 4>(k);
  return norm_kernel_vec<BA_F32, false, 1>(k);
}

// norm.cuh for fp32 tensors, channels last.
#include "norm_launch.cuh"

ba::NormKernel ba::norm_kernel_f32_last(const NormKind& k) {
  if (k.vec == 4) return norm_kernel_vec<BA_F32, true, 4>(k);
  return norm_kernel_vec<BA_F32, true, 1>(k);
}

// norm.cuh for bf16 tensors, channels first.
#include "norm_launch.cuh"

ba::NormKernel ba::norm_kernel_bf16_first(const NormKind& k) {
  if (k.vec == 8) return norm_kernel_vec<BA_BF16, false, 8>(k);
  return norm_kernel_vec<BA_BF16, false, 1>(k);
}

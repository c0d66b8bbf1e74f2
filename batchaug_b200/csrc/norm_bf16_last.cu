// norm.cuh for bf16 tensors, channels last.
#include "norm_launch.cuh"

ba::NormKernel ba::norm_kernel_bf16_last(const NormKind& k) {
  if (k.vec == 8) return norm_kernel_vec<BA_BF16, true, 8>(k);
  if (k.vec == 4) return norm_kernel_vec<BA_BF16, true, 4>(k);
  return norm_kernel_vec<BA_BF16, true, 1>(k);
}

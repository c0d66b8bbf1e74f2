// norm.cuh for bf16 tensors, channels first.
#include "norm_launch.cuh"

void ba::norm_launch_bf16_first(const NormArgs& a, const NormLaunch& l) {
  if (a.f.vec == 8)
    norm_launch_vec<BA_BF16, false, 8>(a, l);
  else
    norm_launch_vec<BA_BF16, false, 1>(a, l);
}

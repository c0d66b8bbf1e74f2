// norm.cuh for bf16 tensors, channels last.
#include "norm_launch.cuh"

void ba::norm_launch_bf16_last(const NormArgs& a, const NormLaunch& l) {
  if (a.f.vec == 8)
    norm_launch_vec<BA_BF16, true, 8>(a, l);
  else if (a.f.vec == 4)
    norm_launch_vec<BA_BF16, true, 4>(a, l);
  else
    norm_launch_vec<BA_BF16, true, 1>(a, l);
}

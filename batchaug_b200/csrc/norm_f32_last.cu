// norm.cuh for fp32 tensors, channels last.
#include "norm_launch.cuh"

void ba::norm_launch_f32_last(const NormArgs& a, const NormLaunch& l) {
  if (a.f.vec == 4)
    norm_launch_vec<BA_F32, true, 4>(a, l);
  else
    norm_launch_vec<BA_F32, true, 1>(a, l);
}

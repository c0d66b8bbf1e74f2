// norm.cuh for fp32 tensors, channels first.
#include "norm_launch.cuh"

void ba::norm_launch_f32_first(const NormArgs& a, const NormLaunch& l) {
  if (a.f.vec == 4)
    norm_launch_vec<BA_F32, false, 4>(a, l);
  else
    norm_launch_vec<BA_F32, false, 1>(a, l);
}

// Launches of norm.cuh's kernels for one dtype and layout; each norm_*.cu
// file instantiates one pair, so that they compile in parallel.
#pragma once

#include "norm.cuh"

namespace ba {

enum { NORM_SUMS = 0, NORM_APPLY = 1, NORM_BWD_SUMS = 2, NORM_BWD_APPLY = 3 };

struct NormLaunch {
  int step;  // NORM_*
  int act;   // ACT_*
  bool drop;
  dim3 grid;
  cudaStream_t stream;
};

void norm_launch_bf16_first(const NormArgs& a, const NormLaunch& l);
void norm_launch_bf16_last(const NormArgs& a, const NormLaunch& l);
void norm_launch_f32_first(const NormArgs& a, const NormLaunch& l);
void norm_launch_f32_last(const NormArgs& a, const NormLaunch& l);

template <int DT, bool LAST, int VEC, int ACT, bool DROP>
void norm_launch_act(const NormArgs& a, const NormLaunch& l) {
  if constexpr (LAST) {
    if (l.step == NORM_APPLY)
      norm_apply_last<DT, VEC, ACT, DROP, false><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
    else if (l.step == NORM_BWD_SUMS)
      norm_sums_last<DT, VEC, ACT, DROP, true><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
    else
      norm_apply_last<DT, VEC, ACT, DROP, true><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
  } else {
    if (l.step == NORM_APPLY)
      norm_apply_first<DT, VEC, ACT, DROP, false><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
    else if (l.step == NORM_BWD_SUMS)
      norm_sums_first<DT, VEC, ACT, DROP, true><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
    else
      norm_apply_first<DT, VEC, ACT, DROP, true><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
  }
}

template <int DT, bool LAST, int VEC, int ACT>
void norm_launch_drop(const NormArgs& a, const NormLaunch& l) {
  if (l.drop)
    norm_launch_act<DT, LAST, VEC, ACT, true>(a, l);
  else
    norm_launch_act<DT, LAST, VEC, ACT, false>(a, l);
}

template <int DT, bool LAST, int VEC>
void norm_launch_vec(const NormArgs& a, const NormLaunch& l) {
  if (l.step == NORM_SUMS) {
    if constexpr (LAST)
      norm_sums_last<DT, VEC, ACT_NONE, false, false><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
    else
      norm_sums_first<DT, VEC, ACT_NONE, false, false><<<l.grid, FEAT_THREADS, 0, l.stream>>>(a);
    return;
  }
  switch (l.act) {
    case ACT_LEAKY: norm_launch_drop<DT, LAST, VEC, ACT_LEAKY>(a, l); break;
    case ACT_SILU: norm_launch_drop<DT, LAST, VEC, ACT_SILU>(a, l); break;
    case ACT_GELU: norm_launch_drop<DT, LAST, VEC, ACT_GELU>(a, l); break;
    default: norm_launch_drop<DT, LAST, VEC, ACT_NONE>(a, l); break;
  }
}

}  // namespace ba

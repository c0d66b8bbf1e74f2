// norm.cuh's kernels for one dtype and layout; each norm_*.cu file
// instantiates one pair, so that they compile in parallel.
#pragma once

#include "norm.cuh"

namespace ba {

struct NormKind {
  int vec;
  int act;  // ACT_*
  int drop;  // DROP_*
  bool backward;
};

using NormKernel = void (*)(NormArgs);

NormKernel norm_kernel_bf16_first(const NormKind& k);
NormKernel norm_kernel_bf16_last(const NormKind& k);
NormKernel norm_kernel_f32_first(const NormKind& k);
NormKernel norm_kernel_f32_last(const NormKind& k);

template <int DT, bool LAST, int VEC, int ACT, int DROP>
NormKernel norm_kernel_drop(const NormKind& k) {
  return k.backward ? norm_kernel<DT, LAST, VEC, ACT, DROP, true>
                    : norm_kernel<DT, LAST, VEC, ACT, DROP, false>;
}

template <int DT, bool LAST, int VEC, int ACT>
NormKernel norm_kernel_act(const NormKind& k) {
  if (k.drop == DROP_PARAM) return norm_kernel_drop<DT, LAST, VEC, ACT, DROP_PARAM>(k);
  if (k.drop == DROP_WORDS) return norm_kernel_drop<DT, LAST, VEC, ACT, DROP_WORDS>(k);
  return norm_kernel_drop<DT, LAST, VEC, ACT, DROP_NONE>(k);
}

template <int DT, bool LAST, int VEC>
NormKernel norm_kernel_vec(const NormKind& k) {
  switch (k.act) {
    case ACT_LEAKY: return norm_kernel_act<DT, LAST, VEC, ACT_LEAKY>(k);
    case ACT_SILU: return norm_kernel_act<DT, LAST, VEC, ACT_SILU>(k);
    case ACT_GELU: return norm_kernel_act<DT, LAST, VEC, ACT_GELU>(k);
    default: return norm_kernel_act<DT, LAST, VEC, ACT_NONE>(k);
  }
}

}  // namespace ba

// ba_norm_forward / ba_norm_backward: host side, and the kernels that merge
// the per-channel partials of norm.cuh into statistics and coefficients.
#include <string.h>

#include "norm_launch.cuh"

namespace ba {
namespace {

// Values a partial of chunk k stands for.
__device__ __forceinline__ int64_t chunk_count(const Feat& f, int64_t k) {
  return min(f.rows, f.S - k * f.rows);
}

// Partial number i (0 .. Cg * nchunk) of group g of element b, its chunk in k.
template <bool LAST>
__device__ __forceinline__ float2 group_part(const NormArgs& a, int64_t b, int64_t g, int64_t i,
                                             int64_t& k) {
  if constexpr (LAST) {
    k = i / a.Cg;
    return a.part[(b * a.f.nchunk + k) * a.f.C + g * a.Cg + (i - k * a.Cg)];
  } else {
    k = i % a.f.nchunk;
    return a.part[(b * a.f.C + g * a.Cg) * a.f.nchunk + i];
  }
}

// One CTA per (element, group): mean and M2 of the group from its partials,
// merged in double: mean = sum n_i mean_i / n, then
// M2 = sum M2_i + n_i (mean_i - mean)^2.
template <bool LAST>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_stats(const __grid_constant__ NormArgs a) {
  __shared__ double tmp[FEAT_WARPS];
  const int64_t b = blockIdx.x / a.G, g = blockIdx.x - b * a.G;
  const int64_t n_parts = a.Cg * a.f.nchunk;
  const double n = (double)a.Cg * (double)a.f.S;
  double s = 0.0, m2 = 0.0;
  int64_t k;
  for (int64_t i = threadIdx.x; i < n_parts; i += FEAT_THREADS) {
    const float2 q = group_part<LAST>(a, b, g, i, k);
    s += (double)chunk_count(a.f, k) * (double)q.x;
  }
  const double mean = block_sum(s, tmp) / n;
  for (int64_t i = threadIdx.x; i < n_parts; i += FEAT_THREADS) {
    const float2 q = group_part<LAST>(a, b, g, i, k);
    const double d = (double)q.x - mean;
    m2 += (double)q.y + (double)chunk_count(a.f, k) * d * d;
  }
  m2 = block_sum(m2, tmp);
  if (threadIdx.x == 0) {
    a.stats[2 * blockIdx.x] = (float)mean;
    a.stats[2 * blockIdx.x + 1] = (float)(1.0 / sqrt(m2 / n + (double)a.eps));
  }
}

// One CTA per (element, group): each channel's sums (one warp a channel), and
// the group's two coefficients.
template <bool LAST>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_coefs(const __grid_constant__ NormArgs a) {
  __shared__ double tmp[FEAT_WARPS];
  const int64_t b = blockIdx.x / a.G, g = blockIdx.x - b * a.G;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  double s1 = 0.0, s2 = 0.0;
  for (int64_t j = warp; j < a.Cg; j += FEAT_WARPS) {
    const int64_t c = g * a.Cg + j;
    double p = 0.0, q = 0.0;
    for (int64_t k = lane; k < a.f.nchunk; k += 32) {
      const float2 t = LAST ? a.part[(b * a.f.nchunk + k) * a.f.C + c]
                            : a.part[(b * a.f.C + c) * a.f.nchunk + k];
      p += (double)t.x;
      q += (double)t.y;
    }
    p = warp_sum(p);
    q = warp_sum(q);
    if (lane == 0) {
      a.chan[b * a.f.C + c] = make_float2((float)p, (float)q);
      const double w = (double)norm_param(a.weight, a.w_bf16, c, 1.0f);
      s1 += w * p;
      s2 += w * q;
    }
  }
  s1 = block_sum(s1, tmp);
  s2 = block_sum(s2, tmp);
  if (threadIdx.x == 0) {
    const double n = (double)a.Cg * (double)a.f.S;
    const double r = (double)a.stats[2 * blockIdx.x + 1];
    a.coef[blockIdx.x] = make_float2((float)(r * s1 / n), (float)(r * r * s2 / n));
  }
}

// The gradients of weight and bias: a channel's sums over the batch.
__global__ void norm_param_grads(const __grid_constant__ NormArgs a) {
  const int64_t c = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (c >= a.f.C) return;
  double db = 0.0, dw = 0.0;
  for (int64_t b = 0; b < a.f.B; ++b) {
    const float2 t = a.chan[b * a.f.C + c];
    db += (double)t.x;
    dw += (double)t.y;
  }
  const int dt = a.w_bf16 ? BA_BF16 : BA_F32;
  if (a.dweight != nullptr) store_f(a.dweight, dt, c, (float)dw);
  if (a.dbias != nullptr) store_f(a.dbias, dt, c, (float)db);
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

struct NormScratch {
  size_t part, coef, chan, total;  // byte offsets
};

NormScratch norm_scratch(const Feat& f, int64_t G, bool backward) {
  NormScratch s;
  s.part = 0;
  s.coef = align16((size_t)(f.B * f.C * f.nchunk) * sizeof(float2));
  s.chan = s.coef + (backward ? align16((size_t)(f.B * G) * sizeof(float2)) : 0);
  s.total = s.chan + (backward ? align16((size_t)(f.B * f.C) * sizeof(float2)) : 0);
  return s;
}

ba_status norm_check(const char* what, const ba_norm_desc* d) {
  BA_REQUIRE(d != nullptr, "%s: desc is NULL", what);
  ba_status st = feat_check(what, d->batch, d->channels, d->H, d->W, d->D, d->dtype, d->layout);
  if (st != BA_OK) return st;
  BA_REQUIRE(d->groups > 0 && d->channels % d->groups == 0,
             "%s: %lld groups do not divide %lld channels", what, (long long)d->groups,
             (long long)d->channels);
  BA_REQUIRE(d->param_dtype == BA_F32 || d->param_dtype == BA_BF16, "%s: bad param_dtype %d", what,
             d->param_dtype);
  BA_REQUIRE(d->activation >= BA_ACT_NONE && d->activation <= BA_ACT_GELU,
             "%s: unknown activation %d", what, d->activation);
  BA_REQUIRE(d->eps >= 0.0f, "%s: eps=%g is negative or NaN", what, (double)d->eps);
  BA_REQUIRE(d->p_elem != nullptr || (d->p >= 0.0f && d->p <= 1.0f), "%s: p=%g not in [0, 1]",
             what, (double)d->p);
  BA_REQUIRE(d->batch * d->groups <= 0x7FFFFFFF, "%s: batch * groups exceeds 2^31 - 1", what);
  return BA_OK;
}

Feat norm_plan(const ba_norm_desc& d, bool backward) {
  const void* ptrs[3] = {d.x, d.out, d.dy};
  return feat_plan(d.batch, d.channels, d.H * d.W * d.D, d.dtype, d.layout, ptrs,
                   backward ? 3 : 2);
}

ba_status norm_run(const char* what, const ba_norm_desc* desc, bool backward, void* workspace,
                   size_t workspace_bytes, cudaStream_t cs) {
  clear_error();
  ba_status st = norm_check(what, desc);
  if (st != BA_OK) return st;
  const ba_norm_desc& d = *desc;
  const int64_t S = d.H * d.W * d.D;
  const size_t esz = d.dtype == BA_BF16 ? 2 : 4, psz = d.param_dtype == BA_BF16 ? 2 : 4;
  if (d.batch * d.channels * S == 0) {
    if (backward && d.channels > 0) {  // sums over nothing
      if ((d.dweight && cudaMemsetAsync(d.dweight, 0, d.channels * psz, cs) != cudaSuccess) ||
          (d.dbias && cudaMemsetAsync(d.dbias, 0, d.channels * psz, cs) != cudaSuccess)) {
        set_error("%s: clearing the parameters' gradients failed", what);
        return BA_ECUDA;
      }
    }
    return BA_OK;
  }
  BA_REQUIRE(d.x && d.stats && (backward ? d.dy : d.out), "%s: NULL tensor", what);
  BA_REQUIRE((uintptr_t)d.x % esz == 0 && (uintptr_t)d.out % esz == 0 &&
                 (!backward || (uintptr_t)d.dy % esz == 0) && (uintptr_t)d.weight % psz == 0 &&
                 (uintptr_t)d.bias % psz == 0 && (uintptr_t)d.dweight % psz == 0 &&
                 (uintptr_t)d.dbias % psz == 0 && (uintptr_t)d.stats % 8 == 0 &&
                 (uintptr_t)d.p_elem % 4 == 0 && (uintptr_t)d.seed_dev % 8 == 0,
             "%s: a pointer is not aligned to its type", what);
  const size_t bytes = (size_t)(d.batch * d.channels * S) * esz;
  BA_REQUIRE(d.out == nullptr || (!feat_overlap(d.x, d.out, bytes) &&
                                  (!backward || !feat_overlap(d.dy, d.out, bytes))),
             "%s: out overlaps an input", what);
  NormArgs a;
  memset(&a, 0, sizeof(a));
  a.f = norm_plan(d, backward);
  const NormScratch sc = norm_scratch(a.f, d.groups, backward);
  BA_REQUIRE(workspace != nullptr && workspace_bytes >= sc.total,
             "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0,
             sc.total);
  BA_REQUIRE((uintptr_t)workspace % 16 == 0, "%s: workspace not 16-byte aligned", what);
  a.x = d.x;
  a.dy = d.dy;
  a.out = d.out;
  a.weight = d.weight;
  a.bias = d.bias;
  a.dweight = d.dweight;
  a.dbias = d.dbias;
  a.w_bf16 = d.param_dtype == BA_BF16;
  a.stats = d.stats;
  a.part = (float2*)((char*)workspace + sc.part);
  a.coef = (float2*)((char*)workspace + sc.coef);
  a.chan = (float2*)((char*)workspace + sc.chan);
  a.G = d.groups;
  a.Cg = d.channels / d.groups;
  a.eps = d.eps;
  a.slope = d.activation == BA_ACT_LEAKY_RELU ? d.slope : 0.0f;
  a.drop = {d.p, d.p_elem, nullptr, (uint32_t)d.seed, (uint32_t)(d.seed >> 32), d.seed_dev,
            d.elem_offset, 1};
  const bool last = d.layout == BA_CHANNELS_LAST;
  NormLaunch l;
  l.act = d.activation == BA_ACT_NONE   ? ACT_NONE
          : d.activation == BA_ACT_SILU ? ACT_SILU
          : d.activation == BA_ACT_GELU ? ACT_GELU
                                        : ACT_LEAKY;
  l.drop = d.p_elem != nullptr || d.p > 0.0f;
  l.stream = cs;
  st = feat_grid(what, a.f, d.layout, &l.grid);
  if (st != BA_OK) return st;
  auto launch = [&](int step) {
    l.step = step;
    if (d.dtype == BA_BF16)
      last ? norm_launch_bf16_last(a, l) : norm_launch_bf16_first(a, l);
    else
      last ? norm_launch_f32_last(a, l) : norm_launch_f32_first(a, l);
    return check_launch(what);
  };
  const unsigned groups = (unsigned)(d.batch * d.groups);
  if ((st = launch(backward ? NORM_BWD_SUMS : NORM_SUMS)) != BA_OK) return st;
  if (!backward) {
    if (last)
      norm_stats<true><<<groups, FEAT_THREADS, 0, cs>>>(a);
    else
      norm_stats<false><<<groups, FEAT_THREADS, 0, cs>>>(a);
    if ((st = check_launch(what)) != BA_OK) return st;
    return launch(NORM_APPLY);
  }
  if (last)
    norm_coefs<true><<<groups, FEAT_THREADS, 0, cs>>>(a);
  else
    norm_coefs<false><<<groups, FEAT_THREADS, 0, cs>>>(a);
  if ((st = check_launch(what)) != BA_OK) return st;
  if (a.dweight != nullptr || a.dbias != nullptr) {
    norm_param_grads<<<(unsigned)((d.channels + 255) / 256), 256, 0, cs>>>(a);
    if ((st = check_launch(what)) != BA_OK) return st;
  }
  return d.out != nullptr ? launch(NORM_BWD_APPLY) : BA_OK;
}

}  // namespace
}  // namespace ba

extern "C" size_t ba_norm_workspace_bytes(const ba_norm_desc* desc, int32_t backward) {
  using namespace ba;
  clear_error();
  if (norm_check("ba_norm_workspace_bytes", desc) != BA_OK) return 0;
  if (desc->batch * desc->channels * desc->H * desc->W * desc->D == 0) return 0;
  return norm_scratch(norm_plan(*desc, backward != 0), desc->groups, backward != 0).total;
}

extern "C" ba_status ba_norm_forward(const ba_norm_desc* desc, void* workspace,
                                     size_t workspace_bytes, ba_stream_t stream) {
  return ba::norm_run("ba_norm_forward", desc, false, workspace, workspace_bytes,
                      (cudaStream_t)stream);
}

extern "C" ba_status ba_norm_backward(const ba_norm_desc* desc, void* workspace,
                                      size_t workspace_bytes, ba_stream_t stream) {
  return ba::norm_run("ba_norm_backward", desc, true, workspace, workspace_bytes,
                      (cudaStream_t)stream);
}

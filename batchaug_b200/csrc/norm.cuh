// Group norm with an activation and a counter-based dropout behind it,
// forward and backward, on (B, C, S) tensors (S = H * W * D) in channels-last
// (B, S, C) or channels-first (B, C, S) memory.
//
//   mean_g, rstd_g = statistics of group g of an element (C / G channels by S
//                    voxels, n values); rstd = 1 / sqrt(var + eps), biased var
//   z = (x - mean) * rstd * w_c + b_c,   y = act(z),   out = keep ? y * k : 0
//   dz = (keep ? dout * k : 0) * act'(z)
//   dw_c = sum dz * xh,  db_c = sum dz   (xh = (x - mean) * rstd; over B and S)
//   dx = rstd * (w dz - sum_g(w dz) / n - xh * sum_g(w dz xh) / n)
//
// Sums are per channel first ("partials": one pair for each channel of each
// chunk of voxels), and merged in a fixed order in double: no atomics, the
// same bits from every run.  A forward partial is (mean, M2), taken with the
// thread's own first value subtracted: that shift is one of the summed
// values, so its distance from the mean is itself part of the variance, and
// M2's relative error stays below the number of values a thread sums times
// 2^-24, whatever the data's offset.
//
// Everything else is one read of the inputs and one write of the output; the
// dropout bits are drawn again where they are needed (dropout.cuh).
#pragma once

#include "feature.cuh"

namespace ba {

enum { ACT_NONE = 0, ACT_LEAKY = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;           // y, or dx
  const void* weight;  // (C,) or NULL
  const void* bias;
  int32_t w_bf16;      // weight and bias are bf16 (else fp32)
  float* stats;        // (B, G, 2): mean, rstd
  float2* part;        // partials
  float2* coef;        // backward (B, G): rstd * sum(w dz) / n, rstd^2 * sum(w dz xh) / n
  float2* chan;        // backward (B, C): sum dz, sum dz xh
  void* dweight;       // (C,) or NULL, of the weight's type
  void* dbias;
  Feat f;
  int64_t G, Cg;
  float eps, slope;
  DropArgs drop;
};

__device__ __forceinline__ float norm_param(const void* p, int bf16, int64_t c, float absent) {
  return p == nullptr ? absent : load_f(p, bf16 ? BA_BF16 : BA_F32, c);
}

// ---------------------------------------------------------------------------
// Activations.  exp and the reciprocal are the hardware's (2 ulp), well below
// the outputs' tolerance in either type.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float z) {
  return __fdividef(1.0f, 1.0f + __expf(-z));
}

template <int ACT>
__device__ __forceinline__ float act_value(float z, float slope) {
  if constexpr (ACT == ACT_LEAKY) return z < 0.0f ? (slope == 0.0f ? 0.0f : z * slope) : z;
  if constexpr (ACT == ACT_SILU) return z * sigmoid(z);
  if constexpr (ACT == ACT_GELU)
    return z * __fmaf_rn(0.5f, erff(z * 0.70710678f), 0.5f);
  return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z, float slope) {
  if constexpr (ACT == ACT_LEAKY) return z > 0.0f ? 1.0f : slope;
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return __fmaf_rn(__fmaf_rn(-s, s, s), z, s);  // s + z s (1 - s)
  }
  if constexpr (ACT == ACT_GELU) {
    const float cdf = __fmaf_rn(0.5f, erff(z * 0.70710678f), 0.5f);
    return __fmaf_rn(z * 0.39894228f, __expf(-0.5f * z * z), cdf);
  }
  return 1.0f;
}

// ---------------------------------------------------------------------------
// A channel's constants.
// ---------------------------------------------------------------------------
struct ChanConst {
  float mean, a, bias;  // z = (x - mean) * a + bias
  float c2, c3;         // dx = a dz - c2 - (x - mean) c3
  float rstd;
};

template <bool COEF>
__device__ __forceinline__ ChanConst chan_const(const NormArgs& a, int64_t b, int64_t c) {
  ChanConst k;
  const int64_t g = b * a.G + c / a.Cg;
  k.mean = a.stats[2 * g];
  k.rstd = a.stats[2 * g + 1];
  k.a = k.rstd * norm_param(a.weight, a.w_bf16, c, 1.0f);
  k.bias = norm_param(a.bias, a.w_bf16, c, 0.0f);
  k.c2 = k.c3 = 0.0f;
  if constexpr (COEF) {
    const float2 q = a.coef[g];
    k.c2 = q.x;
    k.c3 = q.y;
  }
  return k;
}

template <int ACT, bool DROP>
__device__ __forceinline__ float norm_fwd(float x, const ChanConst& k, float slope, bool keep,
                                          float scale) {
  float y = act_value<ACT>(__fmaf_rn(x - k.mean, k.a, k.bias), slope);
  if constexpr (DROP) y = keep ? y * scale : 0.0f;
  return y;
}

// dz from dout
template <int ACT, bool DROP>
__device__ __forceinline__ float norm_dz(float xm, float dy, const ChanConst& k, float slope,
                                         bool keep, float scale) {
  float dz = dy * act_slope<ACT>(ACT == ACT_NONE ? 0.0f : __fmaf_rn(xm, k.a, k.bias), slope);
  if constexpr (DROP) dz = keep ? dz * scale : 0.0f;
  return dz;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sum over the CTA, in every thread; `tmp` holds FEAT_WARPS values.
__device__ __forceinline__ double block_sum(double v, double* tmp) {
  v = warp_sum(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) tmp[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < FEAT_WARPS; ++i) v += tmp[i];
  return v;
}

// ===========================================================================
// Channels last
// ===========================================================================
// The constants of a thread's VEC channels, through shared memory (one
// channel's are resolved once per CTA).
template <int VEC, bool COEF>
__device__ __forceinline__ void last_consts(const NormArgs& a, const LastPlace& p, ChanConst* k,
                                            float (*sm)[FEAT_MAX_COLS]) {
  const int64_t c0 = (int64_t)blockIdx.y * a.f.ncw * VEC;
  for (int i = threadIdx.x; i < a.f.ncw * VEC; i += FEAT_THREADS) {
    if (c0 + i < a.f.C) {
      const ChanConst q = chan_const<COEF>(a, p.b, c0 + i);
      sm[0][i] = q.mean;
      sm[1][i] = q.a;
      sm[2][i] = q.bias;
      if constexpr (COEF) {
        sm[3][i] = q.c2;
        sm[4][i] = q.c3;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int j = p.tx * VEC + i;
    k[i].mean = sm[0][j];
    k[i].a = sm[1][j];
    k[i].bias = sm[2][j];
    if constexpr (COEF) {
      k[i].c2 = sm[3][j];
      k[i].c3 = sm[4][j];
    }
  }
}

// y (BWD = false) or dx of one chunk.
template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_apply_last(const __grid_constant__ NormArgs a) {
  __shared__ float sm[BWD ? 5 : 3][FEAT_MAX_COLS];
  const LastPlace p = last_place<VEC>(a.f);
  ChanConst k[VEC];
  last_consts<VEC, BWD>(a, p, k, sm);
  if (!p.on) return;
  DropRate dr;
  if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  const int64_t base = p.b * a.f.S * a.f.C + p.c;
  for (int64_t r = p.r0 + p.ty * 8; r < p.r1; r += p.nty * 8) {
    Raw<DT, VEC> rx[8], rd[BWD ? 8 : 1];
    const int n = (int)min((int64_t)8, p.r1 - r);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) {
        rx[j] = raw_load<DT, VEC>(a.x, base + (r + j) * a.f.C);
        if constexpr (BWD) rd[j] = raw_load<DT, VEC>(a.dy, base + (r + j) * a.f.C);
      }
    uint32_t keep[VEC];
    if constexpr (DROP) last_keep<VEC>(a.f, dr, p.c, r, keep);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) {
        float v[VEC], d[VEC];
        raw_unpack<DT, VEC>(rx[j], v);
        if constexpr (BWD) raw_unpack<DT, VEC>(rd[j], d);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const bool kp = DROP ? (keep[i] >> j) & 1u : true;
          const float sc = DROP ? dr.scale : 1.0f;
          if constexpr (BWD) {
            const float xm = v[i] - k[i].mean;
            const float dz = norm_dz<ACT, DROP>(xm, d[i], k[i], a.slope, kp, sc);
            v[i] = __fmaf_rn(k[i].a, dz, __fmaf_rn(-xm, k[i].c3, -k[i].c2));
          } else {
            v[i] = norm_fwd<ACT, DROP>(v[i], k[i], a.slope, kp, sc);
          }
        }
        raw_store<DT, VEC>(a.out, base + (r + j) * a.f.C, raw_pack<DT, VEC>(v));
      }
  }
}

// Sum of `v` over the threads of a column (same tx), returned to ty == 0;
// sm holds FEAT_THREADS floats.
__device__ __forceinline__ float column_sum(float v, const LastPlace& p, int ncw, float* sm) {
  __syncthreads();
  sm[threadIdx.x] = v;
  int m = p.nty;
  while (m > 1) {
    __syncthreads();
    const int h = (m + 1) >> 1;
    if (p.ty < m - h) sm[threadIdx.x] += sm[threadIdx.x + h * ncw];
    m = h;
  }
  __syncthreads();
  return sm[p.tx];
}

// The partials of one chunk: (mean, M2) of x, or (sum dz, sum dz xh).
template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_sums_last(const __grid_constant__ NormArgs a) {
  __shared__ float sc[BWD ? 3 : 1][FEAT_MAX_COLS];
  __shared__ float sm[FEAT_THREADS];
  const LastPlace p = last_place<VEC>(a.f);
  const int64_t base = p.b * a.f.S * a.f.C + p.c;
  float s0[VEC], s1[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) s0[i] = s1[i] = 0.0f;
  if constexpr (!BWD) {
    float shift[VEC];
    int64_t cnt = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) shift[i] = 0.0f;
    const int64_t first = p.r0 + p.ty;
    if (p.on && first < p.r1) raw_unpack<DT, VEC>(raw_load<DT, VEC>(a.x, base + first * a.f.C), shift);
    for (int64_t r = first; r < p.r1 && p.on; r += p.nty * 8) {
      Raw<DT, VEC> rx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r + j * p.nty < p.r1) rx[j] = raw_load<DT, VEC>(a.x, base + (r + j * p.nty) * a.f.C);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r + j * p.nty < p.r1) {
          float v[VEC];
          raw_unpack<DT, VEC>(rx[j], v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float t = v[i] - shift[i];
            s0[i] += t;
            s1[i] = __fmaf_rn(t, t, s1[i]);
          }
          ++cnt;
        }
    }
    // the chunk's mean from the threads' sums about the column's first shift,
    // then the sum of squares about that mean
    const float n = (float)cnt, inv = 1.0f / (float)(p.r1 - p.r0);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      __syncthreads();
      if (p.ty == 0) sm[p.tx] = shift[i];
      __syncthreads();
      const float k0 = sm[p.tx];
      const float mt = cnt > 0 ? s0[i] / n : 0.0f;  // the thread's mean - its shift
      const float off = (shift[i] - k0) + mt;       // the thread's mean - k0
      const float m = column_sum(n * off, p, a.f.ncw, sm) * inv;
      const float dm = off - m;
      const float m2 = s1[i] - s0[i] * mt + n * dm * dm;
      s1[i] = column_sum(cnt > 0 ? m2 : 0.0f, p, a.f.ncw, sm);
      s0[i] = k0 + m;
    }
  } else {
    ChanConst k[VEC];
    last_consts<VEC, false>(a, p, k, sc);
    DropRate dr;
    if constexpr (DROP) dr = drop_rate(a.drop, p.b);
    for (int64_t r = p.r0 + p.ty * 8; r < p.r1 && p.on; r += p.nty * 8) {
      Raw<DT, VEC> rx[8], rd[8];
      const int n = (int)min((int64_t)8, p.r1 - r);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) {
          rx[j] = raw_load<DT, VEC>(a.x, base + (r + j) * a.f.C);
          rd[j] = raw_load<DT, VEC>(a.dy, base + (r + j) * a.f.C);
        }
      uint32_t keep[VEC];
      if constexpr (DROP) last_keep<VEC>(a.f, dr, p.c, r, keep);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) {
          float v[VEC], d[VEC];
          raw_unpack<DT, VEC>(rx[j], v);
          raw_unpack<DT, VEC>(rd[j], d);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const bool kp = DROP ? (keep[i] >> j) & 1u : true;
            const float xm = v[i] - k[i].mean;
            const float dz = norm_dz<ACT, DROP>(xm, d[i], k[i], a.slope, kp,
                                                DROP ? dr.scale : 1.0f);
            s0[i] += dz;
            s1[i] = __fmaf_rn(dz, xm, s1[i]);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      s0[i] = column_sum(s0[i], p, a.f.ncw, sm);
      s1[i] = column_sum(s1[i], p, a.f.ncw, sm);
    }
  }
  if (p.on && p.ty == 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float q = s1[i];
      if constexpr (BWD) q *= a.stats[2 * (p.b * a.G + (p.c + i) / a.Cg) + 1];
      a.part[(p.b * a.f.nchunk + p.k) * a.f.C + p.c + i] = make_float2(s0[i], q);
    }
  }
}

// ===========================================================================
// Channels first
// ===========================================================================
// Tiles whose loads are in flight together.
constexpr int FIRST_FLIGHT = 4;

template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_apply_first(const __grid_constant__ NormArgs a) {
  FirstPlace p;
  if (!first_place(a.f, p)) return;
  const ChanConst k = chan_const<BWD>(a, p.b, p.c);
  DropRate dr;
  if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  for (int64_t s = p.s0; s < p.s1; s += FEAT_TILE * FIRST_FLIGHT) {
    FirstTile<DT, VEC> tx[FIRST_FLIGHT], td[BWD ? FIRST_FLIGHT : 1];
#pragma unroll
    for (int u = 0; u < FIRST_FLIGHT; ++u) {
      first_load<DT, VEC>(a.x, p, s + u * FEAT_TILE, tx[u]);
      if constexpr (BWD) first_load<DT, VEC>(a.dy, p, s + u * FEAT_TILE, td[u]);
    }
#pragma unroll
    for (int u = 0; u < FIRST_FLIGHT; ++u) {
      const int64_t su = s + u * FEAT_TILE;
      if (su < p.s1) {
        uint32_t keep = 0xFFu;
        if constexpr (DROP) keep = first_keep<VEC>(a.f, dr, p, su);
        float v[8], d[8];
        first_unpack<DT, VEC>(tx[u], v);
        if constexpr (BWD) first_unpack<DT, VEC>(td[u], d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool kp = DROP ? (keep >> i) & 1u : true;
          const float sc = DROP ? dr.scale : 1.0f;
          if constexpr (BWD) {
            const float xm = v[i] - k.mean;
            const float dz = norm_dz<ACT, DROP>(xm, d[i], k, a.slope, kp, sc);
            v[i] = __fmaf_rn(k.a, dz, __fmaf_rn(-xm, k.c3, -k.c2));
          } else {
            v[i] = norm_fwd<ACT, DROP>(v[i], k, a.slope, kp, sc);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; j += VEC)
          if (su + first_at<VEC>(p.lane, j) < p.s1)
            raw_store<DT, VEC>(a.out, p.base + su + first_at<VEC>(p.lane, j),
                               raw_pack<DT, VEC>(v + j));
      }
    }
  }
}

template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_sums_first(const __grid_constant__ NormArgs a) {
  FirstPlace p;
  if (!first_place(a.f, p)) return;
  float s0 = 0.0f, s1 = 0.0f, shift = 0.0f;
  ChanConst k = {};
  DropRate dr;
  int cnt = 0;
  if constexpr (BWD) {
    k = chan_const<false>(a, p.b, p.c);
    if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  } else if (p.s0 + first_at<VEC>(p.lane, 0) < p.s1) {
    shift = load_f(a.x, DT, p.base + p.s0 + first_at<VEC>(p.lane, 0));
  }
  for (int64_t s = p.s0; s < p.s1; s += FEAT_TILE * FIRST_FLIGHT) {
    FirstTile<DT, VEC> tx[FIRST_FLIGHT], td[BWD ? FIRST_FLIGHT : 1];
#pragma unroll
    for (int u = 0; u < FIRST_FLIGHT; ++u) {
      first_load<DT, VEC>(a.x, p, s + u * FEAT_TILE, tx[u]);
      if constexpr (BWD) first_load<DT, VEC>(a.dy, p, s + u * FEAT_TILE, td[u]);
    }
#pragma unroll
    for (int u = 0; u < FIRST_FLIGHT; ++u) {
      const int64_t su = s + u * FEAT_TILE;
      if (su < p.s1) {
        uint32_t keep = 0xFFu;
        if constexpr (BWD && DROP) keep = first_keep<VEC>(a.f, dr, p, su);
        float v[8], d[8];
        first_unpack<DT, VEC>(tx[u], v);
        if constexpr (BWD) first_unpack<DT, VEC>(td[u], d);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (su + first_at<VEC>(p.lane, i) < p.s1) {
            if constexpr (BWD) {
              const float xm = v[i] - k.mean;
              const float dz = norm_dz<ACT, DROP>(xm, d[i], k, a.slope, (keep >> i) & 1u,
                                                  DROP ? dr.scale : 1.0f);
              s0 += dz;
              s1 = __fmaf_rn(dz, xm, s1);
            } else {
              const float t = v[i] - shift;
              s0 += t;
              s1 = __fmaf_rn(t, t, s1);
              ++cnt;
            }
          }
      }
    }
  }
  if constexpr (BWD) {
    s0 = warp_sum(s0);
    s1 = warp_sum(s1) * k.rstd;
  } else {
    // as norm_sums_last: the run's mean about lane 0's shift, then M2
    const float n = (float)cnt;
    const float k0 = __shfl_sync(0xFFFFFFFFu, shift, 0);
    const float mt = cnt > 0 ? s0 / n : 0.0f;
    const float off = (shift - k0) + mt;
    const float m = warp_sum(cnt > 0 ? n * off : 0.0f) / (float)(p.s1 - p.s0);
    const float dm = off - m;
    s1 = warp_sum(cnt > 0 ? s1 - s0 * mt + n * dm * dm : 0.0f);
    s0 = k0 + m;
  }
  if (p.lane == 0) a.part[p.item] = make_float2(s0, s1);
}

}  // namespace ba

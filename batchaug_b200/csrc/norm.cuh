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
// One launch does it all, a cooperative one where a CTA waits for others that
// are not of its cluster.  A unit is what is normalised on its
// own: a group of an element (channels first), or the groups of a block of
// columns of an element (channels last).  Each set of CTAs takes units in
// waves; its CTAs share a wave's items (equal parts of its units' voxels),
// first for the sums, then for the results.  Every CTA leaves a partial for
// each group of its item, and a CTA that needs a unit's statistics reads the
// partials of all its items and merges them itself, in double and in a fixed
// order (no atomics on sums: the same bits from every run).  A partial's words
// are zero until they are written, so reading them is waiting for them: no
// counter, no fence, no second hop.  The sets' waves together are small
// enough for their inputs to be in L2 still when the results read them again,
// so HBM sees them once; where a unit alone is larger than that, the results
// begin with the items' ends and find those there.  Channels first, the results
// are taken in pieces of an item, first come, first served, the next piece's
// loads behind those of the one at hand (32 units of 8 MB: 153 -> 124 us, with
// the rings on whole lines).  Channels last, the same was slower (2x64x64^3
// forward 41 -> 43 us, backward 64 -> 67; 2x32x128^3 145 -> 146, 233 -> 230), and
// an item's results stay with its CTA.  (The sums' shares are the same every
// time, so that the order of a sum is.)  A unit of up to 512 KB is a cluster of up
// to eight CTAs, unless there are more units than resident CTAs, or (channels
// first) more than 64 channels in a group: its barrier takes the place of the
// waiting, so no zeroed words and no cooperative launch, which is most of what a
// small call costs.
//
// A forward partial is the first and second moment about a value near the
// mean, that value and the count.  A thread sums in fp32 about a centre: its
// first value (channels first, the mean of its first access), and from then on
// the mean of its values so far, taken after 1, 2 and 4 blocks of eight
// accesses and after every fourth (`recentre`).  Sums about the first of n
// values exceed M2 by a factor of n at most (it may be background, the others
// not), those about the mean of as many values before them by 2.  With m <= 64
// values to an accumulator between two centres (16 up to the first), its roundings
// and those of the first moment make 3 m + 2 units: M2's relative error stays
// below 8 * 50 * 2^-24, and 2^-24 more for each centre, whatever the data's offset
// and order.  Where threads' sums meet, they are about a centre of theirs, or in
// double.  (2x64x48^3 bf16 last, two centres a thread: 21.2 us, about the first
// value alone 20.0; 2x32x128^3 and the channels-first volumes the same.)  The
// backward sums have no centre: fp32 over a thread's part, within as many units of
// 2^-24 of their terms' magnitudes as it has values (up to some hundreds at the
// sizes measured), and double from there.
#pragma once

#include "feature.cuh"

namespace ba {

enum { ACT_NONE = 0, ACT_LEAKY = 1, ACT_SILU = 2, ACT_GELU = 3 };

// Blocks of a piece of the results.
constexpr int NORM_PIECE = 4;

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;           // y, or dx (NULL: not wanted)
  const void* weight;  // (C,) or NULL
  const void* bias;
  int32_t w_bf16;      // weight and bias are bf16 (else fp32)
  float* stats;        // (B, G, 2): mean, rstd
  float4* part;        // a partial for each (unit, group of the unit, item):
                       // centre, second and first moment about it, count /
                       // sum w dz, 0, sum w dz xh, 1.  Zeroed before the launch
  float2* chan;        // backward, where weight or bias want a gradient: sum dz,
                       // sum dz xh of each channel of each chunk
  void* dweight;       // (C,) or NULL, of the weight's type
  void* dbias;
  uint32_t* done;      // backward, zeroed: items whose `chan` is written
  unsigned int* timeouts;  // where a wait that gave up is recorded, or NULL
  Feat f;
  uint32_t G, Cg;
  // the schedule (norm.cu)
  uint32_t units;
  uint32_t wave;   // units of a wave
  uint32_t items;  // work items of a unit
  uint32_t ugroups; // groups of a unit
  uint32_t sets;    // the CTAs are so many sets, each taking every sets-th wave
  uint32_t subs;     // channels first: pieces of an item
  int64_t sub_rows;  // voxels of a piece, of a channel
  uint32_t* ticket;  // zeroed: those taken of each unit (subs > 1)
  int32_t reverse;   // results from the last voxels of the items to the first
  int32_t cluster; // a unit is a thread block cluster (small units)
  double inv_n;    // 1 / values of a group
  float eps, slope;
  DropArgs drop;
};

__device__ __forceinline__ float norm_param(const void* p, int bf16, int64_t c, float absent) {
  return p == nullptr ? absent : load_f(p, bf16 ? BA_BF16 : BA_F32, c);
}

// ---------------------------------------------------------------------------
// Activations, on pairs.  exp2 and the reciprocal are the hardware's, within 2^-22
// and 2^-23 of their value: what an fp32 result is off by beside its own
// rounding, and nothing in bf16.  An SM
// makes 16 of them a clock, so they are what an activation costs.  (Sharing
// one reciprocal among four values, 1/a = b (1/(a b)), took 3 to 7 % off a
// forward pass with silu, but a value's last bit then depends on its
// neighbours', of other groups too; it was not kept.)
// ---------------------------------------------------------------------------
__device__ __forceinline__ float exp2_hw(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_hw(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN if either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 exp2_2(F2 t) { return f2(exp2_hw(t.x()), exp2_hw(t.y())); }

__device__ __forceinline__ F2 rcp2(F2 t) { return f2(rcp_hw(t.x()), rcp_hw(t.y())); }

// 1 / (1 + exp(-z)).  The exponent's rounding is |z| 2^-24 of the exponential, which
// for negative z is the value's own; FINE (fp32 results) gives it back to first
// order.  Bf16 has no room for it, and a slope is a sum of order one.
template <bool FINE>
__device__ __forceinline__ F2 sigmoid2(F2 z) {
  if constexpr (FINE) {
    z = f2(min_nan(z.x(), 256.0f), min_nan(z.y(), 256.0f));  // 1 from 18 on, infinity too
    const F2 c = f2(-1.44269504f), a = mul2(z, c);
    F2 r = fma2(z, c, mul2(a, f2(-1.0f)));  // lost of the product and of the constant
    r = fma2(z, f2(-1.9259630e-8f), r);
    return rcp2(fma2(exp2_2(a), fma2(r, f2(0.69314718f), f2(1.0f)), f2(1.0f)));
  }
  return rcp2(add2(exp2_2(mul2(z, f2(-1.44269504f))), f2(1.0f)));
}

// gelu, z Phi(z) = max(z, 0) - x q with x = |z| and the normal distribution's tail
// q = Phi(-x) = t P(t) exp(-x^2 / 2), t = 1 / (1 + c x).  P is by least squares
// weighted towards the largest error (Lawson's iteration) of exp(x^2 / 2) Phi(-x)
// / t, 0 <= x <= 14.5, so the tail keeps its digits (from 1 + erf it has none left
// at x = 5).  fp32: degree 7, 1.7e-7 of q; bf16: degree 5, 4.7e-6.  The exponent is
// rounded twice, x^2 2^-24 of q, which fp32 gets back to first order (then within
// 20 units of 2^-24 down to x = 12.5); bf16 has no room for it.
template <int DT>
__device__ __forceinline__ F2 gelu2(F2 z) {
  // from 15 on the tail is 0, and 256 does for infinity
  const F2 x = f2(min_nan(fabsf(z.x()), 256.0f), min_nan(fabsf(z.y()), 256.0f));
  const F2 xx = mul2(x, x), c = f2(-0.72134752f);  // -log2(e) / 2
  const F2 a = mul2(xx, c);
  F2 e = exp2_2(a);
  F2 t, q;
  if constexpr (DT == BA_F32) {
    F2 r = fma2(xx, c, mul2(a, f2(-1.0f)));           // lost of the product,
    r = fma2(xx, f2(-9.6298149e-9f), r);              // of the constant
    r = fma2(fma2(x, x, mul2(xx, f2(-1.0f))), c, r);  // and of the square
    e = mul2(e, fma2(r, f2(0.69314718f), f2(1.0f)));
    t = rcp2(fma2(x, f2(0.3f), f2(1.0f)));
    q = fma2(t, f2(0.035423707f), f2(-0.15615831f));
    q = fma2(q, t, f2(0.20455652f));
    q = fma2(q, t, f2(-0.052033797f));
    q = fma2(q, t, f2(0.12769167f));
    q = fma2(q, t, f2(0.10017598f));
    q = fma2(q, t, f2(0.12071214f));
    q = fma2(q, t, f2(0.11963201f));
  } else {
    t = rcp2(fma2(x, f2(0.31f), f2(1.0f)));
    q = fma2(t, f2(-0.073929138f), f2(0.18045032f));
    q = fma2(q, t, f2(0.015744729f));
    q = fma2(q, t, f2(0.13342978f));
    q = fma2(q, t, f2(0.12044128f));
    q = fma2(q, t, f2(0.1238607f));
  }
  return fma2(mul2(x, f2(-1.0f)), mul2(mul2(q, t), e),
              f2(fmaxf(z.x(), 0.0f), fmaxf(z.y(), 0.0f)));
}

// For the slope, a sum of order one, errors of 1e-7 are a rounding, and the shorter
// form does (with gelu2's tail the backward pass of 2x48x96^3 took 318 us, not
// 300): the normal distribution function and exp(-z^2 / 2), by Hastings' formula
// (Abramowitz and Stegun 7.1.26: erf(x) = 1 - (a1 t + .. + a5 t^5) exp(-x^2),
// t = 1 / (1 + p x), |error| <= 1.5e-7) with x = |z| / sqrt(2); exp(-x^2) is the
// density that the slope needs, so the slope costs no more exponentials.
__device__ __forceinline__ F2 normal_tail2(F2 t, F2 e) {
  // the coefficients are halved: 1 - cdf(|z|)
  F2 q = fma2(t, f2(0.5f * 1.061405429f), f2(0.5f * -1.453152027f));
  q = fma2(q, t, f2(0.5f * 1.421413741f));
  q = fma2(q, t, f2(0.5f * -0.284496736f));
  q = fma2(q, t, f2(0.5f * 0.254829592f));
  return mul2(mul2(q, t), e);
}
// 0.5 + sign(z) (0.5 - q)
__device__ __forceinline__ F2 normal_side2(F2 z, F2 q) {
  const F2 h = fma2(q, f2(-1.0f), f2(0.5f));
  return add2(f2(copysignf(h.x(), z.x()), copysignf(h.y(), z.y())), f2(0.5f));
}
__device__ __forceinline__ F2 normal_cdf2(F2 z, F2& e) {
  e = exp2_2(mul2(mul2(z, z), f2(-0.72134752f)));  // -log2(e) / 2
  const F2 x = f2(fabsf(z.x()), fabsf(z.y()));
  const F2 t = rcp2(fma2(x, f2(0.3275911f * 0.70710678f), f2(1.0f)));
  return normal_side2(z, normal_tail2(t, e));
}

__device__ __forceinline__ F2 leaky2(F2 z, float slope) {
  // slope 0: +0 for any negative z, infinite ones included
  const F2 n = slope == 0.0f ? f2(0.0f) : mul2(z, f2(slope));
  return f2(z.x() < 0.0f ? n.x() : z.x(), z.y() < 0.0f ? n.y() : z.y());
}

// act(z), and act'(z) of the smooth ones
template <int DT, int ACT>
__device__ __forceinline__ F2 act_value2(F2 z, float slope) {
  if constexpr (ACT == ACT_LEAKY) return leaky2(z, slope);
  if constexpr (ACT == ACT_SILU) return mul2(z, sigmoid2<DT == BA_F32>(z));
  if constexpr (ACT == ACT_GELU) return gelu2<DT>(z);
  return z;
}
template <int ACT>
__device__ __forceinline__ F2 act_slope2(F2 z) {
  if constexpr (ACT == ACT_SILU) {  // s + z s (1 - s)
    const F2 s = sigmoid2<false>(z);
    return fma2(mul2(z, s), fma2(s, f2(-1.0f), f2(1.0f)), s);
  }
  if constexpr (ACT == ACT_GELU) {  // cdf + z pdf
    F2 e;
    const F2 c = normal_cdf2(z, e);
    return fma2(mul2(z, f2(0.39894228f)), e, c);
  }
  return f2(1.0f);
}
// The gradient of act at z for a gradient of g.
template <int ACT>
__device__ __forceinline__ F2 act_grad2(F2 g, F2 z, float slope) {
  if constexpr (ACT == ACT_NONE) return g;
  if constexpr (ACT == ACT_LEAKY) {
    // slope 0: 0 whatever comes in, infinite ones included
    const F2 n = slope == 0.0f ? f2(0.0f) : mul2(g, f2(slope));
    return f2(z.x() > 0.0f ? g.x() : n.x(), z.y() > 0.0f ? g.y() : n.y());
  }
  return mul2(g, act_slope2<ACT>(z));
}

// ---------------------------------------------------------------------------
// A group's numbers, and a channel's constants made of them.
// ---------------------------------------------------------------------------
struct GroupStat {
  float mean, rstd;
  float c2, c3;  // backward: rstd sum(w dz) / n, rstd^2 sum(w dz xh) / n
};

// A pair's constants, negated where they are subtracted.
struct PairConst {
  F2 nmean, a, bias;
  F2 nc2, nc3;
};

// z = (x - mean) * a + bias with a = rstd * w; dx = a dz - c2 - (x - mean) c3.
__device__ __forceinline__ PairConst pair_const(const GroupStat& g, float w, float bias) {
  return {f2(-g.mean), f2(g.rstd * w), f2(bias), f2(-g.c2), f2(-g.c3)};
}

// x -> the results of two pairs (dy: its dropped elements zeroed); scale is
// dropout's, 1 without it.
template <int DT, int ACT, int DROP, bool BWD>
__device__ __forceinline__ void norm_pairs(RawPair<DT>& x0, RawPair<DT>& x1, RawPair<DT> d0,
                                           RawPair<DT> d1, const PairConst& k0,
                                           const PairConst& k1, float slope, float scale) {
  const F2 m0 = add2(pair_value<DT>(x0), k0.nmean), m1 = add2(pair_value<DT>(x1), k1.nmean);
  F2 z0 = fma2(m0, k0.a, k0.bias), z1 = fma2(m1, k1.a, k1.bias);
  if constexpr (BWD) {
    F2 g0 = pair_value<DT>(d0), g1 = pair_value<DT>(d1);
    if constexpr (ACT != ACT_NONE) {
      g0 = act_grad2<ACT>(g0, z0, slope);
      g1 = act_grad2<ACT>(g1, z1, slope);
    }
    const F2 a0 = DROP ? mul2(k0.a, f2(scale)) : k0.a, a1 = DROP ? mul2(k1.a, f2(scale)) : k1.a;
    x0 = pair_raw<DT>(fma2(a0, g0, fma2(m0, k0.nc3, k0.nc2)));
    x1 = pair_raw<DT>(fma2(a1, g1, fma2(m1, k1.nc3, k1.nc2)));
  } else {
    z0 = act_value2<DT, ACT>(z0, slope);
    z1 = act_value2<DT, ACT>(z1, slope);
    if constexpr (DROP) {
      z0 = mul2(z0, f2(scale));
      z1 = mul2(z1, f2(scale));
    }
    x0 = pair_raw<DT>(z0);
    x1 = pair_raw<DT>(z1);
  }
}

// Adds two pairs to their forward (x about the shift) or backward (dz, dz (x -
// mean), without dropout's scale) sums.
template <int DT, int ACT, bool BWD>
__device__ __forceinline__ void norm_add(RawPair<DT> x0, RawPair<DT> x1, RawPair<DT> d0,
                                         RawPair<DT> d1, const PairConst& k0, const PairConst& k1,
                                         float slope, F2& p0, F2& q0, F2& p1, F2& q1) {
  const F2 m0 = add2(pair_value<DT>(x0), k0.nmean), m1 = add2(pair_value<DT>(x1), k1.nmean);
  F2 g0 = m0, g1 = m1;
  if constexpr (BWD) {
    g0 = pair_value<DT>(d0);
    g1 = pair_value<DT>(d1);
    if constexpr (ACT != ACT_NONE) {
      g0 = act_grad2<ACT>(g0, fma2(m0, k0.a, k0.bias), slope);
      g1 = act_grad2<ACT>(g1, fma2(m1, k1.a, k1.bias), slope);
    }
  }
  p0 = add2(p0, g0);
  q0 = fma2(g0, m0, q0);
  p1 = add2(p1, g1);
  q1 = fma2(g1, m1, q1);
}

// After block q of a thread that has more of them.
__device__ __forceinline__ bool recentres(int q) { return q < 2 || (q & 3) == 3; }

// Forward: moves the centre to the mean of the thread's n values.  m2: their
// second moment about the centre, without what is in s1; s0, their first moment,
// keeps what the rounding of the new centre leaves.
__device__ __forceinline__ void recentre(F2& nmean, F2& s0, F2& s1, F2& m2, float n) {
  const F2 to = fma2(s0, f2(-rcp_hw(n)), nmean);
  const F2 by = fma2(nmean, f2(-1.0f), to);  // the step, negated
  const F2 left = fma2(by, f2(n), s0);
  m2 = add2(m2, fma2(by, add2(s0, left), s1));
  s0 = left;
  s1 = f2(0.0f);
  nmean = to;
}
// The same where the pair's halves are sums about one centre.
__device__ __forceinline__ void recentre_one(F2& nmean, F2& s0, F2& s1, F2& m2, float n) {
  s0 = f2(s0.x() + s0.y(), 0.0f);
  s1 = f2(s1.x() + s1.y(), 0.0f);
  recentre(nmean, s0, s1, m2, n);
  nmean = f2(nmean.x());
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// Of N values at once, so that their shuffles and additions overlap.
template <int N>
__device__ __forceinline__ void warp_sums(double* v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
}

// ===========================================================================
// Partials, from the CTA that has them to those that need them.
// ===========================================================================
constexpr unsigned long long NORM_WAIT_NS = 2000000000ull;

__device__ __forceinline__ unsigned long long wall_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void note_timeout(const NormArgs& a) {
  if (a.timeouts != nullptr) atomicOr(a.timeouts, 1u);
}

// Two 8-byte words, each written and read whole, and each not zero: the low
// halves are x and z, the high ones y with a set sign bit (a second moment, or
// 0) and w (not 0).
__device__ __forceinline__ void put_word(void* p, uint32_t lo, uint32_t hi) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"((uint64_t)hi << 32 | lo)
               : "memory");
}
__device__ __forceinline__ uint2 look_word(const void* p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}
__device__ __forceinline__ void put_part(float4* p, float x, float y, float z, uint32_t w) {
  put_word(p, __float_as_uint(x), __float_as_uint(y) | 0x80000000u);
  put_word(reinterpret_cast<uint2*>(p) + 1, __float_as_uint(z), w);
}
__device__ __forceinline__ uint4 look_part(const float4* p) {
  const uint2 a = look_word(p), b = look_word(reinterpret_cast<const uint2*>(p) + 1);
  return make_uint4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ bool is_part(const uint4& t) { return t.y != 0u && t.w != 0u; }

// Sums over the partials k = first, first + step, ... of a group or two, whose
// partials begin at q and, for the second (if `two`), q + next: forward, the
// moments about the centre of the first one (k0); backward, the two sums.  A
// look is a round trip to L2, half a microsecond and more, so NB partials of
// each group are looked at together, and those that are missing again: every
// CTA is resident and writes its partials before it reads any, so they will
// come, or the wait ends without them (false).
template <bool BWD, int GR, int NB>
__device__ __forceinline__ bool sum_parts(const NormArgs& a, const float4* q, bool two,
                                          int64_t next, uint32_t first, uint32_t step, double* s,
                                          double* m, double* k0) {
  unsigned long long t0 = 0;
#pragma unroll
  for (int g = 0; g < GR; ++g) s[g] = m[g] = k0[g] = 0.0;
#pragma unroll 1
  for (uint32_t k = first; k < a.items; k += NB * step) {
    // [NB]: the first partial of the group, for its centre
    uint4 t[GR][NB + 1];
#pragma unroll
    for (int g = 0; g < GR; ++g)
#pragma unroll
      for (int i = 0; i <= NB; ++i) {
        // what does not exist is not waited for
        const bool is = (i < NB ? k + i * step < a.items : !BWD) && (g == 0 || two);
        t[g][i] = make_uint4(0u, is ? 0u : 1u, 0u, is ? 0u : 1u);
      }
    while (true) {
      bool there = true;
#pragma unroll
      for (int g = 0; g < GR; ++g)
#pragma unroll
        for (int i = 0; i <= NB; ++i)
          if (!is_part(t[g][i]))
            t[g][i] = look_part(q + g * next + (i < NB ? k + i * step : 0u));
#pragma unroll
      for (int g = 0; g < GR; ++g)
#pragma unroll
        for (int i = 0; i <= NB; ++i) there = there && is_part(t[g][i]);
      if (there) break;
      const unsigned long long now = wall_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > NORM_WAIT_NS) {
        note_timeout(a);
        return false;
      }
    }
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      if constexpr (!BWD) k0[g] = (double)__uint_as_float(t[g][NB].x);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint4& v = t[g][i];
        if (k + i * step < a.items) {
          const double x = (double)__uint_as_float(v.x), r = (double)__uint_as_float(v.z);
          if constexpr (BWD) {
            s[g] += x;
            m[g] += r;
          } else {
            const double n = (double)v.w, d = x - k0[g], nd = n * d;
            s[g] += nd + r;
            m[g] += (double)__uint_as_float(v.y & 0x7FFFFFFFu) + d * (2.0 * r + nd);
          }
        }
      }
    }
  }
  return true;
}

// A group's partial from sums about k0 (forward), n values.
__device__ __forceinline__ void put_moments(float4* p, double k0, double s, double m, double n) {
  const float c = (float)k0 + (float)s * rcp_hw((float)n);
  const double d = (double)c - k0;
  put_part(p, c, (float)(m - d * (2.0 * s - n * d)), (float)(s - n * d), (uint32_t)n);
}

// A group's numbers from its merged partials.  `keep`: for the backward pass.
template <bool BWD>
__device__ __forceinline__ GroupStat group_stat(const NormArgs& a, int64_t at, double s, double m,
                                                double k0, bool keep) {
  float2* st = reinterpret_cast<float2*>(a.stats) + at;
  const double d = s * a.inv_n;
  if constexpr (BWD) {
    const float2 t = *st;
    return {t.x, t.y, t.y * (float)d, t.y * t.y * (float)(m * a.inv_n)};
  } else {
    const float var = (float)fmax(m * a.inv_n - d * d, 0.0) + a.eps;
    const GroupStat r = {(float)(k0 + d), rsqrtf(isnan(m) ? __int_as_float(0x7FC00000) : var),
                         0.0f, 0.0f};
    if (keep) *st = make_float2(r.mean, r.rstd);
    return r;
  }
}

// The numbers of the unit's one group, in every thread; meet: 2 * FEAT_WARPS
// entries that the CTA's previous call did not use.
template <bool BWD>
__device__ __forceinline__ bool norm_merge_one(const NormArgs& a, uint32_t u, bool keep,
                                               double2* meet, GroupStat& r) {
  double v[2], k0;
  bool ok = sum_parts<BWD, 1, 2>(a, a.part + (int64_t)u * a.items, false, 0, threadIdx.x,
                                 FEAT_THREADS, v, v + 1, &k0);
  // a thread without a partial of its own has not seen the centre
  warp_sums<2>(v);
  if (threadIdx.x % 32 == 0) {
    meet[threadIdx.x / 32] = make_double2(v[0], v[1]);
    if (threadIdx.x == 0) meet[FEAT_WARPS].x = k0;
  }
  ok = __syncthreads_and(ok);
  double s = 0.0, m = 0.0;
#pragma unroll
  for (int i = 0; i < FEAT_WARPS; ++i) {
    s += meet[i].x;
    m += meet[i].y;
  }
  r = group_stat<BWD>(a, u, s, m, meet[FEAT_WARPS].x, keep && threadIdx.x == 0);
  return ok;
}

// The numbers of the unit's groups in shared memory, a warp two groups at a
// time; five partials a lane are one from every SM.
template <bool BWD>
__device__ __forceinline__ bool norm_merge(const NormArgs& a, uint32_t u, bool keep,
                                           GroupStat* gs) {
  bool ok = true;
  const int lane = threadIdx.x % 32;
#pragma unroll 1
  for (uint32_t g = threadIdx.x / 32; g < a.ugroups; g += 2 * FEAT_WARPS) {
    const int64_t at = (int64_t)u * a.ugroups + g;
    const bool two = g + FEAT_WARPS < a.ugroups;
    double v[4], k0[2];
    ok = sum_parts<BWD, 2, 5>(a, a.part + at * a.items, two, (int64_t)FEAT_WARPS * a.items, lane,
                              32, v, v + 2, k0) && ok;
    warp_sums<4>(v);
    // lane 0 has the centres
    if (lane == 0) {
      gs[g] = group_stat<BWD>(a, at, v[0], v[2], k0[0], keep);
      if (two) gs[g + FEAT_WARPS] = group_stat<BWD>(a, at + FEAT_WARPS, v[1], v[3], k0[1], keep);
    }
  }
  return __syncthreads_and(ok) != 0;
}

// All CTAs of the unit have written their partials (a warp's lanes may come
// apart: only some of them write).
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// Backward: the item's `chan` is written, and all items' are.
__device__ __forceinline__ void chan_done(const NormArgs& a) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    asm volatile("red.relaxed.gpu.global.add.u32 [%0], 1;" ::"l"(a.done) : "memory");
  }
}
__device__ __forceinline__ bool chan_wait(const NormArgs& a, uint32_t n) {
  int ok = 1;
  if (threadIdx.x == 0) {
    const unsigned long long t0 = wall_ns();
    uint32_t v;
    do {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(a.done) : "memory");
      if (v != n && wall_ns() - t0 > NORM_WAIT_NS) {
        note_timeout(a);
        ok = 0;
      }
    } while (v != n && ok);
  }
  return __syncthreads_and(ok) != 0;
}

// cp.async of BYTES (8, 16).
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t smem, const void* gmem) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem), "l"(gmem) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(smem), "l"(gmem), "n"(BYTES)
                 : "memory");
}

// ===========================================================================
// A thread's accesses, eight to a block, each thread's own ring of eight slots
// in shared memory: while a block is worked on, the next one is on its way
// (cp.async, no registers held).  Single elements are loaded into registers, a
// block at a time, instead.  What an access costs beside its arithmetic is
// what bounds these kernels after HBM, so the addresses are a pointer to the
// block plus j times a stride, and a block has one count of the accesses that
// exist (negative or more than eight like none and eight).
// ===========================================================================
template <int DT, int VEC, bool BWD>
struct Stream {
  static constexpr int BYTES = VEC * ESIZE<DT>;
  static constexpr int SLOT = FEAT_THREADS * BYTES;
  const char *x, *dy;  // the block after the current one
  char* slot;          // the thread's slot 0
  uint32_t step;       // bytes between the accesses of a block
  int64_t span;        // bytes between blocks, negative if backwards
  int left, dec;       // the current block's count, what the next one has less
  int blocks;          // of the thread
  Raw<DT, 1> rx[VEC == 1 ? 8 : 1], rd[VEC == 1 && BWD ? 8 : 1];

  // To the last block, and from there backwards.
  __device__ __forceinline__ void turn() {
    const int n = blocks - 1;
    if (n > 0) {
      x += n * span;
      dy += n * span;
      left -= n * dec;
    }
    span = -span;
    dec = -dec;
  }

  // accesses j and j + 1 of the next block, `count` of which exist
  __device__ __forceinline__ void issue2(int count, int j) {
    if constexpr (VEC > 1) {
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot) + j * SLOT;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (j + h < count) {
          cp_async<BYTES>(to + h * SLOT, x + (uint64_t)(j + h) * step);
          if constexpr (BWD) cp_async<BYTES>(to + (8 + h) * SLOT, dy + (uint64_t)(j + h) * step);
        }
      cp_async_commit();
    }
  }
  // the first block
  __device__ __forceinline__ void start() {
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) issue2(left, j);
      x += span;
      dy += span;
    }
  }
  // after the current block comes the first one of `o`, of this many accesses
  __device__ __forceinline__ int follow(const Stream& o) {
    if constexpr (VEC > 1) {
      x = o.x;
      dy = o.dy;
    }
    return o.left;
  }
  // what the accesses lack that do not exist: zeros (a block ahead, like them)
  __device__ __forceinline__ void zero(int count) {
    if constexpr (VEC > 1) {
      if (count < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j >= count) {
            *reinterpret_cast<Raw<DT, VEC>*>(slot + j * SLOT) = {};
            if constexpr (BWD) *reinterpret_cast<Raw<DT, VEC>*>(slot + (8 + j) * SLOT) = {};
          }
      }
    }
  }
  // single elements: the whole current block
  __device__ __forceinline__ void fill() {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rx[j] = 0;
        if constexpr (BWD) rd[j] = 0;
        if (j < left) {
          rx[j] = raw_load<DT, 1>(x + (uint64_t)j * step);
          if constexpr (BWD) rd[j] = raw_load<DT, 1>(dy + (uint64_t)j * step);
        }
      }
    }
  }
  // the current block is done with
  __device__ __forceinline__ void next() {
    x += span;
    dy += span;
    left -= dec;
  }
  // accesses j and j + 1 of the block have arrived (those after them not)
  __device__ __forceinline__ void wait2() {
    if constexpr (VEC > 1) cp_async_wait<3>();
  }
  __device__ __forceinline__ Raw<DT, VEC> get_x(int j) const {
    return *reinterpret_cast<const Raw<DT, VEC>*>(slot + j * SLOT);
  }
  __device__ __forceinline__ Raw<DT, VEC> get_dy(int j) const {
    return *reinterpret_cast<const Raw<DT, VEC>*>(slot + (8 + j) * SLOT);
  }
};

// Bytes of a CTA's rings.
template <int DT, int VEC, bool BWD>
constexpr int RING_BYTES = VEC == 1 ? 0 : FEAT_THREADS * VEC * ESIZE<DT> * 8 * (BWD ? 2 : 1);

// Single elements: accesses j .. j + 3 of the block, as two pairs.
template <int DT, int ACT, bool BWD>
__device__ __forceinline__ void single_add(const Stream<DT, 1, BWD>& st, int j,
                                           const RawPair<DT>* d, const PairConst& k, float slope,
                                           F2& s0, F2& s1) {
  F2 p0 = f2(0.0f), q0 = p0, p1 = p0, q1 = p0;
  norm_add<DT, ACT, BWD>(raw_join<DT>(st.rx[j], st.rx[j + 1]),
                         raw_join<DT>(st.rx[j + 2], st.rx[j + 3]), d[0], d[1], k, k, slope, p0, q0,
                         p1, q1);
  // what does not exist adds nothing
  const bool h0 = j < st.left, h1 = j + 1 < st.left, h2 = j + 2 < st.left, h3 = j + 3 < st.left;
  s0 = add2(s0, f2(h0 ? p0.x() : 0.0f, h1 ? p0.y() : 0.0f));
  s1 = add2(s1, f2(h0 ? q0.x() : 0.0f, h1 ? q0.y() : 0.0f));
  s0 = add2(s0, f2(h2 ? p1.x() : 0.0f, h3 ? p1.y() : 0.0f));
  s1 = add2(s1, f2(h2 ? q1.x() : 0.0f, h3 ? q1.y() : 0.0f));
}
template <int DT>
__device__ __forceinline__ void single_store(char* out, uint32_t step, int j, int left,
                                             RawPair<DT> y0, RawPair<DT> y1) {
#pragma unroll
  for (int h = 0; h < 4; ++h)
    if (j + h < left)
      raw_store<DT, 1>(out + (uint64_t)(j + h) * step, raw_half<DT>(h < 2 ? y0 : y1, h & 1));
}

// ===========================================================================
// Channels last
// ===========================================================================
// Weight and bias of a pass's channel threadIdx.x, ahead of their use.
struct ChanParam {
  float w, bias;
};
__device__ __forceinline__ ChanParam chan_param(const NormArgs& a, int64_t c, int64_t end) {
  if (c >= end) return {0.0f, 0.0f};
  return {norm_param(a.weight, a.w_bf16, c, 1.0f), norm_param(a.bias, a.w_bf16, c, 0.0f)};
}

// The constants of a pass's channels in shared memory: plane by plane
// (mean, a, bias, c2, c3, as PairConst has them), a thread's pair i at
// (i * ncw + tx), so that neighbouring threads read neighbouring words.
// sm: 5 * ncw * VEC floats; wt (backward sums): the weights, ncw * VEC.
template <int VEC, bool COEF>
__device__ __forceinline__ void last_consts(const NormArgs& a, const LastPlace& p, uint32_t g0,
                                            const GroupStat* gs, ChanParam own, float* sm,
                                            float* wt) {
  constexpr int P = VEC > 1 ? 2 : 1;
  const int cw = a.f.ncw * VEC;
  const int64_t c0 = p.c - p.tx * VEC;
  for (int i = threadIdx.x; i < cw; i += FEAT_THREADS) {
    if (c0 + i < p.c_end) {
      const uint32_t g = (uint32_t)(c0 + i) / a.Cg - g0;
      const ChanParam cp = i < FEAT_THREADS ? own : chan_param(a, c0 + i, p.c_end);
      const PairConst q = pair_const(gs[g], cp.w, cp.bias);
      float* to = sm + ((i % VEC / P) * a.f.ncw + i / VEC) * P + i % P;
      to[0] = q.nmean.x();
      to[cw] = q.a.x();
      to[2 * cw] = q.bias.x();
      if constexpr (COEF) {
        to[3 * cw] = q.nc2.x();
        to[4 * cw] = q.nc3.x();
      } else {
        wt[i] = cp.w;
      }
    }
  }
  __syncthreads();
}

template <int VEC, bool COEF>
__device__ __forceinline__ PairConst last_const(const NormArgs& a, const LastPlace& p, int i,
                                                const float* sm) {
  const int cw = a.f.ncw * VEC;
  PairConst k = {};
  auto get = [&](int plane) {
    if constexpr (VEC > 1) {
      const float2 v = reinterpret_cast<const float2*>(sm + plane * cw)[i * a.f.ncw + p.tx];
      return f2(v.x, v.y);
    } else {
      return f2(sm[plane * cw + p.tx]);
    }
  };
  k.nmean = get(0);
  k.a = get(1);
  k.bias = get(2);
  if constexpr (COEF) {
    k.nc2 = get(3);
    k.nc3 = get(4);
  }
  return k;
}

template <int DT, int VEC, bool BWD, bool BLOCK>
__device__ __forceinline__ Stream<DT, VEC, BWD> last_stream(const NormArgs& a, const LastPlace& p,
                                                            char* ring) {
  Stream<DT, VEC, BWD> s;
  const uint32_t row = (uint32_t)a.f.C * ESIZE<DT>;
  const int first = BLOCK ? p.ty * 8 : p.ty, span = p.nty * 8;
  const int64_t base = last_base<DT>(a.f, p) + (int64_t)row_at(first, row);
  s.x = (const char*)a.x + base;
  s.dy = (const char*)a.dy + base;
  s.slot = ring + threadIdx.x * VEC * ESIZE<DT>;
  s.step = (BLOCK ? 1 : p.nty) * row;
  s.span = (int64_t)row_at(span, row);
  // rows that are left, or every nty-th of them
  s.dec = BLOCK ? span : 8;
  s.left = BLOCK ? p.rows - first : (p.rows - first + p.nty - 1) / p.nty;
  if (!p.on) s.left = 0;
  s.blocks = s.left > 0 ? (s.left + s.dec - 1) / s.dec : 0;
  return s;
}

// The sums of a pass (256 columns at most) of one item, added to the item's
// groups; the pass's first block is on its way, `first` is its address.
// sm: two planes of nty rows by cw channels, floats (2 * FEAT_THREADS * VEC in
// all), or the constants; meet: max(FEAT_THREADS, cw) entries; acc: the
// groups' sums so far and their centres.
template <int DT, int VEC, int ACT, int DROP, bool BWD>
__device__ __forceinline__ void last_sums(const NormArgs& a, const LastPlace& p,
                                          Stream<DT, VEC, BWD>& st, const char* first, uint32_t g0,
                                          const GroupStat* gs, ChanParam own, float* sm, float* wt,
                                          double2* meet, double2* acc) {
  constexpr bool BLOCK = BWD && DROP != DROP_NONE;
  constexpr int NP = VEC > 1 ? VEC / 2 : 1;  // pairs of channels, or of rows
  if constexpr (BWD) st.zero(st.left);
  F2 s0[NP], s1[NP], m2[NP];
  PairConst k[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) s0[i] = s1[i] = m2[i] = f2(0.0f);
  DropRate dr = {};
  if constexpr (BWD) {
    if constexpr (DROP) dr = drop_rate(a.drop, p.b);
    last_consts<VEC, false>(a, p, g0, gs, own, sm, wt);
#pragma unroll
    for (int i = 0; i < NP; ++i) k[i] = last_const<VEC, false>(a, p, i, sm);
  } else {
    // the thread's first row is its first centre
#pragma unroll
    for (int i = 0; i < NP; ++i) k[i] = {};
    if (st.left > 0) {
      const Raw<DT, VEC> v = raw_load<DT, VEC>(first);
      if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const F2 t = pair_value<DT>(raw_pair<DT, VEC>(v, i));
          k[i].nmean = f2(-t.x(), -t.y());
        }
      } else {
        const F2 t = pair_value<DT>(raw_join<DT>(v, v));
        k[0].nmean = f2(-t.x(), -t.y());
      }
    }
  }
#pragma unroll 1
  for (int q = 0; q < st.blocks; ++q, st.next()) {
    const int more = q + 1 < st.blocks ? st.left - st.dec : 0;
    uint32_t keep[VEC];
    if constexpr (BLOCK) last_keep<VEC, DROP>(a.f, a.drop, dr, p, q * p.nty * 8 + p.ty * 8, keep);
    st.fill();
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j % 2 == 0) st.wait2();
        const Raw<DT, VEC> vx = st.get_x(j);
        Raw<DT, VEC> vd = {};
        if constexpr (BWD) vd = st.get_dy(j);
        // missing rows: a zero dy adds nothing; a zero x would
        if (BWD || j < st.left) {
#pragma unroll
          for (int i = 0; i < NP; i += 2) {
            RawPair<DT> d0 = raw_pair<DT, VEC>(vd, i), d1 = raw_pair<DT, VEC>(vd, i + 1);
            if constexpr (BLOCK) {
              d0 = last_pair_keep<DT>(d0, keep, i, j);
              d1 = last_pair_keep<DT>(d1, keep, i + 1, j);
            }
            norm_add<DT, ACT, BWD>(raw_pair<DT, VEC>(vx, i), raw_pair<DT, VEC>(vx, i + 1), d0, d1,
                                   k[i], k[i + 1], a.slope, s0[i], s1[i], s0[i + 1], s1[i + 1]);
          }
        }
        if (j % 2 == 1) st.issue2(more, j - 1);
      }
      if constexpr (BWD) st.zero(more);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        RawPair<DT> d[2] = {};
        if constexpr (BWD) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            d[h] = raw_join<DT>(st.rd[j + 2 * h], st.rd[j + 2 * h + 1]);
            const uint32_t w = BLOCK ? keep[0] << ((j >> 1) + h) : 0u;
            if constexpr (BLOCK) d[h] = pair_keep<DT, 1, 3>(d[h], w, w);
          }
        }
        single_add<DT, ACT, BWD>(st, j, d, k[0], a.slope, s0[0], s1[0]);
      }
    }
    if constexpr (!BWD) {
      if (q + 1 < st.blocks && recentres(q)) {
        const float n = (float)(8 * q + 8);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if constexpr (VEC > 1)
            recentre(k[i].nmean, s0[i], s1[i], m2[i], n);
          else
            recentre_one(k[i].nmean, s0[i], s1[i], m2[i], n);
        }
      }
    }
  }
  // threads -> channels
  const int cw = a.f.ncw * VEC, rows = p.rows;
  float* plane = sm + p.nty * cw;
  // forward: thread row y has n0 rows of the item, one more below y1
  const int n0 = rows / p.nty, y1 = rows - n0 * p.nty;
  const float inv = 1.0f / (float)(n0 + (p.ty < y1 ? 1 : 0));
  __syncthreads();
  if (p.ty < p.nty) {
    float us[VEC], ws[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int h = VEC > 1 ? i / 2 : 0;
      const float t = VEC == 1 ? s0[0].x() + s0[0].y() : i & 1 ? s0[h].y() : s0[h].x();
      float u = t, w = VEC == 1 ? s1[0].x() + s1[0].y() : i & 1 ? s1[h].y() : s1[h].x();
      if constexpr (!BWD) {
        // a thread's (mean, M2); nothing when it had no row
        const float m = t * inv;
        u = m - (i & 1 ? k[h].nmean.y() : k[h].nmean.x());
        w = __fmaf_rn(-t, m, w + (i & 1 ? m2[h].y() : m2[h].x()));
      }
      us[i] = u;
      ws[i] = w;
    }
    const int at = p.ty * cw + p.tx * VEC;
    if constexpr (VEC > 1) {  // wide, or eight lanes meet in a bank
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        *reinterpret_cast<float4*>(sm + at + i) = make_float4(us[i], us[i + 1], us[i + 2], us[i + 3]);
        *reinterpret_cast<float4*>(plane + at + i) =
            make_float4(ws[i], ws[i + 1], ws[i + 2], ws[i + 3]);
      }
    } else {
      sm[at] = us[0];
      plane[at] = ws[0];
    }
  }
  __syncthreads();
  // rows -> channel parts, about the mean of the part's first row (VEC rows at
  // most, so in fp32: a conversion costs as much as four additions), and from
  // there about that of the group's first channel's first row, in double; then,
  // a warp a group, -> groups, in double
  const int parts = cw >= FEAT_THREADS ? 1 : FEAT_THREADS / cw;
  const int64_t c0 = p.c - p.tx * VEC;
  const int nch = (int)min((int64_t)cw, p.c_end - c0);  // channels of the pass
  const uint32_t ga = (uint32_t)c0 / a.Cg, gb = (uint32_t)(c0 + nch - 1) / a.Cg;
  const float rows0 = (float)n0, rows1 = (float)(n0 + 1);
#pragma unroll 1
  for (int cb = 0; cb < cw; cb += FEAT_THREADS) {
    const int part = parts == 1 ? 0 : (int)threadIdx.x / cw;
    const int ci = cb + (int)threadIdx.x - part * cw;
    if (part >= parts || ci >= nch) continue;
    float u = 0.0f, w = 0.0f, k0 = 0.0f, kp = 0.0f, n = 0.0f;
    const uint32_t g = (uint32_t)(c0 + ci) / a.Cg;
    // about the first channel of the group, which an earlier pass may have had
    if constexpr (!BWD) {
      k0 = g * a.Cg >= (uint32_t)c0 ? sm[g * a.Cg - (uint32_t)c0] : (float)acc[2 * (g - g0) + 1].x;
      kp = part < rows ? sm[part * cw + ci] : k0;
    }
#pragma unroll 4
    for (int y = part; y < p.nty && (BWD || y < rows); y += parts) {
      const float q = sm[y * cw + ci], r = plane[y * cw + ci];
      if constexpr (BWD) {
        u += q;
        w += r;
      } else {
        const float ny = y < y1 ? rows1 : rows0, d = q - kp, nd = ny * d;
        n += ny;
        u += nd;
        w += __fmaf_rn(nd, d, r);
      }
    }
    double2 t = make_double2((double)u, (double)w);
    if constexpr (!BWD) {
      const double d = (double)kp - (double)k0, nd = (double)n * d;
      t.y += d * (2.0 * t.x + nd);
      t.x += nd;
    }
    if constexpr (BWD) {
      const double sc = DROP ? (double)dr.scale : 1.0;
      t.x *= sc;
      t.y *= sc * (double)gs[g - g0].rstd;
    }
    meet[part * cw + ci] = t;
  }
  __syncthreads();
  // a group is always the same warp's, so its sums are too
#pragma unroll 1
  for (uint32_t g = threadIdx.x / 32 + g0; g <= gb; g += 2 * FEAT_WARPS) {
    double v[4] = {0.0, 0.0, 0.0, 0.0};  // two groups' sums, then their second ones
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t gh = g + h * FEAT_WARPS;
      if (gh < ga || gh > gb) continue;
      const int i0 = gh > ga ? (int)(gh * a.Cg - (uint32_t)c0) : 0;
      const int ng = (int)min((int64_t)nch, (int64_t)(gh + 1) * a.Cg - c0) - i0;
      for (int e = threadIdx.x % 32; e < ng * parts; e += 32) {
        const int part = e / ng, i = i0 + e - part * ng;
        const double2 t = meet[part * cw + i];
        const double f = BWD ? (double)wt[i] : 1.0;
        v[h] += f * t.x;
        v[2 + h] += f * t.y;
      }
    }
    warp_sums<4>(v);
    if (threadIdx.x % 32 == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t gh = g + h * FEAT_WARPS;
        if (gh < ga || gh > gb) continue;
        double2* t = acc + 2 * (gh - g0);
        if (gh * a.Cg >= (uint32_t)c0) {
          t[0] = make_double2(v[h], v[2 + h]);
          t[1] = make_double2(BWD ? 0.0 : (double)sm[gh * a.Cg - (uint32_t)c0], 0.0);
        } else {
          t[0].x += v[h];
          t[0].y += v[2 + h];
        }
      }
    }
  }
  if constexpr (BWD) {
    if (a.chan != nullptr)
      for (int ci = threadIdx.x; ci < nch; ci += FEAT_THREADS) {
        double2 t = meet[ci];
        for (int j = 1; j < parts; ++j) {
          t.x += meet[j * cw + ci].x;
          t.y += meet[j * cw + ci].y;
        }
        __stcg(a.chan + (p.b * a.f.nchunk + p.k) * a.f.C + c0 + ci,
               make_float2((float)t.x, (float)t.y));
      }
  }
}

// The item's partials, from the lanes that summed its groups.
template <bool BWD>
__device__ __forceinline__ void last_put(const NormArgs& a, const LastPlace& p, float4* part,
                                         const double2* acc) {
  if (threadIdx.x % 32 != 0) return;
  for (uint32_t g = threadIdx.x / 32; g < a.ugroups; g += FEAT_WARPS) {
    const double2 t = acc[2 * g];
    if constexpr (BWD)
      put_part(part + (int64_t)g * a.items, (float)t.x, 0.0f, (float)t.y, 1u);
    else
      put_moments(part + (int64_t)g * a.items, acc[2 * g + 1].x, t.x, t.y,
                  (double)p.rows * (double)a.Cg);
  }
}

// y or dx of a pass of one item; the pass's first block is on its way.
template <int DT, int VEC, int ACT, int DROP, bool BWD>
__device__ __forceinline__ void last_apply(const NormArgs& a, const LastPlace& p,
                                           Stream<DT, VEC, BWD>& st, uint32_t g0,
                                           const GroupStat* gs, ChanParam own, const DropRate& dr,
                                           float* sm, float* wt) {
  constexpr int NP = VEC > 1 ? VEC / 2 : 1;
  last_consts<VEC, BWD>(a, p, g0, gs, own, sm, wt);
  if (!p.on) return;
  const float scale = DROP ? dr.scale : 1.0f;
  PairConst k[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) k[i] = last_const<VEC, BWD>(a, p, i, sm);
  // the result lies as x does; single elements are not a block ahead
  char* out = (char*)a.out + (st.x - (const char*)a.x) - (VEC > 1 ? st.span : 0);
#pragma unroll 1
  for (int q = 0; q < st.blocks; ++q, st.next(), out += st.span) {
    const int more = q + 1 < st.blocks ? st.left - st.dec : 0;
    uint32_t keep[VEC];
    if constexpr (DROP)
      last_keep<VEC, DROP>(a.f, a.drop, dr, p, (a.reverse ? st.blocks - 1 - q : q) * p.nty * 8 + p.ty * 8, keep);
    st.fill();
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j % 2 == 0) st.wait2();
        Raw<DT, VEC> vx = st.get_x(j), vd = {};
        if constexpr (BWD) vd = st.get_dy(j);
#pragma unroll
        for (int i = 0; i < NP; i += 2) {
          RawPair<DT> y0 = raw_pair<DT, VEC>(vx, i), y1 = raw_pair<DT, VEC>(vx, i + 1);
          RawPair<DT> d0 = raw_pair<DT, VEC>(vd, i), d1 = raw_pair<DT, VEC>(vd, i + 1);
          if constexpr (BWD && DROP) {
            d0 = last_pair_keep<DT>(d0, keep, i, j);
            d1 = last_pair_keep<DT>(d1, keep, i + 1, j);
          }
          norm_pairs<DT, ACT, DROP, BWD>(y0, y1, d0, d1, k[i], k[i + 1], a.slope, scale);
          if constexpr (DROP && !BWD) {
            y0 = last_pair_keep<DT>(y0, keep, i, j);
            y1 = last_pair_keep<DT>(y1, keep, i + 1, j);
          }
          raw_set_pair<DT, VEC>(vx, i, y0);
          raw_set_pair<DT, VEC>(vx, i + 1, y1);
        }
        if (j < st.left) raw_store<DT, VEC>(out + (uint64_t)j * st.step, vx);
        if (j % 2 == 1) st.issue2(more, j - 1);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        RawPair<DT> d[2] = {};
        const uint32_t w[2] = {DROP ? keep[0] << (j >> 1) : 0u, DROP ? keep[0] << ((j >> 1) + 1) : 0u};
        if constexpr (BWD) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            d[h] = raw_join<DT>(st.rd[j + 2 * h], st.rd[j + 2 * h + 1]);
            if constexpr (DROP) d[h] = pair_keep<DT, 1, 3>(d[h], w[h], w[h]);
          }
        }
        RawPair<DT> y0 = raw_join<DT>(st.rx[j], st.rx[j + 1]);
        RawPair<DT> y1 = raw_join<DT>(st.rx[j + 2], st.rx[j + 3]);
        norm_pairs<DT, ACT, DROP, BWD>(y0, y1, d[0], d[1], k[0], k[0], a.slope, scale);
        if constexpr (DROP && !BWD) {
          y0 = pair_keep<DT, 1, 3>(y0, w[0], w[0]);
          y1 = pair_keep<DT, 1, 3>(y1, w[1], w[1]);
        }
        single_store<DT>(out, st.step, j, st.left, y0, y1);
      }
    }
  }
}

// ===========================================================================
// Channels first.  Item i of a group: 8 of its runs (channel, f.rows voxels),
// one for each warp.  An access is 32 * VEC voxels of a warp.
// ===========================================================================
// A piece of a unit's results: piece j of item k, the ends first if reversed.
struct Piece {
  uint32_t k, j;
  __device__ __forceinline__ bool is() const { return k != 0xFFFFFFFFu; }
};
__device__ __forceinline__ Piece piece_of(const NormArgs& a, uint32_t m) {
  const uint32_t j = m / a.items;
  return {j < a.subs ? m - j * a.items : 0xFFFFFFFFu, a.reverse ? a.subs - 1 - j : j};
}

// The next piece of unit u: asked for by thread 0 while the CTA works on one,
// and read by all after the barrier behind it.
struct Tickets {
  Piece* slot;  // two in shared memory
  uint32_t par;
  __device__ __forceinline__ Piece take(const NormArgs& a, uint32_t u) const {
    return piece_of(a, a.items + atomicAdd(a.ticket + u, 1u));
  }
};

// The warp's voxels r .. r + n of its run.
__device__ __forceinline__ void first_item(const NormArgs& a, uint32_t u, uint32_t i, int64_t r,
                                           int64_t n, FirstPlace& p) {
  const uint32_t run = i * FEAT_WARPS + threadIdx.x / 32;
  const uint32_t cl = run / a.f.nchunk, k = run - cl * a.f.nchunk, b = u / a.G;
  p.lane = threadIdx.x % 32;
  p.b = b;
  p.k = k;
  p.c = (u - b * a.G) * a.Cg + cl;
  p.s0 = k * a.f.rows + r;
  p.n = cl < a.Cg ? (int)max((int64_t)0, min(min(n, a.f.rows - r), a.f.S - p.s0)) : 0;
  p.base = (p.b * a.f.C + p.c) * a.f.S + p.s0;
}
__device__ __forceinline__ void first_piece(const NormArgs& a, uint32_t u, Piece m,
                                            FirstPlace& p) {
  first_item(a, u, m.k, (int64_t)m.j * a.sub_rows, a.sub_rows, p);
}

template <int DT, int VEC, bool BWD>
__device__ __forceinline__ void first_count(const FirstPlace& p, Stream<DT, VEC, BWD>& s) {
  constexpr int every = 32 * VEC;
  s.left = (p.n - first_at<VEC>(p.lane, 0) + every - 1) / every;  // towards zero: none below it
  s.dec = 8;
  s.blocks = (p.n + 8 * every - 1) / (8 * every);  // of the warp
}
template <int DT, int VEC, bool BWD>
__device__ __forceinline__ Stream<DT, VEC, BWD> first_stream(const NormArgs& a,
                                                             const FirstPlace& p, char* ring) {
  Stream<DT, VEC, BWD> s;
  constexpr int every = 32 * VEC;  // voxels of a warp's access
  const int64_t base = (p.base + first_at<VEC>(p.lane, 0)) * ESIZE<DT>;
  s.x = (const char*)a.x + base;
  s.dy = (const char*)a.dy + base;
  s.slot = ring + threadIdx.x * VEC * ESIZE<DT>;
  s.step = every * ESIZE<DT>;
  s.span = 8 * every * ESIZE<DT>;
  first_count(p, s);
  return s;
}

// Keep words of accesses j and j + 1 of a block (k: 8 / VEC words a tile; two
// tiles for VEC 8, one for VEC 4; a single element's tile is a block).
template <int VEC, int DROP>
__device__ __forceinline__ void first_block_keep(const NormArgs& a, const DropRate& dr,
                                                 const FirstPlace& p, int s, uint32_t* k) {
  first_keep<VEC, DROP>(a.f, a.drop, dr, p, s, k);
  if constexpr (VEC == 8) first_keep<VEC, DROP>(a.f, a.drop, dr, p, s + FEAT_TILE, k + 1);
}

// The partial of one item.  meet: 2 * FEAT_WARPS entries that the CTA's
// previous call did not use.
template <int DT, int VEC, int ACT, int DROP, bool BWD>
__device__ __forceinline__ void first_sums(const NormArgs& a, uint32_t u_, const FirstPlace& p,
                                           char* ring, double2* meet, float4* part) {
  Stream<DT, VEC, BWD> st = first_stream<DT, VEC, BWD>(a, p, ring);
  const char* first = st.x;
  const int cnt = max(st.left, 0) * VEC;  // the lane's voxels
  st.start();
  if constexpr (BWD) st.zero(st.left);
  F2 s0 = f2(0.0f), s1 = f2(0.0f), u0 = f2(0.0f), u1 = f2(0.0f), m2 = f2(0.0f);
  float weight = 0.0f, rstd = 0.0f;
  PairConst k = {};
  DropRate dr = {};
  if constexpr (BWD) {
    const float2 t = reinterpret_cast<const float2*>(a.stats)[u_];
    const ChanParam cp = chan_param(a, p.c, p.n > 0 ? a.f.C : 0);
    k = pair_const({t.x, t.y, 0.0f, 0.0f}, cp.w, cp.bias);
    weight = cp.w;
    rstd = t.y;
    if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  } else {
    if (cnt > 0) {
      if constexpr (VEC > 1) {  // the mean of the first access: exact for equal values
        const Raw<DT, VEC> v = raw_load<DT, VEC>(first);
        F2 t = add2(pair_value<DT>(raw_pair<DT, VEC>(v, 0)), pair_value<DT>(raw_pair<DT, VEC>(v, 1)));
        if constexpr (VEC == 8)
          t = add2(t, add2(pair_value<DT>(raw_pair<DT, VEC>(v, 2)),
                           pair_value<DT>(raw_pair<DT, VEC>(v, 3))));
        k.nmean = f2((t.x() + t.y()) * (-1.0f / VEC));
      } else {
        k.nmean = f2(-load_f(first, DT, 0));
      }
    } else {
      k.nmean = f2(0.0f);
    }
  }
#pragma unroll 1
  for (int q = 0; q < st.blocks; ++q, st.next()) {
    const int more = q + 1 < st.blocks ? st.left - st.dec : 0;
    st.fill();
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        uint32_t keep[2];
        if constexpr (BWD && DROP)
          first_block_keep<VEC, DROP>(a, dr, p, (q * 8 + j) * 32 * VEC, keep);
        st.wait2();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Raw<DT, VEC> vx = st.get_x(j + h);
          Raw<DT, VEC> vd = {};
          if constexpr (BWD) vd = st.get_dy(j + h);
          if (BWD || j + h < st.left) {
#pragma unroll
            for (int i = 0; i < VEC / 2; i += 2) {
              RawPair<DT> d0 = raw_pair<DT, VEC>(vd, i), d1 = raw_pair<DT, VEC>(vd, i + 1);
              if constexpr (BWD && DROP) {
                d0 = pair_keep<DT, 1, 3>(d0, keep[h] << i, keep[h] << i);
                d1 = pair_keep<DT, 1, 3>(d1, keep[h] << (i + 1), keep[h] << (i + 1));
              }
              norm_add<DT, ACT, BWD>(raw_pair<DT, VEC>(vx, i), raw_pair<DT, VEC>(vx, i + 1), d0,
                                     d1, k, k, a.slope, s0, s1, u0, u1);
            }
          }
        }
        st.issue2(more, j);
      }
      if constexpr (BWD) st.zero(more);
    } else {
      uint32_t keep[8];
      if constexpr (BWD && DROP) first_keep<VEC, DROP>(a.f, a.drop, dr, p, q * 8 * 32 * VEC, keep);
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        RawPair<DT> d[2] = {};
        if constexpr (BWD) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            d[h] = raw_join<DT>(st.rd[j + 2 * h], st.rd[j + 2 * h + 1]);
            if constexpr (DROP)
              d[h] = pair_keep<DT, 3, 3>(d[h], keep[j + 2 * h], keep[j + 2 * h + 1]);
          }
        }
        single_add<DT, ACT, BWD>(st, j, d, k, a.slope, s0, s1);
      }
    }
    if constexpr (!BWD) {
      // a block that another follows is whole in every lane
      if (q + 1 < st.blocks && recentres(q)) {
        s0 = add2(s0, u0);
        s1 = add2(s1, u1);
        u0 = u1 = f2(0.0f);
        recentre_one(k.nmean, s0, s1, m2, (float)((q + 1) * 8 * VEC));
      }
    }
  }
  s0 = add2(s0, u0);
  s1 = add2(s1, u1);
  // lanes -> run -> item, in double; forward, a lane's moments about the first
  // lane's centre, a run's about the first run's
  double u, w, k0 = 0.0;
  if constexpr (BWD) {
    const double sc = DROP ? (double)dr.scale : 1.0;
    u = warp_sum((double)s0.x() + (double)s0.y()) * sc;
    w = warp_sum((double)s1.x() + (double)s1.y()) * sc * (double)rstd;
    if (p.lane == 0 && p.n > 0 && a.chan != nullptr)
      __stcg(a.chan + (p.b * a.f.C + p.c) * a.f.nchunk + p.k, make_float2((float)u, (float)w));
    u *= (double)weight;
    w *= (double)weight;
  } else {
    const float centre = -k.nmean.x();
    k0 = (double)__shfl_sync(0xFFFFFFFFu, centre, 0);
    const double t0 = (double)s0.x() + (double)s0.y();
    const double t1 = (double)s1.x() + (double)s1.y() + (double)m2.x();
    const double d = (double)centre - k0, nd = (double)cnt * d;
    u = warp_sum(cnt > 0 ? t0 + nd : 0.0);
    w = warp_sum(cnt > 0 ? t1 + d * (2.0 * t0 + nd) : 0.0);
  }
  const int warp = threadIdx.x / 32;
  if (p.lane == 0) {
    meet[warp] = make_double2(u, w);
    meet[FEAT_WARPS + warp] = make_double2(k0, (double)p.n);
  }
  __syncthreads();
  if (warp == 0) {
    double n = 0.0;
    u = w = 0.0;
    if (p.lane < FEAT_WARPS) {
      const double2 t = meet[p.lane], e = meet[FEAT_WARPS + p.lane];
      const double d = e.x - k0;
      n = e.y;
      u = t.x + n * d;
      w = t.y + d * (2.0 * t.x + n * d);
      if (n == 0.0) u = w = 0.0;
    }
#pragma unroll
    for (int o = FEAT_WARPS / 2; o > 0; o >>= 1) {
      u += __shfl_down_sync(0xFFFFFFFFu, u, o);
      w += __shfl_down_sync(0xFFFFFFFFu, w, o);
      n += __shfl_down_sync(0xFFFFFFFFu, n, o);
    }
    if (p.lane == 0) {
      if constexpr (BWD)
        put_part(part, (float)u, 0.0f, (float)w, 1u);
      else
        put_moments(part, k0, u, w, n);
    }
  }
}

// y or dx of a piece whose first block is on its way, and of those that the CTA
// draws.  A channel's constants go with the piece.
template <int DT, int VEC, int ACT, int DROP, bool BWD>
__device__ __forceinline__ void first_apply(const NormArgs& a, FirstPlace p,
                                            Stream<DT, VEC, BWD>& st, uint32_t u, Tickets tk,
                                            const GroupStat& gs, ChanParam cp, const DropRate& dr,
                                            char* ring) {
  const float scale = DROP ? dr.scale : 1.0f;
  while (true) {
    Piece next = {0xFFFFFFFFu, 0u}, after = next;
    if (a.subs > 1) next = tk.slot[tk.par];
    if (threadIdx.x == 0 && next.is()) after = tk.take(a, u);
    const PairConst k = pair_const(gs, cp.w, cp.bias);
    char* out = (char*)a.out + (st.x - (const char*)a.x) - (VEC > 1 ? st.span : 0);
#pragma unroll 1
    for (int q = 0; q < st.blocks; ++q, st.next(), out += st.span) {
      int more = st.left - st.dec;
      if (q + 1 == st.blocks) {
        more = 0;
        if (next.is()) {
          FirstPlace pn;
          first_piece(a, u, next, pn);
          more = st.follow(first_stream<DT, VEC, BWD>(a, pn, ring));
        }
      }
      const int s = q * 8 * 32 * VEC;
      st.fill();
      if constexpr (VEC > 1) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          uint32_t keep[2];
          if constexpr (DROP) first_block_keep<VEC, DROP>(a, dr, p, s + j * 32 * VEC, keep);
          st.wait2();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            Raw<DT, VEC> vx = st.get_x(j + h), vd = {};
            if constexpr (BWD) vd = st.get_dy(j + h);
#pragma unroll
            for (int i = 0; i < VEC / 2; i += 2) {
              RawPair<DT> y0 = raw_pair<DT, VEC>(vx, i), y1 = raw_pair<DT, VEC>(vx, i + 1);
              RawPair<DT> d0 = raw_pair<DT, VEC>(vd, i), d1 = raw_pair<DT, VEC>(vd, i + 1);
              const uint32_t w0 = DROP ? keep[h] << i : 0u, w1 = DROP ? keep[h] << (i + 1) : 0u;
              if constexpr (BWD && DROP) {
                d0 = pair_keep<DT, 1, 3>(d0, w0, w0);
                d1 = pair_keep<DT, 1, 3>(d1, w1, w1);
              }
              norm_pairs<DT, ACT, DROP, BWD>(y0, y1, d0, d1, k, k, a.slope, scale);
              if constexpr (DROP && !BWD) {
                y0 = pair_keep<DT, 1, 3>(y0, w0, w0);
                y1 = pair_keep<DT, 1, 3>(y1, w1, w1);
              }
              raw_set_pair<DT, VEC>(vx, i, y0);
              raw_set_pair<DT, VEC>(vx, i + 1, y1);
            }
            if (j + h < st.left) raw_store<DT, VEC>(out + (j + h) * 32 * VEC * ESIZE<DT>, vx);
          }
          st.issue2(more, j);
        }
      } else {
        uint32_t keep[8];
        if constexpr (DROP) first_keep<VEC, DROP>(a.f, a.drop, dr, p, s, keep);
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          RawPair<DT> d[2] = {};
          if constexpr (BWD) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              d[h] = raw_join<DT>(st.rd[j + 2 * h], st.rd[j + 2 * h + 1]);
              if constexpr (DROP)
                d[h] = pair_keep<DT, 3, 3>(d[h], keep[j + 2 * h], keep[j + 2 * h + 1]);
            }
          }
          RawPair<DT> y0 = raw_join<DT>(st.rx[j], st.rx[j + 1]);
          RawPair<DT> y1 = raw_join<DT>(st.rx[j + 2], st.rx[j + 3]);
          norm_pairs<DT, ACT, DROP, BWD>(y0, y1, d[0], d[1], k, k, a.slope, scale);
          if constexpr (DROP && !BWD) {
            y0 = pair_keep<DT, 3, 3>(y0, keep[j], keep[j + 1]);
            y1 = pair_keep<DT, 3, 3>(y1, keep[j + 2], keep[j + 3]);
          }
          single_store<DT>(out, 32 * ESIZE<DT>, j, st.left, y0, y1);
        }
      }
    }
    if (!next.is()) break;
    first_piece(a, u, next, p);
    if (VEC == 1 || st.blocks <= 0) {
      st = first_stream<DT, VEC, BWD>(a, p, ring);
      st.start();
    } else {
      first_count(p, st);
    }
    cp = chan_param(a, p.c, p.n > 0 ? a.f.C : 0);
    if (threadIdx.x == 0) tk.slot[tk.par ^ 1] = after;
    __syncthreads();
    tk.par ^= 1;
  }
}

// The gradients of weight and bias: 8 channels a CTA, 32 threads a channel,
// over the chunks of every element.
template <bool LAST>
static __device__ __forceinline__ void norm_param_grads(const NormArgs& a, double2* meet) {
  const int ci = threadIdx.x % 8, part = threadIdx.x / 8;
  const int dt = a.w_bf16 ? BA_BF16 : BA_F32;
  const uint32_t n = (uint32_t)a.f.B * a.f.nchunk;
  for (int64_t c0 = (int64_t)blockIdx.x * 8; c0 < a.f.C; c0 += (int64_t)gridDim.x * 8) {
    const int64_t c = c0 + ci;
    double db = 0.0, dw = 0.0;
    if (c < a.f.C) {
#pragma unroll 4
      for (uint32_t i = part; i < n; i += 32) {
        const float2 t = __ldcg(
            a.chan + (LAST ? (int64_t)i * a.f.C + c
                           : ((int64_t)(i / a.f.nchunk) * a.f.C + c) * a.f.nchunk +
                                 i % a.f.nchunk));
        db += (double)t.x;
        dw += (double)t.y;
      }
    }
    __syncthreads();
    meet[threadIdx.x] = make_double2(db, dw);
    for (int h = 16; h > 0; h >>= 1) {
      __syncthreads();
      if (part < h) {
        meet[threadIdx.x].x += meet[threadIdx.x + 8 * h].x;
        meet[threadIdx.x].y += meet[threadIdx.x + 8 * h].y;
      }
    }
    if (part == 0 && c < a.f.C) {
      if (a.dweight != nullptr) store_f(a.dweight, dt, c, (float)meet[threadIdx.x].y);
      if (a.dbias != nullptr) store_f(a.dbias, dt, c, (float)meet[threadIdx.x].x);
    }
  }
}

// ===========================================================================
// The kernel.  Its floor is HBM, each tensor once.  Measured on the device:
//   2x32x128^3 bf16, 8 groups, silu, last: 143 us forward, 236 backward; units of
//     134 MB are read twice, 3 and 5 passes of 268 MB at 5.6 and 5.7 TB/s;
//   8x4x128^3 fp32, 4 groups, first: 121 us (4.5 TB/s of input and output);
//   2x64x64^3 bf16, 8 groups, silu, last: 40 and 64 us;
//   2x48x96^3 bf16, 8 groups, gelu, dropout, last: 152 and 300 us, of 52 and 78
//     at the floor: Philox and the normal distribution function, and latency;
//   2x256x8^3 bf16, 32 groups, last: 9.5 us, latency.
// Two CTAs an SM: eight channels' sums, constants and masks take 128 registers,
// and with dropout more (bf16 last, bytes of spill stores: 24 forward, backward 40
// to 76; without dropout the backward pass spills 12 with silu, 20 with gelu).
template <int DT, bool LAST, int VEC, int ACT, int DROP, bool BWD>
__global__ void __launch_bounds__(FEAT_THREADS, 2)
    norm_kernel(const __grid_constant__ NormArgs a) {
  // rings (whole lines: a warp's access is four of them, or five if they begin
  // elsewhere) | meet | group sums | group numbers | tickets | weights | planes
  // or constants
  extern __shared__ __align__(128) char norm_smem[];
  char* ring = norm_smem;
  double2* meet = reinterpret_cast<double2*>(ring + RING_BYTES<DT, VEC, BWD>);
  double2* acc = meet + max(FEAT_THREADS, a.f.ncw * VEC);
  GroupStat* gs = reinterpret_cast<GroupStat*>(acc + 2 * a.ugroups);
  Piece* slot = reinterpret_cast<Piece*>(gs + a.ugroups);
  float* wt = reinterpret_cast<float*>(slot + 2);
  float* sm = wt + (a.f.ncw * VEC + 3) / 4 * 4;
  const uint32_t waves = (a.units + a.wave - 1) / a.wave;
  const unsigned ctas = gridDim.x / (unsigned)a.sets;
  const unsigned set = blockIdx.x / ctas, own = blockIdx.x % ctas;
  const Tickets tk = {slot, 0};
  int turn = 0;  // channels first: the part of `meet` that is free
  for (uint32_t w = set; w < waves; w += a.sets) {
    const uint32_t u0 = w * a.wave, total = min(a.wave, a.units - u0) * a.items;
    for (uint32_t t = own; t < total; t += ctas) {
      const uint32_t u = u0 + t / a.items, i = t % a.items;
      float4* part = a.part + (int64_t)u * a.ugroups * a.items + i;
      if constexpr (LAST) {
        const uint32_t b = u / a.f.colblocks, cb = u - b * a.f.colblocks, g0 = cb * a.ugroups;
        LastPlace p = last_place<VEC>(a.f, b, i, cb);
        bool first_pass = true;
        while (true) {
          Stream<DT, VEC, BWD> st = last_stream<DT, VEC, BWD, (BWD && DROP != DROP_NONE)>(a, p, ring);
          const char* first = st.x;
          st.start();
          ChanParam cp = {};
          __syncthreads();  // the last use of the shared memory is over
          if constexpr (BWD) {
            cp = chan_param(a, p.c - p.tx * VEC + threadIdx.x, p.c_end);
            if (first_pass) {
              const float2* s = reinterpret_cast<const float2*>(a.stats) + (int64_t)u * a.ugroups;
              for (uint32_t g = threadIdx.x; g < a.ugroups; g += FEAT_THREADS)
                gs[g] = {s[g].x, s[g].y, 0.0f, 0.0f};
              __syncthreads();
            }
          }
          last_sums<DT, VEC, ACT, DROP, BWD>(a, p, st, first, g0, gs, cp, sm, wt, meet, acc);
          first_pass = false;
          if (p.c - p.tx * VEC + a.f.ncw * VEC >= p.c_end) break;
          p = last_next<VEC>(a.f, p);
        }
        last_put<BWD>(a, p, part, acc);
      } else {
        FirstPlace p;
        first_item(a, u, i, 0, a.f.rows, p);
        first_sums<DT, VEC, ACT, DROP, BWD>(a, u, p, ring, meet + turn * 2 * FEAT_WARPS, part);
        turn ^= 1;
      }
      if constexpr (BWD) {
        if (a.chan != nullptr && !a.cluster) chan_done(a);
      }
    }
    if (a.out == nullptr) continue;
    if (a.cluster) cluster_barrier();
    for (uint32_t t = own; t < total; t += ctas) {
      const uint32_t u = u0 + t / a.items, i = t % a.items;
      // the first block and what else the results need are on their way while
      // the statistics are waited for
      if constexpr (LAST) {
        const uint32_t b = u / a.f.colblocks, cb = u - b * a.f.colblocks, g0 = cb * a.ugroups;
        LastPlace p = last_place<VEC>(a.f, b, i, cb);
        DropRate dr = {};
        if constexpr (DROP) dr = drop_rate(a.drop, p.b);
        bool first_pass = true;
        while (true) {
          Stream<DT, VEC, BWD> st = last_stream<DT, VEC, BWD, DROP != DROP_NONE>(a, p, ring);
          if (a.reverse) st.turn();
          st.start();
          const ChanParam cp = chan_param(a, p.c - p.tx * VEC + threadIdx.x, p.c_end);
          __syncthreads();  // the last use of the shared memory is over
          if (first_pass && !norm_merge<BWD>(a, u, i == 0, gs)) return;
          first_pass = false;
          last_apply<DT, VEC, ACT, DROP, BWD>(a, p, st, g0, gs, cp, dr, sm, wt);
          if (p.c - p.tx * VEC + a.f.ncw * VEC >= p.c_end) break;
          p = last_next<VEC>(a.f, p);
        }
      } else {
        FirstPlace p;
        first_piece(a, u, piece_of(a, i), p);
        Stream<DT, VEC, BWD> st = first_stream<DT, VEC, BWD>(a, p, ring);
        st.start();
        const ChanParam cp = chan_param(a, p.c, p.n > 0 ? a.f.C : 0);
        DropRate dr = {};
        if constexpr (DROP) dr = drop_rate(a.drop, p.b);
        if (a.subs > 1) {
          __syncthreads();  // the last use of the slots is over
          if (threadIdx.x == 0) slot[0] = tk.take(a, u);
        }
        GroupStat g;
        if (!norm_merge_one<BWD>(a, u, i == 0, meet + (4 + turn * 2) * FEAT_WARPS, g)) return;
        turn ^= 1;
        first_apply<DT, VEC, ACT, DROP, BWD>(a, p, st, u, tk, g, cp, dr, ring);
      }
    }
  }
  if constexpr (BWD) {
    if (a.chan != nullptr && !a.cluster) {
      if (!chan_wait(a, a.units * a.items)) return;
      norm_param_grads<LAST>(a, meet);
    }
  }
}

}  // namespace ba

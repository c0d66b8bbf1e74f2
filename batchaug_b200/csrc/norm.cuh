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
// One cooperative launch does it all.  A unit is what is normalised on its
// own: a group of an element (channels first), or the groups of a block of
// columns of an element (channels last).  Units are taken in waves; the
// resident CTAs share a wave's items (equal parts of its units' voxels), first
// for the sums, then for the results.  Every CTA leaves a partial for each
// group of its item and counts it; a CTA that needs a unit's statistics waits
// for the unit's count and merges the partials itself, in double and in a
// fixed order (no atomics on sums: the same bits from every run).  A wave is
// small enough for its inputs to be in L2 still when the results read them
// again, so HBM sees them once; where a unit alone is larger than that, the
// results run backwards and find its second half there.
//
// A forward partial is (mean, M2), taken with the thread's own first value
// subtracted: that shift is one of the summed values, so its distance from
// the mean is itself part of the variance, and M2's relative error stays
// below the number of values a thread sums times 2^-24, whatever the data's
// offset.
#pragma once

#include "feature.cuh"

namespace ba {

enum { ACT_NONE = 0, ACT_LEAKY = 1, ACT_SILU = 2, ACT_GELU = 3 };

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;           // y, or dx (NULL: not wanted)
  const void* weight;  // (C,) or NULL
  const void* bias;
  int32_t w_bf16;      // weight and bias are bf16 (else fp32)
  float* stats;        // (B, G, 2): mean, rstd
  float4* part;        // a partial for each (unit, item, group of the unit):
                       // mean, M2, count / sum w dz, sum w dz xh
  float2* chan;        // backward, where weight or bias want a gradient: sum dz,
                       // sum dz xh of each channel of each chunk
  void* dweight;       // (C,) or NULL, of the weight's type
  void* dbias;
  uint32_t* sync;      // zeroed: items done, then those of each unit
  unsigned int* timeouts;  // where a wait that gave up is recorded, or NULL
  Feat f;
  int64_t G, Cg;
  // the schedule (norm.cu)
  int64_t units;
  int64_t wave;    // units of a wave
  int32_t items;   // work items of a unit
  int32_t ugroups; // groups of a unit
  int32_t ahead;   // sums of wave w + 1 before the results of wave w
  int32_t reverse; // results from the last voxel to the first
  double inv_n;    // 1 / values of a group
  float eps, slope;
  DropArgs drop;
};

__device__ __forceinline__ float norm_param(const void* p, int bf16, int64_t c, float absent) {
  return p == nullptr ? absent : load_f(p, bf16 ? BA_BF16 : BA_F32, c);
}

// ---------------------------------------------------------------------------
// Activations, on pairs.  exp2 and the reciprocal are the hardware's (2 ulp),
// well below the outputs' tolerance in either type.
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

__device__ __forceinline__ F2 sigmoid2(F2 z) {
  const F2 t = mul2(z, f2(-1.44269504f));
  const F2 d = add2(f2(exp2_hw(t.x), exp2_hw(t.y)), f2(1.0f));
  return f2(rcp_hw(d.x), rcp_hw(d.y));
}

__device__ __forceinline__ F2 normal_cdf2(F2 z) {
  const F2 t = mul2(z, f2(0.70710678f));
  return fma2(f2(erff(t.x), erff(t.y)), f2(0.5f), f2(0.5f));
}

template <int ACT>
__device__ __forceinline__ F2 act_value2(F2 z, float slope) {
  if constexpr (ACT == ACT_LEAKY) {
    // slope 0: +0 for any negative z, infinite ones included
    const F2 n = slope == 0.0f ? f2(0.0f) : mul2(z, f2(slope));
    return f2(z.x < 0.0f ? n.x : z.x, z.y < 0.0f ? n.y : z.y);
  }
  if constexpr (ACT == ACT_SILU) return mul2(z, sigmoid2(z));
  if constexpr (ACT == ACT_GELU) return mul2(z, normal_cdf2(z));
  return z;
}

template <int ACT>
__device__ __forceinline__ F2 act_slope2(F2 z, float slope) {
  if constexpr (ACT == ACT_LEAKY)
    return f2(z.x > 0.0f ? 1.0f : slope, z.y > 0.0f ? 1.0f : slope);
  if constexpr (ACT == ACT_SILU) {  // s + z s (1 - s)
    const F2 s = sigmoid2(z);
    return fma2(mul2(z, s), fma2(s, f2(-1.0f), f2(1.0f)), s);
  }
  if constexpr (ACT == ACT_GELU) {  // cdf + z pdf
    const F2 t = mul2(mul2(z, z), f2(-0.72134752f));
    return fma2(mul2(z, f2(0.39894228f)), f2(exp2_hw(t.x), exp2_hw(t.y)), normal_cdf2(z));
  }
  return f2(1.0f);
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
__device__ __forceinline__ PairConst pair_const(const NormArgs& a, const GroupStat& g,
                                                int64_t c) {
  const float w = norm_param(a.weight, a.w_bf16, c, 1.0f);
  const float bias = norm_param(a.bias, a.w_bf16, c, 0.0f);
  return {f2(-g.mean), f2(g.rstd * w), f2(bias), f2(-g.c2), f2(-g.c3)};
}

// The pair of results of x (and dy, its dropped elements zeroed); scale is
// dropout's, 1 without it.
template <int DT, int ACT, bool DROP, bool BWD>
__device__ __forceinline__ RawPair<DT> norm_pair(RawPair<DT> x, RawPair<DT> dy,
                                                 const PairConst& k, float slope, float scale) {
  const F2 xm = add2(pair_value<DT>(x), k.nmean);
  const F2 z = fma2(xm, k.a, k.bias);
  if constexpr (BWD) {
    F2 dz = pair_value<DT>(dy);
    if constexpr (ACT != ACT_NONE) dz = mul2(dz, act_slope2<ACT>(z, slope));
    const F2 a = DROP ? mul2(k.a, f2(scale)) : k.a;
    return pair_raw<DT>(fma2(a, dz, fma2(xm, k.nc3, k.nc2)));
  } else {
    F2 y = act_value2<ACT>(z, slope);
    if constexpr (DROP) y = mul2(y, f2(scale));
    return pair_raw<DT>(y);
  }
}

// Adds the pair to a forward (x about the shift) or backward (dz, dz (x -
// mean), without dropout's scale) sum.
template <int DT, int ACT, bool BWD>
__device__ __forceinline__ void norm_add(RawPair<DT> x, RawPair<DT> dy, const PairConst& k,
                                         float slope, F2& s0, F2& s1) {
  const F2 xm = add2(pair_value<DT>(x), k.nmean);
  if constexpr (BWD) {
    F2 dz = pair_value<DT>(dy);
    if constexpr (ACT != ACT_NONE) dz = mul2(dz, act_slope2<ACT>(fma2(xm, k.a, k.bias), slope));
    s0 = add2(s0, dz);
    s1 = fma2(dz, xm, s1);
  } else {
    s0 = add2(s0, xm);
    s1 = fma2(xm, xm, s1);
  }
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

// ===========================================================================
// Counting and waiting.
// ===========================================================================
constexpr unsigned long long NORM_WAIT_NS = 2000000000ull;

__device__ __forceinline__ void count_release(uint32_t* p) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}
__device__ __forceinline__ uint32_t load_acquire(const uint32_t* p) {
  uint32_t r;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(r) : "l"(p) : "memory");
  return r;
}
__device__ __forceinline__ unsigned long long wall_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Waits, in every thread, until the counter reads n; false if it did not in
// time.  Every CTA is resident and counts its items before it waits, so the
// wait ends.
static __device__ __noinline__ bool norm_wait(const NormArgs& a, const uint32_t* count,
                                              uint32_t n) {
  int ok = 1;
  if (threadIdx.x == 0) {
    unsigned long long t0 = 0;
    while (load_acquire(count) != n) {
      const unsigned long long t = wall_ns();
      if (t0 == 0) t0 = t;
      if (t - t0 > NORM_WAIT_NS) {
        if (a.timeouts != nullptr) atomicOr(a.timeouts, 1u);
        ok = 0;
        break;
      }
    }
  }
  return __syncthreads_and(ok) != 0;
}

// The item's partials are written.
__device__ __forceinline__ void norm_arrive(const NormArgs& a, int64_t u) {
  __syncthreads();
  if (threadIdx.x == 0) {
    count_release(a.sync + 1 + u);
    count_release(a.sync);
  }
}

// A CTA's shared memory beside its rings.
struct NormShared {
  double2 meet[FEAT_THREADS];
};

// Partials of the unit's groups, merged: thread t < ugroups (looping) writes
// group t's numbers to gs.  The threads split a group's partials and meet in
// shared memory.  Partials are written by other CTAs of this launch, so they
// are read through L2 (ld.global.cg).
template <bool BWD>
static __device__ __noinline__ void norm_merge(const NormArgs& a, int64_t u, int64_t stat0,
                                               double2* meet, GroupStat* gs) {
  const int ng = a.ugroups, gw = min(ng, FEAT_THREADS), parts = FEAT_THREADS / gw;
  const int gi = threadIdx.x % gw, part = threadIdx.x / gw;
  for (int g0 = 0; g0 < ng; g0 += gw) {
    const int g = g0 + gi;
    const float4* q = a.part + (u * a.items) * ng + g;
    double s = 0.0, m2 = 0.0, k0 = 0.0;
    const bool mine = part < parts && g < ng;
    if (mine) {
      if constexpr (!BWD) k0 = (double)__ldcg(q).x;
#pragma unroll 4
      for (int k = part; k < a.items; k += parts) {
        const float4 t = __ldcg(q + (int64_t)k * ng);
        if constexpr (BWD) {
          s += (double)t.x;
          m2 += (double)t.y;
        } else {
          const double n = (double)__float_as_uint(t.z), d = (double)t.x - k0;
          s += n * d;
          m2 += (double)t.y + n * d * d;
        }
      }
    }
    __syncthreads();
    meet[threadIdx.x] = make_double2(s, m2);
    for (int m = parts; m > 1;) {
      __syncthreads();
      const int h = (m + 1) >> 1;
      if (mine && part < m - h) {
        double2 v = meet[threadIdx.x];
        const double2 w = meet[threadIdx.x + h * gw];
        v.x += w.x;
        v.y += w.y;
        meet[threadIdx.x] = v;
      }
      m = h;
    }
    if (mine && part == 0) {
      const double2 v = meet[threadIdx.x];
      GroupStat r;
      float2* st = reinterpret_cast<float2*>(a.stats) + stat0 + g;
      const double d = v.x * a.inv_n;
      if constexpr (BWD) {
        const float2 t = *st;
        r.mean = t.x;
        r.rstd = t.y;
        r.c2 = t.y * (float)d;
        r.c3 = t.y * t.y * (float)(v.y * a.inv_n);
      } else {
        const double var = v.y * a.inv_n - d * d;
        r.mean = (float)(k0 + d);
        r.rstd = __frcp_rn(__fsqrt_rn((float)(var < 0.0 ? 0.0 : var) + a.eps));
        r.c2 = r.c3 = 0.0f;
        // every CTA of the unit has the same; the backward pass wants it once
        if (blockIdx.x == (unsigned)((u % a.wave) * a.items % gridDim.x))
          *st = make_float2(r.mean, r.rstd);
      }
      gs[g] = r;
    }
  }
  __syncthreads();
}

// cp.async of BYTES (4, 8, 16).
template <int BYTES>
__device__ __forceinline__ void cp_async(void* smem, const void* gmem) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(s), "l"(gmem) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(s), "l"(gmem), "n"(BYTES)
                 : "memory");
}

// ===========================================================================
// A thread's accesses, eight to a block, each thread's own ring of eight slots
// in shared memory: while a block is worked on, the next one is on its way
// (cp.async, no registers held).  Single elements are loaded into registers, a
// block at a time, instead.
// ===========================================================================
template <int DT, int VEC, bool BWD>
struct Stream {
  static constexpr int BYTES = VEC * ESIZE<DT>;
  const char *x, *dy;
  char* slot;      // the thread's slot 0
  uint32_t row;    // bytes between accesses of unit index distance
  int n;           // indexes below n exist
  int step;        // index distance inside a block
  Raw<DT, 1> rx[VEC == 1 ? 8 : 1], rd[VEC == 1 && BWD ? 8 : 1];

  __device__ __forceinline__ int at(int r, int j) const { return r + j * step; }
  __device__ __forceinline__ bool has(int r, int j) const { return at(r, j) < n && r >= 0; }

  __device__ __forceinline__ void issue(int r, int j) {
    if constexpr (VEC > 1) {
      if (has(r, j)) {
        const uint64_t o = row_at(at(r, j), row);
        cp_async<BYTES>(slot + j * FEAT_THREADS * BYTES, x + o);
        if constexpr (BWD) cp_async<BYTES>(slot + (8 + j) * FEAT_THREADS * BYTES, dy + o);
      }
      cp_async_commit();
    }
  }
  // the first block
  __device__ __forceinline__ void start(int r) {
#pragma unroll
    for (int j = 0; j < 8; ++j) issue(r, j);
  }
  // single elements: the whole block
  __device__ __forceinline__ void fill(int r) {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rx[j] = 0;
        if constexpr (BWD) rd[j] = 0;
        if (has(r, j)) {
          const uint64_t o = row_at(at(r, j), row);
          rx[j] = raw_load<DT, 1>(x + o);
          if constexpr (BWD) rd[j] = raw_load<DT, 1>(dy + o);
        }
      }
    }
  }
  // accesses j and j + 1 of the block have arrived (those after them not)
  __device__ __forceinline__ void wait2() {
    if constexpr (VEC > 1) cp_async_wait<6>();
  }
  __device__ __forceinline__ Raw<DT, VEC> get_x(int j) const {
    return *reinterpret_cast<const Raw<DT, VEC>*>(slot + j * FEAT_THREADS * BYTES);
  }
  __device__ __forceinline__ Raw<DT, VEC> get_dy(int j) const {
    return *reinterpret_cast<const Raw<DT, VEC>*>(slot + (8 + j) * FEAT_THREADS * BYTES);
  }
};

// Bytes of a CTA's rings.
template <int DT, int VEC, bool BWD>
constexpr int RING_BYTES = VEC == 1 ? 0 : FEAT_THREADS * VEC * ESIZE<DT> * 8 * (BWD ? 2 : 1);

// ===========================================================================
// Channels last
// ===========================================================================
// The constants of a pass's channels in shared memory: plane by plane
// (mean, a, bias, c2, c3, as PairConst has them), a thread's pair i at
// (i * ncw + tx), so that neighbouring threads read neighbouring words.
// sm: 5 * ncw * VEC floats.
template <int VEC, bool COEF>
__device__ __forceinline__ void last_consts(const NormArgs& a, const LastPlace& p, int64_t g0,
                                            const GroupStat* gs, float* sm) {
  constexpr int P = VEC > 1 ? 2 : 1;
  const int cw = a.f.ncw * VEC;
  const int64_t c0 = p.c - p.tx * VEC;
  __syncthreads();
  for (int i = threadIdx.x; i < cw; i += FEAT_THREADS) {
    if (c0 + i < p.c_end) {
      const int g = (int)((uint32_t)(c0 + i) / (uint32_t)a.Cg - (uint32_t)g0);
      const PairConst q = pair_const(a, gs[g], c0 + i);
      float* to = sm + ((i % VEC / P) * a.f.ncw + i / VEC) * P + i % P;
      to[0] = q.nmean.x;
      to[cw] = q.a.x;
      to[2 * cw] = q.bias.x;
      if constexpr (COEF) {
        to[3 * cw] = q.nc2.x;
        to[4 * cw] = q.nc3.x;
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
  const int64_t base = last_base<DT>(a.f, p);
  s.x = (const char*)a.x + base;
  s.dy = (const char*)a.dy + base;
  s.slot = ring + threadIdx.x * VEC * ESIZE<DT>;
  s.row = (uint32_t)a.f.C * ESIZE<DT>;
  s.n = p.on ? p.rows : 0;
  s.step = BLOCK ? 1 : p.nty;
  return s;
}

template <bool BLOCK>
__device__ __forceinline__ int last_first(const LastPlace& p) {
  return BLOCK ? p.ty * 8 : p.ty;
}

// The sums of a pass (256 columns at most) of one item, added to the item's
// groups.  sm: two planes of nty rows by cw channels, floats (2 *
// FEAT_THREADS * VEC in all); acc: the groups' sums so far.
template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__device__ __forceinline__ void last_sums(const NormArgs& a, const LastPlace& p, int64_t g0,
                                          const GroupStat* gs, char* ring, float* sm,
                                          double2* meet, double2* acc, bool first_pass) {
  constexpr bool BLOCK = BWD && DROP;
  constexpr int NP = VEC > 1 ? VEC / 2 : 1;  // pairs of channels, or of rows
  Stream<DT, VEC, BWD> st = last_stream<DT, VEC, BWD, BLOCK>(a, p, ring);
  const int span = p.nty * 8;
  int r = last_first<BLOCK>(p);
  st.start(r);
  F2 s0[NP], s1[NP];
  PairConst k[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) s0[i] = s1[i] = f2(0.0f);
  DropRate dr = {};
  if constexpr (BWD) {
    last_consts<VEC, false>(a, p, g0, gs, sm);
#pragma unroll
    for (int i = 0; i < NP; ++i) k[i] = last_const<VEC, false>(a, p, i, sm);
    if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  } else {
    // the thread's first row is its shift
#pragma unroll
    for (int i = 0; i < NP; ++i) k[i] = {};
    if (st.has(r, 0)) {
      const Raw<DT, VEC> v = raw_load<DT, VEC>(st.x + row_at(r, st.row));
      if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const F2 t = pair_value<DT>(raw_pair<DT, VEC>(v, i));
          k[i].nmean = f2(-t.x, -t.y);
        }
      } else {
        const F2 t = pair_value<DT>(raw_join<DT>(v, v));
        k[0].nmean = f2(-t.x, -t.y);
      }
    }
  }
#pragma unroll 1
  for (; r < st.n; r += span) {
    uint32_t keep[VEC];
    if constexpr (BLOCK) last_keep<VEC>(a.f, dr, p, r, keep);
    st.fill(r);
    if constexpr (VEC > 1) {
#pragma unroll 1
      for (int j = 0; j < 8; j += 2) {
        st.wait2();
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (st.has(r, j + h)) {
            const Raw<DT, VEC> vx = st.get_x(j + h);
            Raw<DT, VEC> vd = {};
            if constexpr (BWD) vd = st.get_dy(j + h);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              RawPair<DT> d = raw_pair<DT, VEC>(vd, i);
              if constexpr (BLOCK) d = last_pair_keep<DT>(d, keep, i, h);
              norm_add<DT, ACT, BWD>(raw_pair<DT, VEC>(vx, i), d, k[i], a.slope, s0[i], s1[i]);
            }
          }
        st.issue(r + span, j);
        st.issue(r + span, j + 1);
        if constexpr (BLOCK) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) keep[i] <<= 1;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const bool h0 = st.has(r, j), h1 = st.has(r, j + 1);
        RawPair<DT> d = {};
        if constexpr (BWD) d = raw_join<DT>(st.rd[j], st.rd[j + 1]);
        if constexpr (BLOCK) d = pair_keep<DT, 1, 3>(d, keep[0] << (j >> 1), keep[0] << (j >> 1));
        F2 t0 = s0[0], t1 = s1[0];
        norm_add<DT, ACT, BWD>(raw_join<DT>(st.rx[j], st.rx[j + 1]), d, k[0], a.slope, t0, t1);
        s0[0] = f2(h0 ? t0.x : s0[0].x, h1 ? t0.y : s0[0].y);
        s1[0] = f2(h0 ? t1.x : s1[0].x, h1 ? t1.y : s1[0].y);
      }
    }
  }
  // threads -> channels
  const int cw = a.f.ncw * VEC, rows = p.rows;
  float* plane = sm + p.nty * cw;
  const float n_own = (float)((rows - p.ty + p.nty - 1) / p.nty);  // forward: rows of this thread
  const float inv = 1.0f / n_own;
  __syncthreads();
  if (p.ty < p.nty) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int h = VEC > 1 ? i / 2 : 0;
      const float t = VEC == 1 ? s0[0].x + s0[0].y : i & 1 ? s0[h].y : s0[h].x;
      float u = t, w = VEC == 1 ? s1[0].x + s1[0].y : i & 1 ? s1[h].y : s1[h].x;
      if constexpr (!BWD) {
        // a thread's (mean, M2); nothing when it had no row
        const float m = t * inv;
        u = m - (i & 1 ? k[h].nmean.y : k[h].nmean.x);
        w = __fmaf_rn(-t, m, w);
      }
      sm[p.ty * cw + p.tx * VEC + i] = u;
      plane[p.ty * cw + p.tx * VEC + i] = w;
    }
  }
  __syncthreads();
  const int parts = cw >= FEAT_THREADS ? 1 : FEAT_THREADS / cw;
  const int64_t c0 = p.c - p.tx * VEC;
#pragma unroll 1
  for (int cb = 0; cb < cw; cb += FEAT_THREADS) {
    const int ci = cb + (parts == 1 ? (int)threadIdx.x : (int)threadIdx.x % cw);
    const int part = parts == 1 ? 0 : threadIdx.x / cw;
    const bool mine = part < parts && ci < cw && c0 + ci < p.c_end;
    double u = 0.0, w = 0.0;
    const double k0 = mine ? (double)sm[ci] : 0.0;
    if (mine)
#pragma unroll 2
      for (int y = part; y < p.nty && (BWD || y < rows); y += parts) {
        const float q = sm[y * cw + ci], m2 = plane[y * cw + ci];
        if constexpr (BWD) {
          u += (double)q;
          w += (double)m2;
        } else {
          const double n = (double)((rows - y + p.nty - 1) / p.nty), d = (double)q - k0;
          u += n * d;
          w += (double)m2 + n * d * d;
        }
      }
    for (int m = parts; m > 1;) {
      meet[threadIdx.x] = make_double2(u, w);
      __syncthreads();
      const int h = (m + 1) >> 1;
      if (mine && part < m - h) {
        u += meet[threadIdx.x + h * cw].x;
        w += meet[threadIdx.x + h * cw].y;
      }
      __syncthreads();
      m = h;
    }
    // (mean, M2) about k0, or the sums, of the channel in place of its row 0
    if (mine && part == 0) {
      if constexpr (BWD) {
        const double sc = DROP ? (double)dr.scale : 1.0;
        const int64_t c = c0 + ci;
        const float rstd = gs[(uint32_t)c / (uint32_t)a.Cg - (uint32_t)g0].rstd;
        u *= sc;
        w *= sc * (double)rstd;
        if (a.chan != nullptr)
          __stcg(a.chan + (p.b * a.f.nchunk + p.k) * a.f.C + c, make_float2((float)u, (float)w));
      } else {
        const double n = (double)rows, d = u / n;
        w -= u * d;
        u = k0 + d;
      }
      sm[ci] = (float)u;
      plane[ci] = (float)w;
    }
  }
  __syncthreads();
  // channels -> groups, a warp a group
  const int cend = (int)min((int64_t)cw, p.c_end - c0);
  const int ga = (int)((uint32_t)c0 / (uint32_t)a.Cg), gb = (int)((uint32_t)(c0 + cend - 1) / (uint32_t)a.Cg);
#pragma unroll 1
  for (int g = ga + (int)threadIdx.x / 32; g <= gb; g += FEAT_WARPS) {
    const int i0 = (int)max((int64_t)0, (int64_t)g * a.Cg - c0);
    const int i1 = (int)min((int64_t)cend, (int64_t)(g + 1) * a.Cg - c0);
    double u = 0.0, w = 0.0;
    const double k0 = first_pass || BWD ? (BWD ? 0.0 : (double)sm[i0]) : acc[2 * (g - g0) + 1].x;
    for (int i = i0 + (int)threadIdx.x % 32; i < i1; i += 32) {
      const double q = (double)sm[i], m2 = (double)plane[i];
      if constexpr (BWD) {
        const double wt = (double)norm_param(a.weight, a.w_bf16, c0 + i, 1.0f);
        u += wt * q;
        w += wt * m2;
      } else {
        const double n = (double)rows, e = q - k0;
        u += n * e;
        w += m2 + n * e * e;
      }
    }
    u = warp_sum(u);
    w = warp_sum(w);
    if (threadIdx.x % 32 == 0) {
      double2* t = acc + 2 * (g - g0);
      if (first_pass) {
        t[0] = make_double2(u, w);
        t[1] = make_double2(k0, 0.0);
      } else {
        t[0].x += u;
        t[0].y += w;
      }
    }
  }
  __syncthreads();
}

// y or dx of a pass of one item; `started`: its first block is on its way.
template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__device__ __forceinline__ void last_apply(const NormArgs& a, const LastPlace& p,
                                           Stream<DT, VEC, BWD>& st, int64_t g0,
                                           const GroupStat* gs, float* sm) {
  constexpr int NP = VEC > 1 ? VEC / 2 : 1;
  const int span = p.nty * 8, end = (p.rows + span - 1) / span * span;
  const int dir = a.reverse ? -span : span;
  int r = last_first<DROP>(p) + (a.reverse ? end - span : 0);
  char* out = (char*)a.out + last_base<DT>(a.f, p);
  last_consts<VEC, BWD>(a, p, g0, gs, sm);
  if (!p.on) return;
  DropRate dr = {};
  if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  const float scale = DROP ? dr.scale : 1.0f;
  PairConst k[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) k[i] = last_const<VEC, BWD>(a, p, i, sm);
#pragma unroll 1
  for (int q = 0; q < end; q += span, r += dir) {
    uint32_t keep[VEC];
    if constexpr (DROP) last_keep<VEC>(a.f, dr, p, r, keep);
    st.fill(r);
    if constexpr (VEC > 1) {
#pragma unroll 1
      for (int j = 0; j < 8; j += 2) {
        st.wait2();
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (st.has(r, j + h)) {
            Raw<DT, VEC> vx = st.get_x(j + h), vd = {};
            if constexpr (BWD) vd = st.get_dy(j + h);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              RawPair<DT> d = raw_pair<DT, VEC>(vd, i);
              if constexpr (BWD && DROP) d = last_pair_keep<DT>(d, keep, i, h);
              RawPair<DT> y = norm_pair<DT, ACT, DROP, BWD>(raw_pair<DT, VEC>(vx, i), d, k[i],
                                                            a.slope, scale);
              if constexpr (DROP && !BWD) y = last_pair_keep<DT>(y, keep, i, h);
              raw_set_pair<DT, VEC>(vx, i, y);
            }
            raw_store<DT, VEC>(out + row_at(st.at(r, j + h), st.row), vx);
          }
        st.issue(r + dir, j);
        st.issue(r + dir, j + 1);
        if constexpr (DROP) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) keep[i] <<= 1;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const uint32_t w = DROP ? keep[0] << (j >> 1) : 0u;
        RawPair<DT> d = {};
        if constexpr (BWD) {
          d = raw_join<DT>(st.rd[j], st.rd[j + 1]);
          if constexpr (DROP) d = pair_keep<DT, 1, 3>(d, w, w);
        }
        RawPair<DT> y = norm_pair<DT, ACT, DROP, BWD>(raw_join<DT>(st.rx[j], st.rx[j + 1]), d,
                                                      k[0], a.slope, scale);
        if constexpr (DROP && !BWD) y = pair_keep<DT, 1, 3>(y, w, w);
        if (st.has(r, j)) raw_store<DT, 1>(out + row_at(st.at(r, j), st.row), raw_half<DT>(y, 0));
        if (st.has(r, j + 1))
          raw_store<DT, 1>(out + row_at(st.at(r, j + 1), st.row), raw_half<DT>(y, 1));
      }
    }
  }
}

// ===========================================================================
// Channels first.  Item i of a group: 8 of its runs (channel, f.rows voxels),
// one for each warp.  An access is 32 * VEC voxels of a warp.
// ===========================================================================
__device__ __forceinline__ bool first_item(const NormArgs& a, int64_t u, int i, FirstPlace& p) {
  const int64_t run = (int64_t)i * FEAT_WARPS + threadIdx.x / 32;
  p.lane = threadIdx.x % 32;
  p.b = u / a.G;
  const int64_t cl = run / a.f.nchunk;
  p.k = run - cl * a.f.nchunk;
  p.c = (u - p.b * a.G) * a.Cg + cl;
  p.s0 = p.k * a.f.rows;
  p.n = cl < a.Cg ? (int)min(a.f.rows, a.f.S - p.s0) : 0;
  p.base = (p.b * a.f.C + p.c) * a.f.S + p.s0;
  return cl < a.Cg;
}

template <int DT, int VEC, bool BWD>
__device__ __forceinline__ Stream<DT, VEC, BWD> first_stream(const NormArgs& a,
                                                             const FirstPlace& p, char* ring) {
  Stream<DT, VEC, BWD> s;
  s.x = (const char*)a.x + p.base * ESIZE<DT>;
  s.dy = (const char*)a.dy + p.base * ESIZE<DT>;
  s.slot = ring + threadIdx.x * VEC * ESIZE<DT>;
  s.row = ESIZE<DT>;  // indexes are voxels
  s.n = p.n;
  s.step = 32 * VEC;
  return s;
}

// Keep words of accesses j and j + 1 of a block (k: 8 / VEC words a tile; two
// tiles for VEC 8, one for VEC 4; a single element's tile is a block).
template <int VEC>
__device__ __forceinline__ void first_block_keep(const NormArgs& a, const DropRate& dr,
                                                 const FirstPlace& p, int s, uint32_t* k) {
  first_keep<VEC>(a.f, dr, p, s, k);
  if constexpr (VEC == 8) first_keep<VEC>(a.f, dr, p, s + FEAT_TILE, k + 1);
}

template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__device__ __forceinline__ void first_sums(const NormArgs& a, const FirstPlace& p,
                                           const GroupStat* gs, char* ring, double2* meet,
                                           float4* part) {
  Stream<DT, VEC, BWD> st = first_stream<DT, VEC, BWD>(a, p, ring);
  const int own = first_at<VEC>(p.lane, 0);
  constexpr int span = 256 * VEC;
  st.start(own);
  F2 s0 = f2(0.0f), s1 = f2(0.0f);
  float shift = 0.0f;
  PairConst k = {};
  DropRate dr = {};
  if constexpr (BWD) {
    if (p.n > 0) {
      k = pair_const(a, gs[0], p.c);
      if constexpr (DROP) dr = drop_rate(a.drop, p.b);
    }
  } else {
    if (own < p.n) shift = load_f(st.x, DT, own);
    k.nmean = f2(-shift);
  }
#pragma unroll 1
  for (int s = 0; s < p.n; s += span) {
    st.fill(s + own);
    if constexpr (VEC > 1) {
#pragma unroll 1
      for (int j = 0; j < 8; j += 2) {
        uint32_t keep[2];
        if constexpr (BWD && DROP) first_block_keep<VEC>(a, dr, p, s + j * 32 * VEC, keep);
        st.wait2();
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (st.has(s + own, j + h)) {
            const Raw<DT, VEC> vx = st.get_x(j + h);
            Raw<DT, VEC> vd = {};
            if constexpr (BWD) vd = st.get_dy(j + h);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
              RawPair<DT> d = raw_pair<DT, VEC>(vd, i);
              if constexpr (BWD && DROP) d = pair_keep<DT, 1, 3>(d, keep[h] << i, keep[h] << i);
              norm_add<DT, ACT, BWD>(raw_pair<DT, VEC>(vx, i), d, k, a.slope, s0, s1);
            }
          }
        st.issue(s + own + span, j);
        st.issue(s + own + span, j + 1);
      }
    } else {
      uint32_t keep[8];
      if constexpr (BWD && DROP) first_keep<VEC>(a.f, dr, p, s, keep);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const bool h0 = st.has(s + own, j), h1 = st.has(s + own, j + 1);
        RawPair<DT> d = {};
        if constexpr (BWD) d = raw_join<DT>(st.rd[j], st.rd[j + 1]);
        if constexpr (BWD && DROP) d = pair_keep<DT, 3, 3>(d, keep[j], keep[j + 1]);
        F2 t0 = s0, t1 = s1;
        norm_add<DT, ACT, BWD>(raw_join<DT>(st.rx[j], st.rx[j + 1]), d, k, a.slope, t0, t1);
        s0 = f2(h0 ? t0.x : s0.x, h1 ? t0.y : s0.y);
        s1 = f2(h0 ? t1.x : s1.x, h1 ? t1.y : s1.y);
      }
    }
  }
  // lanes -> run -> item, in double
  const int warp = threadIdx.x / 32;
  double u, w;
  double* shifts = reinterpret_cast<double*>(meet + 2 * FEAT_WARPS);
  if constexpr (BWD) {
    const double sc = DROP ? (double)dr.scale : 1.0;
    u = warp_sum((double)s0.x + (double)s0.y) * sc;
    w = warp_sum((double)s1.x + (double)s1.y) * sc * (double)gs[0].rstd;
    if (p.lane == 0 && p.n > 0 && a.chan != nullptr)
      __stcg(a.chan + (p.b * a.f.C + p.c) * a.f.nchunk + p.k, make_float2((float)u, (float)w));
    const double wt = p.n > 0 ? (double)norm_param(a.weight, a.w_bf16, p.c, 1.0f) : 0.0;
    u *= wt;
    w *= wt;
  } else {
    // a lane's (mean, M2), about the shift of the CTA's first lane
    if (threadIdx.x == 0) shifts[0] = (double)shift;
    __syncthreads();
    int cnt = 0;
#pragma unroll
    for (int j = 0; j < (VEC == 1 ? 8 : 1); ++j) {
      const int at = own + 32 * j;  // each access of VEC > 1 is whole
      const int every = VEC == 1 ? FEAT_TILE : 32 * VEC;
      cnt += at < p.n ? (p.n - at + every - 1) / every * VEC : 0;
    }
    const double n = (double)cnt;
    const float t0 = s0.x + s0.y, t1 = s1.x + s1.y;
    const float mt = cnt > 0 ? t0 / (float)cnt : 0.0f;
    const double off = (double)shift - shifts[0] + (double)mt;
    u = warp_sum(cnt > 0 ? n * off : 0.0);
    w = warp_sum(cnt > 0 ? (double)__fmaf_rn(-t0, mt, t1) + n * off * off : 0.0);
  }
  if (p.lane == 0) {
    meet[warp] = make_double2(u, w);
    meet[FEAT_WARPS + warp].x = (double)p.n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double n = 0.0;
    u = w = 0.0;
    for (int i = 0; i < FEAT_WARPS; ++i) {
      u += meet[i].x;
      w += meet[i].y;
      n += meet[FEAT_WARPS + i].x;
    }
    if constexpr (BWD) {
      __stcg(part, make_float4((float)u, (float)w, 0.0f, 0.0f));
    } else {
      const double d = u / n;
      __stcg(part, make_float4((float)(shifts[0] + d), (float)(w - u * d),
                               __uint_as_float((uint32_t)n), 0.0f));
    }
  }
}

template <int DT, int VEC, int ACT, bool DROP, bool BWD>
__device__ __forceinline__ void first_apply(const NormArgs& a, const FirstPlace& p,
                                            Stream<DT, VEC, BWD>& st, const GroupStat* gs) {
  if (p.n == 0) return;
  const int own = first_at<VEC>(p.lane, 0);
  constexpr int span = 256 * VEC;
  const int end = (p.n + span - 1) / span * span, dir = a.reverse ? -span : span;
  char* out = (char*)a.out + p.base * ESIZE<DT>;
  const PairConst k = pair_const(a, gs[0], p.c);
  DropRate dr = {};
  if constexpr (DROP) dr = drop_rate(a.drop, p.b);
  const float scale = DROP ? dr.scale : 1.0f;
  int s = a.reverse ? end - span : 0;
#pragma unroll 1
  for (int q = 0; q < end; q += span, s += dir) {
    st.fill(s + own);
    if constexpr (VEC > 1) {
#pragma unroll 1
      for (int j = 0; j < 8; j += 2) {
        uint32_t keep[2];
        if constexpr (DROP) first_block_keep<VEC>(a, dr, p, s + j * 32 * VEC, keep);
        st.wait2();
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (st.has(s + own, j + h)) {
            Raw<DT, VEC> vx = st.get_x(j + h), vd = {};
            if constexpr (BWD) vd = st.get_dy(j + h);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
              RawPair<DT> d = raw_pair<DT, VEC>(vd, i);
              if constexpr (BWD && DROP) d = pair_keep<DT, 1, 3>(d, keep[h] << i, keep[h] << i);
              RawPair<DT> y =
                  norm_pair<DT, ACT, DROP, BWD>(raw_pair<DT, VEC>(vx, i), d, k, a.slope, scale);
              if constexpr (DROP && !BWD) y = pair_keep<DT, 1, 3>(y, keep[h] << i, keep[h] << i);
              raw_set_pair<DT, VEC>(vx, i, y);
            }
            raw_store<DT, VEC>(out + (int64_t)st.at(s + own, j + h) * ESIZE<DT>, vx);
          }
        st.issue(s + own + dir, j);
        st.issue(s + own + dir, j + 1);
      }
    } else {
      uint32_t keep[8];
      if constexpr (DROP) first_keep<VEC>(a.f, dr, p, s, keep);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        RawPair<DT> d = {};
        if constexpr (BWD) d = raw_join<DT>(st.rd[j], st.rd[j + 1]);
        if constexpr (BWD && DROP) d = pair_keep<DT, 3, 3>(d, keep[j], keep[j + 1]);
        RawPair<DT> y = norm_pair<DT, ACT, DROP, BWD>(raw_join<DT>(st.rx[j], st.rx[j + 1]), d, k,
                                                      a.slope, scale);
        if constexpr (DROP && !BWD) y = pair_keep<DT, 3, 3>(y, keep[j], keep[j + 1]);
        if (st.has(s + own, j))
          raw_store<DT, 1>(out + (int64_t)st.at(s + own, j) * ESIZE<DT>, raw_half<DT>(y, 0));
        if (st.has(s + own, j + 1))
          raw_store<DT, 1>(out + (int64_t)st.at(s + own, j + 1) * ESIZE<DT>, raw_half<DT>(y, 1));
      }
    }
  }
}

// The gradients of weight and bias: 8 channels a CTA, 32 threads a channel,
// over the chunks of every element.
template <bool LAST>
static __device__ __noinline__ void norm_param_grads(const NormArgs& a, double2* meet) {
  const int ci = threadIdx.x % 8, part = threadIdx.x / 8;
  const int dt = a.w_bf16 ? BA_BF16 : BA_F32;
  const int64_t n = a.f.B * a.f.nchunk;
  for (int64_t c0 = (int64_t)blockIdx.x * 8; c0 < a.f.C; c0 += (int64_t)gridDim.x * 8) {
    const int64_t c = c0 + ci;
    double db = 0.0, dw = 0.0;
    if (c < a.f.C) {
#pragma unroll 4
      for (int64_t i = part; i < n; i += 32) {
        const float2 t = __ldcg(
            a.chan + (LAST ? i * a.f.C + c
                           : (i / a.f.nchunk * a.f.C + c) * a.f.nchunk + i % a.f.nchunk));
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
template <int DT, bool LAST, int VEC, int ACT, bool DROP, bool BWD>
__global__ void __launch_bounds__(FEAT_THREADS, 2)
    norm_kernel(const __grid_constant__ NormArgs a) {
  // meet | group numbers | group sums | rings | planes or constants
  extern __shared__ double2 norm_smem[];
  double2* meet = norm_smem;
  double2* acc = meet + FEAT_THREADS;
  GroupStat* gs = reinterpret_cast<GroupStat*>(acc + 2 * a.ugroups);
  char* ring = reinterpret_cast<char*>(gs + a.ugroups);
  float* sm = reinterpret_cast<float*>(ring + RING_BYTES<DT, VEC, BWD>);
  const int64_t waves = (a.units + a.wave - 1) / a.wave;
  for (int64_t w = 0; w < waves + a.ahead; ++w) {
    if (w < waves) {
      const int64_t u0 = w * a.wave, total = min(a.wave, a.units - u0) * a.items;
      for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const int64_t u = u0 + t / a.items;
        const int i = (int)(t % a.items);
        float4* part = a.part + (u * a.items + i) * a.ugroups;
        if constexpr (BWD) {
          // mean and rstd of the unit's groups
          __syncthreads();
          const int64_t s0 = u * a.ugroups;
          for (int g = threadIdx.x; g < a.ugroups; g += FEAT_THREADS) {
            const float2 q = reinterpret_cast<const float2*>(a.stats)[s0 + g];
            gs[g] = {q.x, q.y, 0.0f, 0.0f};
          }
          __syncthreads();
        }
        if constexpr (LAST) {
          const int64_t g0 = (u % a.f.colblocks) * a.ugroups;
          LastPlace p = last_place<VEC>(a.f, u / a.f.colblocks, i, u % a.f.colblocks);
          bool first_pass = true;
          while (true) {
            last_sums<DT, VEC, ACT, DROP, BWD>(a, p, g0, gs, ring, sm, meet, acc, first_pass);
            first_pass = false;
            if (p.c - p.tx * VEC + a.f.ncw * VEC >= p.c_end) break;
            p = last_next<VEC>(a.f, p);
          }
          for (int g = threadIdx.x; g < a.ugroups; g += FEAT_THREADS) {
            const double2 q = acc[2 * g];
            if constexpr (BWD) {
              __stcg(part + g, make_float4((float)q.x, (float)q.y, 0.0f, 0.0f));
            } else {
              const double n = (double)p.rows * (double)a.Cg, d = q.x / n;
              __stcg(part + g, make_float4((float)(acc[2 * g + 1].x + d), (float)(q.y - q.x * d),
                                           __uint_as_float((uint32_t)n), 0.0f));
            }
          }
        } else {
          FirstPlace p;
          first_item(a, u, i, p);
          first_sums<DT, VEC, ACT, DROP, BWD>(a, p, gs, ring, meet, part);
        }
        norm_arrive(a, u);
      }
    }
    const int64_t v = w - a.ahead;
    if (v >= 0 && a.out != nullptr) {
      const int64_t u0 = v * a.wave, total = min(a.wave, a.units - u0) * a.items;
      for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const int64_t u = u0 + t / a.items;
        const int i = (int)(t % a.items);
        // the first block is on its way while the statistics are waited for
        if constexpr (LAST) {
          const int64_t g0 = (u % a.f.colblocks) * a.ugroups;
          LastPlace p = last_place<VEC>(a.f, u / a.f.colblocks, i, u % a.f.colblocks);
          bool first_pass = true;
          while (true) {
            Stream<DT, VEC, BWD> st = last_stream<DT, VEC, BWD, DROP>(a, p, ring);
            const int span = p.nty * 8;
            st.start(last_first<DROP>(p) + (a.reverse ? (p.rows - 1) / span * span : 0));
            if (first_pass) {
              if (!norm_wait(a, a.sync + 1 + u, (uint32_t)a.items)) return;
              norm_merge<BWD>(a, u, u * a.ugroups, meet, gs);
            }
            first_pass = false;
            last_apply<DT, VEC, ACT, DROP, BWD>(a, p, st, g0, gs, sm);
            if (p.c - p.tx * VEC + a.f.ncw * VEC >= p.c_end) break;
            p = last_next<VEC>(a.f, p);
          }
        } else {
          FirstPlace p;
          first_item(a, u, i, p);
          Stream<DT, VEC, BWD> st = first_stream<DT, VEC, BWD>(a, p, ring);
          constexpr int span = 256 * VEC;
          st.start(first_at<VEC>(p.lane, 0) +
                   (a.reverse && p.n > 0 ? (p.n - 1) / span * span : 0));
          if (!norm_wait(a, a.sync + 1 + u, (uint32_t)a.items)) return;
          norm_merge<BWD>(a, u, u, meet, gs);
          first_apply<DT, VEC, ACT, DROP, BWD>(a, p, st, gs);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (a.chan != nullptr) {
      if (!norm_wait(a, a.sync, (uint32_t)(a.units * a.items))) return;
      norm_param_grads<LAST>(a, meet);
    }
  }
}

}  // namespace ba

// Counter-based dropout bits, shared by the dropout kernels, the group norm's
// epilogue and the intensity chain.  The mask is never stored: every pass
// that needs it draws it again from the counter.
//
// Voxel s of channel c of global element e owns a 32-bit number r, and stays
// iff r >= ceil(p * 2^32), so it is dropped with probability p to 2^-32.  The
// numbers of 8 consecutive voxels of a channel come from one Philox block:
//   q = c * ceil(S / 8) + s / 8,
//   counter (q, e, e >> 32, STREAM | q >> 32), key = seed;
// its four words are eight 16-bit halves (low half first), the high halves
// of the eight numbers.  The low halves are the same block on a second
// stream, and are drawn only when a high half equals the threshold's high
// half and the threshold's low half is not zero: one block in 8,192 for a
// threshold that needs it.  So eight decisions of 32 bits cost one Philox
// block (ten rounds, ~60 issue slots), not two; a 16-byte vector of bf16 then
// costs fewer issue slots than its HBM time allows.
//
// The bits depend on (seed, global element, channel, voxel) alone: not on
// the memory layout, the launch shape or the batch's sharding.
#pragma once

#include "ba_common.cuh"
#include "philox.cuh"

namespace ba {

constexpr uint32_t STREAM_DROP = 0x44500000u;             // voxels, high halves
constexpr uint32_t STREAM_DROP_LOW = 0x44510000u;         // voxels, low halves
constexpr uint32_t STREAM_DROP_CHANNEL = 0x44520000u;     // channels, high halves
constexpr uint32_t STREAM_DROP_CHANNEL_LOW = 0x44530000u; // channels, low halves

// The drop rate's source and the generator's key, as the host passes them.
struct DropArgs {
  float p;                 // the rate when p_elem is NULL
  const float* p_elem;     // (B,) rates
  const uint8_t* mask;     // (B,) 0/1: elements to drop in, NULL = every one
  uint32_t seed_lo, seed_hi;
  const uint64_t* seed_dev;  // the key in device memory, NULL: seed_lo / seed_hi
  uint64_t elem_offset;
  int rescale;             // scale what stays by 1 / (1 - p)
  uint32_t keys[20];       // the ten rounds' keys of seed_lo / seed_hi (drop_keys)
};

// Where a kernel has the rounds' keys from: the kernel's parameters (the
// constant bank, an operand of the round's XOR; 18 additions of a block's 60
// instructions less), or two words that it adds to.
enum { DROP_NONE = 0, DROP_PARAM = 1, DROP_WORDS = 2 };

inline void drop_keys(DropArgs& a) {
  for (uint32_t i = 0; i < 10; ++i) {
    a.keys[2 * i] = a.seed_lo + i * 0x9E3779B9u;
    a.keys[2 * i + 1] = a.seed_hi + i * 0xBB67AE85u;
  }
}

// An element's rate, resolved.
struct DropRate {
  uint32_t hi, lo;    // halves of the threshold; hi == 0x10000: nothing stays
  uint32_t k0, k1;    // Philox key
  uint32_t e_lo, e_hi;
  float scale;        // of what stays
};

__device__ __forceinline__ DropRate drop_rate(const DropArgs& a, int64_t b) {
  DropRate r;
  const bool on = a.mask == nullptr || a.mask[b] != 0;
  float p = a.p_elem != nullptr ? a.p_elem[b] : a.p;
  p = (on && p > 0.0f) ? p : 0.0f;  // NaN counts as 0
  r.scale = (a.rescale && on) ? (p < 1.0f ? __frcp_rn(1.0f - p) : 0.0f) : 1.0f;
  // p * 2^32 is exact; below 1 it is at most 2^32 - 2^8
  const uint32_t t = p < 1.0f ? __float2uint_ru(p * 4294967296.0f) : 0u;
  r.hi = p < 1.0f ? t >> 16 : 0x10000u;
  r.lo = p < 1.0f ? t & 0xFFFFu : 0u;
  if (a.seed_dev != nullptr) {
    const uint64_t s = *a.seed_dev;
    r.k0 = (uint32_t)s;
    r.k1 = (uint32_t)(s >> 32);
  } else {
    r.k0 = a.seed_lo;
    r.k1 = a.seed_hi;
  }
  const uint64_t e = a.elem_offset + (uint64_t)b;
  r.e_lo = (uint32_t)e;
  r.e_hi = (uint32_t)(e >> 32);
  return r;
}

// philox4x32_10 with each 64-bit product as one instruction.
template <int KEYS>
__device__ __forceinline__ U4 drop_block(const DropArgs& a, const DropRate& r, uint64_t q,
                                         uint32_t stream) {
  uint32_t x = (uint32_t)q, y = r.e_lo, z = r.e_hi, w = stream | (uint32_t)(q >> 32);
  uint32_t k0 = r.k0, k1 = r.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t m = (uint64_t)0xD2511F53u * x, n = (uint64_t)0xCD9E8D57u * z;
    if constexpr (KEYS == DROP_PARAM) {
      k0 = a.keys[2 * i];
      k1 = a.keys[2 * i + 1];
    }
    x = (uint32_t)(n >> 32) ^ y ^ k0;
    y = (uint32_t)n;
    z = (uint32_t)(m >> 32) ^ w ^ k1;
    w = (uint32_t)m;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {x, y, z, w};
}

// Sign bits of the halves: a >= t, for two 16-bit values each.
__device__ __forceinline__ uint32_t ge_halves(uint32_t a, uint32_t t) {
  const uint32_t h = 0x80008000u;
  const uint32_t d = (a | h) - (t & ~h);  // sign: the low 15 bits of a reach t's
  return (a & ~t) | (~(a ^ t) & d);
}

static __device__ __noinline__ uint32_t drop_ties(const DropRate& r, uint64_t q,
                                                  uint32_t stream_low, U4 b) {
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
  const DropArgs none = {};
  const U4 l = drop_block<DROP_WORDS>(none, r, q, stream_low);
  const uint32_t v[4] = {l.x, l.y, l.z, l.w};
  uint32_t lost = 0u;
  for (int j = 0; j < 4; ++j) {
    if ((w[j] & 0xFFFFu) == r.hi && (v[j] & 0xFFFFu) < r.lo) lost |= 1u << (2 * j);
    if ((w[j] >> 16) == r.hi && (v[j] >> 16) < r.lo) lost |= 2u << (2 * j);
  }
  return lost;
}

// The decisions of block q: the sign bits of the halves of g[j] say whether
// the numbers 2 j and 2 j + 1 stay, so that one byte permutation spreads them
// into a mask for a pair of values.
template <int KEYS>
__device__ __forceinline__ void drop_words(const DropArgs& a, const DropRate& r, uint64_t q,
                                           uint32_t* g, uint32_t stream = STREAM_DROP,
                                           uint32_t stream_low = STREAM_DROP_LOW) {
  if (r.hi > 0xFFFFu) {
    g[0] = g[1] = g[2] = g[3] = 0u;
    return;
  }
  const U4 b = drop_block<KEYS>(a, r, q, stream);
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
  const uint32_t t = r.hi * 0x10001u;
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = ge_halves(w[j], t);
  if (r.lo != 0u) {
    // a tie is a zero half of a w ^ t, and of the least of them
    const uint32_t x = __vminu2(__vminu2(w[0] ^ t, w[1] ^ t), __vminu2(w[2] ^ t, w[3] ^ t));
    if ((x - 0x00010001u) & ~x & 0x80008000u) {
      const uint32_t lost = drop_ties(r, q, stream_low, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (lost & (1u << (2 * j))) g[j] &= ~0x8000u;
        if (lost & (2u << (2 * j))) g[j] &= ~0x80000000u;
      }
    }
  }
}

// The same as one word K: number 2 j's decision is bit 15 - j, number
// 2 j + 1's bit 31 - j, so that K << j has the pair's in the sign bits.
constexpr uint32_t KEEP_ALL = 0xF000F000u;

template <int KEYS>
__device__ __forceinline__ uint32_t drop_keep(const DropArgs& a, const DropRate& r, uint64_t q,
                                              uint32_t stream = STREAM_DROP,
                                              uint32_t stream_low = STREAM_DROP_LOW) {
  uint32_t g[4], keep = 0u;
  drop_words<KEYS>(a, r, q, g, stream, stream_low);
#pragma unroll
  for (int j = 0; j < 4; ++j) keep |= (g[j] & 0x80008000u) >> j;
  return keep;
}

// Whether channel c of the element stays (channelwise dropout).
__device__ __forceinline__ bool drop_keep_channel(const DropRate& r, int64_t c) {
  const DropArgs none = {};
  const uint32_t k = drop_keep<DROP_WORDS>(none, r, (uint64_t)c >> 3, STREAM_DROP_CHANNEL,
                                           STREAM_DROP_CHANNEL_LOW);
  const int i = (int)(c & 7);
  return (k >> ((i & 1 ? 31 : 15) - (i >> 1))) & 1u;
}

}  // namespace ba

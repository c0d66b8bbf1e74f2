// How the kernels on a network's feature maps cut a (B, C, S) tensor
// (S = H * W * D voxels) among their threads, in either memory layout, with
// the dropout bits of what a thread holds.  A dropout block is 8 consecutive
// voxels of one channel (dropout.cuh), so both layouts hand a thread whole
// blocks: 8 rows of a column of channels, or 8 voxels of a channel.
#pragma once

#include "ba_common.cuh"
#include "dropout.cuh"

namespace ba {

constexpr int FEAT_THREADS = 256;
constexpr int FEAT_WARPS = FEAT_THREADS / 32;
// channels-first: voxels of a warp tile (32 lanes x 8)
constexpr int FEAT_TILE = 256;

struct Feat {
  int64_t B, C, S;
  int64_t nblk;       // ceil(S / 8): dropout blocks of a channel
  int64_t rows;       // voxels of a chunk, below 2^31
  // counts that index divisions use are 32 bits (a 64-bit division is a call
  // of a hundred instructions, as many as a thread spends on ten accesses)
  uint32_t nchunk;    // chunks of a channel
  uint32_t colblocks; // channels-last: column blocks, of `width` channels
  int64_t width;
  int32_t ncw;        // channels-last: threads of a row (columns of VEC channels)
  int32_t vec;        // elements of a memory access
};

// Host side (feature.cu).
int device_sms();  // of the current device
// Where a kernel records a bounded wait that ran out, for ba_wait_status (of
// the current device; NULL when the first call on a device is made while
// `stream` is being captured: such a wait then ends unrecorded).
unsigned int* wait_timeouts(cudaStream_t stream);
ba_status feat_check(const char* what, int64_t B, int64_t C, int64_t H, int64_t W, int64_t D,
                     int32_t dtype, int32_t layout);
bool feat_overlap(const void* a, const void* b, size_t bytes);
// `ptrs`: every tensor of that shape the kernels touch; the access width is
// the largest that all their addresses and the inner extent allow.
Feat feat_plan(int64_t B, int64_t C, int64_t S, int32_t dtype, int32_t layout,
               const void* const* ptrs, int n_ptrs);
ba_status feat_grid(const char* what, const Feat& f, int32_t layout, dim3* grid);

// ---------------------------------------------------------------------------
// Two fp32 values in a register pair, and sm_100's packed arithmetic on them
// (one issue slot for two results, each rounded as the scalar operation).
// ---------------------------------------------------------------------------
struct F2 {
  unsigned long long v;  // kept whole, so that the pair stays in place
  __device__ __forceinline__ float x() const {
    return __uint_as_float((uint32_t)v);
  }
  __device__ __forceinline__ float y() const {
    return __uint_as_float((uint32_t)(v >> 32));
  }
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ F2 f2(float x) { return f2(x, x); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// ---------------------------------------------------------------------------
// VEC consecutive elements as they lie in memory, and pairs of them.
// ---------------------------------------------------------------------------
template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { using T = uint4; };
template <>
struct RawOf<8> { using T = uint2; };
template <>
struct RawOf<4> { using T = uint32_t; };
template <>
struct RawOf<2> { using T = uint16_t; };

template <int DT>
constexpr int ESIZE = DT == BA_BF16 ? 2 : 4;

template <int DT, int VEC>
using Raw = typename RawOf<VEC * ESIZE<DT>>::T;

// Two elements: one word of bf16, or two of fp32.
template <int DT>
using RawPair = typename RawOf<2 * ESIZE<DT>>::T;

template <int DT>
__device__ __forceinline__ F2 pair_value(RawPair<DT> p) {
  if constexpr (DT == BA_BF16)
    return f2(__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u));
  else
    return f2(__uint_as_float(p.x), __uint_as_float(p.y));
}
template <int DT>
__device__ __forceinline__ RawPair<DT> pair_raw(F2 v) {
  if constexpr (DT == BA_BF16)
    return pack_bf16x2(v.x(), v.y());
  else
    return make_uint2(__float_as_uint(v.x()), __float_as_uint(v.y()));
}

// Pair i of VEC >= 2 elements.
template <int DT, int VEC>
__device__ __forceinline__ RawPair<DT> raw_pair(const Raw<DT, VEC>& r, int i) {
  return reinterpret_cast<const RawPair<DT>*>(&r)[i];
}
template <int DT, int VEC>
__device__ __forceinline__ void raw_set_pair(Raw<DT, VEC>& r, int i, RawPair<DT> p) {
  reinterpret_cast<RawPair<DT>*>(&r)[i] = p;
}
// A pair of two single elements, and its halves.
template <int DT>
__device__ __forceinline__ RawPair<DT> raw_join(Raw<DT, 1> a, Raw<DT, 1> b) {
  if constexpr (DT == BA_BF16)
    return (uint32_t)a | (uint32_t)b << 16;
  else
    return make_uint2(a, b);
}
template <int DT>
__device__ __forceinline__ Raw<DT, 1> raw_half(RawPair<DT> p, int i) {
  if constexpr (DT == BA_BF16)
    return (uint16_t)(i ? p >> 16 : p);
  else
    return i ? p.y : p.x;
}

// prmt with sign replication: a selector of 8 | i fills its byte with the sign
// bit of byte i.
template <int SEL>
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "n"(SEL));
  return r;
}

// The pair with its dropped elements zeroed: element 0 stays if the sign bit
// of byte B0 of k0 is set, element 1 if that of byte B1 of k1 is.
template <int DT, int B0, int B1>
__device__ __forceinline__ RawPair<DT> pair_keep(RawPair<DT> p, uint32_t k0, uint32_t k1) {
  if constexpr (DT == BA_BF16) {
    return p & prmt<(8 | B0) * 0x11 | (12 | B1) * 0x1100>(k0, k1);
  } else {
    p.x &= prmt<(8 | B0) * 0x1111>(k0, 0u);
    p.y &= prmt<(8 | B1) * 0x1111>(k1, 0u);
    return p;
  }
}

// Of memory that nothing writes during the launch.
template <int DT, int VEC>
__device__ __forceinline__ Raw<DT, VEC> raw_load(const char* p) {
  return __ldg(reinterpret_cast<const Raw<DT, VEC>*>(p));
}
// Of memory that the launch may write (a result in place).
template <int DT, int VEC>
__device__ __forceinline__ Raw<DT, VEC> raw_read(const char* p) {
  return *reinterpret_cast<const Raw<DT, VEC>*>(p);
}
template <int DT, int VEC>
__device__ __forceinline__ void raw_store(char* p, const Raw<DT, VEC>& r) {
  *reinterpret_cast<Raw<DT, VEC>*>(p) = r;
}

// ===========================================================================
// Channels last.  A row is one voxel's C channels; a thread owns VEC
// consecutive channels (a column); ncw threads cover the columns of a block
// (256 of them at a time), 256 / ncw threads work down the rows, 8 at a time:
// with dropout 8 consecutive ones, the 8 voxels of one dropout block of each
// of its channels; without, every ncw-th, so that a CTA's accesses are
// contiguous.
// ===========================================================================
struct LastPlace {
  int tx, ty, nty;
  int rows;          // of the item
  int64_t b, k;      // element, item's rows are k * f.rows ..
  int64_t c;         // first channel
  int64_t c_end;     // end of the column block
  int64_t r0;
  bool on;
};

template <int VEC>
__device__ __forceinline__ LastPlace last_place(const Feat& f, uint32_t b, uint32_t k, uint32_t cb) {
  LastPlace p;
  p.tx = threadIdx.x % f.ncw;
  p.ty = threadIdx.x / f.ncw;
  p.nty = FEAT_THREADS / f.ncw;
  p.b = b;
  p.k = k;
  p.c = (int64_t)cb * f.width + p.tx * VEC;
  p.c_end = min(((int64_t)cb + 1) * f.width, f.C);
  p.r0 = (int64_t)k * f.rows;
  p.rows = (int)min(f.rows, f.S - p.r0);
  p.on = p.ty < p.nty && p.c < p.c_end;
  return p;
}

// The next FEAT_THREADS columns of a wider block.
template <int VEC>
__device__ __forceinline__ LastPlace last_next(const Feat& f, LastPlace p) {
  p.c += f.ncw * VEC;
  p.on = p.ty < p.nty && p.c < p.c_end;
  return p;
}

// Bytes from the tensor's start to the thread's columns of the item's row 0.
template <int DT>
__device__ __forceinline__ int64_t last_base(const Feat& f, const LastPlace& p) {
  return ((p.b * f.S + p.r0) * f.C + p.c) * ESIZE<DT>;
}

__device__ __forceinline__ uint64_t row_at(int r, uint32_t row_bytes) {
  return (uint64_t)(uint32_t)r * row_bytes;
}

// Keep words of VEC channels, for the 8 rows from row r of the item
// (r0 + r is a multiple of 8).
template <int VEC, int KEYS>
__device__ __forceinline__ void last_keep(const Feat& f, const DropArgs& a, const DropRate& dr,
                                          const LastPlace& p, int r, uint32_t* keep) {
  const uint64_t q = (uint64_t)(p.c * f.nblk + ((p.r0 + r) >> 3));
#pragma unroll
  for (int i = 0; i < VEC; ++i) keep[i] = drop_keep<KEYS>(a, dr, q + (uint64_t)(i * f.nblk));
}

// Pair i of row j (0 .. 7), its dropped elements zeroed.
template <int DT>
__device__ __forceinline__ RawPair<DT> last_pair_keep(RawPair<DT> p, const uint32_t* keep, int i,
                                                      int j) {
  const uint32_t k0 = keep[2 * i] << (j >> 1), k1 = keep[2 * i + 1] << (j >> 1);
  return j & 1 ? pair_keep<DT, 3, 3>(p, k0, k1) : pair_keep<DT, 1, 1>(p, k0, k1);
}

// ===========================================================================
// Channels first.  A warp takes a run of one channel's voxels in tiles of
// 256, each lane 8 voxels of a tile in accesses of VEC (8 bf16 or 4 fp32: 16
// bytes; 1 where the channel's length or an address does not allow it), each
// access of a warp contiguous.
// ===========================================================================
struct FirstPlace {
  int64_t b, c, k;   // element, channel, run
  int64_t s0;        // the run's first voxel, a multiple of 256
  int64_t base;      // elements before it
  int n;             // its voxels
  int lane;
};

// A lane's value j (0 .. 7) of a tile is the tile's voxel first_at<VEC>(j).
template <int VEC>
__device__ __forceinline__ int first_at(int lane, int j) {
  return lane * VEC + j % VEC + 32 * VEC * (j / VEC);
}

// 8 values of a lane: four pairs.
template <int DT>
struct FirstTile {
  RawPair<DT> p[4];
};

// The tile at voxel s of the run; values beyond the run are not read.
template <int DT, int VEC>
__device__ __forceinline__ void first_load(const char* x, int s, const FirstPlace& p,
                                           FirstTile<DT>& t) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int j = 0; j < 8; j += VEC) {
      const int at = s + first_at<VEC>(p.lane, j);
      if (at < p.n) {
        const Raw<DT, VEC> r = raw_read<DT, VEC>(x + (int64_t)at * ESIZE<DT>);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) t.p[j / 2 + i] = raw_pair<DT, VEC>(r, i);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const int a0 = s + first_at<1>(p.lane, j), a1 = s + first_at<1>(p.lane, j + 1);
      Raw<DT, 1> v0 = 0, v1 = 0;
      if (a0 < p.n) v0 = raw_read<DT, 1>(x + (int64_t)a0 * ESIZE<DT>);
      if (a1 < p.n) v1 = raw_read<DT, 1>(x + (int64_t)a1 * ESIZE<DT>);
      t.p[j / 2] = raw_join<DT>(v0, v1);
    }
  }
}

template <int DT, int VEC>
__device__ __forceinline__ void first_store(char* x, int s, const FirstPlace& p,
                                            const FirstTile<DT>& t) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int j = 0; j < 8; j += VEC) {
      const int at = s + first_at<VEC>(p.lane, j);
      if (at < p.n) {
        Raw<DT, VEC> r;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) raw_set_pair<DT, VEC>(r, i, t.p[j / 2 + i]);
        raw_store<DT, VEC>(x + (int64_t)at * ESIZE<DT>, r);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = s + first_at<1>(p.lane, j);
      if (at < p.n) raw_store<DT, 1>(x + (int64_t)at * ESIZE<DT>, raw_half<DT>(t.p[j / 2], j & 1));
    }
  }
}

// Keep words of a lane's values of the tile at voxel s of the run: lane l
// draws the tile's block l, and where an access is narrower than a block the
// words are handed over from the lanes that drew them.  k[j / VEC] belongs to
// the values j .. j + VEC - 1, shifted so that first_pair_keep finds them.
template <int VEC, int KEYS>
__device__ __forceinline__ void first_keep(const Feat& f, const DropArgs& a, const DropRate& dr,
                                           const FirstPlace& p, int s, uint32_t* k) {
  const uint32_t own =
      drop_keep<KEYS>(a, dr, (uint64_t)(p.c * f.nblk + ((p.s0 + s) >> 3) + p.lane));
#pragma unroll
  for (int j = 0; j < 8; j += VEC) {
    if constexpr (VEC == 8) {
      k[0] = own;
    } else {
      const int v = first_at<VEC>(p.lane, j);
      const uint32_t w = __shfl_sync(0xFFFFFFFFu, own, v >> 3);
      // a single voxel's bit goes to the sign bit of byte 3
      k[j / VEC] = w << (((v & 7) >> 1) + (VEC == 1 && !(v & 1) ? 16 : 0));
    }
  }
}

template <int DT, int VEC>
__device__ __forceinline__ RawPair<DT> first_pair_keep(RawPair<DT> p, const uint32_t* k, int i) {
  if constexpr (VEC == 1) {
    return pair_keep<DT, 3, 3>(p, k[2 * i], k[2 * i + 1]);
  } else {
    const uint32_t w = k[2 * i / VEC] << (i % (VEC / 2));
    return pair_keep<DT, 1, 3>(p, w, w);
  }
}

// A grid-wide list of runs (no units): run number `item`.
__device__ __forceinline__ bool first_place(const Feat& f, uint32_t item, FirstPlace& p) {
  p.lane = threadIdx.x % 32;
  const uint32_t row = item / f.nchunk, k = item - row * f.nchunk, b = row / (uint32_t)f.C;
  p.k = k;
  p.b = b;
  p.c = row - b * (uint32_t)f.C;
  p.s0 = k * f.rows;
  p.n = (int)min(f.rows, f.S - p.s0);
  p.base = row * f.S + p.s0;
  return b < f.B;
}

}  // namespace ba

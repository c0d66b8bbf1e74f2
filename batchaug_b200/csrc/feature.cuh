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
// channels-first: voxels of a warp tile (32 lanes x 8) and tiles of a run
constexpr int FEAT_TILE = 256;
constexpr int FEAT_RUN = 8;
// channels-last: channels of a column block, at most (256 threads x 8)
constexpr int FEAT_MAX_COLS = 2048;

struct Feat {
  int64_t B, C, S;
  int64_t nblk;       // ceil(S / 8): dropout blocks of a channel
  int64_t rows;       // voxels of a chunk
  int64_t nchunk;     // chunks of a channel
  int64_t colblocks;  // channels-last: column blocks
  int32_t ncw;        // channels-last: threads of a row (columns of VEC channels)
  int32_t vec;        // elements of a memory access
};

// Host side (feature.cu).
int device_sms();  // of the current device
ba_status feat_check(const char* what, int64_t B, int64_t C, int64_t H, int64_t W, int64_t D,
                     int32_t dtype, int32_t layout);
bool feat_overlap(const void* a, const void* b, size_t bytes);
// `ptrs`: every tensor of that shape the kernels touch; the access width is
// the largest that all their addresses and the inner extent allow.
Feat feat_plan(int64_t B, int64_t C, int64_t S, int32_t dtype, int32_t layout,
               const void* const* ptrs, int n_ptrs);
ba_status feat_grid(const char* what, const Feat& f, int32_t layout, dim3* grid);

// ---------------------------------------------------------------------------
// VEC consecutive elements as they lie in memory.
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

template <int DT, int VEC>
__device__ __forceinline__ void raw_unpack(const Raw<DT, VEC>& r, float* v) {
  if constexpr (VEC == 1) {
    if constexpr (DT == BA_BF16)
      v[0] = bf16_bits_to_f32(r);
    else
      v[0] = __uint_as_float(r);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < VEC * ESIZE<DT> / 4; ++i) {
      if constexpr (DT == BA_BF16) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        v[i] = __uint_as_float(w[i]);
      }
    }
  }
}

template <int DT, int VEC>
__device__ __forceinline__ Raw<DT, VEC> raw_pack(const float* v) {
  Raw<DT, VEC> r;
  if constexpr (VEC == 1) {
    if constexpr (DT == BA_BF16)
      r = f32_to_bf16_bits(v[0]);
    else
      r = __float_as_uint(v[0]);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < VEC * ESIZE<DT> / 4; ++i) {
      if constexpr (DT == BA_BF16)
        w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else
        w[i] = __float_as_uint(v[i]);
    }
  }
  return r;
}

template <int DT, int VEC>
__device__ __forceinline__ Raw<DT, VEC> raw_load(const void* p, int64_t i) {
  return __ldg(reinterpret_cast<const Raw<DT, VEC>*>((const char*)p + i * ESIZE<DT>));
}

template <int DT, int VEC>
__device__ __forceinline__ void raw_store(void* p, int64_t i, const Raw<DT, VEC>& r) {
  *reinterpret_cast<Raw<DT, VEC>*>((char*)p + i * ESIZE<DT>) = r;
}

// ===========================================================================
// Channels last.  A row is one voxel's C channels; a thread owns VEC
// consecutive channels (a column) and blocks of 8 consecutive rows, which are
// the 8 voxels of one dropout block of each of its channels.  ncw threads
// cover a row (or a block of FEAT_MAX_COLS channels of it), 256 / ncw threads
// work down the rows.
// ===========================================================================
struct LastPlace {
  int tx, ty, nty;
  int64_t b, k, c;       // element, chunk, first channel
  int64_t r0, r1;        // the chunk's rows
  bool on;
};

template <int VEC>
__device__ __forceinline__ LastPlace last_place(const Feat& a) {
  LastPlace p;
  p.tx = threadIdx.x % a.ncw;
  p.ty = threadIdx.x / a.ncw;
  p.nty = FEAT_THREADS / a.ncw;
  p.b = blockIdx.x / a.nchunk;
  p.k = blockIdx.x - p.b * a.nchunk;
  p.c = ((int64_t)blockIdx.y * a.ncw + p.tx) * VEC;
  p.r0 = p.k * a.rows;
  p.r1 = min(p.r0 + a.rows, a.S);
  p.on = p.ty < p.nty && p.c < a.C;
  return p;
}

// Keep bits of 8 rows (bit) by VEC channels, rows r .. r + 7, r % 8 == 0.
template <int VEC>
__device__ __forceinline__ void last_keep(const Feat& a, const DropRate& dr, int64_t c,
                                          int64_t r, uint32_t* keep) {
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    keep[i] = drop_keep8(dr, (uint64_t)((c + i) * a.nblk + (r >> 3)));
}

// ===========================================================================
// Channels first.  A warp takes a run of FEAT_RUN tiles of 256 voxels of one
// channel.  VEC > 1: a lane's 8 consecutive voxels as 16-byte vectors (one
// dropout block).  VEC == 1 (S not a multiple of 8, or unaligned tensors):
// lane l reads voxels l, l + 32, ... so the loads stay coalesced, and the
// dropout blocks, one a lane, are handed round by shuffles.
// ===========================================================================
struct FirstPlace {
  int64_t item;   // (b * C + c) * nchunk + k
  int64_t b, c, k;
  int64_t s0, s1;
  int64_t base;   // of the channel's first voxel
  int lane;
};

__device__ __forceinline__ bool first_place(const Feat& a, FirstPlace& p) {
  p.item = (int64_t)blockIdx.x * FEAT_WARPS + threadIdx.x / 32;
  p.lane = threadIdx.x % 32;
  const int64_t row = p.item / a.nchunk;
  p.k = p.item - row * a.nchunk;
  p.b = row / a.C;
  p.c = row - p.b * a.C;
  p.s0 = p.k * a.rows;
  p.s1 = min(p.s0 + a.rows, a.S);
  p.base = row * a.S;
  return row < a.B * a.C;
}

// A lane's 8 voxels of the tile at s: value j is voxel s + first_at<VEC>(j).
template <int VEC>
__device__ __forceinline__ int first_at(int lane, int j) {
  return VEC > 1 ? lane * 8 + j : lane + 32 * j;
}

template <int DT, int VEC>
struct FirstTile {
  Raw<DT, VEC> w[8 / VEC];
};

template <int DT, int VEC>
__device__ __forceinline__ void first_load(const void* x, const FirstPlace& p, int64_t s,
                                           FirstTile<DT, VEC>& t) {
#pragma unroll
  for (int j = 0; j < 8; j += VEC)
    if (s + first_at<VEC>(p.lane, j) < p.s1)
      t.w[j / VEC] = raw_load<DT, VEC>(x, p.base + s + first_at<VEC>(p.lane, j));
}

template <int DT, int VEC>
__device__ __forceinline__ void first_unpack(const FirstTile<DT, VEC>& t, float* v) {
#pragma unroll
  for (int j = 0; j < 8; j += VEC) raw_unpack<DT, VEC>(t.w[j / VEC], v + j);
}

// Keep bits of a lane's 8 voxels of the tile at s (bit j for value j).
template <int VEC>
__device__ __forceinline__ uint32_t first_keep(const Feat& a, const DropRate& dr,
                                               const FirstPlace& p, int64_t s) {
  const uint32_t own = drop_keep8(dr, (uint64_t)(p.c * a.nblk + (s >> 3) + p.lane));
  if constexpr (VEC > 1) return own;
  uint32_t keep = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t m = __shfl_sync(0xFFFFFFFFu, own, 4 * j + (p.lane >> 3));
    keep |= ((m >> (p.lane & 7)) & 1u) << j;
  }
  return keep;
}

}  // namespace ba

// ba_dropout: one read and one write of the tensor, the mask drawn from the
// counter as it goes (dropout.cuh).
#include "feature.cuh"

namespace ba {
namespace {

struct DropoutArgs {
  const void* src;
  void* dst;
  Feat f;
  DropArgs drop;
  int32_t channelwise;
};

// 8 rows of the thread's columns a pass, each channel's bits from one block, so
// that a block's eight decisions stay in the thread that drew them.  2x64x64^3
// bf16 at p = 0.1: 33 us, 4.1 TB/s of 6.5; the integer units bind (a block is 60
// operations for 8 values): ALU 59 % and issue slots 68 % busy.  The bound of three
// CTAs an SM (80 registers) costs 44 bytes of spill stores there.
template <int DT, int VEC, int KEYS>
__global__ void __launch_bounds__(FEAT_THREADS, 3)
    dropout_last(const __grid_constant__ DropoutArgs a) {
  const uint32_t b = blockIdx.x / a.f.nchunk;
  const LastPlace p = last_place<VEC>(a.f, b, blockIdx.x - b * a.f.nchunk, blockIdx.y);
  if (!p.on) return;
  const DropRate dr = drop_rate(a.drop, p.b);
  const int64_t base = last_base<DT>(a.f, p);
  const char* src = (const char*)a.src + base;
  char* dst = (char*)a.dst + base;
  const uint32_t row = (uint32_t)a.f.C * ESIZE<DT>;
  const F2 scale = f2(dr.scale);
  uint32_t keep[VEC];
  if (a.channelwise) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) keep[i] = drop_keep_channel(dr, p.c + i) ? KEEP_ALL : 0u;
  }
  for (int r = p.ty * 8; r < p.rows; r += p.nty * 8) {
    Raw<DT, VEC> x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (r + j < p.rows) x[j] = raw_read<DT, VEC>(src + row_at(r + j, row));
    if (!a.channelwise) last_keep<VEC, KEYS>(a.f, a.drop, dr, p, r, keep);
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i)
          raw_set_pair<DT, VEC>(
              x[j], i,
              last_pair_keep<DT>(
                  pair_raw<DT>(mul2(pair_value<DT>(raw_pair<DT, VEC>(x[j], i)), scale)), keep, i,
                  j));
        if (r + j < p.rows) raw_store<DT, VEC>(dst + row_at(r + j, row), x[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const uint32_t k = keep[0] << (j >> 1);
        const RawPair<DT> y = pair_keep<DT, 1, 3>(
            pair_raw<DT>(mul2(pair_value<DT>(raw_join<DT>(x[j], x[j + 1])), scale)), k, k);
        if (r + j < p.rows) raw_store<DT, 1>(dst + row_at(r + j, row), raw_half<DT>(y, 0));
        if (r + j + 1 < p.rows) raw_store<DT, 1>(dst + row_at(r + j + 1, row), raw_half<DT>(y, 1));
      }
    }
  }
}

// A warp a run of a channel, four tiles of 256 voxels in flight; a lane's 16
// bytes of bf16 are one dropout block (fp32: words handed over between lanes).
// 16x4x128^3 bf16, a rate for each element: 107 us, 5.0 TB/s, the integer units
// 66 % busy (87 operations for 8 values, where HBM leaves time for 89).
// 2x3x91x109x91 fp32, where no vector width divides a channel: 11.9 us, 3.6 TB/s
// (bf16 there takes 174 registers, one CTA an SM).
template <int DT, int VEC, int KEYS>
__global__ void __launch_bounds__(FEAT_THREADS)
    dropout_first(const __grid_constant__ DropoutArgs a) {
  FirstPlace p;
  if (!first_place(a.f, blockIdx.x * FEAT_WARPS + threadIdx.x / 32, p)) return;
  const DropRate dr = drop_rate(a.drop, p.b);
  constexpr int FLIGHT = 4;
  const char* src = (const char*)a.src + p.base * ESIZE<DT>;
  char* dst = (char*)a.dst + p.base * ESIZE<DT>;
  const F2 scale = f2(dr.scale);
  uint32_t row = 0u;
  if (a.channelwise) row = drop_keep_channel(dr, p.c) ? 0xFFFFFFFFu : 0u;
  for (int s = 0; s < p.n; s += FEAT_TILE * FLIGHT) {
    FirstTile<DT> t[FLIGHT];
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) first_load<DT, VEC>(src, s + u * FEAT_TILE, p, t[u]);
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const int su = s + u * FEAT_TILE;
      if (su < p.n) {
        // a block of its own (four words), or handed-over keep words
        uint32_t keep[VEC == 8 ? 4 : 8 / VEC];
        if (a.channelwise) {
#pragma unroll
          for (int i = 0; i < (VEC == 8 ? 4 : 8 / VEC); ++i) keep[i] = row;
        } else if constexpr (VEC == 8) {
          drop_words<KEYS>(a.drop, dr,
                           (uint64_t)(p.c * a.f.nblk + ((p.s0 + su) >> 3) + p.lane), keep);
        } else {
          first_keep<VEC, KEYS>(a.f, a.drop, dr, p, su, keep);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const RawPair<DT> y = pair_raw<DT>(mul2(pair_value<DT>(t[u].p[i]), scale));
          if constexpr (VEC == 8)
            t[u].p[i] = pair_keep<DT, 1, 3>(y, keep[i], keep[i]);
          else
            t[u].p[i] = first_pair_keep<DT, VEC>(y, keep, i);
        }
        first_store<DT, VEC>(dst, su, p, t[u]);
      }
    }
  }
}

template <int DT, int VEC, int KEYS>
void launch_keys(const DropoutArgs& a, bool last, dim3 grid, cudaStream_t st) {
  if (last)
    dropout_last<DT, VEC, KEYS><<<grid, FEAT_THREADS, 0, st>>>(a);
  else if constexpr (DT == BA_F32 || VEC != 4)
    dropout_first<DT, VEC, KEYS><<<grid, FEAT_THREADS, 0, st>>>(a);
}

template <int DT, int VEC>
void launch(const DropoutArgs& a, bool last, dim3 grid, cudaStream_t st) {
  if (a.drop.seed_dev == nullptr)
    launch_keys<DT, VEC, DROP_PARAM>(a, last, grid, st);
  else
    launch_keys<DT, VEC, DROP_WORDS>(a, last, grid, st);
}

}  // namespace
}  // namespace ba

extern "C" ba_status ba_dropout(const ba_dropout_desc* desc, ba_stream_t stream) {
  using namespace ba;
  clear_error();
  BA_REQUIRE(desc != nullptr, "ba_dropout: desc is NULL");
  const ba_dropout_desc& d = *desc;
  ba_status st = feat_check("ba_dropout", d.batch, d.channels, d.H, d.W, d.D, d.dtype, d.layout);
  if (st != BA_OK) return st;
  BA_REQUIRE((d.flags & ~(BA_DROPOUT_CHANNEL | BA_DROPOUT_RESCALE)) == 0,
             "ba_dropout: unknown flags 0x%x", d.flags);
  BA_REQUIRE(d.p_elem != nullptr || (d.p >= 0.0f && d.p <= 1.0f),
             "ba_dropout: p=%g not in [0, 1]", (double)d.p);
  const int64_t S = d.H * d.W * d.D;
  if (d.batch * d.channels * S == 0) return BA_OK;
  const size_t esz = d.dtype == BA_BF16 ? 2 : 4;
  const size_t bytes = (size_t)(d.batch * d.channels * S) * esz;
  BA_REQUIRE(d.src && d.dst, "ba_dropout: NULL src or dst");
  BA_REQUIRE((uintptr_t)d.src % esz == 0 && (uintptr_t)d.dst % esz == 0,
             "ba_dropout: pointers not aligned to the element size");
  BA_REQUIRE((uintptr_t)d.p_elem % 4 == 0 && (uintptr_t)d.seed_dev % 8 == 0,
             "ba_dropout: p_elem or seed_dev not aligned");
  BA_REQUIRE(d.src == d.dst || !feat_overlap(d.src, d.dst, bytes),
             "ba_dropout: dst partially overlaps src");
  DropoutArgs a;
  a.src = d.src;
  a.dst = d.dst;
  const void* ptrs[2] = {d.src, d.dst};
  a.f = feat_plan(d.batch, d.channels, S, d.dtype, d.layout, ptrs, 2);
  a.drop = {d.p, d.p_elem, d.mask, (uint32_t)d.seed, (uint32_t)(d.seed >> 32), d.seed_dev,
            d.elem_offset, (d.flags & BA_DROPOUT_RESCALE) ? 1 : 0};
  drop_keys(a.drop);
  a.channelwise = (d.flags & BA_DROPOUT_CHANNEL) ? 1 : 0;
  dim3 grid;
  st = feat_grid("ba_dropout", a.f, d.layout, &grid);
  if (st != BA_OK) return st;
  const bool last = d.layout == BA_CHANNELS_LAST;
  cudaStream_t cs = (cudaStream_t)stream;
  if (d.dtype == BA_BF16) {
    if (a.f.vec == 8)
      launch<BA_BF16, 8>(a, last, grid, cs);
    else if (a.f.vec == 4)
      launch<BA_BF16, 4>(a, last, grid, cs);
    else
      launch<BA_BF16, 1>(a, last, grid, cs);
  } else {
    if (a.f.vec == 4)
      launch<BA_F32, 4>(a, last, grid, cs);
    else
      launch<BA_F32, 1>(a, last, grid, cs);
  }
  return check_launch("ba_dropout");
}

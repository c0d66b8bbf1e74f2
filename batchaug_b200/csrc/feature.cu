// Host side of feature.cuh: checks and the cut of a feature map into chunks.
#include "feature.cuh"

#include <algorithm>

namespace ba {

int device_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 0;
    cached[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
                          n > 0
                      ? n
                      : 148;
  }
  return cached[dev];
}

ba_status feat_check(const char* what, int64_t B, int64_t C, int64_t H, int64_t W, int64_t D,
                     int32_t dtype, int32_t layout) {
  BA_REQUIRE(dtype == BA_F32 || dtype == BA_BF16, "%s: bad dtype %d", what, dtype);
  BA_REQUIRE(layout == BA_CHANNELS_FIRST || layout == BA_CHANNELS_LAST, "%s: bad layout %d", what,
             layout);
  BA_REQUIRE(B >= 0 && C >= 0 && H >= 0 && W >= 0 && D >= 0, "%s: negative size", what);
  // every index is computed in 64 bits; the product must not wrap
  int64_t n = 1;
  const int64_t dims[5] = {B, C, H, W, D};
  for (int i = 0; i < 5; ++i)
    if (dims[i] == 0) return BA_OK;
  for (int i = 0; i < 5; ++i) {
    BA_REQUIRE(dims[i] <= ((int64_t)1 << 40) / n, "%s: more than 2^40 values", what);
    n *= dims[i];
  }
  // the dropout blocks of an element are counted in 48 bits
  BA_REQUIRE(B < ((int64_t)1 << 31), "%s: batch exceeds 2^31 - 1", what);
  // a row's bytes are a 32-bit stride
  BA_REQUIRE(C < ((int64_t)1 << 29), "%s: channels exceed 2^29 - 1", what);
  return BA_OK;
}

bool feat_overlap(const void* a, const void* b, size_t bytes) {
  const char *p = (const char*)a, *q = (const char*)b;
  return !(p + bytes <= q || q + bytes <= p);
}

Feat feat_plan(int64_t B, int64_t C, int64_t S, int32_t dtype, int32_t layout,
               const void* const* ptrs, int n_ptrs) {
  Feat f;
  f.B = B;
  f.C = C;
  f.S = S;
  f.nblk = (S + 7) / 8;
  f.colblocks = 1;
  f.ncw = 1;
  f.width = C;
  const int esz = dtype == BA_BF16 ? 2 : 4;
  const bool last = layout == BA_CHANNELS_LAST;
  const int64_t inner = last ? C : S;
  auto fits = [&](int vec) {
    if (inner % vec != 0) return false;
    for (int i = 0; i < n_ptrs; ++i)
      if ((uintptr_t)ptrs[i] % (size_t)(vec * esz) != 0) return false;
    return true;
  };
  f.vec = fits(16 / esz) ? 16 / esz : (last && dtype == BA_BF16 && fits(4)) ? 4 : 1;
  if (last) {
    const int64_t ncol = C / f.vec;
    f.ncw = (int32_t)std::min<int64_t>(ncol, FEAT_THREADS);
    f.width = (int64_t)f.ncw * f.vec;
    f.colblocks = (uint32_t)((ncol + f.ncw - 1) / f.ncw);
    // a pass of the CTA over 8 rows a thread, repeated while there are
    // several times as many chunks as SMs
    const int64_t unit = (int64_t)(FEAT_THREADS / f.ncw) * 8;
    const int64_t units = (S + unit - 1) / unit * B * f.colblocks;
    const int64_t reps = std::min<int64_t>(8, std::max<int64_t>(1, units / (device_sms() * 16)));
    f.rows = unit * reps;
  } else {
    // 4 to 16 tiles a warp: what a warp sets up once is worth two of them
    const int64_t tiles = (S + FEAT_TILE - 1) / FEAT_TILE * B * C;
    const int64_t run = tiles / ((int64_t)device_sms() * 4 * FEAT_WARPS * 4);
    f.rows = (int64_t)FEAT_TILE * std::min<int64_t>(16, std::max<int64_t>(4, run / 4 * 4));
  }
  f.nchunk = (uint32_t)((S + f.rows - 1) / f.rows);
  return f;
}

ba_status feat_grid(const char* what, const Feat& f, int32_t layout, dim3* grid) {
  const int64_t items = f.B * (layout == BA_CHANNELS_LAST ? 1 : f.C) * (int64_t)f.nchunk;
  const int64_t x =
      layout == BA_CHANNELS_LAST ? items : (items + FEAT_WARPS - 1) / FEAT_WARPS;
  const int64_t y = layout == BA_CHANNELS_LAST ? f.colblocks : 1;
  if (x > 0x7FFFFFFF || y > 65535 || items > 0xFFFFFFFF - FEAT_WARPS) {
    set_error("%s: tensor too large for one launch", what);
    return BA_EUNSUPPORTED;
  }
  *grid = dim3((unsigned)x, (unsigned)y);
  return BA_OK;
}

}  // namespace ba

// ba_norm_forward / ba_norm_backward: checks, the schedule, the launch.
#include <string.h>

#include <algorithm>

#include "norm_launch.cuh"

namespace ba {
namespace {

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

// Inputs of the sets' waves together: 32 units of 8 MB took 135 us with waves
// of 36 MB, 127 at 48, 124 at 72 and at 108, and 2x32x64^3 fp32 forward 40, 40,
// 35 and 35 us.  L2 (126 MB, each of the two dies with lines of its own) keeps
// about 32 MB of them from the sums to the results, with the outputs' lines
// beside them, and larger waves read the rest again; but every wave waits once
// and sums its threads' parts once, and that costs more than the reads.
constexpr int64_t NORM_WAVE_BYTES = (int64_t)72 << 20;
constexpr int64_t NORM_L2_BYTES = (int64_t)36 << 20;
constexpr int NORM_MAX_SMEM = 227 << 10;

// The kernel of a call, and how many of its CTAs the device holds at once.
NormKernel norm_kernel_of(const NormKind& k, int32_t dtype, int32_t layout) {
  const bool last = layout == BA_CHANNELS_LAST;
  return dtype == BA_BF16 ? (last ? norm_kernel_bf16_last(k) : norm_kernel_bf16_first(k))
                          : (last ? norm_kernel_f32_last(k) : norm_kernel_f32_first(k));
}

// Shared memory of a CTA: norm_kernel's layout.
size_t norm_smem(const NormArgs& a, bool last, int32_t dtype, bool backward) {
  const Feat& f = a.f;
  const size_t bytes = (size_t)f.vec * (dtype == BA_BF16 ? 2 : 4);
  const size_t ring = f.vec == 1 ? 0 : FEAT_THREADS * bytes * 8 * (backward ? 2 : 1);
  const size_t cw = (size_t)f.ncw * f.vec;
  size_t n = std::max<size_t>(FEAT_THREADS, cw) * sizeof(double2) +
             (size_t)a.ugroups * (2 * sizeof(double2) + sizeof(GroupStat)) + 2 * sizeof(Piece) +
             ring;
  if (last)
    n += ((cw + 3) / 4 * 4 + std::max(5 * cw, (size_t)2 * FEAT_THREADS * f.vec)) * sizeof(float);
  return n;
}

// CTAs of the kernel that an SM holds; also lifts its shared memory limit.
int norm_occupancy(NormKernel fn, const NormKind& k, int32_t dtype, int32_t layout, size_t smem) {
  // an idempotent cache: threads that fill an entry together write the same
  static int cached[64][2][2][3][4][3][2];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  int& c = cached[dev][dtype][layout][k.vec == 1 ? 0 : k.vec == 4 ? 1 : 2][k.act][k.drop]
                 [k.backward];
  if (c == 0) {
    int held = 0;
    if (cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             NORM_MAX_SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, fn, FEAT_THREADS, 0) != cudaSuccess ||
        held < 1) {
      cudaGetLastError();
      return 1;
    }
    c = held;
  }
  // 227 KB a CTA at most and 228 KB an SM, 1 KB of it a CTA's own; three rings
  // cover the memory's latency, and a fourth CTA only adds partials (32 units
  // of 8 MB: 153 us, with four 163)
  return std::min<int>(std::min(c, 3), std::max<int>(1, (int)(((size_t)228 << 10) / (smem + 1024))));
}

// Column blocks (channels last): whole groups, whole columns, and at least 128
// bytes of a row, so that a block's accesses fill their lines.
void norm_columns(NormArgs& a, int32_t dtype) {
  Feat& f = a.f;
  // the least run of channels that is both
  int64_t x = a.Cg, y = f.vec;
  while (y != 0) {
    const int64_t t = x % y;
    x = y;
    y = t;
  }
  const int64_t least = a.Cg / x * f.vec, line = 128 / (dtype == BA_BF16 ? 2 : 4);
  // blocks of m such runs, m a divisor of their number, one to four lines
  // wide if there is such an m; otherwise one block, unless it has so many
  // groups that their sums would fill the shared memory
  const int64_t runs = f.C / least, want = (line + least - 1) / least;
  int64_t m = want;
  while (m < runs && m <= 4 * want && runs % m != 0) ++m;
  if (m > 4 * want && m < runs) m = f.C / a.Cg <= 1024 ? runs : 1;
  m = std::min(m, runs);
  f.width = m * least;
  f.colblocks = (uint32_t)(runs / m);
  f.ncw = (int32_t)std::min<int64_t>(f.width / f.vec, FEAT_THREADS);
  a.ugroups = (uint32_t)(f.width / a.Cg);
}

// The parameters' gradients after a launch of clusters, whose CTAs need not
// all be resident and so cannot wait for each other's sums.
template <bool LAST>
__global__ void __launch_bounds__(FEAT_THREADS)
    norm_param_kernel(const __grid_constant__ NormArgs a) {
  __shared__ double2 meet[FEAT_THREADS];
  norm_param_grads<LAST>(a, meet);
}

// Units of at most so many bytes are clusters of up to eight CTAs: as many as a
// unit has of those that are resident at once, none where that is below one;
// channels first, one for eight channels at least, so that groups of many channels
// may need more than are resident, in rounds.  bf16 with silu, forward / backward
// in us, clusters and waiting launches:
//   2x64x8^3 last           9.0 / 14.1   12.3 / 18.0
//   2x64x12^3 last          9.1 / 14.5   12.2 / 16.5   (216 KB)
//   16x64x16^3 first        9.8 / 13.3   11.1 / 13.4   (64 KB, 128 units)
//   16x64x12^3 first        9.7 / 12.5   10.5 / 12.8   (27 KB; clusters of eight, in
//                                                      three rounds: 24.6 / 34.9)
//   8x512x8^3, 32, first   13.8 / 21.9   17.0 / 21.5   (512 CTAs in clusters of two)
//   16x512x8^3, 8, first   23.8 / 39.9   24.1 / 38.5   (1024 in clusters of eight)
//   2x64x16^3 last         11.3 / 14.1   10.0 / 14.2   (512 KB)
//   16x64x16^3 last        14.9 / 18.2   12.9 / 18.0   (512 KB)
// and a cluster call is 2 us shorter on the host, so at 512 KB they are even.
constexpr int64_t NORM_CLUSTER_BYTES = (int64_t)512 << 10;
constexpr int NORM_CLUSTER = 8;

// The items of a unit whose channels' voxels are cut into `parts`.
void norm_cut(NormArgs& a, bool last, int64_t parts) {
  Feat& f = a.f;
  const int64_t grain = last ? 8 : FEAT_TILE;  // voxels: whole dropout blocks, whole tiles
  const int64_t least = last ? (int64_t)(FEAT_THREADS / f.ncw) * 8 : FEAT_TILE;
  parts = std::min(std::max<int64_t>(1, parts), (f.S + least - 1) / least);
  f.rows = ((f.S + parts - 1) / parts + grain - 1) / grain * grain;
  f.nchunk = (uint32_t)((f.S + f.rows - 1) / f.rows);
  a.items = (uint32_t)(last ? f.nchunk : ((int64_t)a.Cg * f.nchunk + FEAT_WARPS - 1) / FEAT_WARPS);
}

// Cuts the work for `ctas` resident CTAs: waves of units, items of a unit.
void norm_schedule(NormArgs& a, const ba_norm_desc& d, bool backward, int64_t ctas) {
  Feat& f = a.f;
  const bool last = d.layout == BA_CHANNELS_LAST;
  const int64_t units = last ? f.B * f.colblocks : f.B * a.G;
  a.units = (uint32_t)units;
  const int64_t unit_bytes = f.S * (last ? f.width : a.Cg) * (d.dtype == BA_BF16 ? 2 : 4) *
                             (backward ? 2 : 1);
  const int64_t rows_of_unit = last ? 1 : a.Cg;
  const int64_t share = std::min<int64_t>(NORM_CLUSTER, ctas / units);
  if (unit_bytes <= NORM_CLUSTER_BYTES && share >= 1) {
    norm_cut(a, last, last ? share : share * FEAT_WARPS / rows_of_unit);
    a.cluster = a.items <= NORM_CLUSTER;
  }
  if (a.cluster) {
    a.sets = 1;
    a.wave = (uint32_t)units;
    a.reverse = 0;
  } else {
    // two sets of CTAs, so that one streams while the other waits (one set:
    // 2x64x64^3 bf16 backward 86 us, not 65; 2x32x128^3 bf16 157 and 246 us, not 146
    // and 233; four sets of smaller waves were no better)
    const int64_t sets = std::min<int64_t>(units, std::min<int64_t>(2, ctas / device_sms()));
    int64_t wave = std::min((units + sets - 1) / sets,
                            std::max<int64_t>(1, NORM_WAVE_BYTES / unit_bytes / sets));
    const int64_t waves = (units + wave * sets - 1) / (wave * sets) * sets;
    wave = (units + waves - 1) / waves;
    a.sets = (uint32_t)sets;
    a.wave = (uint32_t)wave;
    a.reverse = sets * wave * unit_bytes > NORM_L2_BYTES;
    // parts of a channel's voxels, so that a whole wave has one item for each CTA
    const int64_t workers = ctas / sets * (last ? 1 : FEAT_WARPS);
    norm_cut(a, last, workers / (wave * rows_of_unit));
  }
  // pieces of the results (norm.cuh)
  const bool whole = a.cluster || last;
  a.sub_rows = whole ? f.rows : std::min<int64_t>(f.rows, NORM_PIECE * 256 * f.vec);
  a.subs = (uint32_t)((f.rows + a.sub_rows - 1) / a.sub_rows);
}

struct NormScratch {
  size_t done, ticket, part, chan, total;  // byte offsets; up to chan: zeroed
};

NormScratch norm_scratch(const NormArgs& a, bool backward) {
  NormScratch s;
  s.done = 0;
  s.ticket = 16;
  s.part = s.ticket + (a.subs > 1 ? align16(a.units * sizeof(uint32_t)) : 0);
  s.chan = s.part + (size_t)a.units * a.items * a.ugroups * sizeof(float4);
  s.total = s.chan +
            (backward ? align16((size_t)(a.f.B * a.f.C * a.f.nchunk) * sizeof(float2)) : 0);
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

// Everything of a call that its sizes, types and addresses decide.
struct NormCall {
  NormArgs a;
  NormKernel fn;
  NormScratch scratch;
  size_t smem;
  int64_t ctas;
};

void norm_plan(const ba_norm_desc& d, bool backward, NormCall& c) {
  NormArgs& a = c.a;
  memset(&a, 0, sizeof(a));
  const void* ptrs[3] = {d.x, d.out, d.dy};
  a.f = feat_plan(d.batch, d.channels, d.H * d.W * d.D, d.dtype, d.layout, ptrs,
                  backward ? 3 : 2);
  a.G = (uint32_t)d.groups;
  a.Cg = (uint32_t)(d.channels / d.groups);
  NormKind k;
  k.vec = a.f.vec;
  k.act = d.activation == BA_ACT_NONE   ? ACT_NONE
          : d.activation == BA_ACT_SILU ? ACT_SILU
          : d.activation == BA_ACT_GELU ? ACT_GELU
                                        : ACT_LEAKY;
  k.drop = d.p_elem == nullptr && d.p <= 0.0f ? DROP_NONE
           : d.seed_dev == nullptr            ? DROP_PARAM
                                              : DROP_WORDS;
  k.backward = backward;
  c.fn = norm_kernel_of(k, d.dtype, d.layout);
  const bool last = d.layout == BA_CHANNELS_LAST;
  if (last)
    norm_columns(a, d.dtype);
  else
    a.ugroups = 1;
  c.smem = norm_smem(a, last, d.dtype, backward);
  c.ctas = (int64_t)norm_occupancy(c.fn, k, d.dtype, d.layout, c.smem) * device_sms();
  norm_schedule(a, d, backward, c.ctas);
  c.scratch = norm_scratch(a, backward);
  a.inv_n = 1.0 / ((double)a.Cg * (double)a.f.S);
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
  NormCall c;
  norm_plan(d, backward, c);
  NormArgs& a = c.a;
  const NormScratch& sc = c.scratch;
  // counts are 32 bits: an item's rows, a partial's values, the items of a launch;
  // so are the bytes between a thread's rows (channels last)
  const double row_step = d.layout == BA_CHANNELS_LAST
                              ? (double)(FEAT_THREADS / a.f.ncw) * (double)d.channels * (double)esz
                              : 0.0;
  const double part_values =
      (double)a.f.rows * (double)(d.layout == BA_CHANNELS_LAST ? a.Cg : (uint32_t)FEAT_WARPS);
  if (a.f.rows >= ((int64_t)1 << 31) || part_values >= 4294967296.0 ||
      (double)a.units * (double)a.items * FEAT_WARPS >= 4294967296.0 ||
      (double)a.items * (double)a.subs >= 2147483648.0 ||
      (double)a.f.B * (double)a.f.nchunk >= 4294967296.0 || row_step >= 4294967296.0 ||
      c.smem > (size_t)NORM_MAX_SMEM) {
    set_error("%s: tensor too large for one launch", what);
    return BA_EUNSUPPORTED;
  }
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
  a.done = (uint32_t*)((char*)workspace + sc.done);
  a.ticket = (uint32_t*)((char*)workspace + sc.ticket);
  a.part = (float4*)((char*)workspace + sc.part);
  a.chan = d.dweight || d.dbias ? (float2*)((char*)workspace + sc.chan) : nullptr;
  a.timeouts = wait_timeouts(cs);
  a.eps = d.eps;
  a.slope = d.activation == BA_ACT_LEAKY_RELU ? d.slope : 0.0f;
  a.drop = {d.p, d.p_elem, nullptr, (uint32_t)d.seed, (uint32_t)(d.seed >> 32), d.seed_dev,
            d.elem_offset, 1};
  drop_keys(a.drop);
  void* args[1] = {&a};
  if (a.cluster) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = a.items;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(a.units * a.items);
    cfg.blockDim = dim3(FEAT_THREADS);
    cfg.dynamicSmemBytes = c.smem;
    cfg.stream = cs;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelExC(&cfg, (const void*)c.fn, args);
    if ((st = check_launch(what)) != BA_OK || a.chan == nullptr) return st;
    const unsigned grid = (unsigned)std::min<int64_t>((a.f.C + 7) / 8, 65536);
    if (d.layout == BA_CHANNELS_LAST)
      norm_param_kernel<true><<<grid, FEAT_THREADS, 0, cs>>>(a);
    else
      norm_param_kernel<false><<<grid, FEAT_THREADS, 0, cs>>>(a);
    return check_launch(what);
  }
  if (cudaMemsetAsync(workspace, 0, sc.chan, cs) != cudaSuccess) {
    set_error("%s: clearing the scratch failed: %s", what, cudaGetErrorString(cudaGetLastError()));
    return BA_ECUDA;
  }
  const unsigned grid =
      (unsigned)(a.sets * std::min<int64_t>(c.ctas / a.sets, (int64_t)a.wave * a.items));
  cudaLaunchCooperativeKernel((const void*)c.fn, dim3(grid), dim3(FEAT_THREADS), args, c.smem, cs);
  return check_launch(what);
}

}  // namespace
}  // namespace ba

extern "C" size_t ba_norm_workspace_bytes(const ba_norm_desc* desc, int32_t backward) {
  using namespace ba;
  clear_error();
  if (norm_check("ba_norm_workspace_bytes", desc) != BA_OK) return 0;
  if (desc->batch * desc->channels * desc->H * desc->W * desc->D == 0) return 0;
  NormCall c;
  norm_plan(*desc, backward != 0, c);
  return c.scratch.total;
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

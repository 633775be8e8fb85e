// Planning and launches of the group norm (kernels: groupnorm_2d.cuh), and the sum of its per-image
// weight and bias gradients.
#include <cuda_runtime.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <exception>
#include <limits>
#include <map>
#include <mutex>
#include <numeric>
#include <set>
#include <string>
#include <utility>

#include "cluster.cuh"
#include "groupnorm_2d.h"
#include "ptx.cuh"
#include "../../include/spio_b200.h"

namespace spio_b200 {

int jit_fail(const std::string& msg);  // sets the thread's last-error text, returns 1
bool gw8_pdl_enabled();

namespace {

// dweight[c] / dbias[c] = sums of rows of 2 * c values, in a fixed order: a CTA owns 32 columns, its warps take every
// 32nd row (128-byte rows, coalesced) and are added through shared memory.  Many rows are shared out among the `split`
// CTAs of a cluster.  Bound by the latency of a warp's loads, sixteen at a time: the rows of 4096 images of 64 channels are
// one batch with eight CTAs for 32 columns, eight with one, which takes the backward pass at 7 x 7 pixels from
// 52 to 42 us.
template <bool SPLIT>
__global__ void __launch_bounds__(1024)
groupnorm_2d_bwd_reduce_kernel(float* __restrict__ dweight, float* __restrict__ dbias,
                               const float* __restrict__ part, int c, int rows, int split) {
  __shared__ float sums[32][33];
  __shared__ float total[32];
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (!SPLIT) split = 1;
  const int block = SPLIT ? blockIdx.x / split : blockIdx.x, rank = blockIdx.x - block * split;
  const int col = block * 32 + lane;
  float s = 0.f;
  if (col < 2 * c) {
    const int first = rank * 32 + warp, step = 32 * split;
    const float* at = part + (long long)first * 2 * c + col;
    const long long stride = (long long)step * 2 * c;
    int n = first < rows ? (rows - first - 1) / step + 1 : 0;
    for (; n >= 16; n -= 16, at += 16 * stride) {
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = __ldcg(at + j * stride);
#pragma unroll
      for (int j = 0; j < 16; ++j) s += v[j];
    }
    for (; n > 0; n -= 8, at += 8 * stride) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? __ldcg(at + j * stride) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
  }
  sums[warp][lane] = s;
  __syncthreads();
  s = sums[lane][warp];  // column `warp` of the 32, its warps' sums over the lanes
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (SPLIT) {
    if (lane == 0) total[warp] = s;
    cluster_arrive();
    cluster_wait();
    if (rank == 0) {
      s = lane < split ? cluster_load(total + warp, lane) : 0.f;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    }
    // (the first has read the others' sums, which are there until it has arrived)
    if (rank == 0) cluster_arrive();
    else cluster_arrive_relaxed();
  }
  const int out = block * 32 + warp;
  if (rank == 0 && lane == 0 && out < 2 * c) {
    if (out < c) {
      if (dweight != nullptr) dweight[out] = s;
    } else if (dbias != nullptr) {
      dbias[out - c] = s;
    }
  }
  if (SPLIT) cluster_wait();
}

struct Plan {
  GnGeom g;
  unsigned grid;
  bool one_launch;       // of clusters, else two kernels
  int threads;           // of a CTA
  int smem, slots;       // dynamic shared memory, slots of the ring
  long long rows;        // of the backward pass's partial sums
  size_t stats_bytes;    // forward, two kernels: parts' statistics
  size_t channel_bytes;  // backward: parts' sums for the channels
  size_t group_bytes;    // backward, two kernels: parts' sums for the groups
};

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

#define SPIO_CUDA(call)                                                                        \
  do {                                                                                         \
    const cudaError_t e_ = (call);                                                             \
    if (e_ != cudaSuccess) return jit_fail(std::string("CUDA error: ") + cudaGetErrorString(e_)); \
  } while (0)

struct Device {
  int sms, smem;  // multiprocessors, shared memory a block may have
  int ordinal;
};

int device_of(Device* d) {
  if (cudaGetDevice(&d->ordinal) != cudaSuccess ||
      cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, d->ordinal) != cudaSuccess ||
      cudaDeviceGetAttribute(&d->smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, d->ordinal) != cudaSuccess)
    return jit_fail("CUDA error: no device");
  return 0;
}

// Lets a kernel have more than 48 KB of shared memory and clusters of more than 8 CTAs.  The limits belong to the kernel
// and the device, for all host threads: they are raised as far as they go, once, and never lowered to what one launch
// needs, because a launch of another thread may be on its way that needs more.
int allow(const void* func, const Device& dev) {
  static std::mutex mutex;
  static std::set<std::pair<const void*, int>> raised;
  try {
    std::lock_guard<std::mutex> lock(mutex);
    if (raised.count({func, dev.ordinal})) return 0;
    cudaFuncAttributes attr;
    SPIO_CUDA(cudaFuncGetAttributes(&attr, func));
    SPIO_CUDA(cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, dev.smem - (int)attr.sharedSizeBytes));
    SPIO_CUDA(cudaFuncSetAttribute(func, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    raised.insert({func, dev.ordinal});
  } catch (const std::exception& e) {  // no memory; C callers get an error like any other
    return jit_fail(std::string("GroupNorm2d: ") + e.what());
  }
  return 0;
}

int check_desc(const spio_groupnorm_2d_desc* d) {
  if (d == nullptr) return jit_fail("desc is NULL");
  if (d->n < 0 || d->pixels < 0) return jit_fail("n and pixels must not be negative");
  if (d->c <= 0 || d->c % 8 != 0) return jit_fail("Number of channels must be a multiple of 8.");
  if (d->c > (1 << 20)) return jit_fail("GroupNorm2d supports at most 2^20 channels");
  if (d->groups <= 0 || d->c % d->groups != 0) return jit_fail("Number of channels must be divisible by the number of groups.");
  if (d->pixels > (1ll << 30)) return jit_fail("GroupNorm2d supports at most 2^30 pixels an image");
  if (d->n > (1ll << 30)) return jit_fail("GroupNorm2d supports at most 2^30 images");
  if (d->activation < 0 || d->activation >= kActs) return jit_fail("unknown activation");
  if (d->type < 0 || d->type > 2) return jit_fail("GroupNorm2d: unknown data type");
  const int cpg = d->c / d->groups;
  if (std::lcm(cpg, 8) > kGnWide * 8)
    return jit_fail("GroupNorm2d: groups (rounded up to whole blocks of 8 channels) may span at most 2048 channels");
  return 0;
}

int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

void set_parts(GnGeom* g, int parts, int cluster) {  // cluster: a power of two
  g->parts = parts;
  g->part_px = g->pixels / parts;
  g->part_rest = g->pixels % parts;
  g->cluster = cluster;
  g->log_cluster = 0;
  while ((1 << g->log_cluster) < cluster) ++g->log_cluster;
}

// As many parts of an image as there are CTAs for each slab in one filling of the device, but four pixels a thread at
// least; in pairs, which halves what the second launch has to merge.  (Clusters of four do not fill the device: 46 us
// instead of 43 forward and 72 instead of 62 backward at 1 x 128 x 512 x 512 bf16.)
void set_many_parts(GnGeom* g, const Device& dev, bool backward) {
  const long long want = std::max(1ll, (backward ? 2 : 3) * dev.sms / (g->images * g->slabs));
  const long long cap = g->pixels / (4 * (kGnWide / g->sp));
  const int parts = (int)std::max(1ll, std::min(want, cap));
  set_parts(g, parts >= 2 ? parts / 2 * 2 : 1, parts >= 2 ? 2 : 1);
}

void set_slabs(GnGeom* g, int unit, int most) {  // slabs of at most `most` units, as even as they get
  const int units = g->pieces / unit;
  g->sp = cdiv(units, cdiv(units, most)) * unit;
  g->slabs = cdiv(g->pieces, g->sp);
}

// What the reductions of a CTA need: returns the bytes of shared memory of their arrays.
int set_reduction(GnGeom* g, int threads, bool backward) {
  g->inv_sp = 1.f / (float)g->sp;
  g->slab_groups = g->sp * 8 / g->cpg;
  g->fold = g->cpg % 8 == 0;
  g->run = g->fold ? g->cpg / 8 : g->cpg;
  g->inv_run = 1.f / (float)g->run;
  g->lanes = 0;
  while (g->lanes < 5 && g->slab_groups << (g->lanes + 1) <= threads) ++g->lanes;
  g->run_rows = (1 << g->lanes) / g->run;
  g->run_rest = (1 << g->lanes) % g->run;
  g->column_lanes = 0;
  while (g->column_lanes < 5 && (g->sp * 16) << (g->column_lanes + 1) <= threads) ++g->column_lanes;
  g->plane = g->fold && !backward ? threads : threads * 8;
  return 2 * g->plane * 4 + (backward ? threads * 8 : 0);
}

const GnKernels* kernels_of(int type, bool wide) {
  if (wide)
    return type == 0 ? groupnorm_2d_wide_kernels_0() : type == 1 ? groupnorm_2d_wide_kernels_1() : groupnorm_2d_wide_kernels_2();
  return type == 0 ? groupnorm_2d_narrow_kernels_0() : type == 1 ? groupnorm_2d_narrow_kernels_1() : groupnorm_2d_narrow_kernels_2();
}

// The ring of the kernels (GnBatch): 64 bytes a thread and batch in pieces of x (and dy).
void set_ring(Plan* p, int type, int bytes, bool backward) {
  GnGeom& g = p->g;
  const int pieces = cdiv(cdiv(g.pixels, g.parts), p->threads / g.sp);  // of a thread
  const int batch = (backward ? 4 : 8) / (type == 2 ? 4 : 2);
  g.batches = std::max(1, cdiv(pieces, batch));
  p->slots = 4 * batch;
  const int arrays = set_reduction(&g, p->threads, backward), ring = p->slots * p->threads * bytes;
  const int groups = (3 * g.slab_groups * 8 + 15) / 16 * 16;
  if (p->one_launch) {
    g.planes_at = 0, g.group_at = arrays, g.data_at = arrays + groups;
    p->smem = g.data_at + ring;
  } else {
    g.planes_at = g.data_at = groups, g.group_at = 0;
    p->smem = groups + std::max(arrays, ring);
  }
}

// Which launch to make.  The alternatives differ in the width of a slab, the CTAs of a cluster and their threads, or
// take two launches; none is best for all sizes.  Narrow slabs and large clusters give CTAs enough to fill the
// device, wide slabs whole DRAM sectors, few CTAs little bookkeeping, two launches any number of CTAs for one
// image.  The costs are estimates in cycles with constants fitted to 14000 measured launches of 300 sizes (all types,
// activations and directions; 0.2 to 64 million values): the choice takes 3 % longer than the best of each size on
// average, 15 % or more at one size in 13 and 42 % at worst (28 us instead of 19).
struct Work {
  double piece, piece_bytes;  // instructions a warp spends on a piece in both passes, bytes of it
  double read, written;       // bytes, each once
};

Work work_of(const spio_groupnorm_2d_desc* d, bool backward, bool coded) {
  static const double smooth[kActs] = {0., .2, 1., 1.8};  // instructions of an activation, in those of SiLU
  const double act = smooth[d->activation] * (d->type == 2 ? 2.2 : 1.);  // (fp32: exact functions)
  const double size = d->type == 2 ? 4 : 2;
  const double values = (double)d->n * d->pixels * d->c;
  Work w;
  w.piece_bytes = 8 * size;
  // copies, conversions, sums and stores; the activation (twice backward); the codes; for fp32 the second word of a piece
  w.piece = (backward ? 110 + 85 * act + (coded ? 20 : 0) : 72 + 28 * act + (coded ? 25 : 0)) + (d->type == 2 ? 15 : 0);
  w.read = values * (backward ? size + (coded ? 1.125 : size) : size);
  w.written = values * (size + (coded && !backward ? 1.125 : 0));
  return w;
}

constexpr double kBytesPerCycle = 3420.;  // 6500 GB/s at 1.9 GHz

double cost_of_one_launch(const Plan& p, const Work& w, const Device& dev, bool backward) {
  const GnGeom& g = p.g;
  const double ctas = (double)g.images * g.slabs * g.parts;
  const int pieces = cdiv(cdiv(g.pixels, g.parts), p.threads / g.sp);
  const int on_sm = std::max(1, std::min((backward ? 512 : 768) / p.threads, 228 * 1024 / (p.smem + 1024)));
  const double of_sm = std::ceil(ctas / dev.sms), rounds = std::ceil(of_sm / on_sm);
  const double warps = std::min(of_sm, (double)on_sm) * p.threads / 32;
  // a warp's bookkeeping and reductions, more of them where groups cut pieces, and its pieces; an SM issues up to 3.9 a
  // cycle, a warp .358
  const double instructions = of_sm * p.threads / 32 * ((backward ? 969 : 645) + (g.fold ? 0 : 195) + pieces * w.piece);
  const double compute = instructions / std::min(3.9, .358 * warps);
  const double row = g.sp * w.piece_bytes;
  // what the ring no longer holds is read again, from L2 or DRAM, in bytes of the first reading that take as long
  const double again = std::max(0., 1. - (double)p.slots / pieces) * w.read * (backward ? .845 : 2.54);
  const double filled = std::min(1., 2.19 * ctas * p.threads / (dev.sms * 256.));  // few threads have little on its way
  const double memory =  // (pixels' rows below 64 bytes leave sectors half used)
      (w.read + w.written + again) / kBytesPerCycle / (row >= 64 ? 1. : row >= 32 ? .6 : .36) / filled;
  const double sync = g.cluster > 1 ? 380 + 587 * g.log_cluster : 0;  // starting a cluster, its barriers and loads
  // the CTAs of an SM start together, and load and compute in turn more than at a time: weights of the longer and the
  // shorter; then what each round of CTAs waits for in a row, and launches (backward: the sum of the parts too)
  return .82 * std::max(compute, memory) + 1.45 * std::min(compute, memory) +
         rounds * ((backward ? 1620 : 1270) + sync) + (backward ? 6890 : 3490);
}

double cost_of_two_launches(const Plan& p, const Work& w, const Device& dev, bool backward) {
  const GnGeom& g = p.g;
  if (g.parts == 1) return std::numeric_limits<double>::infinity();  // the same CTAs do it in one launch
  const double of_sm = std::ceil((double)g.images * g.slabs * g.parts / dev.sms);
  const int pieces = cdiv(cdiv(g.pixels, g.parts), p.threads / g.sp);
  const double compute = of_sm * p.threads / 32 * (458 + pieces * (w.piece + 10)) / 2.28;  // as above; 2.28 a cycle
  // pixels' segments that begin and end inside a cache line cost where L2 does not hold them until the rest is wanted
  const double row = g.sp * w.piece_bytes, beyond = std::min(1., std::max(0., (w.read + w.written - 5e7) / 1e8));
  const double torn = g.slabs > 1 && (g.sp * (int)w.piece_bytes) % 128 != 0 ? 14.5 / row * beyond : 0.;
  // (a quarter of the second reading is paid for, the rest is in L2)
  const double memory = (1.25 * w.read + w.written) * (1. + torn) / kBytesPerCycle;
  // rounds of loads in which a CTA of the second launch merges the parts
  const double merges = cdiv(g.slab_groups, 8 * (backward ? 4 : 2)) * cdiv(g.parts / g.cluster, 256);
  return .9 * std::max(compute, memory) + .73 * std::min(compute, memory) + 1020 * merges + (backward ? 14000 : 10100);
}

int choose_plan(const spio_groupnorm_2d_desc* d, const Device& dev, bool backward, bool coded, Plan* best) {
  Plan p{};
  GnGeom& g = p.g;
  g.images = d->n;
  g.pixels = (int)d->pixels;
  g.c = d->c;
  g.pieces = d->c / 8;
  g.groups = d->groups;
  g.cpg = d->c / d->groups;
  g.inv_m = (float)(1.0 / ((double)g.pixels * g.cpg));
  g.inv_pixels = (float)(1.0 / (double)g.pixels);
  g.cpg_magic = (unsigned)(((1ull << 32) + g.cpg - 1) / g.cpg);
  const int unit = std::lcm(g.cpg, 8) / 8, units = g.pieces / unit;
  const int piece = d->type == 2 ? 32 : 16;
  const int bytes = backward ? piece + (coded ? 12 : piece) : piece;  // of a ring's slot
  const Work w = work_of(d, backward, coded);

  // two launches: as many CTAs as fit on the device, but four pixels a thread at least; slabs of at most 64 pieces (1 KB of
  // a pixel) where a group allows it, and narrower ones, which leave each CTA of the second launch less to merge
  double least = std::numeric_limits<double>::infinity();
  p.one_launch = false;
  p.threads = kGnWide;
  for (int most = 64, sp = 0; most >= 8; most /= 2) {
    set_slabs(&g, unit, std::max(1, most / unit));
    if (g.sp == sp) continue;
    sp = g.sp;
    set_many_parts(&g, dev, backward);
    set_ring(&p, d->type, bytes, backward);
    if (p.smem > dev.smem) continue;
    const double cost = cost_of_two_launches(p, w, dev, backward);
    if (cost < least) least = cost, *best = p;
  }

  p.one_launch = true;
  for (int most = std::min(units, std::max(1, 64 / unit)), sp = 0; most >= 1; --most) {
    set_slabs(&g, unit, most);
    if (g.sp == sp) continue;
    sp = g.sp;
    for (int parts = 1; parts <= 16 && parts <= g.pixels; parts *= 2) {
      set_parts(&g, parts, parts);
      for (const int threads : {kGnNarrow, kGnWide}) {
        if (sp > threads) continue;
        p.threads = threads;
        set_ring(&p, d->type, bytes, backward);
        if (p.smem > dev.smem) continue;
        const double cost = cost_of_one_launch(p, w, dev, backward);
        if (cost < least) least = cost, *best = p;
      }
    }
  }
  if (!(least < std::numeric_limits<double>::infinity())) return jit_fail("GroupNorm2d: no launch fits the device");
  const GnGeom& b = best->g;
  const long long grid = b.images * b.slabs * b.parts;
  if (grid > 0x7fffffffll) return jit_fail("GroupNorm2d: too many images for one launch");
  if (((long long)b.part_px + 1) * b.pieces > 0xffffffffll) return jit_fail("GroupNorm2d: an image is too large");
  best->grid = (unsigned)grid;
  best->rows = b.images * b.parts;
  best->stats_bytes = best->one_launch ? 0 : aligned(sizeof(float2) * (size_t)b.images * b.groups * (b.parts / b.cluster));
  best->group_bytes = best->stats_bytes;
  best->channel_bytes = aligned(sizeof(float) * 2 * (size_t)best->rows * b.c);
  return 0;
}

// The choice takes some 10 us: it is made once for each size.
int make_plan(const spio_groupnorm_2d_desc* d, const Device& dev, bool backward, bool coded, Plan* p) {
  typedef std::array<long long, 7> Key;
  static std::mutex mutex;
  static std::map<Key, Plan> plans;
  const Key key = {d->n, d->pixels, d->c, d->groups, d->type * 16 + d->activation, backward * 2 + coded,
                   (long long)dev.sms << 32 | dev.smem};
  try {
    std::lock_guard<std::mutex> lock(mutex);
    auto it = plans.find(key);
    if (it == plans.end()) {
      Plan fresh;
      if (choose_plan(d, dev, backward, coded, &fresh)) return 1;
      if (plans.size() >= 4096) plans.clear();
      it = plans.insert_or_assign(key, fresh).first;
    }
    *p = it->second;
  } catch (const std::exception& e) {  // no memory; C callers get an error like any other
    return jit_fail(std::string("GroupNorm2d: ") + e.what());
  }
  p->g.eps = d->eps;
  return 0;
}

int launch(const void* func, const Device& dev, unsigned grid, int threads, int smem, int cluster, void* stream, void** args) {
  if ((smem > 48 * 1024 || cluster > 8) && allow(func, dev)) return 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (gw8_pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t e = cudaLaunchKernelExC(&cfg, func, args);
  if (e != cudaSuccess) return jit_fail(std::string("CUDA error: ") + cudaGetErrorString(e));
  return 0;
}

int check_pointers(const spio_groupnorm_2d_desc* d, const void* out, const void* a, const void* b, const void* codes,
                   const void* exponents, const void* stats) {
  if (((reinterpret_cast<size_t>(out) | reinterpret_cast<size_t>(a) | reinterpret_cast<size_t>(b)) & 15u) != 0)
    return jit_fail("tensor pointers must be 16-byte aligned");
  if (d->type == 2 && (reinterpret_cast<size_t>(out) & 31u) != 0)
    return jit_fail("fp32 tensors that are written must be 32-byte aligned");
  if ((codes == nullptr) != (exponents == nullptr)) return jit_fail("codes and exponents go together");
  if (((reinterpret_cast<size_t>(codes) | reinterpret_cast<size_t>(stats)) & 7u) != 0)
    return jit_fail("codes and stats must be 8-byte aligned");
  if ((reinterpret_cast<size_t>(exponents) & 3u) != 0) return jit_fail("exponents must be 4-byte aligned");
  return 0;
}

}  // namespace
}  // namespace spio_b200

using namespace spio_b200;

extern "C" {

int spio_groupnorm_2d_plan_for(const spio_groupnorm_2d_desc* desc, int backward, int coded, int sm_count,
                               int smem_optin_bytes, spio_groupnorm_2d_plan_info* info) {
  if (check_desc(desc)) return 1;
  if (info == nullptr) return jit_fail("info is NULL");
  if (desc->n == 0 || desc->pixels == 0) return jit_fail("GroupNorm2d: nothing to plan for an empty tensor");
  if (sm_count <= 0 || smem_optin_bytes <= 0) return jit_fail("GroupNorm2d: no such device");
  const Device dev = {sm_count, smem_optin_bytes, -1};
  Plan p;
  if (choose_plan(desc, dev, backward != 0, coded != 0, &p)) return 1;
  *info = {};
  info->one_launch = p.one_launch;
  info->threads = p.threads;
  info->smem_bytes = p.smem;
  info->slab_pieces = p.g.sp;
  info->slabs = p.g.slabs;
  info->parts = p.g.parts;
  info->cluster = p.g.cluster;
  info->grid = p.grid;
  info->scratch_bytes = backward ? p.channel_bytes + p.group_bytes : p.stats_bytes;
  return 0;
}

size_t spio_groupnorm_2d_fwd_scratch_bytes(const spio_groupnorm_2d_desc* desc) {
  Device dev;
  Plan p, q;
  if (check_desc(desc) || desc->n == 0 || desc->pixels == 0) return 0;
  if (device_of(&dev) || make_plan(desc, dev, false, false, &p) || make_plan(desc, dev, false, true, &q)) return 0;
  return std::max(p.stats_bytes, q.stats_bytes);
}

int spio_groupnorm_2d_fwd(void* y, float* stats, void* codes, void* exponents, const void* x, const float* weight,
                          const float* bias, const spio_groupnorm_2d_desc* desc, void* scratch,
                          size_t scratch_bytes, void* stream) {
  if (check_desc(desc)) return 1;
  if (desc->n == 0 || desc->pixels == 0) return 0;
  if (y == nullptr || x == nullptr) return jit_fail("NULL tensor pointer");
  if (check_pointers(desc, y, x, scratch, codes, exponents, stats)) return 1;
  Device dev;
  Plan p;
  const int coded = codes != nullptr;
  if (device_of(&dev) || make_plan(desc, dev, false, coded, &p)) return 1;
  const GnKernels* k = kernels_of(desc->type, p.threads == kGnWide);
  if (p.one_launch) {
    void* args[] = {&y, &stats, &codes, &exponents, (void*)&x, (void*)&weight, (void*)&bias, &p.g};
    return launch(k->fwd[desc->activation][coded], dev, p.grid, p.threads, p.smem, p.g.cluster, stream, args);
  }
  if (scratch == nullptr || scratch_bytes < p.stats_bytes) return jit_fail("GroupNorm2d scratch buffer is too small");
  void* sargs[] = {&scratch, (void*)&x, &p.g};
  if (launch(k->stats, dev, p.grid, p.threads, p.smem, p.g.cluster, stream, sargs)) return 1;
  void* args[] = {&y, &stats, &codes, &exponents, (void*)&x, (void*)&weight, (void*)&bias, &scratch, &p.g};
  return launch(k->apply[desc->activation][coded], dev, p.grid, p.threads, p.smem, 1, stream, args);
}

size_t spio_groupnorm_2d_bwd_scratch_bytes(const spio_groupnorm_2d_desc* desc) {
  Device dev;
  Plan p, q;
  if (check_desc(desc) || desc->n == 0 || desc->pixels == 0) return 0;
  if (device_of(&dev) || make_plan(desc, dev, true, false, &p) || make_plan(desc, dev, true, true, &q)) return 0;
  return std::max(p.channel_bytes + p.group_bytes, q.channel_bytes + q.group_bytes);
}

int spio_groupnorm_2d_bwd(void* dx, float* dweight, float* dbias, const void* dy, const void* x, const void* codes,
                          const void* exponents, const float* stats, const float* weight, const float* bias,
                          const spio_groupnorm_2d_desc* desc, void* scratch, size_t scratch_bytes, void* stream) {
  if (check_desc(desc)) return 1;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (dx == nullptr && !sums) return 0;
  if (desc->n == 0 || desc->pixels == 0) {  // sums over nothing
    for (float* out : {dweight, dbias})
      if (out != nullptr) {
        const cudaError_t e = cudaMemsetAsync(out, 0, sizeof(float) * (size_t)desc->c, (cudaStream_t)stream);
        if (e != cudaSuccess) return jit_fail(std::string("CUDA error: ") + cudaGetErrorString(e));
      }
    return 0;
  }
  if (dy == nullptr || stats == nullptr || (x == nullptr && codes == nullptr)) return jit_fail("NULL tensor pointer");
  if (check_pointers(desc, dx, dy, codes == nullptr ? x : nullptr, codes, exponents, stats)) return 1;
  if ((reinterpret_cast<size_t>(scratch) & 15u) != 0) return jit_fail("scratch must be 16-byte aligned");
  const int coded = codes != nullptr;
  Device dev;
  Plan p;
  if (device_of(&dev) || make_plan(desc, dev, true, coded, &p)) return 1;
  if (scratch == nullptr || scratch_bytes < p.channel_bytes + p.group_bytes)
    return jit_fail("GroupNorm2d scratch buffer is too small");
  const GnKernels* k = kernels_of(desc->type, p.threads == kGnWide);
  float* part_channel = sums ? static_cast<float*>(scratch) : nullptr;
  if (p.one_launch) {
    void* args[] = {&dx, &part_channel, (void*)&dy, (void*)&x, (void*)&codes, (void*)&exponents,
                    (void*)&stats, (void*)&weight, (void*)&bias, &p.g};
    if (launch(k->bwd[desc->activation][coded], dev, p.grid, p.threads, p.smem, p.g.cluster, stream, args)) return 1;
  } else {
    float2* part_group = dx != nullptr ? reinterpret_cast<float2*>(static_cast<char*>(scratch) + p.channel_bytes) : nullptr;
    void* args[] = {&part_channel, &part_group, (void*)&dy, (void*)&x, (void*)&codes, (void*)&exponents,
                    (void*)&stats, (void*)&weight, (void*)&bias, &p.g};
    if (launch(k->bwd_sums[desc->activation][coded], dev, p.grid, p.threads, p.smem, p.g.cluster, stream, args)) return 1;
    if (dx != nullptr) {
      void* dargs[] = {&dx, &part_group, (void*)&dy, (void*)&x, (void*)&codes, (void*)&exponents,
                       (void*)&stats, (void*)&weight, (void*)&bias, &p.g};
      if (launch(k->bwd_apply[desc->activation][coded], dev, p.grid, p.threads, p.smem, 1, stream, dargs)) return 1;
    }
  }
  if (sums) {
    int c = p.g.c, rows = (int)p.rows, split = 1;  // (the grid has as many CTAs at least: 2^31 - 1 at most)
    // (with 1000 rows the cluster's barriers cost what it saves, 0.7 us)
    while (rows > 1024 && split < 8 && rows / 256 > split) split *= 2;
    void* rargs[] = {&dweight, &dbias, &part_channel, &c, &rows, &split};
    const void* reduce = split > 1 ? (const void*)&groupnorm_2d_bwd_reduce_kernel<true> : (const void*)&groupnorm_2d_bwd_reduce_kernel<false>;
    return launch(reduce, dev, (2 * c + 31) / 32 * split, 1024, 0, split, stream, rargs);
  }
  return 0;
}

}  // extern "C"

// Planning and launches of the group norm (kernels: groupnorm_2d.cuh), and the sum of its per-image
// weight and bias gradients.
#include <cuda_runtime.h>

#include <algorithm>
#include <numeric>
#include <string>

#include "groupnorm_2d.h"
#include "ptx.cuh"
#include "../../include/spio_b200.h"

namespace spio_b200 {

int jit_fail(const std::string& msg);  // sets the thread's last-error text, returns 1
bool gw8_pdl_enabled();

namespace {

// dweight[c] / dbias[c] = sums of rows of 2 * c values, in a fixed order: a CTA owns 32 columns, its
// warps take every 32nd row (128-byte rows, coalesced) and are added through shared memory.
__global__ void __launch_bounds__(1024)
groupnorm_2d_bwd_reduce_kernel(float* __restrict__ dweight, float* __restrict__ dbias,
                               const float* __restrict__ part, int c, long long rows) {
  __shared__ float sums[32][33];
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < 2 * c) {
#pragma unroll 8
    for (long long r = warp; r < rows; r += 32) s += __ldcg(part + r * 2 * c + col);
  }
  sums[warp][lane] = s;
  __syncthreads();
  s = sums[lane][warp];  // column `warp` of the 32, its warps' sums over the lanes
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  const int out = blockIdx.x * 32 + warp;
  if (lane != 0 || out >= 2 * c) return;
  if (out < c) {
    if (dweight != nullptr) dweight[out] = s;
  } else if (dbias != nullptr) {
    dbias[out - c] = s;
  }
}

struct Plan {
  GnGeom g;
  unsigned grid;
  size_t stats_bytes;    // forward: parts' statistics
  size_t channel_bytes;  // backward: parts' sums for the channels
  size_t group_bytes;    // backward: parts' sums for the groups
};

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

int device_sms(int* sms) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return jit_fail("CUDA error: no device");
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
  if (std::lcm(cpg, 8) > kGnMaxSlabPieces * 8)
    return jit_fail("GroupNorm2d: groups (rounded up to whole blocks of 8 channels) may span at most 2048 channels");
  return 0;
}

int make_plan(const spio_groupnorm_2d_desc* d, int sms, Plan* p) {
  GnGeom& g = p->g;
  g.images = d->n;
  g.pixels = (int)d->pixels;
  g.c = d->c;
  g.pieces = d->c / 8;
  g.groups = d->groups;
  g.cpg = d->c / d->groups;
  g.eps = d->eps;
  g.inv_m = (float)(1.0 / ((double)std::max(g.pixels, 1) * g.cpg));
  // slabs: whole groups and whole pieces, 64 pieces (1 KB of a pixel) where a group allows it
  const int unit = std::lcm(g.cpg, 8) / 8;
  const int units = g.pieces / unit;
  const int most = std::max(1, 64 / unit);
  g.slabs = (units + most - 1) / most;
  g.sp = (units + g.slabs - 1) / g.slabs * unit;
  g.slabs = (g.pieces + g.sp - 1) / g.sp;
  // parts: about four CTAs an SM, but four pixels a thread at least
  const int rows = kGnThreads / g.sp;
  const long long ctas = std::max(1ll, g.images * g.slabs);
  const long long want = (4ll * sms + ctas - 1) / ctas;
  const long long cap = std::max(1, g.pixels / (4 * rows));
  const int parts = (int)std::max(1ll, std::min(want, cap));
  g.part_px = std::max(1, (g.pixels + parts - 1) / parts);
  g.parts = std::max(1, (g.pixels + g.part_px - 1) / g.part_px);
  const long long grid = g.images * g.slabs * g.parts;
  if (grid > 0x7fffffffll) return jit_fail("GroupNorm2d: too many images for one launch");
  p->grid = (unsigned)grid;
  p->stats_bytes = aligned(sizeof(float2) * (size_t)g.images * g.groups * g.parts);
  p->group_bytes = p->stats_bytes;
  p->channel_bytes = aligned(sizeof(float) * 2 * (size_t)g.images * g.parts * g.c);
  return 0;
}

const GnKernels* kernels_of(int type) {
  return type == 0 ? groupnorm_2d_kernels_f16() : type == 1 ? groupnorm_2d_kernels_bf16() : groupnorm_2d_kernels_f32();
}

int launch(const void* func, unsigned grid, int threads, void* stream, void** args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = gw8_pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelExC(&cfg, func, args);
  if (e != cudaSuccess) return jit_fail(std::string("CUDA error: ") + cudaGetErrorString(e));
  return 0;
}

int check_pointers(const void* a, const void* b, const void* c, const void* codes, const void* exponents,
                   const void* stats) {
  if (((reinterpret_cast<size_t>(a) | reinterpret_cast<size_t>(b) | reinterpret_cast<size_t>(c)) & 15u) != 0)
    return jit_fail("tensor pointers must be 16-byte aligned");
  if ((codes == nullptr) != (exponents == nullptr)) return jit_fail("codes and exponents go together");
  if (((reinterpret_cast<size_t>(codes) | reinterpret_cast<size_t>(stats)) & 7u) != 0)
    return jit_fail("codes and stats must be 8-byte aligned");
  return 0;
}

}  // namespace
}  // namespace spio_b200

using namespace spio_b200;

extern "C" {

size_t spio_groupnorm_2d_fwd_scratch_bytes(const spio_groupnorm_2d_desc* desc) {
  int sms = 0;
  Plan p;
  if (check_desc(desc) || device_sms(&sms) || make_plan(desc, sms, &p)) return 0;
  return p.stats_bytes;
}

int spio_groupnorm_2d_fwd(void* y, float* stats, void* codes, void* exponents, const void* x, const float* weight,
                          const float* bias, const spio_groupnorm_2d_desc* desc, void* scratch,
                          size_t scratch_bytes, void* stream) {
  if (check_desc(desc)) return 1;
  if (desc->n == 0 || desc->pixels == 0) return 0;
  if (y == nullptr || x == nullptr) return jit_fail("NULL tensor pointer");
  if (check_pointers(y, x, scratch, codes, exponents, stats)) return 1;
  int sms = 0;
  Plan p;
  if (device_sms(&sms) || make_plan(desc, sms, &p)) return 1;
  if (scratch == nullptr || scratch_bytes < p.stats_bytes) return jit_fail("GroupNorm2d scratch buffer is too small");
  const GnKernels* k = kernels_of(desc->type);
  void* sargs[] = {&scratch, (void*)&x, &p.g};
  if (launch(k->stats, p.grid, kGnThreads, stream, sargs)) return 1;
  void* args[] = {&y, &stats, &codes, &exponents, (void*)&x, (void*)&weight, (void*)&bias, &scratch, &p.g};
  return launch(k->apply[desc->activation][codes != nullptr], p.grid, kGnThreads, stream, args);
}

size_t spio_groupnorm_2d_bwd_scratch_bytes(const spio_groupnorm_2d_desc* desc) {
  int sms = 0;
  Plan p;
  if (check_desc(desc) || device_sms(&sms) || make_plan(desc, sms, &p)) return 0;
  return p.channel_bytes + p.group_bytes;
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
  if (check_pointers(dx, dy, codes == nullptr ? x : nullptr, codes, exponents, stats)) return 1;
  if ((reinterpret_cast<size_t>(scratch) & 15u) != 0) return jit_fail("scratch must be 16-byte aligned");
  int sms = 0;
  Plan p;
  if (device_sms(&sms) || make_plan(desc, sms, &p)) return 1;
  if (scratch == nullptr || scratch_bytes < p.channel_bytes + p.group_bytes)
    return jit_fail("GroupNorm2d scratch buffer is too small");
  const GnKernels* k = kernels_of(desc->type);
  const int coded = codes != nullptr;
  float* part_channel = sums ? static_cast<float*>(scratch) : nullptr;
  float2* part_group = dx != nullptr ? reinterpret_cast<float2*>(static_cast<char*>(scratch) + p.channel_bytes) : nullptr;
  void* args[] = {&part_channel, &part_group, (void*)&dy, (void*)&x, (void*)&codes, (void*)&exponents,
                  (void*)&stats, (void*)&weight, (void*)&bias, &p.g};
  if (launch(k->bwd_sums[desc->activation][coded], p.grid, kGnThreads, stream, args)) return 1;
  if (dx != nullptr) {
    void* dargs[] = {&dx, &part_group, (void*)&dy, (void*)&x, (void*)&codes, (void*)&exponents,
                     (void*)&stats, (void*)&weight, (void*)&bias, &p.g};
    if (launch(k->bwd_apply[desc->activation][coded], p.grid, kGnThreads, stream, dargs)) return 1;
  }
  if (sums) {
    long long rows = p.g.images * p.g.parts;
    int c = p.g.c;
    void* rargs[] = {&dweight, &dbias, &part_channel, &c, &rows};
    return launch((const void*)&groupnorm_2d_bwd_reduce_kernel, (2 * c + 31) / 32, 1024, stream, rargs);
  }
  return 0;
}

}  // extern "C"

// Shared by the translation units of the group norm: the geometry a kernel takes by value and the
// table of kernels that each data type's unit exports.
#pragma once

namespace spio_b200 {

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActs = 4 };

// Threads of a CTA: the one-launch kernels are built with both, the wide one serves the two-kernel forms and groups
// that span more pieces of 8 channels than the narrow one has threads.
constexpr int kGnNarrow = 128, kGnWide = 256;

// An image is cut into slabs of whole groups of channels (sp pieces of 8 channels each, the last
// one narrower) and its pixels into parts; a CTA works on one part of one slab of one image.
struct GnGeom {
  long long images;
  int pixels;     // of an image
  int c, pieces;  // channels, c / 8
  int groups, cpg;
  int sp, slabs;        // pieces of a slab, slabs of an image
  int parts, part_px, part_rest;  // parts of an image; pixels of each, one more in the first part_rest
  float inv_m;          // 1 / (pixels * cpg)
  float eps;
  unsigned cpg_magic;     // ceil(2^32 / cpg)
  float inv_sp, inv_pixels;
  // reductions.  fold: a piece lies within one group; lanes: log2 of the lanes that share a group, of which each takes
  // every 2^lanes-th value of the rows' runs of `run` values: run_rows rows and run_rest values on; column_lanes:
  // log2 of the lanes that share a channel
  int fold, lanes, run, run_rows, run_rest, column_lanes;
  float inv_run;
  int slab_groups;  // of a full slab
  int plane;        // values of one of the reductions' arrays
  int planes_at, group_at;  // where these and the groups' values start in the dynamic shared memory
  int cluster, log_cluster;  // CTAs of a cluster, a power of two that divides parts
  int batches, data_at;      // batches of pieces of a thread, where the ring is
};

struct GnKernels {
  const void* stats;
  const void* apply[kActs][2];      // [activation][writes codes]
  const void* bwd_sums[kActs][2];   // [activation][reads codes]
  const void* bwd_apply[kActs][2];
  const void* fwd[kActs][2];        // one launch
  const void* bwd[kActs][2];
};

// type: 0 fp16, 1 bf16, 2 fp32; the narrow tables have the one-launch kernels alone
const GnKernels* groupnorm_2d_wide_kernels_0();
const GnKernels* groupnorm_2d_wide_kernels_1();
const GnKernels* groupnorm_2d_wide_kernels_2();
const GnKernels* groupnorm_2d_narrow_kernels_0();
const GnKernels* groupnorm_2d_narrow_kernels_1();
const GnKernels* groupnorm_2d_narrow_kernels_2();

}  // namespace spio_b200

// Shared by the translation units of the group norm: the geometry a kernel takes by value and the
// table of kernels that each data type's unit exports.
#pragma once

namespace spio_b200 {

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActs = 4 };

constexpr int kGnThreads = 256;
constexpr int kGnMaxSlabPieces = 256;  // a thread owns at most one piece of a pixel's slab

// An image is cut into slabs of whole groups of channels (sp pieces of 8 channels each, the last
// one narrower) and its pixels into parts; a CTA works on one part of one slab of one image.
struct GnGeom {
  long long images;
  int pixels;     // of an image
  int c, pieces;  // channels, c / 8
  int groups, cpg;
  int sp, slabs;        // pieces of a slab, slabs of an image
  int parts, part_px;   // parts of an image, pixels of each (the last one has fewer)
  float inv_m;          // 1 / (pixels * cpg)
  float eps;
};

struct GnKernels {
  const void* stats;
  const void* apply[kActs][2];      // [activation][writes codes]
  const void* bwd_sums[kActs][2];   // [activation][reads codes]
  const void* bwd_apply[kActs][2];
};

const GnKernels* groupnorm_2d_kernels_f16();
const GnKernels* groupnorm_2d_kernels_bf16();
const GnKernels* groupnorm_2d_kernels_f32();

}  // namespace spio_b200

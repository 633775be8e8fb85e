// The group norm's kernels for one data type (GN_TYPE = 0 fp16, 1 bf16, 2 fp32) and one width of CTAs
// (GN_THREADS = 128 or 256).
#if GN_THREADS == 128
#define GN_NAMESPACE gn_narrow
#define GN_TABLE_OF(type) groupnorm_2d_narrow_kernels_##type
#else
#define GN_NAMESPACE gn_wide
#define GN_TABLE_OF(type) groupnorm_2d_wide_kernels_##type
#endif
#define GN_TABLE(type) GN_TABLE_OF(type)

#include "groupnorm_2d.cuh"

namespace spio_b200 {

#if GN_TYPE == 0
typedef __half GnT;
#elif GN_TYPE == 1
typedef __nv_bfloat16 GnT;
#else
typedef float GnT;
#endif

#define GN_BOTH(kernel, act) \
  { (const void*)&GN_NAMESPACE::kernel<GnT, act, false>, (const void*)&GN_NAMESPACE::kernel<GnT, act, true> }
#define GN_ACTS(kernel) \
  { GN_BOTH(kernel, kActNone), GN_BOTH(kernel, kActRelu), GN_BOTH(kernel, kActSilu), GN_BOTH(kernel, kActGelu) }

const GnKernels* GN_TABLE(GN_TYPE)() {
#if GN_THREADS == 128
  static const GnKernels k = {nullptr, {}, {}, {}, GN_ACTS(groupnorm_2d_fwd_kernel), GN_ACTS(groupnorm_2d_bwd_kernel)};
#else
  static const GnKernels k = {(const void*)&GN_NAMESPACE::groupnorm_2d_stats_kernel<GnT>,
                              GN_ACTS(groupnorm_2d_apply_kernel), GN_ACTS(groupnorm_2d_bwd_sums_kernel),
                              GN_ACTS(groupnorm_2d_bwd_apply_kernel), GN_ACTS(groupnorm_2d_fwd_kernel),
                              GN_ACTS(groupnorm_2d_bwd_kernel)};
#endif
  return &k;
}

}  // namespace spio_b200

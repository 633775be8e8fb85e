// The group norm's kernels for one data type (GN_TYPE = 0 fp16, 1 bf16, 2 fp32).
#include "groupnorm_2d.cuh"

namespace spio_b200 {

#if GN_TYPE == 0
typedef __half GnT;
#define GN_TABLE groupnorm_2d_kernels_f16
#elif GN_TYPE == 1
typedef __nv_bfloat16 GnT;
#define GN_TABLE groupnorm_2d_kernels_bf16
#else
typedef float GnT;
#define GN_TABLE groupnorm_2d_kernels_f32
#endif

#define GN_BOTH(kernel, act) \
  { (const void*)&kernel<GnT, act, false>, (const void*)&kernel<GnT, act, true> }
#define GN_ACTS(kernel) \
  { GN_BOTH(kernel, kActNone), GN_BOTH(kernel, kActRelu), GN_BOTH(kernel, kActSilu), GN_BOTH(kernel, kActGelu) }

const GnKernels* GN_TABLE() {
  static const GnKernels k = {(const void*)&groupnorm_2d_stats_kernel<GnT>, GN_ACTS(groupnorm_2d_apply_kernel),
                              GN_ACTS(groupnorm_2d_bwd_sums_kernel), GN_ACTS(groupnorm_2d_bwd_apply_kernel)};
  return &k;
}

}  // namespace spio_b200

// Packing a tensor into the 8-bit form of checkpoint8.cuh and restoring it.
//
// Both are streams: 3.125 bytes a value move for 16-bit data (2 + 1.125), 5.125 for fp32, and what bounds them is
// DRAM.  A thread works on kPieces pieces one CTA width apart, all requested before the first is used.  Two pieces and
// 256 threads were best or within 2 % of it at all sizes: at 256 x 64 x 56 x 56 one piece took 28 us for fp16 instead of
// 24 (too little on its way), eight 25, and at 2 x 64 x 64 x 64, where there are few CTAs, 2.2 us instead of 1.5.
//
// Measured at 256 x 64 x 56 x 56, the inputs not in L2: fp16 packing 23.9 us (6720 GB/s), restoring 25.2 us
// (6370 GB/s); fp32 38.0 us (6940 GB/s) and 40.4 us (6530 GB/s).  A plain copy reaches 6520 GB/s.
#include <cuda_runtime.h>

#include <string>

#include "checkpoint8.cuh"
#include "../../include/spio_b200.h"

namespace spio_b200 {

int jit_fail(const std::string& msg);  // sets the thread's last-error text, returns 1
bool gw8_pdl_enabled();

namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 2;

template <class T>
__global__ void __launch_bounds__(kThreads)
checkpoint8_pack_kernel(uint2* __restrict__ codes, unsigned char* __restrict__ exponents, const T* __restrict__ x,
                        long long blocks) {
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const long long first = (long long)blockIdx.x * (kThreads * kPieces) + threadIdx.x;
  Piece<T> v[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long b = first + k * kThreads;
    if (b < blocks) v[k] = load_piece(x + b * 8);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long b = first + k * kThreads;
    if (b < blocks) {
      const Block8 e = encode_block(v[k], values_of(v[k]));
      __stcs(codes + b, e.codes);
      exponents[b] = (unsigned char)e.exponent;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
checkpoint8_unpack_kernel(T* __restrict__ x, const uint2* __restrict__ codes,
                          const unsigned char* __restrict__ exponents, long long blocks) {
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const long long first = (long long)blockIdx.x * (kThreads * kPieces) + threadIdx.x;
  Block8 v[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long b = first + k * kThreads;
    if (b < blocks) {
      v[k].codes = __ldcs(codes + b);
      v[k].exponent = __ldcs(exponents + b);
    }
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long b = first + k * kThreads;
    if (b < blocks) {
      Piece<T> o;
      to_piece(o, decode_block(v[k]));
      store_piece_keep(x + b * 8, o);
    }
  }
}

int check(const void* x, const void* codes, const void* exponents, long long blocks, int type, bool restore) {
  if (type < 0 || type > 2) return jit_fail("checkpoint8: unknown data type");
  if (blocks < 0) return jit_fail("checkpoint8: the number of blocks must not be negative");
  if (blocks > (1ll << 40)) return jit_fail("checkpoint8: too many blocks");
  if (blocks == 0) return 0;
  if (x == nullptr || codes == nullptr || exponents == nullptr) return jit_fail("NULL tensor pointer");
  if ((reinterpret_cast<size_t>(x) & 15u) != 0) return jit_fail("tensor pointers must be 16-byte aligned");
  if (restore && type == 2 && (reinterpret_cast<size_t>(x) & 31u) != 0)
    return jit_fail("fp32 tensors that are written must be 32-byte aligned");
  if ((reinterpret_cast<size_t>(codes) & 7u) != 0) return jit_fail("codes must be 8-byte aligned");
  return 0;
}

int launch(const void* func, long long blocks, void* stream, void** args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((blocks + kThreads * kPieces - 1) / (kThreads * kPieces)));
  cfg.blockDim = dim3(kThreads);
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

}  // namespace
}  // namespace spio_b200

using namespace spio_b200;

extern "C" {

int spio_checkpoint8_pack(void* codes, void* exponents, const void* x, long long blocks, int type, void* stream) {
  if (check(x, codes, exponents, blocks, type, false)) return 1;
  if (blocks == 0) return 0;
  const void* fn[3] = {(const void*)&checkpoint8_pack_kernel<__half>, (const void*)&checkpoint8_pack_kernel<__nv_bfloat16>,
                       (const void*)&checkpoint8_pack_kernel<float>};
  void* args[] = {&codes, &exponents, (void*)&x, &blocks};
  return launch(fn[type], blocks, stream, args);
}

int spio_checkpoint8_unpack(void* x, const void* codes, const void* exponents, long long blocks, int type,
                            void* stream) {
  if (check(x, codes, exponents, blocks, type, true)) return 1;
  if (blocks == 0) return 0;
  const void* fn[3] = {(const void*)&checkpoint8_unpack_kernel<__half>,
                       (const void*)&checkpoint8_unpack_kernel<__nv_bfloat16>,
                       (const void*)&checkpoint8_unpack_kernel<float>};
  void* args[] = {&x, (void*)&codes, (void*)&exponents, &blocks};
  return launch(fn[type], blocks, stream, args);
}

}  // extern "C"

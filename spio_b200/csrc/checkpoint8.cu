// Packing a tensor into the 8-bit form of checkpoint8.cuh and restoring it.
//
// Both are streams: 3.125 bytes a value move for 16-bit data (2 + 1.125), and what bounds them is DRAM.
// A thread works on kPieces pieces one CTA width apart, all requested before the first is used.
#include <cuda_runtime.h>

#include <string>

#include "checkpoint8.cuh"
#include "../../include/spio_b200.h"

namespace spio_b200 {

int jit_fail(const std::string& msg);  // sets the thread's last-error text, returns 1
bool gw8_pdl_enabled();

namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;

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
#pragma unroll
      for (int i = 0; i < Piece<T>::W; ++i) reinterpret_cast<uint4*>(x + b * 8)[i] = o.u[i];  // read next: keep in L2
    }
  }
}

int check(const void* x, const void* codes, const void* exponents, long long blocks, int type) {
  if (type < 0 || type > 2) return jit_fail("checkpoint8: unknown data type");
  if (blocks < 0) return jit_fail("checkpoint8: the number of blocks must not be negative");
  if (blocks > (1ll << 40)) return jit_fail("checkpoint8: too many blocks");
  if (blocks == 0) return 0;
  if (x == nullptr || codes == nullptr || exponents == nullptr) return jit_fail("NULL tensor pointer");
  if ((reinterpret_cast<size_t>(x) & 15u) != 0) return jit_fail("tensor pointers must be 16-byte aligned");
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
  if (check(x, codes, exponents, blocks, type)) return 1;
  if (blocks == 0) return 0;
  const void* fn[3] = {(const void*)&checkpoint8_pack_kernel<__half>, (const void*)&checkpoint8_pack_kernel<__nv_bfloat16>,
                       (const void*)&checkpoint8_pack_kernel<float>};
  void* args[] = {&codes, &exponents, (void*)&x, &blocks};
  return launch(fn[type], blocks, stream, args);
}

int spio_checkpoint8_unpack(void* x, const void* codes, const void* exponents, long long blocks, int type,
                            void* stream) {
  if (check(x, codes, exponents, blocks, type)) return 1;
  if (blocks == 0) return 0;
  const void* fn[3] = {(const void*)&checkpoint8_unpack_kernel<__half>,
                       (const void*)&checkpoint8_unpack_kernel<__nv_bfloat16>,
                       (const void*)&checkpoint8_unpack_kernel<float>};
  void* args[] = {&x, (void*)&codes, (void*)&exponents, &blocks};
  return launch(fn[type], blocks, stream, args);
}

}  // extern "C"

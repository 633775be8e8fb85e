// The 8-bit form of an activation tensor, and loads and stores of pieces of 8 channels.
//
// A block is 8 consecutive channels of a pixel (one channel group of the gw8 convolution, one
// 16-byte piece of fp16 data).  It is kept as 8 signed codes and one exponent byte E, and stands for
//     value[i] = code[i] * 2^(E - 127),      E = 255: every value is NaN.
// The scale is the smallest power of two, 2^-126 at least, for which the block's largest magnitude
// rounds to at most 127; codes are rounded half to even.  Where rounding up would leave the range of
// the tensor's type (a largest magnitude above 63.5 / 64 of the type's maximum) codes stop at 63, so
// a finite block is restored finite.  A block with an infinity or a NaN is restored as NaN: a loss
// scaler that looks for overflowed gradients still finds them.
//
// Why powers of two and blocks of 8: scaling is exact, so codes are a function of the input alone,
// whatever arithmetic computes them, and a block is one thread's piece: no shuffles, and any split of
// the channels over threads and CTAs sees whole blocks.  1.125 bytes a value; the largest magnitude
// of 8 values is 1.42 standard deviations for normal data, so the step is 1.4 / 91 of one on average.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace spio_b200 {

enum { kTypeF16 = 0, kTypeBf16 = 1, kTypeF32 = 2 };

// ---------------------------------------------------------------- pieces of 8 channels

// 8 values of type T as they lie in memory: W 16-byte words.
template <class T>
struct Piece {
  static constexpr int W = sizeof(T) / 2;
  uint4 u[W];
};

template <class T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> v;
#pragma unroll
  for (int i = 0; i < Piece<T>::W; ++i) v.u[i] = reinterpret_cast<const uint4*>(p)[i];
  return v;
}

// For data that is not read again: first out of the caches.
template <class T>
__device__ __forceinline__ Piece<T> load_piece_streaming(const T* p) {
  Piece<T> v;
#pragma unroll
  for (int i = 0; i < Piece<T>::W; ++i) v.u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return v;
}

template <class T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& v) {
#pragma unroll
  for (int i = 0; i < Piece<T>::W; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, v.u[i]);
}

__device__ __forceinline__ void to_floats(const Piece<__half>& v, float (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v.u[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void to_floats(const Piece<__nv_bfloat16>& v, float (&f)[8]) {
  const u32 w[4] = {v.u[0].x, v.u[0].y, v.u[0].z, v.u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of the fp32 of the same value
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void to_floats(const Piece<float>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(v.u[i].x), f[4 * i + 1] = __uint_as_float(v.u[i].y);
    f[4 * i + 2] = __uint_as_float(v.u[i].z), f[4 * i + 3] = __uint_as_float(v.u[i].w);
  }
}

__device__ __forceinline__ void from_floats(Piece<__half>& v, const float (&f)[8]) {
  __half2* h = reinterpret_cast<__half2*>(&v.u[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void from_floats(Piece<__nv_bfloat16>& v, const float (&f)[8]) {
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v.u[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void from_floats(Piece<float>& v, const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v.u[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                        __float_as_uint(f[4 * i + 3]));
}

// ---------------------------------------------------------------- blocks of 8 codes

// Exponent byte from which codes stop at 63 (see above): the largest magnitude rounds up past the
// top binade of the type.
template <class T>
struct BlockLimit {
  static constexpr u32 top = 249;
};
template <>
struct BlockLimit<__half> {
  static constexpr u32 top = 137;
};

struct Block8 {
  uint2 codes;
  u32 exponent;
};

template <class T>
__device__ __forceinline__ Block8 encode_block(const float (&f)[8]) {
  u32 m = 0;  // magnitudes compare as integers; infinities and NaNs above every finite one
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  Block8 b;
  if (m >= 0x7f800000u) {
    b.codes = make_uint2(0u, 0u);
    b.exponent = 255u;
    return b;
  }
  // exponent field of the largest magnitude, one more where its mantissa is 127/64 or above 127.5/64
  const u32 e = (m + 0x10000u) >> 23;
  b.exponent = e > 7u ? e - 6u : 1u;
  const float inv = __uint_as_float((254u - b.exponent) << 23);
  // f * inv + 1.5 * 2^23 is rounded once, at the unit: its low byte is the code in two's complement
  constexpr float magic = 12582912.f;
  u32 t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = __float_as_uint(fmaf(f[i], inv, magic));
  if (b.exponent >= BlockLimit<T>::top) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      t[i] = __float_as_uint(fminf(fmaxf(__uint_as_float(t[i]), magic - 63.f), magic + 63.f));
  }
  b.codes.x = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
  b.codes.y = __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410);
  return b;
}

__device__ __forceinline__ void decode_block(const Block8& b, float (&f)[8]) {
  // 2^(E - 127); the byte 255 gives a NaN
  const float scale = __uint_as_float(b.exponent == 255u ? 0x7fc00000u : b.exponent << 23);
  // 2^23 + (code + 128) as a float, by placing the byte in the mantissa
  const u32 x = b.codes.x ^ 0x80808080u, y = b.codes.y ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = (__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7540 + i)) - 8388736.f) * scale;
    f[4 + i] = (__uint_as_float(__byte_perm(y, 0x4b000000u, 0x7540 + i)) - 8388736.f) * scale;
  }
}

}  // namespace spio_b200

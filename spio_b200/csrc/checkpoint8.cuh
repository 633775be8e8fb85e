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
// the channels over threads and CTAs sees whole blocks.  1.125 bytes a value; for normal data
// the largest magnitude of 8 values is 1.78 standard deviations on average, and the step 1 / 49 of one.
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

// (The kernels start while the one before them may still be writing what they read, and wait for it: so these are
// loads that stay behind the wait, and that do not take the data for constant during the kernel.)
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> v;
#pragma unroll
  for (int i = 0; i < Piece<T>::W; ++i) v.u[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
  return v;
}

// A piece is stored by one instruction: 32 bytes of fp32 data as two of 16 leave the caches half sectors to put
// together (restoring 51 million fp32 values took 58 us that way, 40 now).
template <class T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& v) {
  __stcs(reinterpret_cast<uint4*>(p), v.u[0]);
}
__device__ __forceinline__ void store_piece(float* p, const Piece<float>& v) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.u[0].x), "r"(v.u[0].y),
               "r"(v.u[0].z), "r"(v.u[0].w), "r"(v.u[1].x), "r"(v.u[1].y), "r"(v.u[1].z), "r"(v.u[1].w)
               : "memory");
}
// The same for data that is read next: no hint that it may leave L2 first.
template <class T>
__device__ __forceinline__ void store_piece_keep(T* p, const Piece<T>& v) {
  *reinterpret_cast<uint4*>(p) = v.u[0];
}
__device__ __forceinline__ void store_piece_keep(float* p, const Piece<float>& v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.u[0].x), "r"(v.u[0].y),
               "r"(v.u[0].z), "r"(v.u[0].w), "r"(v.u[1].x), "r"(v.u[1].y), "r"(v.u[1].z), "r"(v.u[1].w)
               : "memory");
}

// Two fp32 values in a register pair: sm_100 adds, multiplies and fuses them with one instruction, which
// halves the issue slots of the kernels here (they would be issue bound otherwise).
struct Pair {
  u64 v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ Pair pair(float both) { return pair(both, both); }
__device__ __forceinline__ float2 unpair(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// The 8 values of a piece as fp32.
struct Values {
  Pair p[4];
};

__device__ __forceinline__ Values values_of(const Piece<__half>& v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v.u[0]);
  Values r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    r.p[i] = pair(t.x, t.y);
  }
  return r;
}
__device__ __forceinline__ Values values_of(const Piece<__nv_bfloat16>& v) {
  const u32 w[4] = {v.u[0].x, v.u[0].y, v.u[0].z, v.u[0].w};
  Values r;
#pragma unroll
  for (int i = 0; i < 4; ++i)  // a bf16 is the upper half of the fp32 of the same value
    r.p[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  return r;
}
__device__ __forceinline__ Values values_of(const Piece<float>& v) {
  Values r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r.p[2 * i] = pair(__uint_as_float(v.u[i].x), __uint_as_float(v.u[i].y));
    r.p[2 * i + 1] = pair(__uint_as_float(v.u[i].z), __uint_as_float(v.u[i].w));
  }
  return r;
}

// Rounded once, to the piece's type.
__device__ __forceinline__ void to_piece(Piece<__half>& v, const Values& f) {
  __half2* h = reinterpret_cast<__half2*>(&v.u[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __float22half2_rn(unpair(f.p[i]));
}
__device__ __forceinline__ void to_piece(Piece<__nv_bfloat16>& v, const Values& f) {
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v.u[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __float22bfloat162_rn(unpair(f.p[i]));
}
__device__ __forceinline__ void to_piece(Piece<float>& v, const Values& f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = unpair(f.p[2 * i]), b = unpair(f.p[2 * i + 1]);
    v.u[i] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  }
}

// Bits of the largest magnitude, as an fp32: magnitudes compare as integers, infinities and NaNs above
// every finite one.
__device__ __forceinline__ u32 largest_of_words(const uint4& u) {
  const u32 m = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
}
__device__ __forceinline__ u32 largest_magnitude(const Piece<__half>& v) {
  const u32 w = largest_of_words(v.u[0]);
  const u32 m = max(w & 0xffffu, w >> 16);
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}
__device__ __forceinline__ u32 largest_magnitude(const Piece<__nv_bfloat16>& v) {
  const u32 w = largest_of_words(v.u[0]);
  return max(w << 16, w & 0xffff0000u);
}
__device__ __forceinline__ u32 largest_magnitude(const Piece<float>& v) {
  u32 m = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32 k = 0x7fffffffu;
    m = max(m, max(max(v.u[i].x & k, v.u[i].y & k), max(v.u[i].z & k, v.u[i].w & k)));
  }
  return m;
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

// `f`: the values of `v`.
template <class T>
__device__ __forceinline__ Block8 encode_block(const Piece<T>& v, const Values& f) {
  const u32 m = largest_magnitude(v);
  Block8 b;
  if (m >= 0x7f800000u) {
    b.codes = make_uint2(0u, 0u);
    b.exponent = 255u;
    return b;
  }
  // exponent field of the largest magnitude, one more where its mantissa is 127.5 / 64 or above
  const u32 e = (m + 0x10000u) >> 23;
  b.exponent = e > 7u ? e - 6u : 1u;
  const Pair inv = pair(__uint_as_float((254u - b.exponent) << 23));
  // f * inv + 1.5 * 2^23 is rounded once, at the unit: its low byte is the code in two's complement
  constexpr float magic = 12582912.f;
  float t[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 c = unpair(fma2(f.p[i], inv, pair(magic)));
    t[2 * i] = c.x, t[2 * i + 1] = c.y;
  }
  if (b.exponent >= BlockLimit<T>::top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = fminf(fmaxf(t[i], magic - 63.f), magic + 63.f);
  }
  u32 c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = __byte_perm(__float_as_uint(t[2 * i]), __float_as_uint(t[2 * i + 1]), 0x0040);
  b.codes = make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
  return b;
}

__device__ __forceinline__ Values decode_block(const Block8& b) {
  // 2^(E - 127); the byte 255 gives a NaN
  const Pair scale = pair(__uint_as_float(b.exponent == 255u ? 0x7fc00000u : b.exponent << 23));
  // 2^23 + (code + 128) as a float, by placing the byte in the mantissa
  const u32 w[2] = {b.codes.x ^ 0x80808080u, b.codes.y ^ 0x80808080u};
  const Pair offset = pair(-8388736.f);
  Values r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 u = w[i >> 1];
    const int k = 2 * (i & 1);
    r.p[i] = (pair(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + k)),
                   __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541 + k))) + offset) * scale;
  }
  return r;
}

}  // namespace spio_b200

// Group norm with an activation on NHWC data, forward and backward.
//
//   mean, var over the pixels and the c / groups channels of a group of an image (M values)
//   rstd = 1 / sqrt(var + eps),  xhat = (x - mean) * rstd,  z = xhat * weight + bias,  y = act(z)
//   g = dy * act'(z),  dbias = sum_{n,p} g,  dweight = sum_{n,p} g * xhat
//   dx = rstd * (g * weight - s1 - xhat * s2),  s1 = mean_M(g * weight),  s2 = mean_M(g * weight * xhat)
//
// Statistics and sums are fp32.  A thread owns 8 channels (one piece) of the pixels r, r + R, ... of its
// CTA's part and sums differences to its first pixel: the pivot is one of the n samples, so
// (pivot - mean)^2 <= M2 and the cancellation in q - s^2 / n costs at most a factor n of the rounding
// error, whatever the data's offset.  Threads, channels, CTAs are then merged by their means and
// centred squares, in a fixed order: results do not vary from run to run.
#pragma once

#include <cuda_runtime.h>

#include "checkpoint8.cuh"
#include "groupnorm_2d.h"

namespace spio_b200 {

// ---------------------------------------------------------------- activations

// EXACT: for fp32 data, CUDA's own functions.  Otherwise results are rounded to 11 bits or fewer and
// the hardware's exponential and reciprocal (2^-22) are far below that; erfc is Abramowitz and
// Stegun's 7.1.26 (absolute error 1.5e-7, and a factor exp(-x^2) that keeps the tail's relative error
// below the rounding of 16-bit types).
template <int ACT, bool EXACT>
struct Activation {
  static __device__ __forceinline__ float sigmoid(float z) {
    if (EXACT) return 1.f / (1.f + expf(-z));
    return __fdividef(1.f, 1.f + __expf(-z));
  }
  // Phi(z) and exp(-z^2 / 2)
  static __device__ __forceinline__ float normal_cdf(float z, float* e) {
    if (EXACT) {
      *e = expf(-0.5f * z * z);
      return 0.5f * erfcf(-0.70710678118654752f * z);
    }
    *e = __expf(-0.5f * z * z);
    const float u = fabsf(z) * 0.70710678118654752f;
    const float t = __fdividef(1.f, fmaf(0.3275911f, u, 1.f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float tail = 0.5f * p * t * *e;
    return z < 0.f ? tail : 1.f - tail;
  }
  static __device__ __forceinline__ float value(float z) {
    if (ACT == kActRelu) return z < 0.f ? 0.f : z;  // a NaN stays one
    if (ACT == kActSilu) return z * sigmoid(z);
    if (ACT == kActGelu) {
      float e;
      return z * normal_cdf(z, &e);
    }
    return z;
  }
  static __device__ __forceinline__ float slope(float z) {
    if (ACT == kActRelu) return z <= 0.f ? 0.f : 1.f;
    if (ACT == kActSilu) {
      const float s = sigmoid(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    if (ACT == kActGelu) {
      float e;
      const float p = normal_cdf(z, &e);
      return fmaf(z * 0.3989422804014327f, e, p);
    }
    return 1.f;
  }
};

template <class T>
struct IsExact {
  static constexpr bool value = sizeof(T) == 4;
};

// ---------------------------------------------------------------- work of a thread

struct GnWork {
  long long image;
  int slab, part;
  int sp;        // pieces of this slab
  int first;     // first piece of the slab
  int rows;      // rows of threads: pixels worked on at a time
  int r, p;      // this thread's row and piece; r >= rows: none
  int px0, px1;  // pixels of the part
  bool on;
};

__device__ __forceinline__ GnWork gn_work(const GnGeom& g) {
  GnWork w;
  const int b = (int)(blockIdx.x % (unsigned)(g.parts * g.slabs));
  w.image = blockIdx.x / (unsigned)(g.parts * g.slabs);
  w.part = b % g.parts;
  w.slab = b / g.parts;
  w.first = w.slab * g.sp;
  w.sp = min(g.sp, g.pieces - w.first);
  w.rows = kGnThreads / w.sp;
  w.r = threadIdx.x / w.sp;
  w.p = threadIdx.x - w.r * w.sp;
  w.px0 = w.part * g.part_px;
  w.px1 = w.px0 + min(g.part_px, g.pixels - w.px0);
  w.on = w.r < w.rows;
  return w;
}

// index of the first value of piece (pixel, w.p) of the image
__device__ __forceinline__ long long gn_offset(const GnGeom& g, const GnWork& w, int pixel) {
  return (w.image * g.pixels + pixel) * g.c + (long long)(w.first + w.p) * 8;
}

// ---------------------------------------------------------------- sums over a CTA

// Shared memory of the reductions: the tree's staging, then per-channel and per-group values.
struct GnShared {
  float4 tree[4][kGnThreads];
  float ref[kGnMaxSlabPieces * 8];
};

// Adds a[] and b[] of the threads of one piece over the rows; row 0 has the sums afterwards.  The
// halves are folded pairwise, so the order is fixed.
__device__ __forceinline__ void gn_sum_rows(float (&a)[8], float (&b)[8], const GnWork& w, GnShared* sm) {
  int base = 0;  // staging rows used so far: half + half / 2 + ... < rows
  for (int rows = w.rows; rows > 1;) {
    const int half = (rows + 1) >> 1;
    if (w.r >= half && w.r < rows) {
      const int at = (base + w.r - half) * w.sp + w.p;
      sm->tree[0][at] = make_float4(a[0], a[1], a[2], a[3]);
      sm->tree[1][at] = make_float4(a[4], a[5], a[6], a[7]);
      sm->tree[2][at] = make_float4(b[0], b[1], b[2], b[3]);
      sm->tree[3][at] = make_float4(b[4], b[5], b[6], b[7]);
    }
    __syncthreads();
    if (w.r < rows - half) {
      const int at = (base + w.r) * w.sp + w.p;
      const float4 a0 = sm->tree[0][at], a1 = sm->tree[1][at], b0 = sm->tree[2][at], b1 = sm->tree[3][at];
      a[0] += a0.x, a[1] += a0.y, a[2] += a0.z, a[3] += a0.w;
      a[4] += a1.x, a[5] += a1.y, a[6] += a1.z, a[7] += a1.w;
      b[0] += b0.x, b[1] += b0.y, b[2] += b0.z, b[3] += b0.w;
      b[4] += b1.x, b[5] += b1.y, b[6] += b1.z, b[7] += b1.w;
    }
    base += rows - half;
    rows = half;
  }
}

// Sums of a thread over its pixels, as differences to its first one.
struct GnSums {
  float pivot[8], s[8], q[8];
  int n;
  __device__ __forceinline__ void clear() {
    n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) pivot[i] = s[i] = q[i] = 0.f;
  }
  __device__ __forceinline__ void add(const float (&f)[8]) {
    if (n == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) pivot[i] = f[i];
    }
    ++n;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = f[i] - pivot[i];
      s[i] += d;
      q[i] = fmaf(d, d, q[i]);
    }
  }
};

__device__ __forceinline__ float not_below_zero(float v) { return v < 0.f ? 0.f : v; }  // a NaN stays one

// Mean and sum of centred squares of the groups of the slab over the CTA's pixels, by all threads:
// put(group of the slab, mean, m2) is called once for each group by some thread.
template <class Put>
__device__ __forceinline__ void gn_group_stats(const GnGeom& g, const GnWork& w, GnSums& t, GnShared* sm, Put put) {
  // to differences from row 0's mean, which every row can add up
  float a[8], b[8];
  const float n = (float)t.n, inv = t.n > 0 ? 1.f / n : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = t.s[i] * inv;
    b[i] = not_below_zero(t.q[i] - t.s[i] * a[i]);  // centred squares of this thread's pixels
    a[i] += t.pivot[i];
  }
  if (w.r == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sm->ref[w.p * 8 + i] = a[i];
  }
  __syncthreads();
  float ref[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ref[i] = 0.f;
  if (w.on) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ref[i] = sm->ref[w.p * 8 + i];
      const float d = t.n > 0 ? a[i] - ref[i] : 0.f;
      a[i] = n * d;
      b[i] = fmaf(a[i], d, b[i]);
    }
  }
  gn_sum_rows(a, b, w, sm);
  const int px = w.px1 - w.px0;
  float* mean = sm->ref;                                // [channel of the slab]
  float* m2 = reinterpret_cast<float*>(&sm->tree[0][0]);  // the staging is free after the sync
  __syncthreads();
  if (w.r == 0) {
    const float inv_px = 1.f / (float)px;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = a[i] * inv_px;
      mean[w.p * 8 + i] = ref[i] + d;
      m2[w.p * 8 + i] = not_below_zero(b[i] - a[i] * d);
    }
  }
  __syncthreads();
  const int groups = w.sp * 8 / g.cpg;
  const float inv_cpg = 1.f / (float)g.cpg;
  if (g.cpg <= 32) {  // a thread for each group
    for (int k = threadIdx.x; k < groups; k += kGnThreads) {
      const float m0 = mean[k * g.cpg];  // (differences: the mean of equal values is that value)
      float s = 0.f, q = 0.f;
      for (int i = 0; i < g.cpg; ++i) s += mean[k * g.cpg + i] - m0;
      s = fmaf(s, inv_cpg, m0);
      for (int i = 0; i < g.cpg; ++i) {
        const float d = mean[k * g.cpg + i] - s;
        q += fmaf((float)px * d, d, m2[k * g.cpg + i]);
      }
      put(k, s, q);
    }
  } else {  // a warp for each group
    const int lane = threadIdx.x & 31;
    for (int k = threadIdx.x >> 5; k < groups; k += kGnThreads / 32) {
      const float m0 = mean[k * g.cpg];
      float s = 0.f, q = 0.f;
      for (int i = lane; i < g.cpg; i += 32) s += mean[k * g.cpg + i] - m0;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      s = fmaf(s, inv_cpg, m0);
      for (int i = lane; i < g.cpg; i += 32) {
        const float d = mean[k * g.cpg + i] - s;
        q += fmaf((float)px * d, d, m2[k * g.cpg + i]);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) q += __shfl_xor_sync(0xffffffffu, q, d);
      if (lane == 0) put(k, s, q);
    }
  }
}

// Sums of the per-channel values a[], b[] (held by row 0) over the channels of each group.
template <class Put>
__device__ __forceinline__ void gn_group_sums(const GnGeom& g, const GnWork& w, const float (&a)[8],
                                              const float (&b)[8], GnShared* sm, Put put) {
  float* sa = sm->ref;
  float* sb = reinterpret_cast<float*>(&sm->tree[0][0]);
  __syncthreads();
  if (w.r == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sa[w.p * 8 + i] = a[i], sb[w.p * 8 + i] = b[i];
  }
  __syncthreads();
  const int groups = w.sp * 8 / g.cpg;
  if (g.cpg <= 32) {
    for (int k = threadIdx.x; k < groups; k += kGnThreads) {
      float s = 0.f, q = 0.f;
      for (int i = 0; i < g.cpg; ++i) s += sa[k * g.cpg + i], q += sb[k * g.cpg + i];
      put(k, s, q);
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int k = threadIdx.x >> 5; k < groups; k += kGnThreads / 32) {
      float s = 0.f, q = 0.f;
      for (int i = lane; i < g.cpg; i += 32) s += sa[k * g.cpg + i], q += sb[k * g.cpg + i];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, d);
        q += __shfl_xor_sync(0xffffffffu, q, d);
      }
      if (lane == 0) put(k, s, q);
    }
  }
}

// What a thread needs of its 8 channels.
struct GnChannels {
  float mean[8], rstd[8], weight[8], bias[8];
};

// stat(group of the slab) gives {mean, rstd}
template <class Stat>
__device__ __forceinline__ void gn_channels(GnChannels& c, const GnGeom& g, const GnWork& w,
                                            const float* __restrict__ weight, const float* __restrict__ bias,
                                            Stat stat) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int local = w.p * 8 + i, channel = w.first * 8 + local;
    const float2 st = stat(local / g.cpg);
    c.mean[i] = st.x;
    c.rstd[i] = st.y;
    c.weight[i] = weight != nullptr ? __ldg(weight + channel) : 1.f;
    c.bias[i] = bias != nullptr ? __ldg(bias + channel) : 0.f;
  }
}

// ---------------------------------------------------------------- forward, two kernels

constexpr int kGnBatch = 4;  // pieces a thread has in flight

// part_stats[(image * groups + group) * parts + part] = {mean, centred squares} over the part's pixels
template <class T>
__global__ void __launch_bounds__(kGnThreads)
groupnorm_2d_stats_kernel(float2* __restrict__ part_stats, const T* __restrict__ x, const GnGeom g) {
  __shared__ GnShared sm;
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g);
  GnSums t;
  t.clear();
  if (w.on) {
    for (int i = w.px0 + w.r; i < w.px1; i += kGnBatch * w.rows) {
      Piece<T> v[kGnBatch];
#pragma unroll
      for (int k = 0; k < kGnBatch; ++k)
        if (i + k * w.rows < w.px1) v[k] = load_piece(x + gn_offset(g, w, i + k * w.rows));
#pragma unroll
      for (int k = 0; k < kGnBatch; ++k)
        if (i + k * w.rows < w.px1) {
          float f[8];
          to_floats(v[k], f);
          t.add(f);
        }
    }
  }
  const long long first_group = w.image * g.groups + w.first * 8 / g.cpg;
  gn_group_stats(g, w, t, &sm, [&](int k, float mean, float m2) {
    part_stats[(first_group + k) * g.parts + w.part] = make_float2(mean, m2);
  });
}

// Mean and rstd of the slab's groups from the parts' values, into stat[]; all threads, synchronised.
__device__ __forceinline__ void gn_merge_parts(float2* stat, const GnGeom& g, const GnWork& w,
                                               const float2* __restrict__ part_stats) {
  const int groups = w.sp * 8 / g.cpg;
  const long long first_group = w.image * g.groups + w.first * 8 / g.cpg;
  const int lane = threadIdx.x & 31;
  const float inv_pixels = 1.f / (float)g.pixels;
  for (int k = threadIdx.x >> 5; k < groups; k += kGnThreads / 32) {
    const float2* ps = part_stats + (first_group + k) * g.parts;
    const float m0 = __ldcg(ps).x;
    float s = 0.f, q = 0.f;
    for (int i = lane; i < g.parts; i += 32) {
      const float n = (float)min(g.part_px, g.pixels - i * g.part_px);
      s = fmaf(n, __ldcg(ps + i).x - m0, s);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s = fmaf(s, inv_pixels, m0);
    for (int i = lane; i < g.parts; i += 32) {
      const float n = (float)min(g.part_px, g.pixels - i * g.part_px) * (float)g.cpg;
      const float2 v = __ldcg(ps + i);
      const float d = v.x - s;
      q += fmaf(n * d, d, v.y);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) q += __shfl_xor_sync(0xffffffffu, q, d);
    if (lane == 0) stat[k] = make_float2(s, 1.f / sqrtf(fmaf(q, g.inv_m, g.eps)));
  }
  __syncthreads();
}

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads)
groupnorm_2d_apply_kernel(T* __restrict__ y, float2* __restrict__ stats, uint2* __restrict__ codes,
                          unsigned char* __restrict__ exponents, const T* __restrict__ x,
                          const float* __restrict__ weight, const float* __restrict__ bias,
                          const float2* __restrict__ part_stats, const GnGeom g) {
  __shared__ float2 stat[kGnMaxSlabPieces * 8];
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g);
  gn_merge_parts(stat, g, w, part_stats);
  if (stats != nullptr && w.part == 0) {
    const int groups = w.sp * 8 / g.cpg;
    for (int k = threadIdx.x; k < groups; k += kGnThreads)
      stats[w.image * g.groups + w.first * 8 / g.cpg + k] = stat[k];
  }
  if (!w.on) return;
  GnChannels c;
  gn_channels(c, g, w, weight, bias, [&](int k) { return stat[k]; });
#pragma unroll
  for (int i = 0; i < 8; ++i) c.weight[i] *= c.rstd[i];
  for (int i = w.px0 + w.r; i < w.px1; i += kGnBatch * w.rows) {
    Piece<T> v[kGnBatch];
#pragma unroll
    for (int k = 0; k < kGnBatch; ++k)
      if (i + k * w.rows < w.px1) v[k] = load_piece_streaming(x + gn_offset(g, w, i + k * w.rows));
#pragma unroll
    for (int k = 0; k < kGnBatch; ++k)
      if (i + k * w.rows < w.px1) {
        const long long at = gn_offset(g, w, i + k * w.rows);
        float f[8];
        to_floats(v[k], f);
        if (CODES) {
          const Block8 b = encode_block<T>(f);
          codes[at >> 3] = b.codes;
          exponents[at >> 3] = (unsigned char)b.exponent;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          f[j] = Activation<ACT, IsExact<T>::value>::value(fmaf(f[j] - c.mean[j], c.weight[j], c.bias[j]));
        Piece<T> o;
        from_floats(o, f);
        store_piece(y + at, o);
      }
  }
}

// ---------------------------------------------------------------- backward, three kernels

// The input of the norm as it was kept for the backward pass.
template <class T, bool CODES>
struct GnInput {
  Piece<T> v;
  __device__ __forceinline__ void load(const T* x, const uint2*, const unsigned char*, long long at) {
    v = load_piece(x + at);
  }
  __device__ __forceinline__ void floats(float (&f)[8]) const { to_floats(v, f); }
};
template <class T>
struct GnInput<T, true> {
  Block8 b;
  __device__ __forceinline__ void load(const T*, const uint2* codes, const unsigned char* exponents, long long at) {
    b.codes = __ldg(codes + (at >> 3));
    b.exponent = __ldg(exponents + (at >> 3));
  }
  __device__ __forceinline__ void floats(float (&f)[8]) const { decode_block(b, f); }
};

// part_channel[(image * parts + part) * 2 + {0, 1}][c] = sums of g * xhat and of g over the part's pixels;
// part_group[(image * groups + group) * parts + part] = their weighted sums over a group's channels.
template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 2)
groupnorm_2d_bwd_sums_kernel(float* __restrict__ part_channel, float2* __restrict__ part_group,
                             const T* __restrict__ dy, const T* __restrict__ x, const uint2* __restrict__ codes,
                             const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                             const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  __shared__ GnShared sm;
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g);
  const long long first_group = w.image * g.groups + w.first * 8 / g.cpg;
  GnChannels c;
  float sa[8], sb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sa[i] = sb[i] = 0.f;
  if (w.on) {
    gn_channels(c, g, w, weight, bias, [&](int k) { return __ldg(stats + first_group + k); });
    for (int i = w.px0 + w.r; i < w.px1; i += 2 * w.rows) {
      GnInput<T, CODES> v[2];
      Piece<T> d[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (i + k * w.rows < w.px1) {
          const long long at = gn_offset(g, w, i + k * w.rows);
          v[k].load(x, codes, exponents, at);
          d[k] = load_piece(dy + at);
        }
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (i + k * w.rows < w.px1) {
          float f[8], e[8];
          v[k].floats(f);
          to_floats(d[k], e);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float hat = (f[j] - c.mean[j]) * c.rstd[j];
            const float grad =
                e[j] * Activation<ACT, IsExact<T>::value>::slope(fmaf(hat, c.weight[j], c.bias[j]));
            sa[j] = fmaf(grad, hat, sa[j]);
            sb[j] += grad;
          }
        }
    }
  }
  gn_sum_rows(sa, sb, w, &sm);
  if (w.r == 0) {
    if (part_channel != nullptr) {
      float* at = part_channel + ((w.image * g.parts + w.part) * 2) * g.c + (w.first + w.p) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) at[i] = sa[i], at[g.c + i] = sb[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sa[i] *= c.weight[i], sb[i] *= c.weight[i];
  }
  if (part_group != nullptr)
    gn_group_sums(g, w, sa, sb, &sm,
                  [&](int k, float s, float q) { part_group[(first_group + k) * g.parts + w.part] = make_float2(s, q); });
}

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 2)
groupnorm_2d_bwd_apply_kernel(T* __restrict__ dx, const float2* __restrict__ part_group, const T* __restrict__ dy,
                              const T* __restrict__ x, const uint2* __restrict__ codes,
                              const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                              const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  __shared__ float2 mean_of[kGnMaxSlabPieces * 8];  // of g * weight * xhat and g * weight, over a group
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g);
  const long long first_group = w.image * g.groups + w.first * 8 / g.cpg;
  {
    const int groups = w.sp * 8 / g.cpg, lane = threadIdx.x & 31;
    for (int k = threadIdx.x >> 5; k < groups; k += kGnThreads / 32) {
      float s = 0.f, q = 0.f;
      for (int i = lane; i < g.parts; i += 32) {
        const float2 v = __ldcg(part_group + (first_group + k) * g.parts + i);
        s += v.x, q += v.y;
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, d);
        q += __shfl_xor_sync(0xffffffffu, q, d);
      }
      if (lane == 0) mean_of[k] = make_float2(s * g.inv_m, q * g.inv_m);
    }
  }
  __syncthreads();
  if (!w.on) return;
  GnChannels c;
  gn_channels(c, g, w, weight, bias, [&](int k) { return __ldg(stats + first_group + k); });
  float s1[8], s2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = mean_of[(w.p * 8 + i) / g.cpg];
    s2[i] = v.x, s1[i] = v.y;
  }
  for (int i = w.px0 + w.r; i < w.px1; i += 2 * w.rows) {
    GnInput<T, CODES> v[2];
    Piece<T> d[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (i + k * w.rows < w.px1) {
        const long long at = gn_offset(g, w, i + k * w.rows);
        v[k].load(x, codes, exponents, at);
        d[k] = load_piece(dy + at);
      }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (i + k * w.rows < w.px1) {
        float f[8], e[8];
        v[k].floats(f);
        to_floats(d[k], e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float hat = (f[j] - c.mean[j]) * c.rstd[j];
          const float grad = e[j] * Activation<ACT, IsExact<T>::value>::slope(fmaf(hat, c.weight[j], c.bias[j]));
          f[j] = c.rstd[j] * (fmaf(grad, c.weight[j], -s1[j]) - hat * s2[j]);
        }
        Piece<T> o;
        from_floats(o, f);
        store_piece(dx + gn_offset(g, w, i + k * w.rows), o);
      }
  }
}

}  // namespace spio_b200

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
// error, whatever the data's offset.  The threads' sums give the CTA's mean of each group, then their
// squares are moved to that mean and added; CTAs are merged by means and centred squares.  All in a
// fixed order: results do not vary from run to run.
#pragma once

#include <cuda_runtime.h>

#include "checkpoint8.cuh"
#include "groupnorm_2d.h"

#ifndef GN_THREADS
#define GN_THREADS 256
#endif

namespace spio_b200 {
namespace GN_NAMESPACE {

constexpr int kGnThreads = GN_THREADS;  // of a CTA; a thread owns at most one piece of a pixel's slab

// ---------------------------------------------------------------- activations

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// EXACT: for fp32 data, CUDA's own functions.  Otherwise results are rounded to 11 bits or fewer, and the
// hardware's exponential and reciprocal (relative errors of some 2^-22) are far below that; erfc is
// Abramowitz and Stegun's 7.1.26 (absolute error 1.5e-7, with a factor exp(-x^2) that keeps the tail's
// relative error below the rounding of 16-bit types).
template <int ACT, bool EXACT>
struct Activation {
  static __device__ __forceinline__ float exact_sigmoid(float z) { return 1.f / (1.f + expf(-z)); }
  static __device__ __forceinline__ float exact_cdf(float z) { return 0.5f * erfcf(-0.70710678118654752f * z); }

  static __device__ __forceinline__ Pair sigmoid(Pair z) {
    const float2 t = unpair(z * pair(-1.4426950408889634f));
    const float2 d = unpair(pair(exp2_approx(t.x), exp2_approx(t.y)) + pair(1.f));
    return pair(reciprocal_approx(d.x), reciprocal_approx(d.y));
  }
  // Phi(z) and exp(-z^2 / 2)
  static __device__ __forceinline__ Pair normal_cdf(Pair z, Pair* e) {
    const float2 zs = unpair(z);
    const float2 q = unpair(z * z * pair(-0.72134752044448170f));
    *e = pair(exp2_approx(q.x), exp2_approx(q.y));
    const float2 d = unpair(fma2(pair(fabsf(zs.x), fabsf(zs.y)), pair(0.3275911f * 0.70710678118654752f), pair(1.f)));
    const Pair t = pair(reciprocal_approx(d.x), reciprocal_approx(d.y));
    Pair p = fma2(t, pair(0.5f * 1.061405429f), pair(0.5f * -1.453152027f));
    p = fma2(p, t, pair(0.5f * 1.421413741f));
    p = fma2(p, t, pair(0.5f * -0.284496736f));
    p = fma2(p, t, pair(0.5f * 0.254829592f));
    const float2 tail = unpair(p * t * *e);
    return pair(zs.x < 0.f ? tail.x : 1.f - tail.x, zs.y < 0.f ? tail.y : 1.f - tail.y);
  }

  static __device__ __forceinline__ Pair value(Pair z) {
    const float2 f = unpair(z);
    if (ACT == kActRelu) return pair(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);  // a NaN stays one
    if (ACT == kActSilu) return z * (EXACT ? pair(exact_sigmoid(f.x), exact_sigmoid(f.y)) : sigmoid(z));
    if (ACT == kActGelu) {
      Pair e;
      return z * (EXACT ? pair(exact_cdf(f.x), exact_cdf(f.y)) : normal_cdf(z, &e));
    }
    return z;
  }
  // grad * act'(z)
  static __device__ __forceinline__ Pair back(Pair grad, Pair z) {
    const float2 f = unpair(z);
    if (ACT == kActRelu) return grad * pair(f.x <= 0.f ? 0.f : 1.f, f.y <= 0.f ? 0.f : 1.f);
    if (ACT == kActSilu) {
      const Pair s = EXACT ? pair(exact_sigmoid(f.x), exact_sigmoid(f.y)) : sigmoid(z);
      return grad * fma2(z * s, fma2(s, pair(-1.f), pair(1.f)), s);
    }
    if (ACT == kActGelu) {
      Pair e, p;
      if (EXACT) {
        e = pair(expf(-0.5f * f.x * f.x), expf(-0.5f * f.y * f.y));
        p = pair(exact_cdf(f.x), exact_cdf(f.y));
      } else {
        p = normal_cdf(z, &e);
      }
      return grad * fma2(z * pair(0.3989422804014327f), e, p);
    }
    return grad;
  }
};

template <class T>
struct IsExact {
  static constexpr bool value = sizeof(T) == 4;
};

// ---------------------------------------------------------------- work of a thread

__device__ __forceinline__ int gn_part_pixels(const GnGeom& g, int part) { return g.part_px + (part < g.part_rest); }

struct GnWork {
  long long image;
  int part;
  int sp;        // pieces of this slab
  int first;     // first piece of the slab
  int groups;    // of the slab
  int rows;      // rows of threads: pixels worked on at a time
  int r, p;      // this thread's row and piece; r >= rows: none
  int px0, px;   // first pixel of the part, pixels of it
  bool on;
};

// Integer divisions of small numbers.  (A CTA's bookkeeping is paid by every warp of it, for a few thousand
// pieces of work; with the compiler's general divisions it was 1500 instructions a thread, as many as 20 pieces.)

// The group of the slab that channel `local` of it is in: magic = ceil(2^32 / cpg) is less than one too large, which
// is off by less than 2048 / 2^32 here.
__device__ __forceinline__ int gn_group(const GnGeom& g, int local) {
  return g.cpg == 1 ? local : (int)__umulhi((unsigned)local, g.cpg_magic);
}
// a / b with inv_b = 1 / b rounded, for a < 2^20: (a + 0.5) / b is 1 / (2 * b) off a whole number at least
__device__ __forceinline__ int divide(int a, float inv_b) { return (int)(((float)a + 0.5f) * inv_b); }

// CTAs in order: parts of a slab, slabs of an image, images.
__device__ __forceinline__ GnWork gn_work(const GnGeom& g, unsigned block) {
  GnWork w;
  unsigned unit = block;
  w.part = 0;
  if (g.parts > 1) {
    unit = block / (unsigned)g.parts;
    w.part = (int)(block - unit * g.parts);
  }
  w.first = 0;
  w.image = unit;
  w.sp = g.sp;
  float inv_sp = g.inv_sp;
  if (g.slabs > 1) {
    const unsigned image = unit / (unsigned)g.slabs;
    w.image = image;
    w.first = (int)(unit - image * g.slabs) * g.sp;
    if (g.pieces - w.first < g.sp) {  // the last slab may be narrower
      w.sp = g.pieces - w.first;
      inv_sp = 1.f / (float)w.sp;
    }
  }
  w.groups = gn_group(g, w.sp * 8 - 1) + 1;
  w.rows = divide(kGnThreads, inv_sp);
  w.r = divide(threadIdx.x, inv_sp);
  w.p = threadIdx.x - w.r * w.sp;
  w.px0 = w.part * g.part_px + min(w.part, g.part_rest);
  w.px = gn_part_pixels(g, w.part);
  w.on = w.r < w.rows;
  return w;
}

// Index of the slab's first group.  (A slab begins with whole groups; their index may pass 2048.)
__device__ __forceinline__ long long gn_first_group(const GnGeom& g, const GnWork& w) {
  return w.image * g.groups + (w.first == 0 ? 0 : w.first / g.sp * g.slab_groups);
}

// index of the first value of piece (pixel, w.p) of the image
__device__ __forceinline__ long long gn_offset(const GnGeom& g, const GnWork& w, int pixel) {
  return (w.image * g.pixels + pixel) * g.c + (long long)(w.first + w.p) * 8;
}

// ---------------------------------------------------------------- sums over a CTA

// Shared memory of the reductions: two arrays of a value of each channel of each thread, or of each thread
// where a piece lies within one group (g.fold), and two values for each of the slab's groups.
struct GnReduce {
  float* a;
  float* b;        // (backward)
  float2* folded;  // (backward)
  float2* group;
};
constexpr int kGnPlane = kGnThreads * 8;

__device__ __forceinline__ GnReduce gn_reduce(void* at, const GnGeom& g) {
  GnReduce s;
  s.a = reinterpret_cast<float*>(at);
  s.b = s.a + kGnPlane;
  s.folded = reinterpret_cast<float2*>(s.b + kGnPlane);
  s.group = reinterpret_cast<float2*>(reinterpret_cast<char*>(at) + g.group_at);
  return s;
}

__device__ __forceinline__ float not_below_zero(float v) { return v < 0.f ? 0.f : v; }  // a NaN stays one

__device__ __forceinline__ void put8(float* at, const float (&v)[8]) {
  reinterpret_cast<float4*>(at)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(at)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float sum8(const float (&v)[8]) {
  return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// Over 2^log neighbouring lanes.
__device__ __forceinline__ float sum_lanes(float v, int log) {
#pragma unroll
  for (int i = 0; i < 5; ++i)
    if (i < log) v += __shfl_xor_sync(0xffffffffu, v, 1 << i);
  return v;
}

// body(group of the slab, lane of it, live) by the 2^g.lanes neighbouring lanes of each group, all lanes of a warp
// together; `live` where there is such a group.
template <class Body>
__device__ __forceinline__ void gn_groups(const GnGeom& g, const GnWork& w, Body body) {
  const int lane = threadIdx.x & ((1 << g.lanes) - 1), step = kGnThreads >> g.lanes;
  int k = threadIdx.x >> g.lanes;
  for (int base = 0; base < w.groups; base += step, k += step) body(k, lane, k < w.groups);
}

// Calls at(index, channel of the group) for this lane's share of the values of group k: every row's run of them.
template <class At>
__device__ __forceinline__ void gn_run(const GnGeom& g, const GnWork& w, int k, int lane, At at) {
  const int row = g.fold ? w.sp : w.sp * 8;
  int r = divide(lane, g.inv_run), j = lane - r * g.run;
#pragma unroll 4
  while (r < w.rows) {
    at(r * row + k * g.run + j, j);
    r += g.run_rows, j += g.run_rest;
    if (j >= g.run) j -= g.run, ++r;
  }
}

// Sums of a thread over its pixels, as differences to its first one.
struct GnSums {
  Values away, s, q;  // minus the pivot, sums, sums of squares
  int n;
  __device__ __forceinline__ void clear() {
    n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) away.p[i] = s.p[i] = q.p[i] = pair(0.f);
  }
  __device__ __forceinline__ void start(const Values& f) {  // sets the pivot, adds nothing
#pragma unroll
    for (int i = 0; i < 4; ++i) away.p[i] = f.p[i] * pair(-1.f);
  }
  __device__ __forceinline__ void add(const Values& f) {
    ++n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Pair d = f.p[i] + away.p[i];
      s.p[i] = s.p[i] + d;
      q.p[i] = fma2(d, d, q.p[i]);
    }
  }
};

// The 8 values as an array.
__device__ __forceinline__ void spread(const Values& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = unpair(v.p[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
}

// Values of the first pixel of the part, one of each group, to which first-order sums are taken (any value near
// the data does: it keeps the mean of far-off data exact).
template <class T>
__device__ __forceinline__ void gn_origin(float (&o)[8], const GnGeom& g, const GnWork& w, const T* __restrict__ x) {
  if (!w.on) return;
  const T* at = x + (w.image * g.pixels + w.px0) * g.c + w.first * 8;
  if (g.fold) {
    o[0] = (float)at[gn_group(g, w.p * 8) * g.cpg];
#pragma unroll
    for (int i = 1; i < 8; ++i) o[i] = o[0];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)at[gn_group(g, w.p * 8 + i) * g.cpg];
  }
}

// {mean, centred squares} of the groups of the slab over the CTA's pixels, to put(group of the slab, value), by
// all threads.
template <class Put>
__device__ __forceinline__ void gn_group_stats(const GnGeom& g, const GnWork& w, const GnSums& t, const float (&origin)[8],
                                               const GnReduce& red, Put put) {
  float s[8], q[8], d[8];
  const float n = (float)t.n, inv_n = t.n > 0 ? __fdividef(1.f, n) : 0.f;
  const float inv_values = __fdividef(1.f, (float)w.px * (float)g.cpg);  // values of a group in this part
  spread(t.s, s), spread(t.q, q), spread(t.away, d);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float m = s[i] * inv_n;
    q[i] = not_below_zero(q[i] - s[i] * m);  // about this thread's mean of the channel
    d[i] = (m - d[i]) - origin[i];           // that mean, from the origin
    s[i] = n * d[i];
  }
  if (w.on) {
    if (g.fold) red.a[threadIdx.x] = sum8(s);
    else put8(red.a + threadIdx.x * 8, s);
  }
  __syncthreads();
  gn_groups(g, w, [&](int k, int lane, bool live) {
    float v = 0.f;
    if (live) gn_run(g, w, k, lane, [&](int at, int) { v += red.a[at]; });
    v = sum_lanes(v, g.lanes) * inv_values;
    if (live && lane == 0) red.group[k].x = v;  // mean, from the origin
  });
  __syncthreads();
  if (w.on) {
    // (the mean itself is written by a thread that knows the origin: that of the group's first channel)
    if (g.fold) {
      const int k = gn_group(g, w.p * 8);
      const float mean = red.group[k].x;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = d[i] - mean;
        q[i] = fmaf(n * e, e, q[i]);
      }
      if (w.r == 0 && w.p * 8 == k * g.cpg) red.group[k].y = mean + origin[0];
      red.a[threadIdx.x] = sum8(q);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = gn_group(g, w.p * 8 + i);
        const float mean = red.group[k].x, e = d[i] - mean;
        q[i] = fmaf(n * e, e, q[i]);
        if (w.r == 0 && w.p * 8 + i == k * g.cpg) red.group[k].y = mean + origin[i];
      }
      put8(red.a + threadIdx.x * 8, q);
    }
  }
  __syncthreads();
  gn_groups(g, w, [&](int k, int lane, bool live) {
    float v = 0.f;
    if (live) gn_run(g, w, k, lane, [&](int at, int) { v += red.a[at]; });
    v = sum_lanes(v, g.lanes);
    if (live && lane == 0) put(k, make_float2(red.group[k].y, v));
  });
}

// The affine map of a thread's 8 channels.
struct GnAffine {
  Values weight, bias;
};

__device__ __forceinline__ GnAffine gn_affine(const GnWork& w, const float* __restrict__ weight,
                                              const float* __restrict__ bias) {
  GnAffine a;
  const int channel = (w.first + w.p) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a.weight.p[i] = weight != nullptr ? pair(__ldg(weight + channel + 2 * i), __ldg(weight + channel + 2 * i + 1)) : pair(1.f);
    a.bias.p[i] = bias != nullptr ? pair(__ldg(bias + channel + 2 * i), __ldg(bias + channel + 2 * i + 1)) : pair(0.f);
  }
  return a;
}

// What a thread needs of its 8 channels: z = (x + away) * scale + bias.
struct GnChannels {
  Values away, scale, bias;  // -mean, rstd * weight, bias
};

// stat(group of the slab) gives {mean, rstd}
template <class Stat>
__device__ __forceinline__ void gn_channels(GnChannels& c, const GnGeom& g, const GnWork& w, const GnAffine& a, Stat stat) {
  float2 s[8];
  if (g.fold) {
    s[0] = stat(gn_group(g, w.p * 8));
#pragma unroll
    for (int i = 1; i < 8; ++i) s[i] = s[0];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = stat(gn_group(g, w.p * 8 + i));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c.away.p[i] = pair(-s[2 * i].x, -s[2 * i + 1].x);
    c.scale.p[i] = a.weight.p[i] * pair(s[2 * i].y, s[2 * i + 1].y);
    c.bias.p[i] = a.bias.p[i];
  }
}

// The forward pass of a piece.
template <class T, int ACT>
__device__ __forceinline__ Piece<T> gn_forward(const Values& f, const GnChannels& c) {
  Values r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r.p[i] = Activation<ACT, IsExact<T>::value>::value(fma2(f.p[i] + c.away.p[i], c.scale.p[i], c.bias.p[i]));
  Piece<T> o;
  to_piece(o, r);
  return o;
}

// Sums over a thread's pixels, per channel: of g * (x - mean) and of g.
struct GnBackSums {
  Values a, b;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) a.p[i] = b.p[i] = pair(0.f);
  }
  template <class T, int ACT>
  __device__ __forceinline__ void add(const Values& x, const Values& dy, const GnChannels& c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Pair d = x.p[i] + c.away.p[i];
      const Pair grad = Activation<ACT, IsExact<T>::value>::back(dy.p[i], fma2(d, c.scale.p[i], c.bias.p[i]));
      a.p[i] = fma2(grad, d, a.p[i]);
      b.p[i] = b.p[i] + grad;
    }
  }
};

// dx = rstd * weight * g + (x - mean) * slope + level: slope = -rstd^2 * s2, level = -rstd * s1
struct GnInner {
  Values slope, level;
};

template <class Inner>  // inner(group of the slab) gives {slope, level}
__device__ __forceinline__ void gn_inner(GnInner& v, const GnGeom& g, const GnWork& w, Inner inner) {
  float2 s[8];
  if (g.fold) {
    s[0] = inner(gn_group(g, w.p * 8));
#pragma unroll
    for (int i = 1; i < 8; ++i) s[i] = s[0];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = inner(gn_group(g, w.p * 8 + i));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v.slope.p[i] = pair(s[2 * i].x, s[2 * i + 1].x);
    v.level.p[i] = pair(s[2 * i].y, s[2 * i + 1].y);
  }
}

// {slope, level} of a group from its sums of weight * rstd * g * (x - mean) and of weight * g
__device__ __forceinline__ float2 gn_inner_of(float2 sums, float rstd, float inv_m) {
  return make_float2(-rstd * rstd * (sums.x * inv_m), -rstd * (sums.y * inv_m));
}

// The backward pass of a piece.
template <class T, int ACT>
__device__ __forceinline__ Piece<T> gn_backward(const Values& x, const Values& dy, const GnChannels& c,
                                                const GnInner& v) {
  Values r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Pair d = x.p[i] + c.away.p[i];
    const Pair grad = Activation<ACT, IsExact<T>::value>::back(dy.p[i], fma2(d, c.scale.p[i], c.bias.p[i]));
    r.p[i] = fma2(grad, c.scale.p[i], fma2(d, v.slope.p[i], v.level.p[i]));
  }
  Piece<T> o;
  to_piece(o, r);
  return o;
}

// A CTA's backward sums: {sum of weight * g * xhat, sum of weight * g} of the slab's groups, to put(group of the
// slab, value).  stats: {mean, rstd} of the slab's groups.  Leaves the threads' channel sums in shared memory
// for gn_back_channels.
template <class Put>
__device__ __forceinline__ void gn_back_groups(const GnGeom& g, const GnWork& w, const GnBackSums& t,
                                               const float2* __restrict__ stats, const float* __restrict__ weight,
                                               const GnReduce& red, Put put) {
  float a[8], b[8];
  spread(t.a, a), spread(t.b, b);
  if (w.on) {
    put8(red.a + threadIdx.x * 8, a);
    put8(red.b + threadIdx.x * 8, b);
    if (g.fold) {
      if (weight != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = __ldg(weight + (w.first + w.p) * 8 + i);
          a[i] *= f, b[i] *= f;
        }
      }
      red.folded[threadIdx.x] = make_float2(sum8(a), sum8(b));
    }
  }
  __syncthreads();
  gn_groups(g, w, [&](int k, int lane, bool live) {
    float s = 0.f, q = 0.f;
    if (live) {
      if (g.fold) {
        gn_run(g, w, k, lane, [&](int at, int) {
          const float2 v = red.folded[at];
          s += v.x, q += v.y;
        });
      } else {
        gn_run(g, w, k, lane, [&](int at, int ch) {
          const float f = weight != nullptr ? __ldg(weight + w.first * 8 + k * g.cpg + ch) : 1.f;
          s = fmaf(f, red.a[at], s), q = fmaf(f, red.b[at], q);
        });
      }
    }
    s = sum_lanes(s, g.lanes), q = sum_lanes(q, g.lanes);
    if (live && lane == 0) put(k, make_float2(s * __ldg(stats + k).y, q));
  });
}

// The channels' sums over the CTA's pixels, of g * xhat and of g, to out[channel] and out[c + channel].
__device__ __forceinline__ void gn_back_channels(const GnGeom& g, const GnWork& w, const float2* __restrict__ stats,
                                                 const GnReduce& red, float* __restrict__ out) {
  const int columns = w.sp * 16, row = w.sp * 8;  // of a[] and of b[]
  const int lanes = 1 << g.column_lanes, lane = threadIdx.x & (lanes - 1), step = kGnThreads >> g.column_lanes;
  int col = threadIdx.x >> g.column_lanes;
  for (int base = 0; base < columns; base += step, col += step) {
    const bool live = col < columns, second = col >= row;
    const int ch = second ? col - row : col;
    const float* from = (second ? red.b : red.a) + ch;
    float s = 0.f;
    if (live) {
#pragma unroll 4
      for (int r = lane; r < w.rows; r += lanes) s += from[r * row];
    }
    s = sum_lanes(s, g.column_lanes);
    if (live && lane == 0) out[(second ? g.c : 0) + w.first * 8 + ch] = second ? s : s * __ldg(stats + gn_group(g, ch)).y;
  }
}

// ---------------------------------------------------------------- streaming through shared memory
//
// A thread streams its pieces through a ring of slots in shared memory that it alone reads and writes, so the
// copies need no barrier.  The ring is four batches of g.batch slots, each waited for as a whole and
// refilled once used; dynamic shared memory is [reductions][groups of the slab: own, merged][ring].

__device__ __forceinline__ void copy_async_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// the first `bytes` of 4, zeros behind them
__device__ __forceinline__ void copy_async_4(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// A thread's passes over its `count` pieces through the ring: issue(slot, piece) requests a piece, use(slot, piece)
// works on it.  The ring's first filling:
template <class Issue>
__device__ __forceinline__ void gn_request(const GnGeom& g, int count, Issue issue) {
  const int size = g.batch;
  for (int k = 0; k < 4 * size; k += size) {
    for (int i = k; i < min(k + size, count); ++i) issue(i, i);
    copy_commit();
  }
}

// Forwards, behind gn_request.
template <class Issue, class Use>
__device__ __forceinline__ void gn_forwards(const GnGeom& g, int count, Issue issue, Use use) {
  const int size = g.batch;
  int slot = 0;
  for (int k = 0; k < count; k += size) {
    copy_wait<3>();
    const int last = min(k + size, count);
#pragma unroll 2
    for (int i = k; i < last; ++i) use(slot + i - k, i);
    for (int i = k + 4 * size; i < min(k + 5 * size, count); ++i) issue(slot + i - k - 4 * size, i);
    copy_commit();
    slot = slot == 3 * size ? 0 : slot + size;
  }
  copy_wait<0>();
}

// Backwards, behind gn_forwards: the last four batches are in the ring.
template <class Issue, class Use>
__device__ __forceinline__ void gn_backwards(const GnGeom& g, int count, Issue issue, Use use) {
  const int size = g.batch;
  // The same number of batches for all threads, although some have fewer pieces: a batch is requested again four
  // batches ahead of its use, or was among the thread's last four anyway.
  const int batches = g.batches;
  int slot = ((batches - 1) & 3) * size;
  for (int j = batches - 1; j >= 0; --j) {
    if (j < batches - 4) copy_wait<3>();
    const int k = j * size, last = min(k + size, count);
#pragma unroll 2
    for (int i = k; i < last; ++i) use(slot + i - k, i);
    if (j >= 4)
      for (int i = k - 4 * size; i < min(k - 3 * size, count); ++i) issue(slot + i - k + 4 * size, i);
    copy_commit();
    slot = slot == 0 ? 3 * size : slot - size;
  }
}

// Slots of the part that this thread works on.
__device__ __forceinline__ int gn_count(const GnWork& w) {
  return w.on && w.r < w.px ? (w.px - w.r + w.rows - 1) / w.rows : 0;
}

// A piece kept in shared memory: W words, a plane of the CTA's slots apart.
template <class T>
__device__ __forceinline__ Piece<T> kept_piece(const uint4* slot, int plane) {
  Piece<T> v;
#pragma unroll
  for (int i = 0; i < Piece<T>::W; ++i) v.u[i] = slot[i * plane];
  return v;
}
template <class T>
__device__ __forceinline__ void keep_piece(uint4* slot, int plane, const T* from) {
#pragma unroll
  for (int i = 0; i < Piece<T>::W; ++i) copy_async_16(slot + i * plane, reinterpret_cast<const uint4*>(from) + i);
}

// The forward pass of a piece: y, and the 8-bit form of the input.
template <class T, int ACT, bool CODES>
__device__ __forceinline__ void gn_write(T* __restrict__ y, uint2* __restrict__ codes,
                                         unsigned char* __restrict__ exponents, long long at, const Piece<T>& v,
                                         const GnChannels& c) {
  const Values f = values_of(v);
  if (CODES) {
    const Block8 b = encode_block(v, f);
    __stcs(codes + (at >> 3), b.codes);
    exponents[at >> 3] = (unsigned char)b.exponent;
  }
  store_piece(y + at, gn_forward<T, ACT>(f, c));
}

// The norm's input in the ring: pieces of x, or codes (8 bytes a slot) and the 4-byte words that hold their
// exponents.
template <class T, bool CODES>
struct GnKept {
  uint4* slots;
  const T* x;
  __device__ __forceinline__ GnKept(char* at, int, const T* x_, const uint2*, const unsigned char*, long long)
      : slots(reinterpret_cast<uint4*>(at) + threadIdx.x), x(x_) {}
  __device__ __forceinline__ void issue(int slot, int plane, long long at) {
    keep_piece(slots + slot * kGnThreads, plane, x + at);
  }
  __device__ __forceinline__ Values values(int k, int plane, long long) const {
    return values_of(kept_piece<T>(slots + k * kGnThreads, plane));
  }
};
template <class T>
struct GnKept<T, true> {
  uint2* slots;
  u32* words;
  const uint2* codes;
  const unsigned char* exponents;
  long long blocks;
  __device__ __forceinline__ GnKept(char* at, int plane, const T*, const uint2* codes_, const unsigned char* exponents_,
                                    long long blocks_)
      : slots(reinterpret_cast<uint2*>(at) + threadIdx.x),
        words(reinterpret_cast<u32*>(at + 8 * (size_t)plane) + threadIdx.x),
        codes(codes_), exponents(exponents_), blocks(blocks_) {}
  __device__ __forceinline__ void issue(int k, int, long long at) {
    const long long block = at >> 3, word = block & ~3ll;
    copy_async_8(slots + k * kGnThreads, codes + block);
    copy_async_4(words + k * kGnThreads, exponents + word, (int)min(4ll, blocks - word));
  }
  __device__ __forceinline__ Values values(int k, int, long long at) const {
    Block8 b;
    b.codes = slots[k * kGnThreads];
    b.exponent = (words[k * kGnThreads] >> ((int)(at >> 3) & 3) * 8) & 255u;
    return decode_block(b);
  }
};

// What the backward passes read: dy and the norm's input.
template <class T, bool CODES>
struct GnBackRing {
  int plane;
  uint4* grads;
  const T* dy;
  GnKept<T, CODES> kept;
  __device__ __forceinline__ GnBackRing(uint4* dynamic, const GnGeom& g, const T* dy_, const T* x, const uint2* codes,
                                        const unsigned char* exponents)
      : plane(g.slots * kGnThreads),
        grads(reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x),
        dy(dy_),
        kept(reinterpret_cast<char*>(dynamic) + g.data_at + (size_t)g.slots * kGnThreads * 16 * Piece<T>::W,
             g.slots * kGnThreads, x, codes, exponents, g.images * g.pixels * g.pieces) {}
  __device__ __forceinline__ void issue(int slot, long long at) {
    keep_piece(grads + slot * kGnThreads, plane, dy + at);
    kept.issue(slot, plane, at);
  }
  __device__ __forceinline__ Values input(int slot, long long at) const { return kept.values(slot, plane, at); }
  __device__ __forceinline__ Values grad(int slot) const {
    return values_of(kept_piece<T>(grads + slot * kGnThreads, plane));
  }
};

// ---------------------------------------------------------------- two launches
//
// For a few large images: any number of CTAs works on an image, the sums go through memory, and the second launch
// reads the input again.  It may ask for it before the first has ended (its inputs were there before that began) and
// goes through the data backwards, so that it finds in L2 what the first launch read last.

// part_stats[(image * groups + group) * parts + part] = {mean, centred squares} over the part's pixels
template <class T>
__global__ void __launch_bounds__(kGnThreads, 768 / kGnThreads)
groupnorm_2d_stats_kernel(float2* __restrict__ part_stats, const T* __restrict__ x, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  const int plane = g.slots * kGnThreads;
  uint4* data = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x;
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const long long first = gn_offset(g, w, w.px0 + w.r), step = (long long)w.rows * g.c;
  const auto issue = [&](int slot, int k) { keep_piece(data + slot * kGnThreads, plane, x + first + k * step); };
  gn_request(g, count, issue);
  float origin[8];
  gn_origin(origin, g, w, x);
  GnSums t;
  t.clear();
  if (count > 0) t.start(values_of(load_piece(x + first)));
  gn_forwards(g, count, issue,
              [&](int slot, int) { t.add(values_of(kept_piece<T>(data + slot * kGnThreads, plane))); });
  const long long first_group = gn_first_group(g, w);
  gn_group_stats(g, w, t, origin, red, [&](int k, float2 v) { part_stats[(first_group + k) * g.parts + w.part] = v; });
}

// Mean and rstd of the slab's groups from the parts' values, into stat[]; all threads, synchronised.
__device__ __forceinline__ void gn_merge_parts(float2* stat, const GnGeom& g, const GnWork& w,
                                               const float2* __restrict__ part_stats) {
  const long long first_group = gn_first_group(g, w);
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < w.groups; k += kGnThreads / 32) {
    const float2* ps = part_stats + (first_group + k) * g.parts;
    const float m0 = __ldcg(ps).x;
    float s = 0.f, q = 0.f;
    for (int i = lane; i < g.parts; i += 32) {
      const float n = (float)gn_part_pixels(g, i);
      s = fmaf(n, __ldcg(ps + i).x - m0, s);
    }
    s = fmaf(sum_lanes(s, 5), g.inv_pixels, m0);
    for (int i = lane; i < g.parts; i += 32) {
      const float n = (float)gn_part_pixels(g, i) * (float)g.cpg;
      const float2 v = __ldcg(ps + i);
      const float d = v.x - s;
      q += fmaf(n * d, d, v.y);
    }
    q = sum_lanes(q, 5);
    if (lane == 0) stat[k] = make_float2(s, rsqrtf(fmaf(q, g.inv_m, g.eps)));
  }
  __syncthreads();
}

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 768 / kGnThreads)
groupnorm_2d_apply_kernel(T* __restrict__ y, float2* __restrict__ stats, uint2* __restrict__ codes,
                          unsigned char* __restrict__ exponents, const T* __restrict__ x,
                          const float* __restrict__ weight, const float* __restrict__ bias,
                          const float2* __restrict__ part_stats, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  float2* stat = gn_reduce(dynamic, g).group;
  const int plane = g.slots * kGnThreads;
  uint4* data = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x;
  const GnWork w = gn_work(g, gridDim.x - 1 - blockIdx.x);
  const int count = gn_count(w);
  const long long first = gn_offset(g, w, w.px0 + w.r), step = (long long)w.rows * g.c;
  const auto issue = [&](int slot, int k) { keep_piece(data + slot * kGnThreads, plane, x + first + k * step); };
  gn_request(g, count, issue);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  gn_merge_parts(stat, g, w, part_stats);
  if (stats != nullptr && w.part == 0) {
    for (int k = threadIdx.x; k < w.groups; k += kGnThreads) stats[gn_first_group(g, w) + k] = stat[k];
  }
  if (!w.on) return;
  GnChannels c;
  gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return stat[k]; });
  gn_forwards(g, count, issue, [&](int slot, int k) {
    gn_write<T, ACT, CODES>(y, codes, exponents, first + k * step, kept_piece<T>(data + slot * kGnThreads, plane), c);
  });
}

// part_channel[(image * parts + part) * 2 + {0, 1}][c] = sums of g * xhat and of g over the part's pixels;
// part_group[(image * groups + group) * parts + part] = their weighted sums over a group's channels.
template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 512 / kGnThreads)
groupnorm_2d_bwd_sums_kernel(float* __restrict__ part_channel, float2* __restrict__ part_group,
                             const T* __restrict__ dy, const T* __restrict__ x, const uint2* __restrict__ codes,
                             const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                             const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  GnBackRing<T, CODES> ring(dynamic, g, dy, x, codes, exponents);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const long long first = gn_offset(g, w, w.px0 + w.r), step = (long long)w.rows * g.c;
  const auto issue = [&](int slot, int k) { ring.issue(slot, first + k * step); };
  gn_request(g, count, issue);
  const long long first_group = gn_first_group(g, w);
  stats += first_group;
  GnChannels c;
  if (w.on) gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return __ldg(stats + k); });
  GnBackSums t;
  t.clear();
  gn_forwards(g, count, issue,
              [&](int slot, int k) { t.add<T, ACT>(ring.input(slot, first + k * step), ring.grad(slot), c); });
  gn_back_groups(g, w, t, stats, weight, red, [&](int k, float2 v) {
    if (part_group != nullptr) part_group[(first_group + k) * g.parts + w.part] = v;
  });
  if (part_channel != nullptr)
    gn_back_channels(g, w, stats, red, part_channel + (w.image * g.parts + w.part) * 2 * g.c);
}

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 512 / kGnThreads)
groupnorm_2d_bwd_apply_kernel(T* __restrict__ dx, const float2* __restrict__ part_group, const T* __restrict__ dy,
                              const T* __restrict__ x, const uint2* __restrict__ codes,
                              const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                              const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  float2* inner = gn_reduce(dynamic, g).group;
  GnBackRing<T, CODES> ring(dynamic, g, dy, x, codes, exponents);
  const GnWork w = gn_work(g, gridDim.x - 1 - blockIdx.x);
  const int count = gn_count(w);
  const long long first = gn_offset(g, w, w.px0 + w.r), step = (long long)w.rows * g.c;
  const auto issue = [&](int slot, int k) { ring.issue(slot, first + k * step); };
  gn_request(g, count, issue);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const long long first_group = gn_first_group(g, w);
  stats += first_group;
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < w.groups; k += kGnThreads / 32) {
    float s = 0.f, q = 0.f;
    for (int i = lane; i < g.parts; i += 32) {
      const float2 v = __ldcg(part_group + (first_group + k) * g.parts + i);
      s += v.x, q += v.y;
    }
    s = sum_lanes(s, 5), q = sum_lanes(q, 5);
    if (lane == 0) inner[k] = gn_inner_of(make_float2(s, q), __ldg(stats + k).y, g.inv_m);
  }
  __syncthreads();
  if (!w.on) return;
  GnChannels c;
  gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return __ldg(stats + k); });
  GnInner s;
  gn_inner(s, g, w, [&](int k) { return inner[k]; });
  gn_forwards(g, count, issue, [&](int slot, int k) {
    const long long at = first + k * step;
    store_piece(dx + at, gn_backward<T, ACT>(ring.input(slot, at), ring.grad(slot), c, s));
  });
}

// ---------------------------------------------------------------- one launch
//
// The parts of a slab are the CTAs of a cluster (1 to 16) and the sums cross CTAs through distributed shared
// memory, so one launch does both passes and the second one finds its data close by: it goes through the pieces
// backwards, those that are still in the ring first (all of them, where a part fits), the others again from L2,
// which holds what the resident CTAs work on many times over.

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// *p of the CTA `rank` of the cluster
__device__ __forceinline__ float2 cluster_load(const float2* p, int rank) {
  u32 at;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

// Calls body(group, part, live) with the parts of a group in neighbouring lanes (parts is a power of two up
// to 16): all lanes of a warp together, `live` where there is such a group.
template <class Body>
__device__ __forceinline__ void gn_over_parts(const GnGeom& g, const GnWork& w, Body body) {
  const int part = threadIdx.x & (g.parts - 1), step = kGnThreads >> g.log_parts;
  int k = threadIdx.x >> g.log_parts;
  for (int base = 0; base < w.groups; base += step, k += step) body(k, part, k < w.groups);
}

// Every CTA of the cluster has written its `own` values (or this CTA, if it is alone).
__device__ __forceinline__ void gn_cluster_sync(const GnGeom& g) {
  if (g.parts > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
}

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 768 / kGnThreads)
groupnorm_2d_fwd_kernel(T* __restrict__ y, float2* __restrict__ stats, uint2* __restrict__ codes,
                        unsigned char* __restrict__ exponents, const T* __restrict__ x,
                        const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  float2* own = red.group + g.slab_groups;
  float2* stat = own + g.slab_groups;
  const int plane = g.slots * kGnThreads;
  uint4* data = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x;

  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const long long first = gn_offset(g, w, w.px0 + w.r), step = (long long)w.rows * g.c;
  const auto issue = [&](int slot, int k) { keep_piece(data + slot * kGnThreads, plane, x + first + k * step); };
  gn_request(g, count, issue);
  float origin[8];
  gn_origin(origin, g, w, x);
  GnSums t;
  t.clear();
  if (count > 0) t.start(values_of(load_piece(x + first)));
  gn_forwards(g, count, issue,
              [&](int slot, int) { t.add(values_of(kept_piece<T>(data + slot * kGnThreads, plane))); });
  gn_group_stats(g, w, t, origin, red, [&](int k, float2 v) { own[k] = v; });
  const GnAffine affine = w.on ? gn_affine(w, weight, bias) : GnAffine();  // (on its way across the barrier)
  gn_cluster_sync(g);
  gn_over_parts(g, w, [&](int k, int part, bool live) {
    const float2 v = live ? (g.parts > 1 ? cluster_load(own + k, part) : own[k]) : make_float2(0.f, 0.f);
    const float n = (float)gn_part_pixels(g, part);
    float mean = v.x, m2 = v.y;
    if (g.parts > 1) {
      const float m0 = __shfl_sync(0xffffffffu, v.x, 0, g.parts);
      mean = fmaf(sum_lanes(live ? n * (v.x - m0) : 0.f, g.log_parts), g.inv_pixels, m0);
      const float d = v.x - mean;
      m2 = sum_lanes(fmaf(n * (float)g.cpg * d, d, v.y), g.log_parts);
    }
    if (live && part == 0) {
      const float2 st = make_float2(mean, rsqrtf(fmaf(m2, g.inv_m, g.eps)));
      stat[k] = st;
      if (stats != nullptr && w.part == 0) stats[gn_first_group(g, w) + k] = st;
    }
  });
  if (g.parts > 1) cluster_arrive();  // (this CTA has read the others' values; waited for at the end)
  __syncthreads();
  if (w.on) {
    GnChannels c;
    gn_channels(c, g, w, affine, [&](int k) { return stat[k]; });
    gn_backwards(g, count, issue, [&](int slot, int k) {
      gn_write<T, ACT, CODES>(y, codes, exponents, first + k * step, kept_piece<T>(data + slot * kGnThreads, plane), c);
    });
  }
  if (g.parts > 1) cluster_wait();  // no CTA leaves while another reads its values
}

// part_channel as of groupnorm_2d_bwd_sums_kernel; dx may be NULL.
template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 512 / kGnThreads)
groupnorm_2d_bwd_kernel(T* __restrict__ dx, float* __restrict__ part_channel, const T* __restrict__ dy,
                        const T* __restrict__ x, const uint2* __restrict__ codes,
                        const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                        const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  float2* own = red.group + g.slab_groups;
  float2* inner = own + g.slab_groups;
  GnBackRing<T, CODES> ring(dynamic, g, dy, x, codes, exponents);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const long long first = gn_offset(g, w, w.px0 + w.r), step = (long long)w.rows * g.c;
  const auto issue = [&](int slot, int k) { ring.issue(slot, first + k * step); };
  gn_request(g, count, issue);
  stats += gn_first_group(g, w);
  GnChannels c;
  if (w.on) gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return __ldg(stats + k); });
  GnBackSums t;
  t.clear();
  gn_forwards(g, count, issue,
              [&](int slot, int k) { t.add<T, ACT>(ring.input(slot, first + k * step), ring.grad(slot), c); });
  gn_back_groups(g, w, t, stats, weight, red, [&](int k, float2 v) { own[k] = v; });
  if (g.parts > 1) cluster_arrive();
  if (part_channel != nullptr) gn_back_channels(g, w, stats, red, part_channel + (w.image * g.parts + w.part) * 2 * g.c);
  if (g.parts > 1) cluster_wait();
  else __syncthreads();
  gn_over_parts(g, w, [&](int k, int part, bool live) {
    float2 v = live ? (g.parts > 1 ? cluster_load(own + k, part) : own[k]) : make_float2(0.f, 0.f);
    v.x = sum_lanes(v.x, g.log_parts), v.y = sum_lanes(v.y, g.log_parts);
    if (live && part == 0) inner[k] = gn_inner_of(v, __ldg(stats + k).y, g.inv_m);
  });
  if (g.parts > 1) cluster_arrive();
  __syncthreads();
  if (w.on && dx != nullptr) {
    GnInner s;
    gn_inner(s, g, w, [&](int k) { return inner[k]; });
    gn_backwards(g, count, issue, [&](int slot, int k) {
      const long long at = first + k * step;
      store_piece(dx + at, gn_backward<T, ACT>(ring.input(slot, at), ring.grad(slot), c, s));
    });
  }
  if (g.parts > 1) cluster_wait();
}

}  // namespace GN_NAMESPACE
}  // namespace spio_b200

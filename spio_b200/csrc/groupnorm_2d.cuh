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
// error, whatever the data's offset.  Threads, lanes and CTAs are then merged by their counts, means and
// centred squares, in a fixed order: results do not vary from run to run, and the mean of equal values is
// that value.
#pragma once

#include <cuda_runtime.h>

#include "checkpoint8.cuh"
#include "cluster.cuh"
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
// hardware's exponential and reciprocal (relative errors of some 2^-22) are far below that.  The normal distribution
// function is then Abramowitz and Stegun's 7.1.26, off by 7e-8 at most, and GELU by 2.2e-7: for negative z within half a
// step of fp16 down to -3.6 and of bf16 down to -5.3.  Further out, where GELU is 6e-4 and less, its relative error
// grows: 0.05 % at -4, 0.4 % at -6 (half a step of bf16 is 0.2 to 0.4 %), 1 % at -8, 3 % at -12.
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
    if (ACT == kActRelu) {  // chosen, not multiplied: an infinite gradient where ReLU is off counts for nothing
      const float2 d = unpair(grad);
      return pair(f.x <= 0.f ? 0.f : d.x, f.y <= 0.f ? 0.f : d.y);
    }
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
  int each, rest;  // pixels of a row, one more in the first `rest` rows
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
  w.each = w.px / w.rows;
  w.rest = w.px - w.each * w.rows;
  w.on = w.r < w.rows;
  return w;
}

// Index of the slab's first group.  (A slab begins with whole groups; their index may pass 2048.)
__device__ __forceinline__ long long gn_first_group(const GnGeom& g, const GnWork& w) {
  return w.image * g.groups + (w.first == 0 ? 0 : w.first / g.sp * g.slab_groups);
}

// Pieces before the part's first pixel of the slab.  Within the part, 32-bit indices of pieces: one instruction for
// each address.
__device__ __forceinline__ long long gn_part_start(const GnGeom& g, const GnWork& w) {
  return (w.image * g.pixels + w.px0) * g.pieces + w.first;
}
__device__ __forceinline__ u32 gn_first_piece(const GnGeom& g, const GnWork& w) { return (u32)w.r * g.pieces + w.p; }
__device__ __forceinline__ u32 gn_step(const GnGeom& g, const GnWork& w) { return (u32)w.rows * g.pieces; }

// ---------------------------------------------------------------- sums over a CTA

// Shared memory of the reductions: two arrays of a value of each channel of each thread, or of each thread
// (where a piece lies within one group, g.fold) two values of each thread; two values for each of the slab's groups.
struct GnReduce {
  float* a;
  float* b;
  float2* folded;  // (backward)
  float2* group;
};
__device__ __forceinline__ GnReduce gn_reduce(void* at, const GnGeom& g) {
  GnReduce s;
  s.a = reinterpret_cast<float*>(reinterpret_cast<char*>(at) + g.planes_at);
  s.b = s.a + g.plane;
  s.folded = reinterpret_cast<float2*>(s.b + g.plane);
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

// Calls at(index, channel of the group, row) for this lane's share of the values of group k: every row's run of them.
template <class At>
__device__ __forceinline__ void gn_run(const GnGeom& g, const GnWork& w, int k, int lane, At at) {
  const int row = g.fold ? w.sp : w.sp * 8;
  int r = divide(lane, g.inv_run), j = lane - r * g.run;
#pragma unroll 4
  while (r < w.rows) {
    at(r * row + k * g.run + j, j, r);
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

// Count, mean and centred squares of a set of values, and its union with another set.
struct GnSet {
  float n, mean, m2;
  __device__ __forceinline__ void merge(float n_, float mean_, float m2_) {
    const float d = mean_ - mean, share = __fdividef(n_, fmaxf(n + n_, 1.f));
    mean = fmaf(d, share, mean);
    m2 = fmaf(d * share * n, d, m2 + m2_);
    n += n_;
  }
  // with the sets of 2^log neighbouring lanes; lane 0 of them has the union
  __device__ __forceinline__ void merge_lanes(int log) {
#pragma unroll
    for (int i = 0; i < 5; ++i)
      if (i < log)
        merge(__shfl_xor_sync(0xffffffffu, n, 1 << i), __shfl_xor_sync(0xffffffffu, mean, 1 << i),
              __shfl_xor_sync(0xffffffffu, m2, 1 << i));
  }
};

// {mean, centred squares} of the groups of the slab over the CTA's pixels, to put(group of the slab, value), by
// all threads.
template <class Put>
__device__ __forceinline__ void gn_group_stats(const GnGeom& g, const GnWork& w, const GnSums& t, const GnReduce& red,
                                               Put put) {
  if (w.on) {
    float mean[8], m2[8], s[8], away[8];
    const float n = (float)t.n, inv_n = t.n > 0 ? __fdividef(1.f, n) : 0.f;
    spread(t.s, s), spread(t.q, m2), spread(t.away, away);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = s[i] * inv_n;
      m2[i] = fmaf(-s[i], d, m2[i]);
      mean[i] = d - away[i];
    }
    if (g.fold) {
      float d = 0.f, q = 0.f;
#pragma unroll
      for (int i = 1; i < 8; ++i) d += mean[i] - mean[0];
      const float all = fmaf(d, .125f, mean[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) q = fmaf(mean[i] - all, mean[i] - all, q);
      red.a[threadIdx.x] = all;
      red.b[threadIdx.x] = fmaf(q, n, sum8(m2));
    } else {
      put8(red.a + threadIdx.x * 8, mean);
      put8(red.b + threadIdx.x * 8, m2);
    }
  }
  __syncthreads();
  const float scale = g.fold ? 8.f : 1.f;  // channels of a value
  gn_groups(g, w, [&](int k, int lane, bool live) {
    // differences to the lane's first value, which is a mean of members: little cancels
    float n = 0.f, m0 = 0.f, s = 0.f, q = 0.f;
    if (live) {
      gn_run(g, w, k, lane, [&](int at, int, int r) {
        const float mean = red.a[at], count = (float)(w.each + (r < w.rest)) * scale;
        if (n == 0.f) m0 = mean;
        const float d = mean - m0;
        n += count;
        s = fmaf(count, d, s);
        q += fmaf(count * d, d, red.b[at]);
      });
    }
    const float d = n > 0.f ? __fdividef(s, n) : 0.f;
    GnSet set = {n, m0 + d, fmaf(-s, d, q)};
    set.merge_lanes(g.lanes);
    if (live && lane == 0) put(k, make_float2(set.mean, set.m2));
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
    a.weight.p[i] = weight != nullptr ? pair(__ldca(weight + channel + 2 * i), __ldca(weight + channel + 2 * i + 1)) : pair(1.f);
    a.bias.p[i] = bias != nullptr ? pair(__ldca(bias + channel + 2 * i), __ldca(bias + channel + 2 * i + 1)) : pair(0.f);
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
          const float f = __ldca(weight + (w.first + w.p) * 8 + i);
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
        gn_run(g, w, k, lane, [&](int at, int, int) {
          const float2 v = red.folded[at];
          s += v.x, q += v.y;
        });
      } else {
        gn_run(g, w, k, lane, [&](int at, int ch, int) {
          const float f = weight != nullptr ? __ldca(weight + w.first * 8 + k * g.cpg + ch) : 1.f;
          s = fmaf(f, red.a[at], s), q = fmaf(f, red.b[at], q);
        });
      }
    }
    s = sum_lanes(s, g.lanes), q = sum_lanes(q, g.lanes);
    if (live && lane == 0) put(k, make_float2(s * __ldca(stats + k).y, q));
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
    if (live && lane == 0) out[(second ? g.c : 0) + w.first * 8 + ch] = second ? s : s * __ldca(stats + gn_group(g, ch)).y;
  }
}

// ---------------------------------------------------------------- streaming through shared memory
//
// A thread streams its pieces through a ring of slots in shared memory that it alone reads and writes, so the
// copies need no barrier.  The ring is four batches, each waited for as a whole and refilled once used; 256
// bytes a thread in all, so that the CTAs that registers allow on an SM fit beside each other and have 100 KB or more
// on their way.  Dynamic shared memory is [reductions][groups of the slab: own, merged][ring]; the kernels that do not
// come back to the ring reduce in it.
//
// The kernels are bound by instructions as much as by memory (a smooth activation takes 6 to 11 a value), so the
// loops keep their share small: batches have a fixed size and whole ones no bounds checks.

template <class T>
struct GnBatch {  // slots of a quarter of the ring
  static constexpr int forward = 8 / (int)sizeof(T);
  static constexpr int backward = 4 / (int)sizeof(T);
};

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

// A thread's passes over its `count` pieces through the ring, `step` pieces apart: issue(slot, offset) requests a piece,
// use(slot, offset) works on it.  The ring's first filling:
template <int B, class Issue>
__device__ __forceinline__ void gn_request(int count, u32 first, u32 step, Issue issue) {
#pragma unroll
  for (int k = 0; k < 4 * B; ++k) {
    if (k < count) issue(k, first + k * step);
    if (k % B == B - 1) copy_commit();
  }
}

// issue() for the pieces i, i + 1, ... of a batch
template <int B, class Issue>
__device__ __forceinline__ void gn_refill(int slot, int i, int count, u32 offset, u32 step, Issue issue) {
  if (i + B <= count) {
#pragma unroll
    for (int k = 0; k < B; ++k) issue(slot + k, offset + k * step);
  } else {
#pragma unroll
    for (int k = 0; k < B - 1; ++k)
      if (i + k < count) issue(slot + k, offset + k * step);
  }
}

template <int B, class Use>
__device__ __forceinline__ void gn_use(int slot, int i, int count, u32 offset, u32 step, Use use) {
  if (i + B <= count) {
#pragma unroll
    for (int k = 0; k < B; ++k) use(slot + k, offset + k * step);
  } else {
#pragma unroll
    for (int k = 0; k < B - 1; ++k)
      if (i + k < count) use(slot + k, offset + k * step);
  }
}

// Forwards, behind gn_request.
template <int B, class Issue, class Use>
__device__ __forceinline__ void gn_forwards(int count, u32 first, u32 step, Issue issue, Use use) {
  u32 offset = first;
  int slot = 0;
  for (int i = 0; i < count; i += B) {
    copy_wait<3>();
    gn_use<B>(slot, i, count, offset, step, use);
    gn_refill<B>(slot, i + 4 * B, count, offset + 4 * B * step, step, issue);
    copy_commit();
    offset += B * step;
    slot = (slot + B) & (4 * B - 1);
  }
  copy_wait<0>();
}

// Backwards, behind gn_forwards: the last four batches are in the ring.  The same number of batches for all
// threads, although some have fewer pieces: a batch is requested again four batches ahead of its use, or was
// among the thread's last four anyway.
template <int B, class Issue, class Use>
__device__ __forceinline__ void gn_backwards(int batches, int count, u32 first, u32 step, Issue issue, Use use) {
  u32 offset = first + (u32)((batches - 1) * B) * step;
  int slot = ((batches - 1) & 3) * B;
  for (int i = (batches - 1) * B; i >= 0; i -= B) {
    if (i < (batches - 4) * B) copy_wait<3>();
    gn_use<B>(slot, i, count, offset, step, use);
    if (i >= 4 * B) gn_refill<B>(slot, i - 4 * B, count, offset - 4 * B * step, step, issue);
    copy_commit();
    offset -= B * step;
    slot = (slot - B) & (4 * B - 1);
  }
}

// Slots of the part that this thread works on.
__device__ __forceinline__ int gn_count(const GnWork& w) {
  return w.on ? w.each + (w.r < w.rest) : 0;
}

template <class T>
__device__ __forceinline__ T* piece_at(T* p, u32 at) {
  return p + (size_t)at * 8;
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
                                         unsigned char* __restrict__ exponents, u32 at, const Piece<T>& v,
                                         const GnChannels& c) {
  const Values f = values_of(v);
  if (CODES) {
    const Block8 b = encode_block(v, f);
    __stcs(codes + at, b.codes);
    exponents[at] = (unsigned char)b.exponent;
  }
  store_piece(piece_at(y, at), gn_forward<T, ACT>(f, c));
}

// The norm's input in the ring: pieces of x, or codes (8 bytes a slot) and the 4-byte words that hold their
// exponents.  `start`: pieces before the part.
template <class T, bool CODES>
struct GnKept {
  static constexpr int plane = 4 * GnBatch<T>::backward * kGnThreads;
  uint4* slots;
  const T* x;
  __device__ __forceinline__ GnKept(char* at, const GnGeom&, long long start, const T* x_, const uint2*, const unsigned char*)
      : slots(reinterpret_cast<uint4*>(at) + threadIdx.x), x(x_ + start * 8) {}
  __device__ __forceinline__ void issue(int slot, u32 at) { keep_piece(slots + slot * kGnThreads, plane, piece_at(x, at)); }
  __device__ __forceinline__ Values values(int slot, u32) const {
    return values_of(kept_piece<T>(slots + slot * kGnThreads, plane));
  }
};
template <class T>
struct GnKept<T, true> {
  static constexpr int plane = 4 * GnBatch<T>::backward * kGnThreads;
  uint2* slots;
  u32* words;
  const uint2* codes;
  const unsigned char* exponents;  // at a word that begins `shift` bytes before the part's
  u32 shift, bytes;                // bytes: of the exponents from there on (or 2^32 - 1)
  __device__ __forceinline__ GnKept(char* at, const GnGeom& g, long long start, const T*, const uint2* codes_,
                                    const unsigned char* exponents_)
      : slots(reinterpret_cast<uint2*>(at) + threadIdx.x),
        words(reinterpret_cast<u32*>(at + 8 * plane) + threadIdx.x),
        codes(codes_ + start),
        exponents(exponents_ + (start & ~3ll)),
        shift((u32)start & 3u),
        bytes((u32)min(g.images * g.pixels * g.pieces - (start & ~3ll), 0xffffffffll)) {}
  __device__ __forceinline__ void issue(int slot, u32 at) {
    const u32 word = (at + shift) & ~3u;
    copy_async_8(slots + slot * kGnThreads, codes + at);
    copy_async_4(words + slot * kGnThreads, exponents + word, (int)min(4u, bytes - word));
  }
  __device__ __forceinline__ Values values(int slot, u32 at) const {
    Block8 b;
    b.codes = slots[slot * kGnThreads];
    b.exponent = (words[slot * kGnThreads] >> ((at + shift) & 3u) * 8) & 255u;
    return decode_block(b);
  }
};

// What the backward passes read: dy and the norm's input.
template <class T, bool CODES>
struct GnBackRing {
  static constexpr int plane = 4 * GnBatch<T>::backward * kGnThreads;
  uint4* grads;
  const T* dy;
  GnKept<T, CODES> kept;
  __device__ __forceinline__ GnBackRing(uint4* dynamic, const GnGeom& g, long long start, const T* dy_, const T* x,
                                        const uint2* codes, const unsigned char* exponents)
      : grads(reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x),
        dy(dy_ + start * 8),
        kept(reinterpret_cast<char*>(dynamic) + g.data_at + plane * 16 * Piece<T>::W, g, start, x, codes, exponents) {}
  __device__ __forceinline__ void issue(int slot, u32 at) {
    keep_piece(grads + slot * kGnThreads, plane, piece_at(dy, at));
    kept.issue(slot, at);
  }
  __device__ __forceinline__ Values input(int slot, u32 at) const { return kept.values(slot, at); }
  __device__ __forceinline__ Values grad(int slot) const {
    return values_of(kept_piece<T>(grads + slot * kGnThreads, plane));
  }
};

// ---------------------------------------------------------------- sums over a cluster

// Calls body(group, rank, live) with the CTAs of the cluster in neighbouring lanes for each group: all lanes of a warp
// together, `live` where there is such a group.
template <class Body>
__device__ __forceinline__ void gn_over_cluster(const GnGeom& g, const GnWork& w, Body body) {
  const int rank = threadIdx.x & (g.cluster - 1), step = kGnThreads >> g.log_cluster;
  int k = threadIdx.x >> g.log_cluster;
  for (int base = 0; base < w.groups; base += step, k += step) body(k, rank, k < w.groups);
}

// Every CTA of the cluster has written its `own` values (or this CTA, if it is alone).
__device__ __forceinline__ void gn_cluster_sync(const GnGeom& g) {
  if (g.cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
}

// Arrives for the last time, behind the sums over the cluster: a CTA may leave once all have arrived, and with it the
// memory that the others read.  So the warps that gn_over_cluster gave something to read release their arrival; the
// others read nothing and need no order (a release costs a warp some hundred cycles).
__device__ __forceinline__ void gn_cluster_done(const GnGeom& g, const GnWork& w) {
  if (g.cluster == 1) return;
  if ((int)(threadIdx.x & ~31u) >> g.log_cluster < w.groups) cluster_arrive();
  else cluster_arrive_relaxed();
}

__device__ __forceinline__ float2 gn_of_rank(const GnGeom& g, const float2* own, int rank) {
  return g.cluster > 1 ? cluster_load(own, rank) : *own;
}

// The groups' {mean, centred squares} over the cluster's pixels from its CTAs' own, to put(group, value) by one thread
// each, behind gn_cluster_sync.
template <class Put>
__device__ __forceinline__ void gn_cluster_stats(const GnGeom& g, const GnWork& w, const float2* own, Put put) {
  gn_over_cluster(g, w, [&](int k, int rank, bool live) {
    const float2 v = live ? gn_of_rank(g, own + k, rank) : make_float2(0.f, 0.f);
    GnSet set = {(float)gn_part_pixels(g, (w.part & -g.cluster) + rank) * (float)g.cpg, v.x, v.y};
    set.merge_lanes(g.log_cluster);
    if (live && rank == 0) put(k, make_float2(set.mean, set.m2));
  });
}

// The groups' sums over the cluster.
template <class Put>
__device__ __forceinline__ void gn_cluster_sums(const GnGeom& g, const GnWork& w, const float2* own, Put put) {
  gn_over_cluster(g, w, [&](int k, int rank, bool live) {
    float2 v = live ? gn_of_rank(g, own + k, rank) : make_float2(0.f, 0.f);
    v.x = sum_lanes(v.x, g.log_cluster), v.y = sum_lanes(v.y, g.log_cluster);
    if (live && rank == 0) put(k, v);
  });
}

// ---------------------------------------------------------------- two launches
//
// For a few large images: any number of CTAs works on an image, the sums go through memory (one value for each
// cluster), and the second launch reads the input again.  It may ask for it before the first has ended (its inputs
// were there before that began) and goes through the data backwards, so that it finds in L2 what the first launch
// read last.
//
// Measured at 1 x 128 x 512 x 512 bf16 with SiLU and 32 groups: 41.2 us for both launches forward (3260 GB/s counting
// x and y once, where the device copies 6520; under the profiler 19 us for the sums and 27 for the rest, which finds
// nothing in L2 there), one launch of clusters of 16 72 us.  The first launch waits for memory; the second issues in 46 %
// of its cycles and keeps the special functions busy for 65 % of them.

// part_stats[(image * groups + group) * clusters + cluster] = {mean, centred squares} over the cluster's pixels
template <class T>
__global__ void __launch_bounds__(kGnThreads, 768 / kGnThreads)
groupnorm_2d_stats_kernel(float2* __restrict__ part_stats, const T* __restrict__ x, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  constexpr int B = GnBatch<T>::forward, plane = 4 * B * kGnThreads;
  uint4* data = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x;
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const u32 first = gn_first_piece(g, w), step = gn_step(g, w);
  const long long start = gn_part_start(g, w);
  x += start * 8;
  const auto issue = [&](int slot, u32 at) { keep_piece(data + slot * kGnThreads, plane, piece_at(x, at)); };
  gn_request<B>(count, first, step, issue);
  GnSums t;
  t.clear();
  if (count > 0) t.start(values_of(load_piece(piece_at(x, first))));
  gn_forwards<B>(count, first, step, issue, [&](int slot, u32) {
    t.add(values_of(kept_piece<T>(data + slot * kGnThreads, plane)));
  });
  float2* own = red.group + g.slab_groups;
  __syncthreads();  // the ring is free for the reductions
  gn_group_stats(g, w, t, red, [&](int k, float2 v) { own[k] = v; });
  gn_cluster_sync(g);
  if ((w.part & (g.cluster - 1)) == 0) {
    const long long first_group = gn_first_group(g, w);
    const int clusters = g.parts >> g.log_cluster, cluster = w.part >> g.log_cluster;
    gn_cluster_stats(g, w, own, [&](int k, float2 v) { part_stats[(first_group + k) * clusters + cluster] = v; });
  }
  if (g.cluster > 1) gn_cluster_sync(g);  // no CTA leaves while another reads its values
}

// Pixels of an image before part i.
__device__ __forceinline__ int gn_part_begin(const GnGeom& g, int i) { return i * g.part_px + min(i, g.part_rest); }

// body(which, value, cluster) for this lane's share of the clusters' values of G groups, kGnWarps apart from group k on
// (zeros behind the last cluster and for groups that there are not).  G * 8 loads at a time: every CTA of the second launch does this before anything else,
// and one load after the other took it 17 us for the 222 clusters of 1 x 128 x 512 x 512.
constexpr int kGnWarps = kGnThreads / 32;
template <int G, class Body>
__device__ __forceinline__ void gn_each_cluster(const float2* __restrict__ values, int clusters, int k, int groups,
                                                Body body) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < clusters; base += 256) {
    float2 v[G][8];
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const float2* from = values + (long long)(k + h * kGnWarps) * clusters;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = base + j * 32 + lane;
        v[h][j] = k + h * kGnWarps < groups && i < clusters ? __ldcg(from + i) : make_float2(0.f, 0.f);
      }
    }
#pragma unroll
    for (int h = 0; h < G; ++h) {
#pragma unroll
      for (int j = 0; j < 8; ++j) body(h, v[h][j], base + j * 32 + lane);
    }
  }
}

// Mean and rstd of the slab's groups from the clusters' values, into stat[]; all threads, synchronised.
__device__ __forceinline__ void gn_merge_parts(float2* stat, const GnGeom& g, const GnWork& w,
                                               const float2* __restrict__ part_stats) {
  constexpr int G = 2;
  const int clusters = g.parts >> g.log_cluster;
  const float2* first = part_stats + gn_first_group(g, w) * clusters;
  for (int k = threadIdx.x >> 5; k < w.groups; k += G * kGnWarps) {
    float m0[G], s[G] = {}, q[G] = {};
    gn_each_cluster<G>(first, clusters, k, w.groups, [&](int h, float2 v, int i) {
      if (i == (int)(threadIdx.x & 31)) m0[h] = __shfl_sync(0xffffffffu, v.x, 0);  // (differences to the first mean: little cancels)
      const float n = i < clusters
                          ? (float)(gn_part_begin(g, (i + 1) << g.log_cluster) - gn_part_begin(g, i << g.log_cluster))
                          : 0.f;
      const float d = v.x - m0[h];
      s[h] = fmaf(n, d, s[h]);
      q[h] += fmaf(n * (float)g.cpg * d, d, v.y);
    });
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const float sum = sum_lanes(s[h], 5), square = sum_lanes(q[h], 5);
      const float d = sum * g.inv_pixels, m2 = not_below_zero(fmaf(-sum * (float)g.cpg, d, square));
      if ((threadIdx.x & 31) == 0 && k + h * kGnWarps < w.groups)
        stat[k + h * kGnWarps] = make_float2(m0[h] + d, rsqrtf(fmaf(m2, g.inv_m, g.eps)));
    }
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
  constexpr int B = GnBatch<T>::forward, plane = 4 * B * kGnThreads;
  uint4* data = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x;
  const GnWork w = gn_work(g, gridDim.x - 1 - blockIdx.x);
  const int count = gn_count(w);
  const u32 first = gn_first_piece(g, w), step = gn_step(g, w);
  const long long start = gn_part_start(g, w);
  x += start * 8;
  y += start * 8;
  if (CODES) codes += start, exponents += start;
  const auto issue = [&](int slot, u32 at) { keep_piece(data + slot * kGnThreads, plane, piece_at(x, at)); };
  gn_request<B>(count, first, step, issue);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  gn_merge_parts(stat, g, w, part_stats);
  if (stats != nullptr && w.part == 0) {
    for (int k = threadIdx.x; k < w.groups; k += kGnThreads) stats[gn_first_group(g, w) + k] = stat[k];
  }
  if (!w.on) return;
  GnChannels c;
  gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return stat[k]; });
  gn_forwards<B>(count, first, step, issue, [&](int slot, u32 at) {
    gn_write<T, ACT, CODES>(y, codes, exponents, at, kept_piece<T>(data + slot * kGnThreads, plane), c);
  });
}

// part_channel[(image * parts + part) * 2 + {0, 1}][c] = sums of g * xhat and of g over the part's pixels;
// part_group[(image * groups + group) * clusters + cluster] = their weighted sums over a group's channels and the
// cluster's pixels.
template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 512 / kGnThreads)
groupnorm_2d_bwd_sums_kernel(float* __restrict__ part_channel, float2* __restrict__ part_group,
                             const T* __restrict__ dy, const T* __restrict__ x, const uint2* __restrict__ codes,
                             const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                             const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const u32 first = gn_first_piece(g, w), step = gn_step(g, w);
  const long long start = gn_part_start(g, w);
  GnBackRing<T, CODES> ring(dynamic, g, start, dy, x, codes, exponents);
  const auto issue = [&](int slot, u32 at) { ring.issue(slot, at); };
  constexpr int B = GnBatch<T>::backward;
  gn_request<B>(count, first, step, issue);
  const long long first_group = gn_first_group(g, w);
  stats += first_group;
  GnChannels c;
  if (w.on) gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return __ldca(stats + k); });
  GnBackSums t;
  t.clear();
  gn_forwards<B>(count, first, step, issue,
                 [&](int slot, u32 at) { t.add<T, ACT>(ring.input(slot, at), ring.grad(slot), c); });
  float2* own = red.group + g.slab_groups;
  __syncthreads();  // the ring is free for the reductions
  gn_back_groups(g, w, t, stats, weight, red, [&](int k, float2 v) { own[k] = v; });
  if (g.cluster > 1) cluster_arrive();
  if (part_channel != nullptr)
    gn_back_channels(g, w, stats, red, part_channel + (w.image * g.parts + w.part) * 2 * g.c);
  if (g.cluster > 1) cluster_wait();
  else __syncthreads();
  if (part_group != nullptr && (w.part & (g.cluster - 1)) == 0) {
    const int clusters = g.parts >> g.log_cluster, cluster = w.part >> g.log_cluster;
    gn_cluster_sums(g, w, own, [&](int k, float2 v) { part_group[(first_group + k) * clusters + cluster] = v; });
  }
  if (g.cluster > 1) gn_cluster_sync(g);
}

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 512 / kGnThreads)
groupnorm_2d_bwd_apply_kernel(T* __restrict__ dx, const float2* __restrict__ part_group, const T* __restrict__ dy,
                              const T* __restrict__ x, const uint2* __restrict__ codes,
                              const unsigned char* __restrict__ exponents, const float2* __restrict__ stats,
                              const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  float2* inner = gn_reduce(dynamic, g).group;
  const GnWork w = gn_work(g, gridDim.x - 1 - blockIdx.x);
  const int count = gn_count(w);
  const u32 first = gn_first_piece(g, w), step = gn_step(g, w);
  const long long start = gn_part_start(g, w);
  GnBackRing<T, CODES> ring(dynamic, g, start, dy, x, codes, exponents);
  dx += start * 8;
  const auto issue = [&](int slot, u32 at) { ring.issue(slot, at); };
  constexpr int B = GnBatch<T>::backward;
  gn_request<B>(count, first, step, issue);
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const long long first_group = gn_first_group(g, w);
  stats += first_group;
  constexpr int G = 4;
  const int clusters = g.parts >> g.log_cluster;
  for (int k = threadIdx.x >> 5; k < w.groups; k += G * kGnWarps) {
    float s[G] = {}, q[G] = {};
    gn_each_cluster<G>(part_group + first_group * clusters, clusters, k, w.groups,
                       [&](int h, float2 v, int) { s[h] += v.x, q[h] += v.y; });
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const float a = sum_lanes(s[h], 5), b = sum_lanes(q[h], 5);
      if ((threadIdx.x & 31) == 0 && k + h * kGnWarps < w.groups)
        inner[k + h * kGnWarps] = gn_inner_of(make_float2(a, b), __ldca(stats + k + h * kGnWarps).y, g.inv_m);
    }
  }
  __syncthreads();
  if (!w.on) return;
  GnChannels c;
  gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return __ldca(stats + k); });
  GnInner s;
  gn_inner(s, g, w, [&](int k) { return inner[k]; });
  gn_forwards<B>(count, first, step, issue, [&](int slot, u32 at) {
    store_piece(piece_at(dx, at), gn_backward<T, ACT>(ring.input(slot, at), ring.grad(slot), c, s));
  });
}

// ---------------------------------------------------------------- one launch
//
// The parts of a slab are the CTAs of a cluster (1 to 16) and the sums cross CTAs through distributed shared
// memory, so one launch does both passes and the second one finds its data close by: it goes through the pieces
// backwards, those that are still in the ring first (all of them, where a part fits), the others again from L2.
//
// Measured at 256 x 64 x 56 x 56 fp16 with SiLU and 8 groups: 49.9 us forward (4120 GB/s counting x and y once, 63 % of
// what a copy reaches), 87.0 us backward with the sum of the parts (3550 GB/s, 54 %); 29.6 and 42.4 us at
// 128 x 192 x 28 x 28 with 8-bit codes.  Nothing is used up: forward 53 % of the issue slots and 53 % of the special
// functions (two a value), backward 50 % and 59 % (four a value).  What bounds them is this structure: a thread asks for
// its own 16 bytes at a time and waits for them, and the CTAs of an SM begin together, so that they load and compute in
// turn more than at a time.  It is not the activation: 53 and 85 us without one.  What did not help: a CTA
// that goes on to the next image and requests it during its second pass (the bookkeeping of an image came back as
// waiting, in every warp), five CTAs of 96 registers instead of four of 128 (88.6 us backward instead of 87 then),
// smaller parts (the second pass of the backward kernel finds 130 of 206 MB no longer in L2; parts of a quarter of that
// size took 88.3 us, because they pay the reductions more often), one reciprocal for two values, keeping the first
// pass's gradients in shared memory.  Not tried: a producer warp that fetches whole rows by bulk copies for the others.

template <class T, int ACT, bool CODES>
__global__ void __launch_bounds__(kGnThreads, 768 / kGnThreads)
groupnorm_2d_fwd_kernel(T* __restrict__ y, float2* __restrict__ stats, uint2* __restrict__ codes,
                        unsigned char* __restrict__ exponents, const T* __restrict__ x,
                        const float* __restrict__ weight, const float* __restrict__ bias, const GnGeom g) {
  extern __shared__ uint4 dynamic[];
  const GnReduce red = gn_reduce(dynamic, g);
  float2* own = red.group + g.slab_groups;
  float2* stat = own + g.slab_groups;
  constexpr int B = GnBatch<T>::forward, plane = 4 * B * kGnThreads;
  uint4* data = reinterpret_cast<uint4*>(reinterpret_cast<char*>(dynamic) + g.data_at) + threadIdx.x;

  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const u32 first = gn_first_piece(g, w), step = gn_step(g, w);
  const long long start = gn_part_start(g, w);
  x += start * 8;
  y += start * 8;
  if (CODES) codes += start, exponents += start;
  const auto issue = [&](int slot, u32 at) { keep_piece(data + slot * kGnThreads, plane, piece_at(x, at)); };
  gn_request<B>(count, first, step, issue);
  GnSums t;
  t.clear();
  if (count > 0) t.start(values_of(load_piece(piece_at(x, first))));
  gn_forwards<B>(count, first, step, issue, [&](int slot, u32) {
    t.add(values_of(kept_piece<T>(data + slot * kGnThreads, plane)));
  });
  gn_group_stats(g, w, t, red, [&](int k, float2 v) { own[k] = v; });
  const GnAffine affine = w.on ? gn_affine(w, weight, bias) : GnAffine();  // (on its way across the barrier)
  gn_cluster_sync(g);
  gn_cluster_stats(g, w, own, [&](int k, float2 v) {
    const float2 st = make_float2(v.x, rsqrtf(fmaf(not_below_zero(v.y), g.inv_m, g.eps)));
    stat[k] = st;
    if (stats != nullptr && w.part == 0) stats[gn_first_group(g, w) + k] = st;
  });
  __syncthreads();
  gn_cluster_done(g, w);  // waited for at the end
  if (w.on) {
    GnChannels c;
    gn_channels(c, g, w, affine, [&](int k) { return stat[k]; });
    gn_backwards<B>(g.batches, count, first, step, issue, [&](int slot, u32 at) {
      gn_write<T, ACT, CODES>(y, codes, exponents, at, kept_piece<T>(data + slot * kGnThreads, plane), c);
    });
  }
  if (g.cluster > 1) cluster_wait();  // no CTA leaves while another reads its values
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
  grid_dependency_wait();
  grid_dependency_launch_dependents();
  const GnWork w = gn_work(g, blockIdx.x);
  const int count = gn_count(w);
  const u32 first = gn_first_piece(g, w), step = gn_step(g, w);
  const long long start = gn_part_start(g, w);
  GnBackRing<T, CODES> ring(dynamic, g, start, dy, x, codes, exponents);
  if (dx != nullptr) dx += start * 8;
  const auto issue = [&](int slot, u32 at) { ring.issue(slot, at); };
  constexpr int B = GnBatch<T>::backward;
  gn_request<B>(count, first, step, issue);
  stats += gn_first_group(g, w);
  GnChannels c;
  if (w.on) gn_channels(c, g, w, gn_affine(w, weight, bias), [&](int k) { return __ldca(stats + k); });
  GnBackSums t;
  t.clear();
  gn_forwards<B>(count, first, step, issue,
                 [&](int slot, u32 at) { t.add<T, ACT>(ring.input(slot, at), ring.grad(slot), c); });
  gn_back_groups(g, w, t, stats, weight, red, [&](int k, float2 v) { own[k] = v; });
  if (g.cluster > 1) cluster_arrive();
  if (part_channel != nullptr) gn_back_channels(g, w, stats, red, part_channel + (w.image * g.parts + w.part) * 2 * g.c);
  if (g.cluster > 1) cluster_wait();
  else __syncthreads();
  gn_cluster_sums(g, w, own, [&](int k, float2 v) { inner[k] = gn_inner_of(v, __ldca(stats + k).y, g.inv_m); });
  __syncthreads();
  gn_cluster_done(g, w);
  if (w.on && dx != nullptr) {
    GnInner s;
    gn_inner(s, g, w, [&](int k) { return inner[k]; });
    gn_backwards<B>(g.batches, count, first, step, issue, [&](int slot, u32 at) {
      store_piece(piece_at(dx, at), gn_backward<T, ACT>(ring.input(slot, at), ring.grad(slot), c, s));
    });
  }
  if (g.cluster > 1) cluster_wait();
}

}  // namespace GN_NAMESPACE
}  // namespace spio_b200

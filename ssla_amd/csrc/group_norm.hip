// Group norm with an activation, channels last, on gfx950:
//   y = act((x - mean) rstd w + b)
// over the positions of a sample and the C / G channels of a group, with its
// backward.  x is [N, L, C]: a group's values are L runs of C / G channels.
// Bound by memory: the forward moves x and y, the backward x, dy and dx.  Measured:
// 32,768 rows of 8 groups of 64, silu, bf16 18 us (3.8 TB/s); 8 grids of 4,560
// positions and 64 channels, relu, fp32, forward 16 us in two launches, backward 23
// in three.
//
// Values are read W at a time (16 bytes where the groups allow it) and held in
// registers, so the variance is that of the centred values at no second read.
// * A group of up to 64 lanes x 32 values belongs to SG lanes of a wavefront
//   (SG a power of two): means are shuffles among them, nothing is shared.
// * Larger groups: a workgroup takes a slice of a sample, 256 threads x 32
//   values, with a fixed channel vector a thread.  A sample of one slice is
//   normalised in the same kernel; else every slice leaves count, mean and
//   centred sum of squares of its part, which are joined by the formula for the
//   moments of two sets, and a second pass normalises.
// The gradients of weight and bias are sums of fixed order: per thread, per
// workgroup or lane group in memory, then down the columns in two steps.
#include "vec.h"

namespace ssla {
namespace {

constexpr int kNone = SSLA_ACT_NONE, kRelu = SSLA_ACT_RELU, kSilu = SSLA_ACT_SILU;
constexpr int kHold = 32;   // values of x that a thread holds

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == kRelu) return z > 0.f ? z : (z != z ? z : 0.f);
  if (act == kSilu) return z / (1.f + fast_exp2(-kLog2e * z));
  return z;
}
// d act / dz
__device__ __forceinline__ float act_grad(int act, float z) {
  if (act == kRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kSilu) {
    const float s = 1.f / (1.f + fast_exp2(-kLog2e * z));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  return 1.f;
}

struct NormArgs {
  const void *x, *dy;
  const float *w, *b;
  void *y;             // y, or dx (may be NULL in the backward)
  float *stats;        // [N, G, 2]: written by the forward (may be NULL), read by the backward
  float *part;         // moments or sums of the slices
  float *cols;         // backward: rows of dw and db sums, [rows][2][C]; NULL: not wanted
  int64_t N, L;
  int C, G, act, join;
  float eps;
};

// The backward's per-value factor: h = dy act'(z) w, dz = dy act'(z).
struct Point { float xh, dz, h; };
__device__ __forceinline__ Point point_of(float x, float dy, float mean, float rstd, float w, float b, int act) {
  Point p;
  p.xh = (x - mean) * rstd;
  p.dz = dy * act_grad(act, fmaf(p.xh, w, b));
  p.h = p.dz * w;
  return p;
}

// W values of a weight vector, or of its default.
template <int W>
__device__ __forceinline__ void load_row(const float *p, int c, bool on, float other, float (&x)[W]) {
#pragma unroll
  for (int e = 0; e < W; ++e) x[e] = other;
  if (!p || !on) return;
  if constexpr (W >= 4) {   // (rows of channels begin at a multiple of 16 bytes of an aligned vector: see widest)
#pragma unroll
    for (int e = 0; e < W; e += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4 *>(p + c + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[e + i] = v[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) x[e] = p[c + e];
  }
}

// --------------------------------------------------- groups of one wavefront --
// Lane j of the SG lanes of a group has its vectors j, j + SG, ...; the lane
// groups of a launch step over the samples, each with one group of channels.
template <int DT, int W, int NV, bool BWD>
__global__ __launch_bounds__(256) void norm_lanes_kernel(const NormArgs a, int SG, int64_t slots) {
  const int per = a.C / a.G, pv = per / W, nv = static_cast<int>(a.L) * pv;
  const int64_t sub = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / SG;
  const int j = threadIdx.x & (SG - 1), g = static_cast<int>(sub % a.G);
  const bool on = sub < slots * a.G;
  const float inv = 1.f / static_cast<float>(a.L * per);
  int off[NV];
  bool ok[NV];
  float w[NV][W], b[NV][W], sw[BWD ? NV : 1][W], sb[BWD ? NV : 1][W];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = j + SG * i, row = v / pv, c = g * per + (v - row * pv) * W;
    ok[i] = on && v < nv;
    off[i] = row * a.C + c;
    load_row<W>(a.w, c, ok[i], 1.f, w[i]);
    load_row<W>(a.b, c, ok[i], 0.f, b[i]);
    if constexpr (BWD)
#pragma unroll
      for (int e = 0; e < W; ++e) sw[i][e] = sb[i][e] = 0.f;
  }
  auto sum = [&](float x) __attribute__((always_inline)) {
    for (int d = 1; d < SG; d <<= 1) x += __shfl_xor(x, d);
    return x;
  };
  Vec<DT, W> x[NV], nx[NV], dy[BWD ? NV : 1], ndy[BWD ? NV : 1];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t n) __attribute__((always_inline)) {
    const int64_t base = n * a.L * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (ok[i]) {
        nx[i] = load_vec<DT, W>(a.x, base + off[i]);
        if constexpr (BWD) ndy[i] = load_vec<DT, W>(a.dy, base + off[i]);
      }
    if constexpr (BWD) {
      nmean = a.stats[2 * (n * a.G + g)];
      nrstd = a.stats[2 * (n * a.G + g) + 1];
    }
  };
  if (!on) return;   // (whole lane groups)
  fetch(sub / a.G);
  for (int64_t n = sub / a.G; n < a.N; n += slots) {
    const int64_t base = n * a.L * a.C, st = 2 * (n * a.G + g);
    const float mean_in = nmean, rstd_in = nrstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      if constexpr (BWD) dy[i] = ndy[i];
    }
    if (n + slots < a.N) fetch(n + slots);   // the next sample's, in flight meanwhile
    if constexpr (!BWD) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (ok[i])
#pragma unroll
          for (int e = 0; e < W; ++e) s += x[i][e];
      const float mean = sum(s) * inv;
      s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (ok[i])
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float d = x[i][e] - mean;
            s = fmaf(d, d, s);
          }
      const float rstd = 1.f / sqrtf(sum(s) * inv + a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (ok[i]) {
          Vec<DT, W> y;
#pragma unroll
          for (int e = 0; e < W; ++e) y.set(e, act_of(a.act, fmaf((x[i][e] - mean) * rstd, w[i][e], b[i][e])));
          store_vec<DT, W>(a.y, base + off[i], y);
        }
      if (a.stats && j == 0) {
        a.stats[st] = mean;
        a.stats[st + 1] = rstd;
      }
    } else {
      const float mean = mean_in, rstd = rstd_in;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (ok[i])
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const Point p = point_of(x[i][e], dy[i][e], mean, rstd, w[i][e], b[i][e], a.act);
            s0 += p.h;
            s1 = fmaf(p.h, p.xh, s1);
            sb[i][e] += p.dz;
            sw[i][e] = fmaf(p.dz, p.xh, sw[i][e]);
          }
      if (a.y) {
        s0 = sum(s0) * inv;
        s1 = sum(s1) * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (ok[i]) {
            Vec<DT, W> dx;
#pragma unroll
            for (int e = 0; e < W; ++e) {
              const Point p = point_of(x[i][e], dy[i][e], mean, rstd, w[i][e], b[i][e], a.act);
              dx.set(e, rstd * (p.h - s0 - p.xh * s1));
            }
            store_vec<DT, W>(a.y, base + off[i], dx);
          }
      }
    }
  }
  if constexpr (BWD) {
    if (a.cols) {
      // row (slot, position): a position's channels of every slot
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (ok[i]) {
          const int row = off[i] / a.C, c = off[i] - row * a.C;
          float *dst = a.cols + ((sub / a.G) * a.L + row) * 2 * a.C + c;
#pragma unroll
          for (int e = 0; e < W; ++e) {
            dst[e] = sw[i][e];
            dst[a.C + e] = sb[i][e];
          }
        }
    }
  }
}

// --------------------------------------------------------------- slices --
// A slice: RT x NR rows by up to 256 / RT channel vectors; thread (rt, cv) has
// rows rt, rt + RT, ... of vector cv.
struct Slice {
  int cv, CT, RT, cblocks, rblocks;
};
__host__ __device__ inline Slice slice_of(int64_t L, int C, int W) {
  Slice s;
  s.cv = C / W;
  s.CT = s.cv < 256 ? s.cv : 256;
  s.RT = 256 / s.CT;
  s.cblocks = (s.cv + s.CT - 1) / s.CT;
  const int64_t rows = static_cast<int64_t>(s.RT) * (kHold / W);
  s.rblocks = static_cast<int>((L + rows - 1) / rows);
  return s;
}

// Sums of a and b over the rows rt, then over each group's vectors of the block:
// thread (group, 8 lanes); the sums of local group k land in sa[k], sb[k].
struct SliceSmem {
  float a[256], b[256], sa[256], sb[256];
};
__device__ __forceinline__ void group_sums(SliceSmem &sm, const Slice &s, int c0, int cw, int pv, float xa, float xb) {
  const int tid = threadIdx.x;
  __syncthreads();
  sm.a[tid] = xa;
  sm.b[tid] = xb;
  __syncthreads();
  float ya = 0.f, yb = 0.f;
  if (tid < s.CT)
    for (int r = 0; r < s.RT; ++r) {
      ya += sm.a[r * s.CT + tid];
      yb += sm.b[r * s.CT + tid];
    }
  __syncthreads();
  sm.a[tid] = ya;
  sm.b[tid] = yb;
  __syncthreads();
  const int g0 = c0 / pv, ng = (c0 + cw - 1) / pv - g0 + 1;
  for (int k0 = 0; k0 < ng; k0 += 32) {
    const int k = k0 + (tid >> 3);
    const int lo = max((g0 + k) * pv - c0, 0), hi = min((g0 + k + 1) * pv - c0, cw);
    ya = yb = 0.f;
    if (k < ng)
      for (int v = lo + (tid & 7); v < hi; v += 8) {
        ya += sm.a[v];
        yb += sm.b[v];
      }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
      ya += __shfl_xor(ya, d);
      yb += __shfl_xor(yb, d);
    }
    if (k < ng && (tid & 7) == 0) {
      sm.sa[k] = ya;
      sm.sb[k] = yb;
    }
  }
  __syncthreads();
}

// Joins the slices of group i of all groups on one wavefront (every lane returns
// the result): mean and centred squares, or the two sums.  A slice whose channels
// lie elsewhere holds nothing of the group and wrote nothing.
template <bool BWD>
__device__ __forceinline__ void join_slices(const float *__restrict__ part, const Slice &s, int64_t i, int g, int pv,
                                            float &u, float &v) {
  const int lane = threadIdx.x & 63;
  const int b0 = g * pv / s.CT, b1 = ((g + 1) * pv - 1) / s.CT, nb = b1 - b0 + 1;   // its channel blocks
  float cnt = 0.f;
  u = v = 0.f;
  auto join = [&](float c2, float u2, float v2) __attribute__((always_inline)) {
    if constexpr (BWD) {
      u += u2;
      v += v2;
    } else if (c2 > 0.f) {
      const float c = cnt + c2, d = u2 - u, f = c2 / c;
      u = fmaf(d, f, u);
      v += v2 + d * d * cnt * f;
      cnt = c;
    }
  };
  for (int64_t k = lane; k < static_cast<int64_t>(s.rblocks) * nb; k += 64) {
    const float *p = part + ((i * s.rblocks + k / nb) * s.cblocks + b0 + k % nb) * (BWD ? 2 : 3);
    if constexpr (BWD) join(0.f, p[0], p[1]);
    else join(p[0], p[1], p[2]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float c2 = __shfl_xor(cnt, d), u2 = __shfl_xor(u, d), v2 = __shfl_xor(v, d);
    if constexpr (!BWD) {   // both lanes join in the same order
      const bool up = lane & d;
      const float cx = up ? cnt : c2, ux = up ? u : u2, vx = up ? v : v2;
      cnt = up ? c2 : cnt;
      u = up ? u2 : u;
      v = up ? v2 : v;
      if (cnt == 0.f) { cnt = cx; u = ux; v = vx; }
      else join(cx, ux, vx);
    } else {
      u += u2;
      v += v2;
    }
  }
}

// STAGE 0: a sample is one slice, all in one pass; 1: the slices' moments (or
// sums) and, in the backward, the columns' sums; 2: y (or dx) from the joined
// ones, which a workgroup of a few slices joins itself (a.join: one launch less).
template <int DT, int W, bool BWD, int STAGE>
__global__ __launch_bounds__(256) void norm_slice_kernel(const NormArgs a) {
  constexpr int NR = kHold / W;
  __shared__ SliceSmem sm;
  const Slice s = slice_of(a.L, a.C, W);
  const int per = a.C / a.G, pv = per / W;
  const int cb = static_cast<int>(blockIdx.x % s.cblocks);
  const int64_t rest = blockIdx.x / s.cblocks, rb = rest % s.rblocks, n = rest / s.rblocks;
  const int rt = threadIdx.x / s.CT, cl = threadIdx.x - rt * s.CT, c0 = cb * s.CT, cw = min(s.CT, s.cv - c0);
  const int c = (c0 + cl) * W, g = min((c0 + cl) / pv, a.G - 1), k = g - c0 / pv;   // channel, group, group in the block
  const bool on = rt < s.RT && cl < cw;
  const int64_t r0 = rb * s.RT * NR, rows = min(static_cast<int64_t>(s.RT) * NR, a.L - r0);
  const int64_t base = (n * a.L + r0) * a.C + c;
  float w[W], b[W];
  load_row<W>(a.w, c, on, 1.f, w);
  load_row<W>(a.b, c, on, 0.f, b);
  Vec<DT, W> x[NR], dy[BWD ? NR : 1];
#pragma unroll
  for (int i = 0; i < NR; ++i)
    if (on && rt + s.RT * i < rows) {
      const int64_t at = base + static_cast<int64_t>(rt + s.RT * i) * a.C;
      x[i] = load_vec<DT, W>(a.x, at);
      if constexpr (BWD) dy[i] = load_vec<DT, W>(a.dy, at);
    }
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (on && rt + s.RT * i < rows)
#pragma unroll
        for (int e = 0; e < W; ++e) f(i, e);
  };
  const int64_t st = 2 * (n * a.G + g);
  if (STAGE == 2 && a.join) {
    const int g0 = c0 / pv, ng = (c0 + cw - 1) / pv - g0 + 1;
    for (int i = threadIdx.x >> 6; i < ng; i += 4) {
      float u, v;
      join_slices<BWD>(a.part, s, n * a.G + g0 + i, g0 + i, pv, u, v);
      if ((threadIdx.x & 63) == 0) {
        sm.sa[i] = u;
        sm.sb[i] = BWD ? v : 1.f / sqrtf(v / (static_cast<float>(a.L) * per) + a.eps);
      }
    }
    __syncthreads();
  }
  if constexpr (!BWD) {
    float mean = 0.f, rstd = 0.f;
    if constexpr (STAGE == 2) {
      mean = a.join ? sm.sa[k] : a.stats[st];
      rstd = a.join ? sm.sb[k] : a.stats[st + 1];
      if (a.join && a.stats && on && rb == 0 && rt == 0 && (c0 + cl) % pv == 0) {
        a.stats[st] = mean;
        a.stats[st + 1] = rstd;
      }
    } else {
      const float cnt = static_cast<float>(rows) * W *
                        static_cast<float>(min((g + 1) * pv, c0 + cw) - max(g * pv, c0));   // values of the group in the slice
      float t = 0.f;
      each([&](int i, int e) { t += x[i][e]; });
      group_sums(sm, s, c0, cw, pv, on ? t : 0.f, 0.f);
      mean = sm.sa[k] / cnt;
      t = 0.f;
      each([&](int i, int e) {
        const float d = x[i][e] - mean;
        t = fmaf(d, d, t);
      });
      group_sums(sm, s, c0, cw, pv, on ? t : 0.f, 0.f);
      // the first lane of the group's first vector in the block speaks for it
      const bool first = on && rt == 0 && (cl == 0 || (c0 + cl) % pv == 0);
      if constexpr (STAGE == 1) {
        if (first) {
          float *dst = a.part + (((n * a.G + g) * s.rblocks + rb) * s.cblocks + cb) * 3;
          dst[0] = cnt;
          dst[1] = mean;
          dst[2] = sm.sa[k];
        }
        return;
      }
      rstd = 1.f / sqrtf(sm.sa[k] / cnt + a.eps);
      if (a.stats && first) {
        a.stats[st] = mean;
        a.stats[st + 1] = rstd;
      }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (on && rt + s.RT * i < rows) {
        Vec<DT, W> y;
#pragma unroll
        for (int e = 0; e < W; ++e) y.set(e, act_of(a.act, fmaf((x[i][e] - mean) * rstd, w[e], b[e])));
        store_vec<DT, W>(a.y, base + static_cast<int64_t>(rt + s.RT * i) * a.C, y);
      }
  } else {
    const float mean = a.stats[st], rstd = a.stats[st + 1], inv = 1.f / (static_cast<float>(a.L) * per);
    float s0 = 0.f, s1 = 0.f;
    if constexpr (STAGE < 2) {
      float sw[W], sb[W];
#pragma unroll
      for (int e = 0; e < W; ++e) sw[e] = sb[e] = 0.f;
      each([&](int i, int e) {
        const Point p = point_of(x[i][e], dy[i][e], mean, rstd, w[e], b[e], a.act);
        s0 += p.h;
        s1 = fmaf(p.h, p.xh, s1);
        sb[e] += p.dz;
        sw[e] = fmaf(p.dz, p.xh, sw[e]);
      });
      if (a.y) {
        group_sums(sm, s, c0, cw, pv, on ? s0 : 0.f, on ? s1 : 0.f);
        s0 = sm.sa[k] * inv;
        s1 = sm.sb[k] * inv;
        if (STAGE == 1 && on && rt == 0 && (cl == 0 || (c0 + cl) % pv == 0)) {
          float *dst = a.part + (((n * a.G + g) * s.rblocks + rb) * s.cblocks + cb) * 2;
          dst[0] = s0;
          dst[1] = s1;
        }
      }
      if (a.cols) {   // the block's columns over the rows rt
#pragma unroll
        for (int e = 0; e < W; ++e) {
          __syncthreads();
          sm.a[threadIdx.x] = on ? sw[e] : 0.f;
          sm.b[threadIdx.x] = on ? sb[e] : 0.f;
          __syncthreads();
          if (rt == 0 && on) {
            float ya = 0.f, yb = 0.f;
            for (int r = 0; r < s.RT; ++r) {
              ya += sm.a[r * s.CT + cl];
              yb += sm.b[r * s.CT + cl];
            }
            float *dst = a.cols + (n * s.rblocks + rb) * 2 * a.C + c + e;
            dst[0] = ya;
            dst[a.C] = yb;
          }
        }
      }
      if constexpr (STAGE == 1) return;
    } else {
      s0 = a.join ? sm.sa[k] : a.part[st];
      s1 = a.join ? sm.sb[k] : a.part[st + 1];
    }
    if (!a.y) return;
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (on && rt + s.RT * i < rows) {
        Vec<DT, W> dx;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const Point p = point_of(x[i][e], dy[i][e], mean, rstd, w[e], b[e], a.act);
          dx.set(e, rstd * (p.h - s0 - p.xh * s1));
        }
        store_vec<DT, W>(a.y, base + static_cast<int64_t>(rt + s.RT * i) * a.C, dx);
      }
  }
}

template <bool BWD>
__global__ __launch_bounds__(256) void norm_join_kernel(const float *__restrict__ part, int64_t groups, int G, int per,
                                                        int W, int64_t L, int C, float eps, float *__restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= groups) return;   // whole wavefront
  float u, v;
  join_slices<BWD>(part, slice_of(L, C, W), i, static_cast<int>(i % G), per / W, u, v);
  if ((threadIdx.x & 63) == 0) {
    out[2 * i] = u;
    out[2 * i + 1] = BWD ? v : 1.f / sqrtf(v / (static_cast<float>(L) * per) + eps);
  }
}

// Sums down R rows of [R][cols]: workgroup (64 columns, split s of S), 16
// wavefronts with every 16 S-th row each.
__global__ __launch_bounds__(1024) void norm_cols_kernel(const float *__restrict__ src, int64_t R, int64_t cols, int S,
                                                         float *__restrict__ dst, int C, float *__restrict__ dw,
                                                         float *__restrict__ db) {
  __shared__ float sm[16][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t nb = (cols + 63) / 64, c = (blockIdx.x % nb) * 64 + lane, s = blockIdx.x / nb;
  float t = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = s * 16 + w; r < R; r += 16 * S) t += src[r * cols + c];
  }
  sm[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < cols) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += sm[i][lane];
    if (dst) dst[s * cols + c] = t;
    else if (c < C) {
      if (dw) dw[c] = t;
    } else if (db) db[c - C] = t;
  }
}

// ----------------------------------------------------------------- launches --
// How a call runs, from its sizes and the widest vector its addresses allow.
struct NormPlan {
  int W;            // values of a vector
  bool lanes;       // groups of one wavefront
  int SG, NV;
  int64_t slots;    // lane groups a group of channels
  Slice s;
  bool one;         // a sample is one slice
  int64_t part_floats, col_rows;
  int S;            // splits of the column sums
};
constexpr int kColSplits = 64;
// The backward's lane groups keep their columns' sums over the samples they step
// over: 512 workgroups (two a CU) leave 2,048 rows of sums of 8 heads of 64
// channels to add.
constexpr int64_t kBwdBlocks = 512, kFwdBlocks = 4096;

NormPlan plan_of(int64_t N, int64_t L, int C, int G, int W, bool bwd) {
  NormPlan p{};
  const int per = C / G;
  p.W = W;
  const int64_t nv = L * (per / W);
  p.lanes = nv <= 64 * (kHold / W) && L * C <= 0x7fffffff;   // (offsets inside a sample are 32 bits there)
  if (p.lanes) {
    p.SG = 1;
    while (p.SG < 64 && p.SG < nv) p.SG *= 2;
    p.NV = 1;
    while (static_cast<int64_t>(p.SG) * p.NV < nv) p.NV *= 2;
    p.slots = std::min<int64_t>(N, std::max<int64_t>(1, (bwd ? kBwdBlocks : kFwdBlocks) * 256 / p.SG / G));
    p.col_rows = p.slots * L;
  } else {
    p.s = slice_of(L, C, W);
    p.one = p.s.rblocks == 1 && p.s.cblocks == 1;
    p.part_floats = p.one ? 0 : (bwd ? 2 : 3) * N * G * p.s.rblocks * p.s.cblocks + 2 * N * G;
    p.col_rows = N * p.s.rblocks;
  }
  // (one step adds up to 64 rows a wavefront; more are split over the GPU first)
  p.S = p.col_rows <= 1024 ? 1 : static_cast<int>(std::min<int64_t>(kColSplits, p.col_rows / 128));
  return p;
}
int64_t ws_floats(const NormPlan &p, int C, bool bwd) {
  const int64_t part = (p.part_floats + 3) / 4 * 4;
  return bwd ? part + p.col_rows * 2 * C + static_cast<int64_t>(p.S) * 2 * C : part;
}
size_t ws_bytes(int64_t N, int64_t L, int C, int G, bool bwd) {   // whatever vectors the addresses allow
  if (N <= 0 || L <= 0 || C <= 0 || G <= 0 || C % G) return 0;
  int64_t most = 0;
  for (int W = 1; W <= 8; W *= 2)
    if (W != 2 && C / G % W == 0) most = std::max(most, ws_floats(plan_of(N, L, C, G, W, bwd), C, bwd));
  return static_cast<size_t>(most) * sizeof(float);
}

int check_sizes(const char *what, int64_t N, int64_t L, int C, int G, int act) {
  SSLA_CHECK_ARG(N >= 0 && L >= 0 && C > 0 && G > 0 && C % G == 0 && act >= kNone && act <= kSilu,
                 "%s: bad sizes N=%lld L=%lld C=%d G=%d act=%d", what, (long long)N, (long long)L, C, G, act);
  if (N > 0x7fffffff || N * G > 0x7fffffff || L > 0x3fffffff) {
    set_error("%s: too many groups or positions", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  return SSLA_OK;
}

int widest(int per, int dtype, std::initializer_list<const void *> tensors, std::initializer_list<const float *> rows) {
  const int es = dtype == SSLA_F32 ? 4 : 2;
  for (const float *t : rows)
    if (!aligned(t, 16)) return 1;   // (NULL is aligned)
  for (int W = 16 / es; W >= 4; W /= 2) {
    bool ok = per % W == 0;
    for (const void *t : tensors) ok = ok && aligned(t, W * es);
    if (ok) return W;
  }
  return 1;
}

inline dim3 grid_of(int64_t n) { return dim3(static_cast<unsigned>(n)); }

template <int DT, int W, bool BWD>
void launch_norm(const NormPlan &p, const NormArgs &a, float *joined, hipStream_t st) {
  const dim3 block(256);
  if (p.lanes) {
    const dim3 grid = grid_of((p.slots * a.G * p.SG + 255) / 256);
#define SSLA_LANES(NV_)                                                                                             \
  if constexpr (NV_ * W <= kHold)                                                                                   \
    if (p.NV == NV_) hipLaunchKernelGGL((norm_lanes_kernel<DT, W, NV_, BWD>), grid, block, 0, st, a, p.SG, p.slots)
    SSLA_LANES(1);
    SSLA_LANES(2);
    SSLA_LANES(4);
    SSLA_LANES(8);
    SSLA_LANES(16);
    SSLA_LANES(32);
#undef SSLA_LANES
    return;
  }
  const dim3 grid = grid_of(a.N * p.s.rblocks * p.s.cblocks);
  if (p.one) {
    hipLaunchKernelGGL((norm_slice_kernel<DT, W, BWD, 0>), grid, block, 0, st, a);
    return;
  }
  hipLaunchKernelGGL((norm_slice_kernel<DT, W, BWD, 1>), grid, block, 0, st, a);
  if (BWD && !a.y) return;
  NormArgs second = a;
  // up to 64 slices a sample (one a lane) are joined by each workgroup that needs them
  second.join = p.s.rblocks * p.s.cblocks <= 64;
  if (second.join) {
    hipLaunchKernelGGL((norm_slice_kernel<DT, W, BWD, 2>), grid, block, 0, st, second);
    return;
  }
  if (BWD) second.part = joined;
  else second.stats = joined;
  hipLaunchKernelGGL((norm_join_kernel<BWD>), grid_of((a.N * a.G + 3) / 4), block, 0, st, a.part, a.N * a.G, a.G,
                     a.C / a.G, W, a.L, a.C, a.eps, joined);
  hipLaunchKernelGGL((norm_slice_kernel<DT, W, BWD, 2>), grid, block, 0, st, second);
}

template <bool BWD>
int launch_dtype(const char *what, const NormPlan &p, const NormArgs &a, float *joined, int dtype, hipStream_t st) {
  if (p.lanes ? p.slots * a.G > (static_cast<int64_t>(0x7fffffff) * 256) / p.SG
              : a.N * p.s.rblocks * p.s.cblocks > 0x7fffffff) {
    set_error("%s: too many workgroups", what);
    return SSLA_ERR_UNSUPPORTED;
  }
#define SSLA_NORM(DT_)                                            \
  do {                                                            \
    if (DT_ != SSLA_F32 && p.W == 8) {                            \
      if constexpr (DT_ != SSLA_F32) launch_norm<DT_, 8, BWD>(p, a, joined, st); \
    } else if (p.W == 4) launch_norm<DT_, 4, BWD>(p, a, joined, st); \
    else launch_norm<DT_, 1, BWD>(p, a, joined, st);              \
  } while (0)
  if (dtype == SSLA_F32) SSLA_NORM(SSLA_F32);
  else if (dtype == SSLA_BF16) SSLA_NORM(SSLA_BF16);
  else SSLA_NORM(SSLA_F16);
#undef SSLA_NORM
  return SSLA_OK;
}

int check_dtype(const char *what, int dtype) {
  if (dtype == SSLA_F32 || dtype == SSLA_BF16 || dtype == SSLA_F16) return SSLA_OK;
  set_error("%s: unsupported dtype %d", what, dtype);
  return SSLA_ERR_DTYPE;
}
int check_ws(const char *what, const void *ws, size_t have, size_t need) {
  if (need == 0 || (ws && have >= need && aligned(ws, 16))) return SSLA_OK;
  set_error("%s: needs %zu bytes of workspace, got %zu", what, need, have);
  return SSLA_ERR_WORKSPACE;
}

}  // namespace
}  // namespace ssla

extern "C" size_t ssla_group_norm_workspace_size(int64_t N, int64_t L, int C, int G) {
  return ssla::ws_bytes(N, L, C, G, false);
}

extern "C" int ssla_group_norm_fwd(const void *x, int64_t N, int64_t L, int C, int G, const float *weight,
                                   const float *bias, float eps, int act, void *y, float *stats, int dtype,
                                   void *workspace, size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("group_norm_fwd", N, L, C, G, act)) return e;
  if (N == 0 || L == 0) return SSLA_OK;
  SSLA_CHECK_ARG(x && y, "group_norm_fwd: null pointer");
  if (const int e = check_dtype("group_norm_fwd", dtype)) return e;
  if (const int e = check_ws("group_norm_fwd", workspace, workspace_bytes, ws_bytes(N, L, C, G, false))) return e;
  const NormPlan p = plan_of(N, L, C, G, widest(C / G, dtype, {x, y}, {weight, bias}), false);
  float *part = static_cast<float *>(workspace);
  NormArgs a{};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.stats = stats; a.part = part;
  a.N = N; a.L = L; a.C = C; a.G = G; a.act = act; a.eps = eps;
  float *joined = stats ? stats : part + (p.part_floats - 2 * N * G);
  if (const int e = launch_dtype<false>("group_norm_fwd", p, a, joined, dtype, static_cast<hipStream_t>(stream)))
    return e;
  return launch_status("group_norm_fwd");
}

extern "C" size_t ssla_group_norm_bwd_workspace_size(int64_t N, int64_t L, int C, int G) {
  return ssla::ws_bytes(N, L, C, G, true);
}

extern "C" int ssla_group_norm_bwd(const void *dy, const void *x, const float *stats, int64_t N, int64_t L, int C,
                                   int G, const float *weight, const float *bias, int act, void *dx, float *dweight,
                                   float *dbias, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("group_norm_bwd", N, L, C, G, act)) return e;
  const bool none = N == 0 || L == 0;
  SSLA_CHECK_ARG(none || (dy && x && stats), "group_norm_bwd: null pointer");
  if (const int e = check_dtype("group_norm_bwd", dtype)) return e;
  if (const int e = check_ws("group_norm_bwd", workspace, workspace_bytes, ws_bytes(N, L, C, G, true))) return e;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool sums = dweight || dbias;
  NormPlan p{};
  float *part = static_cast<float *>(workspace), *cols = nullptr, *split = nullptr;
  if (!none) {
    if (!dx && !sums) return SSLA_OK;
    p = plan_of(N, L, C, G, widest(C / G, dtype, dx ? std::initializer_list<const void *>{x, dy, dx}
                                                    : std::initializer_list<const void *>{x, dy}, {weight, bias}), true);
    cols = part + (p.part_floats + 3) / 4 * 4;
    split = cols + p.col_rows * 2 * C;
    NormArgs a{};
    a.x = x; a.dy = dy; a.w = weight; a.b = bias; a.y = dx; a.stats = const_cast<float *>(stats); a.part = part;
    a.cols = sums ? cols : nullptr;
    a.N = N; a.L = L; a.C = C; a.G = G; a.act = act;
    if (const int e = launch_dtype<true>("group_norm_bwd", p, a, part + (p.part_floats - 2 * N * G), dtype, st)) return e;
  }
  if (sums) {
    const int64_t wide = 2 * static_cast<int64_t>(C), nb = (wide + 63) / 64;
    const dim3 block(1024);
    if (p.S > 1) {
      hipLaunchKernelGGL(norm_cols_kernel, grid_of(nb * p.S), block, 0, st, cols, p.col_rows, wide, p.S, split, C,
                         dweight, dbias);
      hipLaunchKernelGGL(norm_cols_kernel, grid_of(nb), block, 0, st, split, static_cast<int64_t>(p.S), wide, 1,
                         static_cast<float *>(nullptr), C, dweight, dbias);
    } else {   // (no rows at all: zeros)
      hipLaunchKernelGGL(norm_cols_kernel, grid_of(nb), block, 0, st, cols, none ? 0 : p.col_rows, wide, 1,
                         static_cast<float *>(nullptr), C, dweight, dbias);
    }
  }
  return launch_status("group_norm_bwd");
}

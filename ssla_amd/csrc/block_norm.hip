// Norms around a block, by rows, with their backward passes.
//
// Gated: the norm of an attention's output by groups of channels, times its gate,
//   y = (n w + b) act(z),  n = (x - mean) rstd  (or x rstd),
//   dz = dy (n w + b) act'(z),  dv = dy act(z),  dw = sum dv n,  db = sum dv,
//   dx = rstd (h - mean(h) - n mean(h n)),  h = dv w   (no mean(h) without a mean)
// Residual: a stream's step from one block to the next,
//   p = norm2(x) w2 (or x),  s = r + c keep p,  y = norm(s) w + b
// with c = alpha gamma / (1 - p) and keep a mask that is drawn again in the backward:
//   ds = ds' + norm'(dy),  dr = ds,  dgamma = sum ds keep p,  dp = c keep ds,
//   dw2 = sum dp n2,  dx = norm2'(dp).
//
// Bound by memory: each tensor is read or written once in either direction.  A row
// (a group of one) lies in the registers of S lanes, S a power of two: up to 64
// lanes of a wavefront with up to 8 values each, whose sums are shuffles, or more
// than one wavefront, whose sums are joined in LDS.  Nothing of a norm is kept for the backward: with x (and r)
// at hand again its sums cost shuffles, not memory.  Lane groups step over the rows
// with the next one on its way.  Sums over rows stay with their lanes, are added up
// in the workgroup and then down the workgroups, in a fixed order.
// Measured: 32,768 rows of 8 heads of 64, bf16 18.3 us (5.5 TB/s); 32,768 rows of 1,024
// channels, bf16 with an fp32 stream, dropout and both norms: forward 79 (5.1 TB/s),
// backward 145 (4.2 TB/s, vector units busy 59 % of the time).
#include "philox.h"
#include "vec.h"

#include <math.h>

namespace ssla {
namespace {

constexpr int kHold = 8;        // values that a lane holds of a row
constexpr int kMostLanes = 1024;
constexpr int kFwdThreads = 256, kBwdThreads = 256;   // of a workgroup, unless a row needs more

struct RowArgs {
  const void *x, *r, *z, *dy, *ds;   // ds, and dy of the residual's backward, may be NULL
  int64_t ldx, ldz;                  // elements from row to row of x and z (gated)
  const float *w, *b, *w2, *gamma;   // may be NULL
  void *y, *s;                       // y and the stream, or dx and dr (the backward's may be NULL)
  void *dz;
  float *part;                       // [workgroups][kinds][C] sums over rows; NULL: not wanted
  int64_t N;                         // rows
  int C, G, per, S, layer, post, silu;
  int64_t slots;                     // rows at once, of each group
  float eps, alpha;
  Draw draw;
};

// ------------------------------------------------------------- a row's lanes --
template <int CTRL>
__device__ __forceinline__ float dpp_of(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
// The sum over S neighbouring lanes (a power of two up to 64), the same on each, by lane
// swaps on the VALU: neighbours, pairs, mirrored fours and eights (equal inside them by
// then), rows of 16 and halves.
__device__ __forceinline__ float lane_sum(float x, int S) {
  if (S > 1) x += dpp_of<0xB1>(x);
  if (S > 2) x += dpp_of<0x4E>(x);
  if (S > 4) x += dpp_of<0x141>(x);
  if (S > 8) x += dpp_of<0x140>(x);
  if (S > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (S > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// The sums of M values over a row's lanes, in the same order on every lane.  WIDE: over
// several wavefronts, all threads of the workgroup at once.
template <int WIDE, int M>
__device__ __forceinline__ void row_sums(float (&x)[M], int S, float *sm, int &turn) {
#pragma unroll
  for (int k = 0; k < M; ++k) x[k] = lane_sum(x[k], WIDE ? 64 : S);
  if constexpr (WIDE != 0) {
    float *at = sm + (turn ^= 32);   // (two places in turn: one barrier a sum)
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < M; ++k) at[16 * k + (threadIdx.x >> 6)] = x[k];
    __syncthreads();
    const int waves = S >> 6, first = threadIdx.x / S * waves;
#pragma unroll
    for (int k = 0; k < M; ++k) {
      x[k] = 0.f;
      for (int i = 0; i < waves; ++i) x[k] += at[16 * k + first + i];
    }
  }
}

// f(i, e) of all values held.  Lanes without a value hold zeros that their sums take in.
template <int W, int NV, typename F>
__device__ __forceinline__ void each(F f) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) f(i, e);
}

// Where a lane works: its place j among the S lanes of a row, the group of channels g
// and the first row; lane groups that have none (`on` false) idle along.  A lane's values
// are NV vectors of W neighbouring channels.  FULL: whole ones at their borders, else as
// many of them as the group has channels, read one by one.
template <int W, int NV, bool FULL>
struct Place {
  int j, g, c[NV];
  int64_t row, first;               // its first row, and the workgroup's
  bool on, live;                    // has rows; has one to work on now
  int cols[NV], has[NV], now[NV];   // values that exist; with a row at all; with the row worked on
  __device__ __forceinline__ explicit Place(const RowArgs &a) {
    const int64_t sub = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / a.S;
    j = threadIdx.x & (a.S - 1);
    g = static_cast<int>(sub % a.G);
    row = sub / a.G;
    first = static_cast<int64_t>(blockIdx.x) * blockDim.x / a.S / a.G;
    on = row < a.slots;
    live = on && row < a.N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      c[i] = (j + a.S * i) * W;
      cols[i] = min(max(a.per - c[i], 0), W);
      has[i] = on ? cols[i] : 0;
      now[i] = live ? has[i] : 0;
      c[i] = (cols[i] ? c[i] : 0) + g * a.per;
    }
  }
  // Row n is the one worked on: lanes behind the last row idle along.
  __device__ __forceinline__ void at(int64_t n, int64_t N) {
    live = on && n < N;
#pragma unroll
    for (int i = 0; i < NV; ++i) now[i] = live ? has[i] : 0;
  }
  // The workgroup goes on behind row n (the same for all its threads).
  __device__ __forceinline__ bool again(int64_t n, const RowArgs &a) const { return n - row + first + a.slots < a.N; }
  __device__ __forceinline__ bool is(int i, int e) const { return FULL ? now[i] != 0 : e < now[i]; }
};

// W values of a vector over the channels, or of its default.
template <int W, int NV, bool FULL>
__device__ __forceinline__ void load_weights(const float *p, const Place<W, NV, FULL> &l, int i, float other, float (&x)[W]) {
#pragma unroll
  for (int e = 0; e < W; ++e) x[e] = other;
  if (!p) return;
  if constexpr (FULL) {
#pragma unroll
    for (int e = 0; e < W; e += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4 *>(p + l.c[i] + e);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[e + k] = v[k];
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < l.cols[i]) x[e] = p[l.c[i] + e];
  }
}

// A row's values, zeros where there are none.
template <int DT, int W, int NV, bool FULL>
__device__ __forceinline__ void load_row(Held<DT, W> (&x)[NV], const void *p, int64_t at, const Place<W, NV, FULL> &l, bool on) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    x[i] = Held<DT, W>{};
    if constexpr (FULL) {
      if (l.has[i] && on) x[i] = load_held<DT, W>(p, at + l.c[i]);
    } else if (on) {
      const typename Elem<DT>::T *from = static_cast<const typename Elem<DT>::T *>(p) + at + l.c[i];
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (e < l.has[i]) {
          if constexpr (DT == SSLA_F32) x[i].w[e] = __float_as_uint(from[e]);
          else x[i].w[e >> 1] |= static_cast<uint32_t>(from[e]) << (e & 1 ? 16 : 0);
        }
    }
  }
}
template <int DT, int W, int NV, bool FULL>
__device__ __forceinline__ void store_row(void *p, int64_t at, const Place<W, NV, FULL> &l, int i, const Vec<DT, W> &x) {
  if constexpr (FULL) {
    if (l.now[i]) store_vec<DT, W>(p, at + l.c[i], x);
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < l.now[i]) static_cast<typename Elem<DT>::T *>(p)[at + l.c[i] + e] = x.e[e];
  }
}

// x becomes its normalised values; returns 1 / deviation.
template <int WIDE, bool FULL, int W, int NV>
__device__ __forceinline__ float normalise(float (&x)[NV][W], const Place<W, NV, FULL> &l, const RowArgs &a, float *sm, int &turn) {
  const float inv = 1.f / static_cast<float>(a.per);
  if (a.layer) {
    float t[1] = {0.f};
    each<W, NV>([&](int i, int e) { t[0] += x[i][e]; });
    row_sums<WIDE>(t, a.S, sm, turn);
    const float mean = t[0] * inv;
    each<W, NV>([&](int i, int e) { x[i][e] = l.is(i, e) ? x[i][e] - mean : 0.f; });
  }
  float t[1] = {0.f};
  each<W, NV>([&](int i, int e) { t[0] = fmaf(x[i][e], x[i][e], t[0]); });
  row_sums<WIDE>(t, a.S, sm, turn);
  const float rstd = l.live ? 1.f / sqrtf(t[0] * inv + a.eps) : 0.f;   // (idle lanes stay at zeros)
  each<W, NV>([&](int i, int e) { x[i][e] *= rstd; });
  return rstd;
}
// h, the gradient of normalised values n, becomes that of what they were made of.
template <int WIDE, bool FULL, int W, int NV>
__device__ __forceinline__ void normalise_back(float (&h)[NV][W], const float (&n)[NV][W], float rstd,
                                               const Place<W, NV, FULL> &l, const RowArgs &a, float *sm, int &turn) {
  const float inv = 1.f / static_cast<float>(a.per);
  float t[2] = {0.f, 0.f};
  each<W, NV>([&](int i, int e) {
    t[0] += h[i][e];
    t[1] = fmaf(h[i][e], n[i][e], t[1]);
  });
  row_sums<WIDE>(t, a.S, sm, turn);
  const float m = a.layer ? t[0] * inv : 0.f, v = t[1] * inv;
  each<W, NV>([&](int i, int e) { h[i][e] = l.is(i, e) ? rstd * (h[i][e] - m - n[i][e] * v) : 0.f; });
}

// Adds the workgroup's sums over rows and leaves them in rows of a.part ([rows][KINDS][C]):
// a row a workgroup, or a row a slot where a workgroup has not all groups of channels.
// Lane groups of one group of channels are G apart.  Four or more are added up by all threads,
// a sum each, fewer by the first lane group for its own channels (forward and backward,
// us, the first against the second: 16,384 rows of 4 groups of 16 channels 19, 40;
// 32,768 rows of 1,024 221, 214).
template <int W, int NV, bool FULL, int KINDS>
__device__ __forceinline__ void leave_sums(const RowArgs &a, const Place<W, NV, FULL> &l, const float (&sum)[KINDS][NV][W], float *sm) {
  const int lanes = blockDim.x, groups = lanes / a.S, mine = threadIdx.x / a.S;   // lane groups
  const bool all = a.G <= groups;
  const int64_t to = all ? static_cast<int64_t>(blockIdx.x) : l.row;
  const int own = a.G * a.S;   // lanes before the first group of channels comes again
#pragma unroll
  for (int k = 0; k < KINDS; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) sm[(e * NV + i) * lanes + threadIdx.x] = l.has[i] ? sum[k][i][e] : 0.f;
    __syncthreads();
    if (4 * own <= lanes) {
      for (int o = threadIdx.x; o < own * W * NV; o += lanes) {
        const uint32_t v = static_cast<uint32_t>(o) / own, at = o - v * own, q = at / a.S, j = at - q * a.S;
        const uint32_t g = (blockIdx.x * groups + q) % a.G, c = (j + a.S * (v % NV)) * W + v / NV;
        if (c >= static_cast<uint32_t>(a.per)) continue;
        float t = 0.f;
#pragma unroll 8
        for (int x = at; x < lanes; x += own) t += sm[v * lanes + x];
        a.part[(to * KINDS + k) * a.C + g * a.per + c] = t;
      }
    } else if (mine < a.G && (all || l.on)) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (e < l.cols[i]) {
            float t = 0.f;
            for (int q = mine; q < groups; q += a.G) t += sm[(e * NV + i) * lanes + q * a.S + l.j];
            a.part[(to * KINDS + k) * a.C + l.c[i] + e] = t;
          }
    }
  }
}

__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * z)); }

// -------------------------------------------------------------------- gated --
template <int DT, int W, int NV, bool FULL, int WIDE>
__global__ __launch_bounds__(WIDE ? WIDE : kFwdThreads) void gated_fwd_kernel(const RowArgs a) {
  __shared__ float sm[64];
  int turn = 0;
  Place<W, NV, FULL> l(a);
  Held<DT, W> x[NV], z[NV], nx[NV], nz[NV];
  load_row<DT, W, NV, FULL>(nx, a.x, l.row * a.ldx, l, l.row < a.N);
  load_row<DT, W, NV, FULL>(nz, a.z, l.row * a.ldz, l, l.row < a.N);
  for (int64_t n = l.row; n - l.row + l.first < a.N; n += a.slots) {   // (as often in the whole workgroup)
    l.at(n, a.N);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      z[i] = nz[i];
    }
    if (l.again(n, a)) {
      const bool more = n + a.slots < a.N;
      load_row<DT, W, NV, FULL>(nx, a.x, (n + a.slots) * a.ldx, l, more);
      load_row<DT, W, NV, FULL>(nz, a.z, (n + a.slots) * a.ldz, l, more);
    }
    float v[NV][W];
    each<W, NV>([&](int i, int e) { v[i][e] = x[i][e]; });
    normalise<WIDE, FULL, W, NV>(v, l, a, sm, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[W], b[W];
      load_weights(a.w, l, i, 1.f, w);
      load_weights(a.b, l, i, 0.f, b);
      Vec<DT, W> y;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float g = z[i][e], s = sigmoid_of(g);
        y.set(e, fmaf(v[i][e], w[e], b[e]) * (a.silu ? g * s : s));
      }
      store_row<DT>(a.y, n * a.C, l, i, y);
    }
  }
}

template <int DT, int W, int NV, bool FULL, int WIDE>
__global__ __launch_bounds__(WIDE ? WIDE : kBwdThreads) void gated_bwd_kernel(const RowArgs a) {
  __shared__ float sm[(WIDE ? WIDE : kBwdThreads) * kHold];
  int turn = 0;
  Place<W, NV, FULL> l(a);
  float sum[2][NV][W];   // of w and b
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) sum[0][i][e] = sum[1][i][e] = 0.f;
  Held<DT, W> x[NV], z[NV], dy[NV], nx[NV], nz[NV], ndy[NV];
  auto fetch = [&](int64_t n, bool on) {
    load_row<DT, W, NV, FULL>(nx, a.x, n * a.ldx, l, on);
    load_row<DT, W, NV, FULL>(nz, a.z, n * a.ldz, l, on);
    load_row<DT, W, NV, FULL>(ndy, a.dy, n * a.C, l, on);
  };
  fetch(l.row, l.row < a.N);
  for (int64_t n = l.row; n - l.row + l.first < a.N; n += a.slots) {   // (as often in the whole workgroup)
    l.at(n, a.N);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      z[i] = nz[i];
      dy[i] = ndy[i];
    }
    if (l.again(n, a)) fetch(n + a.slots, n + a.slots < a.N);   // (zeros behind the last row: those lanes add nothing)
    float v[NV][W], h[NV][W];
    each<W, NV>([&](int i, int e) { v[i][e] = x[i][e]; });
    const float rstd = normalise<WIDE, FULL, W, NV>(v, l, a, sm, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[W], b[W];
      load_weights(a.w, l, i, 1.f, w);
      load_weights(a.b, l, i, 0.f, b);
      Vec<DT, W> dz;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float g = z[i][e], s = sigmoid_of(g), o = sigmoid_of(-g);
        const float act = a.silu ? g * s : s, slope = a.silu ? fmaf(g * s, o, s) : s * o;
        const float d = dy[i][e], dv = d * act;
        dz.set(e, d * fmaf(v[i][e], w[e], b[e]) * slope);
        sum[0][i][e] = fmaf(dv, v[i][e], sum[0][i][e]);
        sum[1][i][e] += dv;
        h[i][e] = dv * w[e];
      }
      if (a.dz) store_row<DT>(a.dz, n * a.C, l, i, dz);
    }
    if (a.y) {
      normalise_back<WIDE, FULL, W, NV>(h, v, rstd, l, a, sm, turn);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Vec<DT, W> dx;
#pragma unroll
        for (int e = 0; e < W; ++e) dx.set(e, h[i][e]);
        store_row<DT>(a.y, n * a.C, l, i, dx);
      }
    }
  }
  if (a.part) leave_sums<W, NV, FULL, 2>(a, l, sum, sm);
}

// ----------------------------------------------------------------- residual --
// The stream's value before its norm and, for the backward, what is kept of the way
// there: the branch's normalised values, their 1 / deviation and the mask.
template <int DT, int DTR, int W, int NV, bool FULL, int WIDE>
struct Stream {
  float s[NV][W], n2[NV][W], rstd2;
  uint32_t keep[NV];
  __device__ __forceinline__ void run(const RowArgs &a, const Place<W, NV, FULL> &l, const Held<DT, W> (&x)[NV], const Held<DTR, W> (&r)[NV],
                                      float scale, uint64_t seed, int64_t n, float *sm, int &turn) {
    each<W, NV>([&](int i, int e) { n2[i][e] = x[i][e]; });
    rstd2 = a.post ? normalise<WIDE, FULL, W, NV>(n2, l, a, sm, turn) : 1.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      keep[i] = ~0u;
      if (a.draw.threshold) keep[i] = kept<W, FULL>(a.draw, seed, static_cast<uint64_t>(n) * a.C + l.c[i]);
      float w2[W], c[W];
      load_weights(a.w2, l, i, 1.f, w2);
      load_weights(a.gamma, l, i, 1.f, c);
#pragma unroll
      for (int e = 0; e < W; ++e) s[i][e] = r[i][e] + (keep[i] >> e & 1 ? c[e] * scale * (n2[i][e] * w2[e]) : 0.f);
    }
  }
};

template <int DT, int DTR, int W, int NV, bool FULL, int WIDE>
__global__ __launch_bounds__(WIDE ? WIDE : kFwdThreads) void residual_fwd_kernel(const RowArgs a) {
  __shared__ float sm[64];
  int turn = 0;
  Place<W, NV, FULL> l(a);
  const float scale = a.alpha * (a.draw.threshold ? a.draw.scale : 1.f);
  const uint64_t seed = a.draw.threshold ? static_cast<uint64_t>(*a.draw.seed) : 0;
  Held<DT, W> x[NV], nx[NV];
  Held<DTR, W> r[NV], nr[NV];
  load_row<DT, W, NV, FULL>(nx, a.x, l.row * a.C, l, l.row < a.N);
  load_row<DTR, W, NV, FULL>(nr, a.r, l.row * a.C, l, l.row < a.N);
  for (int64_t n = l.row; n - l.row + l.first < a.N; n += a.slots) {   // (as often in the whole workgroup)
    l.at(n, a.N);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      r[i] = nr[i];
    }
    if (l.again(n, a)) {
      const bool more = n + a.slots < a.N;
      load_row<DT, W, NV, FULL>(nx, a.x, (n + a.slots) * a.C, l, more);
      load_row<DTR, W, NV, FULL>(nr, a.r, (n + a.slots) * a.C, l, more);
    }
    Stream<DT, DTR, W, NV, FULL, WIDE> t;
    t.run(a, l, x, r, scale, seed, n, sm, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec<DTR, W> s;
#pragma unroll
      for (int e = 0; e < W; ++e) s.set(e, t.s[i][e]);
      store_row<DTR>(a.s, n * a.C, l, i, s);
    }
    normalise<WIDE, FULL, W, NV>(t.s, l, a, sm, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[W], b[W];
      load_weights(a.w, l, i, 1.f, w);
      load_weights(a.b, l, i, 0.f, b);
      Vec<DT, W> y;
#pragma unroll
      for (int e = 0; e < W; ++e) y.set(e, fmaf(t.s[i][e], w[e], b[e]));
      store_row<DT>(a.y, n * a.C, l, i, y);
    }
  }
}

template <int DT, int DTR, int W, int NV, bool FULL, int WIDE>
__global__ __launch_bounds__(WIDE ? WIDE : kBwdThreads) void residual_bwd_kernel(const RowArgs a) {
  __shared__ float sm[(WIDE ? WIDE : kBwdThreads) * kHold];
  int turn = 0;
  Place<W, NV, FULL> l(a);
  float sum[4][NV][W];   // of w, b, gamma, w2
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) sum[0][i][e] = sum[1][i][e] = sum[2][i][e] = sum[3][i][e] = 0.f;
  const float scale = a.alpha * (a.draw.threshold ? a.draw.scale : 1.f);
  const uint64_t seed = a.draw.threshold ? static_cast<uint64_t>(*a.draw.seed) : 0;
  Held<DT, W> x[NV], nx[NV], dy[NV], ndy[NV];
  Held<DTR, W> r[NV], nr[NV], ds[NV], nds[NV];
  auto fetch = [&](int64_t n, bool on) {
    load_row<DT, W, NV, FULL>(nx, a.x, n * a.C, l, on);
    load_row<DTR, W, NV, FULL>(nr, a.r, n * a.C, l, on);
    load_row<DT, W, NV, FULL>(ndy, a.dy, n * a.C, l, on && a.dy);
    load_row<DTR, W, NV, FULL>(nds, a.ds, n * a.C, l, on && a.ds);
  };
  fetch(l.row, l.row < a.N);
  for (int64_t n = l.row; n - l.row + l.first < a.N; n += a.slots) {   // (as often in the whole workgroup)
    l.at(n, a.N);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      r[i] = nr[i];
      dy[i] = ndy[i];
      ds[i] = nds[i];
    }
    if (l.again(n, a)) fetch(n + a.slots, n + a.slots < a.N);   // (zeros behind the last row: those lanes add nothing)
    Stream<DT, DTR, W, NV, FULL, WIDE> t;
    t.run(a, l, x, r, scale, seed, n, sm, turn);
    float d[NV][W];
    if (a.dy) {
      const float rstd = normalise<WIDE, FULL, W, NV>(t.s, l, a, sm, turn);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float w[W];
        load_weights(a.w, l, i, 1.f, w);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float g = dy[i][e];
          sum[0][i][e] = fmaf(g, t.s[i][e], sum[0][i][e]);
          sum[1][i][e] += g;
          d[i][e] = g * w[e];
        }
      }
      normalise_back<WIDE, FULL, W, NV>(d, t.s, rstd, l, a, sm, turn);
      each<W, NV>([&](int i, int e) { d[i][e] += ds[i][e]; });   // (zeros without one)
    } else {
      each<W, NV>([&](int i, int e) { d[i][e] = ds[i][e]; });
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (a.s) {
        Vec<DTR, W> dr;
#pragma unroll
        for (int e = 0; e < W; ++e) dr.set(e, d[i][e]);
        store_row<DTR>(a.s, n * a.C, l, i, dr);
      }
      float w2[W], c[W];
      load_weights(a.w2, l, i, 1.f, w2);
      load_weights(a.gamma, l, i, 1.f, c);
#pragma unroll
      for (int e = 0; e < W; ++e) {   // (what was dropped is 0 whatever it was)
        const bool on = t.keep[i] >> e & 1;
        const float g = on ? d[i][e] * scale : 0.f, v = on ? t.n2[i][e] : 0.f, dp = g * c[e];
        sum[2][i][e] = fmaf(g, v * w2[e], sum[2][i][e]);
        sum[3][i][e] = fmaf(dp, v, sum[3][i][e]);
        d[i][e] = dp * w2[e];
      }
    }
    if (a.y) {
      if (a.post) normalise_back<WIDE, FULL, W, NV>(d, t.n2, t.rstd2, l, a, sm, turn);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Vec<DT, W> dx;
#pragma unroll
        for (int e = 0; e < W; ++e) dx.set(e, d[i][e]);
        store_row<DT>(a.y, n * a.C, l, i, dx);
      }
    }
  }
  if (a.part) leave_sums<W, NV, FULL, 4>(a, l, sum, sm);
}

// Sums down R rows of [R][KINDS C]: 64 columns a workgroup, 16 wavefronts with every
// 16th row each.
struct Sums { float *to[4]; };
__global__ __launch_bounds__(1024) void row_cols_kernel(const float *__restrict__ src, int64_t R, int64_t cols, int C, Sums out) {
  __shared__ float sm[16][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float t = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = w; r < R; r += 16) t += src[r * cols + c];
  }
  sm[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < cols) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += sm[i][lane];
    float *to = out.to[c / C];
    if (to) to[c % C] = t;
  }
}

// ----------------------------------------------------------------- launches --
// How the rows are dealt, from the sizes and the widest vector the addresses allow.
struct RowPlan {
  int W, NV, S, threads;
  bool full, wide;
  int64_t slots, blocks, rows;   // rows: of sums
};
// Wavefronts: the forward's lane groups have a few rows each, the backward's about as many
// as run at once: their sums over rows go through memory once a workgroup.  Three
// workgroups a CU fit where a lane has 168 registers or less: all gated ones, and residual
// ones of 16-bit tensors in vectors of 8 (149 to 168); of fp32 (169 to 200) and some odd
// widths or vectors of 4 twice (171 to 183) two fit, and a third of the workgroups run behind the
// others.  Of 1,024 threads one fits.
constexpr int64_t kFwdWaves = 256 * 32, kBwdWaves[3] = {256 * 12, 256 * 8, 256 * 16};   // (256 CUs; workgroups of 256, 512, 1,024 threads)

RowPlan plan_of(int64_t N, int per, int G, int W, int dtype, bool bwd) {   // W 0: no vectors
  RowPlan p{};
  p.full = W != 0;
  if (!W) W = dtype == SSLA_F32 ? 4 : 8;
  p.W = W;
  const int nv = (per + W - 1) / W, most = kHold / W;
  p.S = 1;
  while (p.S < nv && (p.S < 64 || static_cast<int64_t>(p.S) * most < nv)) p.S *= 2;
  p.wide = p.S > 64;
  p.threads = std::max(bwd ? kBwdThreads : kFwdThreads, p.S);
  p.NV = 1;
  while (p.NV < most && (p.wide || !p.full || static_cast<int64_t>(p.S) * p.NV < nv)) p.NV *= 2;
  const int64_t groups = p.threads / p.S;   // lane groups of a workgroup
  const int64_t need = (N * G + groups - 1) / groups;
  p.blocks = std::min(need, (bwd ? kBwdWaves[p.threads / 512] : kFwdWaves) * 64 / p.threads);
  // a lane group keeps its group of channels, so all groups have as many (one row at a time at least)
  p.slots = std::min(N, std::max<int64_t>(1, p.blocks * groups / G));
  p.slots = (N + (N + p.slots - 1) / p.slots - 1) / ((N + p.slots - 1) / p.slots);   // all as many rows as the busiest, or one less
  p.blocks = (p.slots * G + groups - 1) / groups;
  p.rows = G <= groups ? p.blocks : p.slots;
  return p;
}

struct Tensor { const void *p; int64_t ld; int dtype; };
int widest(int per, int dtype, std::initializer_list<Tensor> tensors, std::initializer_list<const float *> weights) {
  for (const float *w : weights)
    if (!aligned(w, 16)) return 0;   // (NULL is aligned)
  for (int W = dtype == SSLA_F32 ? 4 : 8; W >= 4; W /= 2) {
    bool ok = per % W == 0;
    for (const Tensor &t : tensors) {
      const int bytes = std::min(16, W * (t.dtype == SSLA_F32 ? 4 : 2));
      ok = ok && aligned(t.p, bytes) && t.ld * (t.dtype == SSLA_F32 ? 4 : 2) % bytes == 0;
    }
    if (ok) return W;
  }
  return 0;
}

size_t sums_bytes(int64_t N, int per, int G, int kinds) {   // whatever type and vectors the call has
  int64_t most = 0;
  for (int dtype : {SSLA_F32, SSLA_BF16})
    for (int W : {0, 4, 8})
      if (!W || per % W == 0) most = std::max(most, plan_of(N, per, G, W, dtype, true).rows);
  return static_cast<size_t>(most) * kinds * per * G * sizeof(float);
}

int check_sizes(const char *what, int64_t N, int C, int G, int kind, int dtype, int r_dtype) {
  SSLA_CHECK_ARG(N >= 0 && C > 0 && G > 0 && C % G == 0 && (kind == SSLA_NORM_RMS || kind == SSLA_NORM_LAYER),
                 "%s: bad sizes N=%lld C=%d G=%d kind=%d", what, (long long)N, C, G, kind);
  const bool known = dtype == SSLA_F32 || dtype == SSLA_BF16 || dtype == SSLA_F16;
  if (!known || (r_dtype != dtype && r_dtype != SSLA_F32)) {
    set_error("%s: unsupported dtypes %d, %d", what, dtype, r_dtype);
    return SSLA_ERR_DTYPE;
  }
  if (C / G > kHold * kMostLanes || C > 1 << 24 || N > (1ll << 40) / C) {
    set_error("%s: at most %d channels in a group and 2^40 values", what, kHold * kMostLanes);
    return SSLA_ERR_UNSUPPORTED;
  }
  return SSLA_OK;
}
int check_ws(const char *what, const void *ws, size_t have, size_t need) {
  if (need == 0 || (ws && have >= need && aligned(ws, 16))) return SSLA_OK;
  set_error("%s: needs %zu bytes of workspace, got %zu", what, need, have);
  return SSLA_ERR_WORKSPACE;
}
int check_draw(const char *what, float p, const int64_t *seed, Draw &d) {
  SSLA_CHECK_ARG(p >= 0.f && p <= 1.f, "%s: p must lie in [0, 1], got %g", what, static_cast<double>(p));
  d.threshold = static_cast<uint32_t>(lrint(static_cast<double>(p) * 65536.0));
  SSLA_CHECK_ARG(d.threshold == 0 || seed, "%s: seed is NULL", what);
  d.seed = seed;
  d.scale = d.threshold < 65536 ? static_cast<float>(65536.0 / (65536.0 - d.threshold)) : 0.f;
  return SSLA_OK;
}

// Launches K<..., W, NV, FULL, WIDE> by the plan (WIDE: the threads whose registers a row of
// several wavefronts has to do with; 0: rows of one wavefront).
#define SSLA_ROWS_NV(K, W_, NV_, FULL_, ...)                                                                 \
  if (p.W == W_ && p.NV == NV_ && p.full == FULL_) {                                                         \
    if (p.wide) {                                                                                            \
      if constexpr (W_ * NV_ == kHold) {                                                                     \
        if (p.threads <= 512) hipLaunchKernelGGL((K<__VA_ARGS__, W_, NV_, FULL_, 512>), grid, block, 0, st, a); \
        else hipLaunchKernelGGL((K<__VA_ARGS__, W_, NV_, FULL_, kMostLanes>), grid, block, 0, st, a);        \
      }                                                                                                      \
    } else {                                                                                                 \
      hipLaunchKernelGGL((K<__VA_ARGS__, W_, NV_, FULL_, 0>), grid, block, 0, st, a);                        \
    }                                                                                                        \
  }
#define SSLA_ROWS(K, D, ...)                                  \
  do {                                                        \
    const dim3 grid(static_cast<unsigned>(p.blocks)), block(p.threads); \
    if constexpr (D != SSLA_F32) {                            \
      SSLA_ROWS_NV(K, 8, 1, true, __VA_ARGS__)                \
      SSLA_ROWS_NV(K, 8, 1, false, __VA_ARGS__)               \
    } else {                                                  \
      SSLA_ROWS_NV(K, 4, 2, false, __VA_ARGS__)               \
    }                                                         \
    SSLA_ROWS_NV(K, 4, 1, true, __VA_ARGS__)                  \
    SSLA_ROWS_NV(K, 4, 2, true, __VA_ARGS__)                  \
  } while (0)
#define SSLA_GATED(K)                                             \
  if (dtype == SSLA_F32) SSLA_ROWS(K, SSLA_F32, SSLA_F32);        \
  else if (dtype == SSLA_BF16) SSLA_ROWS(K, SSLA_BF16, SSLA_BF16); \
  else SSLA_ROWS(K, SSLA_F16, SSLA_F16)
#define SSLA_RESIDUAL(K)                                                                 \
  if (dtype == SSLA_F32) SSLA_ROWS(K, SSLA_F32, SSLA_F32, SSLA_F32);                     \
  else if (dtype == SSLA_BF16 && r_dtype == SSLA_F32) SSLA_ROWS(K, SSLA_BF16, SSLA_BF16, SSLA_F32); \
  else if (dtype == SSLA_BF16) SSLA_ROWS(K, SSLA_BF16, SSLA_BF16, SSLA_BF16);            \
  else if (r_dtype == SSLA_F32) SSLA_ROWS(K, SSLA_F16, SSLA_F16, SSLA_F32);              \
  else SSLA_ROWS(K, SSLA_F16, SSLA_F16, SSLA_F16)

void set_plan(RowArgs &a, const RowPlan &p) {
  a.S = p.S;
  a.slots = p.slots;
}
void add_columns(const float *part, int64_t rows, int kinds, int C, Sums out, hipStream_t st) {
  const int64_t cols = static_cast<int64_t>(kinds) * C;
  hipLaunchKernelGGL(row_cols_kernel, dim3(static_cast<unsigned>((cols + 63) / 64)), dim3(1024), 0, st, part, rows, cols, C, out);
}

}  // namespace
}  // namespace ssla

extern "C" int ssla_gated_norm_fwd(const void *x, int64_t ldx, const void *z, int64_t ldz, int64_t N, int C, int G, int kind,
                                   const float *weight, const float *bias, float eps, int act, void *y, int dtype,
                                   void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("gated_norm_fwd", N, C, G, kind, dtype, dtype)) return e;
  SSLA_CHECK_ARG((act == SSLA_ACT_SILU || act == SSLA_ACT_SIGMOID) && (N <= 1 || (ldx >= C && ldz >= C)),
                 "gated_norm_fwd: bad activation %d or row strides %lld, %lld", act, (long long)ldx, (long long)ldz);
  if (N == 0) return SSLA_OK;
  SSLA_CHECK_ARG(x && z && y, "gated_norm_fwd: null pointer");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  RowArgs a{};
  a.x = x; a.z = z; a.ldx = ldx; a.ldz = ldz; a.w = weight; a.b = bias; a.y = y;
  a.N = N; a.C = C; a.G = G; a.per = C / G; a.layer = kind == SSLA_NORM_LAYER; a.silu = act == SSLA_ACT_SILU; a.eps = eps;
  const RowPlan p = plan_of(N, C / G, G, widest(C / G, dtype, {{x, ldx, dtype}, {z, ldz, dtype}, {y, C, dtype}}, {weight, bias}), dtype, false);
  set_plan(a, p);
  SSLA_GATED(gated_fwd_kernel);
  return launch_status("gated_norm_fwd");
}

extern "C" size_t ssla_gated_norm_bwd_workspace_size(int64_t N, int C, int G) {
  return N > 0 && C > 0 && G > 0 && C % G == 0 ? ssla::sums_bytes(N, C / G, G, 2) : 0;
}

extern "C" int ssla_gated_norm_bwd(const void *dy, const void *x, int64_t ldx, const void *z, int64_t ldz, int64_t N, int C,
                                   int G, int kind, const float *weight, const float *bias, float eps, int act, void *dx,
                                   void *dz, float *dweight, float *dbias, int dtype, void *workspace,
                                   size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("gated_norm_bwd", N, C, G, kind, dtype, dtype)) return e;
  SSLA_CHECK_ARG((act == SSLA_ACT_SILU || act == SSLA_ACT_SIGMOID) && (N <= 1 || (ldx >= C && ldz >= C)),
                 "gated_norm_bwd: bad activation %d or row strides %lld, %lld", act, (long long)ldx, (long long)ldz);
  SSLA_CHECK_ARG(N == 0 || (dy && x && z), "gated_norm_bwd: null pointer");
  const bool sums = dweight || dbias;
  if (N == 0 && !sums) return SSLA_OK;
  if (const int e = check_ws("gated_norm_bwd", workspace, workspace_bytes,
                             sums ? ssla_gated_norm_bwd_workspace_size(N, C, G) : 0)) return e;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  RowPlan p{};
  if (N > 0) {
    RowArgs a{};
    a.x = x; a.z = z; a.dy = dy; a.ldx = ldx; a.ldz = ldz; a.w = weight; a.b = bias; a.y = dx; a.dz = dz;
    a.part = sums ? static_cast<float *>(workspace) : nullptr;
    a.N = N; a.C = C; a.G = G; a.per = C / G; a.layer = kind == SSLA_NORM_LAYER; a.silu = act == SSLA_ACT_SILU; a.eps = eps;
    p = plan_of(N, C / G, G, widest(C / G, dtype, {{x, ldx, dtype}, {z, ldz, dtype}, {dy, C, dtype}, {dx, C, dtype}, {dz, C, dtype}},
                                    {weight, bias}), dtype, true);
    set_plan(a, p);
    SSLA_GATED(gated_bwd_kernel);
  }
  if (sums) add_columns(static_cast<const float *>(workspace), p.rows, 2, C, {{dweight, dbias, nullptr, nullptr}}, st);
  return launch_status("gated_norm_bwd");
}

extern "C" int ssla_residual_norm_fwd(const void *x, const void *residual, int64_t N, int C, int kind, const float *weight,
                                      const float *bias, float eps, float alpha, const float *gamma, int post,
                                      const float *post_weight, float p, const int64_t *seed, uint32_t subsequence, void *y,
                                      void *sum, int dtype, int r_dtype, void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("residual_norm_fwd", N, C, 1, kind, dtype, r_dtype)) return e;
  RowArgs a{};
  if (const int e = check_draw("residual_norm_fwd", p, seed, a.draw)) return e;
  SSLA_CHECK_ARG(post || !post_weight, "residual_norm_fwd: a weight of a norm that is not asked for");
  if (N == 0) return SSLA_OK;
  SSLA_CHECK_ARG(x && residual && y && sum, "residual_norm_fwd: null pointer");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  a.draw.subsequence = subsequence;
  a.x = x; a.r = residual; a.w = weight; a.b = bias; a.w2 = post_weight; a.gamma = gamma; a.y = y; a.s = sum;
  a.N = N; a.C = a.per = C; a.G = 1; a.layer = kind == SSLA_NORM_LAYER; a.post = post != 0; a.eps = eps; a.alpha = alpha;
  const RowPlan pl = plan_of(N, C, 1, widest(C, dtype, {{x, C, dtype}, {residual, C, r_dtype}, {y, C, dtype}, {sum, C, r_dtype}},
                                             {weight, bias, post_weight, gamma}), dtype, false);
  {
    const RowPlan &p = pl;
    set_plan(a, p);
    SSLA_RESIDUAL(residual_fwd_kernel);
  }
  return launch_status("residual_norm_fwd");
}

extern "C" size_t ssla_residual_norm_bwd_workspace_size(int64_t N, int C) {
  return N > 0 && C > 0 ? ssla::sums_bytes(N, C, 1, 4) : 0;
}

extern "C" int ssla_residual_norm_bwd(const void *dy, const void *dsum, const void *x, const void *residual, int64_t N, int C,
                                      int kind, const float *weight, float eps, float alpha, const float *gamma, int post,
                                      const float *post_weight, float p, const int64_t *seed, uint32_t subsequence, void *dx,
                                      void *dresidual, float *dweight, float *dbias, float *dgamma, float *dpost_weight,
                                      int dtype, int r_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("residual_norm_bwd", N, C, 1, kind, dtype, r_dtype)) return e;
  RowArgs a{};
  if (const int e = check_draw("residual_norm_bwd", p, seed, a.draw)) return e;
  SSLA_CHECK_ARG(post || (!post_weight && !dpost_weight), "residual_norm_bwd: a weight of a norm that is not asked for");
  SSLA_CHECK_ARG(N == 0 || ((dy || dsum) && x && residual), "residual_norm_bwd: null pointer");
  const bool sums = dweight || dbias || dgamma || dpost_weight;
  if (N == 0 && !sums) return SSLA_OK;
  if (const int e = check_ws("residual_norm_bwd", workspace, workspace_bytes,
                             sums ? ssla_residual_norm_bwd_workspace_size(N, C) : 0)) return e;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  int64_t rows = 0;
  if (N > 0) {
    a.draw.subsequence = subsequence;
    a.x = x; a.r = residual; a.dy = dy; a.ds = dsum; a.w = weight; a.w2 = post_weight; a.gamma = gamma; a.y = dx; a.s = dresidual;
    a.part = sums ? static_cast<float *>(workspace) : nullptr;
    a.N = N; a.C = a.per = C; a.G = 1; a.layer = kind == SSLA_NORM_LAYER; a.post = post != 0; a.eps = eps; a.alpha = alpha;
    const RowPlan p = plan_of(N, C, 1, widest(C, dtype, {{x, C, dtype}, {residual, C, r_dtype}, {dy, C, dtype}, {dsum, C, r_dtype},
                                                         {dx, C, dtype}, {dresidual, C, r_dtype}}, {weight, post_weight, gamma}), dtype, true);
    rows = p.rows;
    set_plan(a, p);
    SSLA_RESIDUAL(residual_bwd_kernel);
  }
  if (sums) add_columns(static_cast<const float *>(workspace), rows, 4, C, {{dweight, dbias, dgamma, dpost_weight}}, st);
  return launch_status("residual_norm_bwd");
}

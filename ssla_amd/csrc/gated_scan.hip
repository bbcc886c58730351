// Gated linear recurrence over packed sequences, per channel:
//   h_t = a_t h_{t-1} + u_t,  a_t = g_t, e^(g_t) or sigmoid(g_t),  o_t = q_t h_t (or h_t)
// with its backward, from an initial state to the final one.  With e_t the
// gradient of h_t:
//   e_t = q_t do_t + a_{t+1} e_{t+1} (dht_n behind a sequence's last row)
//   du_t = e_t,  da_t = e_t h_{t-1},  dq_t = do_t h_t,  dh0_n = a_first e_first
//
// Bound by memory: the forward moves u, g, q and o, the backward u, g, q, do and the
// three gradients, each once.  The packed rows are one time axis, cut into tiles of
// rows by channels whatever the sequences; a row that begins a sequence takes its
// state from h0 and nothing from the rows before.
//
// A lane holds R rows of W neighbouring channels in registers.  Over its rows the
// recurrence is a map h -> A h + U; the maps of a tile's row groups are joined in
// LDS, one thread a channel.  A tile publishes its map and finds its entering state
// from the tiles before: the nearest one whose leaving state is known, and the maps
// from there on, applied in their order, so the result does not depend on which
// were known.  A tile with a sequence's start publishes its leaving state at once.
// Tiles are handed out in order by a ticket and publish before they wait, so every
// tile waited for has started and the wait ends.  A word says by itself whether it
// is there (an all-ones word is not): no fences.
// The backward does the same from the last tile on; the states it needs come from
// the forward, which leaves one every 64 rows, and are computed again in between.
#include "vec.h"

namespace ssla {
namespace {

constexpr int kValue = SSLA_GATE_VALUE, kLog = SSLA_GATE_LOG, kSigmoid = SSLA_GATE_SIGMOID;

// e^x with the product x log2(e) in two parts: off by 4 2^-24 at any x whose e^x is a
// normal number (e^x of one product by up to 100 2^-24).
__device__ __forceinline__ float exp_of(float x) {
  const float y = x * kLog2e;
  const float e = fast_exp2(y);
  return fabsf(y) < 126.f ? fmaf(e * 0.6931472f, fmaf(x, 1.925963e-8f, fmaf(x, kLog2e, -y)), e) : e;   // (past that 0, infinite or near it)
}

// The gate and its derivative.  sigmoid from e^-|g|: both it and 1 - it keep their
// relative precision on either side.
struct Gate { float a, slope; };
__device__ __forceinline__ Gate gate_of(int kind, float g) {
  if (kind == kValue) return {g, 1.f};
  if (kind == kLog) {
    const float a = exp_of(g);
    return {a, a};
  }
  const float t = exp_of(-fabsf(g)), r = __builtin_amdgcn_rcpf(1.f + t), s = t * r;
  return {g >= 0.f ? r : s, r * s};
}

constexpr int R = 8;             // rows of a lane
constexpr int kBlock = 256;
constexpr int kKeepRows = 64;    // rows between the states left for the backward
constexpr int kMostValues = kBlock * 8;   // (row group, channel) pairs of a tile

struct ScanArgs {
  const void *u, *g, *q, *dout;   // q may be NULL
  int64_t ldu, ldg, ldq;          // elements from row to row
  const int64_t *cu;
  int n_seq;
  int64_t T;
  int C, gate;
  const float *h0, *dht;          // may be NULL
  void *o, *du, *dg, *dq;
  float *ht, *dh0, *keep;         // may be NULL (keep: not in the backward)
  int CT, RG, cblocks;            // lanes of a row, row groups, channel blocks
  int64_t tiles;
  uint32_t *ticket;               // NULL: one tile of rows
  uint64_t *maps;                 // [tiles][cblocks CT W]: A and U
  uint32_t *states;               // the state that leaves a tile
};

// ------------------------------------------------------- tiles and sequences --
// What a tile's rows are: mark[row] the sequence that begins there, kInside, or
// kOutside of all sequences; fin[row] the sequence that ends with the row, or -1.
constexpr int kInside = -1, kOutside = -2;

// Fills mark and fin of the rows r0 .. r0 + rows; false where all rows are kInside
// and none ends a sequence.  Two rounds of 256 probes for up to 65,536 sequences.
__device__ bool mark_rows(const ScanArgs &a, int64_t r0, int rows, int *mark, int *fin) {
  const int tid = threadIdx.x;
  for (int i = tid; i < rows; i += kBlock) {
    mark[i] = kInside;
    fin[i] = -1;
  }
  if (a.n_seq == 0) {
    __syncthreads();
    for (int i = tid; i < rows; i += kBlock) mark[i] = kOutside;
    __syncthreads();
    return true;
  }
  int lo = 0, hi = a.n_seq;   // the last sequence that begins at r0 or before is in [lo, hi)
  while (hi - lo > kBlock) {  // (the same for all threads)
    const int step = (hi - lo + kBlock - 1) / kBlock;
    const int64_t i = lo + static_cast<int64_t>(tid) * step;
    const int cnt = __syncthreads_count(i < hi && a.cu[i] <= r0);
    lo += max(cnt - 1, 0) * step;
    hi = min(hi, lo + step);
  }
  const int64_t first = min(max(a.cu[0], (int64_t)0), a.T), last = min(max(a.cu[a.n_seq], first), a.T);
  __syncthreads();
  bool some = false;
  for (int n0 = lo; n0 < a.n_seq; n0 += kBlock) {
    const int n = n0 + tid;
    bool past = true;
    if (n < a.n_seq) {
      const int64_t b = min(max(a.cu[n], (int64_t)0), a.T), e = min(max(a.cu[n + 1], b), a.T);
      past = b >= r0 + rows;
      if (e > b) {
        if (b >= r0 && b < r0 + rows) {
          mark[b - r0] = n;
          some = true;
        }
        if (e > r0 && e <= r0 + rows) {
          fin[e - 1 - r0] = n;
          some = true;
        }
      }
    }
    if (__syncthreads_or(past)) break;
  }
  for (int i = tid; i < rows; i += kBlock)
    if (r0 + i < first || r0 + i >= last) {
      mark[i] = kOutside;
      some = true;
    }
  return __syncthreads_or(some);
}

// --------------------------------------------------- states between the tiles --
constexpr uint32_t kNone32 = 0xffffffffu;
constexpr uint64_t kNone64 = ~0ull;

// A value's bits as a word that can be told from one that is not there.
__device__ __forceinline__ uint32_t word_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b == kNone32 ? 0x7fc00000u : b;
}
template <typename T>
__device__ __forceinline__ T look(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ void show(T *p, T x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// (a factor that overflowed must not meet a state of zero)
__device__ __forceinline__ float apply(float A, float x, float U) { return x == 0.f ? U : fmaf(A, x, U); }
__device__ __forceinline__ float apply(uint64_t m, float x) {
  return apply(__uint_as_float(static_cast<uint32_t>(m)), x, __uint_as_float(static_cast<uint32_t>(m >> 32)));
}

// The state that enters tile k > 0 in column c of `wide`.
__device__ float entering_state(const ScanArgs &a, int64_t k, int64_t c, int64_t wide) {
  constexpr int NW = 8;   // tiles of a round trip
  const uint64_t *maps = a.maps + c;
  const uint32_t *states = a.states + c;
  int64_t near = k - 1;
  for (;;) {
    uint64_t m[NW];
    uint32_t s[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const int64_t at = max(near - i, (int64_t)0) * wide;
      s[i] = look(states + at);
      m[i] = look(maps + at);
    }
    int found = -1, ready = NW;
#pragma unroll
    for (int i = NW - 1; i >= 0; --i) {
      if (s[i] != kNone32) found = i;
      else if (m[i] == kNone64) {
        ready = i;
        found = -1;
      }
    }
    // (found: the nearest known state, with every map this side of it)
    if (found >= 0) {
      float x = 0.f;
#pragma unroll
      for (int i = NW - 1; i >= 0; --i) {
        if (i == found) x = __uint_as_float(s[i]);
        else if (i < found) x = apply(m[i], x);
      }
      // the maps of the rounds before this one
      for (int64_t at = near + 1; at < k; at += NW) {
#pragma unroll
        for (int i = 0; i < NW; ++i) m[i] = look(maps + min(at + i, k - 1) * wide);
#pragma unroll
        for (int i = 0; i < NW; ++i)
          if (at + i < k) x = apply(m[i], x);
      }
      return x;
    }
    if (ready == NW) near -= NW;
    else __builtin_amdgcn_s_sleep(1);
  }
}

__global__ __launch_bounds__(256) void scan_clear_kernel(uint32_t *ticket, uint64_t *words, int64_t n) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    words[i] = kNone64;
}

// Which tile and channel block a workgroup has.
__device__ __forceinline__ int64_t take_tile(const ScanArgs &a, uint32_t *slot) {
  if (!a.ticket) return blockIdx.x;
  if (threadIdx.x == 0) *slot = atomicAdd(a.ticket, 1u);
  __syncthreads();
  return *slot;
}

// Joins the maps of the RG row groups of channel c (LDS, `cw` channels a row group)
// from the first or the last on; cut[k]: the state leaving group k is U, whatever enters.
struct Joined { float A, U; bool cut; };
template <bool BACK>
__device__ __forceinline__ Joined join_groups(const float *A, const float *U, const int *cut, int RG, int cw, int c) {
  Joined j{1.f, 0.f, false};
#pragma unroll 8
  for (int i = 0; i < RG; ++i) {
    const int k = BACK ? RG - 1 - i : i;
    const float x = A[k * cw + c], y = U[k * cw + c];
    const bool r = cut[k];
    j.U = r ? y : apply(x, j.U, y);
    j.A *= x;
    j.cut |= r;
  }
  return j;
}
// Puts each group's entering state in U.
template <bool BACK>
__device__ __forceinline__ void enter_groups(const float *A, float *U, const int *cut, int RG, int cw, int c, float x) {
#pragma unroll 8
  for (int i = 0; i < RG; ++i) {
    const int k = BACK ? RG - 1 - i : i;
    const float f = A[k * cw + c], y = U[k * cw + c];
    U[k * cw + c] = x;
    x = cut[k] ? y : apply(f, x, y);
  }
}
// A channel's part between its maps: publishes, finds the entering state (`closed`:
// the tile's first row takes none) and fills U.
template <bool BACK>
__device__ __forceinline__ void enter_tile(const ScanArgs &a, int64_t k, int64_t col, int64_t wide, const float *A, float *U,
                                           const int *cut, bool closed, int cw, int c) {
  float x = 0.f;
  if (a.ticket) {
    const Joined j = join_groups<BACK>(A, U, cut, a.RG, cw, c);
    const int64_t at = k * wide + col;
    const bool known = k == 0 || j.cut;
    if (known) show(a.states + at, word_of(j.U));
    else show(a.maps + at, static_cast<uint64_t>(word_of(j.A)) | static_cast<uint64_t>(__float_as_uint(j.U)) << 32);
    asm volatile("" ::: "memory");   // (published before anything is waited for)
    if (k > 0 && !closed) x = entering_state(a, k, col, wide);
    if (!known) show(a.states + at, word_of(apply(j.A, x, j.U)));
  }
  enter_groups<BACK>(A, U, cut, a.RG, cw, c, x);
}

template <int DT, int W>
__device__ __forceinline__ void load_rows(Vec<DT, W> (&x)[R], const void *p, int64_t ld, int64_t row0, int64_t T, int c) {
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (row0 + i < T) x[i] = load_vec<DT, W>(p, (row0 + i) * ld + c);
}

// ------------------------------------------------------------------ forward --
template <int DT, int DTG, int W>
__global__ __launch_bounds__(kBlock) void scan_fwd_kernel(const ScanArgs a) {
  __shared__ float sA[kMostValues], sU[kMostValues];
  __shared__ int mark[kBlock * R], fin[kBlock * R], cut[kBlock];
  __shared__ uint32_t slot;
  const int64_t id = take_tile(a, &slot);
  const int64_t k = id / a.cblocks;
  const int cb = static_cast<int>(id - k * a.cblocks), cw = a.CT * W, tid = threadIdx.x;
  const int rg = tid / a.CT, cl = tid - rg * a.CT, rows = a.RG * R;
  const int64_t r0 = k * rows, row0 = r0 + rg * R;
  const int c = (cb * a.CT + cl) * W;
  const bool on = rg < a.RG && c < a.C;
  Vec<DT, W> u[R], q[R];
  Vec<DTG, W> g[R];
  if (on) {
    load_rows<DT, W>(u, a.u, a.ldu, row0, a.T, c);
    load_rows<DTG, W>(g, a.g, a.ldg, row0, a.T, c);
    if (a.q) load_rows<DT, W>(q, a.q, a.ldq, row0, a.T, c);
  }
  const bool some = mark_rows(a, r0, rows, mark, fin);
  float f[R][W];
  if (on) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) f[i][e] = gate_of(a.gate, g[i][e]).a;
    float A[W], U[W];
    bool reset = false;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      A[e] = 1.f;
      U[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int m = some ? mark[rg * R + i] : kInside;
      if (m == kInside) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          U[e] = fmaf(f[i][e], U[e], u[i][e]);
          A[e] *= f[i][e];
        }
      } else {
        reset = true;
#pragma unroll
        for (int e = 0; e < W; ++e)
          U[e] = m < 0 ? 0.f : fmaf(f[i][e], a.h0 ? a.h0[static_cast<int64_t>(m) * a.C + c + e] : 0.f, u[i][e]);
      }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      sA[rg * cw + cl * W + e] = A[e];
      sU[rg * cw + cl * W + e] = U[e];
    }
    if (cl == 0) cut[rg] = reset;
  }
  __syncthreads();
  const int64_t wide = static_cast<int64_t>(a.cblocks) * cw;
  if (tid < cw && cb * cw + tid < a.C)
    enter_tile<false>(a, k, static_cast<int64_t>(cb) * cw + tid, wide, sA, sU, cut, some && mark[0] != kInside, cw, tid);
  __syncthreads();
  if (on) {
    float h[W];
#pragma unroll
    for (int e = 0; e < W; ++e) h[e] = sU[rg * cw + cl * W + e];
    if (a.keep && row0 % kKeepRows == 0 && row0 < a.T)
#pragma unroll
      for (int e = 0; e < W; ++e) a.keep[row0 / kKeepRows * a.C + c + e] = h[e];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (row0 + i >= a.T) break;
      const int m = some ? mark[rg * R + i] : kInside;
      Vec<DT, W> o;
      if (m == kOutside) {
#pragma unroll
        for (int e = 0; e < W; ++e) o.set(e, 0.f);
      } else {
        if (m >= 0)
#pragma unroll
          for (int e = 0; e < W; ++e) h[e] = a.h0 ? a.h0[static_cast<int64_t>(m) * a.C + c + e] : 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          h[e] = fmaf(f[i][e], h[e], u[i][e]);
          o.set(e, a.q ? h[e] * q[i][e] : h[e]);
        }
        const int n = some ? fin[rg * R + i] : -1;
        if (a.ht && n >= 0)
#pragma unroll
          for (int e = 0; e < W; ++e) a.ht[static_cast<int64_t>(n) * a.C + c + e] = h[e];
      }
      store_vec<DT, W>(a.o, (row0 + i) * a.C + c, o);
    }
  }
  if (a.ht)   // empty sequences, dealt over the tiles
    for (int64_t n = k; n < a.n_seq; n += a.tiles) {
      const int64_t b = min(max(a.cu[n], (int64_t)0), a.T);
      if (a.cu[n + 1] <= b && tid < cw && cb * cw + tid < a.C)
        a.ht[n * a.C + cb * cw + tid] = a.h0 ? a.h0[n * a.C + cb * cw + tid] : 0.f;
    }
}

// ----------------------------------------------------------------- backward --
template <int DT, int DTG, int W>
__global__ __launch_bounds__(kBlock) void scan_bwd_kernel(const ScanArgs a) {
  __shared__ float sA[kMostValues], sU[kMostValues], sE[kMostValues];
  __shared__ int mark[kBlock * R], fin[kBlock * R], cut[kBlock];
  __shared__ uint32_t slot;
  const int64_t id = take_tile(a, &slot);
  const int64_t back = id / a.cblocks, k = a.tiles - 1 - back;
  const int cb = static_cast<int>(id - back * a.cblocks), cw = a.CT * W, tid = threadIdx.x;
  const int rg = tid / a.CT, cl = tid - rg * a.CT, rows = a.RG * R;
  const int64_t r0 = k * rows, row0 = r0 + rg * R;
  const int c = (cb * a.CT + cl) * W;
  const bool on = rg < a.RG && c < a.C;
  Vec<DT, W> u[R], q[R], d[R];
  Vec<DTG, W> g[R];
  if (on) {
    load_rows<DT, W>(u, a.u, a.ldu, row0, a.T, c);
    load_rows<DTG, W>(g, a.g, a.ldg, row0, a.T, c);
    load_rows<DT, W>(d, a.dout, a.C, row0, a.T, c);
    if (a.q) load_rows<DT, W>(q, a.q, a.ldq, row0, a.T, c);
  }
  const bool some = mark_rows(a, r0, rows, mark, fin);
  Gate f[R][W];
  auto state0 = [&](int m, int e) __attribute__((always_inline)) {
    return a.h0 ? a.h0[static_cast<int64_t>(m) * a.C + c + e] : 0.f;
  };
  auto grad_of = [&](int i, int e) __attribute__((always_inline)) { return a.q ? d[i][e] * q[i][e] : d[i][e]; };
  if (on) {
    float A[W], U[W], E[W];
    bool reset = false;
#pragma unroll
    for (int e = 0; e < W; ++e) {
      A[e] = 1.f;
      U[e] = E[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int m = some ? mark[rg * R + i] : kInside;
      reset |= m != kInside;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        f[i][e] = gate_of(a.gate, g[i][e]);
        U[e] = m == kOutside ? 0.f : fmaf(f[i][e].a, m >= 0 ? state0(m, e) : U[e], u[i][e]);
        A[e] *= f[i][e].a;
      }
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const int m = some ? mark[rg * R + i] : kInside, n = some ? fin[rg * R + i] : -1;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (n >= 0) E[e] = a.dht ? a.dht[static_cast<int64_t>(n) * a.C + c + e] : 0.f;
        E[e] = m == kInside ? f[i][e].a * (grad_of(i, e) + E[e]) : 0.f;   // (nothing goes past a beginning)
      }
      // a sequence's end takes nothing from the rows behind it
      reset |= n >= 0;
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      sA[rg * cw + cl * W + e] = A[e];
      sU[rg * cw + cl * W + e] = U[e];
      sE[rg * cw + cl * W + e] = E[e];
    }
    if (cl == 0) cut[rg] = reset;
  }
  __syncthreads();
  const int64_t wide = static_cast<int64_t>(a.cblocks) * cw;
  // one half of the threads takes the states forward, the other the gradients back
  const int half = tid < kBlock / 2 ? tid : tid - kBlock / 2;
  if (half < cw && cb * cw + half < a.C) {
    if (tid < kBlock / 2)
      enter_groups<false>(sA, sU, cut, a.RG, cw, half, r0 < a.T ? a.keep[r0 / kKeepRows * a.C + cb * cw + half] : 0.f);
    else
      enter_tile<true>(a, back, static_cast<int64_t>(cb) * cw + half, wide, sA, sE, cut,
                       some && (mark[rows - 1] == kOutside || fin[rows - 1] >= 0), cw, half);
  }
  __syncthreads();
  if (on) {
    float h[W], x[W], before[R][W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      h[e] = sU[rg * cw + cl * W + e];
      x[e] = sE[rg * cw + cl * W + e];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int m = some ? mark[rg * R + i] : kInside;
      Vec<DT, W> dq;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (m >= 0) h[e] = state0(m, e);
        before[i][e] = h[e];
        h[e] = fmaf(f[i][e].a, h[e], u[i][e]);
        dq.set(e, m == kOutside ? 0.f : d[i][e] * h[e]);
      }
      if (a.q && row0 + i < a.T) store_vec<DT, W>(a.dq, (row0 + i) * a.C + c, dq);
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const int m = some ? mark[rg * R + i] : kInside, n = some ? fin[rg * R + i] : -1;
      Vec<DT, W> du;
      Vec<DTG, W> dg;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (n >= 0) x[e] = a.dht ? a.dht[static_cast<int64_t>(n) * a.C + c + e] : 0.f;
        const float s = grad_of(i, e) + x[e];
        du.set(e, m == kOutside ? 0.f : s);
        dg.set(e, m == kOutside ? 0.f : s * before[i][e] * f[i][e].slope);
        x[e] = f[i][e].a * s;
        if (m >= 0 && a.dh0) a.dh0[static_cast<int64_t>(m) * a.C + c + e] = x[e];
      }
      if (row0 + i < a.T) {
        store_vec<DT, W>(a.du, (row0 + i) * a.C + c, du);
        store_vec<DTG, W>(a.dg, (row0 + i) * a.C + c, dg);
      }
    }
  }
  if (a.dh0)   // empty sequences
    for (int64_t n = k; n < a.n_seq; n += a.tiles) {
      const int64_t b = min(max(a.cu[n], (int64_t)0), a.T);
      if (a.cu[n + 1] <= b && tid < cw && cb * cw + tid < a.C)
        a.dh0[n * a.C + cb * cw + tid] = a.dht ? a.dht[n * a.C + cb * cw + tid] : 0.f;
    }
}

// --------------------------------------------------------- single tokens --
struct StepArgs {
  const int32_t *at;
  const void *u, *g, *q;
  int64_t ldu, ldg, ldq;
  float *state;
  void *o;
  int32_t *status;
  int n, rows, C, gate;
};
template <int DT, int DTG>
__global__ __launch_bounds__(256) void scan_step_kernel(const StepArgs a) {
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (x >= static_cast<int64_t>(a.n) * a.C) return;
  const int64_t i = x / a.C;
  const int c = static_cast<int>(x % a.C), row = a.at[i];
  if (row < 0 || row >= a.rows || (i > 0 && a.at[i - 1] >= row)) {
    Elem<DT>::store(a.o, x, 0.f);
    if (a.status) __hip_atomic_store(a.status, SSLA_ERR_ARG, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return;
  }
  float &s = a.state[static_cast<int64_t>(row) * a.C + c];
  s = fmaf(gate_of(a.gate, Elem<DTG>::load(a.g, i * a.ldg + c)).a, s, Elem<DT>::load(a.u, i * a.ldu + c));
  Elem<DT>::store(a.o, x, a.q ? s * Elem<DT>::load(a.q, i * a.ldq + c) : s);
}

// --------------------------------------------------------------- launches --
int check_sizes(const char *what, int n_seq, int64_t T, int C, int gate, int dtype, int g_dtype, int64_t ldu, int64_t ldg,
                int64_t ldq) {
  SSLA_CHECK_ARG(n_seq >= 0 && T >= 0 && C > 0 && gate >= kValue && gate <= kSigmoid,
                 "%s: bad sizes n_seq=%d T=%lld C=%d gate=%d", what, n_seq, (long long)T, C, gate);
  SSLA_CHECK_ARG(T <= 1 || (ldu >= C && ldg >= C && ldq >= C), "%s: rows of %d channels overlap at strides %lld, %lld, %lld",
                 what, C, (long long)ldu, (long long)ldg, (long long)ldq);
  const bool known = dtype == SSLA_F32 || dtype == SSLA_BF16 || dtype == SSLA_F16;
  if (!known || (g_dtype != dtype && g_dtype != SSLA_F32)) {
    set_error("%s: unsupported dtypes %d, gates %d", what, dtype, g_dtype);
    return SSLA_ERR_DTYPE;
  }
  if (T > (1ll << 40) / C || static_cast<int64_t>(n_seq) * C > (1ll << 38)) {
    set_error("%s: too many values", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  return SSLA_OK;
}

#define SSLA_SCAN_TYPES(CALL)                                                                       \
  do {                                                                                              \
    if (dtype == SSLA_F32) { CALL(SSLA_F32, SSLA_F32); }                                            \
    else if (dtype == SSLA_BF16) { if (g_dtype == SSLA_F32) { CALL(SSLA_BF16, SSLA_F32); } else { CALL(SSLA_BF16, SSLA_BF16); } } \
    else { if (g_dtype == SSLA_F32) { CALL(SSLA_F16, SSLA_F32); } else { CALL(SSLA_F16, SSLA_F16); } } \
  } while (0)

// How the rows and channels are cut for vectors of W values: up to kLanes lanes a
// row, as many row groups as a workgroup has room for (a power of two, so that a
// tile is a multiple of kKeepRows rows).
constexpr int kLanes = 16;
struct ScanPlan {
  int CT, RG, cblocks;
  int64_t tiles;
};
ScanPlan plan_of(int64_t T, int C, int W, int lanes) {
  ScanPlan p;
  const int cv = C / W;
  p.CT = (cv + (cv + lanes - 1) / lanes - 1) / ((cv + lanes - 1) / lanes);
  p.cblocks = (cv + p.CT - 1) / p.CT;
  p.RG = kKeepRows / R;
  while (2 * p.RG * p.CT <= kBlock) p.RG *= 2;
  p.tiles = std::max<int64_t>(1, (T + p.RG * R - 1) / (p.RG * R));
  return p;
}
constexpr size_t kHead = 256;   // the ticket's line
int64_t word_count(const ScanPlan &p, int W) {   // 64-bit words of maps and states
  return (p.tiles * p.cblocks * p.CT * W * 3 + 1) / 2;
}
size_t ws_bytes(int64_t T, int C) {   // whatever vectors the addresses allow
  int64_t most = 0;
  for (int W = 1; W <= 8; W *= 2)
    if (W != 2 && C % W == 0) {
      const ScanPlan p = plan_of(T, C, W, kLanes);
      if (p.tiles > 1) most = std::max(most, word_count(p, W));
    }
  return most ? kHead + static_cast<size_t>(most) * 8 : 0;
}

int size_of(int dtype) { return dtype == SSLA_F32 ? 4 : 2; }

// The widest vector that all rows of the tensors allow.
struct Rows { const void *p; int64_t ld; int dtype; };
int widest(int C, int most, std::initializer_list<Rows> all) {
  for (int W = most; W >= 4; W /= 2) {
    bool ok = C % W == 0;
    for (const Rows &r : all) {
      const int bytes = std::min(16, W * size_of(r.dtype));
      ok = ok && aligned(r.p, bytes) && r.ld * size_of(r.dtype) % bytes == 0;
    }
    if (ok) return W;
  }
  return 1;
}

// Sets the plan, clears the words and launches `kernel`.
template <typename Kernel>
int launch_scan(const char *what, ScanArgs &a, int W, Kernel kernel, void *workspace, size_t workspace_bytes, hipStream_t st) {
  const ScanPlan p = plan_of(a.T, a.C, W, kLanes);
  const size_t need = p.tiles > 1 ? kHead + static_cast<size_t>(word_count(p, W)) * 8 : 0;
  if (need && !(workspace && workspace_bytes >= need && aligned(workspace, 16))) {
    set_error("%s: needs %zu bytes of workspace, got %zu", what, ws_bytes(a.T, a.C), workspace_bytes);
    return SSLA_ERR_WORKSPACE;
  }
  if (p.tiles * p.cblocks > 0x7fffffff) {
    set_error("%s: too many workgroups", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  a.CT = p.CT; a.RG = p.RG; a.cblocks = p.cblocks; a.tiles = p.tiles;
  if (need) {
    const int64_t n = word_count(p, W);
    a.ticket = static_cast<uint32_t *>(workspace);
    a.maps = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + kHead);
    a.states = reinterpret_cast<uint32_t *>(a.maps + p.tiles * p.cblocks * p.CT * W);
    hipLaunchKernelGGL(scan_clear_kernel, dim3(static_cast<unsigned>(std::min<int64_t>((n + 1023) / 1024, 2048))), dim3(256), 0,
                       st, a.ticket, a.maps, n);
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.tiles * p.cblocks)), dim3(kBlock), 0, st, a);
  return SSLA_OK;
}

}  // namespace
}  // namespace ssla

extern "C" size_t ssla_gated_scan_workspace_size(int64_t T, int C) { return T > 0 && C > 0 ? ssla::ws_bytes(T, C) : 0; }

extern "C" size_t ssla_gated_scan_keep_size(int64_t T, int C) {
  return T > 0 && C > 0 ? static_cast<size_t>((T + ssla::kKeepRows - 1) / ssla::kKeepRows) * C * sizeof(float) : 0;
}

extern "C" int ssla_gated_scan_fwd(const void *u, int64_t ldu, const void *g, int64_t ldg, const void *q, int64_t ldq,
                                   const int64_t *cu_seqlens, int n_seq, int64_t T, int C, int gate, const float *h0,
                                   void *o, float *ht, void *keep, int dtype, int g_dtype, void *workspace,
                                   size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("gated_scan_fwd", n_seq, T, C, gate, dtype, g_dtype, ldu, ldg, q ? ldq : ldu)) return e;
  SSLA_CHECK_ARG(n_seq == 0 || cu_seqlens, "gated_scan_fwd: cu_seqlens is NULL");
  SSLA_CHECK_ARG(T == 0 || (u && g && o), "gated_scan_fwd: null pointer");
  if (T == 0 && n_seq == 0) return SSLA_OK;
  ScanArgs a{};
  a.u = u; a.g = g; a.q = q; a.ldu = ldu; a.ldg = ldg; a.ldq = ldq;
  a.cu = cu_seqlens; a.n_seq = n_seq; a.T = T; a.C = C; a.gate = gate;
  a.h0 = h0; a.o = o; a.ht = ht; a.keep = static_cast<float *>(keep);
  const int W = widest(C, dtype == SSLA_F32 ? 4 : 8, {{u, ldu, dtype}, {g, ldg, g_dtype}, {q, q ? ldq : 0, dtype}, {o, C, dtype}});
  int status = SSLA_OK;
#define SSLA_LAUNCH(D, G, W_) \
  status = launch_scan("gated_scan_fwd", a, W_, scan_fwd_kernel<D, G, W_>, workspace, workspace_bytes, static_cast<hipStream_t>(stream))
#define SSLA_CALL(D, G)                                              \
  if (W == 8) { if constexpr (D != SSLA_F32) SSLA_LAUNCH(D, G, 8); } \
  else if (W == 4) SSLA_LAUNCH(D, G, 4);                             \
  else SSLA_LAUNCH(D, G, 1)
  SSLA_SCAN_TYPES(SSLA_CALL);
#undef SSLA_CALL
#undef SSLA_LAUNCH
  return status == SSLA_OK ? launch_status("gated_scan_fwd") : status;
}

extern "C" int ssla_gated_scan_bwd(const void *u, int64_t ldu, const void *g, int64_t ldg, const void *q, int64_t ldq,
                                   const int64_t *cu_seqlens, int n_seq, int64_t T, int C, int gate, const float *h0,
                                   const void *keep, const void *dout, const float *dht, void *du, void *dg, void *dq,
                                   float *dh0, int dtype, int g_dtype, void *workspace, size_t workspace_bytes,
                                   void *stream) {
  using namespace ssla;
  clear_error();
  if (const int e = check_sizes("gated_scan_bwd", n_seq, T, C, gate, dtype, g_dtype, ldu, ldg, q ? ldq : ldu)) return e;
  SSLA_CHECK_ARG(n_seq == 0 || cu_seqlens, "gated_scan_bwd: cu_seqlens is NULL");
  SSLA_CHECK_ARG(T == 0 || (u && g && dout && keep && du && dg && (!q || dq)), "gated_scan_bwd: null pointer");
  if (T == 0 && n_seq == 0) return SSLA_OK;
  ScanArgs a{};
  a.u = u; a.g = g; a.q = q; a.dout = dout; a.ldu = ldu; a.ldg = ldg; a.ldq = ldq;
  a.cu = cu_seqlens; a.n_seq = n_seq; a.T = T; a.C = C; a.gate = gate;
  a.h0 = h0; a.dht = dht; a.du = du; a.dg = dg; a.dq = dq; a.dh0 = dh0;
  a.keep = static_cast<float *>(const_cast<void *>(keep));
  const int W = widest(C, 4, {{u, ldu, dtype}, {g, ldg, g_dtype}, {q, q ? ldq : 0, dtype}, {dout, C, dtype}, {du, C, dtype},
                              {dg, C, g_dtype}, {dq, C, dtype}});
  int status = SSLA_OK;
#define SSLA_LAUNCH(D, G, W_) \
  status = launch_scan("gated_scan_bwd", a, W_, scan_bwd_kernel<D, G, W_>, workspace, workspace_bytes, static_cast<hipStream_t>(stream))
#define SSLA_CALL(D, G)             \
  if (W == 4) SSLA_LAUNCH(D, G, 4); \
  else SSLA_LAUNCH(D, G, 1)
  SSLA_SCAN_TYPES(SSLA_CALL);
#undef SSLA_CALL
#undef SSLA_LAUNCH
  return status == SSLA_OK ? launch_status("gated_scan_bwd") : status;
}

extern "C" int ssla_sparse_gated_step(const int32_t *row_idx, int n_active, const void *u, int64_t ldu, const void *g,
                                      int64_t ldg, const void *q, int64_t ldq, float *state, int n_rows, int C, int gate,
                                      void *o, int32_t *status, int dtype, int g_dtype, void *stream) {
  using namespace ssla;
  clear_error();
  SSLA_CHECK_ARG(n_rows >= 0, "sparse_gated_step: bad sizes n_rows=%d", n_rows);
  if (const int e = check_sizes("sparse_gated_step", n_active, n_active, C, gate, dtype, g_dtype, ldu, ldg, q ? ldq : ldu))
    return e;
  if (n_active == 0) return SSLA_OK;
  SSLA_CHECK_ARG(row_idx && u && g && o && (state || n_rows == 0), "sparse_gated_step: null pointer");
  StepArgs a{row_idx, u, g, q, ldu, ldg, ldq, state, o, status, n_active, n_rows, C, gate};
  const int64_t blocks = (static_cast<int64_t>(n_active) * C + 255) / 256;
#define SSLA_CALL(D, G) \
  hipLaunchKernelGGL((scan_step_kernel<D, G>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, \
                     static_cast<hipStream_t>(stream), a)
  SSLA_SCAN_TYPES(SSLA_CALL);
#undef SSLA_CALL
  return launch_status("sparse_gated_step");
}

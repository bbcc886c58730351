// Gated delta rule on gfx950, token by token: per sequence and head
//   S <- e^(g_t) S,  u_t = beta_t (v_t - S^T k_t),  S <- S + k_t u_t^T,
//   o_t = scale S^T q_t.
// Both products read the state before the token's write: with r = S^T k and
// p = S^T q of the old state, u = beta (v - e^g r), o = scale (e^g p +
// (k . q) u) and S <- e^g S + k u^T, so a token waits on one reduction over
// the keys, not on two.
//
// Sequences: one wavefront per (sequence, head, NC value columns), lane = (key
// group of 64 / NC, column), each with KR state rows in fp32; the value columns of
// a state are independent of each other.  NC is 16, and 8 (half the instructions
// a token, twice the wavefronts) for batches that leave SIMDs without one.  Tokens are fetched BT at a time with
// 16-byte loads while the block before runs, and parked in LDS of the wavefront's
// own as fp32, with the decays and the products k . q, so a token's chain is the
// sum S^T k, u and the update.  Bound by vector instructions (4,510 histories of 13
// tokens, 4 heads of 32, fp32: 87 us, 3.1 TB/s; VALU busy 66 % of the time, 69
// instructions a token and 16 columns where its formula takes about 50: blocks are
// staged and dotted for 16 tokens), long histories by the chain, 0.20 us a token of
// 32 keys, 0.27 of 64 and 0.41 of 128.
//
// Single tokens: one wavefront per (row, head, 4 VL value columns), the whole of
// a state's columns in registers as 16-byte pieces, every load in flight at once.
// Bound by memory: a state is read and written (1,024 rows, 8 heads of 128 x 128:
// 210 us, 5.1 TB/s).
#include "delta_tile.h"

namespace ssla {
namespace {

struct DeltaArgs {
  const void *q, *k, *v;
  const float *g, *beta;
  const int64_t *cu;      // NULL: sequence n is row n
  const int32_t *row_of;  // NULL: sequence n's state is row n
  const float *h0;
  float *ht;
  void *o;
  int32_t *status;
  int64_t T, longest;     // sequences of more rows are left to another kernel
  int n_seq, Hk, H, K, V, n_rows, kvec, vvec;   // k and q, v and o: rows of whole 16-byte pieces
  float scale;
};

// The state's row of sequence n, or -1 where the list's entry must be skipped.
__device__ __forceinline__ int64_t state_row(const DeltaArgs &a, int64_t n) {
  if (!a.row_of) return n;
  const int64_t row = a.row_of[n];
  return row < 0 || row >= a.n_rows || (n > 0 && a.row_of[n - 1] >= row) ? -1 : row;
}
__device__ __forceinline__ void report(const DeltaArgs &a) {
  if (a.status && (threadIdx.x & 63) == 0)
    __hip_atomic_store(a.status, SSLA_ERR_ARG, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Orders this wavefront's LDS accesses (its lanes read what others wrote; LDS
// serves one wavefront in order, so only the compiler needs to be told).
__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Sum over the lanes of a column (the key groups): lane swaps on the VALU, where a
// shuffle would be a trip through LDS in every token's chain.  A value swapped
// with itself gives both partners' values to both.
template <int NC>
__device__ __forceinline__ float sum_groups(float x) {
  if constexpr (NC == 8)
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));
  const uint32_t b = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  const uint32_t y = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// ROWS rows of `n` values (n <= N) at a stride, 16 bytes a lane and load where
// vec, into registers and from there to LDS rows of LD floats (zeros behind).
template <int DT, int ROWS, int N, int LD>
struct Rows {
  typedef typename Elem<DT>::T E;
  static constexpr int ES = sizeof(E), P = 16 / ES, PIECES = ROWS * N / P, L = (PIECES + 63) / 64;
  struct Piece { E e[P]; };
  Piece p[L];
  __device__ __forceinline__ void fetch(const Rsrc &rs, int64_t stride, int n, bool vec) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int u = lane + 64 * i, row = u / (N / P), col = (u % (N / P)) * P;
      const uint32_t at = u < PIECES ? static_cast<uint32_t>(row * stride + col) * ES : kOutside;
      if (vec) {
        p[i] = __builtin_bit_cast(Piece, __builtin_amdgcn_raw_buffer_load_b128(rs, col + P <= n ? at : kOutside, 0, 0));
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) p[i].e[j] = load_one<E>(rs, u < PIECES && col + j < n ? at + j * ES : kOutside);
      }
    }
  }
  __device__ __forceinline__ void park(float *lds) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int u = lane + 64 * i, row = u / (N / P), col = (u % (N / P)) * P;
      if (u < PIECES)
#pragma unroll
        for (int j = 0; j < P; j += 4)
          *reinterpret_cast<f32x4 *>(lds + row * LD + col + j) =
              f32x4{of_elem<DT>(p[i].e[j]), of_elem<DT>(p[i].e[j + 1]), of_elem<DT>(p[i].e[j + 2]), of_elem<DT>(p[i].e[j + 3])};
    }
  }
  // the other way: LDS rows to memory
  static __device__ __forceinline__ void put(const float *lds, const Rsrc &rs, int64_t stride, int n, bool vec) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int u = lane + 64 * i, row = u / (N / P), col = (u % (N / P)) * P;
      const uint32_t at = u < PIECES ? static_cast<uint32_t>(row * stride + col) * ES : kOutside;
      Piece x;
#pragma unroll
      for (int j = 0; j < P; ++j) x.e[j] = to_elem<DT>(u < PIECES ? lds[row * LD + col + j] : 0.f);
      if (vec) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(__attribute__((ext_vector_type(4))) uint32_t, x), rs,
                                               col + P <= n ? at : kOutside, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) store_one<E>(rs, u < PIECES && col + j < n ? at + j * ES : kOutside, x.e[j]);
      }
    }
  }
};

template <int NC, int KR, int BT>
struct BlockLds {   // one wavefront's
  static constexpr int KT = 64 / NC * KR;
  float k[BT][KT], q[BT][KT], v[BT][NC], gb[BT][4];   // gb: decay, beta, k . q
};

template <int NC, int KR, int BT, int DT>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(const DeltaArgs a) {
  typedef typename Elem<DT>::T ET;
  constexpr int ES = sizeof(ET);
  typedef BlockLds<NC, KR, BT> Lds;
  constexpr int KT = Lds::KT;
  __shared__ __align__(16) Lds sm[4];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Lds &m = sm[w];
  const int n_vt = (a.V + NC - 1) / NC;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + w;
  if (item >= static_cast<int64_t>(a.n_seq) * a.H * n_vt) return;   // whole wavefront
  const int vt = static_cast<int>(item % n_vt), h = static_cast<int>((item / n_vt) % a.H);
  const int64_t n = item / (static_cast<int64_t>(n_vt) * a.H);
  const int hk = h / (a.H / a.Hk), c0 = vt * NC, nc = min(NC, a.V - c0);
  const int col = lane % NC, kg = lane / NC;

  // (clamped to [0, T): no offset addresses memory outside the tensors)
  int64_t bos = n, eos = n + 1;
  if (a.cu) {
    bos = min(max(a.cu[n], (int64_t)0), a.T);
    eos = min(max(a.cu[n + 1], bos), a.T);
  }
  if (eos - bos > a.longest) return;   // whole wavefront
  const int64_t row = state_row(a, n), vstride = static_cast<int64_t>(a.H) * a.V, kstride = static_cast<int64_t>(a.Hk) * a.K;
  if (row < 0) {
    report(a);
    for (int64_t t = bos; t < eos; ++t)
      if (lane < nc) Elem<DT>::store(a.o, (t * a.H + h) * a.V + c0 + lane, 0.f);
    return;
  }

  // state: rows kg KR .. of this lane's column
  const int64_t s0 = (row * a.H + h) * a.K * a.V;
  const uint32_t soff = col < nc ? static_cast<uint32_t>(kg * KR * a.V + c0 + col) * 4 : kOutside;
  float S[KR];
  {
    const Rsrc rs = rsrc_of(a.h0 + s0, a.h0 ? static_cast<int64_t>(a.K) * a.V * 4 : 0);
#pragma unroll
    for (int i = 0; i < KR; ++i) S[i] = load_one<float>(rs, soff + i * a.V * 4);
  }

  Rows<DT, BT, KT, KT> kr, qr;
  Rows<DT, BT, NC, NC> vr;
  float gr = 0.f;
  auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(BT), eos - t0));
    const int64_t kat = (t0 * a.Hk + hk) * a.K;
    kr.fetch(rows_rsrc(a.k, kat, rows, kstride, a.K, ES), kstride, a.K, a.kvec);
    qr.fetch(rows_rsrc(a.q, kat, rows, kstride, a.K, ES), kstride, a.K, a.kvec);
    vr.fetch(rows_rsrc(a.v, (t0 * a.H + h) * a.V + c0, rows, vstride, nc, ES), vstride, nc, a.vvec);
    const int r = lane & 31;   // lanes 0 .. : gates, lanes 32 .. : weights
    gr = r < rows ? (lane < 32 ? a.g : a.beta)[(t0 + r) * a.H + h] : 0.f;
  };
  if (bos < eos) fetch(bos);
  for (int64_t t0 = bos; t0 < eos; t0 += BT) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(BT), eos - t0));
    kr.park(&m.k[0][0]);
    qr.park(&m.q[0][0]);
    vr.park(&m.v[0][0]);
    if ((lane & 31) < BT) m.gb[lane & 31][lane >> 5] = lane < 32 ? fast_exp2(gr * kLog2e) : gr;
    lds_order();
    if (t0 + BT < eos) fetch(t0 + BT);   // the next block's, in flight meanwhile
    {   // k . q of all tokens: four lanes each
      const int t = lane >> 2, j0 = (lane & 3) * (KT / 4);
      float s = 0.f;
      if (t < BT)
#pragma unroll
        for (int i = 0; i < KT / 4; ++i) s = fmaf(m.k[t][j0 + i], m.q[t][j0 + i], s);
      s += __shfl_xor(s, 1);
      s += __shfl_xor(s, 2);
      if (t < BT && (lane & 3) == 0) m.gb[t][2] = s;
    }
    lds_order();
    struct Token {
      f32x4 k[KR / 4], q[KR / 4], gb;
      float v;
    };
    auto read = [&](Token &x, int t) __attribute__((always_inline)) {
      t = min(t, BT - 1);
      x.gb = *reinterpret_cast<const f32x4 *>(&m.gb[t][0]);
      x.v = m.v[t][col];
#pragma unroll
      for (int i = 0; i < KR / 4; ++i) {
        x.k[i] = *reinterpret_cast<const f32x4 *>(&m.k[t][kg * KR + 4 * i]);
        x.q[i] = *reinterpret_cast<const f32x4 *>(&m.q[t][kg * KR + 4 * i]);
      }
    };
    auto write = [&](const Token &x, int t) __attribute__((always_inline)) {
      float r0 = 0.f, r1 = 0.f, p0 = 0.f, p1 = 0.f;
#pragma unroll
      for (int i = 0; i < KR; i += 2) {
        r0 = fmaf(x.k[i >> 2][i & 3], S[i], r0);
        r1 = fmaf(x.k[i >> 2][(i & 3) + 1], S[i + 1], r1);
        p0 = fmaf(x.q[i >> 2][i & 3], S[i], p0);
        p1 = fmaf(x.q[i >> 2][(i & 3) + 1], S[i + 1], p1);
      }
      const float eg = x.gb[0], r = sum_groups<NC>(r0 + r1), p = sum_groups<NC>(p0 + p1);
      const float u = x.gb[1] * fmaf(-eg, r, x.v);
#pragma unroll
      for (int i = 0; i < KR; ++i) S[i] = fmaf(x.k[i >> 2][i & 3], u, eg * S[i]);
      if (kg == 0) m.v[t][col] = a.scale * fmaf(x.gb[2], u, eg * p);   // o in the place of v
    };
    // a token's values are read while the one before runs (two sets of registers,
    // where the keys' leave room for them)
    Token x, y;
    read(x, 0);
    if constexpr (KR <= 16) {
      for (int t = 0; t < rows; t += 2) {
        read(y, t + 1);
        write(x, t);
        if (t + 1 == rows) break;
        read(x, t + 2);
        write(y, t + 1);
      }
    } else {
      for (int t = 0; t < rows; ++t) {
        write(x, t);
        read(x, t + 1);
      }
    }
    lds_order();
    Rows<DT, BT, NC, NC>::put(&m.v[0][0], rows_rsrc(a.o, (t0 * a.H + h) * a.V + c0, rows, vstride, nc, ES), vstride, nc,
                              a.vvec);
    lds_order();
  }

  if (a.ht) {
    const Rsrc rs = rsrc_of(a.ht + s0, static_cast<int64_t>(a.K) * a.V * 4);
#pragma unroll
    for (int i = 0; i < KR; ++i) store_one<float>(rs, soff + i * a.V * 4, S[i]);
  }
}

// One token of every row: lane = (key group of 64 / VL, 16-byte piece of the
// columns), RPL state rows each.
template <int VL, int RPL, int DT>
__global__ __launch_bounds__(256) void delta_step_kernel(const DeltaArgs a) {
  typedef typename Elem<DT>::T ET;
  constexpr int CW = 4 * VL;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n_vt = (a.V + CW - 1) / CW;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + w;
  if (item >= static_cast<int64_t>(a.n_seq) * a.H * n_vt) return;   // whole wavefront
  const int vt = static_cast<int>(item % n_vt), h = static_cast<int>((item / n_vt) % a.H);
  const int64_t n = item / (static_cast<int64_t>(n_vt) * a.H);
  const int hk = h / (a.H / a.Hk), c = vt * CW + (lane % VL) * 4, k0 = (lane / VL) * RPL;
  const bool col_ok = c < a.V;   // (V is a multiple of 4)
  const int64_t at = (n * a.H + h) * a.V + c, row = state_row(a, n);
  if (row < 0) {
    report(a);
    if (lane < VL && col_ok)
#pragma unroll
      for (int j = 0; j < 4; ++j) Elem<DT>::store(a.o, at + j, 0.f);
    return;
  }
  const int64_t s0 = (row * a.H + h) * a.K * a.V, bytes = static_cast<int64_t>(a.K) * a.V * 4;
  const uint32_t soff = col_ok ? static_cast<uint32_t>(k0 * a.V + c) * 4 : kOutside;
  const Rsrc rs = rsrc_of(a.h0 + s0, a.h0 ? bytes : 0);
  f32x4 S[RPL];
#pragma unroll
  for (int i = 0; i < RPL; ++i)
    S[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, soff + i * a.V * 4, 0, 0));
  const int64_t kat = (n * a.Hk + hk) * a.K;
  const Rsrc rk = rows_rsrc(a.k, kat, 1, 0, a.K, sizeof(ET)), rq = rows_rsrc(a.q, kat, 1, 0, a.K, sizeof(ET));
  struct Run { ET e[RPL]; } ke, qe;
  if constexpr (sizeof(Run) % 16 == 0) {
    constexpr int W = sizeof(Run) / 16, P = 16 / sizeof(ET);
    if (a.kvec) {
      struct Raw { uint4 x[W]; } kw, qw;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint32_t off = static_cast<uint32_t>(k0 + j * P) * sizeof(ET);
        kw.x[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, off, 0, 0));
        qw.x[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rq, off, 0, 0));
      }
      ke = __builtin_bit_cast(Run, kw);
      qe = __builtin_bit_cast(Run, qw);
    }
  }
  if (sizeof(Run) % 16 != 0 || !a.kvec) {
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      ke.e[i] = load_one<ET>(rk, (k0 + i) * sizeof(ET));
      qe.e[i] = load_one<ET>(rq, (k0 + i) * sizeof(ET));
    }
  }
  const float eg = fast_exp2(a.g[n * a.H + h] * kLog2e), b = a.beta[n * a.H + h];
  f32x4 vv = f32x4{0.f, 0.f, 0.f, 0.f};
  if (col_ok)
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = Elem<DT>::load(a.v, at + j);
  f32x4 r = f32x4{0.f, 0.f, 0.f, 0.f}, p = r;
  float kq = 0.f;
#pragma unroll
  for (int i = 0; i < RPL; ++i) {
    const float kx = of_elem<DT>(ke.e[i]), qx = of_elem<DT>(qe.e[i]);
    kq = fmaf(kx, qx, kq);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] = fmaf(kx, S[i][j], r[j]);
      p[j] = fmaf(qx, S[i][j], p[j]);
    }
  }
#pragma unroll
  for (int d = VL; d < 64; d <<= 1) {
    kq += __shfl_xor(kq, d);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] += __shfl_xor(r[j], d);
      p[j] += __shfl_xor(p[j], d);
    }
  }
  const f32x4 u = b * (vv - eg * r);
  const Rsrc wt = rsrc_of(a.ht + s0, a.ht ? bytes : 0);
#pragma unroll
  for (int i = 0; i < RPL; ++i) {
    const f32x4 x = eg * S[i] + of_elem<DT>(ke.e[i]) * u;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(__attribute__((ext_vector_type(4))) uint32_t, x), wt,
                                           soff + i * a.V * 4, 0, 0);
  }
  if (lane < VL && col_ok)
#pragma unroll
    for (int j = 0; j < 4; ++j) Elem<DT>::store(a.o, at + j, a.scale * fmaf(kq, u[j], eg * p[j]));
}

template <int VL, int DT>
bool launch_step(const DeltaArgs &a, dim3 grid, hipStream_t st) {
  const int rpl = (a.K + 64 / VL - 1) / (64 / VL);
#define SSLA_STEP(R_)                                                                          \
  if (rpl <= R_) {                                                                             \
    hipLaunchKernelGGL((delta_step_kernel<VL, R_, DT>), grid, dim3(256), 0, st, a);            \
    return true;                                                                               \
  }
  SSLA_STEP(2) SSLA_STEP(4) SSLA_STEP(8) SSLA_STEP(16) SSLA_STEP(32)
#undef SSLA_STEP
  return false;
}

template <int DT>
int launch_delta(const char *what, const DeltaArgs &a, hipStream_t st) {
  // single tokens: 16-byte pieces of the states' rows, at most 32 rows a lane
  const int vl = a.V <= 16 ? 4 : a.V <= 32 ? 8 : 16;
  const bool step = a.cu == nullptr && a.V % 4 == 0 && aligned(a.h0, 16) && aligned(a.ht, 16) && (a.K + 64 / vl - 1) / (64 / vl) <= 32;
  // fewer wavefronts than the 1,024 SIMDs: 8 columns each (71 histories of 9,001
  // tokens, 4 heads of 32: 568 wavefronts of 16 columns 157 us, twice as many of 8 125 us)
  const int64_t seqs = static_cast<int64_t>(a.n_seq) * a.H;
  const bool narrow = !step && seqs * ((a.V + 15) / 16) < 1024 && a.V > 8;
  const int64_t tiles = step ? (a.V + 4 * vl - 1) / (4 * vl) : narrow ? (a.V + 7) / 8 : (a.V + 15) / 16;
  const int64_t blocks = (seqs * tiles + 3) / 4;
  if (blocks > 0x7fffffff) {
    set_error("%s: too many (sequence, head, tile) items", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  if (step) {
    if (vl == 4) launch_step<4, DT>(a, grid, st);
    else if (vl == 8) launch_step<8, DT>(a, grid, st);
    else launch_step<16, DT>(a, grid, st);
    return launch_status(what);
  }
#define SSLA_DELTA(KR_, BT_)                                                                                   \
  do {                                                                                                         \
    if (narrow) hipLaunchKernelGGL((delta_recurrent_kernel<8, (KR_ > 4 ? KR_ / 2 : 4), BT_, DT>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((delta_recurrent_kernel<16, KR_, BT_, DT>), grid, block, 0, st, a);                \
  } while (0)
  if (a.K <= 16) SSLA_DELTA(4, 16);
  else if (a.K <= 32) SSLA_DELTA(8, 16);
  else if (a.K <= 64) SSLA_DELTA(16, 16);
  else if (a.K <= 128) SSLA_DELTA(32, 8);
  else SSLA_DELTA(64, 4);
#undef SSLA_DELTA
  return launch_status(what);
}

}  // namespace

int delta_recurrent_up_to(const char *what, int64_t longest, const void *q, const void *k, const void *v, const float *g,
                          const float *beta, const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk, int H, int K, int V,
                          float scale, const float *h0, void *o, float *ht, const int32_t *state_idx, int n_state_rows,
                          int32_t *status, int dtype, hipStream_t st) {
  const int64_t es = dtype == SSLA_F32 ? 4 : 2;
  const int kvec = K * es % 16 == 0 && aligned(q, 16) && aligned(k, 16);
  const int vvec = V * es % 16 == 0 && aligned(v, 16) && aligned(o, 16);
  const DeltaArgs a{q, k, v, g, beta, cu_seqlens, state_idx, h0, ht, o, status, T, longest, n_seq, Hk, H, K, V,
                    n_state_rows, kvec, vvec, scale};
  switch (dtype) {
    case SSLA_F32: return launch_delta<SSLA_F32>(what, a, st);
    case SSLA_BF16: return launch_delta<SSLA_BF16>(what, a, st);
    case SSLA_F16: return launch_delta<SSLA_F16>(what, a, st);
  }
  set_error("%s: unsupported dtype %d", what, dtype);
  return SSLA_ERR_DTYPE;
}

}  // namespace ssla

extern "C" int ssla_gated_delta_recurrent(const void *q, const void *k, const void *v, const float *g,
                                          const float *beta, const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk,
                                          int H, int K, int V, float scale, const float *h0, void *o, float *ht,
                                          const int32_t *state_idx, int n_state_rows, int32_t *status, int dtype,
                                          void *stream) {
  using namespace ssla;
  clear_error();
  SSLA_CHECK_ARG(n_seq >= 0 && T >= 0 && Hk > 0 && H > 0 && H % Hk == 0 && K > 0 && V > 0,
                 "gated_delta_recurrent: bad sizes n_seq=%d T=%lld Hk=%d H=%d K=%d V=%d", n_seq, (long long)T, Hk, H, K,
                 V);
  if (K > 256) {
    set_error("gated_delta_recurrent: K=%d exceeds 256", K);
    return SSLA_ERR_UNSUPPORTED;
  }
  if (n_seq == 0) return SSLA_OK;
  SSLA_CHECK_ARG(cu_seqlens != nullptr || T == n_seq, "gated_delta_recurrent: no cu_seqlens and T != n_seq");
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta && o), "gated_delta_recurrent: null tensor pointer");
  SSLA_CHECK_ARG(state_idx == nullptr || (n_state_rows >= 0 && h0 && ht),
                 "gated_delta_recurrent: state_idx without a state table");
  if (const int e = check_widths("gated_delta_recurrent", 16, Hk, H, K, V)) return e;
  return delta_recurrent_up_to("gated_delta_recurrent", INT64_MAX, q, k, v, g, beta, cu_seqlens, n_seq, T, Hk, H, K, V,
                               scale, h0, o, ht, state_idx, n_state_rows, status, dtype, static_cast<hipStream_t>(stream));
}

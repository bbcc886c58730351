// Chunked gated delta rule, forward, on gfx950.
//
// Per sequence and head, S <- e^(g_t) S, u_t = beta_t (v_t - S^T k_t),
// S <- S + k_t u_t^T, o_t = scale S^T q_t.  In a chunk of 64 rows, with G the
// inclusive sum of g from the chunk's start and S the state entering it,
//   u = Tm X,  X_i = beta_i (v_i - e^(G_i) S^T k_i),
//   Tm = (I + A)^-1,  A_ij = beta_i e^(G_i - G_j) k_i . k_j  (j < i),
//   o_i = scale e^(G_i) S^T q_i + sum_(j <= i) P_ij u_j,
//   P_ij = scale e^(G_i - G_j) q_i . k_j,
//   S' = e^(G_last) S + sum_j k_j (e^(G_last - G_j) u_j)^T.
// Tm needs no state: one kernel computes it for all chunks side by side (unit
// lower triangular, by forward substitution in 16 x 16 blocks whose inverses
// are joined: no power of A, so equal keys lose no digits).  The walk then
// carries the states from chunk to chunk, one wavefront per 16 value columns,
// which do not need each other.
//
// Long sequences are cut into segments that run side by side: over a segment
// the state goes through an affine map S -> M S + L, and the columns of M are
// columns of a state that enters as the identity with v = 0.  A pass over all
// segments but a sequence's last computes L and M (the first segment's from the
// initial state, so it needs no M), a fold carries the states over the segments,
// and the walk starts every segment from its state.
//
// Measured at 8 sequences of 4096 rows, 8 heads of 64, bf16: matrices 31 us,
// segments 66, fold 9, walk 60; 151 a pass among others, 0.9 TB/s of the inputs
// and outputs.  Bound by latency: a SIMD has two (walk) or three (segments)
// wavefronts, VALU busy 37 % and matrix cores 20 % of the time; more wavefronts
// need fewer registers than the states, one operand's parts and the next chunk's
// loads take.
//
// Values that are not finite: a row whose beta, g or k . k is not finite makes all
// columns of its head NaN from that row on, one in v or in a state its own
// column; earlier rows are computed without them.
#include "delta_tile.h"
#include "seq_slots.h"

namespace ssla {
namespace {

// (what rounds to an infinity in bf16 counts as one)
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < 3.38e38f; }

// -------------------------------------------------- matrices of the chunks --
// One workgroup per (chunk slot, head): the row factors and Tm.
template <int DT, int KP>
__global__ __launch_bounds__(256) void delta_prep_kernel(const void *__restrict__ k, const float *__restrict__ g,
                                                         const float *__restrict__ beta,
                                                         const int64_t *__restrict__ cu, int n_seq, int64_t T, int Hk,
                                                         int H, int K, int vec, int mixed, float scale,
                                                         float *__restrict__ tm, int tm_floats,
                                                         float *__restrict__ rowv) {
  constexpr int NP = Parts<DT>::n, LD = 68;
  constexpr int SK = NP * kChunk * KP * 2, SA = kChunk * LD * 4;
  __shared__ __align__(16) char buf[SK > SA ? SK : SA];
  auto sk = reinterpret_cast<uint16_t(*)[kChunk * KP]>(buf);   // k, until its Gram matrix is in registers
  auto A = reinterpret_cast<float(*)[LD]>(buf);                // then I + A, then Tm
  __shared__ float sv[kRowVecs][kChunk];
  __shared__ float diag[kChunk];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int h = static_cast<int>(blockIdx.x % H), hk = h / (H / Hk);
  const int64_t slot = blockIdx.x / H;
  int n;
  int64_t bos, eos, first;
  auto slot_of = [&](int64_t row, int i) __attribute__((always_inline)) { return chunk_slot(row, i, 0, mixed); };
  if (!seq_of_slot_by(cu, n_seq, T, slot, slot_of, n, bos, eos, first)) return;   // workgroup-uniform
  if (mixed && eos - bos <= kChunk) return;
  const int64_t t0 = bos + (slot - first) * kChunk;
  if (t0 >= eos) return;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0));

  RowTile<DT, KP> kt;
  kt.fetch(rows_rsrc(k, (t0 * Hk + hk) * K, rows, Hk * K, K, RowTile<DT, KP>::ES), Hk * K, K, vec);
  // the row factors, while k is on its way: e^-150 is 0 in fp32; sums in 64 bits,
  // kept as two floats, so that differences of far sums stay exact
  float gv = 0.f, bv = 0.f;
  auto factors = [&]() __attribute__((always_inline)) {
    double G = static_cast<double>(fmaxf(gv, -150.f)) * 1.4426950408889634;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double up = __shfl_up(G, d);
      if (lane >= d) G += up;
    }
    const float hi = static_cast<float>(G), lo = static_cast<float>(G - static_cast<double>(hi));
    const float eg = fast_exp2(hi) * fast_exp2(lo), last = __shfl(hi, 63), last_lo = __shfl(lo, 63);
    sv[kBeta][lane] = bv;
    sv[kBetaG][lane] = bv * eg;
    sv[kScaleG][lane] = scale * eg;
    sv[kToEnd][lane] = fast_exp2((last - hi) + (last_lo - lo));
    sv[kGHi][lane] = hi;
    sv[kGLo][lane] = lo;
  };
  if (w == 0) {
    if (lane < rows) {
      gv = g[(t0 + lane) * H + h];
      bv = beta[(t0 + lane) * H + h];
    }
    factors();
  }
  kt.store(&sk[0][0], kChunk * KP);
  __syncthreads();

  // Gram matrix k k^T: wavefront w computes the row tile w
  f32x4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KP / 32; ++ks) {
    bf16x8 a[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) a[i] = op_rows<KP>(sk[i], w, ks, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > (w | 1)) continue;   // columns past the rows' pair: above the diagonal
      bf16x8 b[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) b[i] = op_rows<KP>(sk[i], j, ks, lane);
      acc[j] = mul<2>(a, b, acc[j]);
    }
  }
  {   // the diagonal tells whether a row of k is finite
    const int r = (lane >> 4) * 4, m = lane & 15;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j == w && m >= r && m < r + 4) {
        const f32x4 v4 = acc[j];
        diag[idx_of(w, m)] = m == r ? v4[0] : m == r + 1 ? v4[1] : m == r + 2 ? v4[2] : v4[3];
      }
  }
  __syncthreads();
  if (w == 0) {
    // a row that is not finite (a gate of -inf is: it empties the state) and
    // those after it are left out of Tm; its beta becomes NaN, which the walk
    // turns into NaN for all that follows
    const bool bad = lane < rows && !(finite(diag[lane]) && finite(bv) && gv < 3.38e38f);
    const unsigned long long any = __ballot(bad);
    const int r0 = any ? __ffsll(static_cast<long long>(any)) - 1 : kChunk;
    if (any) {
      if (lane >= r0) {
        gv = 0.f;
        bv = lane == r0 ? __builtin_nanf("") : 0.f;
      }
      factors();
    }
    diag[lane] = lane < r0 ? bv : 0.f;   // now: beta of the rows that Tm takes
  }
  __syncthreads();
  {
    const int col = lane & 15, row = idx_of(w, (lane >> 4) * 4);   // and the three rows behind it
    const f32x4 hi = *reinterpret_cast<const f32x4 *>(&sv[kGHi][row]), lo = *reinterpret_cast<const f32x4 *>(&sv[kGLo][row]);
    const f32x4 bt = *reinterpret_cast<const f32x4 *>(&diag[row]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > (w | 1)) continue;
      const int c = idx_of(j, col);
      const float chi = sv[kGHi][c], clo = sv[kGLo][c];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = bt[i] * acc[j][i] * fast_exp2((hi[i] - chi) + (lo[i] - clo));
        // (a selection, not a product: what is above the diagonal or left out may be NaN)
        A[row + i][c] = row + i == c ? 1.f : keep(c < row + i && bt[i] != 0.f, x);
      }
    }
  }
  // (rows r0.. have beta 0, so row r0's NaN keys reach no other row: row > c >= r0 is left out by its own beta)
  __syncthreads();
  // the four diagonal blocks of 16, inverted in place: lane = (block, column)
  if (w == 0) {
    const int b = 16 * (lane >> 4), c = lane & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-A[b + i][b + j], x[j], s);
      x[i] = s;
    }
    // (one wavefront: all reads above are done before the writes)
#pragma unroll
    for (int i = 0; i < 16; ++i) A[b + i][b + c] = i < c ? 0.f : x[i];
  }
  __syncthreads();
  // joins: [[P, 0], [C, Q]]^-1 = [[P^-1, 0], [-Q^-1 C P^-1, Q^-1]], in fp32
  const int m = lane & 15, gr = lane >> 4;
  if (w < 2) {   // blocks of 16, a pair for each of two wavefronts
    const int b = 32 * w;
    float x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = A[b + 16 + m][b + 4 * gr + j];
      y[j] = A[b + 4 * gr + j][b + m];
    }
    f32x4 c = mul_f32(x, y, f32x4{0.f, 0.f, 0.f, 0.f});   // rows 4 gr + i = the next product's contraction
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = A[b + 16 + m][b + 16 + 4 * gr + j];
      y[j] = c[j];
    }
    c = mul_f32(x, y, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int i = 0; i < 4; ++i) A[b + 16 + 4 * gr + i][b + m] = -c[i];
  }
  __syncthreads();
  {   // blocks of 32: wavefront w has 16 columns; both row tiles of C P^-1 feed its column of the second product
    const int ct = 16 * (w & 1), rt = 16 * (w >> 1);
    float x[8], y[8];
    f32x4 c[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = A[8 * gr + j][ct + m];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = A[32 + idx_of(t, m)][8 * gr + j];
      c[t] = mul_f32(x, y, f32x4{0.f, 0.f, 0.f, 0.f});
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = A[32 + rt + m][32 + 8 * gr + j];
      y[j] = c[j >> 2][j & 3];
    }
    c[0] = mul_f32(x, y, f32x4{0.f, 0.f, 0.f, 0.f});
    __syncthreads();   // C is read
#pragma unroll
    for (int i = 0; i < 4; ++i) A[32 + rt + 4 * gr + i][ct + m] = -c[0][i];
  }
  __syncthreads();
  // operands: thread (b, lane, half of its eight values) has sets b, 2 + b, 4 + b
  f32x4 *dst = reinterpret_cast<f32x4 *>(tm + (slot * H + h) * tm_floats) + tid;
  const int b = tid >> 7, om = (tid >> 1) & 15, oc = 8 * ((tid >> 5) & 3) + 4 * (tid & 1);
#pragma unroll
  for (int i = 0; i < 3; ++i) {   // Tm: row tiles 0, 1 need the first half, 2, 3 both
    const int t = i == 0 ? b : i + 1, ks = i == 0 ? 0 : b;
    dst[256 * i] = *reinterpret_cast<const f32x4 *>(&A[idx_of(t, om)][32 * ks + oc]);
  }
  if (tm_floats > kTriFloats) {   // and Tm^T: row tiles 0, 1 need both halves, 2, 3 the second
    dst += kTriFloats / 4;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int t = i == 2 ? 2 + b : i, ks = i == 2 ? 1 : b;
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = A[32 * ks + oc + j][idx_of(t, om)];
      dst[256 * i] = x;
    }
  }
  float *dv = rowv + (slot * H + h) * kRowFloats;
  for (int e = tid; e < kRowFloats; e += 256) dv[e] = (&sv[0][0])[e];
}

// ----------------------------------------------------------------- the walk --
// kOutput walks a segment from its entering state and writes o (and ht behind the
// sequence's last row); kStates does so and writes every chunk's entering state
// and u instead (for the backward); kSegment walks an inner segment from zero
// (a sequence's first from its initial state) and from the identity and writes L
// and M.
enum { kOutput, kStates, kSegment };

template <int DT, int KP, bool OUT>
struct WalkSmem {
  static constexpr int NP = Parts<DT>::n, NO = DT == SSLA_F32 ? 3 : 2;
  uint16_t k[NP][kChunk * KP];
  uint16_t q[OUT ? NP : 1][OUT ? kChunk * KP : 8];
  uint16_t tm[3][kTriSets * 512];
  uint16_t p[OUT ? NO : 1][OUT ? kTriSets * 512 : 8];
  float rowv[kRowVecs][kChunk];
};

// Four wavefronts, each with 16 columns of the state (its rows: the keys).
template <int DT, int KP, int MODE>
__global__ __launch_bounds__(256, (DT == SSLA_F32 && KP == 128) ? 1 : MODE == kSegment && KP < 128 ? 3 : 2) void delta_walk_kernel(const WalkArgs a) {
  constexpr int NP = Parts<DT>::n, NO = DT == SSLA_F32 ? 3 : 2, LIMO = NO - 1, NT = KP / 16;
  constexpr bool OUT = MODE == kOutput, SEG = MODE == kSegment;
  typedef Elem<DT> E;
  typedef typename E::T ET;
  __shared__ __align__(16) WalkSmem<DT, KP, OUT> sm;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, G = lane >> 4;
  const int n_vt = (a.V + 15) >> 4, n_groups = (n_vt + (SEG ? NT : 0) + 3) >> 2;
  int64_t b = blockIdx.x;
  const int grp = static_cast<int>(b % n_groups);
  b /= n_groups;
  const int h = static_cast<int>(b % a.H), hk = h / (a.H / a.Hk);
  const int64_t slot = b / a.H;
  const int64_t unit = static_cast<int64_t>(a.per) * kChunk;
  int n;
  int64_t bos, eos, first;
  // (segments have at least 4 chunks: in a mixed batch 64 rows a slot do)
  auto slot_of = [&](int64_t row, int i) __attribute__((always_inline)) {
    return MODE == kOutput && a.mixed ? row / kChunk : pieces_before(row, unit, a.T) + (SEG ? 0 : i);
  };
  if (!seq_of_slot_by(a.cu, a.n_seq, a.T, slot, slot_of, n, bos, eos, first)) return;   // workgroup-uniform
  if (MODE == kOutput && a.mixed && eos - bos <= kChunk) return;
  const int64_t seg = slot - first, t_begin = bos + seg * unit;
  if (SEG ? t_begin + unit >= eos : (t_begin >= eos && seg > 0)) return;
  if (SEG && seg == 0 && grp * 4 >= n_vt) return;   // (a first segment's M)
  const int64_t t_end = min(t_begin + unit, eos);
  const int tile = grp * 4 + w;
  const bool is_map = SEG && tile >= n_vt;                   // this wavefront's columns are M's
  const int vcol = tile * 16 + col, mcol = (tile - n_vt) * 16 + col;
  const bool active = is_map ? mcol < KP : tile < n_vt, v_ok = !is_map && vcol < a.V;
  const int64_t KV = static_cast<int64_t>(a.K) * a.V;

  const StateCols<NT> cols(a.K, a.V, vcol, v_ok, G);
  f32x4 S[NT];
  cols.load(seg > 0 ? (SEG ? nullptr : a.seg_state + ((bos / unit + seg - 1) * a.H + h) * KV)
            : a.h0  ? a.h0 + (static_cast<int64_t>(n) * a.H + h) * KV : nullptr, S);
  if (is_map) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][r] = idx_of(t, 4 * G + r) == mcol ? 1.f : 0.f;
  }
  // byte offset of row 8 G in this lane's column of v, o and u (in values of 4 bytes for u)
  constexpr int ES = sizeof(ET);
  const uint32_t vrow = static_cast<uint32_t>(a.H) * a.V, voff = v_ok ? (8 * G * vrow + vcol) * ES : kOutside;

  RowTile<DT, KP> kt, qt;
  f32x4 tmr[3], rvr;
  ET vr[16];
  // (a chunk past the segment: resources of no bytes, zeros and no traffic)
  auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
    const int rows = t0 < t_end ? static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0)) : 0;
    const int64_t at = (t0 * a.Hk + hk) * a.K;
    const int stride = a.Hk * a.K;
    kt.fetch(rows_rsrc(a.k, at, rows, stride, a.K, ES), stride, a.K, a.vec);
    if constexpr (OUT) qt.fetch(rows_rsrc(a.q, at, rows, stride, a.K, ES), stride, a.K, a.vec);
    const int64_t c = chunk_slot(bos, n, (t0 - bos) / kChunk, MODE != kStates && a.mixed) * a.H + h;
    const Rsrc rt = rsrc_of(a.tm + c * a.tm_floats, rows > 0 ? kTriFloats * 4 : 0);
    const Rsrc rr = rsrc_of(a.rowv + c * kRowFloats, rows > 0 ? kRowFloats * 4 : 0);
    tmr[0] = load4(rt, tid * 32);
    tmr[1] = load4(rt, tid * 32 + 16);
    tmr[2] = load4(rt, 8192 + tid * 16);
    rvr = load4(rr, tid * 16);   // (96 threads' worth)
    const Rsrc rv = rows_rsrc(a.v, (t0 * a.H + h) * a.V, rows, vrow, a.V, ES);
#pragma unroll
    for (int i = 0; i < 16; ++i) vr[i] = load_one<ET>(rv, voff + idx_of(i >> 2, i & 3) * vrow * ES);
  };
  auto stage = [&]() __attribute__((always_inline)) {
    kt.store(&sm.k[0][0], kChunk * KP);
    if constexpr (OUT) qt.store(&sm.q[0][0], kChunk * KP);
    {   // sets 0 .. 3: a lane's eight values of one thread
      bf16x8 s[3];
      split(join(tmr[0], tmr[1]), s);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4 *>(&sm.tm[i][tid * 8]) = to_bits(s[i]);
    }
    {   // sets 4, 5: half a lane's values of each thread
      uint2 s[3];
      split(tmr[2], s);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2 *>(&sm.tm[i][2048 + tid * 4]) = s[i];
    }
    if (tid < kRowFloats / 4) reinterpret_cast<f32x4 *>(&sm.rowv[0][0])[tid] = rvr;
  };
  auto row8 = [&](int vec, int p) __attribute__((always_inline)) {   // rows 32 p + 8 G .. + 7 of a row vector
    const f32x4 *s = reinterpret_cast<const f32x4 *>(&sm.rowv[vec][32 * p + 8 * G]);
    return join(s[0], s[1]);
  };

  if (t_begin < t_end) fetch(t_begin);
  for (int64_t t0 = t_begin; t0 < t_end; t0 += kChunk) {
    stage();
    f32x8 vv[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      vv[i >> 3][i & 7] = of_elem<DT>(vr[i]);
    }
    if constexpr (MODE == kStates)
      cols.store(a.chunk_state + (chunk_slot(bos, n, (t0 - bos) / kChunk) * a.H + h) * KV, S);
    __syncthreads();

    if constexpr (OUT) {
      // P of this wavefront's row tile: k q^T has row j of P^T in the lanes that
      // the operand needs (columns: the rows i of P)
      const int i = idx_of(w, col);
      const float hi = sm.rowv[kGHi][i], lo = sm.rowv[kGLo][i];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks > (w >> 1)) continue;
        f32x4 d[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kk = 0; kk < KP / 32; ++kk) {
          bf16x8 qb[NP];
#pragma unroll
          for (int j = 0; j < NP; ++j) qb[j] = op_rows<KP>(sm.q[j], w, kk, lane);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            bf16x8 ka[NP];
#pragma unroll
            for (int j = 0; j < NP; ++j) ka[j] = op_rows<KP>(sm.k[j], 2 * ks + x, kk, lane);
            d[x] = mul<LIMO>(ka, qb, d[x]);
          }
        }
        f32x8 pv = join(d[0], d[1]);
        const f32x8 ghi = row8(kGHi, ks), glo = row8(kGLo, ks);
#pragma unroll
        for (int j = 0; j < 8; ++j)   // (a selection: rows behind i may hold NaN)
          pv[j] = keep(32 * ks + 8 * G + j <= i, a.scale * pv[j] * fast_exp2((hi - ghi[j]) + (lo - glo[j])));
        bf16x8 s[NO];
        split(pv, s);
#pragma unroll
        for (int j = 0; j < NO; ++j)
          *reinterpret_cast<uint4 *>(&sm.p[j][(tri_set(w, ks) * 64 + lane) * 8]) = to_bits(s[j]);
      }
    }

    // R = k S (and q S): rows in pairs of tiles, this wavefront's columns
    f32x4 R[4], O[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) R[t] = O[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KP / 32; ++ks) {
      bf16x8 s[3];
      split(join(S[2 * ks], S[2 * ks + 1]), s);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        bf16x8 x[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) x[j] = op_rows<KP>(sm.k[j], t, ks, lane);
        R[t] = mul<2>(x, s, R[t]);
        if constexpr (OUT) {
#pragma unroll
          for (int j = 0; j < NP; ++j) x[j] = op_rows<KP>(sm.q[j], t, ks, lane);
          O[t] = mul<LIMO>(x, s, O[t]);
        }
      }
    }
    f32x8 X[2], U[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const f32x8 bt = row8(kBeta, p), bg = row8(kBetaG, p), r = join(R[2 * p], R[2 * p + 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) X[p][j] = fmaf(-bg[j], r[j], bt[j] * vv[p][j]);
    }
    int r0 = kChunk;   // this lane's column is not finite from this row on
    for (bool sane = false;; sane = true) {
      bf16x8 x[2][3];
      f32x4 u[4];
#pragma unroll
      for (int p = 0; p < 2; ++p) split(X[p], x[p]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        u[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks <= t / 2; ++ks) {
          bf16x8 m[3];
#pragma unroll
          for (int j = 0; j < 3; ++j)
            m[j] = from_bits<bf16x8>(*reinterpret_cast<const uint4 *>(&sm.tm[j][(tri_set(t, ks) * 64 + lane) * 8]));
          u[t] = mul<2>(m, x[ks], u[t]);
        }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) U[p] = join(u[2 * p], u[2 * p + 1]);
      // every row of tile 3 sums over all of X: one value tells
      if (sane || __ballot(!finite(U[1][4])) == 0) break;   // wavefront-uniform
#pragma unroll
      for (int i = 15; i >= 0; --i)
        if (!finite(X[i >> 3][i & 7])) r0 = 32 * (i >> 3) + 8 * G + (i & 7);
      r0 = min(r0, __shfl_xor(r0, 16));
      r0 = min(r0, __shfl_xor(r0, 32));
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * (i >> 3) + 8 * G + (i & 7) >= r0) X[i >> 3][i & 7] = 0.f;
    }
    if (__ballot(r0 < kChunk)) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * (i >> 3) + 8 * G + (i & 7) >= r0) U[i >> 3][i & 7] = 0.f;
    }

    if constexpr (OUT) {
      bf16x8 us[2][NO];
#pragma unroll
      for (int p = 0; p < 2; ++p) split(U[p], us[p]);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const f32x8 eg = row8(kScaleG, p);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          O[2 * p][r] *= eg[r];
          O[2 * p + 1][r] *= eg[4 + r];
        }
      }
      __syncthreads();   // P is written
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ks = 0; ks <= t / 2; ++ks) {
          bf16x8 m[NO];
#pragma unroll
          for (int j = 0; j < NO; ++j)
            m[j] = from_bits<bf16x8>(*reinterpret_cast<const uint4 *>(&sm.p[j][(tri_set(t, ks) * 64 + lane) * 8]));
          O[t] = mul<LIMO>(m, us[ks], O[t]);
        }
      const int rows = static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0));
      const Rsrc ro = rows_rsrc(a.o, (t0 * a.H + h) * a.V, rows, vrow, a.V, ES);
      if (__ballot(r0 < kChunk)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * (i >> 3) + 8 * G + (i & 7) >= r0) O[i >> 2][i & 3] = __builtin_nanf("");
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        store_one<ET>(ro, voff + idx_of(i >> 2, i & 3) * vrow * ES, to_elem<DT>(O[i >> 2][i & 3]));
    }
    if constexpr (MODE == kStates) {
      const int rows = static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0));
      const Rsrc ru = rows_rsrc(a.u, (t0 * a.H + h) * a.V, rows, vrow, a.V, 4);
      const uint32_t uoff = v_ok ? (8 * G * vrow + vcol) * 4 : kOutside;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        store_one<float>(ru, uoff + idx_of(i >> 2, i & 3) * vrow * 4,
                         32 * (i >> 3) + 8 * G + (i & 7) >= r0 ? __builtin_nanf("") : U[i >> 3][i & 7]);
    }

    // the next chunk's, in flight meanwhile (from here on fewer values are live: at
    // the chunk's start it took 60 registers more, 175 against 154 us for 16,411
    // ragged rows of 4 heads of 128)
    fetch(t0 + kChunk);

    // S <- e^(G_last) S + k^T (e^(G_last - G) u)
    bf16x8 ws[2][3];
#pragma unroll
    for (int p = 0; p < 2; ++p) split(U[p] * row8(kToEnd, p), ws[p]);
    const float through = fast_exp2(sm.rowv[kGHi][kChunk - 1]) * fast_exp2(sm.rowv[kGLo][kChunk - 1]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      S[t] *= through;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8 x[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) x[j] = op_cols<KP>(sm.k[j], t, ks, lane);
        S[t] = mul<2>(x, ws[ks], S[t]);
      }
      if (r0 < kChunk) S[t] = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
    }
    __syncthreads();   // the chunk's tiles are read
  }

  if (!SEG) {
    if (a.ht && t_end == eos) cols.store(a.ht + (static_cast<int64_t>(n) * a.H + h) * KV, S);
  } else if (is_map) {
    if (active && seg > 0) {
      uint16_t *dst = a.seg_map + (slot * a.H + h) * (3 * KP * KP) + mcol;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = S[t][r];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const uint16_t bits = f32_to_bf16_bits(x);
            x -= bf16_bits_to_f32(bits);
            dst[(p * KP + idx_of(t, 4 * G + r)) * KP] = bits;
          }
        }
    }
  } else {
    cols.store(a.seg_state + (slot * a.H + h) * KV, S);
  }
}

// The fold (see delta_fold): one workgroup per (sequence, head, 16 columns), a
// segment after the other.  A wavefront owns one or two of the state's key tiles,
// reads its rows of M from memory as operands, kAhead segments in flight, and passes
// its keys' parts to the other wavefronts through LDS (two buffers: one barrier a
// segment).  Bound by what one CU can read past its L2, 28 KB a segment of K = 64:
// 62 segments of 65,536 rows take 51 us, 58 where the columns of a head read M
// through different L2s, and the same with 2 to 8 segments in flight or half the
// instructions; 86 with M staged in LDS for 64 columns by one CU.
// Of many short sequences few are cut: a workgroup then takes an inner segment's slot
// (n_slots of them) and serves the sequence whose first one it is; otherwise sequence i.
__device__ __forceinline__ bool fold_rows(const int64_t *cu, int n_seq, int64_t T, int64_t unit, int n_slots, int i,
                                          int64_t &bos, int64_t &eos) {
  if (n_slots < n_seq) {
    int n;
    int64_t first;
    return seq_of_slot<false>(cu, n_seq, T, unit, i, n, bos, eos, first) && first == i;
  }
  bos = min(max(cu[i], (int64_t)0), T);
  eos = min(max(cu[i + 1], bos), T);
  return true;
}

template <int KP>
struct FoldSize {
  static constexpr int NT = KP / 16, WAVES = NT < 4 ? NT : 4, TPW = NT / WAVES, KS = KP / 32;
  static constexpr int kAhead = KP == 128 ? 2 : 4;
};
template <int KP>
__global__ __launch_bounds__(64 * FoldSize<KP>::WAVES) void delta_fold_kernel(
    const int64_t *__restrict__ cu, int n_seq, int n_slots, int64_t T, int H, int K, int V, int per,
    const uint16_t *__restrict__ seg_map, float *__restrict__ states) {
  typedef FoldSize<KP> F;
  constexpr int PLANE = KP * KP, D = F::kAhead;
  __shared__ __align__(16) uint2 parts[2][F::KS][3][64][2];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, G = lane >> 4;
  // (a sequence and head's columns are 8 workgroups apart: on one die, whose L2 then
  // holds M for all of them, and next to each other there, on CUs of their own,
  // however many sequences without a fold lie between)
  const int units = min(n_seq, n_slots) * H, n_cols = (V + 15) >> 4, b = static_cast<int>(blockIdx.x >> 3);
  const int u = b / n_cols * 8 + static_cast<int>(blockIdx.x & 7);
  if (u >= units) return;
  const int vcol = (b % n_cols) * 16 + col, h = u % H;
  const int64_t unit = static_cast<int64_t>(per) * kChunk, KV = static_cast<int64_t>(K) * V;
  int64_t bos, eos;
  if (!fold_rows(cu, n_seq, T, unit, n_slots, u / H, bos, eos)) return;   // workgroup-uniform
  const int inner = static_cast<int>((eos - bos + unit - 1) / unit) - 1;   // segments but the last
  if (inner < 2) return;   // the only state is there already
  const StateCols<F::NT> cols(K, V, vcol, vcol < V, G);
  struct Step {
    bf16x8 m[F::TPW][F::KS][3];
    f32x4 L[F::TPW];
  };
  Step ahead[D];
  f32x4 S[F::TPW];
  // pointers that move on by a segment: with one wavefront a SIMD, what a step costs
  // is its instructions, of which addresses from a segment's number were a third
  const int64_t first = (bos / unit) * H + h, ds = H * KV, dm = static_cast<int64_t>(H) * (3 * PLANE);
  float *out = states + first * KV;
  const float *in = out;
  const uint16_t *map = seg_map + first * (3 * PLANE);
  uint32_t moff[F::TPW], soff[F::TPW][4];
#pragma unroll
  for (int t = 0; t < F::TPW; ++t) {
    moff[t] = (idx_of(w * F::TPW + t, col) * KP + 8 * G) * 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) soff[t][i] = cols.off + idx_of(w * F::TPW + t, i) * cols.V4;
  }
  auto state = [&](f32x4 (&x)[F::TPW]) __attribute__((always_inline)) {
    const Rsrc r = cols.rs(in);
#pragma unroll
    for (int t = 0; t < F::TPW; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[t][i] = load_one<float>(r, soff[t][i]);
  };
  int next = 0;   // the segment that is fetched next
  auto fetch = [&](Step &x) __attribute__((always_inline)) {
    const bool on = ++next < inner;   // (past the end: the last one again)
    map += on ? dm : 0;
    in += on ? ds : 0;
    const Rsrc r = rsrc_of(map, 3 * PLANE * 2);
#pragma unroll
    for (int t = 0; t < F::TPW; ++t)
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int ks = 0; ks < F::KS; ++ks)
          x.m[t][ks][p] = from_bits<bf16x8>(__builtin_bit_cast(
              uint4, __builtin_amdgcn_raw_buffer_load_b128(r, moff[t] + 64 * ks, p * PLANE * 2, 0)));
    state(x.L);
  };
  state(S);
#pragma unroll
  for (int d = 0; d + 1 < D; ++d) fetch(ahead[d]);
  // a segment; meanwhile a later one goes into the operands that the one before had
  auto step = [&](int parity, const Step &x, auto ahead_of) __attribute__((always_inline)) {
    auto &buf = parts[parity];
#pragma unroll
    for (int t = 0; t < F::TPW; ++t) {
      const int tile = w * F::TPW + t;
      uint2 s[3];
      split(S[t], s);
#pragma unroll
      for (int p = 0; p < 3; ++p) buf[tile >> 1][p][lane][tile & 1] = s[p];
    }
    __syncthreads();
    ahead_of();
    // (a chain of products for each 32 keys, step by step side by side)
    bf16x8 s[F::KS][3];
    f32x4 c[F::TPW][F::KS];
#pragma unroll
    for (int ks = 0; ks < F::KS; ++ks) {
#pragma unroll
      for (int p = 0; p < 3; ++p) s[ks][p] = from_bits<bf16x8>(*reinterpret_cast<const uint4 *>(&buf[ks][p][lane][0]));
#pragma unroll
      for (int t = 0; t < F::TPW; ++t) c[t][ks] = ks ? f32x4{0.f, 0.f, 0.f, 0.f} : x.L[t];
    }
#pragma unroll
    for (int o = 2; o >= 0; --o)
#pragma unroll
      for (int i = 0; i <= o; ++i)
#pragma unroll
        for (int ks = 0; ks < F::KS; ++ks)
#pragma unroll
          for (int t = 0; t < F::TPW; ++t)
            c[t][ks] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.m[t][ks][i], s[ks][o - i], c[t][ks], 0, 0, 0);
#pragma unroll
    for (int t = 0; t < F::TPW; ++t) {
      if constexpr (F::KS == 1) S[t] = c[t][0];
      else if constexpr (F::KS == 2) S[t] = c[t][0] + c[t][1];
      else S[t] = (c[t][0] + c[t][1]) + (c[t][2] + c[t][3]);
    }
    // (a load behind each product: in one piece they would hold up the chain)
    __builtin_amdgcn_sched_group_barrier(0x100, 3 * F::KS, 0);
#pragma unroll
    for (int i = 0; i < 6 * F::KS * F::TPW; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    out += ds;
    const Rsrc r = cols.rs(out);
#pragma unroll
    for (int t = 0; t < F::TPW; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) store_one<float>(r, soff[t][i], S[t][i]);
  };
  static_assert(D % 2 == 0, "a step's buffer is known");
  int j = 1;
  for (; j + D <= inner; j += D) {   // (no way out inside: the loads' order stays known)
#pragma unroll
    for (int d = 0; d < D; ++d)
      step((d + 1) & 1, ahead[d], [&]() __attribute__((always_inline)) { fetch(ahead[(d + D - 1) % D]); });
  }
#pragma unroll
  for (int d = 0; d + 1 < D; ++d)
    if (j + d < inner) step((d + 1) & 1, ahead[d], []() {});
}

// The fold in reverse, with M^T: one workgroup per (sequence, head, 64 columns).  A
// segment's M is staged in LDS for the four wavefronts, which read it by columns;
// the next one is in flight.
template <int KP>
__global__ __launch_bounds__(256) void delta_fold_reverse_kernel(const int64_t *__restrict__ cu, int n_seq, int n_slots,
                                                                 int64_t T, int H, int K, int V,
                                                                 int per, const uint16_t *__restrict__ seg_map,
                                                                 float *__restrict__ states) {
  constexpr int NT = KP / 16, PLANE = KP * KP, N = (3 * PLANE / 8 + 255) / 256;
  __shared__ __align__(16) uint16_t sm[3 * PLANE];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, col = lane & 15, G = lane >> 4;
  const int n_groups = (((V + 15) >> 4) + 3) >> 2;
  const int vcol = ((blockIdx.x % n_groups) * 4 + w) * 16 + col;
  const int h = static_cast<int>((blockIdx.x / n_groups) % H);
  const int64_t unit = static_cast<int64_t>(per) * kChunk, KV = static_cast<int64_t>(K) * V;
  int64_t bos, eos;
  if (!fold_rows(cu, n_seq, T, unit, n_slots, static_cast<int>(blockIdx.x / n_groups / H), bos, eos)) return;   // workgroup-uniform
  const int64_t inner = (eos - bos + unit - 1) / unit - 1;   // segments but the last
  if (inner < 2) return;   // the only state is there already
  const StateCols<NT> cols(K, V, vcol, vcol < V, G);
  auto slot = [&](int64_t j) __attribute__((always_inline)) { return (bos / unit + j) * H + h; };
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 pm[N];
  f32x4 S[NT], L[NT];
  auto fetch = [&](int64_t i) __attribute__((always_inline)) {   // step i: M of segment inner - i
    const uint16_t *m = seg_map + slot(inner - i) * (3 * PLANE);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (tid + 256 * e < 3 * PLANE / 8) pm[e] = reinterpret_cast<const u32x4 *>(m)[tid + 256 * e];
    cols.load(states + slot(inner - 1 - i) * KV, L);
  };
  cols.load(states + slot(inner - 1) * KV, S);
  fetch(1);
  for (int64_t i = 1; i < inner; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int u = tid + 256 * e, p = u / (PLANE / 8), r = u % (PLANE / 8);
      if (u < 3 * PLANE / 8)
        *reinterpret_cast<u32x4 *>(&sm[p * PLANE + sw<KP>(r / (KP / 8), (r % (KP / 8)) * 8)]) = pm[e];
    }
    bf16x8 s[NT / 2][3];
#pragma unroll
    for (int ks = 0; ks < NT / 2; ++ks) split(join(S[2 * ks], S[2 * ks + 1]), s[ks]);
#pragma unroll
    for (int t = 0; t < NT; ++t) S[t] = L[t];
    __syncthreads();
    if (i + 1 < inner) fetch(i + 1);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int ks = 0; ks < NT / 2; ++ks) {
        bf16x8 x[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) x[p] = op_cols<KP>(sm + p * PLANE, t, ks, lane);
        S[t] = mul<2>(x, s[ks], S[t]);
      }
    cols.store(states + slot(inner - 1 - i) * KV, S);
    __syncthreads();   // M is read
  }
}

// ------------------------------------------------------------------ launches --
inline dim3 grid_of(int64_t n) { return dim3(static_cast<unsigned>(n)); }
inline int v_groups(int V) { return ((V + 15) / 16 + 3) / 4; }

int check_grids(const char *what, const DeltaLayout &L, const WalkArgs &a) {
  const int64_t walk = L.seg_slots * a.H * v_groups(a.V), prep = L.chunk_slots * a.H;
  const int64_t inner = L.inner_slots * a.H * (v_groups(a.V) + L.KP / 64 + 1);
  if (std::max({prep, walk, inner, (static_cast<int64_t>(a.n_seq) * a.H + 7) * ((a.V + 15) / 16)}) > 0x7fffffff) {
    set_error("%s: too many workgroups", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  return SSLA_OK;
}

template <int DT, int KP>
void launch_chunk(const DeltaLayout &L, const WalkArgs &a, const float *g, const float *beta, bool states,
                  bool have_segs, hipStream_t st) {
  const dim3 block(256);
  hipLaunchKernelGGL((delta_prep_kernel<DT, KP>), grid_of(L.chunk_slots * a.H), block, 0, st, a.k, g, beta, a.cu, a.n_seq,
                     a.T, a.Hk, a.H, a.K, a.vec, a.mixed, a.scale, const_cast<float *>(a.tm), a.tm_floats,
                     const_cast<float *>(a.rowv));
  if (L.inner_slots > 0 && !have_segs) {
    const int groups = ((a.V + 15) / 16 + KP / 16 + 3) / 4;
    hipLaunchKernelGGL((delta_walk_kernel<DT, KP, kSegment>), grid_of(L.inner_slots * a.H * groups), block, 0, st, a);
    delta_fold(L, a, a.seg_state, false, st);
  }
  const dim3 grid = grid_of(L.seg_slots * a.H * v_groups(a.V));
  if (states) hipLaunchKernelGGL((delta_walk_kernel<DT, KP, kStates>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((delta_walk_kernel<DT, KP, kOutput>), grid, block, 0, st, a);
}

template <int DT>
void launch_keys(const DeltaLayout &L, const WalkArgs &a, const float *g, const float *beta, bool states,
                 bool have_segs, hipStream_t st) {
  switch (L.KP) {
    case 32: return launch_chunk<DT, 32>(L, a, g, beta, states, have_segs, st);
    case 64: return launch_chunk<DT, 64>(L, a, g, beta, states, have_segs, st);
    default: return launch_chunk<DT, 128>(L, a, g, beta, states, have_segs, st);
  }
}

int launch_dtype(const char *what, const DeltaLayout &L, const WalkArgs &a, const float *g, const float *beta,
                 bool states, bool have_segs, int dtype, hipStream_t st) {
  if (const int e = check_grids(what, L, a)) return e;
  if (dtype == SSLA_F32) launch_keys<SSLA_F32>(L, a, g, beta, states, have_segs, st);
  else if (dtype == SSLA_BF16) launch_keys<SSLA_BF16>(L, a, g, beta, states, have_segs, st);
  else if (dtype == SSLA_F16) launch_keys<SSLA_F16>(L, a, g, beta, states, have_segs, st);
  else {
    set_error("%s: unsupported dtype %d", what, dtype);
    return SSLA_ERR_DTYPE;
  }
  return launch_status(what);
}

}  // namespace

int delta_forward_states(const DeltaLayout &L, const WalkArgs &a, const float *g, const float *beta, bool have_segs,
                         int dtype, hipStream_t st) {
  return launch_dtype("gated_delta_chunk_bwd", L, a, g, beta, true, have_segs, dtype, st);
}

int delta_fold(const DeltaLayout &L, const WalkArgs &a, float *states, bool reverse, hipStream_t st) {
  if (L.inner_slots < 2) return launch_status("gated_delta_chunk");   // no sequence of three segments
  const int n_slots = static_cast<int>(std::min<int64_t>(L.inner_slots, 0x7fffffff));
  const int64_t units = static_cast<int64_t>(std::min(a.n_seq, n_slots)) * a.H;
  const dim3 ahead = grid_of((units + 7) / 8 * 8 * ((a.V + 15) / 16)), back = grid_of(units * v_groups(a.V));
#define SSLA_FOLD(KP_)                                                                                               \
  do {                                                                                                               \
    if (reverse)                                                                                                     \
      hipLaunchKernelGGL((delta_fold_reverse_kernel<KP_>), back, dim3(256), 0, st, a.cu, a.n_seq, n_slots, a.T, a.H, \
                         a.K, a.V, a.per, a.seg_map, states);                                                        \
    else                                                                                                             \
      hipLaunchKernelGGL((delta_fold_kernel<KP_>), ahead, dim3(64 * FoldSize<KP_>::WAVES), 0, st, a.cu, a.n_seq,     \
                         n_slots, a.T, a.H, a.K, a.V, a.per, a.seg_map, states);                                     \
  } while (0)
  if (L.KP == 32) SSLA_FOLD(32);
  else if (L.KP == 64) SSLA_FOLD(64);
  else SSLA_FOLD(128);
#undef SSLA_FOLD
  return launch_status("gated_delta_chunk");
}

}  // namespace ssla

extern "C" size_t ssla_gated_delta_chunk_workspace_size(int n_seq, int64_t T, int H, int K, int V) {
  if (n_seq < 0 || T < 0 || H <= 0 || K <= 0 || K > 128 || V <= 0) return 0;
  return ssla::delta_layout(n_seq, T, H, H, K, V, false).total;
}

extern "C" size_t ssla_gated_delta_chunk_segments_size(int n_seq, int64_t T, int H, int K, int V) {
  if (n_seq < 0 || T < 0 || H <= 0 || K <= 0 || K > 128 || V <= 0) return 0;
  return ssla::delta_layout(n_seq, T, H, H, K, V, false).seg_bytes;
}

namespace ssla {
namespace {

// Rows too wide for the chunk kernels' offsets, but not for a token's.
bool tokens_alone(int H, int K, int V) { return check_widths("gated_delta_mixed_fwd", kChunk, 1, H, K, V) != SSLA_OK; }

}  // namespace
}  // namespace ssla

extern "C" size_t ssla_gated_delta_mixed_workspace_size(int64_t T, int H, int K, int V) {
  if (T < 0 || H <= 0 || K <= 0 || K > 128 || V <= 0 || ssla::tokens_alone(H, K, V)) return 0;
  return ssla::delta_layout(1, T, H, H, K, V, false, true).total;
}

namespace ssla {
namespace {

// mixed: up to kChunk rows token by token, longer sequences by chunks, both kinds of
// kernels over the whole batch (a workgroup whose sequence is the other kind's
// ends after its search).  Measured, 4 heads, bf16: a prompt of 15,900 rows among 512
// single rows 84 us at K = 32, 149 at 64 and 466 at 128 (all token by token 3,684,
// 5,002 and 10,675, all by chunks 104, 235 and 457); without a long one the empty
// launches are added to the tokens' time: 4,096 sequences of 16 rows 68 -> 98 us at K =
// 32 and 274 -> 296 at 64 (by chunks 347 and 415), 32 of 20 rows 13 -> 25 (20).
int chunk_fwd(const char *what, bool mixed, const void *q, const void *k, const void *v, const float *g, const float *beta,
              const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk, int H, int K, int V, float scale, const float *h0,
              void *o, float *ht, void *segments, int dtype, void *workspace, size_t workspace_bytes, hipStream_t st) {
  clear_error();
  SSLA_CHECK_ARG(n_seq >= 0 && T >= 0 && Hk > 0 && H > 0 && H % Hk == 0 && K > 0 && V > 0,
                 "%s: bad sizes n_seq=%d T=%lld Hk=%d H=%d K=%d V=%d", what, n_seq, (long long)T, Hk, H, K, V);
  if (K > 128) {
    set_error("%s: K=%d exceeds 128", what, K);
    return SSLA_ERR_UNSUPPORTED;
  }
  if (n_seq == 0) return SSLA_OK;
  SSLA_CHECK_ARG(cu_seqlens != nullptr, "%s: cu_seqlens is NULL", what);
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta && o), "%s: null tensor pointer", what);
  if (mixed && tokens_alone(H, K, V)) {
    clear_error();
    if (const int e = check_widths(what, 16, Hk, H, K, V)) return e;
    return delta_recurrent_up_to(what, INT64_MAX, q, k, v, g, beta, cu_seqlens, n_seq, T, Hk, H, K, V, scale, h0, o, ht,
                                 nullptr, 0, nullptr, dtype, st);
  }
  if (const int e = check_widths(what, kChunk, Hk, H, K, V)) return e;
  const DeltaLayout L = delta_layout(n_seq, T, Hk, H, K, V, false, mixed);
  if (!workspace || workspace_bytes < L.total || !aligned(workspace, 16)) {
    set_error("%s: needs %zu bytes of workspace, got %zu", what, L.total, workspace_bytes);
    return SSLA_ERR_WORKSPACE;
  }
  SSLA_CHECK_ARG(aligned(segments, 16), "%s: segments must be 16-byte aligned", what);
  WalkArgs a = walk_args(L, static_cast<char *>(workspace), q, k, v, cu_seqlens, n_seq, T, Hk, H, K, V, scale, h0, dtype,
                         false, segments);
  a.o = o;
  a.ht = ht;
  a.mixed = mixed;
  if (mixed) {
    if (const int e = check_grids(what, L, a)) return e;
    if (const int e = delta_recurrent_up_to(what, kChunk, q, k, v, g, beta, cu_seqlens, n_seq, T, Hk, H, K, V, scale, h0, o,
                                            ht, nullptr, 0, nullptr, dtype, st))
      return e;
    if (T <= kChunk) return SSLA_OK;   // no longer sequence
  }
  return launch_dtype(what, L, a, g, beta, false, false, dtype, st);
}

}  // namespace
}  // namespace ssla

extern "C" int ssla_gated_delta_chunk_fwd(const void *q, const void *k, const void *v, const float *g,
                                          const float *beta, const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk,
                                          int H, int K, int V, float scale, const float *h0, void *o, float *ht,
                                          void *segments, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  return ssla::chunk_fwd("gated_delta_chunk_fwd", false, q, k, v, g, beta, cu_seqlens, n_seq, T, Hk, H, K, V, scale, h0, o,
                         ht, segments, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int ssla_gated_delta_mixed_fwd(const void *q, const void *k, const void *v, const float *g,
                                          const float *beta, const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk,
                                          int H, int K, int V, float scale, const float *h0, void *o, float *ht, int dtype,
                                          void *workspace, size_t workspace_bytes, void *stream) {
  return ssla::chunk_fwd("gated_delta_mixed_fwd", true, q, k, v, g, beta, cu_seqlens, n_seq, T, Hk, H, K, V, scale, h0, o,
                         ht, nullptr, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

// Chunked gated delta rule, backward, on gfx950.
//
// Notation of delta_chunk.hip; do the gradient of o, D that of the state
// leaving a chunk, S the state entering it.  Per chunk
//   du = P^T do + e^(G_last - G) (k D),   dX = Tm^T du,   dv = beta dX,
//   D' = e^(G_last) D + q^T (scale e^G do) - k^T (beta e^G dX)
// (D' leaves the chunk before).  Each column of D goes its own way, so this is
// the forward's walk in reverse over the same segments: over a segment the
// gradient goes through D -> M^T D + L with the forward's M, so only L is walked
// for (the last segment's from the final state's gradient), then folded.  With the products' factors known for every chunk,
//   dP_ij = scale e^(G_i - G_j) do_i . u_j (j <= i),
//   dN_ij = -e^(G_i - G_j) dX_i . u_j (j < i),
//   dq = scale e^G (do S^T) + dP k,
//   dk = dP^T q + beta (dN k) + (beta dN)^T k - beta e^G (dX S^T)
//        + e^(G_last - G) (u D^T),
//   dbeta_i = dX_i . v_i - e^(G_i) k_i . (S dX_i) + k_i . (dN k)_i
// for all chunks side by side.  A gate's gradient is the sum over everything its
// step scales: the terms between rows i >= t > j of dP and dN, from the state to
// rows i >= t, from rows j < t to the next state, and from state to state.  Row
// and column sums of the first kind are dot products of the rows of q and k with
// the pieces of dq and dk, so no second Gram matrix is formed.
// Measured at 8 sequences of 4096 rows, 8 heads of 64, bf16: reverse segments 59
// us, fold 16, reverse walk 81, chunk gradients 158 (495 MB, 3.1 TB/s: bound by the
// loads of u, dX, S and D between barriers, VALU busy 51 % and matrix cores 22 % of
// the time at four wavefronts a SIMD; 167 at two, where every wavefront had both
// sides of its rows and the next loads in flight).
// Shared key heads: every value head's dq and dk in fp32, added in the order of
// the heads.
#include "delta_tile.h"
#include "seq_slots.h"

namespace ssla {
namespace {

struct GradArgs {
  WalkArgs w;
  const void *dout;
  const float *dht;
  float *seg_grad;     // per inner segment: after the fold the gradient leaving it
  float *chunk_grad;   // per chunk: D
  float *dx;           // [T, H, V]
  void *dq, *dk, *dv;
  float *dq_part, *dk_part;   // [T, H, K] where key heads are shared
  float *dg, *dbeta, *dh0;
  int vvec, dvec;
};

// Operand set of row tile t, contraction half ks (>= t / 2), of an upper triangular matrix.
__device__ __forceinline__ constexpr int upper_set(int t, int ks) { return t < 2 ? 2 * t + ks : t + 2; }

template <int DT, int KP>
struct ReverseSmem {
  static constexpr int NP = Parts<DT>::n;
  uint16_t k[NP][kChunk * KP];
  uint16_t q[NP][kChunk * KP];
  uint16_t tm[3][kTriSets * 512];
  uint16_t p[3][kTriSets * 512];
  float rowv[kRowVecs][kChunk];
};

// SEG: a segment with a predecessor from zero (a sequence's last from dht): what it
// adds to the gradient leaving that predecessor.  Otherwise: a segment from the gradient leaving
// it; writes every chunk's D and dX, dv, and dh0 before the sequence's first row.
template <int DT, int KP, bool SEG>
__global__ __launch_bounds__(256, (DT == SSLA_F32 && KP == 128) ? 1 : 2) void delta_reverse_kernel(const GradArgs ga) {
  constexpr int NP = Parts<DT>::n, NT = KP / 16;
  typedef Elem<DT> E;
  typedef typename E::T ET;
  const WalkArgs &a = ga.w;
  __shared__ __align__(16) ReverseSmem<DT, KP> sm;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, G = lane >> 4;
  const int n_vt = (a.V + 15) >> 4, n_groups = (n_vt + 3) >> 2;
  int64_t b = blockIdx.x;
  const int grp = static_cast<int>(b % n_groups);
  b /= n_groups;
  const int h = static_cast<int>(b % a.H), hk = h / (a.H / a.Hk);
  const int64_t slot = b / a.H;
  const int64_t unit = static_cast<int64_t>(a.per) * kChunk;
  int n;
  int64_t bos, eos, first;
  if (!seq_of_slot<!SEG>(a.cu, a.n_seq, a.T, unit, slot, n, bos, eos, first)) return;   // workgroup-uniform
  const int64_t seg = slot - first + (SEG ? 1 : 0), t_begin = bos + seg * unit;
  if (t_begin >= eos && seg > 0) return;
  const int64_t t_end = min(t_begin + unit, eos);
  const int tile = grp * 4 + w;
  const int vcol = tile * 16 + col;
  const bool v_ok = vcol < a.V;
  const int64_t KV = static_cast<int64_t>(a.K) * a.V;

  const StateCols<NT> cols(a.K, a.V, vcol, v_ok, G);
  f32x4 D[NT];
  cols.load(t_end < eos ? (SEG ? nullptr : ga.seg_grad + ((bos / unit + seg) * a.H + h) * KV)
            : ga.dht    ? ga.dht + (static_cast<int64_t>(n) * a.H + h) * KV : nullptr, D);
  // byte offset of row 8 G in this lane's column of do and dv, and of dX (4 bytes)
  constexpr int ES = sizeof(ET);
  const uint32_t vrow = static_cast<uint32_t>(a.H) * a.V;
  const uint32_t voff = v_ok ? (8 * G * vrow + vcol) * ES : kOutside, xoff = v_ok ? (8 * G * vrow + vcol) * 4 : kOutside;

  RowTile<DT, KP> kt, qt;
  f32x4 tmr[3], rvr;
  ET dr[16];
  // (a chunk before the segment: resources of no bytes, zeros and no traffic)
  auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
    const int rows = t0 >= t_begin ? static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0)) : 0;
    const int64_t at = (t0 * a.Hk + hk) * a.K;
    const int stride = a.Hk * a.K;
    kt.fetch(rows_rsrc(a.k, at, rows, stride, a.K, ES), stride, a.K, a.vec);
    qt.fetch(rows_rsrc(a.q, at, rows, stride, a.K, ES), stride, a.K, a.vec);
    const int64_t c = chunk_slot(bos, n, (t0 - bos) / kChunk) * a.H + h;
    const Rsrc rt = rsrc_of(a.tm + c * a.tm_floats + kTriFloats, rows > 0 ? kTriFloats * 4 : 0);
    const Rsrc rr = rsrc_of(a.rowv + c * kRowFloats, rows > 0 ? kRowFloats * 4 : 0);
    tmr[0] = load4(rt, tid * 32);
    tmr[1] = load4(rt, tid * 32 + 16);
    tmr[2] = load4(rt, 8192 + tid * 16);
    rvr = load4(rr, tid * 16);   // (96 threads' worth)
    const Rsrc rd = rows_rsrc(ga.dout, (t0 * a.H + h) * a.V, rows, vrow, a.V, ES);
#pragma unroll
    for (int i = 0; i < 16; ++i) dr[i] = load_one<ET>(rd, voff + idx_of(i >> 2, i & 3) * vrow * ES);
  };
  auto stage = [&]() __attribute__((always_inline)) {
    kt.store(&sm.k[0][0], kChunk * KP);
    qt.store(&sm.q[0][0], kChunk * KP);
    bf16x8 s[3];
    split(join(tmr[0], tmr[1]), s);   // sets 0 .. 3: a lane's eight values of one thread
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4 *>(&sm.tm[i][tid * 8]) = to_bits(s[i]);
    uint2 half[3];
    split(tmr[2], half);   // sets 4, 5: half a lane's values
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2 *>(&sm.tm[i][2048 + tid * 4]) = half[i];
    if (tid < kRowFloats / 4) reinterpret_cast<f32x4 *>(&sm.rowv[0][0])[tid] = rvr;
  };
  auto row8 = [&](int vec, int p) __attribute__((always_inline)) {
    const f32x4 *s = reinterpret_cast<const f32x4 *>(&sm.rowv[vec][32 * p + 8 * G]);
    return join(s[0], s[1]);
  };
  auto set_of = [&](const uint16_t (&m)[3][kTriSets * 512], int set, bf16x8 (&x)[3]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 3; ++j) x[j] = from_bits<bf16x8>(*reinterpret_cast<const uint4 *>(&m[j][(set * 64 + lane) * 8]));
  };

  const int64_t n_chunks = (t_end - t_begin + kChunk - 1) / kChunk;
  if (n_chunks > 0) fetch(t_begin + (n_chunks - 1) * kChunk);
  for (int64_t c = n_chunks - 1; c >= 0; --c) {
    const int64_t t0 = t_begin + c * kChunk;
    stage();
    f32x8 dov[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) dov[i >> 3][i & 7] = of_elem<DT>(dr[i]);
    if constexpr (!SEG)
      cols.store(ga.chunk_grad + (chunk_slot(bos, n, (t0 - bos) / kChunk) * a.H + h) * KV, D);
    __syncthreads();

    {   // P^T of this wavefront's row tile (rows j): q k^T has row i of P in the lanes that the operand needs
      const int j = idx_of(w, col);
      const float hi = sm.rowv[kGHi][j], lo = sm.rowv[kGLo][j];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks < (w >> 1)) continue;
        f32x4 d[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kk = 0; kk < KP / 32; ++kk) {
          bf16x8 kb[NP];
#pragma unroll
          for (int i = 0; i < NP; ++i) kb[i] = op_rows<KP>(sm.k[i], w, kk, lane);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            bf16x8 qa[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) qa[i] = op_rows<KP>(sm.q[i], 2 * ks + x, kk, lane);
            d[x] = mul<2>(qa, kb, d[x]);
          }
        }
        f32x8 pv = join(d[0], d[1]);
        const f32x8 ghi = row8(kGHi, ks), glo = row8(kGLo, ks);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          pv[i] = keep(32 * ks + 8 * G + i >= j, a.scale * pv[i] * fast_exp2((ghi[i] - hi) + (glo[i] - lo)));
        bf16x8 s[3];
        split(pv, s);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          *reinterpret_cast<uint4 *>(&sm.p[i][(upper_set(w, ks) * 64 + lane) * 8]) = to_bits(s[i]);
      }
    }

    f32x4 u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) u[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KP / 32; ++ks) {
      bf16x8 s[3];
      split(join(D[2 * ks], D[2 * ks + 1]), s);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        bf16x8 x[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) x[j] = op_rows<KP>(sm.k[j], t, ks, lane);
        u[t] = mul<2>(x, s, u[t]);
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const f32x8 el = row8(kToEnd, p);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        u[2 * p][r] *= el[r];
        u[2 * p + 1][r] *= el[4 + r];
      }
    }
    {
      bf16x8 d[2][NP];
#pragma unroll
      for (int p = 0; p < 2; ++p) split(dov[p], d[p]);
      __syncthreads();   // P^T is written
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ks = t / 2; ks < 2; ++ks) {
          bf16x8 m[3];
          set_of(sm.p, upper_set(t, ks), m);
          u[t] = mul<2>(m, d[ks], u[t]);
        }
    }
    f32x8 dX[2];
    {
      bf16x8 x[2][3];
#pragma unroll
      for (int p = 0; p < 2; ++p) split(join(u[2 * p], u[2 * p + 1]), x[p]);
      f32x4 y[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        y[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = t / 2; ks < 2; ++ks) {
          bf16x8 m[3];
          set_of(sm.tm, upper_set(t, ks), m);
          y[t] = mul<2>(m, x[ks], y[t]);
        }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) dX[p] = join(y[2 * p], y[2 * p + 1]);
    }
    if constexpr (!SEG) {
      const int rows = static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0));
      const int64_t at = (t0 * a.H + h) * a.V;
      const Rsrc rv = rows_rsrc(ga.dv, at, rows, vrow, a.V, ES), rx = rows_rsrc(ga.dx, at, rows, vrow, a.V, 4);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const f32x8 dv = row8(kBeta, p) * dX[p];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          store_one<float>(rx, xoff + (32 * p + i) * vrow * 4, dX[p][i]);
          store_one<ET>(rv, voff + (32 * p + i) * vrow * ES, to_elem<DT>(dv[i]));
        }
      }
    }
    fetch(t0 - kChunk);   // the next chunk's, in flight meanwhile (here: fewer values are live)

    // D <- e^(G_last) D + q^T (scale e^G do) - k^T (beta e^G dX)
    bf16x8 x1[2][3], x2[2][3];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      split(row8(kScaleG, p) * dov[p], x1[p]);
      split(-row8(kBetaG, p) * dX[p], x2[p]);
    }
    const float through = fast_exp2(sm.rowv[kGHi][kChunk - 1]) * fast_exp2(sm.rowv[kGLo][kChunk - 1]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      D[t] *= through;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8 x[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) x[j] = op_cols<KP>(sm.q[j], t, ks, lane);
        D[t] = mul<2>(x, x1[ks], D[t]);
#pragma unroll
        for (int j = 0; j < NP; ++j) x[j] = op_cols<KP>(sm.k[j], t, ks, lane);
        D[t] = mul<2>(x, x2[ks], D[t]);
      }
    }
    __syncthreads();   // the chunk's tiles are read
  }

  if (!SEG) {
    if (ga.dh0 && seg == 0) cols.store(ga.dh0 + (static_cast<int64_t>(n) * a.H + h) * KV, D);
  } else {
    cols.store(ga.seg_grad + (slot * a.H + h) * KV, D);
  }
}

// ------------------------------------------------------ the chunks' gradients --
// 64 rows of 32 columns, four columns for each of 512 threads.
template <int DT>
struct ColTile {
  typedef typename Elem<DT>::T E;
  static constexpr int ES = sizeof(E);
  struct Piece { E e[4]; };
  Piece p;

  __device__ __forceinline__ void fetch(const Rsrc &rs, int thread, int stride, int n_cols, bool vec) {
    const int row = thread >> 3, col = (thread & 7) * 4;
    const uint32_t at = static_cast<uint32_t>(row * stride + col) * ES;
    if (vec) {
      const uint32_t off = col + 4 <= n_cols ? at : kOutside;
      if constexpr (ES == 2) p = __builtin_bit_cast(Piece, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
      else p = __builtin_bit_cast(Piece, load4(rs, off));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) p.e[j] = load_one<E>(rs, col + j < n_cols ? at + ES * j : kOutside);
    }
  }
  __device__ __forceinline__ float value(int j) const { return of_elem<DT>(p.e[j]); }
  // plane j at t + j * stride elements
  __device__ __forceinline__ void store(uint16_t *t, int stride) const {
    uint16_t *dst = t + sw<32>(threadIdx.x >> 3, (threadIdx.x & 7) * 4);
    if constexpr (DT == SSLA_BF16) {
      *reinterpret_cast<uint2 *>(dst) = __builtin_bit_cast(uint2, p);
    } else {
      uint2 w[Parts<DT>::n];
      split(f32x4{value(0), value(1), value(2), value(3)}, w);
#pragma unroll
      for (int j = 0; j < Parts<DT>::n; ++j) *reinterpret_cast<uint2 *>(dst + j * stride) = w[j];
    }
  }
};

template <int DT, int KP>
struct GradSmem {
  static constexpr int NP = Parts<DT>::n, KR = KP < 64 ? 64 : KP;
  struct Values {   // 32 value columns at a time
    uint16_t dout[NP][kChunk * 32], u[3][kChunk * 32], dx[3][kChunk * 32], S[3][KR * 32], D[3][KR * 32];
  };
  struct Keys {
    uint16_t q[NP][kChunk * KP], k[NP][kChunk * KP];
  };
  struct Pass {   // what the rows' wavefronts add to dk
    f32x4 dk[KP / 16][256];
  };
  // side by side where two workgroups a CU still fit: q and k then come with the first columns
  static constexpr bool kApart = std::max(sizeof(Values), sizeof(Pass)) + sizeof(Keys) <= 76 * 1024;
  union Front { Values v; Pass x; };
  struct Apart { Front f; Keys k; };
  struct Behind { Pass x; Keys k; };
  union Over { Values v; Behind b; };
  std::conditional_t<kApart, Apart, Over> m;
  float rowv[kRowVecs][kChunk];
  float base[2][kChunk], to_next[kChunk], dxv[kChunk], db[kChunk], eg[kChunk];
  float sd[8];
  __device__ __forceinline__ Values &values() {
    if constexpr (kApart) return m.f.v;
    else return m.v;
  }
  __device__ __forceinline__ Keys &keys() {
    if constexpr (kApart) return m.k;
    else return m.b.k;
  }
  __device__ __forceinline__ Pass &pass() {
    if constexpr (kApart) return m.f.x;
    else return m.b.x;
  }
};

// One workgroup per (chunk slot, head), two wavefronts per row tile w: one has what
// the rows i of the tile read (do, dX with S and the rows before: dq), one what the
// rows j write (u with D and the rows behind: dk, to which the first adds its dN k
// and dX S^T).
template <int DT, int KP>
__global__ __launch_bounds__(512, KP == 128 ? 2 : 4) void delta_grad_kernel(const GradArgs ga) {
  constexpr int NP = Parts<DT>::n, KT = KP / 16;
  typedef Elem<DT> E;
  typedef typename E::T ET;
  const WalkArgs &a = ga.w;
  typedef GradSmem<DT, KP> Smem;
  __shared__ __align__(16) Smem sm;
  typename Smem::Values &sv = sm.values();
  typename Smem::Keys &sk = sm.keys();
  const int tid = threadIdx.x, lane = tid & 63, w8 = __builtin_amdgcn_readfirstlane(tid >> 6), w = w8 & 3;
  const bool reads = w8 < 4;
  const int col = lane & 15, G = lane >> 4;
  const int h = static_cast<int>(blockIdx.x % a.H), hk = h / (a.H / a.Hk);
  const int64_t slot = blockIdx.x / a.H;
  int n;
  int64_t bos, eos, first;
  if (!seq_of_slot(a.cu, a.n_seq, a.T, kChunk, slot, n, bos, eos, first)) return;   // workgroup-uniform
  const int64_t t0 = bos + (slot - first) * kChunk;
  if (t0 >= eos) return;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kChunk), eos - t0));
  const int64_t KV = static_cast<int64_t>(a.K) * a.V;
  const float *Sp = a.chunk_state + (slot * a.H + h) * KV, *Dp = ga.chunk_grad + (slot * a.H + h) * KV;
  const int64_t vat = (t0 * a.H + h) * a.V;
  const int vrow = a.H * a.V;
  constexpr int ES = sizeof(ET);

  const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
  float dxv = 0.f, sd = 0.f;
  const int pair = w >> 1;
  auto keys = [&]() __attribute__((always_inline)) {   // the first four wavefronts q, the others k
    RowTile<DT, KP> x;
    const int64_t at = (t0 * a.Hk + hk) * a.K;
    const int stride = a.Hk * a.K;
    x.fetch(rows_rsrc(reads ? a.q : a.k, at, rows, stride, a.K, ES), stride, a.K, a.vec);
    x.store(reads ? &sk.q[0][0] : &sk.k[0][0], kChunk * KP);
  };
  if (tid < kRowFloats / 4)
    reinterpret_cast<f32x4 *>(&sm.rowv[0][0])[tid] =
        reinterpret_cast<const f32x4 *>(a.rowv + (slot * a.H + h) * kRowFloats)[tid];
  if (Smem::kApart) keys();
  // 32 value columns: the values' rows, and the states' (64 keys a tile)
  constexpr int KH = (KP + 63) / 64, KR = Smem::KR;
  auto columns = [&](int c0) __attribute__((always_inline)) {
    const int nc = a.V - c0;
    int thread = tid;   // (taken anew: offsets kept over the loop would cost a wavefront's registers)
    asm volatile("" : "+v"(thread));
    ColTile<DT> dt, vt;
    ColTile<SSLA_F32> ut, xt, st[KH], gt[KH];
    dt.fetch(rows_rsrc(ga.dout, vat + c0, rows, vrow, nc, ES), thread, vrow, nc, ga.dvec);
    vt.fetch(rows_rsrc(a.v, vat + c0, rows, vrow, nc, ES), thread, vrow, nc, ga.dvec);
    ut.fetch(rows_rsrc(a.u, vat + c0, rows, vrow, nc, 4), thread, vrow, nc, ga.vvec);
    xt.fetch(rows_rsrc(ga.dx, vat + c0, rows, vrow, nc, 4), thread, vrow, nc, ga.vvec);
#pragma unroll
    for (int i = 0; i < KH; ++i) {
      const int64_t at = static_cast<int64_t>(64 * i) * a.V + c0;
      st[i].fetch(rows_rsrc(Sp, at, a.K - 64 * i, a.V, nc, 4), thread, a.V, nc, ga.vvec);
      gt[i].fetch(rows_rsrc(Dp, at, a.K - 64 * i, a.V, nc, 4), thread, a.V, nc, ga.vvec);
    }
    __syncthreads();   // the columns before are read
    dt.store(&sv.dout[0][0], kChunk * 32);
    ut.store(&sv.u[0][0], kChunk * 32);
    xt.store(&sv.dx[0][0], kChunk * 32);
#pragma unroll
    for (int j = 0; j < 4; ++j) dxv = fmaf(vt.value(j), xt.value(j), dxv);
#pragma unroll
    for (int i = 0; i < KH; ++i) {
      st[i].store(&sv.S[0][64 * i * 32], KR * 32);
      gt[i].store(&sv.D[0][64 * i * 32], KR * 32);
#pragma unroll
      for (int j = 0; j < 4; ++j) sd = fmaf(st[i].value(j), gt[i].value(j), sd);
    }
    __syncthreads();
  };
  auto behind_columns = [&]() __attribute__((always_inline)) {
    __syncthreads();   // the last columns are read
    if (!Smem::kApart) keys();
    dxv += __shfl_xor(dxv, 1);
    dxv += __shfl_xor(dxv, 2);
    dxv += __shfl_xor(dxv, 4);
    if ((tid & 7) == 0) sm.dxv[tid >> 3] = dxv;
#pragma unroll
    for (int d = 32; d; d >>= 1) sd += __shfl_xor(sd, d);
    if (lane == 0) sm.sd[w8] = sd;
    if (w8 == 7) sm.eg[lane] = fast_exp2(sm.rowv[kGHi][lane]) * fast_exp2(sm.rowv[kGLo][lane]);
    __syncthreads();
  };
  auto row8 = [&](int vec, int p) __attribute__((always_inline)) {
    const f32x4 *s = reinterpret_cast<const f32x4 *>(&sm.rowv[vec][32 * p + 8 * G]);
    return join(s[0], s[1]);
  };
  const bool part = ga.dq_part != nullptr;   // every value head's in fp32
  const int krow = (part ? a.H : a.Hk) * a.K, GS = part ? 4 : ES;
  const int64_t kat = part ? (t0 * a.H + h) * a.K : (t0 * a.Hk + hk) * a.K;
  const Rsrc rs = rows_rsrc(reads ? (part ? static_cast<const void *>(ga.dq_part) : ga.dq)
                                  : (part ? static_cast<const void *>(ga.dk_part) : ga.dk),
                            kat, rows, krow, a.K, GS);
  const int row0 = idx_of(w, 4 * G), me = idx_of(w, col);   // own rows row0 .. + 3 in accumulators, own row in operands
  auto put = [&](int t, const f32x4 &x) __attribute__((always_inline)) {
    const int key = idx_of(t, col);
    const uint32_t off = key < a.K ? static_cast<uint32_t>(row0 * krow + key) * GS : kOutside;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (part) store_one<float>(rs, off + r * krow * 4, x[r]);
      else store_one<ET>(rs, off + r * krow * ES, to_elem<DT>(x[r]));
    }
  };
  // own rows of the column operands of half `pair`: elements 4 (w & 1) .. + 3
  auto own = [&](const bf16x8 (&x)[NP]) __attribute__((always_inline)) {
    f32x4 y = zero;
#pragma unroll
    for (int j = NP - 1; j >= 0; --j) {
      const uint4 u = to_bits(x[j]);
      const uint32_t lo = w & 1 ? u.z : u.x, hi = w & 1 ? u.w : u.y;
      y += f32x4{__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16),
                 __uint_as_float(hi & 0xffff0000u)};
    }
    return y;
  };
  // (each kind of wavefronts runs its own loop, with as many barriers as the other's)
  if (reads) {
    f32x4 A1[KT], A2[KT], C1[4], C2[4];   // do S^T, dX S^T; u do^T, u dX^T of the row tiles up to the own one's pair
#pragma unroll
    for (int i = 0; i < KT; ++i) A1[i] = A2[i] = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) C1[i] = C2[i] = zero;
    for (int c0 = 0; c0 < a.V; c0 += 32) {
      columns(c0);
      bf16x8 od[NP], ox[3];   // this wavefront's rows of do, dX
#pragma unroll
      for (int i = 0; i < NP; ++i) od[i] = op_rows<32>(sv.dout[i], w, 0, lane);
#pragma unroll
      for (int i = 0; i < 3; ++i) ox[i] = op_rows<32>(sv.dx[i], w, 0, lane);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 s[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] = op_rows<32>(sv.S[i], t, 0, lane);
        A1[t] = mul<2>(od, s, A1[t]);
        A2[t] = mul<2>(ox, s, A2[t]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if ((t >> 1) > pair) continue;
        bf16x8 x[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) x[i] = op_rows<32>(sv.u[i], t, 0, lane);
        C1[t] = mul<2>(x, od, C1[t]);
        C2[t] = mul<2>(x, ox, C2[t]);
      }
    }
    behind_columns();
    const f32x4 bt4 = *reinterpret_cast<const f32x4 *>(&sm.rowv[kBeta][row0]);
    const float mhi = sm.rowv[kGHi][me], mlo = sm.rowv[kGLo][me];
    // dP, dN with this wavefront's rows i in the lanes (contraction j <= i), one
    // after the other: parts of both would take more registers than there are
    f32x8 n1[2];
    bf16x8 p[2][3];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks > pair) continue;
      const f32x8 ghi = row8(kGHi, ks), glo = row8(kGLo, ks);
      f32x8 p1 = join(C1[2 * ks], C1[2 * ks + 1]);
      n1[ks] = join(C2[2 * ks], C2[2 * ks + 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 32 * ks + 8 * G + j;
        const float e = fast_exp2((mhi - ghi[j]) + (mlo - glo[j]));
        p1[j] = keep(r <= me, a.scale * p1[j] * e);
        n1[ks][j] = keep(r < me, -n1[ks][j] * e);
      }
      split(p1, p[ks]);
    }
    // per own row: q . dq, k . (dN k), k . (dX S^T)
    f32x4 qa = zero, kd = zero, ky = zero;
    {
      const f32x4 sg = *reinterpret_cast<const f32x4 *>(&sm.rowv[kScaleG][row0]);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        f32x4 b = zero, qv = zero;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          if (ks > pair) continue;
          bf16x8 x[NP];
#pragma unroll
          for (int i = 0; i < NP; ++i) x[i] = op_cols<KP>(sk.k[i], t, ks, lane);
          b = mul<2>(p[ks], x, b);
          if (ks == pair) {
#pragma unroll
            for (int i = 0; i < NP; ++i) x[i] = op_cols<KP>(sk.q[i], t, ks, lane);
            qv = own(x);
          }
        }
        b += sg * A1[t];
        qa += qv * b;
        put(t, b);
      }
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      if (ks <= pair) split(n1[ks], p[ks]);
    const f32x4 bg = *reinterpret_cast<const f32x4 *>(&sm.rowv[kBetaG][row0]);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      f32x4 d = zero, kv = zero;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks > pair) continue;
        bf16x8 x[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = op_cols<KP>(sk.k[i], t, ks, lane);
        d = mul<2>(p[ks], x, d);
        if (ks == pair) kv = own(x);
      }
      kd += kv * d;
      ky += kv * A2[t];
      sm.pass().dk[t][tid] = bt4 * d - bg * A2[t];
    }
    const f32x4 eg = *reinterpret_cast<const f32x4 *>(&sm.eg[row0]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {   // the keys' sums, of what the row needs
      const float base = row_sum((qa[r] - bg[r] * ky[r]) + bt4[r] * kd[r]);
      const float db = row_sum(fmaf(-eg[r], ky[r], kd[r]));
      if (col == 0) {
        sm.base[0][row0 + r] = base;
        sm.db[row0 + r] = db;
      }
    }
    __syncthreads();
  } else {
    f32x4 A1[KT], C1[4], C2[4];   // u D^T; do u^T, dX u^T of the row tiles from the own one's pair on
#pragma unroll
    for (int i = 0; i < KT; ++i) A1[i] = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) C1[i] = C2[i] = zero;
    for (int c0 = 0; c0 < a.V; c0 += 32) {
      columns(c0);
      bf16x8 ou[3];   // this wavefront's rows of u
#pragma unroll
      for (int i = 0; i < 3; ++i) ou[i] = op_rows<32>(sv.u[i], w, 0, lane);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 s[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] = op_rows<32>(sv.D[i], t, 0, lane);
        A1[t] = mul<2>(ou, s, A1[t]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if ((t >> 1) < pair) continue;
        bf16x8 x[3], y[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) y[i] = op_rows<32>(sv.dout[i], t, 0, lane);
        C1[t] = mul<2>(y, ou, C1[t]);
#pragma unroll
        for (int i = 0; i < 3; ++i) x[i] = op_rows<32>(sv.dx[i], t, 0, lane);
        C2[t] = mul<2>(x, ou, C2[t]);
      }
    }
    behind_columns();
    const float mhi = sm.rowv[kGHi][me], mlo = sm.rowv[kGLo][me];
    bf16x8 p[2][3], m[2][3];
    // dP^T, dN^T with the own rows j in the lanes (contraction i >= j)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks < pair) continue;
      const f32x8 ghi = row8(kGHi, ks), glo = row8(kGLo, ks), bt = row8(kBeta, ks);
      f32x8 p2 = join(C1[2 * ks], C1[2 * ks + 1]), n2 = join(C2[2 * ks], C2[2 * ks + 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 32 * ks + 8 * G + j;
        const float e = fast_exp2((ghi[j] - mhi) + (glo[j] - mlo));
        p2[j] = keep(r >= me, a.scale * p2[j] * e);
        n2[j] = keep(r > me, -bt[j] * n2[j] * e);
      }
      split(p2, p[ks]);
      split(n2, m[ks]);
    }
    const f32x4 te = *reinterpret_cast<const f32x4 *>(&sm.rowv[kToEnd][row0]);
    // per own row: k . (dP^T q + (beta dN)^T k), k . (u D^T)
    f32x4 kc = zero, kw = zero;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      f32x4 c = zero, e = zero, kv = zero;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks < pair) continue;
        bf16x8 x[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = op_cols<KP>(sk.k[i], t, ks, lane);
        e = mul<2>(m[ks], x, e);
        if (ks == pair) kv = own(x);
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = op_cols<KP>(sk.q[i], t, ks, lane);
        c = mul<2>(p[ks], x, c);
      }
      const f32x4 hw = te * A1[t];
      c += e;
      kc += kv * c;
      kw += kv * hw;
      A1[t] = hw + c;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float base = row_sum(-kc[r]), next = row_sum(kw[r]);
      if (col == 0) {
        sm.base[1][row0 + r] = base;
        sm.to_next[row0 + r] = next;
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < KT; ++t) put(t, sm.pass().dk[t][tid - 256] + A1[t]);
  }
  if (w8 == 0) {
    // dg_t = sum_(i >= t) base_i + sum_(j < t) to_next_j + e^(G_last) <S, D>
    float s = sm.base[0][lane] + sm.base[1][lane], p = sm.to_next[lane];
    const float mine = p;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const float down = __shfl_down(s, d), up = __shfl_up(p, d);
      if (lane + d < 64) s += down;
      if (lane >= d) p += up;
    }
    float sdt = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sdt += sm.sd[i];
    if (lane < rows) {
      ga.dg[(t0 + lane) * a.H + h] = s + fmaf(sm.eg[kChunk - 1], sdt, p - mine);
      ga.dbeta[(t0 + lane) * a.H + h] = sm.dxv[lane] + sm.db[lane];
    }
  }
}

// dq, dk of the key heads: their value heads' in order.
template <int DT>
__global__ __launch_bounds__(256) void delta_heads_kernel(const int64_t *__restrict__ cu, int n_seq, int64_t T, int Hk,
                                                          int rep, int K, const float *__restrict__ dq_part,
                                                          const float *__restrict__ dk_part, void *__restrict__ dq,
                                                          void *__restrict__ dk) {
  const int64_t start = min(max(cu[0], (int64_t)0), T), end = min(max(cu[n_seq], start), T);
  const int64_t per = static_cast<int64_t>(Hk) * K, n = (end - start) * per;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < n; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t t = start + e / per, hk = (e % per) / K, key = e % K;
    const int64_t src = ((t * Hk + hk) * rep) * K + key, dst = start * per + e;
    float s = 0.f, x = 0.f;
    for (int r = 0; r < rep; ++r) {
      s += dq_part[src + static_cast<int64_t>(r) * K];
      x += dk_part[src + static_cast<int64_t>(r) * K];
    }
    Elem<DT>::store(dq, dst, s);
    Elem<DT>::store(dk, dst, x);
  }
}

// Zeros in the rows of no sequence: n elements of `wide` 2- or 4-byte values a row.
template <typename U>
__device__ __forceinline__ void zero_rows(void *p, int64_t row, int64_t wide) {
  for (int64_t i = threadIdx.x; i < wide; i += 256) static_cast<U *>(p)[row * wide + i] = U(0);
}
template <typename U>
__global__ __launch_bounds__(256) void delta_outside_kernel(const GradArgs ga) {
  const WalkArgs &a = ga.w;
  const int64_t start = min(max(a.cu[0], (int64_t)0), a.T), end = min(max(a.cu[a.n_seq], start), a.T);
  const int64_t n = start + (a.T - end);
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t row = i < start ? i : end + (i - start);
    zero_rows<U>(ga.dq, row, static_cast<int64_t>(a.Hk) * a.K);
    zero_rows<U>(ga.dk, row, static_cast<int64_t>(a.Hk) * a.K);
    zero_rows<U>(ga.dv, row, static_cast<int64_t>(a.H) * a.V);
    zero_rows<float>(ga.dg, row, a.H);
    zero_rows<float>(ga.dbeta, row, a.H);
  }
}

// ------------------------------------------------------------------ launches --
inline dim3 grid_of(int64_t n) { return dim3(static_cast<unsigned>(n)); }

template <int DT, int KP>
int launch_bwd(const DeltaLayout &L, const GradArgs &ga, hipStream_t st) {
  const WalkArgs &a = ga.w;
  const dim3 block(256);
  const int vg = ((a.V + 15) / 16 + 3) / 4;
  if (L.inner_slots > 0) {
    hipLaunchKernelGGL((delta_reverse_kernel<DT, KP, true>), grid_of(L.inner_slots * a.H * vg), block, 0, st, ga);
    if (const int e = delta_fold(L, a, ga.seg_grad, true, st)) return e;
  }
  hipLaunchKernelGGL((delta_reverse_kernel<DT, KP, false>), grid_of(L.seg_slots * a.H * vg), block, 0, st, ga);
  hipLaunchKernelGGL((delta_grad_kernel<DT, KP>), grid_of(L.chunk_slots * a.H), dim3(512), 0, st, ga);
  return launch_status("gated_delta_chunk_bwd");
}

template <int DT>
int launch_keys(const DeltaLayout &L, const GradArgs &ga, hipStream_t st) {
  int e;
  if (L.KP == 32) e = launch_bwd<DT, 32>(L, ga, st);
  else if (L.KP == 64) e = launch_bwd<DT, 64>(L, ga, st);
  else e = launch_bwd<DT, 128>(L, ga, st);
  if (e) return e;
  const WalkArgs &a = ga.w;
  if (ga.dq_part && a.T > 0) {
    const int64_t n = a.T * a.Hk * a.K;
    hipLaunchKernelGGL((delta_heads_kernel<DT>), grid_of(std::min<int64_t>((n + 255) / 256, 1 << 16)), dim3(256), 0, st,
                       a.cu, a.n_seq, a.T, a.Hk, a.H / a.Hk, a.K, ga.dq_part, ga.dk_part, ga.dq, ga.dk);
  }
  return launch_status("gated_delta_chunk_bwd");
}

}  // namespace
}  // namespace ssla

extern "C" size_t ssla_gated_delta_chunk_bwd_workspace_size(int n_seq, int64_t T, int Hk, int H, int K, int V) {
  if (n_seq < 0 || T < 0 || Hk <= 0 || H <= 0 || H % Hk || K <= 0 || K > 128 || V <= 0) return 0;
  return ssla::delta_layout(n_seq, T, Hk, H, K, V, true).total;
}

extern "C" int ssla_gated_delta_chunk_bwd(const void *q, const void *k, const void *v, const float *g,
                                          const float *beta, const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk,
                                          int H, int K, int V, float scale, const float *h0, const void *dout,
                                          const float *dht, void *dq, void *dk, void *dv, float *dg, float *dbeta,
                                          float *dh0, const void *segments, int dtype, void *workspace, size_t workspace_bytes,
                                          void *stream) {
  using namespace ssla;
  clear_error();
  SSLA_CHECK_ARG(n_seq >= 0 && T >= 0 && Hk > 0 && H > 0 && H % Hk == 0 && K > 0 && V > 0,
                 "gated_delta_chunk_bwd: bad sizes n_seq=%d T=%lld Hk=%d H=%d K=%d V=%d", n_seq, (long long)T, Hk, H, K,
                 V);
  if (K > 128) {
    set_error("gated_delta_chunk_bwd: K=%d exceeds 128", K);
    return SSLA_ERR_UNSUPPORTED;
  }
  SSLA_CHECK_ARG(cu_seqlens != nullptr, "gated_delta_chunk_bwd: cu_seqlens is NULL");
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta && dout && dq && dk && dv && dg && dbeta),
                 "gated_delta_chunk_bwd: null tensor pointer");
  if (dtype != SSLA_F32 && dtype != SSLA_BF16 && dtype != SSLA_F16) {
    set_error("gated_delta_chunk_bwd: unsupported dtype %d", dtype);
    return SSLA_ERR_DTYPE;
  }
  if (const int e = check_widths("gated_delta_chunk_bwd", kChunk, Hk, H, K, V)) return e;
  const DeltaLayout L = delta_layout(n_seq, T, Hk, H, K, V, true);
  if (!workspace || workspace_bytes < L.total || !aligned(workspace, 16)) {
    set_error("gated_delta_chunk_bwd: needs %zu bytes of workspace, got %zu", L.total, workspace_bytes);
    return SSLA_ERR_WORKSPACE;
  }
  char *ws = static_cast<char *>(workspace);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  GradArgs ga{};
  ga.w = walk_args(L, ws, q, k, v, cu_seqlens, n_seq, T, Hk, H, K, V, scale, h0, dtype, true,
                   const_cast<void *>(segments));
  ga.dout = dout;
  ga.dht = dht;
  ga.seg_grad = reinterpret_cast<float *>(ws + L.seg_grad);
  ga.chunk_grad = reinterpret_cast<float *>(ws + L.chunk_grad);
  ga.dx = reinterpret_cast<float *>(ws + L.dx);
  ga.dq = dq; ga.dk = dk; ga.dv = dv; ga.dg = dg; ga.dbeta = dbeta; ga.dh0 = dh0;
  if (H > Hk) {
    ga.dq_part = reinterpret_cast<float *>(ws + L.dq);
    ga.dk_part = reinterpret_cast<float *>(ws + L.dk);
  }
  ga.vvec = V % 4 == 0;
  ga.dvec = (static_cast<int64_t>(V) * (dtype == SSLA_F32 ? 4 : 2)) % 16 == 0 && aligned(dout, 16) && aligned(v, 16);
  if (T > 0) {
    const dim3 grid = grid_of(std::min<int64_t>(T, 256));
    if (dtype == SSLA_F32) hipLaunchKernelGGL((delta_outside_kernel<float>), grid, dim3(256), 0, st, ga);
    else hipLaunchKernelGGL((delta_outside_kernel<uint16_t>), grid, dim3(256), 0, st, ga);
  }
  if (n_seq == 0) return launch_status("gated_delta_chunk_bwd");
  if (const int e = delta_forward_states(L, ga.w, g, beta, segments != nullptr, dtype, st)) return e;
  switch (dtype) {
    case SSLA_F32: return launch_keys<SSLA_F32>(L, ga, st);
    case SSLA_BF16: return launch_keys<SSLA_BF16>(L, ga, st);
    default: return launch_keys<SSLA_F16>(L, ga, st);
  }
}

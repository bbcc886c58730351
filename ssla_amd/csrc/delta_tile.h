// Tiles and products of the chunked gated delta rule (forward and backward).
//
// Products run on v_mfma_f32_16x16x32_bf16.  An fp32 value is the exact sum of
// three bf16 (a head and two rounded remainders, 24 bits in all), an fp16 value
// of two, a bf16 value is one: a product of two operands is the sum of the
// products of their parts whose orders add up to at most two, which leaves out
// up to 2^-24 of the operands' product, 2^-27 in the mean (computed for random
// values).  Where only an o of 16 bits follows: two parts an operand and orders up to
// one, which leaves out up to 2^-15, 2^-18 in the mean; o's own rounding is up to 2^-8
// (bf16) or 2^-11 (fp16).  Parts below 2^-126 count as 0 in the products, so values
// below 2^-110 have less than three.  States, sums and the values that are carried on keep the precision of fp32 that way, at a sixth of the bf16
// rate for two fp32 operands and a third where one is a bf16 input; the fp32
// matrix instructions run at a sixteenth.
//
// Index order.  Rows (or keys) are taken 32 at a time as a pair of 16-row
// accumulator tiles 2 p and 2 p + 1: row 4 G + r of tile 2 p + a is index
// 32 p + 8 G + 4 a + r.  Lane group G (lanes 16 G .. 16 G + 15) then holds the
// eight consecutive indices 32 p + 8 G .. + 7 of a column in its two
// accumulators, which is what the next product's operand needs of it: results
// go on to the next product without leaving their lanes.
#pragma once
#include <type_traits>

#include "lds_tile.h"

namespace ssla {

constexpr int kChunk = 64;            // rows of a chunk
constexpr int kTriSets = 6;           // 16 x 32 operands of a lower triangular 64 x 64 matrix
constexpr int kTriFloats = kTriSets * 512;
typedef float f32x8 __attribute__((ext_vector_type(8)));

// Index of row m (0..15) of tile t in the order above.
__device__ __forceinline__ int idx_of(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }
// The operand set of row tile t (0..3), contraction half ks (<= t / 2), of a lower triangular matrix.
__device__ __forceinline__ constexpr int tri_set(int t, int ks) { return t < 2 ? t : 2 * t - 2 + ks; }

template <int DT> struct Parts { static constexpr int n = DT == SSLA_BF16 ? 1 : DT == SSLA_F16 ? 2 : 3; };

// x as a sum of N bf16 vectors.  (Two values a conversion, taken apart again by
// a shift and a mask: the vector conversion back would convert each value anew.)
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int N, int P>
__device__ __forceinline__ void split_pairs(const float (&x)[2 * P], uint32_t (&w)[N][P]) {
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
      if (i + 1 < N) {
        a -= __uint_as_float(w[i][j] << 16);
        b -= __uint_as_float(w[i][j] & 0xffff0000u);
      }
    }
  }
}
template <int N>
__device__ __forceinline__ void split(const f32x8 &x, bf16x8 (&p)[N]) {
  const float v[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
  uint32_t w[N][4];
  split_pairs<N, 4>(v, w);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = from_bits<bf16x8>(make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]));
}
template <int N>
__device__ __forceinline__ void split(const f32x4 &x, uint2 (&p)[N]) {
  const float v[4] = {x[0], x[1], x[2], x[3]};
  uint32_t w[N][2];
  split_pairs<N, 2>(v, w);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = make_uint2(w[i][0], w[i][1]);
}
// Sum over the 16 lanes of a DPP row, in every lane of it.
__device__ __forceinline__ float row_sum(float x) {
  auto turn = [&](auto n) __attribute__((always_inline)) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + decltype(n)::value,
                                                                 0xf, 0xf, false));
  };
  x += turn(std::integral_constant<int, 8>{});
  x += turn(std::integral_constant<int, 4>{});
  x += turn(std::integral_constant<int, 2>{});
  x += turn(std::integral_constant<int, 1>{});
  return x;
}
// x where on, else 0, also where x is not finite; without a branch around what computes x
__device__ __forceinline__ float keep(bool on, float x) {
  asm("" : "+v"(x));
  return on ? x : 0.f;
}
__device__ __forceinline__ f32x8 join(const f32x4 &a, const f32x4 &b) {
  return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// c += a b over the parts whose orders add up to at most LIM, small ones first.
template <int LIM, int NA, int NB>
__device__ __forceinline__ f32x4 mul(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 c) {
#pragma unroll
  for (int s = LIM; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
  return c;
}

// A 64 x KP tile of bf16 in LDS: the 16-byte segments of a row are permuted so
// that both the operand reads (rows idx_of(t, 0..7) of one segment) and the
// transposing reads (four rows, four segments) spread over the banks.
template <int KP>
__device__ __forceinline__ int sw(int row, int col) {
  const int a = row & 1, b = (row >> 1) & 1, c = (row >> 3) & 1;
  const int key = KP == 32 ? (b << 1 | c) : KP == 64 ? (b << 2 | a << 1 | c) : (a << 3 | b << 2 | a << 1 | c);
  return row * KP + ((((col >> 3) ^ key) << 3) | (col & 7));
}
// Operand with lane (m, G) = row idx_of(t, m), columns 32 ks + 8 G .. + 7.
template <int KP>
__device__ __forceinline__ bf16x8 op_rows(const uint16_t *t, int tile, int ks, int lane) {
  return from_bits<bf16x8>(*reinterpret_cast<const uint4 *>(t + sw<KP>(idx_of(tile, lane & 15), 32 * ks + 8 * (lane >> 4))));
}
// Operand with lane (m, G) = column idx_of(tile, m), rows 32 ks + 8 G .. + 7
// (ds_read_b64_tr_b16: see tr_read4; source lane s reads row + s / 4, four
// columns from 8 (s % 4)).
template <int KP>
__device__ __forceinline__ bf16x8 op_cols(const uint16_t *t, int tile, int ks, int lane) {
  const int s = lane & 15, row = 32 * ks + 8 * (lane >> 4) + (s >> 2), col = 32 * (tile >> 1) + 8 * (s & 3) + 4 * (tile & 1);
  uint2 u[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t *p = t + sw<KP>(row + 4 * i, col);
    u[i] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<__attribute__((address_space(3))) s16x4 *>(reinterpret_cast<uintptr_t>(p))));
  }
  return from_bits<bf16x8>(make_uint4(u[0].x, u[0].y, u[1].x, u[1].y));
}

// Global memory goes through buffer resources that cover a chunk's rows (or one
// state): the hardware reads zeros past their end and drops stores there, so
// rows behind a sequence and columns behind a matrix need no branches.  Offsets
// are 32 bits inside a resource; what is outside gets kOutside.
constexpr uint32_t kOutside = 0x80000000u;
typedef __amdgpu_buffer_rsrc_t Rsrc;
__device__ __forceinline__ Rsrc rsrc_of(const void *base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), static_cast<short>(0), static_cast<int>(bytes),
                                           0x00020000);   // raw 32-bit data, range checked
}
// rows of `width` values at a stride (in values of es bytes)
__device__ __forceinline__ Rsrc rows_rsrc(const void *base, int64_t at, int rows, int64_t stride, int width, int es) {
  return rsrc_of(static_cast<const char *>(base) + at * es, rows > 0 ? ((rows - 1) * stride + width) * es : 0);
}
template <typename E>
__device__ __forceinline__ E load_one(const Rsrc &rs, uint32_t off) {
  if constexpr (sizeof(E) == 2) return static_cast<E>(__builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0));
  else return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0));
}
__device__ __forceinline__ f32x4 load4(const Rsrc &rs, uint32_t off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
}
template <typename E>
__device__ __forceinline__ void store_one(const Rsrc &rs, uint32_t off, E x) {
  if constexpr (sizeof(E) == 2) __builtin_amdgcn_raw_buffer_store_b16(x, rs, off, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), rs, off, 0, 0);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T to_elem(float x) {
  if constexpr (DT == SSLA_BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  else if constexpr (DT == SSLA_F16) return f32_to_f16_bits(x);
  else return x;
}
template <int DT>
__device__ __forceinline__ float of_elem(typename Elem<DT>::T x) {
  if constexpr (DT == SSLA_BF16) return bf16_bits_to_f32(x);
  else if constexpr (DT == SSLA_F16) return f16_bits_to_f32(x);
  else return x;
}

// 64 rows of a matrix with row stride `stride` (values), fetched into registers
// by 256 threads (or once by each 256 of them) and stored to LDS as Parts<DT>::n tiles of bf16; rows past the
// resource and columns from n_cols on are zero.  Where rows are whole 16-byte
// pieces at aligned addresses (vec) they are read 16 bytes at a time.
template <int DT, int KP>
struct RowTile {
  static constexpr int U = KP / 32;   // 8-column pieces of a thread
  typedef typename Elem<DT>::T E;
  static constexpr int ES = sizeof(E), W = ES / 2;   // 16-byte loads of a piece
  struct Piece { E e[8]; };
  Piece p[U];

  __device__ __forceinline__ void fetch(const Rsrc &rs, int stride, int n_cols, bool vec) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = (threadIdx.x & 255) + 256 * i, row = u / (KP / 8), col = (u % (KP / 8)) * 8;
      const uint32_t at = static_cast<uint32_t>(row * stride + col) * ES;
      if (vec) {
        struct Raw { uint4 w[W]; } raw;
#pragma unroll
        for (int j = 0; j < W; ++j)
          raw.w[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
              rs, col + 8 / W * (j + 1) <= n_cols ? at + 16 * j : kOutside, 0, 0));
        p[i] = __builtin_bit_cast(Piece, raw);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[i].e[j] = load_one<E>(rs, col + j < n_cols ? at + ES * j : kOutside);
      }
    }
  }
  __device__ __forceinline__ float value(int i, int j) const { return of_elem<DT>(p[i].e[j]); }   // column j of piece i
  // plane j at t + j * stride elements
  __device__ __forceinline__ void store(uint16_t *t, int stride) const {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = (threadIdx.x & 255) + 256 * i, row = u / (KP / 8), col = (u % (KP / 8)) * 8;
      uint16_t *dst = t + sw<KP>(row, col);
      if constexpr (DT == SSLA_BF16) {
        *reinterpret_cast<uint4 *>(dst) = __builtin_bit_cast(uint4, p[i]);
      } else {
        f32x8 x;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = value(i, j);
        bf16x8 s[Parts<DT>::n];
        split(x, s);
#pragma unroll
        for (int j = 0; j < Parts<DT>::n; ++j) *reinterpret_cast<uint4 *>(dst + j * stride) = to_bits(s[j]);
      }
    }
  }
};

// The chunks' matrices and row factors that every pass reads, written once by
// the first kernel: per (chunk slot, head) the operands of Tm = (I + A)^-1 in
// fp32 (set by set, 64 lanes of 8 values), for the backward those of its
// transpose behind them, and kRowVecs vectors of 64 floats.
enum { kBeta = 0, kBetaG, kScaleG, kToEnd, kGHi, kGLo, kRowVecs };
constexpr int kRowFloats = kRowVecs * kChunk;

// Chunk c (of 64 rows) of sequence n that starts at row bos has slot
// bos / 64 + n + c; see seq_of_slot.  In a mixed batch (sequences of up to kChunk
// rows run token by token) it has bos / 32 + c.
__device__ __forceinline__ int64_t chunk_slot(int64_t bos, int n, int64_t c, bool mixed = false) {
  return (bos >> (mixed ? 5 : 6)) + (mixed ? 0 : n) + c;
}

inline size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
inline int padded_keys(int K) { return K <= 32 ? 32 : K <= 64 ? 64 : 128; }

// Chunks per segment: as many as leave about 512 workgroups of 64 value columns (two
// a CU, where the kernel's LDS admits two), and at least 4; where heads are few, with
// c chunks in an average sequence at least sqrt(c / 5), where the walks over a
// segment (3.5 us a chunk) take about as long as the folds over the segments (0.8 us
// each, 1.3 in reverse).  Measured: 8 x 4096 rows of 8 heads of 64 143 us at 8 chunks,
// 172 at 4; 65,536 rows of one head of 128 384 us at 15, 420 at 11, 496 at 8; of one
// head of 64 172 at 15, 165 at 11, 170 at 8; 16,384 of one head of 64 96 at 8, 90 at 5 and
// 6 (c / 8 instead of c / 5 took 379 us instead of 348 for 32,768 rows of 4 heads of 128).
// The average may come of sequences that are hardly there, beside a long one: no
// batch is cut into more than 128 segments unless one sequence of all rows would be.
// Measured for 65,536 rows of one head, 4 and 8 chunks: one sequence beside 63 single
// rows 241 and 171 us at 64 columns, 872 and 496 at 128; 64 equal sequences 69 and 77,
// 164 and 131.  (8 at least for fewer rows too: 12 sequences in 8,209 rows, a training
// step, 222 and 299.)
inline int seg_chunks(int n_seq, int64_t T, int H, int V) {
  const int64_t chunks = (T + kChunk - 1) / kChunk, work = chunks * H * ((V + 63) / 64);
  int64_t per = std::max<int64_t>(4, (work + 511) / 512);
  while (per * per * 5 < chunks && (per * per * 5 * n_seq < chunks || per * 128 < chunks)) ++per;
  return static_cast<int>(std::min<int64_t>(1 << 20, per));
}

// Workspace of the forward, and (grad) of the backward.  The segments' states and
// maps come first in a block of their own (seg_bytes), which a forward can leave
// to its backward.
struct DeltaLayout {
  size_t map, seg_bytes, segs, tm, rowv, seg_grad, chunk_state, chunk_grad, u, dx, dq, dk, total;
  int64_t chunk_slots, seg_slots, inner_slots;
  int per, KP;
};
inline DeltaLayout delta_layout(int n_seq, int64_t T, int Hk, int H, int K, int V, bool grad, bool mixed = false) {
  DeltaLayout L{};
  L.KP = padded_keys(K);
  // (a mixed batch may be one long sequence and nothing else)
  L.per = seg_chunks(mixed ? 1 : std::max(n_seq, 1), T, H, V);
  const int64_t unit = static_cast<int64_t>(L.per) * kChunk;
  L.chunk_slots = mixed ? T / (kChunk / 2) + 1 : T / kChunk + n_seq + 1;
  L.seg_slots = mixed ? T / kChunk + 1 : T / unit + n_seq + 1;
  L.inner_slots = T > 0 ? (T - 1) / unit : 0;   // 0: no sequence is cut
  size_t p = 0;
  auto take = [&](size_t bytes) {
    const size_t at = p;
    p = align256(p + bytes);
    return at;
  };
  const size_t kv = static_cast<size_t>(K) * V * sizeof(float);
  L.tm = take(sizeof(float) * kTriFloats * (grad ? 2 : 1) * L.chunk_slots * H);
  L.rowv = take(sizeof(float) * kRowFloats * L.chunk_slots * H);
  L.map = align256(kv * L.inner_slots * H);
  L.seg_bytes = L.map + align256(sizeof(uint16_t) * 3 * L.inner_slots * H * L.KP * L.KP);
  L.segs = take(L.seg_bytes);
  if (grad) {
    L.seg_grad = take(kv * L.inner_slots * H);
    L.chunk_state = take(kv * L.chunk_slots * H);
    L.chunk_grad = take(kv * L.chunk_slots * H);
    L.u = take(sizeof(float) * T * H * V);
    L.dx = take(sizeof(float) * T * H * V);
    L.dq = take(H > Hk ? sizeof(float) * T * H * K : 0);
    L.dk = take(H > Hk ? sizeof(float) * T * H * K : 0);
  }
  L.total = p;
  return L;
}

// 16 x 16 x 4 N product in fp32 (operand value j of lane group G: contraction
// index N G + j), for the few products whose operands are not kept in parts.
template <int N>
__device__ __forceinline__ f32x4 mul_f32(const float (&a)[N], const float (&b)[N], f32x4 c) {
#pragma unroll
  for (int j = 0; j < N; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// 16 columns of a [K, V] fp32 state as accumulator tiles: lane = (key group,
// column); keys from K on and columns from V on are zero and not stored.
template <int NT>
struct StateCols {
  uint32_t off;   // of key 8 G in this lane's column
  int K, V4;
  __device__ __forceinline__ StateCols(int K_, int V, int vcol, bool on, int G)
      : off(on ? static_cast<uint32_t>(8 * G * V + vcol) * 4u : kOutside), K(K_), V4(V * 4) {}
  __device__ __forceinline__ Rsrc rs(const float *base) const { return rsrc_of(base, base ? static_cast<int64_t>(K) * V4 : 0); }
  __device__ __forceinline__ void load(const float *base, f32x4 (&S)[NT]) const {
    const Rsrc r = rs(base);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[t][i] = load_one<float>(r, off + idx_of(t, i) * V4);
  }
  __device__ __forceinline__ void store(float *base, const f32x4 (&S)[NT]) const {
    const Rsrc r = rs(base);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) store_one<float>(r, off + idx_of(t, i) * V4, S[t][i]);
  }
};

struct WalkArgs {
  const void *q, *k, *v;
  const int64_t *cu;
  const float *tm, *rowv;
  const float *h0;
  void *o;
  float *ht;
  // per inner segment (all but a sequence's last): L, after the fold the state
  // entering the next segment, and (but for a sequence's first) M as three bf16 matrices
  float *seg_state;
  uint16_t *seg_map;
  float *chunk_state;     // per chunk: the state entering it
  float *u;               // [T, H, V]
  int64_t T;
  int n_seq, Hk, H, K, V, per, vec, tm_floats, mixed;
  float scale;
};

inline WalkArgs walk_args(const DeltaLayout &L, char *ws, const void *q, const void *k, const void *v, const int64_t *cu,
                          int n_seq, int64_t T, int Hk, int H, int K, int V, float scale, const float *h0, int dtype,
                          bool grad, void *segs) {
  WalkArgs a{};
  a.q = q; a.k = k; a.v = v; a.cu = cu; a.h0 = h0;
  a.tm = reinterpret_cast<float *>(ws + L.tm);
  a.rowv = reinterpret_cast<float *>(ws + L.rowv);
  char *sg = segs ? static_cast<char *>(segs) : ws + L.segs;
  a.seg_state = reinterpret_cast<float *>(sg);
  a.seg_map = reinterpret_cast<uint16_t *>(sg + L.map);
  if (grad) {
    a.chunk_state = reinterpret_cast<float *>(ws + L.chunk_state);
    a.u = reinterpret_cast<float *>(ws + L.u);
  }
  a.T = T; a.n_seq = n_seq; a.Hk = Hk; a.H = H; a.K = K; a.V = V; a.per = L.per; a.scale = scale;
  a.tm_floats = kTriFloats * (grad ? 2 : 1);
  a.vec = (static_cast<int64_t>(K) * (dtype == SSLA_F32 ? 4 : 2)) % 16 == 0 && aligned(q, 16) && aligned(k, 16);
  return a;
}

// Offsets inside `rows` rows, or inside a state (of up to 256 padded keys), are 32 bits.
inline int check_widths(const char *what, int rows, int Hk, int H, int K, int V) {
  if (std::max(static_cast<int64_t>(Hk) * K, static_cast<int64_t>(H) * std::max(K, V)) * rows * 4 > 0x7fffffff ||
      V > 1 << 20) {
    set_error("%s: rows of %d x %d or %d x %d values are too wide", what, Hk, K, H, V);
    return SSLA_ERR_UNSUPPORTED;
  }
  return SSLA_OK;
}

// The chunks' matrices, unless they are there (have_segs) the segments' states and
// maps, and every chunk's entering state and u (delta_chunk.hip), for the backward.
int delta_forward_states(const DeltaLayout &L, const WalkArgs &a, const float *g, const float *beta, bool have_segs,
                         int dtype, hipStream_t st);

// Token by token, the sequences of up to `longest` rows (delta_recurrent.hip).
int delta_recurrent_up_to(const char *what, int64_t longest, const void *q, const void *k, const void *v, const float *g,
                          const float *beta, const int64_t *cu_seqlens, int n_seq, int64_t T, int Hk, int H, int K, int V,
                          float scale, const float *h0, void *o, float *ht, const int32_t *state_idx, int n_state_rows,
                          int32_t *status, int dtype, hipStream_t st);

// Carries states over a sequence's segments (delta_chunk.hip).  Forward: with M and
// L of segments 1 .., and L of segment 0 the state behind it, L of segment j
// becomes the state behind segment j.  In reverse (states: of the gradient, slot j
// what segment j + 1 adds to the gradient leaving segment j) slot j becomes the
// gradient leaving segment j.
int delta_fold(const DeltaLayout &L, const WalkArgs &a, float *states, bool reverse, hipStream_t st);

}  // namespace ssla

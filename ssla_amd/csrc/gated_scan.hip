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
// Over few channels, where long chains of tiles run at once, 16 tiles are a span that
// publishes a map and a state of its own (262,144 rows of 64 channels 58 us, without 95).
// Tiles are handed out in order by a ticket and publish before they wait, so every
// tile waited for has started and the wait ends.  A word says by itself whether it
// is there, a map or a state: no fences.
// The backward does the same from the last tile on; the states it needs come from
// the forward, which leaves one every 64 rows, and are computed again in between.
// Measured: 65,536 rows of 1,024 channels, bf16, with q 133 us (4.0 TB/s; vector units
// busy 41 % of the time, wavefronts waiting 58 %); 8 x 4,096 rows forward 74, backward 127;
// 65,536 sequences of one row 231 with their states (4.6 TB/s); 912 single tokens of
// 2,048 channels 5.9 (5.1 TB/s).
#include "vec.h"

#include <type_traits>

namespace ssla {
namespace {

constexpr int kValue = SSLA_GATE_VALUE, kLog = SSLA_GATE_LOG, kSigmoid = SSLA_GATE_SIGMOID;

// e^x with the product x log2(e) in two parts: off by 4 2^-24 (e^x of one product by up to
// 100 2^-24) at any x whose e^x is a normal number and, unless UP, at most 2^126.
template <bool UP>
__device__ __forceinline__ float exp_of(float x) {
  const float y = x * kLog2e, e = fast_exp2(y);
  const float lo = fmaf(x, 1.925963e-8f, fmaf(x, kLog2e, -y));
  const bool inside = UP ? y >= -126.f && y < 128.f : fabsf(y) <= 126.f;   // (past that 0, infinite or next to it)
  return inside ? fmaf(e, lo * 0.6931472f, e) : e;
}

// The gate; and with its derivative, sigmoid's from e^-|g|: both it and 1 - it keep
// their relative precision on either side.
struct Gate { float a, slope; };
template <int KIND>
__device__ __forceinline__ float gate_value(float g) {
  if constexpr (KIND == kValue) return g;
  if constexpr (KIND == kLog) return exp_of<true>(g);
  return __builtin_amdgcn_rcpf(1.f + exp_of<false>(-g));   // (e^-g infinite: 0; past 2^126 no normal number)
}
template <int KIND>
__device__ __forceinline__ Gate gate_of(float g) {
  if constexpr (KIND == kSigmoid) {
    const float t = exp_of<false>(-fabsf(g)), r = __builtin_amdgcn_rcpf(1.f + t), s = t * r;
    return {g >= 0.f ? r : s, r * s};
  }
  const float a = gate_value<KIND>(g);
  return {a, KIND == kLog ? a : 1.f};
}

// Rows of a lane, and threads: large tiles are few steps between them, small ones leave
// registers for more workgroups.  65,536 rows of 1,024 channels, forward (us): 8 rows 135
// with 512 threads, 145 with 256, 172 with 1,024; 4 rows 230.  The backward of 8 x 4,096
// rows holds twice as much a row: 4 rows 127, 8 rows 14 % more.
constexpr int kFwdRows = 8, kBwdRows = 4;
constexpr int kMostRows = 8;
constexpr int kBlock = 512;
constexpr int kKeepRows = 64;    // rows between the states left for the backward
constexpr int kMostLanes = 16;   // lanes of a row
constexpr int kMostGroups = 64;  // row groups of a tile
constexpr int kMostValues = kBlock * 4;   // (row group, channel) pairs of a tile
constexpr int kMostWidth = 1 << 20;       // elements from row to row: offsets in a tile are 32 bits

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
  int tiles;                      // of rows
  uint32_t *ticket;               // NULL: one tile of rows
  uint64_t *words, *span_words;   // [tiles], [spans][cblocks CT W]: what a tile (spans of more), a span says of itself
  uint32_t *hints;                // [cblocks][spans]
};

// ------------------------------------------------------- tiles and sequences --
// What a tile's rows are: mark[row] the sequence that begins there, kInside, or
// kOutside of all sequences; fin[row] the sequence that ends with the row, or -1.
constexpr int kInside = -1, kOutside = -2;

struct Span { int64_t b, e; };   // a sequence's rows
__device__ __forceinline__ Span span_of(const ScanArgs &a, int n) {
  Span s;
  s.b = min(max(a.cu[n], (int64_t)0), a.T);
  s.e = min(max(a.cu[n + 1], s.b), a.T);
  return s;
}

// Fills mark and fin of the rows r0 .. r0 + rows; false where all rows are kInside
// and none ends a sequence.  `mine`: sequence threadIdx.x, `all` the rows of any.  More
// than kBlock sequences are searched, two rounds of probes for up to 65,536.
__device__ __forceinline__ bool mark_rows(const ScanArgs &a, const Span &mine, const Span &all, int64_t r0, int rows, int *mark,
                                          int *fin) {
  const int tid = threadIdx.x;
  bool some = false;
  for (int i = tid; i < rows; i += kBlock) {
    const bool out = r0 + i < all.b || r0 + i >= all.e;
    mark[i] = out ? kOutside : kInside;
    fin[i] = -1;
    some |= out;
  }
  auto put = [&](const Span &s, int n) {
    if (s.e > s.b) {
      if (s.b >= r0 && s.b < r0 + rows) {
        mark[s.b - r0] = n;
        some = true;
      }
      if (s.e > r0 && s.e <= r0 + rows) {
        fin[s.e - 1 - r0] = n;
        some = true;
      }
    }
  };
  if (a.n_seq <= kBlock) {   // (the same for all threads)
    __syncthreads();
    if (tid < a.n_seq) put(mine, tid);
  } else {
    int lo = 0, hi = a.n_seq;   // the last sequence that begins at r0 or before is in [lo, hi)
    while (hi - lo > kBlock) {
      const int step = (hi - lo + kBlock - 1) / kBlock;
      const int64_t i = lo + static_cast<int64_t>(tid) * step;
      const int cnt = __syncthreads_count(i < hi && a.cu[i] <= r0);
      lo += max(cnt - 1, 0) * step;
      hi = min(hi, lo + step);
    }
    for (bool past = false; lo < a.n_seq && !past; lo += kBlock) {
      const int n = lo + tid;
      Span s{r0 + rows, 0};
      if (n < a.n_seq) s = span_of(a, n);
      past = __syncthreads_or(s.b >= r0 + rows);
      put(s, n);
    }
  }
  return __syncthreads_or(some);
}

// --------------------------------------------------- states between the tiles --
// A tile's word in a channel: nothing yet (all ones), its map (A low, U high), or the
// state that leaves it (kState low, the state high).
constexpr uint64_t kNone = ~0ull;
constexpr uint32_t kState = 0xfffffffeu;

__device__ __forceinline__ uint64_t state_word(float x) {
  return static_cast<uint64_t>(__float_as_uint(x)) << 32 | kState;
}
__device__ __forceinline__ uint64_t map_word(float A, float U) {   // (a NaN of A's like the marks is made the usual one)
  const uint32_t b = __float_as_uint(A);
  return static_cast<uint64_t>(__float_as_uint(U)) << 32 | (b >= kState ? 0x7fc00000u : b);
}
__device__ __forceinline__ bool is_state(uint64_t w) { return static_cast<uint32_t>(w) == kState; }
template <typename T>
__device__ __forceinline__ T look(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ void show(T *p, T x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A product of gates too small for fp32, none of them 0, is held as +-2^-149 (kFaded: its
// bits): an infinite state goes on, a finite one is off by 2^-149 of itself at most.
constexpr uint32_t kFaded = 1;
// The product A of factors; zero: one of them is 0 (whatever overflowed beside it).
__device__ __forceinline__ float settled(float A, bool zero) {
  return zero ? 0.f : A == 0.f ? __uint_as_float((__float_as_uint(A) & 0x80000000u) | kFaded) : A;
}
// (a factor that overflowed must not meet a state of zero)
__device__ __forceinline__ float apply(float A, float x, float U) { return x == 0.f ? U : fmaf(A, x, U); }
// The state behind a tile that x enters: the same bits whichever of its words was there.
__device__ __forceinline__ float apply(uint64_t w, float x) {
  const float U = __uint_as_float(static_cast<uint32_t>(w >> 32));
  return is_state(w) ? U : apply(__uint_as_float(static_cast<uint32_t>(w)), x, U);
}

// What the last tile of a span has published of it in a channel block, told by a word of
// its own next to its neighbours': a wavefront sees 64 spans at one read.  Only a hint
// where to look: the words say by themselves whether they are there.
constexpr uint32_t kNoHint = ~0u, kMapHint = 1, kStateHint = 2;

// The nearest span before k > 0 whose state is known, with maps from there on; for a
// whole wavefront.
__device__ __forceinline__ int known_span(const uint32_t *hints, int k) {
  const int lane = threadIdx.x & 63;
  for (int near = k - 1;;) {
    const int t = near - lane;
    const uint32_t h = t >= 0 ? look(hints + t) : kMapHint;
    const uint64_t states = __ballot(h == kStateHint), nothing = __ballot(h == kNoHint);
    const int s = states ? __builtin_ctzll(states) : 64, n = nothing ? __builtin_ctzll(nothing) : 64;
    if (s < n) return near - s;
    if (n == 64) near -= 64;   // (span 0 is known or not there: it stays at 0 or above)
    else __builtin_amdgcn_s_sleep(1);
  }
}

__global__ __launch_bounds__(256) void scan_clear_kernel(uint32_t *ticket, uint64_t *words, int64_t n) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    words[i] = kNone;
}

// Which tile and channel block a workgroup has.
__device__ __forceinline__ int take_tile(const ScanArgs &a, uint32_t *slot) {
  if (!a.ticket) return blockIdx.x;
  if (threadIdx.x == 0) *slot = atomicAdd(a.ticket, 1u);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*slot);
}

// Joins the maps of the RG row groups of channel c (LDS, `cw` channels a row group)
// from the first or the last on; cut[k]: the state leaving group k is U, whatever enters.
struct Joined { float A, U; };
template <bool BACK>
__device__ __forceinline__ Joined join_groups(const float *A, const float *U, const int *cut, int RG, int cw, int c) {
  Joined j{1.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < RG; ++i) {
    const int k = BACK ? RG - 1 - i : i;
    const float x = A[k * cw + c], y = U[k * cw + c];
    const bool r = cut[k];
    j.U = r ? y : apply(x, j.U, y);
    j.A *= x;
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
// What the threads share between a tile's maps.
constexpr int kSpanLog2 = 4, kSpan = 1 << kSpanLog2;   // tiles of a span, where there is more than one
constexpr int kWords = 48;   // spans of a round trip
struct TileSmem {
  float A[kMostValues], U[kMostValues];
  uint64_t words[(kSpan + kWords) * kMostLanes * 4];
  int mark[kMostGroups * kMostRows], fin[kMostGroups * kMostRows], cut[kMostGroups];
  int flags[kBlock];   // of a channel: one of its gates is 0; later of empty_states
  int from;
  uint32_t slot;
};

// Between a tile's maps, for the whole workgroup: publishes, finds the entering states
// (`closed`: the tile's first row takes none) and fills U.  The threads from `first` on
// have a channel each; all of them fetch the words.
//
// 2^SPAN tiles are a span.  Its last tile joins their maps to the span's; the states behind
// spans come of the states before and the spans' maps, those inside a span of the state
// before it and its tiles' maps, always in this order: the same bits whoever is first.
template <bool BACK, int SPAN>
__device__ __forceinline__ void enter_tile(const ScanArgs &a, TileSmem &sm, float *U, int k, int cb, bool closed, int cw,
                                           int first) {
  const int tid = threadIdx.x, c = tid - first, mine = a.C - cb * cw;   // (channels that exist)
  const bool on = c >= 0 && c < cw && c < mine;
  float x = 0.f;
  if (a.ticket) {
    const int64_t wide = static_cast<int64_t>(a.cblocks) * cw;
    const int s = k >> SPAN, in = k - (s << SPAN);
    const bool last = in + 1 == 1 << SPAN, open = k > 0 && !closed;
    uint64_t *words = a.words + static_cast<int64_t>(cb) * cw, *above = a.span_words + static_cast<int64_t>(cb) * cw;
    uint64_t *span = above + s * wide;
    uint32_t *hints = a.hints + static_cast<int64_t>(cb) * (a.tiles >> SPAN);   // (of the whole spans)
    // the words of n tiles or spans, from slot `at` on
    auto fetch = [&](const uint64_t *from, int n, int at, bool state) {
      const int per = kBlock / cw, i0 = tid / cw, cc = tid - i0 * cw;
      if (i0 < per && cc < mine)
        for (int i = i0; i < n; i += 4 * per) {
          uint64_t w[4];
          bool there;
          do {   // (a word may come after its hint)
            there = true;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = i + e * per;
              w[e] = t < n ? look(from + t * wide + cc) : 0;
              there = there && w[e] != kNone && (t > 0 || !state || is_state(w[e]));
            }
          } while (!there);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e * per < n) sm.words[(at + i + e * per) * cw + cc] = w[e];
        }
      __syncthreads();
    };
    auto pass = [&](int at, int n) {   // x through n words
      for (int i = 0; i < n; i += 8) {   // (eight reads on their way at once)
        uint64_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = sm.words[(at + min(i + e, n - 1)) * cw + c];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < n) x = apply(w[e], x);
      }
    };
    bool known = k == 0;
    Joined j{0.f, 0.f};
    if (c >= 0 && c < 64) {   // (a whole wavefront)
      known |= __any(c < a.RG && sm.cut[c] != 0);
      if (on) {
        j = join_groups<BACK>(sm.A, U, sm.cut, a.RG, cw, c);
        j.A = settled(j.A, sm.flags[c]);
        const uint64_t w = known ? state_word(j.U) : map_word(j.A, j.U);
        if (SPAN > 0) show(words + k * wide + c, w);
        if (last && (known || SPAN == 0)) show(span + c, w);
      }
      if (last && (known || SPAN == 0) && c == 0) show(hints + s, known ? kStateHint : kMapHint);
    }
    asm volatile("" ::: "memory");   // (published before anything is waited for)
    if (open) {
      if (SPAN > 0 && in > 0) fetch(words + (k - in) * wide, in, 0, false);
      if (c >= 0 && c < 64) {
        bool cut = false;   // (the same for all channels)
        if (SPAN > 0 && on && last) {
          Joined m{1.f, 0.f};
          bool zero = j.A == 0.f;
          for (int i = 0; i < in; ++i) {
            const uint64_t w = sm.words[i * cw + c];
            const float f = __uint_as_float(static_cast<uint32_t>(w));
            cut |= is_state(w);
            m.U = apply(w, m.U);
            m.A *= f;
            zero |= f == 0.f;
          }
          j = {settled(m.A * j.A, zero), apply(j.A, m.U, j.U)};
        } else if (SPAN > 0 && on) {
          for (int i = 0; i < in; ++i) cut |= is_state(sm.words[i * cw + c]);
        }
        if (SPAN > 0) cut = __any(cut);
        if (SPAN > 0 && last && !known) {
          if (on) show(span + c, cut ? state_word(j.U) : map_word(j.A, j.U));
          if (c == 0) show(hints + s, cut ? kStateHint : kMapHint);
        }
        known |= cut;
        const int from = cut ? -1 : known_span(hints, s);
        if (c == 0) sm.from = from;
      }
      __syncthreads();
      const int from = __builtin_amdgcn_readfirstlane(sm.from);
      if (from >= 0)
        for (int at = from; at < s; at += kWords) {
          const int n = min(s - at, kWords);
          fetch(above + at * wide, n, kSpan, at == from);
          if (on) pass(kSpan, n);
          if (at + kWords < s) __syncthreads();
        }
      if (last && !known) {
        if (on) show(span + c, state_word(apply(j.A, x, j.U)));
        if (c == 0) show(hints + s, kStateHint);
      }
      if (SPAN > 0 && on && in > 0) pass(0, in);
    }
  }
  if (on) enter_groups<BACK>(sm.A, U, sm.cut, a.RG, cw, c, x);
}

// R rows of W values from channel c of row `row` of a tile that begins at `first`, ld
// apart; behind the last row that exists, that one again.
template <int DT, int W, int R>
__device__ __forceinline__ void load_rows(Vec<DT, W> (&x)[R], const void *p, int64_t first, int64_t ld, int row, int last, int c) {
  const typename Elem<DT>::T *base = static_cast<const typename Elem<DT>::T *>(p) + first * ld;
#pragma unroll
  for (int i = 0; i < R; ++i)
    x[i] = load_vec<DT, W>(base, static_cast<uint32_t>(min(row + i, last)) * static_cast<uint32_t>(ld) + c);
}

// Keeps the values as they were read: without this their 32-bit forms are kept over
// the wait, twice the registers.
template <typename V, int R>
__device__ __forceinline__ void as_read(V (&x)[R]) {
  struct Raw { uint32_t w[(sizeof(V) + 3) / 4]; };
  if constexpr (sizeof(V) % 4 == 0)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      Raw r = __builtin_bit_cast(Raw, x[i]);
#pragma unroll
      for (uint32_t &w : r.w) asm volatile("" : "+v"(w));
      x[i] = __builtin_bit_cast(V, r);
    }
}

// f(i, e) of all values held.
template <int R, int W, typename F>
__device__ __forceinline__ void each(F f) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) f(i, e);
}
// The products A of a lane's gates(i, e), and a flag for each channel with a gate of 0.
// A product of 0 (or 0 times one that overflowed) is rare enough to look at the gates
// again: a count of them in join_groups, on every tile's way, is 1 % of any call, this
// 2 to 3 % of calls with gates of 0 in most tiles.
template <int R, int W, typename F>
__device__ __forceinline__ void settle(float (&A)[W], int *zeros, F gates) {
#pragma unroll
  for (int e = 0; e < W; ++e)
    if (!(fabsf(A[e]) > 0.f)) {
      bool zero = false;
#pragma unroll
      for (int i = 0; i < R; ++i) zero |= gates(i, e) == 0.f;
      A[e] = settled(A[e], zero);
      if (zero) zeros[e] = 1;
    }
}
// W values of a row of states (fp32, at any 4-byte border).
template <int W>
struct __attribute__((aligned(4))) States { float x[W]; };
template <int W>
__device__ __forceinline__ const States<W> &states_at(const float *p, int64_t i) {
  return *reinterpret_cast<const States<W> *>(p + i);
}
// The rows n[0 .. B - 1] of p where they are rows and p is there: zeros otherwise.  All on
// their way at once (a wait for each of many short sequences' is most of their time).
template <int W, int B>
__device__ __forceinline__ void load_states(States<W> (&s)[B], const float *p, const int (&n)[B], int C, int c) {
#pragma unroll
  for (int i = 0; i < B; ++i) {
    s[i] = States<W>{};
    if (p && n[i] >= 0) s[i] = states_at<W>(p, static_cast<int64_t>(n[i]) * C + c);
  }
}

// f(KIND as a constant) of a call's kind of gate: decided once for all values held.
template <typename F>
__device__ __forceinline__ void by_kind(int kind, F f) {
  if (kind == kSigmoid) f(std::integral_constant<int, kSigmoid>());
  else if (kind == kLog) f(std::integral_constant<int, kLog>());
  else f(std::integral_constant<int, kValue>());
}

// The states of empty sequences, dealt over the tiles in blocks: what enters leaves.  For
// the whole workgroup, flags: kBlock integers of its own.
__device__ __forceinline__ void empty_states(const ScanArgs &a, const float *from, float *to, int k, int cb, int cw, int *flags) {
  const int tid = threadIdx.x, c = cb * cw + tid, per = (a.n_seq + a.tiles - 1) / a.tiles;
  const int last = static_cast<int>(min(static_cast<int64_t>(k + 1) * per, static_cast<int64_t>(a.n_seq)));
  for (int64_t n0 = static_cast<int64_t>(k) * per; n0 < last; n0 += kBlock) {
    const int64_t n = n0 + tid;
    bool none = false;
    if (n < last) {
      const Span s = span_of(a, static_cast<int>(n));
      none = s.e == s.b;
    }
    if (!__syncthreads_or(none)) continue;
    flags[tid] = none;
    __syncthreads();
    for (int i = 0; i < kBlock && n0 + i < last; ++i)
      if (flags[i] && tid < cw && c < a.C) to[(n0 + i) * a.C + c] = from ? from[(n0 + i) * a.C + c] : 0.f;
    __syncthreads();
  }
}

// ------------------------------------------------------------------ forward --
// Two workgroups a CU (128 registers; the LDS holds no third) in 16 bits: measured in bf16,
// which spills none (7 with fp32 gates), while fp16 with a read-out gate spills 10 to 19
// (65,536 rows of 1,024 channels 150 us, bf16 131).  fp32 values do without the second one
// sooner than without registers (8 x 4,096 rows: 130 us, 162 at 128 registers).
template <int DT, int DTG, int W, bool READ, int SPAN>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(DT == SSLA_F32 ? 2 : 4))) void scan_fwd_kernel(const ScanArgs a) {
  constexpr int R = kFwdRows, B = 4;   // B: rows whose states are read at once
  __shared__ TileSmem sm;
  const int tid = threadIdx.x, cw = a.CT * W, rows = a.RG * R;
  const int rg = tid / a.CT, cl = tid - rg * a.CT;
  const Span all = a.n_seq ? Span{span_of(a, 0).b, span_of(a, a.n_seq - 1).e} : Span{0, 0};
  const Span mine = tid < a.n_seq ? span_of(a, tid) : Span{0, 0};
  const int id = take_tile(a, &sm.slot);
  const int k = id / a.cblocks, cb = id - k * a.cblocks;
  if (a.T == 0) {   // (one tile without rows)
    if (a.ht) empty_states(a, a.h0, a.ht, k, cb, cw, sm.flags);
    return;
  }
  const int64_t r0 = static_cast<int64_t>(k) * rows;
  const int row = rg * R;
  const int exist = static_cast<int>(min(a.T - r0, static_cast<int64_t>(rows))), left = exist - row;
  const bool on = rg < a.RG && (cb * a.CT + cl) * W < a.C;
  const int c = on ? (cb * a.CT + cl) * W : 0;   // (lanes without a channel read the first)
  Vec<DT, W> u[R], q[READ ? R : 1];
  Vec<DTG, W> g[R];
  load_rows<DT, W, R>(u, a.u, r0, a.ldu, row, exist - 1, c);
  load_rows<DTG, W, R>(g, a.g, r0, a.ldg, row, exist - 1, c);
  if constexpr (READ) load_rows<DT, W, R>(q, a.q, r0, a.ldq, row, exist - 1, c);
  if (tid < cw) sm.flags[tid] = 0;   // (mark_rows waits)
  const bool some = mark_rows(a, mine, all, r0, rows, sm.mark, sm.fin);
  float f[R][W];
  by_kind(a.gate, [&](auto kind) { each<R, W>([&](int i, int e) { f[i][e] = gate_value<kind()>(g[i][e]); }); });
  if (on) {
    float A[W], U[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      A[e] = 1.f;
      U[e] = 0.f;
    }
    bool reset = false;
    if (!some) {
      each<R, W>([&](int i, int e) {
        U[e] = fmaf(f[i][e], U[e], u[i][e]);
        A[e] *= f[i][e];
      });
    } else {
#pragma unroll
      for (int i0 = 0; i0 < R; i0 += B) {
        int m[B];
        States<W> s0[B];
#pragma unroll
        for (int i = 0; i < B; ++i) m[i] = sm.mark[row + i0 + i];
        load_states(s0, a.h0, m, a.C, c);
#pragma unroll
        for (int i = 0; i < B; ++i) {
          reset |= m[i] != kInside;
#pragma unroll
          for (int e = 0; e < W; ++e) {
            U[e] = m[i] == kOutside ? 0.f : fmaf(f[i0 + i][e], m[i] >= 0 ? s0[i].x[e] : U[e], u[i0 + i][e]);
            A[e] *= f[i0 + i][e];
          }
        }
      }
    }
    settle<R, W>(A, sm.flags + cl * W, [&](int i, int e) { return f[i][e]; });
#pragma unroll
    for (int e = 0; e < W; ++e) {
      sm.A[rg * cw + cl * W + e] = A[e];
      sm.U[rg * cw + cl * W + e] = U[e];
    }
    if (cl == 0) sm.cut[rg] = reset;
  }
  __syncthreads();
  enter_tile<false, SPAN>(a, sm, sm.U, k, cb, some && sm.mark[0] != kInside, cw, 0);
  __syncthreads();
  as_read(u);
  if constexpr (READ) as_read(q);
  if (on) {
    float h[W];
#pragma unroll
    for (int e = 0; e < W; ++e) h[e] = sm.U[rg * cw + cl * W + e];
    if (a.keep && (r0 + row) % kKeepRows == 0 && left > 0)
#pragma unroll
      for (int e = 0; e < W; ++e) a.keep[(r0 + row) / kKeepRows * a.C + c + e] = h[e];
    typename Elem<DT>::T *out = static_cast<typename Elem<DT>::T *>(a.o) + r0 * a.C;
    const uint32_t at = row * a.C + c;
    if (!some) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        Vec<DT, W> o;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          h[e] = fmaf(f[i][e], h[e], u[i][e]);
          o.set(e, READ ? h[e] * q[READ ? i : 0][e] : h[e]);
        }
        store_vec<DT, W>(out, at + static_cast<uint32_t>(i) * a.C, o);
      }
    } else {
#pragma unroll
      for (int i0 = 0; i0 < R; i0 += B) {
        int m[B];
        States<W> s0[B];
#pragma unroll
        for (int i = 0; i < B; ++i) m[i] = sm.mark[row + i0 + i];
        load_states(s0, a.h0, m, a.C, c);
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const int n = sm.fin[row + i0 + i];
          Vec<DT, W> o;
#pragma unroll
          for (int e = 0; e < W; ++e) {
            h[e] = fmaf(f[i0 + i][e], m[i] >= 0 ? s0[i].x[e] : h[e], u[i0 + i][e]);
            o.set(e, m[i] == kOutside ? 0.f : READ ? h[e] * q[READ ? i0 + i : 0][e] : h[e]);
          }
          if (a.ht && n >= 0) {
            States<W> out_state;
#pragma unroll
            for (int e = 0; e < W; ++e) out_state.x[e] = h[e];
            *reinterpret_cast<States<W> *>(a.ht + static_cast<int64_t>(n) * a.C + c) = out_state;
          }
          if (i0 + i < left) store_vec<DT, W>(out, at + static_cast<uint32_t>(i0 + i) * a.C, o);
        }
      }
    }
  }
  if (a.ht) empty_states(a, a.h0, a.ht, k, cb, cw, sm.flags);
}

// ----------------------------------------------------------------- backward --
template <int DT, int DTG, int W, bool READ, int SPAN>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(4))) void scan_bwd_kernel(const ScanArgs a) {
  constexpr int R = kBwdRows;
  static_assert(R == 4, "rows whose states are read at once");
  __shared__ TileSmem sm;
  __shared__ float sE[kMostValues];
  const int tid = threadIdx.x, cw = a.CT * W, rows = a.RG * R;
  const int rg = tid / a.CT, cl = tid - rg * a.CT;
  const Span all = a.n_seq ? Span{span_of(a, 0).b, span_of(a, a.n_seq - 1).e} : Span{0, 0};
  const Span mine = tid < a.n_seq ? span_of(a, tid) : Span{0, 0};
  const int id = take_tile(a, &sm.slot);
  const int back = id / a.cblocks, k = a.tiles - 1 - back, cb = id - back * a.cblocks;
  if (a.T == 0) {
    if (a.dh0) empty_states(a, a.dht, a.dh0, k, cb, cw, sm.flags);
    return;
  }
  const int64_t r0 = static_cast<int64_t>(k) * rows;
  const int row = rg * R;
  const int exist = static_cast<int>(min(a.T - r0, static_cast<int64_t>(rows))), left = exist - row;
  const bool on = rg < a.RG && (cb * a.CT + cl) * W < a.C;
  const int c = on ? (cb * a.CT + cl) * W : 0;   // (lanes without a channel read the first)
  Vec<DT, W> u[R], q[READ ? R : 1], d[R];
  Vec<DTG, W> g[R];
  load_rows<DT, W, R>(u, a.u, r0, a.ldu, row, exist - 1, c);
  load_rows<DTG, W, R>(g, a.g, r0, a.ldg, row, exist - 1, c);
  load_rows<DT, W, R>(d, a.dout, r0, a.C, row, exist - 1, c);
  if constexpr (READ) load_rows<DT, W, R>(q, a.q, r0, a.ldq, row, exist - 1, c);
  // (the forward left the state that enters the tile)
  const float entering = tid < cw && cb * cw + tid < a.C ? a.keep[r0 / kKeepRows * a.C + cb * cw + tid] : 0.f;
  if (tid < cw) sm.flags[tid] = 0;   // (mark_rows waits)
  const bool some = mark_rows(a, mine, all, r0, rows, sm.mark, sm.fin);
  Gate f[R][W];
  auto grad_of = [&](int i, int e) { return READ ? d[i][e] * q[READ ? i : 0][e] : d[i][e]; };
  by_kind(a.gate, [&](auto kind) { each<R, W>([&](int i, int e) { f[i][e] = gate_of<kind()>(g[i][e]); }); });
  if (on) {
    float A[W], U[W], E[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      A[e] = 1.f;
      U[e] = E[e] = 0.f;
    }
    bool reset = false;
    if (!some) {
      each<R, W>([&](int i, int e) {
        U[e] = fmaf(f[i][e].a, U[e], u[i][e]);
        A[e] *= f[i][e].a;
      });
      each<R, W>([&](int i, int e) { E[e] = f[R - 1 - i][e].a * (grad_of(R - 1 - i, e) + E[e]); });
    } else {
      int m[R], n[R];
      States<W> s0[R];   // (states, then gradients of final ones)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        m[i] = sm.mark[row + i];
        n[i] = sm.fin[row + i];
      }
      load_states(s0, a.h0, m, a.C, c);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        reset |= m[i] != kInside || n[i] >= 0;   // (nothing goes past a beginning or an end)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          U[e] = m[i] == kOutside ? 0.f : fmaf(f[i][e].a, m[i] >= 0 ? s0[i].x[e] : U[e], u[i][e]);
          A[e] *= f[i][e].a;
        }
      }
      load_states(s0, a.dht, n, a.C, c);
#pragma unroll
      for (int i = R - 1; i >= 0; --i) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float x = n[i] >= 0 ? s0[i].x[e] : E[e];
          E[e] = m[i] == kInside ? f[i][e].a * (grad_of(i, e) + x) : 0.f;
        }
      }
    }
    settle<R, W>(A, sm.flags + cl * W, [&](int i, int e) { return f[i][e].a; });
#pragma unroll
    for (int e = 0; e < W; ++e) {
      sm.A[rg * cw + cl * W + e] = A[e];
      sm.U[rg * cw + cl * W + e] = U[e];
      sE[rg * cw + cl * W + e] = E[e];
    }
    if (cl == 0) sm.cut[rg] = reset;
  }
  __syncthreads();
  // the first threads take the states forward, those from half on the gradients back
  if (tid < cw && cb * cw + tid < a.C) enter_groups<false>(sm.A, sm.U, sm.cut, a.RG, cw, tid, entering);
  enter_tile<true, SPAN>(a, sm, sE, back, cb, some && (sm.mark[rows - 1] == kOutside || sm.fin[rows - 1] >= 0), cw, kBlock / 2);
  __syncthreads();
  as_read(u);
  as_read(d);
  if constexpr (READ) as_read(q);
  if (on) {
    float h[W], x[W], before[R][W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      h[e] = sm.U[rg * cw + cl * W + e];
      x[e] = sE[rg * cw + cl * W + e];
    }
    const int64_t first = r0 * a.C;
    const uint32_t at = row * a.C + c;
    typedef typename Elem<DT>::T TU;
    typedef typename Elem<DTG>::T TG;
    int mark[R], fin[R];
    States<W> s0[R];   // (states, then gradients of final ones)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      mark[i] = some ? sm.mark[row + i] : kInside;
      fin[i] = some ? sm.fin[row + i] : -1;
    }
    if (some) load_states(s0, a.h0, mark, a.C, c);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int m = mark[i];
      Vec<DT, W> dq;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (m >= 0) h[e] = s0[i].x[e];
        before[i][e] = h[e];
        h[e] = fmaf(f[i][e].a, h[e], u[i][e]);
        dq.set(e, m == kOutside ? 0.f : d[i][e] * h[e]);
      }
      if (READ && i < left) store_vec<DT, W>(static_cast<TU *>(a.dq) + first, at + static_cast<uint32_t>(i) * a.C, dq);
    }
    if (some) load_states(s0, a.dht, fin, a.C, c);
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      const int m = mark[i], n = fin[i];
      Vec<DT, W> du;
      Vec<DTG, W> dg;
      States<W> first_grad;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if (n >= 0) x[e] = s0[i].x[e];
        const float s = grad_of(i, e) + x[e];
        du.set(e, m == kOutside ? 0.f : s);
        dg.set(e, m == kOutside ? 0.f : s * before[i][e] * f[i][e].slope);
        x[e] = f[i][e].a * s;
        first_grad.x[e] = x[e];
      }
      if (m >= 0 && a.dh0) *reinterpret_cast<States<W> *>(a.dh0 + static_cast<int64_t>(m) * a.C + c) = first_grad;
      if (i < left) {
        store_vec<DT, W>(static_cast<TU *>(a.du) + first, at + static_cast<uint32_t>(i) * a.C, du);
        store_vec<DTG, W>(static_cast<TG *>(a.dg) + first, at + static_cast<uint32_t>(i) * a.C, dg);
      }
    }
  }
  if (a.dh0) empty_states(a, a.dht, a.dh0, k, cb, cw, sm.flags);
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
// W channels a thread.
template <int DT, int DTG, int W>
__global__ __launch_bounds__(256) void scan_step_kernel(const StepArgs a) {
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int cv = a.C / W;
  if (x >= static_cast<int64_t>(a.n) * cv) return;
  const int64_t i = x / cv;
  const int c = static_cast<int>(x - i * cv) * W, row = a.at[i];
  Vec<DT, W> o;
  if (row < 0 || row >= a.rows || (i > 0 && a.at[i - 1] >= row)) {
#pragma unroll
    for (int e = 0; e < W; ++e) o.set(e, 0.f);
    store_vec<DT, W>(a.o, i * a.C + c, o);
    if (a.status) __hip_atomic_store(a.status, SSLA_ERR_ARG, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return;
  }
  const Vec<DT, W> u = load_vec<DT, W>(a.u, i * a.ldu + c);
  const Vec<DTG, W> g = load_vec<DTG, W>(a.g, i * a.ldg + c);
  Vec<DT, W> q;
  if (a.q) q = load_vec<DT, W>(a.q, i * a.ldq + c);
  States<W> &s = *reinterpret_cast<States<W> *>(a.state + static_cast<int64_t>(row) * a.C + c);
  States<W> h = s;
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const float f = a.gate == kSigmoid ? gate_value<kSigmoid>(g[e]) : a.gate == kLog ? gate_value<kLog>(g[e]) : g[e];
    h.x[e] = fmaf(f, h.x[e], u[e]);
    o.set(e, a.q ? h.x[e] * q[e] : h.x[e]);
  }
  s = h;
  store_vec<DT, W>(a.o, i * a.C + c, o);
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
  if (C > kMostWidth || (T > 1 && (ldu > kMostWidth || ldg > kMostWidth || ldq > kMostWidth))) {
    set_error("%s: rows of more than %d values, or that far apart", what, kMostWidth);
    return SSLA_ERR_UNSUPPORTED;
  }
  // (the kernels add sequences, tiles and threads in 32 bits)
  if (T > (1ll << 40) / C || static_cast<int64_t>(n_seq) * C > (1ll << 38) || n_seq > 1 << 30) {
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

// How the rows and channels are cut for vectors of W values and R rows a lane: up to kMostLanes lanes a
// row, as many row groups as a workgroup has room for (a power of two, so that a
// tile is a multiple of kKeepRows rows).
struct ScanPlan {
  int CT, RG, cblocks, span;
  int64_t tiles;
};
ScanPlan plan_of(int64_t T, int C, int W, int R) {
  ScanPlan p;
  const int cv = C / W;
  p.CT = (cv + (cv + kMostLanes - 1) / kMostLanes - 1) / ((cv + kMostLanes - 1) / kMostLanes);
  p.cblocks = (cv + p.CT - 1) / p.CT;
  p.RG = kKeepRows / R;
  while (2 * p.RG * p.CT <= kBlock && p.RG < kMostGroups) p.RG *= 2;
  p.tiles = std::max<int64_t>(1, (T + p.RG * R - 1) / (p.RG * R));
  // Some 512 workgroups run at once.  Over few channel blocks that is a long chain of tiles
  // each, which spans shorten (one sequence, spans of 16 against 1: 262,144 rows of 64 channels
  // 58 us, 95; 65,536 of 96 31, 42; of 256 55, 55); over more blocks spans are one wait more
  // (65,536 of 1,024 139, 133; 16,384 of 512 32, 30).
  p.span = p.cblocks <= 4 ? kSpanLog2 : 0;
  return p;
}
constexpr size_t kHead = 256;   // the ticket's line
constexpr int64_t kMostThreads = 0xffffffff;   // of a launch
int64_t word_count(const ScanPlan &p, int W) {   // words and hints
  const int64_t spans = p.tiles >> p.span;
  return ((p.span ? p.tiles : 0) + spans) * p.cblocks * p.CT * W + (spans * p.cblocks + 1) / 2;
}
size_t ws_bytes(int64_t T, int C) {   // whatever vectors the addresses allow
  int64_t most = 0;
  for (int W = 1; W <= 4; W *= 4)
    if (C % W == 0)
      for (int R : {kFwdRows, kBwdRows}) {
        const ScanPlan p = plan_of(T, C, W, R);
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

// Sets the plan, clears the words and launches `kernel`, or `spans` where there are any.
template <typename Kernel>
int launch_scan(const char *what, ScanArgs &a, int W, int R, Kernel kernel, Kernel spans, void *workspace, size_t workspace_bytes, hipStream_t st) {
  const ScanPlan p = plan_of(a.T, a.C, W, R);
  const size_t need = p.tiles > 1 ? kHead + static_cast<size_t>(word_count(p, W)) * 8 : 0;
  if (need && !(workspace && workspace_bytes >= need && aligned(workspace, 16))) {
    set_error("%s: needs %zu bytes of workspace, got %zu", what, ws_bytes(a.T, a.C), workspace_bytes);
    return SSLA_ERR_WORKSPACE;
  }
  if (p.tiles * p.cblocks > kMostThreads / kBlock) {
    set_error("%s: too many workgroups", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  a.CT = p.CT; a.RG = p.RG; a.cblocks = p.cblocks; a.tiles = static_cast<int>(p.tiles);
  if (need) {
    const int64_t n = word_count(p, W);
    a.ticket = static_cast<uint32_t *>(workspace);
    const int64_t wide = static_cast<int64_t>(p.cblocks) * p.CT * W;
    a.words = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + kHead);
    a.span_words = a.words + (p.span ? p.tiles * wide : 0);
    a.hints = reinterpret_cast<uint32_t *>(a.span_words + (p.tiles >> p.span) * wide);
    hipLaunchKernelGGL(scan_clear_kernel, dim3(static_cast<unsigned>(std::min<int64_t>((n + 1023) / 1024, 2048))), dim3(256), 0,
                       st, a.ticket, a.words, n);
  }
  hipLaunchKernelGGL(need && p.span ? spans : kernel, dim3(static_cast<unsigned>(p.tiles * p.cblocks)), dim3(kBlock), 0, st, a);
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
  const int W = widest(C, 4, {{u, ldu, dtype}, {g, ldg, g_dtype}, {q, q ? ldq : 0, dtype}, {o, C, dtype}});
  const hipStream_t st = static_cast<hipStream_t>(stream);
  int status = SSLA_OK;
#define SSLA_LAUNCH(D, G, W_) \
  status = q ? launch_scan("gated_scan_fwd", a, W_, kFwdRows, scan_fwd_kernel<D, G, W_, true, 0>, scan_fwd_kernel<D, G, W_, true, kSpanLog2>,    \
                           workspace, workspace_bytes, st)                                                                         \
             : launch_scan("gated_scan_fwd", a, W_, kFwdRows, scan_fwd_kernel<D, G, W_, false, 0>, scan_fwd_kernel<D, G, W_, false, kSpanLog2>, \
                           workspace, workspace_bytes, st)
#define SSLA_CALL(D, G)             \
  if (W == 4) SSLA_LAUNCH(D, G, 4); \
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  int status = SSLA_OK;
#define SSLA_LAUNCH(D, G, W_) \
  status = q ? launch_scan("gated_scan_bwd", a, W_, kBwdRows, scan_bwd_kernel<D, G, W_, true, 0>, scan_bwd_kernel<D, G, W_, true, kSpanLog2>,    \
                           workspace, workspace_bytes, st)                                                                         \
             : launch_scan("gated_scan_bwd", a, W_, kBwdRows, scan_bwd_kernel<D, G, W_, false, 0>, scan_bwd_kernel<D, G, W_, false, kSpanLog2>, \
                           workspace, workspace_bytes, st)
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
  const int W = widest(C, 4, {{u, ldu, dtype}, {g, ldg, g_dtype}, {q, q ? ldq : 0, dtype}, {o, C, dtype}});
  const int64_t blocks = (static_cast<int64_t>(n_active) * (C / W) + 255) / 256;
  if (blocks > kMostThreads / 256) {
    set_error("sparse_gated_step: too many workgroups");
    return SSLA_ERR_UNSUPPORTED;
  }
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SSLA_CALL(D, G)                                                                \
  if (W == 4) hipLaunchKernelGGL((scan_step_kernel<D, G, 4>), grid, block, 0, st, a);   \
  else hipLaunchKernelGGL((scan_step_kernel<D, G, 1>), grid, block, 0, st, a)
  SSLA_SCAN_TYPES(SSLA_CALL);
#undef SSLA_CALL
  return launch_status("sparse_gated_step");
}

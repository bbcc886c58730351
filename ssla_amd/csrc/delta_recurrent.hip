// Gated delta rule on gfx950, token by token: per sequence and head
//   S <- e^(g_t) S,  u_t = beta_t (v_t - S^T k_t),  S <- S + k_t u_t^T,
//   o_t = scale S^T q_t.
// Both products read the state before the token's write: with r = S^T k and
// p = S^T q of the old state, u = beta (v - e^g r), o = scale (e^g p +
// (k . q) u) and S <- e^g S + k u^T, so a token waits on one reduction over
// the keys, not on two.
//
// One wavefront per (sequence, head, 16 value columns): lane = (key group of
// four, column), each holding KR state rows in fp32.  The value columns of a
// state are independent of each other.
#include "common.h"

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
  int64_t T;
  int n_seq, Hk, H, K, V, n_rows;
  float scale;
};

template <int KR, int DT>
__global__ __launch_bounds__(256) void delta_recurrent_kernel(const DeltaArgs a) {
  typedef Elem<DT> E;
  const int lane = threadIdx.x & 63;
  const int n_vt = (a.V + 15) >> 4;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= static_cast<int64_t>(a.n_seq) * a.H * n_vt) return;   // whole wavefront
  const int vt = static_cast<int>(item % n_vt), h = static_cast<int>((item / n_vt) % a.H);
  const int n = static_cast<int>(item / (static_cast<int64_t>(n_vt) * a.H));
  const int hk = h / (a.H / a.Hk);
  const int col = vt * 16 + (lane & 15), k0 = (lane >> 4) * KR;
  const bool col_ok = col < a.V;

  // (clamped to [0, T): no offset addresses memory outside the tensors)
  int64_t bos = n, eos = n + 1;
  if (a.cu) {
    bos = min(max(a.cu[n], (int64_t)0), a.T);
    eos = min(max(a.cu[n + 1], bos), a.T);
  }
  int64_t row = n;
  if (a.row_of) {
    row = a.row_of[n];
    if (row < 0 || row >= a.n_rows || (n > 0 && a.row_of[n - 1] >= row)) {
      if (a.status && lane == 0)
        __hip_atomic_store(a.status, SSLA_ERR_ARG, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      for (int64_t t = bos; t < eos; ++t)
        if (lane < 16 && col_ok) E::store(a.o, (t * a.H + h) * a.V + col, 0.f);
      return;
    }
  }

  const int64_t s0 = (row * a.H + h) * a.K;
  float S[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i)
    S[i] = (a.h0 && col_ok && k0 + i < a.K) ? a.h0[(s0 + k0 + i) * a.V + col] : 0.f;

  for (int64_t t = bos; t < eos; ++t) {
    const float eg = fast_exp2(a.g[t * a.H + h] * kLog2e), b = a.beta[t * a.H + h];
    const float vv = col_ok ? E::load(a.v, (t * a.H + h) * a.V + col) : 0.f;
    const int64_t kb = (t * a.Hk + hk) * a.K + k0;
    float kk[KR], r = 0.f, p = 0.f, kq = 0.f;
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const bool ok = k0 + i < a.K;
      kk[i] = ok ? E::load(a.k, kb + i) : 0.f;
      const float qq = ok ? E::load(a.q, kb + i) : 0.f;
      r = fmaf(kk[i], S[i], r);
      p = fmaf(qq, S[i], p);
      kq = fmaf(kk[i], qq, kq);
    }
    r += __shfl_xor(r, 16);
    p += __shfl_xor(p, 16);
    kq += __shfl_xor(kq, 16);
    r += __shfl_xor(r, 32);
    p += __shfl_xor(p, 32);
    kq += __shfl_xor(kq, 32);
    const float u = b * fmaf(-eg, r, vv);
#pragma unroll
    for (int i = 0; i < KR; ++i) S[i] = fmaf(kk[i], u, eg * S[i]);
    if (lane < 16 && col_ok) E::store(a.o, (t * a.H + h) * a.V + col, a.scale * fmaf(kq, u, eg * p));
  }

  if (a.ht && col_ok) {
#pragma unroll
    for (int i = 0; i < KR; ++i)
      if (k0 + i < a.K) a.ht[(s0 + k0 + i) * a.V + col] = S[i];
  }
}

template <int DT>
int launch_delta(const DeltaArgs &a, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(a.n_seq) * a.H * ((a.V + 15) / 16);
  const int64_t blocks = (items + 3) / 4;
  if (blocks > 0x7fffffff) {
    set_error("gated_delta_recurrent: too many (sequence, head, tile) items");
    return SSLA_ERR_UNSUPPORTED;
  }
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
#define SSLA_DELTA(KR_) hipLaunchKernelGGL((delta_recurrent_kernel<KR_, DT>), grid, block, 0, st, a)
  if (a.K <= 16) SSLA_DELTA(4);
  else if (a.K <= 32) SSLA_DELTA(8);
  else if (a.K <= 64) SSLA_DELTA(16);
  else if (a.K <= 128) SSLA_DELTA(32);
  else SSLA_DELTA(64);
#undef SSLA_DELTA
  return launch_status("gated_delta_recurrent");
}

}  // namespace
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
  const DeltaArgs a{q, k, v, g, beta, cu_seqlens, state_idx, h0, ht, o, status, T, n_seq, Hk, H, K, V, n_state_rows,
                    scale};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SSLA_F32: return launch_delta<SSLA_F32>(a, st);
    case SSLA_BF16: return launch_delta<SSLA_BF16>(a, st);
    case SSLA_F16: return launch_delta<SSLA_F16>(a, st);
  }
  set_error("gated_delta_recurrent: unsupported dtype %d", dtype);
  return SSLA_ERR_DTYPE;
}

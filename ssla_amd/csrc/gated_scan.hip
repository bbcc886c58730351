// Gated linear recurrence over packed sequences, per channel:
//   h_t = a_t h_{t-1} + u_t,  a_t = g_t, e^(g_t) or sigmoid(g_t),  o_t = q_t h_t (or h_t)
// with its backward, from an initial state to the final one.  With e_t the
// gradient of h_t:
//   e_t = q_t do_t + a_{t+1} e_{t+1} (dht_n behind a sequence's last row)
//   du_t = e_t,  da_t = e_t h_{t-1},  dq_t = do_t h_t,  dh0_n = a_first e_first
// A thread walks one channel of one sequence.
#include "common.h"

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

struct ScanArgs {
  const void *u, *g, *q, *dout;   // q may be NULL
  int64_t ldu, ldg, ldq;          // elements from row to row
  const int64_t *cu;
  int n_seq;
  int64_t T;
  int C, gate;
  const float *h0, *dht;          // may be NULL
  void *o, *du, *dg, *dq;
  float *ht, *dh0, *keep;         // may be NULL
};

__device__ __forceinline__ void bounds(const ScanArgs &a, int n, int64_t &b, int64_t &e) {
  b = min(max(a.cu[n], (int64_t)0), a.T);
  e = min(max(a.cu[n + 1], b), a.T);
}

template <int DT, int DTG>
__global__ __launch_bounds__(256) void scan_fwd_kernel(const ScanArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(a.n_seq) * a.C) return;
  const int n = static_cast<int>(i / a.C), c = static_cast<int>(i % a.C);
  int64_t b, e;
  bounds(a, n, b, e);
  float h = a.h0 ? a.h0[i] : 0.f;
  for (int64_t t = b; t < e; ++t) {
    const float gate = gate_of(a.gate, Elem<DTG>::load(a.g, t * a.ldg + c)).a;
    h = fmaf(gate, h, Elem<DT>::load(a.u, t * a.ldu + c));
    Elem<DT>::store(a.o, t * a.C + c, a.q ? h * Elem<DT>::load(a.q, t * a.ldq + c) : h);
    if (a.keep) a.keep[t * a.C + c] = h;
  }
  if (a.ht) a.ht[i] = h;
}

template <int DT, int DTG>
__global__ __launch_bounds__(256) void scan_bwd_kernel(const ScanArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(a.n_seq) * a.C) return;
  const int n = static_cast<int>(i / a.C), c = static_cast<int>(i % a.C);
  int64_t b, e;
  bounds(a, n, b, e);
  float d = a.dht ? a.dht[i] : 0.f;
  for (int64_t t = e - 1; t >= b; --t) {
    const Gate gate = gate_of(a.gate, Elem<DTG>::load(a.g, t * a.ldg + c));
    float s = Elem<DT>::load(a.dout, t * a.C + c);
    if (a.q) {
      Elem<DT>::store(a.dq, t * a.C + c, s * a.keep[t * a.C + c]);
      s *= Elem<DT>::load(a.q, t * a.ldq + c);
    }
    s += d;
    const float before = t > b ? a.keep[(t - 1) * a.C + c] : a.h0 ? a.h0[i] : 0.f;
    Elem<DT>::store(a.du, t * a.C + c, s);
    Elem<DTG>::store(a.dg, t * a.C + c, s * before * gate.slope);
    d = gate.a * s;
  }
  if (a.dh0) a.dh0[i] = d;
}

// Zeros on the rows in no sequence.
template <int DT>
__global__ __launch_bounds__(256) void scan_outside_kernel(const ScanArgs a, void *x) {
  const int64_t lo = a.n_seq ? min(max(a.cu[0], (int64_t)0), a.T) : a.T;
  const int64_t hi = a.n_seq ? min(max(a.cu[a.n_seq], lo), a.T) : a.T;
  const int64_t head = lo * a.C, all = head + (a.T - hi) * a.C;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256)
    Elem<DT>::store(x, i < head ? i : hi * a.C + i - head, 0.f);
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

}  // namespace
}  // namespace ssla

extern "C" size_t ssla_gated_scan_workspace_size(int64_t, int) { return 0; }

extern "C" size_t ssla_gated_scan_keep_size(int64_t T, int C) {
  return T > 0 && C > 0 ? static_cast<size_t>(T) * C * sizeof(float) : 0;
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  ScanArgs a{};
  a.u = u; a.g = g; a.q = q; a.ldu = ldu; a.ldg = ldg; a.ldq = ldq;
  a.cu = cu_seqlens; a.n_seq = n_seq; a.T = T; a.C = C; a.gate = gate;
  a.h0 = h0; a.o = o; a.ht = ht; a.keep = static_cast<float *>(keep);
  const int64_t blocks = (static_cast<int64_t>(n_seq) * C + 255) / 256;
#define SSLA_CALL(D, G)                                                                                               \
  if (n_seq > 0) hipLaunchKernelGGL((scan_fwd_kernel<D, G>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a); \
  if (T > 0) hipLaunchKernelGGL((scan_outside_kernel<D>), dim3(64), dim3(256), 0, st, a, a.o)
  SSLA_SCAN_TYPES(SSLA_CALL);
#undef SSLA_CALL
  return launch_status("gated_scan_fwd");
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  ScanArgs a{};
  a.u = u; a.g = g; a.q = q; a.dout = dout; a.ldu = ldu; a.ldg = ldg; a.ldq = ldq;
  a.cu = cu_seqlens; a.n_seq = n_seq; a.T = T; a.C = C; a.gate = gate;
  a.h0 = h0; a.dht = dht; a.du = du; a.dg = dg; a.dq = dq; a.dh0 = dh0;
  a.keep = static_cast<float *>(const_cast<void *>(keep));
  const int64_t blocks = (static_cast<int64_t>(n_seq) * C + 255) / 256;
#define SSLA_CALL(D, G)                                                                                               \
  if (n_seq > 0) hipLaunchKernelGGL((scan_bwd_kernel<D, G>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a); \
  if (T > 0) {                                                                                                        \
    hipLaunchKernelGGL((scan_outside_kernel<D>), dim3(64), dim3(256), 0, st, a, a.du);                                \
    hipLaunchKernelGGL((scan_outside_kernel<G>), dim3(64), dim3(256), 0, st, a, a.dg);                                \
    if (q) hipLaunchKernelGGL((scan_outside_kernel<D>), dim3(64), dim3(256), 0, st, a, a.dq);                         \
  }
  SSLA_SCAN_TYPES(SSLA_CALL);
#undef SSLA_CALL
  return launch_status("gated_scan_bwd");
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

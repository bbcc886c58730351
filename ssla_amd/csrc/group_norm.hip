// Group norm with an activation, channels last, on gfx950:
//   y = act((x - mean) rstd w + b)
// over the positions of a sample and the C / G channels of a group, with its
// backward.  x is [N, L, C]: a group's values are L runs of C / G channels.
// Sums are fp32; the variance is that of the centred values.
#include "common.h"

namespace ssla {
namespace {

constexpr int kNone = SSLA_ACT_NONE, kRelu = SSLA_ACT_RELU, kSilu = SSLA_ACT_SILU;

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

__device__ __forceinline__ float block_sum(float x, float *sm) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = x;
  __syncthreads();
  return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// One workgroup per (sample, group).
template <int DT>
__global__ __launch_bounds__(256) void group_norm_fwd_kernel(const void *__restrict__ x, int64_t L, int C, int G,
                                                             const float *__restrict__ w, const float *__restrict__ b,
                                                             float eps, int act, void *__restrict__ y,
                                                             float *__restrict__ stats) {
  typedef Elem<DT> E;
  __shared__ float sm[4];
  const int64_t n = blockIdx.x / G;
  const int g = static_cast<int>(blockIdx.x % G), per = C / G;
  const int64_t base = n * L * C + g * per, m = L * per;
  auto at = [&](int64_t i) { return base + (i / per) * C + i % per; };
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < m; i += 256) s += E::load(x, at(i));
  const float mean = block_sum(s, sm) / static_cast<float>(m);
  s = 0.f;
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    const float d = E::load(x, at(i)) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = 1.f / sqrtf(block_sum(s, sm) / static_cast<float>(m) + eps);
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    const int c = g * per + static_cast<int>(i % per);
    const float z = fmaf((E::load(x, at(i)) - mean) * rstd, w ? w[c] : 1.f, b ? b[c] : 0.f);
    E::store(y, at(i), act_of(act, z));
  }
  if (stats && threadIdx.x == 0) {
    stats[2 * static_cast<int64_t>(blockIdx.x)] = mean;
    stats[2 * static_cast<int64_t>(blockIdx.x) + 1] = rstd;
  }
}

// dx: with h = dy act'(z) w and x^ = (x - mean) rstd,
//   dx = rstd (h - mean(h) - x^ mean(h x^)).
template <int DT>
__global__ __launch_bounds__(256) void group_norm_dx_kernel(const void *__restrict__ dy, const void *__restrict__ x,
                                                            const float *__restrict__ stats, int64_t L, int C, int G,
                                                            const float *__restrict__ w, const float *__restrict__ b,
                                                            int act, void *__restrict__ dx) {
  typedef Elem<DT> E;
  __shared__ float sm[4];
  const int64_t n = blockIdx.x / G;
  const int g = static_cast<int>(blockIdx.x % G), per = C / G;
  const int64_t base = n * L * C + g * per, m = L * per;
  const float mean = stats[2 * static_cast<int64_t>(blockIdx.x)], rstd = stats[2 * static_cast<int64_t>(blockIdx.x) + 1];
  auto at = [&](int64_t i) { return base + (i / per) * C + i % per; };
  auto grad = [&](int64_t i, float &xh) {
    const int c = g * per + static_cast<int>(i % per);
    xh = (E::load(x, at(i)) - mean) * rstd;
    const float wc = w ? w[c] : 1.f;
    return E::load(dy, at(i)) * act_grad(act, fmaf(xh, wc, b ? b[c] : 0.f)) * wc;
  };
  float s0 = 0.f, s1 = 0.f;
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    float xh;
    const float h = grad(i, xh);
    s0 += h;
    s1 = fmaf(h, xh, s1);
  }
  s0 = block_sum(s0, sm) / static_cast<float>(m);
  s1 = block_sum(s1, sm) / static_cast<float>(m);
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    float xh;
    const float h = grad(i, xh);
    E::store(dx, at(i), rstd * (h - s0 - xh * s1));
  }
}

// dw_c = sum dy act'(z) x^, db_c = sum dy act'(z): one workgroup per channel.
template <int DT>
__global__ __launch_bounds__(256) void group_norm_dwb_kernel(const void *__restrict__ dy, const void *__restrict__ x,
                                                             const float *__restrict__ stats, int64_t N, int64_t L,
                                                             int C, int G, const float *__restrict__ w,
                                                             const float *__restrict__ b, int act,
                                                             float *__restrict__ dw, float *__restrict__ db) {
  typedef Elem<DT> E;
  __shared__ float sm[4];
  const int c = blockIdx.x, g = c / (C / G);
  const float wc = w ? w[c] : 1.f, bc = b ? b[c] : 0.f;
  float s0 = 0.f, s1 = 0.f;
  for (int64_t i = threadIdx.x; i < N * L; i += 256) {
    const int64_t n = i / L;
    const float xh = (E::load(x, i * C + c) - stats[2 * (n * G + g)]) * stats[2 * (n * G + g) + 1];
    const float d = E::load(dy, i * C + c) * act_grad(act, fmaf(xh, wc, bc));
    s0 += d;
    s1 = fmaf(d, xh, s1);
  }
  s0 = block_sum(s0, sm);
  s1 = block_sum(s1, sm);
  if (threadIdx.x == 0) {
    if (dw) dw[c] = s1;
    if (db) db[c] = s0;
  }
}

int check_sizes(const char *what, int64_t N, int64_t L, int C, int G, int act) {
  SSLA_CHECK_ARG(N >= 0 && L >= 0 && C > 0 && G > 0 && C % G == 0 && act >= kNone && act <= kSilu,
                 "%s: bad sizes N=%lld L=%lld C=%d G=%d act=%d", what, (long long)N, (long long)L, C, G, act);
  if (N * G > 0x7fffffff) {
    set_error("%s: too many groups", what);
    return SSLA_ERR_UNSUPPORTED;
  }
  return SSLA_OK;
}

}  // namespace
}  // namespace ssla

extern "C" size_t ssla_group_norm_workspace_size(int64_t N, int64_t L, int C, int G) {
  (void)N, (void)L, (void)C, (void)G;
  return 0;
}

extern "C" int ssla_group_norm_fwd(const void *x, int64_t N, int64_t L, int C, int G, const float *weight,
                                   const float *bias, float eps, int act, void *y, float *stats, int dtype,
                                   void *workspace, size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  (void)workspace, (void)workspace_bytes;
  if (const int e = check_sizes("group_norm_fwd", N, L, C, G, act)) return e;
  if (N == 0 || L == 0) return SSLA_OK;
  SSLA_CHECK_ARG(x && y, "group_norm_fwd: null pointer");
  const dim3 grid(static_cast<unsigned>(N * G)), block(256);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SSLA_GN(DT_) \
  hipLaunchKernelGGL((group_norm_fwd_kernel<DT_>), grid, block, 0, st, x, L, C, G, weight, bias, eps, act, y, stats)
  if (dtype == SSLA_F32) SSLA_GN(SSLA_F32);
  else if (dtype == SSLA_BF16) SSLA_GN(SSLA_BF16);
  else if (dtype == SSLA_F16) SSLA_GN(SSLA_F16);
  else {
    set_error("group_norm_fwd: unsupported dtype %d", dtype);
    return SSLA_ERR_DTYPE;
  }
#undef SSLA_GN
  return launch_status("group_norm_fwd");
}

extern "C" size_t ssla_group_norm_bwd_workspace_size(int64_t N, int64_t L, int C, int G) {
  (void)N, (void)L, (void)C, (void)G;
  return 0;
}

extern "C" int ssla_group_norm_bwd(const void *dy, const void *x, const float *stats, int64_t N, int64_t L, int C,
                                   int G, const float *weight, const float *bias, int act, void *dx, float *dweight,
                                   float *dbias, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace ssla;
  clear_error();
  (void)workspace, (void)workspace_bytes;
  if (const int e = check_sizes("group_norm_bwd", N, L, C, G, act)) return e;
  const bool none = N == 0 || L == 0;
  SSLA_CHECK_ARG(none || (dy && x && stats), "group_norm_bwd: null pointer");
  const dim3 grid(static_cast<unsigned>(N * G)), block(256);
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SSLA_GN(DT_)                                                                                                 \
  do {                                                                                                               \
    if (dx && !none)                                                                                                 \
      hipLaunchKernelGGL((group_norm_dx_kernel<DT_>), grid, block, 0, st, dy, x, stats, L, C, G, weight, bias, act,  \
                         dx);                                                                                        \
    if (dweight || dbias)                                                                                            \
      hipLaunchKernelGGL((group_norm_dwb_kernel<DT_>), dim3(C), block, 0, st, dy, x, stats, N, L, C, G, weight, bias, \
                         act, dweight, dbias);                                                                       \
  } while (0)
  if (dtype == SSLA_F32) SSLA_GN(SSLA_F32);
  else if (dtype == SSLA_BF16) SSLA_GN(SSLA_BF16);
  else if (dtype == SSLA_F16) SSLA_GN(SSLA_F16);
  else {
    set_error("group_norm_bwd: unsupported dtype %d", dtype);
    return SSLA_ERR_DTYPE;
  }
#undef SSLA_GN
  return launch_status("group_norm_bwd");
}

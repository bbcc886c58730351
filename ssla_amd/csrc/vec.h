// Neighbouring values read and written together.
#pragma once
#include "common.h"

namespace ssla {

template <int DT, int W>
struct Vec {
  typename Elem<DT>::T e[W];
  __device__ __forceinline__ float operator[](int i) const { return Elem<DT>::load(e, i); }
  __device__ __forceinline__ void set(int i, float x) {
    if constexpr (DT == SSLA_BF16) e[i] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    else Elem<DT>::store(e, i, x);
  }
};
// The border that a vector's address lies at: 16 bytes at most, as the callers check.
template <int DT, int W>
constexpr size_t vec_border() { return sizeof(Vec<DT, W>) < 16 ? sizeof(Vec<DT, W>) : 16; }
template <int DT, int W>
__device__ __forceinline__ Vec<DT, W> load_vec(const void *p, int64_t i) {
  struct __attribute__((aligned((vec_border<DT, W>())))) A { Vec<DT, W> v; };
  return reinterpret_cast<const A *>(static_cast<const typename Elem<DT>::T *>(p) + i)->v;
}
template <int DT, int W>
__device__ __forceinline__ void store_vec(void *p, int64_t i, const Vec<DT, W> &x) {
  struct __attribute__((aligned((vec_border<DT, W>())))) A { Vec<DT, W> v; };
  reinterpret_cast<A *>(static_cast<typename Elem<DT>::T *>(p) + i)->v = x;
}

// The same to be held for a while: as the words they came in.  (16-bit values of a Vec
// that are chosen or kept over a branch take a register each.)
template <int DT, int W>
struct Held {
  static constexpr int kBytes = static_cast<int>(sizeof(typename Elem<DT>::T)) * W, kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (DT == SSLA_F32) return __uint_as_float(w[e]);
    else if constexpr (DT == SSLA_BF16) return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    else return f16_bits_to_f32(static_cast<uint16_t>(e & 1 ? w[e >> 1] >> 16 : w[e >> 1]));
  }
};
template <int DT, int W>
__device__ __forceinline__ Held<DT, W> load_held(const void *p, int64_t i) {
  const typename Elem<DT>::T *at = static_cast<const typename Elem<DT>::T *>(p) + i;
  Held<DT, W> h;
  if constexpr (Held<DT, W>::kBytes < 4) {
    h.w[0] = *at;
  } else {
    typedef uint32_t V __attribute__((ext_vector_type(Held<DT, W>::kWords > 4 ? 4 : Held<DT, W>::kWords)));
    constexpr int n = Held<DT, W>::kWords > 4 ? 4 : Held<DT, W>::kWords;
#pragma unroll
    for (int k = 0; k < Held<DT, W>::kWords; k += n) {
      if constexpr (n == 1) {
        h.w[k] = *reinterpret_cast<const uint32_t *>(at);
      } else {
        const V v = *(reinterpret_cast<const V *>(at) + k / n);
#pragma unroll
        for (int e = 0; e < n; ++e) h.w[k + e] = v[e];
      }
    }
  }
  return h;
}

}  // namespace ssla

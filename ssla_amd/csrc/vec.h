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
template <int DT, int W>
__device__ __forceinline__ Vec<DT, W> load_vec(const void *p, int64_t i) {
  struct __attribute__((aligned(sizeof(Vec<DT, W>)))) A { Vec<DT, W> v; };
  return reinterpret_cast<const A *>(static_cast<const typename Elem<DT>::T *>(p) + i)->v;
}
template <int DT, int W>
__device__ __forceinline__ void store_vec(void *p, int64_t i, const Vec<DT, W> &x) {
  struct __attribute__((aligned(sizeof(Vec<DT, W>)))) A { Vec<DT, W> v; };
  reinterpret_cast<A *>(static_cast<typename Elem<DT>::T *>(p) + i)->v = x;
}

}  // namespace ssla

// Element types and unaligned vector access of the kernels that take fp32, bf16 and fp16 tensors of any alignment
// (embedding.hip, grad_norm.hip).
#pragma once
#include "nr_common.h"

namespace {

// N elements of T at an address that is aligned to T only: one wide access (gfx950 reads and writes any byte address; the type
// says so to the compiler, which would split a plain vector access that it cannot prove aligned)
template <typename T, int N>
struct alignas(alignof(T)) NrPack {
  typedef T vec __attribute__((ext_vector_type(N), aligned(alignof(T))));
  vec v;
};

template <typename T, int N>
__device__ __forceinline__ void nr_load_pack(const T* __restrict__ p, float (&x)[N]) {
  const auto v = reinterpret_cast<const NrPack<T, N>*>(p)->v;
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = (float)v[k];
}
// one rounding to T (to nearest even), of a value held in fp32
template <typename T, int N>
__device__ __forceinline__ void nr_store_pack(T* __restrict__ p, const float (&x)[N]) {
  typename NrPack<T, N>::vec v;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = (T)x[k];
  reinterpret_cast<NrPack<T, N>*>(p)->v = v;
}
// the same without a place in the caches, for results that are larger than those: what they would push out is read again
template <typename T, int N>
__device__ __forceinline__ void nr_store_pack_stream(T* __restrict__ p, const float (&x)[N]) {
  typename NrPack<T, N>::vec v;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = (T)x[k];
  __builtin_nontemporal_store(v, reinterpret_cast<typename NrPack<T, N>::vec*>(p));
}
// Results beyond this size leave through nr_store_pack_stream: the 256 MB cache in front of the memory cannot hold them for
// whoever reads them next, and writing them past it leaves it to the inputs.  Measured: 537 MB of rows from a table of 268 MB
// 171 -> 114 us; a norm (613 MB) after a scaling that wrote as much 124 -> 94 us; 134 MB the same either way.
constexpr int64_t kStreamBytes = (int64_t)256 << 20;
// the first m of N elements (the end of a row or of a tensor)
template <typename T, int N>
__device__ __forceinline__ void nr_load_some(const T* __restrict__ p, int m, float (&x)[N]) {
  if (m >= N) {
    nr_load_pack<T, N>(p, x);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = k < m ? (float)p[k] : 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void nr_store_some(T* __restrict__ p, int m, const float (&x)[N]) {
  if (m >= N) {
    nr_store_pack<T, N>(p, x);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < m) p[k] = (T)x[k];
  }
}

}  // namespace

// Element types and unaligned vector access of the kernels that take fp32, bf16 and fp16 tensors of any alignment
// (embedding.hip, grad_norm.hip).
#pragma once
#include <type_traits>

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
// One rounding to T (to nearest even) of a value held in fp32.  The compiler may form a product and round it to fp16 in one instruction
// (v_fma_mixlo_f16: once, not first to fp32), and does so in some loops and not in others: an element's bits would depend on where in
// its tensor it lies.  So the value is taken as it stands in its register.
template <typename T>
__device__ __forceinline__ T nr_round(float x) {
  if constexpr (std::is_same_v<T, _Float16>) asm("" : "+v"(x));
  return (T)x;
}
template <typename T, int N>
__device__ __forceinline__ void nr_store_pack(T* __restrict__ p, const float (&x)[N]) {
  typename NrPack<T, N>::vec v;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = nr_round<T>(x[k]);
  reinterpret_cast<NrPack<T, N>*>(p)->v = v;
}
// the same without a place in the caches, for results that are larger than those: what they would push out is read again
template <typename T, int N>
__device__ __forceinline__ void nr_store_pack_stream(T* __restrict__ p, const float (&x)[N]) {
  typename NrPack<T, N>::vec v;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = nr_round<T>(x[k]);
  __builtin_nontemporal_store(v, reinterpret_cast<typename NrPack<T, N>::vec*>(p));
}
// Results beyond this size leave through nr_store_pack_stream: the 256 MB cache in front of the memory cannot hold them for
// whoever reads them next, and writing them past it leaves it to the inputs.  Measured: 537 MB of rows from a table of 268 MB
// 171 -> 114 us; a norm (613 MB) after a scaling that wrote as much 124 -> 94 us; 134 MB the same either way.
constexpr int64_t kStreamBytes = (int64_t)256 << 20;

// The first m of N elements (the end of a row or of a tensor): 8, 4 and 2 bytes, up to three accesses and not m.  The vector
// is held as two integers that are shifted, never as an array that is indexed, so that it stays in registers.  Measured against one
// element at a time: a gradient of 3 822 rows of 7 fp16 values 27 -> 14 us, a lookup of 200 000 rows of 5 6.6 -> 4.3.
template <typename W, typename T>
struct NrPiece {
  typedef W __attribute__((may_alias, aligned(alignof(T)))) type;
};
template <typename T, int N>
__device__ __forceinline__ void nr_load_some(const T* __restrict__ p, int m, float (&x)[N]) {
  if (m >= N) {
    nr_load_pack<T, N>(p, x);
    return;
  }
  if constexpr (N * sizeof(T) > 16) {
    float half[N / 2], rest[N / 2];
    nr_load_some<T, N / 2>(p, m, half);
    nr_load_some<T, N / 2>(p + N / 2, m > N / 2 ? m - N / 2 : 0, rest);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      x[k] = half[k];
      x[N / 2 + k] = rest[k];
    }
    return;
  }
  const int bytes = m * (int)sizeof(T);
  const char* at = reinterpret_cast<const char*>(p);
  uint64_t low = 0, eight = 0;
  if (bytes & 8) {
    eight = *reinterpret_cast<const typename NrPiece<uint64_t, T>::type*>(at);
    at += 8;
  }
  if (bytes & 4) {
    low = *reinterpret_cast<const typename NrPiece<uint32_t, T>::type*>(at);
    at += 4;
  }
  if (sizeof(T) == 2 && (bytes & 2)) {
    const uint64_t two = *reinterpret_cast<const typename NrPiece<uint16_t, T>::type*>(at);
    low |= (bytes & 4) ? two << 32 : two;
  }
  typedef uint64_t two64 __attribute__((ext_vector_type(2)));
  const two64 all = {(bytes & 8) ? eight : low, (bytes & 8) ? low : 0};
  typedef T whole __attribute__((ext_vector_type(16 / sizeof(T))));
  const whole v = __builtin_bit_cast(whole, all);
#pragma unroll
  for (int k = 0; k < N && k < (int)(16 / sizeof(T)); ++k) x[k] = (float)v[k];
}
template <typename T, int N>
__device__ __forceinline__ void nr_store_some(T* __restrict__ p, int m, const float (&x)[N]) {
  if (m >= N) {
    nr_store_pack<T, N>(p, x);
    return;
  }
  if constexpr (N * sizeof(T) > 16) {
    float half[N / 2], rest[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      half[k] = x[k];
      rest[k] = x[N / 2 + k];
    }
    nr_store_some<T, N / 2>(p, m, half);
    nr_store_some<T, N / 2>(p + N / 2, m > N / 2 ? m - N / 2 : 0, rest);
    return;
  }
  typedef uint64_t two64 __attribute__((ext_vector_type(2)));
  typedef T whole __attribute__((ext_vector_type(16 / sizeof(T))));
  whole v = {};
#pragma unroll
  for (int k = 0; k < N && k < (int)(16 / sizeof(T)); ++k) v[k] = nr_round<T>(x[k]);
  const two64 all = __builtin_bit_cast(two64, v);
  const int bytes = m * (int)sizeof(T);
  char* at = reinterpret_cast<char*>(p);
  uint64_t low = all[0];
  if (bytes & 8) {
    *reinterpret_cast<typename NrPiece<uint64_t, T>::type*>(at) = low;
    at += 8;
    low = all[1];
  }
  if (bytes & 4) {
    *reinterpret_cast<typename NrPiece<uint32_t, T>::type*>(at) = (uint32_t)low;
    at += 4;
    low >>= 32;
  }
  if (sizeof(T) == 2 && (bytes & 2)) *reinterpret_cast<typename NrPiece<uint16_t, T>::type*>(at) = (uint16_t)low;
}

}  // namespace

// The global norm of a list of gradients, and their clipping (torch.nn.utils.clip_grad_norm_; the reference clips a parameter
// group's gradients to `max_norm` in engine/optimizers.py).
//
//   N = (sum x^2)^(1/2), sum |x| or max |x| over every element of every tensor;  f = min(1, max_norm / (N + 1e-6));  y = round(f x)
//
// Bound by memory: the norm reads every element once, the clipping reads it again (the factor is known only when the last element
// has been seen) and writes it.  One launch covers up to kList tensors of any sizes and types: their addresses travel as kernel
// arguments (nothing is copied to the device, so a captured graph holds them), a block finds its tensor by bisection and takes one
// fixed piece of it.  Every block leaves one partial result; one block adds those up in order: the same bits on every call.
// Sums are held in fp64: a vector FMA in fp64 costs what one in fp32 does, and no square of an fp32 value over- or underflows in
// it.  NaN and infinity travel as in torch: the maximum compares bit patterns of |x|, where NaN is the largest.
// Measured: 153 M fp32 (613 MB) norm 95 to 97 us = 6.4 TB/s, finish 5 us, scaling into other buffers 214 us = 5.7 TB/s (a copy of this
// size: 5.0); 288 bf16 tensors of 134 MB in all: 3 x 10 + 3 + 3 x 15 us; 24 small tensors: 3.8 + 1.7 us, two launches; 75 tensors of
// 1.8 MB clipped: 4.4 + 5.2 us, two launches.
#include "rows_dev.h"

namespace {

constexpr int kThreads = 256;
constexpr int kList = 96;                    // tensors of one launch (kernel arguments: 3 KB of the 4 KB there are)
constexpr int kUnroll = 4;                   // 16-byte accesses in flight per thread
constexpr int kPiece = kThreads * kUnroll * 8;  // elements: pieces of whole batches for 16-bit and 32-bit types
constexpr int64_t kMaxBlocks = 16384;        // pieces that a list is cut into, about
constexpr int kFinishThreads = 1024;
constexpr int64_t kFew = 1024;               // partial results that a block adds up beside other work

enum { kNormMax = 0, kNormSum = 1, kNormTwo = 2 };

struct List {
  const void* in[kList];
  void* out[kList];
  int64_t numel[kList];
  uint32_t first[kList + 1];  // first block of each tensor
  uint8_t in_dtype[kList], out_dtype[kList];
  int count;
  int64_t piece;              // elements per block, a multiple of kPiece
};

__device__ __forceinline__ int tensor_of(const List& l, uint32_t block) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (l.first[mid] <= block) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int KIND>
struct Acc {
  double v = 0.0;
  __device__ __forceinline__ void take(float x) {
    if constexpr (KIND == kNormTwo) v = fma((double)x, (double)x, v);
    else v += (double)fabsf(x);
  }
  __device__ __forceinline__ void join(double o) { v += o; }
};
template <>
struct Acc<kNormMax> {
  double v = 0.0;        // (after the block's reduction)
  uint32_t bits = 0u;    // of |x|: ordered like the values, NaN above infinity
  __device__ __forceinline__ void take(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    bits = b > bits ? b : bits;
  }
  __device__ __forceinline__ void join(double o) {
    const uint32_t b = __float_as_uint((float)o) & 0x7FFFFFFFu;
    bits = b > bits ? b : bits;
  }
};

__device__ __forceinline__ double shfl_down_f64(double v, int d) {
  const int lo = __shfl_down(__double2loint(v), d, NR_WAVE), hi = __shfl_down(__double2hiint(v), d, NR_WAVE);
  return __hiloint2double(hi, lo);
}

// over the block, in thread 0
template <int KIND, int THREADS>
__device__ __forceinline__ double block_reduce(Acc<KIND> acc) {
  __shared__ double part[THREADS / NR_WAVE];
  if constexpr (KIND == kNormMax) acc.v = (double)__uint_as_float(acc.bits);
#pragma unroll
  for (int d = NR_WAVE / 2; d > 0; d >>= 1) {
    const double o = shfl_down_f64(acc.v, d);
    acc.join(o);
    if constexpr (KIND == kNormMax) acc.v = (double)__uint_as_float(acc.bits);
  }
  if (nr_lane() == 0) part[threadIdx.x / NR_WAVE] = acc.v;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / NR_WAVE; ++w) acc.join(part[w]);
    if constexpr (KIND == kNormMax) acc.v = (double)__uint_as_float(acc.bits);
  }
  return acc.v;
}

// Elements [lo, hi) of x: a lane takes 16 bytes, a wave a kilobyte, a block four such stretches in flight.
template <int KIND, typename T>
__device__ __forceinline__ void piece_norm(Acc<KIND>& acc, const T* __restrict__ x, int64_t lo, int64_t hi) {
  constexpr int N = 16 / (int)sizeof(T), kStep = kThreads * N;
  int64_t i = lo + threadIdx.x * N;
  for (; i + (kUnroll - 1) * kStep + N <= hi; i += kUnroll * kStep) {
    float v[kUnroll][N];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) nr_load_pack<T, N>(x + i + u * kStep, v[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) acc.take(v[u][k]);
  }
  for (; i < hi; i += kStep) {
    float v[N];
    nr_load_some<T, N>(x + i, hi - i < N ? (int)(hi - i) : N, v);
#pragma unroll
    for (int k = 0; k < N; ++k) acc.take(v[k]);
  }
}

template <int KIND>
__global__ void __launch_bounds__(kThreads)
norm_kernel(List l, double* __restrict__ partial) {
  const int t = tensor_of(l, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - l.first[t]) * l.piece;
  const int64_t hi = lo + l.piece < l.numel[t] ? lo + l.piece : l.numel[t];
  Acc<KIND> acc;
  if (l.in_dtype[t] == NR_DTYPE_F32) piece_norm<KIND, float>(acc, static_cast<const float*>(l.in[t]), lo, hi);
  else if (l.in_dtype[t] == NR_DTYPE_BF16) piece_norm<KIND, __bf16>(acc, static_cast<const __bf16*>(l.in[t]), lo, hi);
  else piece_norm<KIND, _Float16>(acc, static_cast<const _Float16*>(l.in[t]), lo, hi);
  const double v = block_reduce<KIND, kThreads>(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// The partial results' norm, and the factor that clips to max_norm, in thread 0 of the block.
template <int KIND, int THREADS>
__device__ __forceinline__ void finish(const double* __restrict__ partial, int64_t count, double max_norm, float& norm, float& factor) {
  Acc<KIND> acc;
  for (int64_t i = threadIdx.x; i < count; i += 4 * THREADS) {
    double v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = i + u * THREADS < count ? partial[i + u * THREADS] : 0.0;
#pragma unroll
    for (int u = 0; u < 4; ++u) acc.join(v[u]);
  }
  double v = block_reduce<KIND, THREADS>(acc);
  if constexpr (KIND == kNormTwo) v = sqrt(v);
  const double f = max_norm / (v + 1e-6);
  norm = (float)v;
  factor = f > 1.0 ? 1.0f : (float)f;  // (NaN stays NaN)
}

// result[0] = norm, result[1] = factor
template <int KIND, int THREADS>
__global__ void __launch_bounds__(THREADS)
norm_finish_kernel(const double* __restrict__ partial, int64_t count, double max_norm, float* __restrict__ result) {
  float norm, factor;
  finish<KIND, THREADS>(partial, count, max_norm, norm, factor);
  if (threadIdx.x == 0) {
    result[0] = norm;
    result[1] = factor;
  }
}

template <typename T, typename O, bool STREAM>
__device__ __forceinline__ void piece_scale(const T* __restrict__ x, O* __restrict__ y, int64_t lo, int64_t hi, float f) {
  constexpr int N = 16 / (int)sizeof(T), kStep = kThreads * N;
  int64_t i = lo + threadIdx.x * N;
  for (; i + (kUnroll - 1) * kStep + N <= hi; i += kUnroll * kStep) {
    float v[kUnroll][N];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) nr_load_pack<T, N>(x + i + u * kStep, v[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[u][k] *= f;
      if constexpr (STREAM) nr_store_pack_stream<O, N>(y + i + u * kStep, v[u]);
      else nr_store_pack<O, N>(y + i + u * kStep, v[u]);
    }
  }
  for (; i < hi; i += kStep) {
    const int m = hi - i < N ? (int)(hi - i) : N;
    float v[N];
    nr_load_some<T, N>(x + i, m, v);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] *= f;
    nr_store_some<O, N>(y + i, m, v);
  }
}
template <typename T, bool STREAM>
__device__ __forceinline__ void piece_scale_to(const T* x, void* y, int out_dtype, int64_t lo, int64_t hi, float f) {
  if (out_dtype == NR_DTYPE_F32) piece_scale<T, float, STREAM>(x, static_cast<float*>(y), lo, hi, f);
  else if (out_dtype == NR_DTYPE_BF16) piece_scale<T, __bf16, STREAM>(x, static_cast<__bf16*>(y), lo, hi, f);
  else piece_scale<T, _Float16, STREAM>(x, static_cast<_Float16*>(y), lo, hi, f);
}

template <bool STREAM>
__device__ __forceinline__ void scale_block(const List& l, uint32_t block, float f) {
  const int t = tensor_of(l, block);
  if (f == 1.0f && l.in[t] == l.out[t]) return;  // in place and within the norm: nothing to do
  const int64_t lo = (int64_t)(block - l.first[t]) * l.piece;
  const int64_t hi = lo + l.piece < l.numel[t] ? lo + l.piece : l.numel[t];
  if (l.in_dtype[t] == NR_DTYPE_F32) piece_scale_to<float, STREAM>(static_cast<const float*>(l.in[t]), l.out[t], l.out_dtype[t], lo, hi, f);
  else if (l.in_dtype[t] == NR_DTYPE_BF16) piece_scale_to<__bf16, STREAM>(static_cast<const __bf16*>(l.in[t]), l.out[t], l.out_dtype[t], lo, hi, f);
  else piece_scale_to<_Float16, STREAM>(static_cast<const _Float16*>(l.in[t]), l.out[t], l.out_dtype[t], lo, hi, f);
}

template <bool STREAM>
__global__ void __launch_bounds__(kThreads)
scale_kernel(List l, const float* __restrict__ result) {
  // backwards: what the norm read last is what the cache still holds
  scale_block<STREAM>(l, gridDim.x - 1 - blockIdx.x, result[1]);
}

// The same straight from the partial results, where they are few: every block adds them up for itself, in the finishing launch's
// order, and that launch (3 us with the wait for it) is saved.
template <int KIND>
__global__ void __launch_bounds__(kThreads)
finish_scale_kernel(List l, const double* __restrict__ partial, int64_t count, double max_norm, float* __restrict__ result) {
  __shared__ float s_factor;
  float norm, factor;
  finish<KIND, kThreads>(partial, count, max_norm, norm, factor);
  if (threadIdx.x == 0) {
    s_factor = factor;
    if (blockIdx.x == 0) {  // (of every launch of a long list: the same values)
      result[0] = norm;
      result[1] = factor;
    }
  }
  __syncthreads();
  scale_block<false>(l, gridDim.x - 1 - blockIdx.x, s_factor);
}

// ---------------------------------------------------------------------------------------------------------------- host
bool dtype_ok(int dtype) { return dtype == NR_DTYPE_F32 || dtype == NR_DTYPE_BF16 || dtype == NR_DTYPE_F16; }

struct Cut {
  int64_t piece, blocks;
};
// Pieces of a size that follows from the list's total: large lists in about kMaxBlocks of them, small ones in whole steps.
bool cut_list(const int64_t* numel, int count, Cut* c) {
  int64_t total = 0;
  if (count < 0 || (count > 0 && numel == nullptr)) return false;
  for (int t = 0; t < count; ++t) {
    if (numel[t] < 0 || numel[t] > ((int64_t)1 << 40)) return false;
    total += numel[t];
  }
  c->piece = nr_cdiv(total > 0 ? total : 1, kMaxBlocks * kPiece) * kPiece;
  c->blocks = 0;
  for (int t = 0; t < count; ++t) c->blocks += nr_cdiv(numel[t], c->piece);
  return c->blocks <= 0x7FFFFFFF;
}

// Calls launch(list, blocks, blocks before) for runs of up to kList non-empty tensors.
template <typename Launch>
int for_each_run(const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype, const int32_t* out_dtype, int count,
                 const Cut& c, Launch launch) {
  List l;
  l.piece = c.piece;
  int64_t before = 0;
  int t = 0;
  while (t < count) {
    l.count = 0;
    uint32_t blocks = 0;
    for (; t < count && l.count < kList; ++t) {
      if (numel[t] == 0) continue;
      const int k = l.count++;
      l.in[k] = in[t];
      l.out[k] = out != nullptr ? out[t] : nullptr;
      l.numel[k] = numel[t];
      l.in_dtype[k] = (uint8_t)in_dtype[t];
      l.out_dtype[k] = (uint8_t)(out_dtype != nullptr ? out_dtype[t] : in_dtype[t]);
      l.first[k] = blocks;
      blocks += (uint32_t)nr_cdiv(numel[t], c.piece);
    }
    if (l.count == 0) break;
    l.first[l.count] = blocks;
    if (int rc = launch(l, blocks, before)) return rc;
    before += blocks;
  }
  return 0;
}

bool list_ok(const void* const* in, const int64_t* numel, const int32_t* dtype, int count) {
  if (count > 0 && (in == nullptr || dtype == nullptr)) return false;
  for (int t = 0; t < count; ++t) {
    if (!dtype_ok(dtype[t]) || (numel[t] > 0 && in[t] == nullptr)) return false;
    const uintptr_t mask = dtype[t] == NR_DTYPE_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(in[t]) & mask) != 0) return false;
  }
  return true;
}

// A tensor in place is scaled in its own type: as another one, blocks would write what others have not read yet.
bool places_ok(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, const int32_t* out_dtypes, int count) {
  if (!list_ok(grads, numel, dtypes, count) || !list_ok(outs, numel, out_dtypes, count)) return false;
  for (int t = 0; t < count; ++t)
    if (numel[t] > 0 && grads[t] == outs[t] && dtypes[t] != out_dtypes[t]) return false;
  return true;
}

template <int KIND>
int run_partials(const void* const* in, const int64_t* numel, const int32_t* dtype, int count, const Cut& c, double* partial, hipStream_t stream) {
  return for_each_run(in, nullptr, numel, dtype, nullptr, count, c, [&](const List& l, uint32_t blocks, int64_t before) {
    hipLaunchKernelGGL(norm_kernel<KIND>, dim3(blocks), dim3(kThreads), 0, stream, l, partial + before);
    NR_LAUNCH_CHECK();
    return 0;
  });
}

template <int KIND>
int run_norm(const void* const* in, const int64_t* numel, const int32_t* dtype, int count, const Cut& c, double max_norm, float* result,
             double* partial, hipStream_t stream) {
  if (int rc = run_partials<KIND>(in, numel, dtype, count, c, partial, stream)) return rc;
  if (c.blocks <= kFew)
    hipLaunchKernelGGL((norm_finish_kernel<KIND, kThreads>), dim3(1), dim3(kThreads), 0, stream, partial, c.blocks, max_norm, result);
  else
    hipLaunchKernelGGL((norm_finish_kernel<KIND, kFinishThreads>), dim3(1), dim3(kFinishThreads), 0, stream, partial, c.blocks, max_norm, result);
  NR_LAUNCH_CHECK();
  return 0;
}

int run_scale(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, const int32_t* out_dtypes, int count,
              const Cut& c, const float* result, hipStream_t stream) {
  int64_t bytes = 0;
  for (int t = 0; t < count; ++t) bytes += numel[t] * (out_dtypes[t] == NR_DTYPE_F32 ? 4 : 2);
  const bool past = bytes > kStreamBytes;
  return for_each_run(grads, outs, numel, dtypes, out_dtypes, count, c, [&](const List& l, uint32_t blocks, int64_t) {
    if (past) hipLaunchKernelGGL(scale_kernel<true>, dim3(blocks), dim3(kThreads), 0, stream, l, result);
    else hipLaunchKernelGGL(scale_kernel<false>, dim3(blocks), dim3(kThreads), 0, stream, l, result);
    NR_LAUNCH_CHECK();
    return 0;
  });
}

template <int KIND>
int run_clip(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, const int32_t* out_dtypes, int count,
             const Cut& c, double max_norm, float* result, double* partial, hipStream_t stream) {
  if (c.blocks == 0 || c.blocks > kFew) {
    if (int rc = run_norm<KIND>(grads, numel, dtypes, count, c, max_norm, result, partial, stream)) return rc;
    return run_scale(grads, outs, numel, dtypes, out_dtypes, count, c, result, stream);
  }
  if (int rc = run_partials<KIND>(grads, numel, dtypes, count, c, partial, stream)) return rc;
  return for_each_run(grads, outs, numel, dtypes, out_dtypes, count, c, [&](const List& l, uint32_t blocks, int64_t) {
    hipLaunchKernelGGL(finish_scale_kernel<KIND>, dim3(blocks), dim3(kThreads), 0, stream, l, partial, c.blocks, max_norm, result);
    NR_LAUNCH_CHECK();
    return 0;
  });
}

bool norm_args_ok(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count, int norm_type, double max_norm,
                  const float* result, const void* workspace, Cut* c) {
  return cut_list(numel, count, c) && list_ok(grads, numel, dtypes, count) && norm_type >= 0 && norm_type <= 2 && max_norm >= 0.0 &&
         result != nullptr && !(c->blocks > 0 && workspace == nullptr) && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0;
}

}  // namespace

extern "C" int64_t nr_grad_norm_workspace_bytes(const int64_t* numel, int count) {
  Cut c;
  if (!cut_list(numel, count, &c)) return NR_EINVAL;
  return c.blocks * (int64_t)sizeof(double);
}

extern "C" int nr_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count, int norm_type, double max_norm,
                            float* result, void* workspace, nr_stream_t stream) {
  Cut c;
  if (!norm_args_ok(grads, numel, dtypes, count, norm_type, max_norm, result, workspace, &c)) return NR_EINVAL;
  auto run = norm_type == kNormMax ? run_norm<kNormMax> : norm_type == kNormSum ? run_norm<kNormSum> : run_norm<kNormTwo>;
  return run(grads, numel, dtypes, count, c, max_norm, result, static_cast<double*>(workspace), nr_s(stream));
}

extern "C" int nr_grad_scale(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, const int32_t* out_dtypes,
                             int count, const float* result, nr_stream_t stream) {
  Cut c;
  if (!cut_list(numel, count, &c) || !places_ok(grads, outs, numel, dtypes, out_dtypes, count) || result == nullptr) return NR_EINVAL;
  return run_scale(grads, outs, numel, dtypes, out_dtypes, count, c, result, nr_s(stream));
}

extern "C" int nr_grad_clip(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, const int32_t* out_dtypes,
                            int count, int norm_type, double max_norm, float* result, void* workspace, nr_stream_t stream) {
  Cut c;
  if (!norm_args_ok(grads, numel, dtypes, count, norm_type, max_norm, result, workspace, &c) ||
      !places_ok(grads, outs, numel, dtypes, out_dtypes, count))
    return NR_EINVAL;
  auto run = norm_type == kNormMax ? run_clip<kNormMax> : norm_type == kNormSum ? run_clip<kNormSum> : run_clip<kNormTwo>;
  return run(grads, outs, numel, dtypes, out_dtypes, count, c, max_norm, result, static_cast<double*>(workspace), nr_s(stream));
}

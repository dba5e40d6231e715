// Kernels of the gradient norm and clipping (grad_norm.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "grad_norm.h"

namespace ft {
namespace gn {
namespace {

constexpr int NT = 256;

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

// Sum over the block, the same in every thread; `red` has room for 32.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

// Squares of K values: in fp32, or in fp64 where that is infinite or has lost small values.
template <int K>
__device__ __forceinline__ double squares(const float (&v)[K]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < K; ++i) s = fmaf(v[i], v[i], s);
  double r = s;
  if (s < 0x1p-90f || s > 0x1p126f) {
    r = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) r = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), r);
  }
  return r;
}

// Values before the first 16-byte boundary
template <typename T>
__device__ __forceinline__ int ahead(const T* p) {
  return static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
}

template <typename T>
__device__ __forceinline__ double sum_chunk(const T* x, int n) {
  constexpr int V = 16 / sizeof(T);
  double acc = 0;
  const int h = min(n, ahead(x));
  if (static_cast<int>(threadIdx.x) < h) {
    const float one[1] = {to_f(x[threadIdx.x])};
    acc += squares(one);
  }
  const int nv = (n - h) / V;
  const uint4* xv = reinterpret_cast<const uint4*>(x + h);
  constexpr int U = 4;
  for (int i = threadIdx.x; i < nv; i += NT * U) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = i + u * NT < nv ? __ldg(xv + i + u * NT) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * NT >= nv) break;
      const T* e = reinterpret_cast<const T*>(&q[u]);
      float v[V];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = to_f(e[k]);
      acc += squares(v);
    }
  }
  for (int i = h + nv * V + threadIdx.x; i < n; i += NT) {
    const float one[1] = {to_f(x[i])};
    acc += squares(one);
  }
  return acc;
}

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t.chunk_end[mid] > chunk) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// This block's run of chunks: [first, last)
__device__ __forceinline__ void run_of(int chunks, int& first, int& last) {
  first = static_cast<int>(static_cast<int64_t>(chunks) * blockIdx.x / gridDim.x);
  last = static_cast<int>(static_cast<int64_t>(chunks) * (blockIdx.x + 1) / gridDim.x);
}

template <int N>
__global__ void __launch_bounds__(NT) sumsq_kernel(const __grid_constant__ Table<N> t, int n_slots,
                                                   double* __restrict__ partial) {
  __shared__ double red[32];
  int c, last;
  run_of(t.chunks, c, last);
  double sums[MAX_SLOTS];
#pragma unroll
  for (int s = 0; s < MAX_SLOTS; ++s) sums[s] = 0;
  int i = tensor_of(t, c);
  while (c < last) {
    while (t.chunk_end[i] <= c) ++i;
    const int begin = i ? t.chunk_end[i - 1] : 0, stop = min(last, t.chunk_end[i]);
    double acc = 0;
    for (; c < stop; ++c) {
      const int64_t at = static_cast<int64_t>(c - begin) * CHUNK;
      const int n = static_cast<int>(min(static_cast<int64_t>(CHUNK), t.n[i] - at));
      if (t.type[i] == F32) acc += sum_chunk(static_cast<const float*>(t.x[i]) + at, n);
      else if (t.type[i] == BF16) acc += sum_chunk(static_cast<const __nv_bfloat16*>(t.x[i]) + at, n);
      else acc += sum_chunk(static_cast<const __half*>(t.x[i]) + at, n);
    }
#pragma unroll
    for (int s = 0; s < MAX_SLOTS; ++s)
      if (t.slot[i] == s) sums[s] += acc;
  }
#pragma unroll
  for (int s = 0; s < MAX_SLOTS; ++s) {
    if (s >= n_slots) break;
    const double v = block_sum(sums[s], red);
    if (threadIdx.x == 0) partial[static_cast<int64_t>(blockIdx.x) * n_slots + s] = v;
  }
}

__global__ void __launch_bounds__(NT) finish_kernel(const double* __restrict__ partial, int blocks, int n_slots,
                                                    double* __restrict__ sums) {
  __shared__ double red[32];
  for (int s = 0; s < n_slots; ++s) {
    double v = 0;
    for (int b = threadIdx.x; b < blocks; b += NT) v += partial[static_cast<int64_t>(b) * n_slots + s];
    v = block_sum(v, red);
    if (threadIdx.x == 0) sums[s] = v;
  }
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* x, T* y, int n, float f) {
  constexpr int V = 16 / sizeof(T);
  int h = n, nv = 0;
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0) {
    h = min(n, ahead(x));
    nv = (n - h) / V;
  }
  for (int i = threadIdx.x; i < h; i += NT) y[i] = from_f<T>(to_f(x[i]) * f);
  const uint4* xv = reinterpret_cast<const uint4*>(x + h);
  uint4* yv = reinterpret_cast<uint4*>(y + h);
  constexpr int U = 4;
  for (int i = threadIdx.x; i < nv; i += NT * U) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * NT < nv) q[u] = xv[i + u * NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * NT >= nv) break;
      T* e = reinterpret_cast<T*>(&q[u]);
#pragma unroll
      for (int k = 0; k < V; ++k) e[k] = from_f<T>(to_f(e[k]) * f);
      yv[i + u * NT] = q[u];
    }
  }
  for (int i = h + nv * V + threadIdx.x; i < n; i += NT) y[i] = from_f<T>(to_f(x[i]) * f);
}

template <int N>
__global__ void __launch_bounds__(NT) scale_kernel(const __grid_constant__ Table<N> t, const __grid_constant__ Factor f) {
  __shared__ double red[32];
  float c;
  if (f.coef) {
    c = *f.coef;
  } else {
    double v = 0;
    for (int b = threadIdx.x; b < f.blocks; b += NT) v += f.partial[b];
    const float norm = static_cast<float>(sqrt(block_sum(v, red)));
    c = f.max_norm / (norm + 1e-6f);
    if (c > 1.f) c = 1.f;  // a norm that is not a number stays one
    if (blockIdx.x == 0 && threadIdx.x == 0) *f.norm = norm;
  }
  if (f.in_place && c == 1.f) return;
  int k, last;
  run_of(t.chunks, k, last);
  int i = tensor_of(t, k);
  for (; k < last; ++k) {
    while (t.chunk_end[i] <= k) ++i;
    const int64_t at = static_cast<int64_t>(k - (i ? t.chunk_end[i - 1] : 0)) * CHUNK;
    const int n = static_cast<int>(min(static_cast<int64_t>(CHUNK), t.n[i] - at));
    if (t.type[i] == F32) scale_chunk(static_cast<const float*>(t.x[i]) + at, static_cast<float*>(t.y[i]) + at, n, c);
    else if (t.type[i] == BF16)
      scale_chunk(static_cast<const __nv_bfloat16*>(t.x[i]) + at, static_cast<__nv_bfloat16*>(t.y[i]) + at, n, c);
    else scale_chunk(static_cast<const __half*>(t.x[i]) + at, static_cast<__half*>(t.y[i]) + at, n, c);
  }
}

}  // namespace

// Eight blocks of 256 threads on each of 148 SMs; fewer chunks than that take a block each.
int sumsq_blocks(int chunks) { return std::min(chunks, 148 * 8); }

template <int N>
cudaError_t launch_sumsq(const Table<N>& t, int n_slots, double* partial, cudaStream_t st) {
  sumsq_kernel<N><<<sumsq_blocks(t.chunks), NT, 0, st>>>(t, n_slots, partial);
  return cudaGetLastError();
}

cudaError_t launch_finish(const double* partial, int blocks, int n_slots, double* sums, cudaStream_t st) {
  finish_kernel<<<1, NT, 0, st>>>(partial, blocks, n_slots, sums);
  return cudaGetLastError();
}

template <int N>
cudaError_t launch_scale(const Table<N>& t, const Factor& f, cudaStream_t st) {
  scale_kernel<N><<<sumsq_blocks(t.chunks), NT, 0, st>>>(t, f);
  return cudaGetLastError();
}

template cudaError_t launch_sumsq<64>(const Table<64>&, int, double*, cudaStream_t);
template cudaError_t launch_sumsq<MAX_TENSORS>(const Table<MAX_TENSORS>&, int, double*, cudaStream_t);
template cudaError_t launch_scale<64>(const Table<64>&, const Factor&, cudaStream_t);
template cudaError_t launch_scale<MAX_TENSORS>(const Table<MAX_TENSORS>&, const Factor&, cudaStream_t);

}  // namespace gn
}  // namespace ft

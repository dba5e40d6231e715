// Kernels of the embedding lookup and its sorted gradient (embedding.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "embedding.h"

namespace ft {
namespace emb {
namespace {

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

__device__ __forceinline__ int64_t id_at(const void* ids, bool wide, int64_t t) {
  return wide ? static_cast<const int64_t*>(ids)[t] : static_cast<const int*>(ids)[t];
}

// ------------------------------------------------------------------------------ lookup
// One block per (token, piece of the row) with 16 bytes per thread; one per token, eight loads in flight, where rows are not
// on 16-byte boundaries.
template <typename T, int VEC>
__global__ void __launch_bounds__(128) fwd_kernel(const FwdArgs a) {
  const int64_t t = blockIdx.x;
  const int c = VEC == 1 ? threadIdx.x : (blockIdx.y * 128 + threadIdx.x) * VEC;
  if (c >= a.H) return;
  const int64_t id = id_at(a.ids, a.ids64, t) - a.vstart;
  const bool has = id >= 0 && id < a.V;
  const T* w = static_cast<const T*>(a.table) + id * a.H + c;
  T* o = static_cast<T*>(a.out) + t * a.H + c;
  if constexpr (VEC == 1) {
    const int n = (a.H - c + 127) / 128;
    for (int i0 = 0; i0 < n; i0 += 8) {
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = has && i0 + i < n ? w[(i0 + i) * 128] : from_f<T>(0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < n) o[(i0 + i) * 128] = from_f<T>(to_f(v[i]) * a.scale);
    }
  } else {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (has) {
      q = __ldg(reinterpret_cast<const uint4*>(w));
      T* e = reinterpret_cast<T*>(&q);
#pragma unroll
      for (int k = 0; k < VEC; ++k) e[k] = from_f<T>(to_f(e[k]) * a.scale);
    }
    *reinterpret_cast<uint4*>(o) = q;
  }
}

template <typename T>
void fwd_of(const FwdArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const dim3 grid(static_cast<unsigned>(a.T), a.vec ? (a.H + 128 * V - 1) / (128 * V) : 1);
  if (a.vec) fwd_kernel<T, V><<<grid, 128, 0, st>>>(a);
  else fwd_kernel<T, 1><<<grid, 128, 0, st>>>(a);
}

// ------------------------------------------------------------------------------ sort
// Least significant digit first; each pass counts the digits of every block's tokens, scans the counts digit
// by digit over the blocks, and moves each token behind the equal digits before it.
constexpr int SORT_NT = 256, SORT_WARPS = SORT_NT / 32, PER_WARP = SORT_CHUNK / SORT_WARPS;

struct Pass {
  int shift, bits;
  bool first;  // keys still come from the ids
  const uint32_t *key, *pos;
  uint32_t *key_out, *pos_out;
};

__device__ __forceinline__ uint32_t key_at(const SortArgs& a, const Pass& p, int t) {
  if (!p.first) return p.key[t];
  const int64_t id = id_at(a.ids, a.ids64, t) - a.vstart;
  return static_cast<uint32_t>(id >= 0 && id < a.V ? id : a.V);
}

__global__ void __launch_bounds__(SORT_NT) count_kernel(const SortArgs a, const Pass p) {
  __shared__ uint32_t bins[MAX_BINS];
  const int n = 1 << p.bits;
  for (int i = threadIdx.x; i < n; i += SORT_NT) bins[i] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * SORT_CHUNK, t1 = min(a.T, t0 + SORT_CHUNK);
  for (int t = t0 + threadIdx.x; t < t1; t += SORT_NT) atomicAdd(&bins[(key_at(a, p, t) >> p.shift) & (n - 1)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += SORT_NT) a.counts[static_cast<int64_t>(i) * a.blocks + blockIdx.x] = bins[i];
}

// Exclusive scan of n counts in place; one block.
__global__ void __launch_bounds__(1024) scan_kernel(uint32_t* __restrict__ x, int n) {
  __shared__ uint32_t warps[32];
  uint32_t carry = 0;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i0 = 0; i0 < n; i0 += 4096) {
    const int i = i0 + threadIdx.x * 4;
    uint32_t v[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = i + e < n ? x[i + e] : 0;
      sum += v[e];
    }
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffff, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) warps[w] = inc;
    __syncthreads();
    uint32_t before = carry, all = 0;
    for (int k = 0; k < 32; ++k) {
      if (k < w) before += warps[k];
      all += warps[k];
    }
    uint32_t at = before + inc - sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e < n) x[i + e] = at;
      at += v[e];
    }
    carry += all;
  }
}

__global__ void __launch_bounds__(SORT_NT) move_kernel(const SortArgs a, const Pass p) {
  extern __shared__ uint32_t at[];  // [warps][bins]: where a warp's next token of a digit goes
  const int n = 1 << p.bits, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < n * SORT_WARPS; i += SORT_NT) at[i] = 0;
  __syncthreads();
  uint32_t* mine = at + w * n;
  const int t0 = blockIdx.x * SORT_CHUNK + w * PER_WARP;
  for (int r = 0; r < PER_WARP; r += 32) {
    const int t = t0 + r + lane;
    if (t < a.T) atomicAdd(&mine[(key_at(a, p, t) >> p.shift) & (n - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += SORT_NT) {
    uint32_t base = a.counts[static_cast<int64_t>(i) * a.blocks + blockIdx.x];
    for (int k = 0; k < SORT_WARPS; ++k) {
      const uint32_t c = at[k * n + i];
      at[k * n + i] = base;
      base += c;
    }
  }
  __syncthreads();
  for (int r = 0; r < PER_WARP; r += 32) {
    const int t = t0 + r + lane;
    const bool in = t < a.T;
    const uint32_t key = in ? key_at(a, p, t) : 0;
    const uint32_t digit = in ? (key >> p.shift) & (n - 1) : n;  // n: no token
    const uint32_t same = __match_any_sync(0xffffffff, digit);
    const uint32_t rank = __popc(same & ((1u << lane) - 1));
    uint32_t to = 0;
    if (in) to = mine[digit] + rank;
    __syncwarp();
    if (in && rank == 0) mine[digit] += __popc(same);
    __syncwarp();
    if (in) {
      p.key_out[to] = key;
      p.pos_out[to] = p.first ? t : p.pos[t];
    }
  }
}

// The same passes for up to SMALL_SORT tokens, in the shared memory of one block; a warp's tokens are neighbours, so equal
// digits keep their order.
constexpr int SMALL_NT = 1024, SMALL_WARPS = SMALL_NT / 32, SMALL_BINS = 1 << SMALL_BITS, ROUNDS = SMALL_SORT / SMALL_NT;
struct SmallSort {
  uint32_t key[2][SMALL_SORT];
  uint16_t pos[2][SMALL_SORT];
  uint16_t at[SMALL_WARPS][SMALL_BINS];  // counts, then where a warp's next token of a digit goes
  uint32_t warps[SMALL_WARPS];
};

__global__ void __launch_bounds__(SMALL_NT) small_sort_kernel(const SortArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");  // clearing may run beside this block
  extern __shared__ uint8_t raw[];
  SmallSort& s = *reinterpret_cast<SmallSort*>(raw);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int t = threadIdx.x; t < a.T; t += SMALL_NT) {
    const int64_t id = id_at(a.ids, a.ids64, t) - a.vstart;
    s.key[0][t] = static_cast<uint32_t>(id >= 0 && id < a.V ? id : a.V);
    s.pos[0][t] = static_cast<uint16_t>(t);
  }
  const int rounds = (a.T + SMALL_NT - 1) / SMALL_NT, t0 = w * rounds * 32;
  int shift = 0;
  for (int pass = 0; pass < a.passes; ++pass) {
    const int bins = 1 << a.bits[pass], from = pass & 1;
    for (int i = threadIdx.x; i < SMALL_WARPS * bins / 2; i += SMALL_NT)
      reinterpret_cast<uint32_t*>(s.at)[i / (bins / 2) * (SMALL_BINS / 2) + i % (bins / 2)] = 0;
    __syncthreads();
    // a token's place among its warp's equal digits, kept for the move (matching is what takes the time)
    uint16_t place[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if (r >= rounds) break;
      const int t = t0 + r * 32 + lane;
      const bool in = t < a.T;
      const uint32_t digit = in ? (s.key[from][t] >> shift) & (bins - 1) : bins;
      const uint32_t same = __match_any_sync(0xffffffff, digit), rank = __popc(same & ((1u << lane) - 1));
      const uint32_t before = in ? s.at[w][digit] : 0;
      place[r] = static_cast<uint16_t>(before + rank);
      __syncwarp();
      if (in && rank == 0) s.at[w][digit] = static_cast<uint16_t>(before + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    // exclusive scan, digit by digit over the warps
    uint32_t sum = 0;
    if (static_cast<int>(threadIdx.x) < bins)
      for (int k = 0; k < SMALL_WARPS; ++k) sum += s.at[k][threadIdx.x];
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffff, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) s.warps[w] = inc;
    __syncthreads();
    uint32_t base = inc - sum;
    for (int k = 0; k < w; ++k) base += s.warps[k];
    if (static_cast<int>(threadIdx.x) < bins)
      for (int k = 0; k < SMALL_WARPS; ++k) {
        const uint32_t c = s.at[k][threadIdx.x];
        s.at[k][threadIdx.x] = static_cast<uint16_t>(base);
        base += c;
      }
    __syncthreads();
    const bool last = pass + 1 == a.passes;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if (r >= rounds) break;
      const int t = t0 + r * 32 + lane;
      const bool in = t < a.T;
      const uint32_t key = in ? s.key[from][t] : 0;
      const uint32_t to = in ? s.at[w][(key >> shift) & (bins - 1)] + place[r] : 0;
      if (in) {
        if (last) {
          a.key[0][to] = key;
          a.pos[0][to] = s.pos[from][t];
        } else {
          s.key[from ^ 1][to] = key;
          s.pos[from ^ 1][to] = s.pos[from][t];
        }
      }
    }
    __syncthreads();
    shift += a.bits[pass];
  }
}

// ------------------------------------------------------------------------------ sums
template <typename D, int VEC>
__device__ __forceinline__ void put(D* d, const float (&v)[VEC], float scale, bool add) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const float x = v[k] * scale;
    d[k] = from_f<D>(add ? to_f(d[k]) + x : x);
  }
}

template <typename D, int VEC>
__device__ __forceinline__ void put_row(void* dw, int64_t at, const float (&v)[VEC], float scale, bool add) {
  D* d = static_cast<D*>(dw) + at;
  if constexpr (VEC == 1) {
    put<D, 1>(d, v, scale, add);
  } else {
    constexpr int Q = VEC * sizeof(D) / 16 > 0 ? VEC * sizeof(D) / 16 : 1;
    __align__(16) D buf[VEC];
    uint4* b4 = reinterpret_cast<uint4*>(buf);
    uint4* d4 = reinterpret_cast<uint4*>(d);
    if constexpr (VEC * sizeof(D) % 16 == 0) {
      if (add)
#pragma unroll
        for (int q = 0; q < Q; ++q) b4[q] = d4[q];
      put<D, VEC>(buf, v, scale, add);
#pragma unroll
      for (int q = 0; q < Q; ++q) d4[q] = b4[q];
    } else {  // 4 values of 2 bytes
      uint2* b2 = reinterpret_cast<uint2*>(buf);
      if (add) *b2 = *reinterpret_cast<uint2*>(d);
      put<D, VEC>(buf, v, scale, add);
      *reinterpret_cast<uint2*>(d) = *b2;
    }
  }
}

// A block sums 32 sorted tokens over 128 VEC columns, eight rows in flight at a time.
template <typename T, typename D, int VEC>
__global__ void __launch_bounds__(128) sum_kernel(const GradArgs a) {
  __shared__ uint32_t key[PIECE + 2], pos[PIECE];  // key[0]: of the token before the piece, key[n + 1]: behind it
  const int e0 = blockIdx.x * PIECE, n = min(PIECE, a.T - e0);
  if (static_cast<int>(threadIdx.x) < n + 2) {
    const int e = e0 + static_cast<int>(threadIdx.x) - 1;
    key[threadIdx.x] = e >= 0 && e < a.T ? a.key[e] : 0xffffffffu;
  }
  if (static_cast<int>(threadIdx.x) < n) pos[threadIdx.x] = a.pos[e0 + threadIdx.x];
  __syncthreads();
  const int c = (blockIdx.y * 128 + threadIdx.x) * VEC;
  if (c >= a.H) return;
  const T* dout = static_cast<const T*>(a.dout) + c;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  bool begun = key[0] != key[1];  // did the present run begin in this piece
  constexpr int U = VEC == 1 ? 8 : 4;
  for (int i0 = 0; i0 < n; i0 += U) {
    T in[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i < n && key[i + 1] < static_cast<uint32_t>(a.V)) {
        const T* src = dout + static_cast<int64_t>(pos[i]) * a.H;
        if constexpr (VEC == 1) in[u][0] = src[0];
        else *reinterpret_cast<uint4*>(in[u]) = __ldg(reinterpret_cast<const uint4*>(src));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= n || key[i + 1] >= static_cast<uint32_t>(a.V)) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += to_f(in[u][k]);
      if (key[i + 2] != key[i + 1] || i + 1 == n) {
        const bool ends = key[i + 2] != key[i + 1];
        if (begun && ends) {
          put_row<D, VEC>(a.dw, static_cast<int64_t>(key[i + 1]) * a.H + c, acc, a.scale, a.accumulate);
        } else {
          float* part = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (begun ? 1 : 0)) * a.H + c;
#pragma unroll
          for (int k = 0; k < VEC; ++k) part[k] = acc[k];
        }
        begun = true;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
      }
    }
  }
}

// A block whose piece begins a run that goes on into the next one adds that run's partial sums up.
template <typename D, int VEC>
__global__ void __launch_bounds__(128) join_kernel(const GradArgs a) {
  const int e1 = (blockIdx.x + 1) * PIECE;
  if (e1 >= a.T) return;
  const uint32_t key = a.key[e1 - 1];
  if (key >= static_cast<uint32_t>(a.V) || a.key[e1] != key) return;
  const int e0 = e1 - PIECE;
  if (a.key[e0] == key && e0 > 0 && a.key[e0 - 1] == key) return;  // the run began before this piece
  const int c = (blockIdx.y * 128 + threadIdx.x) * VEC;
  if (c >= a.H) return;
  float acc[VEC];
  const float* part = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + 1) * a.H + c;
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = part[k];
  for (int b = blockIdx.x + 1; b < a.pieces && a.key[b * PIECE] == key; ++b) {
    const float* more = a.partial + static_cast<int64_t>(b) * 2 * a.H + c;
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += more[k];
  }
  put_row<D, VEC>(a.dw, static_cast<int64_t>(key) * a.H + c, acc, a.scale, a.accumulate);
}

template <typename T, typename D, int VEC>
void grad_of(const GradArgs& a, cudaStream_t st) {
  const dim3 grid(a.pieces, (a.H + 128 * VEC - 1) / (128 * VEC));
  sum_kernel<T, D, VEC><<<grid, 128, 0, st>>>(a);
  if (a.pieces > 1) join_kernel<D, VEC><<<grid, 128, 0, st>>>(a);
}

template <typename T>
void grad_to(const GradArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  auto go = [&](auto d) {
    using D = decltype(d);
    if (a.vec) grad_of<T, D, V>(a, st);
    else grad_of<T, D, 1>(a, st);
  };
  if (a.dw_type == F32) go(float());
  else if (a.dw_type == BF16) go(__nv_bfloat16());
  else go(__half());
}

}  // namespace

cudaError_t launch_fwd(const FwdArgs& a, cudaStream_t st) {
  if (a.type == F32) fwd_of<float>(a, st);
  else if (a.type == BF16) fwd_of<__nv_bfloat16>(a, st);
  else fwd_of<__half>(a, st);
  return cudaGetLastError();
}

// 16 bytes per store, four per thread, in many small blocks: 2.1 GB in 280 us.  (A block of 1024 threads per SM, beside the
// block that sorts, took 350 us; the runtime's memset 337.)  Behind the sort in one block it may start beside it, as it reads
// nothing of it; what follows on the stream waits for this kernel, so one of its blocks waits for the sort.
__global__ void __launch_bounds__(256) clear_kernel(uint4* __restrict__ x, int64_t words) {
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (i0 + u * 256 < words) x[i0 + u * 256] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

cudaError_t launch_clear(void* x, int64_t bytes, bool beside_sort, cudaStream_t st) {
  const int64_t words = bytes / 16, blocks = (words + 1023) / 1024;
  if (reinterpret_cast<uintptr_t>(x) % 16 || bytes % 16 || blocks >= (int64_t(1) << 31)) return cudaMemsetAsync(x, 0, bytes, st);
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = beside_sort ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, clear_kernel, static_cast<uint4*>(x), words);
}

cudaError_t launch_small_sort(const SortArgs& a, cudaStream_t st) {
  static unsigned long long done = 0;
  smem_attr_once(small_sort_kernel, sizeof(SmallSort), done);
  small_sort_kernel<<<1, SMALL_NT, sizeof(SmallSort), st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_sort(const SortArgs& a, cudaStream_t st) {
  int shift = 0;
  for (int i = 0; i < a.passes; ++i) {
    const Pass p{shift, a.bits[i], i == 0, a.key[i & 1], a.pos[i & 1], a.key[(i + 1) & 1], a.pos[(i + 1) & 1]};
    const int bins = 1 << a.bits[i];
    count_kernel<<<a.blocks, SORT_NT, 0, st>>>(a, p);
    scan_kernel<<<1, 1024, 0, st>>>(a.counts, bins * a.blocks);
    move_kernel<<<a.blocks, SORT_NT, bins * SORT_WARPS * sizeof(uint32_t), st>>>(a, p);
    shift += a.bits[i];
  }
  return cudaGetLastError();
}

cudaError_t launch_grad(const GradArgs& a, cudaStream_t st) {
  if (a.dout_type == F32) grad_to<float>(a, st);
  else if (a.dout_type == BF16) grad_to<__nv_bfloat16>(a, st);
  else grad_to<__half>(a, st);
  return cudaGetLastError();
}

}  // namespace emb
}  // namespace ft

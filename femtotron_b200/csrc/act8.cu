// Activations kept in 8 bits between forward and backward (sm_100a).
//
// Format: a row of n values is cut into groups of G (32, 64, 128 or 256; the last one may be
// short).  With top = max |x| of the group,
//   q  = rint(x * (127 * (1 / top)))      int8, ties to even        (0 where top < 2^-120)
//   x8 = q * (top * (1 / 127))            what the 8 bits stand for, |x8 - x| <= top / 254
// The scale top / 127 is kept in fp32.  Each step is one IEEE fp32 operation, so the codes are
// the same on every device.  A group with a NaN or an infinity comes back as NaN throughout.
// Codes of a row start on a 16-byte boundary (pitch = n rounded up to 16).
//
// One thread owns 16 neighbouring values: one 32-byte bf16 load where rows allow it (else two of
// 16), one 16-byte code store.  The
// G / 16 threads of a group are neighbours in one warp and find the maximum with shuffles, so
// every value is read from memory once.  All kernels here are bound by HBM bandwidth once the
// instructions per value are few: conversions by added constants and byte permutes (see encode16,
// decode16), row and chunk of a thread by one multiplication.  Measured among others of its kind
// (bytes moved / time): quantise 8192 x 4096 bf16 20.4 us (4.9 TB/s), dequantise 18.5 us (5.5),
// RMSNorm 4096 x 8192 forward 33.5 us (5.0), backward 48.6 us (4.8), SwiGLU 4096 x 14336
// forward 84 us (5.6), backward 105 us (5.6).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "checks.h"
#include "common.cuh"

namespace ft {
namespace {

constexpr int kChunk = 16;                // values per thread
constexpr float kTiny = 7.52316385e-37f;  // 2^-120
constexpr float kInv127 = 1.0f / 127.0f;

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

// How rows lie in memory: 16-value chunks on 32-byte boundaries (one 256-bit access per 16
// bf16), on 16-byte ones, or neither.
enum Rows { kRows32, kRows16, kRowsAny };

// N 32-bit words of p, N = 4, 8 or 16.
template <int N, Rows R>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (R == kRows32 && N >= 8) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      asm("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
          : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]),
            "=r"(w[i + 6]), "=r"(w[i + 7])
          : "l"(__cvta_generic_to_global(static_cast<const uint32_t*>(p) + i))
          : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(p) + i);
      w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
    }
  }
}
template <int N, Rows R>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[N]) {
  if constexpr (R == kRows32 && N >= 8) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
      asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]),
                   "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7]),
                   "l"(__cvta_generic_to_global(static_cast<uint32_t*>(p) + i))
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<uint4*>(static_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}

// 16 values and their packed words (two 16-bit values per word, the lower one first).
__device__ __forceinline__ void unpack(const uint32_t (&w)[8], float (&v)[16], __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint32_t (&w)[8], float (&v)[16], __half) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const uint32_t (&w)[16], float (&v)[16], float) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void pack(const float (&v)[16], uint32_t (&w)[8], __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void pack(const float (&v)[16], uint32_t (&w)[8], __half) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void pack(const float (&v)[16], uint32_t (&w)[16], float) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
}

// Up to 16 values starting at p (`left` of them exist) as fp32, zeros after them.
template <typename T, Rows R>
__device__ __forceinline__ void load16(const T* p, int left, float (&v)[16]) {
  if (R != kRowsAny && left >= 16) {
    uint32_t w[4 * sizeof(T)];
    load_words<4 * sizeof(T), R>(p, w);
    unpack(w, v, T{});
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < left ? to_f(p[i]) : 0.f;
  }
}
template <typename T, Rows R>
__device__ __forceinline__ void store16(T* p, int left, const float (&v)[16]) {
  if (R != kRowsAny && left >= 16) {
    uint32_t w[4 * sizeof(T)];
    pack(v, w, T{});
    store_words<4 * sizeof(T), R>(p, w);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}

// Rows on no 16-byte boundary: the warp takes its lanes' chunks two at a time, 16 lanes on
// neighbouring values of one, and hands them over through shared memory (17 words per chunk: no bank
// conflicts).  Every lane of the warp takes part, with left <= 0 where it has no chunk.
template <typename T>
__device__ __forceinline__ void load16_any(const T* p, int left, float (&v)[16], float* box) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int from = 2 * i + lane / 16, k = lane % 16;
    const T* q = reinterpret_cast<const T*>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
    const int have = __shfl_sync(0xffffffffu, left, from);
    v[i] = k < have ? to_f(q[k]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) box[(2 * i + lane / 16) * 17 + lane % 16] = v[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = box[lane * 17 + i];
}
template <typename T>
__device__ __forceinline__ void store16_any(T* p, int left, const float (&v)[16], float* box) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int i = 0; i < 16; ++i) box[lane * 17 + i] = v[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int from = 2 * i + lane / 16, k = lane % 16;
    T* q = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
    const int have = __shfl_sync(0xffffffffu, left, from);
    if (k < have) q[k] = from_f<T>(box[from * 17 + k]);
  }
}
template <Rows R> constexpr int kBoxes = R == kRowsAny ? 8 * 32 * 17 : 1;

// Largest magnitude over the 2^lanes_log2 neighbouring threads that share a group.  NaN has to win,
// so magnitudes are compared as their bit patterns (for non-negative floats the integer order
// is the order of the values, with NaN above infinity).
__device__ __forceinline__ float group_top(const float (&v)[16], int lanes_log2) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {  // groups have 2 to 16 threads
    const uint32_t other = __shfl_xor_sync(0xffffffffu, m, o);
    if (o < (1 << lanes_log2)) m = max(m, other);
  }
  return __uint_as_float(m);
}

// Codes of 16 values; returns the group's scale.  top = inf or NaN gives the scale NaN.
// Adding 1.5 * 2^23 rounds the product to an integer (ties to even) whose two's complement is the
// low byte of the sum: no conversion instruction, which would run at a quarter of the rate.
// |x * mul| <= 127 (1 + 2^-22), so the codes need no clamp.
__device__ __forceinline__ float encode16(const float (&v)[16], float top, uint4& out) {
  const bool fine = top < INFINITY;  // false for NaN
  const bool kept = fine && top >= kTiny;
  const float mul = kept ? __fmul_rn(__frcp_rn(top), 127.0f) : 0.f;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[4 * j + i], mul), 12582912.f));
    w[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  out = kept ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0, 0, 0, 0);
  return kept ? __fmul_rn(top, kInv127) : fine ? 0.f : __int_as_float(0x7fffffff);
}

// The reverse trick: a byte b + 128 under the exponent of 2^23 is the float 2^23 + b + 128.
// v = code * scale.
__device__ __forceinline__ void decode16(const uint4& q, float scale, float (&v)[16]) {
  const uint32_t w[4] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u, q.z ^ 0x80808080u, q.w ^ 0x80808080u};
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[4 * j + i] = __fmul_rn(
          __fadd_rn(__uint_as_float(__byte_perm(w[j], 0x4b000000u, 0x7440 + i)), -8388736.f), scale);
}

// Row and chunk of a thread (the launch has fewer than 2^31 threads).
__device__ __forceinline__ void split_index(const FastDiv& slots, int64_t& row, int& slot) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t r = slots.div(idx);
  row = r;
  slot = static_cast<int>(idx - r * slots.d);
}

__device__ __forceinline__ float sigmoid(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return r;
}

// ------------------------------------------------------------------ quantise / dequantise
template <typename T, Rows R>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                       float* __restrict__ scale, int64_t rows, int n,
                                                       int64_t ldx, int64_t pitch, int groups, int lanes_log2,
                                                       FastDiv slots) {
  // `slots` threads per row: whole groups
  int64_t row;
  int slot;
  split_index(slots, row, slot);
  const int c = slot * kChunk;
  const int left = row < rows ? n - c : 0;
  float v[16];
  if constexpr (R == kRowsAny) {
    __shared__ float boxes[kBoxes<R>];
    load16_any(x + row * ldx + c, left, v, boxes + threadIdx.x / 32 * (32 * 17));
  } else {
    load16<T, R>(x + row * ldx + c, left, v);
  }
  const float top = group_top(v, lanes_log2);
  uint4 code;
  const float s = encode16(v, top, code);
  if (left > 0) {
    *reinterpret_cast<uint4*>(q + row * pitch + c) = code;
    if ((slot & ((1 << lanes_log2) - 1)) == 0) scale[row * groups + (slot >> lanes_log2)] = s;
  }
}

template <typename T, Rows R>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* __restrict__ q,
                                                         const float* __restrict__ scale,
                                                         T* __restrict__ x, int64_t rows, int n,
                                                         int64_t ldx, int64_t pitch, int groups, int lanes_log2,
                                                         FastDiv slots) {
  int64_t row;
  int slot;
  split_index(slots, row, slot);
  const int c = slot * kChunk;
  const int left = row < rows ? n - c : 0;
  if (R != kRowsAny && left <= 0) return;
  float v[16];
  if (left > 0)
    decode16(*reinterpret_cast<const uint4*>(q + row * pitch + c), scale[row * groups + (slot >> lanes_log2)], v);
  if constexpr (R == kRowsAny) {
    __shared__ float boxes[kBoxes<R>];
    if (left <= 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    store16_any(x + row * ldx + c, left, v, boxes + threadIdx.x / 32 * (32 * 17));
  } else {
    store16<T, R>(x + row * ldx + c, left, v);
  }
}

// ------------------------------------------------------------------ RMSNorm
// y = w x r, r = rsqrt(mean x^2 + eps), and the 8-bit copy of x, from one read of x.
// NT threads share a row (VPT chunks each); blocks of max(NT, 128) threads.
template <int NT, int VPT, Rows R>
__global__ void __launch_bounds__(NT > 128 ? NT : 128)
    rms_norm8_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ w,
                     __nv_bfloat16* __restrict__ y, float* __restrict__ rstd, int8_t* __restrict__ q,
                     float* __restrict__ scale, int64_t rows, int H, int64_t ldx, int64_t ldy,
                     int64_t pitch, int groups, int lanes_log2, float eps) {
  __shared__ float red[NT / 32];
  constexpr int RPB = NT >= 128 ? 1 : 128 / NT;
  const int t = threadIdx.x % NT;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / NT;
  const bool here = row < rows;
  float v[VPT][16];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * NT) * kChunk;
    load16<__nv_bfloat16, R>(x + row * ldx + c, here ? H - c : 0, v[i]);
#pragma unroll
    for (int j = 0; j < 16; ++j) ss += v[i][j] * v[i][j];
  }
  ss = warp_sum(ss);
  if (NT > 32 && t % 32 == 0) red[t / 32] = ss;
  // the codes need no sum: they are written while the row's warps come together
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int slot = t + i * NT;
    const float top = group_top(v[i], lanes_log2);
    uint4 code;
    const float s = encode16(v[i], top, code);
    if (here && slot * kChunk < H) {
      *reinterpret_cast<uint4*>(q + row * pitch + slot * kChunk) = code;
      if ((slot & ((1 << lanes_log2) - 1)) == 0) scale[row * groups + (slot >> lanes_log2)] = s;
    }
  }
  if (NT > 32) {
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) ss += red[i];
  }
  const float r = rsqrtf(ss / H + eps);
  if (here && t == 0) rstd[row] = r;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * NT) * kChunk;
    if (!here || c >= H) continue;
    float wv[16];
    load16<__nv_bfloat16, R>(w + c, H - c, wv);
#pragma unroll
    for (int j = 0; j < 16; ++j) wv[j] *= v[i][j] * r;
    store16<__nv_bfloat16, R>(y + row * ldy + c, H - c, wv);
  }
}

// n = x8 r,  dx = r (dy w - n mean(dy w n)),  y8 = n w,  dw = sum over rows of dy n.
// A walker (NT threads) takes a run of rows; its share of dw stays in registers and goes to
// part[walker], which dw_sum_kernel adds up in walker order (no atomics: the same sums on
// every run).  This form is for short rows, one warp each.
template <int VPT, Rows R>
__global__ void __launch_bounds__(128)
    rms_norm8_bwd_warp_kernel(const __nv_bfloat16* __restrict__ dy, const int8_t* __restrict__ q,
                              const float* __restrict__ scale, const __nv_bfloat16* __restrict__ w,
                              const float* __restrict__ rstd, __nv_bfloat16* __restrict__ dx,
                              __nv_bfloat16* __restrict__ y8, float* __restrict__ part, int64_t rows, int H,
                              int64_t lddy, int64_t pitch, int groups, int lanes_log2, int rows_per_walker) {
  const int t = threadIdx.x % 32;
  const int64_t walker = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int64_t r0 = walker * rows_per_walker, r1 = min(rows, r0 + rows_per_walker);
  float dw[VPT][16];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) dw[i][j] = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const float r = rstd[row];
    float n[VPT][16], g[VPT][16];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int slot = t + i * 32;
      const int c = slot * kChunk;
      if (c < H) {
        decode16(*reinterpret_cast<const uint4*>(q + row * pitch + c), scale[row * groups + (slot >> lanes_log2)], n[i]);
        load16<__nv_bfloat16, R>(dy + row * lddy + c, H - c, g[i]);
        float wv[16];
        load16<__nv_bfloat16, R>(w + c, H - c, wv);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          n[i][j] *= r;
          dw[i][j] += g[i][j] * n[i][j];
          g[i][j] *= wv[j];
          dot += g[i][j] * n[i][j];
          wv[j] *= n[i][j];
        }
        store16<__nv_bfloat16, R>(y8 + row * H + c, H - c, wv);
      }
    }
    dot = warp_sum(dot) / H;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * 32) * kChunk;
      if (c < H) {
#pragma unroll
        for (int j = 0; j < 16; ++j) g[i][j] = r * (g[i][j] - n[i][j] * dot);
        store16<__nv_bfloat16, R>(dx + row * H + c, H - c, g[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * 32) * kChunk;
    if (c < H && r0 < rows) store16<float, kRows16>(part + walker * H + c, H - c, dw[i]);
  }
}

__device__ __forceinline__ uint64_t clock_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Long rows: a block per walker.  The rows' codes and dy come through a ring of kStages bulk
// copies into shared memory, so the next rows are on their way during this one's reduction.
// One barrier per row: the sums of the warps alternate between two buffers, and the stage that the
// previous row used is refilled after this row's barrier.  After a wait that ran out nothing more is
// fetched, and the block stays (for a bounded time) until what is on its way has landed.
constexpr int kStages = 3;
constexpr int kErrNormWait = 302;  // a bulk copy did not arrive

template <int NT, int VPT, Rows R>
__global__ void __launch_bounds__(NT, 512 / NT)
    rms_norm8_bwd_kernel(const __nv_bfloat16* __restrict__ dy, const int8_t* __restrict__ q,
                         const float* __restrict__ scale, const __nv_bfloat16* __restrict__ w,
                         const float* __restrict__ rstd, __nv_bfloat16* __restrict__ dx,
                         __nv_bfloat16* __restrict__ y8, float* __restrict__ part, int64_t rows, int H,
                         int64_t lddy, int64_t pitch, int groups, int lanes_log2, int rows_per_walker,
                         int* __restrict__ err) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kStages];
  __shared__ float red[2][NT / 32];
  const int t = threadIdx.x;
  const int64_t r0 = (int64_t)blockIdx.x * rows_per_walker;
  const int count = static_cast<int>(min(rows - r0, (int64_t)rows_per_walker));
  const uint32_t code_bytes = static_cast<uint32_t>(pitch), dy_bytes = 2u * H;
  const uint32_t stage_bytes = code_bytes + dy_bytes;
  auto arrived = [&](int k) {  // waits for row k, about two seconds at most
    if (mbar_try_wait(&full[k % kStages], (k / kStages) & 1)) return true;
    const uint64_t start = clock_ns();
    while (!mbar_try_wait(&full[k % kStages], (k / kStages) & 1))
      if (clock_ns() - start > 2000000000ull) return false;
    return true;
  };
  auto fetch = [&](int k) {  // one thread
    uint8_t* s = ring + (k % kStages) * stage_bytes;
    mbar_arrive_expect_tx(&full[k % kStages], stage_bytes);
    bulk_load(s, q + (r0 + k) * pitch, code_bytes, &full[k % kStages]);
    bulk_load(s + code_bytes, dy + (r0 + k) * lddy, dy_bytes, &full[k % kStages]);
  };
  if (t == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
    for (int k = 0; k < min(count, kStages - 1); ++k) fetch(k);
  }
  uint32_t wq[VPT][8];
  float dw[VPT][16], sc[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int slot = t + i * NT, c = slot * kChunk;
#pragma unroll
    for (int j = 0; j < 8; ++j) wq[i][j] = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) dw[i][j] = 0.f;
    sc[i] = 0.f;
    if (c < H) {
      float wv[16];
      load16<__nv_bfloat16, R>(w + c, H - c, wv);
      pack(wv, wq[i], __nv_bfloat16{});
      sc[i] = scale[r0 * groups + (slot >> lanes_log2)];
    }
  }
  float r = rstd[r0];
  __syncthreads();  // barriers are initialised
  int late = count;  // the first row that did not arrive: the results are marked by err
  for (int k = 0; k < count; ++k) {
    const int64_t row = r0 + k;
    const uint8_t* s = ring + (k % kStages) * stage_bytes;
    // the next row's scalars
    float sc_next[VPT], r_next = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int slot = t + i * NT;
      sc_next[i] = (k + 1 < count && slot * kChunk < H) ? scale[(row + 1) * groups + (slot >> lanes_log2)] : 0.f;
    }
    if (k + 1 < count) r_next = rstd[row + 1];
    if (late == count && !arrived(k)) {
      atomicCAS(err, 0, kErrNormWait);
      late = k;
    }
    // n and dy w of a chunk; kept in registers over the barrier where one chunk is a thread's share
    auto chunk = [&](int i, float (&n)[16], float (&g)[16]) {
      const int c = (t + i * NT) * kChunk;
      decode16(*reinterpret_cast<const uint4*>(s + c), sc[i] * r, n);
      load16<__nv_bfloat16, kRows16>(reinterpret_cast<const __nv_bfloat16*>(s + code_bytes) + c, H - c, g);
    };
    float n[16], g[16];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * NT) * kChunk;
      if (c < H) {
        float wv[16], y[16];
        chunk(i, n, g);
        unpack(wq[i], wv, __nv_bfloat16{});
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          dw[i][j] += g[j] * n[j];
          g[j] *= wv[j];
          dot += g[j] * n[j];
          y[j] = wv[j] * n[j];
        }
        store16<__nv_bfloat16, R>(y8 + row * H + c, H - c, y);
      }
    }
    dot = warp_sum(dot);
    if (t % 32 == 0) red[k & 1][t / 32] = dot;
    __syncthreads();
    if (t == 0 && late == count && k + kStages - 1 < count) fetch(k + kStages - 1);
    dot = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) dot += red[k & 1][i];
    dot /= H;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * NT) * kChunk;
      if (c < H) {
        if (VPT > 1) {
          float wv[16];
          chunk(i, n, g);
          unpack(wq[i], wv, __nv_bfloat16{});
#pragma unroll
          for (int j = 0; j < 16; ++j) g[j] *= wv[j];
        }
        float d[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) d[j] = r * (g[j] - n[j] * dot);
        store16<__nv_bfloat16, R>(dx + row * H + c, H - c, d);
      }
      sc[i] = sc_next[i];
    }
    r = r_next;
  }
  if (t == 0)  // the rows that had been fetched when it gave up
    for (int k = late; k < min(count, late + kStages - 1); ++k) arrived(k);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * NT) * kChunk;
    if (c < H) store16<float, kRows16>(part + (int64_t)blockIdx.x * H + c, H - c, dw[i]);
  }
}

// dw[c] = sum of part[0..walkers)[c]: 32 columns per block, 32 rows of threads.
__global__ void __launch_bounds__(1024) dw_sum_kernel(const float* __restrict__ part, float* __restrict__ dw,
                                                      int walkers, int H) {
  __shared__ float red[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, k = threadIdx.x / 32;
  float s = 0.f;
  if (c < H)
    for (int i = k; i < walkers; i += 32) s += part[(int64_t)i * H + c];
  red[k][threadIdx.x % 32] = s;
  __syncthreads();
  s = warp_sum(red[threadIdx.x % 32][k]);  // warp k adds column k
  if (threadIdx.x % 32 == 0 && blockIdx.x * 32 + k < H) dw[blockIdx.x * 32 + k] = s;
}

// ------------------------------------------------------------------ SwiGLU
// gu = [gate F | up F] -> h = silu(g) u, and the 8-bit copies of both halves (groups do not
// cross from gate to up: each half is a row of its own in the code, pitch bytes apart).
// Five blocks per SM: 84.0 us for 4096 x 14336, 90.0 without the bound on registers, 85.3 with six.
template <Rows R>
__global__ void __launch_bounds__(256, 5) swiglu8_kernel(const __nv_bfloat16* __restrict__ gu,
                                                      __nv_bfloat16* __restrict__ h, int8_t* __restrict__ q,
                                                      float* __restrict__ scale, int64_t rows, int F,
                                                      int64_t ldgu, int64_t ldh, int64_t pitch, int groups,
                                                      int lanes_log2, FastDiv slots) {
  int64_t row;
  int slot;
  split_index(slots, row, slot);
  const int c = slot * kChunk;
  const int left = row < rows ? F - c : 0;
  float g[16], u[16];
  load16<__nv_bfloat16, R>(gu + row * ldgu + c, left, g);
  load16<__nv_bfloat16, R>(gu + row * ldgu + F + c, left, u);
  const float tg = group_top(g, lanes_log2), tu = group_top(u, lanes_log2);
  uint4 cg, cu;
  const float sg = encode16(g, tg, cg), su = encode16(u, tu, cu);
  if (left <= 0) return;
  *reinterpret_cast<uint4*>(q + 2 * row * pitch + c) = cg;
  *reinterpret_cast<uint4*>(q + (2 * row + 1) * pitch + c) = cu;
  if ((slot & ((1 << lanes_log2) - 1)) == 0) {
    scale[2 * row * groups + (slot >> lanes_log2)] = sg;
    scale[(2 * row + 1) * groups + (slot >> lanes_log2)] = su;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = g[i] * sigmoid(g[i]) * u[i];  // g u may leave fp32's range
  store16<__nv_bfloat16, R>(h + row * ldh + c, left, g);
}

// s = sigmoid(g8): dg = dh u8 s (1 + g8 (1 - s)), du = dh g8 s, h8 = g8 s u8.
template <Rows R>
__global__ void __launch_bounds__(256) swiglu8_bwd_kernel(const __nv_bfloat16* __restrict__ dh,
                                                          const int8_t* __restrict__ q,
                                                          const float* __restrict__ scale,
                                                          __nv_bfloat16* __restrict__ dgu,
                                                          __nv_bfloat16* __restrict__ h8, int64_t rows, int F,
                                                          int64_t lddh, int64_t lddgu, int64_t ldh,
                                                          int64_t pitch, int groups, int lanes_log2,
                                                          FastDiv slots) {
  int64_t row;
  int slot;
  split_index(slots, row, slot);
  if (row >= rows) return;
  const int c = slot * kChunk;
  float d[16], g[16], u[16], hv[16];
  load16<__nv_bfloat16, R>(dh + row * lddh + c, F - c, d);
  decode16(*reinterpret_cast<const uint4*>(q + 2 * row * pitch + c), scale[2 * row * groups + (slot >> lanes_log2)], g);
  decode16(*reinterpret_cast<const uint4*>(q + (2 * row + 1) * pitch + c),
           scale[(2 * row + 1) * groups + (slot >> lanes_log2)], u);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float s = sigmoid(g[i]);
    const float gs = g[i] * s;
    hv[i] = gs * u[i];
    u[i] = s * (1.f + g[i] * (1.f - s)) * u[i] * d[i];  // dg: s first, d u may leave fp32's range
    g[i] = d[i] * gs;                                   // du
  }
  store16<__nv_bfloat16, R>(dgu + row * lddgu + c, F - c, u);
  store16<__nv_bfloat16, R>(dgu + row * lddgu + F + c, F - c, g);
  store16<__nv_bfloat16, R>(h8 + row * ldh + c, F - c, hv);
}

// ------------------------------------------------------------------ host side
unsigned blocks_for(int64_t threads) {  // 2^31 threads are 2^35 values
  TORCH_CHECK_VALUE(threads < (int64_t(1) << 31) - 256, "act8: tensor too large for one launch");
  return static_cast<unsigned>((threads + 255) / 256);
}

int log2_lanes(int64_t group) { return group == 32 ? 1 : group == 64 ? 2 : group == 128 ? 3 : 4; }

FastDiv divider(int64_t slots) {
  FastDiv f;
  f.set(static_cast<uint32_t>(slots));
  return f;
}

Rows rows_of(const torch::Tensor& t) {
  const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
  const int64_t pitch = (t.dim() > 1 && t.size(0) > 1 ? t.stride(0) : 0) * t.element_size();
  return p % 32 == 0 && pitch % 32 == 0 ? kRows32 : p % 16 == 0 && pitch % 16 == 0 ? kRows16 : kRowsAny;
}

void check_group(int64_t group) {
  TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128 || group == 256,
                    "act8: group must be 32, 64, 128 or 256, got ", group);
}

// x as rows over its last dimension, with a unit inner stride; `vec`: on 16-byte boundaries too.
torch::Tensor as_rows(const torch::Tensor& x, const char* name, bool vec) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "act8: ", name, " needs at least one dimension");
  TORCH_CHECK_VALUE(x.is_cuda(), "act8: ", name, " must be a CUDA tensor");
  const int64_t n = x.size(-1);
  int64_t rows = 1;
  for (int i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  torch::Tensor r = x.dim() == 2 ? x : x.reshape({rows, n});
  if (n > 1 && r.stride(1) != 1) r = r.contiguous();
  if (vec) {
    TORCH_CHECK(x.scalar_type() == at::kBFloat16, "act8: ", name, " must be bf16 on CUDA, got ", x.scalar_type());
    TORCH_CHECK(n >= 8 && n % 8 == 0, "act8: rows of ", name, " must hold a multiple of 8 values, got ", n);
    if (rows_of(r) == kRowsAny) r = r.clone(at::MemoryFormat::Contiguous);
  }
  return r;
}

std::pair<torch::Tensor, torch::Tensor> code_buffers(const torch::Tensor& like, int64_t rows, int64_t n,
                                                     int64_t group) {
  return {torch::empty({rows, (n + 15) / 16 * 16}, like.options().dtype(at::kChar)),
          torch::empty({rows, (n + group - 1) / group}, like.options().dtype(at::kFloat))};
}

void check_code(const torch::Tensor& q, const torch::Tensor& scale, int64_t code_rows, int64_t n, int64_t group) {
  check_group(group);
  TORCH_CHECK(q.is_cuda() && scale.is_cuda() && q.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat,
              "act8: codes must be int8 and scales fp32 CUDA tensors");
  TORCH_CHECK(q.dim() == 2 && q.is_contiguous() && q.size(0) == code_rows && q.size(1) == (n + 15) / 16 * 16 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "act8: codes must be contiguous [rows, n rounded up to 16] on a 16-byte boundary");
  TORCH_CHECK(scale.dim() == 2 && scale.is_contiguous() && scale.size(0) == code_rows &&
                  scale.size(1) == (n + group - 1) / group,
              "act8: scales must be contiguous [rows, groups]");
}

torch::Tensor check_weight(const torch::Tensor& w, int64_t H) {
  TORCH_CHECK(w.is_cuda() && w.scalar_type() == at::kBFloat16 && w.numel() == H,
              "act8: the weight must be a bf16 CUDA vector of ", H, " values");
  return w.is_contiguous() && rows_of(w) != kRowsAny ? w : w.clone(at::MemoryFormat::Contiguous);
}

const __nv_bfloat16* bf16(const torch::Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); }
__nv_bfloat16* bf16_out(torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }

template <typename T>
void launch_quantize(Rows r, unsigned grid, cudaStream_t st, const torch::Tensor& x, torch::Tensor& q,
                     torch::Tensor& scale, int lanes) {
  auto kern = r == kRows32 ? quantize_kernel<T, kRows32>
                           : r == kRows16 ? quantize_kernel<T, kRows16> : quantize_kernel<T, kRowsAny>;
  kern<<<grid, 256, 0, st>>>(reinterpret_cast<const T*>(x.data_ptr()), q.data_ptr<int8_t>(), scale.data_ptr<float>(),
                             x.size(0), x.size(1), x.stride(0), q.size(1), scale.size(1), lanes,
                             divider(scale.size(1) << lanes));
}
template <typename T>
void launch_dequantize(Rows r, unsigned grid, cudaStream_t st, const torch::Tensor& q, const torch::Tensor& scale,
                       torch::Tensor& x, int64_t rows, int n, int lanes) {
  auto kern = r == kRows32 ? dequantize_kernel<T, kRows32>
                           : r == kRows16 ? dequantize_kernel<T, kRows16> : dequantize_kernel<T, kRowsAny>;
  kern<<<grid, 256, 0, st>>>(q.data_ptr<int8_t>(), scale.data_ptr<float>(), reinterpret_cast<T*>(x.data_ptr()), rows,
                             n, n, q.size(1), scale.size(1), lanes, divider((n + kChunk - 1) / kChunk));
}

}  // namespace

// (codes, scales) of x (bf16, fp16 or fp32), groups along its last dimension.
std::tuple<torch::Tensor, torch::Tensor> act8_quantize(const torch::Tensor& x, int64_t group) {
  check_group(group);
  const auto type = x.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
              "act8.quantize: bf16, fp16 or fp32 expected, got ", type);
  const c10::cuda::CUDAGuard guard(x.device());
  const torch::Tensor r = as_rows(x, "x", false);
  const int64_t rows = r.size(0), n = r.size(1);
  TORCH_CHECK_VALUE(n < (int64_t(1) << 31), "act8: rows too long");
  auto [q, scale] = code_buffers(r, rows, n, group);
  if (rows == 0 || n == 0) return {q, scale};
  auto st = at::cuda::getCurrentCUDAStream();
  const int lanes = log2_lanes(group);
  const unsigned grid = blocks_for(rows * (scale.size(1) << lanes));
  if (type == at::kBFloat16) launch_quantize<__nv_bfloat16>(rows_of(r), grid, st, r, q, scale, lanes);
  else if (type == at::kHalf) launch_quantize<__half>(rows_of(r), grid, st, r, q, scale, lanes);
  else launch_quantize<float>(rows_of(r), grid, st, r, q, scale, lanes);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, scale};
}

// The kept values as a contiguous tensor of `sizes` (rows of n values).
torch::Tensor act8_dequantize(const torch::Tensor& q, const torch::Tensor& scale, const std::vector<int64_t>& sizes,
                              int64_t n, torch::ScalarType dtype, int64_t group) {
  check_one_device("act8.dequantize", q, scale);
  check_code(q, scale, q.size(0), n, group);
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat,
              "act8.dequantize: bf16, fp16 or fp32 expected, got ", dtype);
  const c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor x = torch::empty(sizes, q.options().dtype(dtype));
  const int64_t rows = q.size(0);
  TORCH_CHECK(x.numel() == rows * n, "act8.dequantize: codes of ", rows * n, " values do not fit ", x.sizes());
  if (x.numel() == 0) return x;
  auto st = at::cuda::getCurrentCUDAStream();
  const int lanes = log2_lanes(group);
  const unsigned grid = blocks_for(rows * ((n + kChunk - 1) / kChunk));
  const int64_t pitch = n * x.element_size();  // the allocation itself starts on a 512-byte boundary
  const Rows r = rows == 1 || pitch % 32 == 0 ? kRows32 : pitch % 16 == 0 ? kRows16 : kRowsAny;
  if (dtype == at::kBFloat16) launch_dequantize<__nv_bfloat16>(r, grid, st, q, scale, x, rows, n, lanes);
  else if (dtype == at::kHalf) launch_dequantize<__half>(r, grid, st, q, scale, x, rows, n, lanes);
  else launch_dequantize<float>(r, grid, st, q, scale, x, rows, n, lanes);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return x;
}

// Threads per row and chunks per thread for a row of H values.
#define FT_NORM8_SIZES(LAUNCH)          \
  if (H <= 512) LAUNCH(32, 1);          \
  else if (H <= 1024) LAUNCH(32, 2);    \
  else if (H <= 2048) LAUNCH(128, 1);   \
  else if (H <= 4096) LAUNCH(256, 1);   \
  else if (H <= 8192) LAUNCH(512, 1);   \
  else LAUNCH(512, 2)

// (y, rstd, codes, scales)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> act8_rms_norm(const torch::Tensor& x,
                                                                                     const torch::Tensor& weight,
                                                                                     double eps, int64_t group) {
  check_group(group);
  check_one_device("act8.rms_norm", x, weight);
  const c10::cuda::CUDAGuard guard(x.device());
  const torch::Tensor r = as_rows(x, "x", true);
  const int64_t rows = r.size(0);
  const int H = r.size(1);
  TORCH_CHECK(H <= 16384, "act8.rms_norm: at most 16384 values per row, got ", H);
  const torch::Tensor w = check_weight(weight, H);
  torch::Tensor y = torch::empty(x.sizes(), r.options());
  torch::Tensor rstd = torch::empty({rows}, r.options().dtype(at::kFloat));
  auto [q, scale] = code_buffers(r, rows, H, group);
  if (rows == 0) return {y, rstd, q, scale};
  auto st = at::cuda::getCurrentCUDAStream();
  const int lanes = log2_lanes(group), groups = scale.size(1);
  const bool wide = H % 16 == 0 && rows_of(r) == kRows32 && rows_of(w) == kRows32;
#define FT_L(NT, VPT)                                                                                             \
  do {                                                                                                            \
    constexpr int rpb = NT >= 128 ? 1 : 128 / NT;                                                                 \
    auto kern = wide ? rms_norm8_kernel<NT, VPT, kRows32> : rms_norm8_kernel<NT, VPT, kRows16>;                   \
    kern<<<static_cast<unsigned>((rows + rpb - 1) / rpb), rpb * NT, 0, st>>>(                                     \
        bf16(r), bf16(w), bf16_out(y), rstd.data_ptr<float>(), q.data_ptr<int8_t>(), scale.data_ptr<float>(), rows, \
        H, r.stride(0), H, q.size(1), groups, lanes, static_cast<float>(eps));                                    \
  } while (0)
  FT_NORM8_SIZES(FT_L);
#undef FT_L
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {y, rstd, q, scale};
}

// (dx, dw, y8)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> act8_rms_norm_bwd(
    const torch::Tensor& dy, const torch::Tensor& q, const torch::Tensor& scale, const torch::Tensor& weight,
    const torch::Tensor& rstd, int64_t group, torch::Tensor& err) {
  check_one_device("act8.rms_norm_bwd", dy, q, scale, weight, rstd, err);
  const c10::cuda::CUDAGuard guard(dy.device());
  const torch::Tensor g = as_rows(dy, "dy", true);
  const int64_t rows = g.size(0);
  const int H = g.size(1);
  TORCH_CHECK(H <= 16384, "act8.rms_norm_bwd: at most 16384 values per row, got ", H);
  check_code(q, scale, rows, H, group);
  const torch::Tensor w = check_weight(weight, H);
  TORCH_CHECK(rstd.is_cuda() && rstd.scalar_type() == at::kFloat && rstd.numel() == rows && rstd.is_contiguous());
  const auto f32 = g.options().dtype(at::kFloat);
  torch::Tensor dx = torch::empty(dy.sizes(), g.options()), y8 = torch::empty(dy.sizes(), g.options());
  if (rows == 0) return {dx, torch::zeros({H}, f32), y8};
  auto st = at::cuda::getCurrentCUDAStream();
  // as many walkers as blocks (or, for short rows, warps) are resident, or one per row: 512
  // threads per SM with everything in registers (49.1 us for 4096 x 8192) do better than 1024 that
  // decode a row twice (55.0 us), and write half as many shares of dw
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t most = H <= 1024 ? sms * 16 : H <= 2048 ? sms * 4 : H <= 4096 ? sms * 2 : sms;
  const int64_t per = (rows + most - 1) / most, walkers = (rows + per - 1) / per;
  torch::Tensor dw = torch::empty({H}, f32), part = torch::empty({walkers, H}, f32);
  const int lanes = log2_lanes(group), groups = scale.size(1);
  const bool wide = H % 16 == 0 && rows_of(g) == kRows32 && rows_of(w) == kRows32;
  const int smem = kStages * static_cast<int>(q.size(1) + 2 * (int64_t)H);
#define FT_ARGS                                                                                                  \
  bf16(g), q.data_ptr<int8_t>(), scale.data_ptr<float>(), bf16(w), rstd.data_ptr<float>(), bf16_out(dx),         \
      bf16_out(y8), part.data_ptr<float>(), rows, H, g.stride(0), q.size(1), groups, lanes, static_cast<int>(per)
#define FT_L(NT, VPT)                                                                                            \
  do {                                                                                                           \
    if constexpr (NT == 32) {                                                                                    \
      auto kern = wide ? rms_norm8_bwd_warp_kernel<VPT, kRows32> : rms_norm8_bwd_warp_kernel<VPT, kRows16>;      \
      kern<<<static_cast<unsigned>((walkers + 3) / 4), 128, 0, st>>>(FT_ARGS);                                   \
    } else {                                                                                                     \
      constexpr int nt = NT < 128 ? 128 : NT;                                                                    \
      auto kern = wide ? rms_norm8_bwd_kernel<nt, VPT, kRows32> : rms_norm8_bwd_kernel<nt, VPT, kRows16>;        \
      static unsigned long long done[2] = {0, 0};                                                                \
      smem_attr_once(kern, kStages * 3 * 16 * nt * VPT, done[wide]);                                             \
      kern<<<static_cast<unsigned>(walkers), nt, smem, st>>>(FT_ARGS, err.data_ptr<int>());                      \
    }                                                                                                            \
  } while (0)
  FT_NORM8_SIZES(FT_L);
#undef FT_L
#undef FT_ARGS
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  dw_sum_kernel<<<(H + 31) / 32, 1024, 0, st>>>(part.data_ptr<float>(), dw.data_ptr<float>(),
                                                static_cast<int>(walkers), H);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dx, dw, y8};
}

// (h, codes, scales) of gu = [gate | up]
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> act8_swiglu(const torch::Tensor& gu, int64_t group) {
  check_group(group);
  const c10::cuda::CUDAGuard guard(gu.device());
  const torch::Tensor r = as_rows(gu, "gate and up", true);
  const int64_t rows = r.size(0);
  const int F = r.size(1) / 2;
  TORCH_CHECK(r.size(1) % 16 == 0, "act8.swiglu: gate and up must hold a multiple of 8 values each, got ", r.size(1));
  std::vector<int64_t> sizes = gu.sizes().vec();
  sizes.back() = F;
  torch::Tensor h = torch::empty(sizes, r.options());
  auto [q, scale] = code_buffers(r, 2 * rows, F, group);
  if (rows == 0) return {h, q, scale};
  const int lanes = log2_lanes(group), groups = scale.size(1);
  auto kern = F % 16 == 0 && rows_of(r) == kRows32 ? swiglu8_kernel<kRows32> : swiglu8_kernel<kRows16>;
  kern<<<blocks_for(rows * ((int64_t)groups << lanes)), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      bf16(r), bf16_out(h), q.data_ptr<int8_t>(), scale.data_ptr<float>(), rows, F, r.stride(0), F, q.size(1), groups,
      lanes, divider((int64_t)groups << lanes));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {h, q, scale};
}

// (dgu, h8)
std::tuple<torch::Tensor, torch::Tensor> act8_swiglu_bwd(const torch::Tensor& dh, const torch::Tensor& q,
                                                         const torch::Tensor& scale, int64_t group) {
  check_one_device("act8.swiglu_bwd", dh, q, scale);
  const c10::cuda::CUDAGuard guard(dh.device());
  const torch::Tensor r = as_rows(dh, "dh", true);
  const int64_t rows = r.size(0);
  const int F = r.size(1);
  check_code(q, scale, 2 * rows, F, group);
  std::vector<int64_t> sizes = dh.sizes().vec();
  sizes.back() = 2 * F;
  torch::Tensor dgu = torch::empty(sizes, r.options()), h8 = torch::empty(dh.sizes(), r.options());
  if (rows == 0) return {dgu, h8};
  const int lanes = log2_lanes(group), groups = scale.size(1);
  auto kern = F % 16 == 0 && rows_of(r) == kRows32 ? swiglu8_bwd_kernel<kRows32> : swiglu8_bwd_kernel<kRows16>;
  kern<<<blocks_for(rows * ((F + kChunk - 1) / kChunk)), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      bf16(r), q.data_ptr<int8_t>(), scale.data_ptr<float>(), bf16_out(dgu), bf16_out(h8), rows, F, r.stride(0),
      2 * (int64_t)F, F, q.size(1), groups, lanes, divider((F + kChunk - 1) / kChunk));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dgu, h8};
}

}  // namespace ft

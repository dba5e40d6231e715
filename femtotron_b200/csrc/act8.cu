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
// One thread owns 16 neighbouring values: two 16-byte bf16 loads, one 16-byte code store.  The
// G / 16 threads of a group are neighbours in one warp and find the maximum with shuffles, so
// every value is read from memory once.  All kernels here are bound by HBM bandwidth.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ft {
namespace {

constexpr int kChunk = 16;            // values per thread
constexpr float kTiny = 7.52316385e-37f;  // 2^-120
constexpr float kInv127 = 1.0f / 127.0f;

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

template <typename T> struct alignas(16) Vec16 { T v[16 / sizeof(T)]; };

// Up to 16 values starting at p (`left` of them exist) as fp32, zeros after them.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load16(const T* p, int left, float (&v)[16]) {
  constexpr int PER = 16 / sizeof(T);
  if (ALIGNED && left >= 16) {
#pragma unroll
    for (int j = 0; j < 16 / PER; ++j) {
      const Vec16<T> q = *reinterpret_cast<const Vec16<T>*>(p + j * PER);
#pragma unroll
      for (int i = 0; i < PER; ++i) v[j * PER + i] = to_f(q.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < left ? to_f(p[i]) : 0.f;
  }
}
template <typename T, bool ALIGNED>
__device__ __forceinline__ void store16(T* p, int left, const float (&v)[16]) {
  constexpr int PER = 16 / sizeof(T);
  if (ALIGNED && left >= 16) {
#pragma unroll
    for (int j = 0; j < 16 / PER; ++j) {
      Vec16<T> q;
#pragma unroll
      for (int i = 0; i < PER; ++i) q.v[i] = from_f<T>(v[j * PER + i]);
      *reinterpret_cast<Vec16<T>*>(p + j * PER) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) p[i] = from_f<T>(v[i]);
  }
}

// Largest magnitude over the `lanes` neighbouring threads that share a group.  NaN has to win,
// so magnitudes are compared as their bit patterns (for non-negative floats the integer order
// is the order of the values, with NaN above infinity).
__device__ __forceinline__ float group_top(const float (&v)[16], int lanes) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  for (int o = lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return __uint_as_float(m);
}

// Codes of 16 values; returns the group's scale.  top = inf or NaN gives the scale NaN.
__device__ __forceinline__ float encode16(const float (&v)[16], float top, uint4& out) {
  const bool fine = top < INFINITY;  // false for NaN
  const float mul = (fine && top >= kTiny) ? __fmul_rn(__fdiv_rn(1.0f, top), 127.0f) : 0.f;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = __float2int_rn(__fmul_rn(v[4 * j + i], mul));
      x |= (static_cast<uint32_t>(min(127, max(-127, q))) & 0xffu) << (8 * i);
    }
    w[j] = x;
  }
  out = make_uint4(w[0], w[1], w[2], w[3]);
  return fine ? (top >= kTiny ? __fmul_rn(top, kInv127) : 0.f) : __int_as_float(0x7fffffff);
}

__device__ __forceinline__ void decode16(const uint4& q, float scale, float (&v)[16]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[4 * j + i] = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[j] >> (8 * i))), scale);
}

// ------------------------------------------------------------------ quantise / dequantise
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int8_t* __restrict__ q,
                                                       float* __restrict__ scale, int64_t rows, int n,
                                                       int64_t ldx, int64_t pitch, int groups, int lanes) {
  const int slots = groups * lanes;  // threads per row, whole groups
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / slots;
  const int slot = static_cast<int>(idx - row * slots);
  const int c = slot * kChunk;
  const int left = row < rows ? n - c : 0;
  float v[16];
  load16<T, ALIGNED>(x + row * ldx + c, left, v);
  const float top = group_top(v, lanes);
  uint4 code;
  const float s = encode16(v, top, code);
  if (left > 0) {
    *reinterpret_cast<uint4*>(q + row * pitch + c) = code;
    if (slot % lanes == 0) scale[row * groups + slot / lanes] = s;
  }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* __restrict__ q,
                                                         const float* __restrict__ scale,
                                                         T* __restrict__ x, int64_t rows, int n,
                                                         int64_t ldx, int64_t pitch, int groups, int lanes) {
  const int slots = (n + kChunk - 1) / kChunk;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / slots;
  if (row >= rows) return;
  const int slot = static_cast<int>(idx - row * slots);
  const int c = slot * kChunk;
  float v[16];
  decode16(*reinterpret_cast<const uint4*>(q + row * pitch + c), scale[row * groups + slot / lanes], v);
  store16<T, ALIGNED>(x + row * ldx + c, n - c, v);
}

// ------------------------------------------------------------------ RMSNorm
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (NT > 32) {
    const int w = threadIdx.x / 32;
    __syncthreads();  // the previous use of red is over
    if (threadIdx.x % 32 == 0) red[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) v += red[i];
  }
  return v;
}

// y = w x r, r = rsqrt(mean x^2 + eps), and the 8-bit copy of x, from one read of x.
// NT threads share a row (VPT chunks each); blocks of max(NT, 128) threads.
template <int NT, int VPT>
__global__ void __launch_bounds__(NT > 128 ? NT : 128)
    rms_norm8_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ w,
                     __nv_bfloat16* __restrict__ y, float* __restrict__ rstd, int8_t* __restrict__ q,
                     float* __restrict__ scale, int64_t rows, int H, int64_t ldx, int64_t ldy,
                     int64_t pitch, int groups, int lanes, float eps) {
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
    load16<__nv_bfloat16, true>(x + row * ldx + c, here ? H - c : 0, v[i]);
#pragma unroll
    for (int j = 0; j < 16; ++j) ss += v[i][j] * v[i][j];
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int slot = t + i * NT;
    const float top = group_top(v[i], lanes);
    uint4 code;
    const float s = encode16(v[i], top, code);
    if (here && slot * kChunk < H) {
      *reinterpret_cast<uint4*>(q + row * pitch + slot * kChunk) = code;
      if (slot % lanes == 0) scale[row * groups + slot / lanes] = s;
    }
  }
  ss = row_sum<NT>(ss, red);
  const float r = rsqrtf(ss / H + eps);
  if (here && t == 0) rstd[row] = r;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * NT) * kChunk;
    if (!here || c >= H) continue;
    float wv[16];
    load16<__nv_bfloat16, true>(w + c, H - c, wv);
#pragma unroll
    for (int j = 0; j < 16; ++j) wv[j] *= v[i][j] * r;
    store16<__nv_bfloat16, true>(y + row * ldy + c, H - c, wv);
  }
}

// n = x8 r,  dx = r (dy w - n mean(dy w n)),  y8 = n w,  dw = sum over rows of dy n.
// A block walks a run of rows; its share of dw stays in registers and goes to part[block],
// which dw_sum_kernel adds up in block order (no atomics: the same sums on every run).
template <int NT, int VPT>
__global__ void __launch_bounds__(NT > 128 ? NT : 128)
    rms_norm8_bwd_kernel(const __nv_bfloat16* __restrict__ dy, const int8_t* __restrict__ q,
                         const float* __restrict__ scale, const __nv_bfloat16* __restrict__ w,
                         const float* __restrict__ rstd, __nv_bfloat16* __restrict__ dx,
                         __nv_bfloat16* __restrict__ y8, float* __restrict__ part, int64_t rows, int H,
                         int64_t lddy, int64_t lddx, int64_t ldy, int64_t pitch, int groups, int lanes,
                         int rows_per_walker) {
  __shared__ float red[NT / 32];
  constexpr int RPB = NT >= 128 ? 1 : 128 / NT;
  const int t = threadIdx.x % NT;
  const int64_t walker = (int64_t)blockIdx.x * RPB + threadIdx.x / NT;
  const int64_t r0 = walker * rows_per_walker;
  float dw[VPT][16];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) dw[i][j] = 0.f;
  for (int k = 0; k < rows_per_walker; ++k) {
    const int64_t row = r0 + k;
    const bool here = row < rows;
    if (!here && NT >= 32) break;  // the whole row's threads leave together
    const float r = rstd[row];
    float n[VPT][16], g[VPT][16];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int slot = t + i * NT;
      const int c = slot * kChunk;
      if (c < H) {
        decode16(*reinterpret_cast<const uint4*>(q + row * pitch + c), scale[row * groups + slot / lanes], n[i]);
        load16<__nv_bfloat16, true>(dy + row * lddy + c, H - c, g[i]);
        float wv[16];
        load16<__nv_bfloat16, true>(w + c, H - c, wv);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          n[i][j] *= r;
          dw[i][j] += g[i][j] * n[i][j];
          g[i][j] *= wv[j];
          dot += g[i][j] * n[i][j];
          wv[j] *= n[i][j];
        }
        store16<__nv_bfloat16, true>(y8 + row * ldy + c, H - c, wv);
      }
    }
    dot = row_sum<NT>(dot, red) / H;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * NT) * kChunk;
      if (c < H) {
#pragma unroll
        for (int j = 0; j < 16; ++j) g[i][j] = r * (g[i][j] - n[i][j] * dot);
        store16<__nv_bfloat16, true>(dx + row * lddx + c, H - c, g[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * NT) * kChunk;
    if (c < H && r0 < rows) store16<float, true>(part + walker * H + c, H - c, dw[i]);
  }
}

// dw[c] = sum of part[0..walkers)[c]: 32 columns per block, 8 rows of threads.
__global__ void __launch_bounds__(256) dw_sum_kernel(const float* __restrict__ part, float* __restrict__ dw,
                                                     int walkers, int H) {
  __shared__ float red[8][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, k = threadIdx.x / 32;
  float s = 0.f;
  if (c < H)
    for (int i = k; i < walkers; i += 8) s += part[(int64_t)i * H + c];
  red[k][threadIdx.x % 32] = s;
  __syncthreads();
  if (k == 0 && c < H) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
    dw[c] = s;
  }
}

// ------------------------------------------------------------------ SwiGLU
// gu = [gate F | up F] -> h = silu(g) u, and the 8-bit copies of both halves (groups do not
// cross from gate to up: each half is a row of its own in the code, pitch bytes apart).
__global__ void __launch_bounds__(256) swiglu8_kernel(const __nv_bfloat16* __restrict__ gu,
                                                      __nv_bfloat16* __restrict__ h, int8_t* __restrict__ q,
                                                      float* __restrict__ scale, int64_t rows, int F,
                                                      int64_t ldgu, int64_t ldh, int64_t pitch, int groups,
                                                      int lanes) {
  const int slots = groups * lanes;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / slots;
  const int slot = static_cast<int>(idx - row * slots);
  const int c = slot * kChunk;
  const int left = row < rows ? F - c : 0;
  float g[16], u[16];
  load16<__nv_bfloat16, true>(gu + row * ldgu + c, left, g);
  load16<__nv_bfloat16, true>(gu + row * ldgu + F + c, left, u);
  const float tg = group_top(g, lanes), tu = group_top(u, lanes);
  uint4 cg, cu;
  const float sg = encode16(g, tg, cg), su = encode16(u, tu, cu);
  if (left <= 0) return;
  *reinterpret_cast<uint4*>(q + 2 * row * pitch + c) = cg;
  *reinterpret_cast<uint4*>(q + (2 * row + 1) * pitch + c) = cu;
  if (slot % lanes == 0) {
    scale[2 * row * groups + slot / lanes] = sg;
    scale[(2 * row + 1) * groups + slot / lanes] = su;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = g[i] * u[i] * __fdividef(1.f, 1.f + __expf(-g[i]));
  store16<__nv_bfloat16, true>(h + row * ldh + c, left, g);
}

// s = sigmoid(g8): dg = dh u8 s (1 + g8 (1 - s)), du = dh g8 s, h8 = g8 s u8.
__global__ void __launch_bounds__(256) swiglu8_bwd_kernel(const __nv_bfloat16* __restrict__ dh,
                                                          const int8_t* __restrict__ q,
                                                          const float* __restrict__ scale,
                                                          __nv_bfloat16* __restrict__ dgu,
                                                          __nv_bfloat16* __restrict__ h8, int64_t rows, int F,
                                                          int64_t lddh, int64_t lddgu, int64_t ldh,
                                                          int64_t pitch, int groups, int lanes) {
  const int slots = (F + kChunk - 1) / kChunk;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / slots;
  if (row >= rows) return;
  const int slot = static_cast<int>(idx - row * slots);
  const int c = slot * kChunk;
  float d[16], g[16], u[16], hv[16];
  load16<__nv_bfloat16, true>(dh + row * lddh + c, F - c, d);
  decode16(*reinterpret_cast<const uint4*>(q + 2 * row * pitch + c), scale[2 * row * groups + slot / lanes], g);
  decode16(*reinterpret_cast<const uint4*>(q + (2 * row + 1) * pitch + c),
           scale[(2 * row + 1) * groups + slot / lanes], u);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float s = __fdividef(1.f, 1.f + __expf(-g[i]));
    const float gs = g[i] * s;
    hv[i] = gs * u[i];
    u[i] = d[i] * u[i] * s * (1.f + g[i] * (1.f - s));  // dg
    g[i] = d[i] * gs;                                   // du
  }
  store16<__nv_bfloat16, true>(dgu + row * lddgu + c, F - c, u);
  store16<__nv_bfloat16, true>(dgu + row * lddgu + F + c, F - c, g);
  store16<__nv_bfloat16, true>(h8 + row * ldh + c, F - c, hv);
}

// ------------------------------------------------------------------ host side
unsigned blocks_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256;
  TORCH_CHECK(b < (int64_t(1) << 31), "act8: tensor too large for one launch");
  return static_cast<unsigned>(b);
}

bool aligned16(const torch::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.stride(0) * t.element_size()) % 16 == 0;
}

void check_code(const torch::Tensor& q, const torch::Tensor& scale, int64_t code_rows, int64_t n, int64_t group) {
  TORCH_CHECK(group == 32 || group == 64 || group == 128 || group == 256,
              "act8: group must be 32, 64, 128 or 256, got ", group);
  TORCH_CHECK(q.is_cuda() && scale.is_cuda() && q.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat,
              "act8: codes must be int8 and scales fp32 CUDA tensors");
  TORCH_CHECK(q.dim() == 2 && q.is_contiguous() && q.size(0) == code_rows && q.size(1) == (n + 15) / 16 * 16,
              "act8: codes must be contiguous [rows, n rounded up to 16]");
  TORCH_CHECK(scale.dim() == 2 && scale.is_contiguous() && scale.size(0) == code_rows &&
                  scale.size(1) == (n + group - 1) / group,
              "act8: scales must be contiguous [rows, groups]");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0, "act8: codes must be 16-byte aligned");
}

void check_rows(const torch::Tensor& t, int64_t rows, int64_t n, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(0) == rows &&
                  t.size(1) == n && t.stride(1) == 1 && aligned16(t),
              "act8: ", name, " must be a bf16 CUDA tensor [", rows, ", ", n,
              "] with unit inner stride and 16-byte aligned rows");
}

}  // namespace

void act8_quantize(const torch::Tensor& x, torch::Tensor& q, torch::Tensor& scale, int64_t group) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1),
              "act8_quantize: a 2-D CUDA tensor with unit inner stride is required");
  const int64_t rows = x.size(0);
  const int n = x.size(1);
  check_code(q, scale, rows, n, group);
  if (rows == 0 || n == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int lanes = group / kChunk, groups = scale.size(1);
  const unsigned grid = blocks_for(rows * groups * lanes);
  const bool al = aligned16(x);
#define FT_Q(T, AL)                                                                                    \
  quantize_kernel<T, AL><<<grid, 256, 0, st>>>(reinterpret_cast<const T*>(x.data_ptr()),               \
                                               q.data_ptr<int8_t>(), scale.data_ptr<float>(), rows, n, \
                                               x.stride(0), q.size(1), groups, lanes)
#define FT_QA(T) do { if (al) FT_Q(T, true); else FT_Q(T, false); } while (0)
  if (x.scalar_type() == at::kBFloat16) FT_QA(__nv_bfloat16);
  else if (x.scalar_type() == at::kHalf) FT_QA(__half);
  else if (x.scalar_type() == at::kFloat) FT_QA(float);
  else TORCH_CHECK(false, "act8_quantize: bf16, fp16 or fp32 expected, got ", x.scalar_type());
#undef FT_QA
#undef FT_Q
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void act8_dequantize(const torch::Tensor& q, const torch::Tensor& scale, torch::Tensor& x, int64_t group) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1),
              "act8_dequantize: a 2-D CUDA output with unit inner stride is required");
  const int64_t rows = x.size(0);
  const int n = x.size(1);
  check_code(q, scale, rows, n, group);
  if (rows == 0 || n == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int lanes = group / kChunk, groups = scale.size(1);
  const unsigned grid = blocks_for(rows * ((n + kChunk - 1) / kChunk));
  const bool al = aligned16(x);
#define FT_D(T, AL)                                                                                        \
  dequantize_kernel<T, AL><<<grid, 256, 0, st>>>(q.data_ptr<int8_t>(), scale.data_ptr<float>(),            \
                                                 reinterpret_cast<T*>(x.data_ptr()), rows, n, x.stride(0), \
                                                 q.size(1), groups, lanes)
#define FT_DA(T) do { if (al) FT_D(T, true); else FT_D(T, false); } while (0)
  if (x.scalar_type() == at::kBFloat16) FT_DA(__nv_bfloat16);
  else if (x.scalar_type() == at::kHalf) FT_DA(__half);
  else if (x.scalar_type() == at::kFloat) FT_DA(float);
  else TORCH_CHECK(false, "act8_dequantize: bf16, fp16 or fp32 expected, got ", x.scalar_type());
#undef FT_DA
#undef FT_D
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Threads per row and chunks per thread for a row of H values.
#define FT_NORM8_SIZES(LAUNCH)          \
  if (H <= 512) LAUNCH(32, 1);          \
  else if (H <= 1024) LAUNCH(32, 2);    \
  else if (H <= 2048) LAUNCH(128, 1);   \
  else if (H <= 4096) LAUNCH(256, 1);   \
  else if (H <= 8192) LAUNCH(512, 1);   \
  else LAUNCH(512, 2)

void act8_rms_norm(const torch::Tensor& x, const torch::Tensor& w, torch::Tensor& y, torch::Tensor& rstd,
                   torch::Tensor& q, torch::Tensor& scale, int64_t group, double eps) {
  const int64_t rows = x.size(0);
  const int H = x.size(1);
  TORCH_CHECK(H % 8 == 0 && H >= 8 && H <= 16384, "act8_rms_norm: H must be a multiple of 8, at most 16384");
  check_rows(x, rows, H, "x");
  check_rows(y, rows, H, "y");
  check_code(q, scale, rows, H, group);
  TORCH_CHECK(w.is_cuda() && w.scalar_type() == at::kBFloat16 && w.numel() == H && w.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
              "act8_rms_norm: w must be a contiguous bf16 vector of H values");
  TORCH_CHECK(rstd.is_cuda() && rstd.scalar_type() == at::kFloat && rstd.numel() == rows && rstd.is_contiguous());
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int lanes = group / kChunk, groups = scale.size(1);
#define FT_L(NT, VPT)                                                                                       \
  rms_norm8_kernel<NT, VPT><<<(rows + (NT >= 128 ? 1 : 128 / NT) - 1) / (NT >= 128 ? 1 : 128 / NT),         \
                              NT >= 128 ? NT : 128, 0, st>>>(                                               \
      reinterpret_cast<const __nv_bfloat16*>(x.data_ptr()),                                                 \
      reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()), reinterpret_cast<__nv_bfloat16*>(y.data_ptr()), \
      rstd.data_ptr<float>(), q.data_ptr<int8_t>(), scale.data_ptr<float>(), rows, H, x.stride(0),          \
      y.stride(0), q.size(1), groups, lanes, static_cast<float>(eps))
  FT_NORM8_SIZES(FT_L);
#undef FT_L
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Rows that may write a share of dw: the size of the workspace that act8_rms_norm_bwd needs.
int64_t act8_norm_walkers(int64_t rows, int64_t H) {
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t most = H <= 1024 ? sms * 16 : H <= 2048 ? sms * 8 : H <= 4096 ? sms * 4 : sms * 2;
  const int64_t per = (rows + most - 1) / most;
  return rows == 0 ? 0 : (rows + per - 1) / per;
}

void act8_rms_norm_bwd(const torch::Tensor& dy, const torch::Tensor& q, const torch::Tensor& scale,
                       const torch::Tensor& w, const torch::Tensor& rstd, torch::Tensor& dx, torch::Tensor& y8,
                       torch::Tensor& dw, torch::Tensor& part, int64_t group) {
  const int64_t rows = dy.size(0);
  const int H = dy.size(1);
  TORCH_CHECK(H % 8 == 0 && H >= 8 && H <= 16384, "act8_rms_norm_bwd: H must be a multiple of 8, at most 16384");
  check_rows(dy, rows, H, "dy");
  check_rows(dx, rows, H, "dx");
  check_rows(y8, rows, H, "y8");
  check_code(q, scale, rows, H, group);
  TORCH_CHECK(w.is_cuda() && w.scalar_type() == at::kBFloat16 && w.numel() == H && w.is_contiguous() &&
                  reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0);
  TORCH_CHECK(rstd.is_cuda() && rstd.scalar_type() == at::kFloat && rstd.numel() == rows && rstd.is_contiguous());
  TORCH_CHECK(dw.is_cuda() && dw.scalar_type() == at::kFloat && dw.numel() == H && dw.is_contiguous());
  const int64_t walkers = act8_norm_walkers(rows, H);
  TORCH_CHECK(part.is_cuda() && part.scalar_type() == at::kFloat && part.is_contiguous() &&
                  part.numel() >= walkers * H && reinterpret_cast<uintptr_t>(part.data_ptr()) % 16 == 0,
              "act8_rms_norm_bwd: workspace too small");
  const c10::cuda::CUDAGuard guard(dy.device());
  auto st = at::cuda::getCurrentCUDAStream();
  if (rows > 0) {
    const int rpw = static_cast<int>((rows + walkers - 1) / walkers);
    const int lanes = group / kChunk, groups = scale.size(1);
#define FT_L(NT, VPT)                                                                                          \
  rms_norm8_bwd_kernel<NT, VPT><<<(walkers + (NT >= 128 ? 1 : 128 / NT) - 1) / (NT >= 128 ? 1 : 128 / NT),     \
                                  NT >= 128 ? NT : 128, 0, st>>>(                                              \
      reinterpret_cast<const __nv_bfloat16*>(dy.data_ptr()), q.data_ptr<int8_t>(), scale.data_ptr<float>(),    \
      reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()), rstd.data_ptr<float>(),                            \
      reinterpret_cast<__nv_bfloat16*>(dx.data_ptr()), reinterpret_cast<__nv_bfloat16*>(y8.data_ptr()),        \
      part.data_ptr<float>(), rows, H, dy.stride(0), dx.stride(0), y8.stride(0), q.size(1), groups, lanes, rpw)
    FT_NORM8_SIZES(FT_L);
#undef FT_L
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  dw_sum_kernel<<<(H + 31) / 32, 256, 0, st>>>(part.data_ptr<float>(), dw.data_ptr<float>(),
                                               static_cast<int>(walkers), H);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void act8_swiglu(const torch::Tensor& gu, torch::Tensor& h, torch::Tensor& q, torch::Tensor& scale, int64_t group) {
  const int64_t rows = h.size(0);
  const int F = h.size(1);
  TORCH_CHECK(F % 8 == 0 && F >= 8, "act8_swiglu: F must be a multiple of 8");
  check_rows(gu, rows, 2 * (int64_t)F, "gu");
  check_rows(h, rows, F, "h");
  check_code(q, scale, 2 * rows, F, group);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(gu.device());
  const int lanes = group / kChunk, groups = scale.size(1);
  swiglu8_kernel<<<blocks_for(rows * groups * lanes), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      reinterpret_cast<const __nv_bfloat16*>(gu.data_ptr()), reinterpret_cast<__nv_bfloat16*>(h.data_ptr()),
      q.data_ptr<int8_t>(), scale.data_ptr<float>(), rows, F, gu.stride(0), h.stride(0), q.size(1), groups, lanes);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void act8_swiglu_bwd(const torch::Tensor& dh, const torch::Tensor& q, const torch::Tensor& scale,
                     torch::Tensor& dgu, torch::Tensor& h8, int64_t group) {
  const int64_t rows = dh.size(0);
  const int F = dh.size(1);
  TORCH_CHECK(F % 8 == 0 && F >= 8, "act8_swiglu_bwd: F must be a multiple of 8");
  check_rows(dh, rows, F, "dh");
  check_rows(dgu, rows, 2 * (int64_t)F, "dgu");
  check_rows(h8, rows, F, "h8");
  check_code(q, scale, 2 * rows, F, group);
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(dh.device());
  const int lanes = group / kChunk, groups = scale.size(1);
  swiglu8_bwd_kernel<<<blocks_for(rows * ((F + kChunk - 1) / kChunk)), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      reinterpret_cast<const __nv_bfloat16*>(dh.data_ptr()), q.data_ptr<int8_t>(), scale.data_ptr<float>(),
      reinterpret_cast<__nv_bfloat16*>(dgu.data_ptr()), reinterpret_cast<__nv_bfloat16*>(h8.data_ptr()), rows, F,
      dh.stride(0), dgu.stride(0), h8.stride(0), q.size(1), groups, lanes);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace ft

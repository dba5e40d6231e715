// Rotary positions over all or part of each head, in half or interleaved layout (sm_100a).
//
// With r = rot / 2 pairs per head and position p, pair i of every head is turned by the angle
// whose cosine and sine are cos[p][i], sin[p][i] (fp32 tables, so scaled frequencies and
// positions of a long context keep their precision):
//   a' = a c - b s,   b' = b c + a s        (inverse, the backward pass: s -> -s)
// half layout: (a, b) = (x[i], x[r + i]); interleaved: (a, b) = (x[2 i], x[2 i + 1]).
// Values at rot .. d are passed through.
//
// The work is one read and one write of q and k, so HBM bandwidth bounds it.  A thread turns
// the same P pairs (16 bytes of each half where alignment allows) of up to kHeads heads of one
// token: cos and sin are read once for all of them, and the loads of all heads are in flight
// before the first is used.  Threads of a warp take neighbouring pairs, then neighbouring heads.
// Input and output may be the same memory: a thread reads its pairs before it writes them.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ft {
namespace {

constexpr int kHeads = 4;           // heads per thread
constexpr int kErrPosition = 301;   // a position outside the tables

struct RotaryParams {
  const void* in[2];   // q, k
  void* out[2];
  int64_t is[2][3], os[2][3];  // strides of batch, token, head
  const float* cos;
  const float* sin;
  const void* pos;     // int32 or int64, or null: the token index
  int64_t pb, ps;      // its strides
  int* err;
  int64_t tokens;      // batch * sequence
  int seq, nq, heads, max_pos;
  int rot, d;
  int slots, turning;  // P-pair slots per head; the first `turning` of them rotate
  int groups;          // head groups of kHeads
  int pos64, inverse;
};

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T as_type(float v);
template <> __device__ __forceinline__ __nv_bfloat16 as_type(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half as_type(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float as_type(float v) { return v; }

template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack { T v[N]; };

// A slot's 2P values as two packs: the two halves of P pairs (half layout), or 2P neighbours.
template <typename T, int P, bool IL>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  using V = Pack<T, P>;
  const int per_token = p.groups * p.slots;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= p.tokens * per_token) return;
  int64_t token;
  int rest;
  if (idx <= 0x7fffffff) {  // 32-bit division unless the launch is that large
    token = static_cast<uint32_t>(idx) / static_cast<uint32_t>(per_token);
  } else {
    token = idx / per_token;
  }
  rest = static_cast<int>(idx - token * per_token);
  const int g = rest / p.slots;
  const int slot = rest - g * p.slots;
  const int b = static_cast<int>(token / p.seq);
  const int t = static_cast<int>(token - (int64_t)b * p.seq);
  const bool turns = slot < p.turning;
  const int r = p.rot / 2;
  // element offsets of the two packs inside a head
  const int o0 = (turns && !IL) ? slot * P : slot * 2 * P;
  const int o1 = (turns && !IL) ? o0 + r : o0 + P;
  V x[kHeads][2];
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const int h = g + j * p.groups;
    if (h < p.heads) {
      const int w = h >= p.nq;
      const T* base = reinterpret_cast<const T*>(p.in[w]) + b * p.is[w][0] + t * p.is[w][1] +
                      (h - (w ? p.nq : 0)) * p.is[w][2];
      x[j][0] = *reinterpret_cast<const V*>(base + o0);
      if (o1 < p.d) x[j][1] = *reinterpret_cast<const V*>(base + o1);
    }
  }
  float c[P], s[P];
  if (turns) {
    int64_t at = t;
    if (p.pos) {
      const int64_t k = b * p.pb + t * p.ps;
      at = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[k] : reinterpret_cast<const int*>(p.pos)[k];
    }
    if (at < 0 || at >= p.max_pos) {
      if (slot == 0 && g == 0) atomicCAS(p.err, 0, kErrPosition);
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    } else {
      using F = Pack<float, (P < 4 ? P : 4)>;
      const float* cp = p.cos + at * r + slot * P;
      const float* sp = p.sin + at * r + slot * P;
#pragma unroll
      for (int i = 0; i < P; i += (P < 4 ? P : 4)) {
        const F cv = *reinterpret_cast<const F*>(cp + i), sv = *reinterpret_cast<const F*>(sp + i);
#pragma unroll
        for (int j = 0; j < (P < 4 ? P : 4); ++j) {
          c[i + j] = cv.v[j];
          s[i + j] = p.inverse ? -sv.v[j] : sv.v[j];
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    const int h = g + j * p.groups;
    if (h < p.heads) {
      const int w = h >= p.nq;
      T* base = reinterpret_cast<T*>(p.out[w]) + b * p.os[w][0] + t * p.os[w][1] +
                (h - (w ? p.nq : 0)) * p.os[w][2];
      V y0 = x[j][0], y1 = x[j][1];
      if (turns) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          // flat position of a and b of pair i in the 2P values of the slot
          const int ia = IL ? 2 * i : i, ib = IL ? 2 * i + 1 : P + i;
          const float a = as_float<T>(ia < P ? x[j][0].v[ia % P] : x[j][1].v[ia % P]);
          const float bb = as_float<T>(ib < P ? x[j][0].v[ib % P] : x[j][1].v[ib % P]);
          const T na = as_type<T>(a * c[i] - bb * s[i]), nb = as_type<T>(bb * c[i] + a * s[i]);
          if (ia < P) y0.v[ia % P] = na; else y1.v[ia % P] = na;
          if (ib < P) y0.v[ib % P] = nb; else y1.v[ib % P] = nb;
        }
      }
      *reinterpret_cast<V*>(base + o0) = y0;
      if (o1 < p.d) *reinterpret_cast<V*>(base + o1) = y1;
    }
  }
}

}  // namespace

// q [B, S, nq, d] and k [B, S, nkv, d] (any strides with a unit inner one) -> the same shapes.
// cos, sin: contiguous fp32 [max_pos, rot / 2]; pos: int32 or int64 [B or 1, S], or none.
// A position outside the tables gives NaN and records an error code in err.
void rotary_qk(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& cos_t,
               const torch::Tensor& sin_t, const c10::optional<torch::Tensor>& pos, torch::Tensor& oq,
               torch::Tensor& ok, bool interleaved, bool inverse, torch::Tensor& err) {
  const torch::Tensor* in[2] = {&q, &k};
  torch::Tensor* out[2] = {&oq, &ok};
  const auto type = q.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
              "rotary_qk: bf16, fp16 or fp32 expected, got ", type);
  const int64_t B = q.size(0), S = q.size(1), d = q.size(3);
  RotaryParams p;
  const int64_t rot = 2 * cos_t.size(1);
  TORCH_CHECK(cos_t.is_cuda() && sin_t.is_cuda() && cos_t.scalar_type() == at::kFloat &&
                  sin_t.scalar_type() == at::kFloat && cos_t.dim() == 2 && cos_t.sizes() == sin_t.sizes() &&
                  cos_t.is_contiguous() && sin_t.is_contiguous(),
              "rotary_qk: cos and sin must be contiguous fp32 CUDA tables [positions, rot / 2]");
  TORCH_CHECK(rot <= d, "rotary_qk: ", rot, " rotated values do not fit a head of ", d);
  const int64_t es = q.element_size();
  const int widest = static_cast<int>(16 / es);
  // P: the widest pack that every address of the launch is aligned to, and that neither the
  // rotated part nor the rest of a head splits
  int P = widest;
  auto fits = [&](int64_t elems, int pack) { return elems % pack == 0; };
  for (int w = 0; w < 2; ++w) {
    const torch::Tensor &a = *in[w], &o = *out[w];
    TORCH_CHECK(a.is_cuda() && o.is_cuda() && a.dim() == 4 && o.dim() == 4 && a.scalar_type() == type &&
                    o.scalar_type() == type && a.sizes() == o.sizes() && a.size(0) == B && a.size(1) == S &&
                    a.size(3) == d && (d == 1 || (a.stride(3) == 1 && o.stride(3) == 1)),
                "rotary_qk: q and k must be CUDA tensors [B, S, heads, d] of one type with unit inner stride");
    p.in[w] = a.data_ptr();
    p.out[w] = o.data_ptr();
    for (int i = 0; i < 3; ++i) {
      p.is[w][i] = a.stride(i);
      p.os[w][i] = o.stride(i);
      while (P > 1 && !((a.size(i) == 1 || fits(a.stride(i), P)) && (o.size(i) == 1 || fits(o.stride(i), P)))) P /= 2;
    }
    while (P > 1 && (reinterpret_cast<uintptr_t>(a.data_ptr()) % (P * es) ||
                     reinterpret_cast<uintptr_t>(o.data_ptr()) % (P * es)))
      P /= 2;
  }
  while (P > 1 && (!fits(rot / 2, P) || !fits(d - rot, 2 * P) ||
                   reinterpret_cast<uintptr_t>(cos_t.data_ptr()) % (4 * std::min(P, 4)) ||
                   reinterpret_cast<uintptr_t>(sin_t.data_ptr()) % (4 * std::min(P, 4))))
    P /= 2;
  const int64_t nq = q.size(2), nkv = k.size(2), heads = nq + nkv;
  if (B * S == 0 || heads == 0 || d == 0) return;
  TORCH_CHECK(B * S < (int64_t(1) << 31) && heads < (1 << 20) && d < (1 << 20) && cos_t.size(0) < (int64_t(1) << 31),
              "rotary_qk: sizes out of range");
  p.pos = nullptr;
  p.pb = p.ps = 0;
  p.pos64 = 0;
  if (pos.has_value()) {
    TORCH_CHECK(pos->is_cuda() && (pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt) &&
                    pos->dim() == 2 && pos->size(1) == S && (pos->size(0) == B || pos->size(0) == 1),
                "rotary_qk: pos must be an int32 or int64 CUDA tensor [B or 1, S]");
    p.pos = pos->data_ptr();
    p.pb = pos->size(0) == 1 ? 0 : pos->stride(0);
    p.ps = pos->stride(1);
    p.pos64 = pos->scalar_type() == at::kLong;
  }
  for (int w = 0; w < 2; ++w)
    TORCH_CHECK(p.in[w] != p.out[w] || in[w]->numel() == 0 || in[w]->strides() == out[w]->strides(),
                "rotary_qk: an output in the memory of its input needs the same strides");
  const bool in_place = p.in[0] == p.out[0] && p.in[1] == p.out[1];
  p.cos = cos_t.data_ptr<float>();
  p.sin = sin_t.data_ptr<float>();
  p.err = err.data_ptr<int>();
  p.tokens = B * S;
  p.seq = S;
  p.nq = nq;
  p.heads = heads;
  p.max_pos = cos_t.size(0);
  p.rot = rot;
  p.d = d;
  p.turning = rot / 2 / P;
  // what is passed through needs no copy where input and output are the same memory
  p.slots = in_place ? p.turning : p.turning + static_cast<int>((d - rot + 2 * P - 1) / (2 * P));
  p.groups = (heads + kHeads - 1) / kHeads;
  p.inverse = inverse;
  if (p.slots == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int64_t blocks = (p.tokens * p.groups * p.slots + 255) / 256;
  TORCH_CHECK(blocks < (int64_t(1) << 31), "rotary_qk: tensor too large for one launch");
#define FT_R(T, PP)                                                                              \
  do {                                                                                           \
    if (interleaved) rotary_kernel<T, PP, true><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p); \
    else rotary_kernel<T, PP, false><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);          \
  } while (0)
#define FT_R16(T)                  \
  do {                             \
    if (P == 8) FT_R(T, 8);        \
    else if (P == 4) FT_R(T, 4);   \
    else if (P == 2) FT_R(T, 2);   \
    else FT_R(T, 1);               \
  } while (0)
  if (type == at::kBFloat16) FT_R16(__nv_bfloat16);
  else if (type == at::kHalf) FT_R16(__half);
  else if (P == 4) FT_R(float, 4);
  else if (P == 2) FT_R(float, 2);
  else FT_R(float, 1);
#undef FT_R16
#undef FT_R
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace ft

// Rotary positions over all or part of each head, in half or interleaved layout (sm_100a).
//
// With r = rot / 2 pairs per head and position p, pair i of every head is turned by the angle
// whose cosine and sine are cos[p][i], sin[p][i] (fp32 tables, so scaled frequencies and
// positions of a long context keep their precision):
//   a' = a c - b s,   b' = b c + a s        (inverse, the backward pass: s -> -s)
// half layout: (a, b) = (x[i], x[r + i]); interleaved: (a, b) = (x[2 i], x[2 i + 1]).
// Values at rot .. d are passed through.
//
// The work is one read and one write of q and k, so HBM bandwidth bounds it, provided that a
// token's positions, table rows and addresses are not worked out for every head anew: a thread
// turns the same P pairs (16 bytes of each half where alignment allows) of several heads of one
// token, one after the other (with two or four heads' loads in flight it needs so many registers
// that fewer warps hide less: 69.9 and 87.1 us instead of 63.2 for 2 x 8192 tokens of 40 heads
// of 128, bf16).  Threads of a warp take neighbouring pairs, then neighbouring heads.  The input
// is read past L2's reuse (61.3 us: 5.6 TB/s, 0.86 of the copy rate).
// Input and output may be the same memory: a thread reads its pairs before it writes them.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdlib>
#include <type_traits>
#include <utility>

#include "checks.h"
#include "common.cuh"

namespace ft {
namespace {

constexpr int kErrPosition = 301;   // a position outside the tables

struct RotaryParams {
  const void* in[2];   // q, k
  void* out[2];
  int64_t is[2][2], os[2][2];  // strides of batch and token
  int ih[2], oh[2];            // of a head
  FastDiv by_token, by_slots, by_seq;
  const float* cos;
  const float* sin;
  const void* pos;     // int32 or int64, or null: the token index
  int64_t pb, ps;      // its strides
  int* err;
  int64_t tokens;      // batch * sequence
  int seq, nq, heads, max_pos;
  int rot, d;
  int slots, turning;  // P-pair slots per head; the first `turning` of them rotate
  int groups;          // a thread takes heads g, g + groups, ...
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

// A pack read once: first out of L2.
template <typename V>
__device__ __forceinline__ void streamed(V& v, const V* p) {
  if constexpr (sizeof(V) == 16) *reinterpret_cast<uint4*>(&v) = __ldcs(reinterpret_cast<const uint4*>(p));
  else if constexpr (sizeof(V) == 8) *reinterpret_cast<uint2*>(&v) = __ldcs(reinterpret_cast<const uint2*>(p));
  else if constexpr (sizeof(V) == 4) *reinterpret_cast<unsigned*>(&v) = __ldcs(reinterpret_cast<const unsigned*>(p));
  else v = *p;
}

// N floats to N values of T, two at a time where T has a conversion of pairs.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> rounded(const float* f) {
  Pack<T, N> y;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if constexpr (std::is_same_v<T, __half>)
        *reinterpret_cast<__half2*>(&y.v[i]) = __floats2half2_rn(f[i], f[i + 1]);
      else
        *reinterpret_cast<__nv_bfloat162*>(&y.v[i]) = __floats2bfloat162_rn(f[i], f[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) y.v[i] = as_type<T>(f[i]);
  }
  return y;
}

// A slot's 2P values as two packs: the two halves of P pairs (half layout), or 2P neighbours.
template <typename T, int P, bool IL>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  using V = Pack<T, P>;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const int token = p.by_token.div(idx);
  if (token >= p.tokens) return;
  const int rest = idx - token * p.by_token.d;
  const int g = p.by_slots.div(rest);
  const int slot = rest - g * p.slots;
  const int b = p.by_seq.div(token);
  const int t = token - b * p.seq;
  const bool turns = slot < p.turning;
  int64_t at = t;
  if (p.pos && turns) {
    const int64_t k = b * p.pb + t * p.ps;
    at = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[k] : reinterpret_cast<const int*>(p.pos)[k];
  }
  const int r = p.rot / 2;
  // element offsets of the two packs inside a head
  const int o0 = (turns && !IL) ? slot * P : slot * 2 * P;
  const int o1 = (turns && !IL) ? o0 + r : o0 + P;
  const bool two = o1 < p.d;
  // head h of this token: base + h * stride, with the k heads counted on from the q heads
  const T* iq = reinterpret_cast<const T*>(p.in[0]) + b * p.is[0][0] + t * p.is[0][1];
  const T* ik = reinterpret_cast<const T*>(p.in[1]) + b * p.is[1][0] + t * p.is[1][1] - (int64_t)p.nq * p.ih[1];
  T* oq = reinterpret_cast<T*>(p.out[0]) + b * p.os[0][0] + t * p.os[0][1];
  T* ok = reinterpret_cast<T*>(p.out[1]) + b * p.os[1][0] + t * p.os[1][1] - (int64_t)p.nq * p.oh[1];

  V x[2];
  auto load = [&](int h) {
    if (h < p.heads) {
      const T* base = h < p.nq ? iq + (int64_t)h * p.ih[0] : ik + (int64_t)h * p.ih[1];
      streamed(x[0], reinterpret_cast<const V*>(base + o0));
      if (two) streamed(x[1], reinterpret_cast<const V*>(base + o1));
    }
  };
  load(g);
  float c[P], s[P];
  if (turns) {
    if (at < 0 || at >= p.max_pos) {
      if (slot == 0 && g == 0) atomicCAS(p.err, 0, kErrPosition);
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    } else {
      constexpr int F = P < 4 ? P : 4;
      const float* cp = p.cos + at * r + slot * P;
      const float* sp = p.sin + at * r + slot * P;
#pragma unroll
      for (int i = 0; i < P; i += F) {
        const Pack<float, F> cv = *reinterpret_cast<const Pack<float, F>*>(cp + i);
        const Pack<float, F> sv = *reinterpret_cast<const Pack<float, F>*>(sp + i);
#pragma unroll
        for (int j = 0; j < F; ++j) {
          c[i + j] = cv.v[j];
          s[i + j] = p.inverse ? -sv.v[j] : sv.v[j];
        }
      }
    }
  }
  for (int h = g; h < p.heads; h += p.groups) {
    T* base = h < p.nq ? oq + (int64_t)h * p.oh[0] : ok + (int64_t)h * p.oh[1];
    if (turns) {
      float f[2 * P];  // in the order of memory: pair i is (i, P + i) or (2 i, 2 i + 1)
#pragma unroll
      for (int i = 0; i < P; ++i) {
        f[i] = as_float<T>(x[0].v[i]);
        f[P + i] = as_float<T>(x[1].v[i]);
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float &u = f[IL ? 2 * i : i], &v = f[IL ? 2 * i + 1 : P + i];
        const float a = u, bb = v;
        u = a * c[i] - bb * s[i];
        v = bb * c[i] + a * s[i];
      }
      x[0] = rounded<T, P>(f);
      x[1] = rounded<T, P>(f + P);
    }
    *reinterpret_cast<V*>(base + o0) = x[0];
    if (two) *reinterpret_cast<V*>(base + o1) = x[1];
    load(h + p.groups);
  }
}

// Elements from the first to the last one of x, or -1 where, going up the strides, a step does not
// clear what lies below it: then elements share memory.
int64_t reach_of(const torch::Tensor& x) {
  std::pair<int64_t, int64_t> dims[4];
  int n = 0;
  for (int i = 0; i < 4; ++i)
    if (x.size(i) > 1) dims[n++] = {x.stride(i), x.size(i)};
  std::sort(dims, dims + n);
  int64_t reach = 0;
  for (int i = 0; i < n; ++i) {
    if (dims[i].first <= reach) return -1;
    reach += dims[i].first * (dims[i].second - 1);
  }
  return reach;
}

struct Steps { int64_t stride, up, down; };  // and the most steps along it in q and in k

// Whether steps of q less steps of k can come to `rest`.
bool meet(const Steps* dims, int n, int64_t rest) {
  if (n == 0) return rest == 0;
  int64_t below = 0;
  for (int i = 1; i < n; ++i) below += dims[i].stride * std::max(dims[i].up, dims[i].down);
  // below spans a few strides at most: q and k do not overlap themselves
  const int64_t st = dims[0].stride;
  for (int64_t c = std::max(-dims[0].down, (rest - below) / st - 1); c <= dims[0].up && c * st - rest <= below; ++c)
    if (std::abs(c * st - rest) <= below && meet(dims + 1, n - 1, rest - c * st)) return true;
  return false;
}

// Whether q or k overlaps itself, or q and k, laid out alike, have an element in common.
bool written_twice(const torch::Tensor& q, const torch::Tensor& k) {
  const int64_t rq = q.numel() ? reach_of(q) : 0, rk = k.numel() ? reach_of(k) : 0;
  if (rq < 0 || rk < 0) return true;
  if (q.numel() == 0 || k.numel() == 0) return false;
  const int64_t bytes = reinterpret_cast<intptr_t>(k.data_ptr()) - reinterpret_cast<intptr_t>(q.data_ptr());
  const int64_t es = q.element_size(), apart = bytes / es;
  if (apart > rq || apart < -rk || bytes % es) return false;
  Steps dims[4];
  int n = 0;
  for (int i = 0; i < 4; ++i) {
    if (q.size(i) > 1 && k.size(i) > 1 && q.stride(i) != k.stride(i)) return false;  // not laid out alike
    if (q.size(i) > 1 || k.size(i) > 1)
      dims[n++] = {q.size(i) > 1 ? q.stride(i) : k.stride(i), q.size(i) - 1, k.size(i) - 1};
  }
  std::sort(dims, dims + n, [](const Steps& a, const Steps& b) { return a.stride > b.stride; });
  return meet(dims, n, apart);
}

}  // namespace

// q [B, S, nq, d] and k [B, S, nkv, d] (any strides with a unit inner one) -> turned copies, or
// q and k themselves turned in place.  cos, sin: contiguous fp32 [max_pos, rot / 2]; pos: int32
// or int64 [B or 1, S], or none.  A position outside the tables gives NaN and an error code in err.
std::tuple<torch::Tensor, torch::Tensor> rotary_qk(const torch::Tensor& q_, const torch::Tensor& k_,
                                                   const torch::Tensor& cos_t, const torch::Tensor& sin_t,
                                                   const c10::optional<torch::Tensor>& pos_, bool interleaved,
                                                   bool inverse, bool inplace, torch::Tensor& err) {
  torch::Tensor q = q_, k = k_;
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "rotary_qk: q and k must be [batch, tokens, heads, d], got ",
                    q.sizes(), " and ", k.sizes());
  const int64_t B = q.size(0), S = q.size(1), d = q.size(3);
  const auto type = q.scalar_type();
  TORCH_CHECK_VALUE(k.size(0) == B && k.size(1) == S && k.size(3) == d && k.scalar_type() == type &&
                        k.device() == q.device(),
                    "rotary_qk: q and k must agree in batch, tokens, d, dtype and device");
  check_one_device("rotary_qk", q, cos_t, sin_t, err);
  if (pos_.has_value()) check_one_device("rotary_qk", q, *pos_);
  TORCH_CHECK(q.is_cuda() && (type == at::kBFloat16 || type == at::kHalf || type == at::kFloat),
              "rotary_qk: bf16, fp16 or fp32 CUDA tensors expected, got ", type);
  TORCH_CHECK_VALUE(cos_t.dim() == 2 && cos_t.sizes() == sin_t.sizes() && cos_t.scalar_type() == at::kFloat &&
                        sin_t.scalar_type() == at::kFloat,
                    "rotary_qk: cos and sin must be fp32 tables [positions, rot/2] of one shape");
  TORCH_CHECK(cos_t.is_cuda() && sin_t.is_cuda() && cos_t.is_contiguous() && sin_t.is_contiguous(),
              "rotary_qk: cos and sin must be contiguous CUDA tables");
  const int64_t rot = 2 * cos_t.size(1);
  TORCH_CHECK_VALUE(rot <= d, "rotary_qk: ", rot, " rotated values do not fit a head of ", d);
  const c10::cuda::CUDAGuard guard(q.device());
  if (d > 1 && (q.stride(3) != 1 || k.stride(3) != 1)) {
    TORCH_CHECK_VALUE(!inplace, "rotary_qk: in place needs a unit inner stride");
    q = q.contiguous();
    k = k.contiguous();
  }
  // threads would race on an element with two names
  TORCH_CHECK(!inplace || !written_twice(q, k), "rotary_qk: in place on q and k that name an element more than once");
  RotaryParams p;
  p.pos = nullptr;
  p.pb = p.ps = 0;
  p.pos64 = 0;
  if (pos_.has_value()) {
    const torch::Tensor& pos = *pos_;
    TORCH_CHECK_TYPE(pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt,
                     "rotary_qk: positions must be int32 or int64, got ", pos.scalar_type());
    TORCH_CHECK(pos.is_cuda(), "rotary_qk: positions must be a CUDA tensor");
    const int64_t pd = pos.dim();
    TORCH_CHECK_VALUE((pd == 1 || (pd == 2 && (pos.size(0) == B || pos.size(0) == 1))) && pos.size(pd - 1) == S,
                      "rotary_qk: positions of shape ", pos.sizes(), " do not match [", B, " or 1, ", S, "]");
    p.pos = pos.data_ptr();
    p.pb = pd == 1 || pos.size(0) == 1 ? 0 : pos.stride(0);
    p.ps = pos.stride(pd - 1);
    p.pos64 = pos.scalar_type() == at::kLong;
  } else {
    TORCH_CHECK_VALUE(S <= cos_t.size(0), "rotary_qk: ", S, " tokens, tables of ", cos_t.size(0), " positions");
  }
  torch::Tensor oq = inplace ? q_ : torch::empty(q.sizes(), q.options());
  torch::Tensor ok = inplace ? k_ : torch::empty(k.sizes(), k.options());

  const int64_t es = q.element_size();
  // P: the widest pack (16 bytes at most) that every address of the launch is aligned to, and
  // that neither the rotated part nor the rest of a head splits
  int P = static_cast<int>(16 / es);
  auto narrow_to = [&](int64_t elems, int packs) {
    while (P > 1 && elems % (packs * P)) P /= 2;
  };
  const torch::Tensor* in[2] = {&q, &k};
  const torch::Tensor* out[2] = {&oq, &ok};
  for (int w = 0; w < 2; ++w) {
    p.in[w] = in[w]->data_ptr();
    p.out[w] = out[w]->data_ptr();
    for (int i = 0; i < 3; ++i) {
      const int64_t a = in[w]->stride(i), o = out[w]->stride(i);
      if (i < 2) {
        p.is[w][i] = a;
        p.os[w][i] = o;
      }
      if (in[w]->size(i) > 1) {
        narrow_to(a, 1);
        narrow_to(o, 1);
      }
    }
    const bool one = in[w]->size(2) <= 1;  // the stride of one head does not matter
    TORCH_CHECK_VALUE(one || (std::abs(in[w]->stride(2)) < (int64_t(1) << 31) &&
                              std::abs(out[w]->stride(2)) < (int64_t(1) << 31)),
                      "rotary_qk: heads too far apart");
    p.ih[w] = one ? 0 : static_cast<int>(in[w]->stride(2));
    p.oh[w] = one ? 0 : static_cast<int>(out[w]->stride(2));
    narrow_to(reinterpret_cast<intptr_t>(p.in[w]) / es, 1);
    narrow_to(reinterpret_cast<intptr_t>(p.out[w]) / es, 1);
  }
  narrow_to(rot / 2, 1);
  narrow_to(d - rot, 2);
  while (P > 1 && (reinterpret_cast<uintptr_t>(cos_t.data_ptr()) % (4 * std::min(P, 4)) ||
                   reinterpret_cast<uintptr_t>(sin_t.data_ptr()) % (4 * std::min(P, 4))))
    P /= 2;
  const int64_t nq = q.size(2), nkv = k.size(2), heads = nq + nkv;
  if (B * S == 0 || heads == 0 || d == 0) return {oq, ok};
  TORCH_CHECK_VALUE(B * S < (int64_t(1) << 31) && heads < (1 << 20) && d < (1 << 20) &&
                        cos_t.size(0) < (int64_t(1) << 31),
                    "rotary_qk: sizes out of range");
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
  p.slots = inplace ? p.turning : p.turning + static_cast<int>((d - rot + 2 * P - 1) / (2 * P));
  p.inverse = inverse;
  if (p.slots == 0) return {oq, ok};
  // heads per thread: as many as leave two rounds of threads for the GPU
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t most = std::min<int64_t>(16, std::max<int64_t>(1, p.tokens * heads * p.slots / (sms * 3072)));
  p.groups = static_cast<int>((heads + most - 1) / most);
  p.by_slots.set(p.slots);
  p.by_token.set(p.groups * p.slots);
  p.by_seq.set(p.seq);
  auto st = at::cuda::getCurrentCUDAStream();
  const int64_t threads = p.tokens * p.groups * p.slots;
  TORCH_CHECK_VALUE(threads < (int64_t(1) << 31) - 256, "rotary_qk: tensor too large for one launch");
  const int64_t blocks = (threads + 255) / 256;
#define FT_R(T, PP)                                                                    \
  do {                                                                                 \
    auto kern = interleaved ? rotary_kernel<T, PP, true> : rotary_kernel<T, PP, false>; \
    kern<<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);                            \
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
  return {oq, ok};
}

}  // namespace ft

// Entry points of the attention over a mask of intervals (masked_attn.h): checks of the operands and launches.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>

#include "masked_attn.h"
#include "tmap.h"

namespace ft {
namespace ma {
namespace {

// A kernel reads all its operands by address, so they have to lie on the device that it runs on.
template <class... Tensors>
void one_device(const at::Tensor& first, const Tensors&... rest) {
  const at::Tensor* all[] = {&rest...};
  for (const at::Tensor* t : all)
    TORCH_CHECK(t->device() == first.device(), "masked_attention: all operands must be on one device, got ", first.device(),
                " and ", t->device());
}

// tiles of 128 rows that stay, of STEP rows that go past
CUtensorMap heads_map(const at::Tensor& x, int rows) {
  auto stride = [&](int i) { return x.size(i) == 1 ? x.size(3) : x.stride(i); };  // of one element: never taken
  return make_tmap_heads(x.data_ptr(), x.size(3), x.size(2), x.size(1), x.size(0), stride(2), stride(1), stride(0), rows);
}

// x itself where TMA and 16-byte accesses take it, else a contiguous copy
at::Tensor usable(const at::Tensor& x) {
  bool fine = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && (x.stride(3) == 1 || x.size(3) == 1);
  for (int i = 0; i < 3; ++i) fine = fine && (x.size(i) == 1 || (x.stride(i) % 8 == 0 && x.stride(i) > 0));
  return fine ? x : x.clone(at::MemoryFormat::Contiguous);
}

struct Shape {
  int64_t B, S, nq, nkv, d;
};

Shape check(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& rows,
            const at::Tensor& tiles, const at::Tensor& order, const c10::optional<at::Tensor>& slopes,
            const at::Tensor& err) {
  TORCH_CHECK(q.is_cuda(), "masked_attention: q must be a CUDA tensor");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "masked_attention: q, k, v must be [batch, tokens, heads, d]");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16,
              "masked_attention: q, k, v must be bfloat16 on CUDA");
  const Shape n{q.size(0), q.size(1), q.size(2), k.size(2), q.size(3)};
  TORCH_CHECK(k.size(0) == n.B && k.size(1) == n.S && k.size(3) == n.d && v.sizes() == k.sizes(),
              "masked_attention: q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not match");
  TORCH_CHECK(n.d % 8 == 0 && n.d >= 8 && n.d <= 128, "masked_attention: the head size must be a multiple of 8 up to 128, got ",
              n.d);
  TORCH_CHECK(n.nkv > 0 && n.nq % n.nkv == 0, "masked_attention: ", n.nq, " query heads do not share ", n.nkv, " key heads evenly");
  one_device(q, k, v, rows, tiles, order, err);
  const int64_t nt = (n.S + TILE - 1) / TILE;
  TORCH_CHECK(rows.scalar_type() == at::kInt && rows.is_contiguous() && rows.dim() == 3 && rows.size(1) == nt * TILE &&
                  rows.size(2) == 2 && tiles.scalar_type() == at::kInt && tiles.is_contiguous() && tiles.dim() == 3 &&
                  tiles.size(1) == nt && tiles.size(2) == 4 && tiles.size(0) == rows.size(0) &&
                  order.scalar_type() == at::kInt && order.is_contiguous() && order.dim() == 2 &&
                  order.size(0) == rows.size(0) && order.size(1) == nt,
              "masked_attention: the mask was not made for ", n.S, " tokens");
  TORCH_CHECK(rows.size(0) == 1 || rows.size(0) == n.B, "masked_attention: a mask of ", rows.size(0),
              " sequences for a batch of ", n.B);
  if (slopes.has_value()) {
    one_device(q, *slopes);
    TORCH_CHECK(slopes->scalar_type() == at::kFloat && slopes->is_contiguous() && slopes->dim() == 1 &&
                    slopes->size(0) == n.nq,
                "masked_attention: slopes must be one fp32 number per query head");
  }
  TORCH_CHECK(n.B <= 65535 && n.nq <= 8192 && n.B * n.nq < (int64_t(1) << 31), "masked_attention: at most 65535 sequences of ",
              "8192 heads, got ", n.B, " of ", n.nq);
  return n;
}

void fill(Common& p, const Shape& n, const at::Tensor& rows, const at::Tensor& tiles,
          const at::Tensor& order, double scale, double softcap,
          const c10::optional<at::Tensor>& slopes, float* neg_lse2, at::Tensor& err) {
  p.B = n.B; p.S = n.S; p.nq = n.nq; p.nkv = n.nkv; p.d = n.d;
  p.ntiles = (n.S + TILE - 1) / TILE;
  p.padded = p.ntiles * TILE;
  p.group = n.nq / n.nkv;
  p.ksteps = (n.d + 15) / 16;
  p.rows = reinterpret_cast<const int2*>(rows.data_ptr<int>());
  p.tiles = reinterpret_cast<const int4*>(tiles.data_ptr<int>());
  p.rows_stride = rows.size(0) == 1 ? 0 : p.padded;
  p.tiles_stride = rows.size(0) == 1 ? 0 : p.ntiles;
  p.order = order.data_ptr<int>();
  p.slopes = slopes.has_value() ? slopes->data_ptr<float>() : nullptr;
  p.scale = static_cast<float>(scale);
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  p.cap_in = softcap > 0 ? static_cast<float>(2 * scale * 1.4426950408889634 / softcap) : 0.f;
  p.cap_out = static_cast<float>(softcap * 1.4426950408889634);
  // tanh(x) / x at the Chebyshev nodes of x^2 in [0, 0.49] as a polynomial in x^2, with x = scale s / c put in
  const double poly[5] = {0.999999702, -0.333301812, 0.132807881, -0.0508257188, 0.0137630384};
  const double r = softcap > 0 ? scale / softcap : 0.0;
  p.cap_small = softcap > 0 ? static_cast<float>(0.7 / r) : 0.f;
  for (int i = 0; i < 5; ++i) p.cap_poly[i] = static_cast<float>(poly[i] * std::pow(r, 2 * i + 1));
  if (!std::isfinite(p.cap_poly[4])) p.cap_small = -1.f;  // a cap so small that only the other form serves
  p.neg_lse2 = neg_lse2;
  p.err = err.data_ptr<int>();
}

Out out_of(const at::Tensor& x) {
  return Out{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}

void check_out(const at::Tensor& x, const at::Tensor& like, const char* name) {
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.sizes() == like.sizes() && x.device() == like.device(),
              "masked_attention: ", name, " must have its operand's shape, type and device");
  bool fine = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && (x.stride(3) == 1 || x.size(3) == 1);
  for (int i = 0; i < 3; ++i) fine = fine && (x.stride(i) % 8 == 0 || x.size(i) == 1);
  TORCH_CHECK(fine, "masked_attention: ", name, " must lie on 16-byte boundaries");
}

}  // namespace
}  // namespace ma

std::tuple<at::Tensor, at::Tensor, at::Tensor> attn_mask(int64_t B, int64_t S, bool causal, int64_t window,
                                                         const c10::optional<at::Tensor>& docs,
                                                   const c10::optional<at::Tensor>& marks, at::Device device) {
  using namespace ma;
  TORCH_CHECK(B > 0 && S > 0, "attention_mask: needs at least one sequence of one token");
  TORCH_CHECK(S <= int64_t(MAX_TILES) * TILE, "attention_mask: sequences of up to ", MAX_TILES * TILE, " tokens, got ", S);
  MaskArgs a{};
  if (docs.has_value()) {
    TORCH_CHECK(docs->device() == device && docs->dim() == 2 && docs->size(0) == B && docs->size(1) == S &&
                    (docs->stride(1) == 1 || S == 1) &&
                    (docs->scalar_type() == at::kInt || docs->scalar_type() == at::kLong),
                "attention_mask: docs must be [batch, tokens] int32 or int64 on the mask's device");
    a.docs = docs->data_ptr();
    a.docs_stride = docs->stride(0);
    a.docs64 = docs->scalar_type() == at::kLong;
  }
  if (marks.has_value()) {
    TORCH_CHECK(marks->device() == device && marks->dim() == 2 && marks->size(0) == B && marks->size(1) == S &&
                    (marks->stride(1) == 1 || S == 1) && marks->scalar_type() == at::kBool,
                "attention_mask: prefix must be [batch, tokens] bool on the mask's device");
    a.marks = marks->data_ptr<bool>();
    a.marks_stride = marks->stride(0);
  }
  const c10::cuda::CUDAGuard g(device);
  const int64_t nt = (S + TILE - 1) / TILE;
  auto opt = at::TensorOptions().dtype(at::kInt).device(device);
  at::Tensor rows = at::empty({B, nt * TILE, 2}, opt), tiles = at::empty({B, nt, 4}, opt);
  at::Tensor order = at::empty({B, nt}, opt);
  a.rows = reinterpret_cast<int2*>(rows.data_ptr<int>());
  a.tiles = reinterpret_cast<int4*>(tiles.data_ptr<int>());
  a.order = order.data_ptr<int>();
  a.S = S;
  a.padded = nt * TILE;
  a.window = window > 0 && window < 0x40000000 ? window : 0x40000000;
  a.causal = causal;
  C10_CUDA_CHECK(launch_mask(a, B, at::cuda::getCurrentCUDAStream()));
  return {rows, tiles, order};
}

// o [B, S, nq, d] and, where `graded`, the statistics [B, nq, padded] and the rest of o that the backward reads
std::tuple<at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>> masked_attn_fwd(
    const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& rows,
    const at::Tensor& tiles, const at::Tensor& order, double scale, double softcap,
    const c10::optional<at::Tensor>& slopes, bool graded, at::Tensor& err) {
  using namespace ma;
  const Shape n = check(q_, k_, v_, rows, tiles, order, slopes, err);
  const c10::cuda::CUDAGuard g(q_.device());
  at::Tensor o = at::empty({n.B, n.S, n.nq, n.d}, q_.options().memory_format(c10::MemoryFormat::Contiguous));
  c10::optional<at::Tensor> lse, low;
  const int64_t nt = (n.S + TILE - 1) / TILE;
  if (graded) low = at::empty_like(o);
  if (graded) lse = at::empty({n.B, n.nq, nt * TILE}, q_.options().dtype(at::kFloat));
  if (n.B == 0 || n.S == 0 || n.nq == 0) return {o, lse, low};
  const at::Tensor q = usable(q_), k = usable(k_), v = usable(v_);
  FwdParams p;
  fill(p, n, rows, tiles, order, scale, softcap, slopes, graded ? lse->data_ptr<float>() : nullptr, err);
  p.rest = graded;
  C10_CUDA_CHECK(launch_fwd(heads_map(q, TILE), heads_map(k, STEP), heads_map(v, STEP), heads_map(o, TILE),
                            heads_map(graded ? *low : o, TILE), p, softcap > 0, slopes.has_value(),
                            at::cuda::getCurrentCUDAStream()));
  return {o, lse, low};
}

// returns the number of kernels launched
int64_t masked_attn_bwd(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& o,
                     const at::Tensor& low, const at::Tensor& do_, const at::Tensor& lse, const at::Tensor& rows,
                     const at::Tensor& tiles, const at::Tensor& order, double scale, double softcap,
                     const c10::optional<at::Tensor>& slopes, at::Tensor& dq, at::Tensor& dk, at::Tensor& dv,
                     at::Tensor& err) {
  using namespace ma;
  const Shape n = check(q_, k_, v_, rows, tiles, order, slopes, err);
  one_device(q_, o, low, do_, lse);
  const int64_t nt = (n.S + TILE - 1) / TILE;
  TORCH_CHECK(o.sizes() == q_.sizes() && do_.sizes() == q_.sizes() && o.scalar_type() == at::kBFloat16 &&
                  do_.scalar_type() == at::kBFloat16 && o.is_contiguous() && low.sizes() == o.sizes() &&
                  low.scalar_type() == at::kBFloat16 && low.is_contiguous(),
              "masked_attention: the output and its gradient must have the queries' shape and type");
  TORCH_CHECK(lse.is_contiguous() && lse.scalar_type() == at::kFloat && lse.numel() == n.B * n.nq * nt * TILE,
              "masked_attention: statistics of another call");
  check_out(dq, q_, "dq");
  check_out(dk, k_, "dk");
  check_out(dv, v_, "dv");
  if (n.B == 0 || n.S == 0 || n.nq == 0) return 0;
  const c10::cuda::CUDAGuard g(q_.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const at::Tensor q = usable(q_), k = usable(k_), v = usable(v_), dout = usable(do_);
  at::Tensor delta = at::empty_like(lse);
  BwdParams p;
  fill(p, n, rows, tiles, order, scale, softcap, slopes, lse.data_ptr<float>(), err);
  p.neg_delta = delta.data_ptr<float>();
  p.o = out_of(o);
  p.low = low.data_ptr();
  p.dk = out_of(dk);
  p.dv = out_of(dv);
  // Few key tiles leave SMs idle and one block with the whole group's work: then the group is split, as far as
  // two blocks per SM, where a block keeps 16 tiles to work through.  (16384 tokens, 8 heads over 1: 128 blocks
  // took 2.19 ms, 512 blocks 1.11; joining their sums takes 14 us.)
  p.split = 1;
  while (n.B * n.nkv * nt * p.split < 2 * 148 && p.group / p.split >= 2 && nt * p.group / p.split >= 32) {
    int next = p.split + 1;
    while (p.group % next) ++next;
    p.split = next;
  }
  at::Tensor part;
  if (p.split > 1) {
    part = at::empty({p.split, 2, n.B * n.nkv, p.padded, n.d}, lse.options());
    p.part = part.data_ptr<float>();
  }
  C10_CUDA_CHECK(launch_delta(p, out_of(dout), st));
  C10_CUDA_CHECK(launch_dkv(heads_map(q, STEP), heads_map(k, TILE), heads_map(v, TILE), heads_map(dout, STEP),
                            heads_map(dk, TILE), heads_map(dv, TILE), p, softcap > 0, slopes.has_value(), st));
  C10_CUDA_CHECK(launch_dq(heads_map(q, TILE), heads_map(k, STEP), heads_map(v, STEP), heads_map(dout, TILE),
                           heads_map(dq, TILE), p, softcap > 0, slopes.has_value(), st));  // right behind: see there
  if (p.split > 1) C10_CUDA_CHECK(launch_join(p, st));
  return p.split > 1 ? 4 : 3;
}

}  // namespace ft

// Entry points of the gradient norm and clipping (grad_norm.h).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <memory>
#include <vector>

#include "grad_norm.h"

namespace ft {
namespace gn {
namespace {

struct Item {
  const void* x;
  void* y;
  int64_t n;
  uint8_t type, slot;
};

constexpr int SIZE[] = {4, 2, 2};  // bytes by Type

uint8_t type_of(const char* op, const at::Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return F32;
    case at::kBFloat16: return BF16;
    case at::kHalf: return F16;
    default: TORCH_CHECK_TYPE(false, op, ": fp32, bf16 or fp16 tensors are required, got ", x.scalar_type());
  }
}

void check(const char* op, const std::vector<at::Tensor>& xs) {
  for (const at::Tensor& x : xs) {
    TORCH_CHECK_VALUE(x.is_cuda() && x.device() == xs[0].device(), op, ": all tensors must be on one CUDA device, got ",
                xs[0].device(), " and ", x.device());
    type_of(op, x);
  }
}

// The tables of a list: one of up to 64 tensors, or as many large ones as it takes.
struct Tables {
  std::unique_ptr<Table<64>> small;
  std::vector<std::unique_ptr<Table<MAX_TENSORS>>> large;

  explicit Tables(const std::vector<Item>& items) {
    if (items.size() <= 64) {
      small = std::make_unique<Table<64>>();
      fill(*small, items, 0, items.size());
      return;
    }
    for (size_t from = 0; from < items.size(); from += MAX_TENSORS) {
      large.push_back(std::make_unique<Table<MAX_TENSORS>>());
      fill(*large.back(), items, from, std::min(items.size(), from + MAX_TENSORS));
    }
  }
  template <class F>
  void each(F&& go) const {
    if (small) go(*small);
    for (const auto& t : large) go(*t);
  }

 private:
  template <int N>
  static void fill(Table<N>& t, const std::vector<Item>& items, size_t from, size_t to) {
    t.count = static_cast<int>(to - from);
    int64_t chunks = 0;
    for (size_t i = from; i < to; ++i) {
      const size_t k = i - from;
      chunks += (items[i].n + CHUNK - 1) / CHUNK;
      TORCH_CHECK(chunks < (int64_t(1) << 31), "grad_norm: more values than one launch takes");
      t.x[k] = items[i].x;
      t.y[k] = items[i].y;
      t.n[k] = items[i].n;
      t.type[k] = items[i].type;
      t.slot[k] = items[i].slot;
      t.chunk_end[k] = static_cast<int>(chunks);
    }
    t.chunks = static_cast<int>(chunks);
  }
};

// Memory of one call's outputs: no value may be written by two of them, nor read by another one.
void check_apart(const char* op, const std::vector<Item>& items) {
  struct Span {
    uintptr_t from, to;
    size_t who;
  };
  std::vector<Span> out;
  for (size_t i = 0; i < items.size(); ++i) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(items[i].y);
    out.push_back({p, p + items[i].n * SIZE[items[i].type], i});
  }
  auto before = [](const Span& a, const Span& b) { return a.from < b.from; };
  if (!std::is_sorted(out.begin(), out.end(), before)) std::sort(out.begin(), out.end(), before);
  for (size_t i = 1; i < out.size(); ++i)
    TORCH_CHECK(out[i].from >= out[i - 1].to, op, ": two of the tensors written share memory");
  for (size_t i = 0; i < items.size(); ++i) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(items[i].x), e = p + items[i].n * SIZE[items[i].type];
    auto at = std::upper_bound(out.begin(), out.end(), p, [](uintptr_t v, const Span& s) { return v < s.to; });
    for (; at != out.end() && at->from < e; ++at)
      TORCH_CHECK(at->who == i && at->from == p, op, ": a tensor written shares memory with one that is read");
  }
}

at::Tensor dense(const at::Tensor& x) { return x.is_non_overlapping_and_dense() ? x : x.contiguous(); }

// What is read and written, with copies in the place of tensors that are no solid piece of memory
struct Plan {
  std::vector<Item> items;
  std::vector<at::Tensor> held;                            // the copies
  std::vector<std::pair<at::Tensor, at::Tensor>> back;     // (to, from) once the kernel is done
  bool in_place;
};

Plan plan_of(const char* op, const std::vector<at::Tensor>& xs, const std::vector<at::Tensor>& outs) {
  check(op, xs);
  Plan p;
  p.in_place = outs.empty();
  TORCH_CHECK_VALUE(p.in_place || outs.size() == xs.size(), op, ": ", xs.size(), " tensors and ", outs.size(), " outputs");
  for (size_t i = 0; i < xs.size(); ++i) {
    const at::Tensor& o = p.in_place ? xs[i] : outs[i];
    TORCH_CHECK_VALUE(o.sizes() == xs[i].sizes() && o.scalar_type() == xs[i].scalar_type() && o.device() == xs[0].device(), op,
                      ": an output of ", o.scalar_type(), " ", o.sizes(), " for ", xs[i].scalar_type(), " ", xs[i].sizes());
    if (xs[i].numel() == 0) continue;
    if (!o.is_non_overlapping_and_dense()) at::assert_no_internal_overlap(o);
    at::Tensor src = dense(xs[i]);
    at::Tensor dst = o.is_non_overlapping_and_dense() && o.strides() == src.strides() ? o : at::Tensor();
    if (!dst.defined()) {
      dst = p.in_place ? src : at::empty_like(src);  // in place: src is a copy already
      p.back.emplace_back(o, dst);
    }
    p.held.push_back(src);
    p.held.push_back(dst);
    p.items.push_back({src.data_ptr(), dst.data_ptr(), src.numel(), type_of(op, src), 0});
  }
  check_apart(op, p.items);
  // Written by a copy: as far as first addresses tell, as the columns of one matrix are no solid pieces but lie apart.
  for (size_t i = 0; i < p.back.size(); ++i) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p.back[i].first.data_ptr());
    for (const Item& t : p.items) {
      const uintptr_t y = reinterpret_cast<uintptr_t>(t.y);  // (or a copy's own memory, where no tensor of the caller's lies)
      TORCH_CHECK(a < y || a >= y + t.n * SIZE[t.type], op, ": two of the tensors written share memory");
    }
    for (size_t k = 0; k < i; ++k)
      TORCH_CHECK(a != reinterpret_cast<uintptr_t>(p.back[k].first.data_ptr()), op, ": two of the tensors written share memory");
  }
  return p;
}

// Once the kernels are launched: copies go back, and autograd learns that what was written has changed.
void finish(const Plan& p, const std::vector<at::Tensor>& written) {
  for (const auto& [to, from] : p.back) to.copy_(from);
  for (const at::Tensor& x : written)
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

// Launches the sums of all tables; the partial sums [blocks, n_slots].
at::Tensor partials(const Tables& tables, int64_t n_slots, const at::Device& dev, cudaStream_t st) {
  int64_t blocks = 0;
  tables.each([&](const auto& t) { blocks += sumsq_blocks(t.chunks); });
  at::Tensor part = at::empty({blocks, n_slots}, at::TensorOptions().dtype(at::kDouble).device(dev));
  double* at_ = part.data_ptr<double>();
  tables.each([&](const auto& t) {
    C10_CUDA_CHECK(launch_sumsq(t, static_cast<int>(n_slots), at_, st));
    at_ += sumsq_blocks(t.chunks) * n_slots;
  });
  return part;
}

}  // namespace
}  // namespace gn

at::Tensor grad_sumsq(const std::vector<at::Tensor>& xs, const std::vector<int64_t>& slots, int64_t n_slots) {
  using namespace gn;
  TORCH_CHECK(!xs.empty(), "sum_of_squares: no tensors");
  check("sum_of_squares", xs);
  TORCH_CHECK(n_slots >= 1 && n_slots <= MAX_SLOTS, "sum_of_squares: 1 to ", MAX_SLOTS, " slots, got ", n_slots);
  TORCH_CHECK(slots.size() == xs.size(), "sum_of_squares: one slot per tensor is needed");
  const c10::cuda::CUDAGuard g(xs[0].device());
  auto st = at::cuda::getCurrentCUDAStream();
  std::vector<Item> items;
  std::vector<at::Tensor> held;
  for (size_t i = 0; i < xs.size(); ++i) {
    TORCH_CHECK(slots[i] >= 0 && slots[i] < n_slots, "sum_of_squares: slot ", slots[i], " of ", n_slots);
    if (xs[i].numel() == 0) continue;
    held.push_back(dense(xs[i]));
    items.push_back({held.back().data_ptr(), nullptr, xs[i].numel(), type_of("sum_of_squares", xs[i]),
                     static_cast<uint8_t>(slots[i])});
  }
  at::Tensor sums = at::empty({n_slots}, at::TensorOptions().dtype(at::kDouble).device(xs[0].device()));
  if (items.empty()) return sums.zero_();
  const at::Tensor part = partials(Tables(items), n_slots, xs[0].device(), st);
  C10_CUDA_CHECK(launch_finish(part.data_ptr<double>(), static_cast<int>(part.size(0)), static_cast<int>(n_slots),
                               sums.data_ptr<double>(), st));
  return sums;
}

void grad_scale(const std::vector<at::Tensor>& xs, const at::Tensor& coef, const std::vector<at::Tensor>& outs) {
  using namespace gn;
  if (xs.empty()) return;
  const Plan p = plan_of("scale_grads", xs, outs);
  TORCH_CHECK(coef.scalar_type() == at::kFloat && coef.numel() == 1 && coef.device() == xs[0].device(),
              "scale_grads: the factor must be one fp32 number on the tensors' device");
  const c10::cuda::CUDAGuard g(xs[0].device());
  auto st = at::cuda::getCurrentCUDAStream();
  if (p.items.empty()) return;
  const Tables tables(p.items);
  const Factor f{coef.data_ptr<float>(), nullptr, 0, 0.f, nullptr, p.in_place};
  tables.each([&](const auto& t) { C10_CUDA_CHECK(launch_scale(t, f, st)); });
  finish(p, outs.empty() ? xs : outs);
}

at::Tensor grad_clip(const std::vector<at::Tensor>& xs, double max_norm, const std::vector<at::Tensor>& outs) {
  using namespace gn;
  TORCH_CHECK(!xs.empty(), "clip_grads: no tensors");
  const Plan p = plan_of("clip_grads", xs, outs);
  const c10::cuda::CUDAGuard g(xs[0].device());
  auto st = at::cuda::getCurrentCUDAStream();
  at::Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(xs[0].device()));
  if (p.items.empty()) return norm.zero_();
  const Tables tables(p.items);
  const at::Tensor part = partials(tables, 1, xs[0].device(), st);
  const Factor f{nullptr, part.data_ptr<double>(), static_cast<int>(part.size(0)), static_cast<float>(max_norm),
                 norm.data_ptr<float>(), p.in_place};
  tables.each([&](const auto& t) { C10_CUDA_CHECK(launch_scale(t, f, st)); });
  finish(p, outs.empty() ? xs : outs);
  return norm;
}

}  // namespace ft

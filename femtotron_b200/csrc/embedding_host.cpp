// Entry points of the embedding lookup and its sorted gradient (embedding.h).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "embedding.h"

namespace ft {
namespace emb {
namespace {

int type_of(const char* what, const at::Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return F32;
    case at::kBFloat16: return BF16;
    case at::kHalf: return F16;
    default: TORCH_CHECK(false, "embedding: ", what, " must be fp32, bf16 or fp16, got ", x.scalar_type());
  }
}

bool aligned(const at::Tensor& x) {
  return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.size(-1) * x.element_size() % 16 == 0;
}

void check_ids(const at::Tensor& ids, const at::Tensor& other) {
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "embedding: ids must be int32 or int64, got ",
              ids.scalar_type());
  TORCH_CHECK(ids.is_cuda() && ids.device() == other.device(), "embedding: all operands must be on one device, got ",
              ids.device(), " and ", other.device());
  TORCH_CHECK(ids.numel() <= (int64_t(1) << 30), "embedding: at most 2^30 ids, got ", ids.numel());
}

}  // namespace
}  // namespace emb

at::Tensor embed_lookup(const at::Tensor& ids_, const at::Tensor& table, int64_t vstart, double scale) {
  using namespace emb;
  TORCH_CHECK(table.dim() == 2 && table.is_contiguous(), "embedding: the table must be a contiguous [words, values] tensor");
  check_ids(ids_, table);
  const c10::cuda::CUDAGuard g(table.device());
  const at::Tensor ids = ids_.contiguous();
  auto sizes = ids_.sizes().vec();
  sizes.push_back(table.size(1));
  at::Tensor out = at::empty(sizes, table.options());
  if (out.numel() == 0) return out;
  TORCH_CHECK(table.size(1) <= 65535 * 128, "embedding: rows of up to ", 65535 * 128, " values");
  const FwdArgs a{ids.data_ptr(), table.data_ptr(), out.data_ptr(), ids.numel(), table.size(0), vstart,
                  static_cast<int>(table.size(1)), type_of("the table", table), ids.scalar_type() == at::kLong,
                  aligned(table), static_cast<float>(scale)};
  C10_CUDA_CHECK(launch_fwd(a, at::cuda::getCurrentCUDAStream()));
  return out;
}

// dst [words, values] = (accumulate: +=) the gradient; returns the number of kernels launched
int64_t embed_sorted_grad(const at::Tensor& ids_, const at::Tensor& dout_, at::Tensor& dst, bool accumulate, int64_t vstart,
                          double scale) {
  using namespace emb;
  TORCH_CHECK(dst.dim() == 2 && dst.is_contiguous(), "embedding: the gradient must be a contiguous [words, values] tensor");
  check_ids(ids_, dst);
  const int64_t T = ids_.numel(), V = dst.size(0), H = dst.size(1);
  TORCH_CHECK(dout_.device() == dst.device(), "embedding: all operands must be on one device, got ", dout_.device(), " and ",
              dst.device());
  TORCH_CHECK(dout_.dim() == 2 && dout_.size(0) == T && dout_.size(1) == H, "embedding: an output gradient of ", dout_.sizes(),
              " for ", T, " ids and rows of ", H);
  TORCH_CHECK(V < (int64_t(1) << 30), "embedding: too many words");
  type_of("the output gradient", dout_);
  type_of("the gradient", dst);
  const c10::cuda::CUDAGuard g(dst.device());
  auto st = at::cuda::getCurrentCUDAStream();
  if (dst.numel() == 0) return 0;
  TORCH_CHECK(H <= 65535 * 128, "embedding: rows of up to ", 65535 * 128, " values");
  const bool small = T > 0 && T <= SMALL_SORT;
  if (!accumulate && !small) C10_CUDA_CHECK(launch_clear(dst.data_ptr(), dst.nbytes(), false, st));
  if (T == 0) return accumulate ? 0 : 1;
  const at::Tensor ids = ids_.contiguous(), dout = dout_.contiguous();
  SortArgs s{};
  s.ids = ids.data_ptr();
  s.ids64 = ids.scalar_type() == at::kLong;
  s.vstart = vstart;
  s.V = V;
  s.T = static_cast<int>(T);
  s.blocks = static_cast<int>((T + SORT_CHUNK - 1) / SORT_CHUNK);
  int bits = 1;
  while ((int64_t(1) << bits) <= V) ++bits;  // keys 0 ... V
  const int digit = small ? SMALL_BITS : 10;
  s.passes = (bits + digit - 1) / digit;
  TORCH_CHECK(s.passes <= 4, "embedding: too many words");
  int most = 0;
  for (int i = 0; i < s.passes; ++i) {
    s.bits[i] = (bits - i + s.passes - 1) / s.passes;
    most = std::max(most, s.bits[i]);
  }
  const int64_t pieces = (T + PIECE - 1) / PIECE;
  const int64_t words = small ? 2 * T : 4 * T + (int64_t(1) << most) * s.blocks;
  at::Tensor work = at::empty({words}, dst.options().dtype(at::kInt));
  uint32_t* w = reinterpret_cast<uint32_t*>(work.data_ptr<int>());
  for (int i = 0; i < (small ? 1 : 2); ++i) {
    s.key[i] = w + 2 * i * T;
    s.pos[i] = w + (2 * i + 1) * T;
  }
  s.counts = w + 4 * T;
  if (small) {
    C10_CUDA_CHECK(launch_small_sort(s, st));
    if (!accumulate) C10_CUDA_CHECK(launch_clear(dst.data_ptr(), dst.nbytes(), true, st));
  } else C10_CUDA_CHECK(launch_sort(s, st));
  at::Tensor partial = at::empty({pieces, 2, H}, dst.options().dtype(at::kFloat));
  GradArgs a{};
  a.key = s.key[small ? 0 : s.passes & 1];
  a.pos = s.pos[small ? 0 : s.passes & 1];
  a.dout = dout.data_ptr();
  a.dw = dst.data_ptr();
  a.partial = partial.data_ptr<float>();
  a.T = s.T;
  a.H = static_cast<int>(H);
  a.V = static_cast<int>(V);
  a.pieces = static_cast<int>(pieces);
  a.dout_type = type_of("the output gradient", dout);
  a.dw_type = type_of("the gradient", dst);
  a.accumulate = accumulate;
  // 16 bytes of dout per thread; as many values of dw and of the partial sums are then on boundaries too
  a.vec = aligned(dout) && reinterpret_cast<uintptr_t>(dst.data_ptr()) % 16 == 0 &&
          (dst.element_size() >= dout.element_size() || H % 8 == 0);
  a.scale = static_cast<float>(scale);
  C10_CUDA_CHECK(launch_grad(a, st));
  return (accumulate ? 0 : 1) + (small ? 1 : 3 * s.passes) + (pieces > 1 ? 2 : 1);
}

}  // namespace ft

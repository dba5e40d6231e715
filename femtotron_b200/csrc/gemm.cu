// Entry points of the general GEMM: D[M,N] (op)= A[M,K] * B[N,K]^T with the fused epilogues of
// gemm_core.cuh (store, fp32 / bf16 accumulation, residual, SwiGLU, scatter to peer ranks).
#include "gemm_core.cuh"

namespace ft {
namespace gemm {

template <bool A_MN, bool B_MN>
static void dispatch_bn(int bn, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p,
                        int num_tiles, cudaStream_t stream) {
  if (bn == 256)
    launch<A_MN, B_MN, 256, 4>(ta, tb, p, num_tiles, stream);
  else
    launch<A_MN, B_MN, 128, 6>(ta, tb, p, num_tiles, stream);
}

// Pick BN: 256-wide tiles (better operand reuse per UMMA) unless N is small, measured
// faster or equal on every Llama-3-8B projection shape; FT_GEMM_BN=128|256 forces one.
static int choose_bn(int M, int N, bool swiglu) {
  if (swiglu) return 256;
  static int forced = [] {
    const char* e = getenv("FT_GEMM_BN");
    return e ? atoi(e) : 0;
  }();
  if (forced == 128 || forced == 256) return forced;
  (void)M;
  return N > 128 ? 256 : 128;
}

}  // namespace gemm

int64_t gate_reserved_sms() { return gemm::GATE_RESERVED_SMS; }

struct GateScatter {
  int64_t gate_flags = 0;
  int gate_op = 0;
  int gate_epoch = 0;
  int64_t gate_off = 0, gate_row_elems = 1, gate_chunk_elems = 1;
  std::vector<int64_t> scatter_ptrs;
  int scatter_rows = 0;
  int64_t m_rot_rows = 0;
  int reserved_sms = 0;
};

void gemm_tc_impl(const torch::Tensor& A, const torch::Tensor& B, torch::Tensor& D, bool a_mn,
                  bool b_mn, int64_t mode, const c10::optional<torch::Tensor>& R,
                  const c10::optional<torch::Tensor>& GU, int64_t gate_up_off, torch::Tensor& err,
                  const GateScatter& gs);

// A: [M,K] (a_mn=false) or [K,M] (a_mn=true); B: [N,K] (b_mn=false) or [K,N] (b_mn=true).
// D: [M,N] bf16 or fp32 per `mode`.  All operands row-major with unit inner stride.
void gemm_tc(const torch::Tensor& A, const torch::Tensor& B, torch::Tensor& D, bool a_mn,
             bool b_mn, int64_t mode, const c10::optional<torch::Tensor>& R,
             const c10::optional<torch::Tensor>& GU, int64_t gate_up_off, torch::Tensor& err) {
  gemm_tc_impl(A, B, D, a_mn, b_mn, mode, R, GU, gate_up_off, err, GateScatter());
}

// Fused-communication GEMM: K-major operands, optional operand gate and scatter epilogue.
//   gate_op 1/2 gates A/B rows on int32 flags at `gate_flags` (device address);
//   mode 6 stores row r of D into scatter_ptrs[r / scatter_rows] (row stride D.stride(0));
//   m_rot_rows (a multiple of 256, or 0) starts the tile order at that output row;
//   reserved_sms (> 0) is how many SMs a gated launch leaves to the streams releasing it.
void gemm_tc_fused(const torch::Tensor& A, const torch::Tensor& B, torch::Tensor& D, bool a_mn,
                   bool b_mn, int64_t mode,
                   const c10::optional<torch::Tensor>& R, const c10::optional<torch::Tensor>& GU,
                   int64_t gate_up_off, torch::Tensor& err, int64_t gate_flags, int64_t gate_op,
                   int64_t gate_epoch, int64_t gate_off, int64_t gate_row_elems,
                   int64_t gate_chunk_elems, const std::vector<int64_t>& scatter_ptrs,
                   int64_t scatter_rows, int64_t m_rot_rows, int64_t reserved_sms) {
  GateScatter gs;
  gs.gate_flags = gate_flags;
  gs.gate_op = static_cast<int>(gate_op);
  gs.gate_epoch = static_cast<int>(gate_epoch);
  gs.gate_off = gate_off;
  gs.gate_row_elems = std::max<int64_t>(1, gate_row_elems);
  gs.gate_chunk_elems = std::max<int64_t>(1, gate_chunk_elems);
  gs.scatter_ptrs = scatter_ptrs;
  gs.scatter_rows = static_cast<int>(scatter_rows);
  gs.m_rot_rows = m_rot_rows;
  gs.reserved_sms = static_cast<int>(std::max<int64_t>(0, reserved_sms));
  TORCH_CHECK(scatter_ptrs.size() <= 8, "gemm_tc_fused: at most 8 scatter owners");
  if (mode == 6) TORCH_CHECK(scatter_rows > 0 && !scatter_ptrs.empty(), "gemm_tc_fused: scatter needs owners");
  TORCH_CHECK(gs.gate_op == 0 || (gs.gate_op == 1 && !a_mn) || (gs.gate_op == 2 && !b_mn),
              "gemm_tc_fused: only K-major operands can be gated");
  gemm_tc_impl(A, B, D, a_mn, b_mn, mode, R, GU, gate_up_off, err, gs);
}

void gemm_tc_impl(const torch::Tensor& A, const torch::Tensor& B, torch::Tensor& D, bool a_mn,
                  bool b_mn, int64_t mode, const c10::optional<torch::Tensor>& R,
                  const c10::optional<torch::Tensor>& GU, int64_t gate_up_off, torch::Tensor& err,
                  const GateScatter& gs) {
  using namespace gemm;
  TORCH_CHECK(A.is_cuda() && B.is_cuda() && D.is_cuda(), "gemm_tc: CUDA tensors required");
  TORCH_CHECK(A.scalar_type() == at::kBFloat16 && B.scalar_type() == at::kBFloat16,
              "gemm_tc: bf16 operands required");
  TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && D.dim() == 2, "gemm_tc: 2-D operands required");
  TORCH_CHECK(A.stride(1) == 1 && B.stride(1) == 1 && (mode == 6 || D.stride(1) == 1),
              "gemm_tc: unit inner stride required");
  const int M = a_mn ? A.size(1) : A.size(0);
  const int K = a_mn ? A.size(0) : A.size(1);
  const bool swiglu = (mode == EPI_SWIGLU_BF16);
  const int N = D.size(1);
  const int Kb = b_mn ? B.size(0) : B.size(1);
  TORCH_CHECK(K == Kb, "gemm_tc: K mismatch ", K, " vs ", Kb);
  TORCH_CHECK(D.size(0) == M, "gemm_tc: D rows mismatch");
  const bool scatter = (mode == 6);
  if (swiglu) {
    TORCH_CHECK(!b_mn, "gemm_tc: swiglu epilogue needs a K-major B");
    TORCH_CHECK(B.size(0) >= gate_up_off + N, "gemm_tc: swiglu B too small");
    TORCH_CHECK(GU.has_value() && GU->size(0) == M && GU->size(1) >= gate_up_off + N,
                "gemm_tc: swiglu needs GU [M, gate_up_off+N]");
    TORCH_CHECK(N % 8 == 0 && gate_up_off % 8 == 0, "gemm_tc: swiglu sizes must be multiples of 8");
  } else {
    const int Nb = b_mn ? B.size(1) : B.size(0);
    TORCH_CHECK(Nb == N, "gemm_tc: N mismatch ", Nb, " vs ", N);
  }
  TORCH_CHECK(N % 8 == 0, "gemm_tc: N must be a multiple of 8");
  const bool out_f32 = (mode == EPI_STORE_F32 || mode == EPI_ACC_F32);
  TORCH_CHECK(D.scalar_type() == (out_f32 ? at::kFloat : at::kBFloat16), "gemm_tc: D dtype");
  if (!scatter)
    TORCH_CHECK(D.stride(0) % (out_f32 ? 4 : 8) == 0 &&
                    reinterpret_cast<uintptr_t>(D.data_ptr()) % 16 == 0,
                "gemm_tc: D must be 16-byte aligned with an aligned row stride");
  if (mode == EPI_RESID_BF16) {
    TORCH_CHECK(R.has_value() && R->scalar_type() == at::kBFloat16 && R->size(0) == M &&
                    R->size(1) == N && R->stride(1) == 1 && R->stride(0) % 8 == 0,
                "gemm_tc: bad residual");
  }
  const c10::cuda::CUDAGuard guard(A.device());
  auto stream = at::cuda::getCurrentCUDAStream();

  static const int pair_mode = [] {
    const char* e = getenv("FT_GEMM_PAIR");
    return e ? atoi(e) : 1;
  }();
  const bool use_pair = pair_mode != 0 && M > 128 && (swiglu || N > 128);
  // Pair tile width: 256 (best operand reuse) unless 128-wide tiles fill the last wave of
  // CTA pairs enough better.  Cost model: waves x (tile width x k-blocks + a fixed per-tile
  // pipeline fill/drain worth 8 k-blocks of a 256-wide tile), 5% extra for the narrow tile.
  int pbn = 256;
  if (use_pair && !swiglu) {
    const long pairs = std::max(1, num_sms() / 2);
    const long tm = (M + 255) / 256;
    const long kb = (K + BK - 1) / BK;
    const long c256 = (tm * ((N + 255) / 256) + pairs - 1) / pairs * (256 * kb + 2048);
    const long c128 = (tm * ((N + 127) / 128) + pairs - 1) / pairs * (128 * kb + 2048);
    if (c128 * 105 < c256 * 100) pbn = 128;
    if (pair_mode == 2) pbn = 256;
    if (pair_mode == 3) pbn = 128;
  }
  const int bn = use_pair ? pbn : choose_bn(M, N, swiglu);
  const auto BF16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const int a_rows = use_pair ? 128 : BM;            // rows of A staged per CTA
  const int b_rows = use_pair ? bn / 2 : (swiglu ? 128 : bn);  // K-major B rows per TMA box
  CUtensorMap ta = a_mn ? make_tmap_2d(A.data_ptr(), BF16, 2, M, K, A.stride(0), 64, 64, true)
                        : make_tmap_2d(A.data_ptr(), BF16, 2, K, M, A.stride(0), 64, a_rows, true);
  CUtensorMap tb;
  if (b_mn)
    tb = make_tmap_2d(B.data_ptr(), BF16, 2, B.size(1), K, B.stride(0), 64, 64, true);
  else
    tb = make_tmap_2d(B.data_ptr(), BF16, 2, K, B.size(0), B.stride(0), 64, b_rows, true);

  Params p;
  p.M = M; p.N = N; p.K = K;
  p.D = scatter ? nullptr : D.data_ptr();
  p.ldd = scatter ? N : D.stride(0);
  p.R = R.has_value() ? reinterpret_cast<const __nv_bfloat16*>(R->data_ptr()) : nullptr;
  p.ldr = R.has_value() ? R->stride(0) : 0;
  p.GU = GU.has_value() ? reinterpret_cast<__nv_bfloat16*>(GU->data_ptr()) : nullptr;
  p.ldgu = GU.has_value() ? GU->stride(0) : 0;
  p.mode = static_cast<int>(mode);
  p.gate_up_off = static_cast<int>(gate_up_off);
  p.group_m = 8;
  p.err = err.data_ptr<int>();
  p.gate_flags = reinterpret_cast<const int*>(gs.gate_flags);
  p.gate_op = gs.gate_op;
  p.gate_epoch = gs.gate_epoch;
  p.gate_off = gs.gate_off;
  p.gate_row_elems = gs.gate_row_elems;
  p.gate_chunk_elems = gs.gate_chunk_elems;
  // rotation in whole 256-row tiles (both the 128-row and the paired 256-row tilings)
  p.reserved_sms = gs.reserved_sms;
  p.split_rows = 0;
  p.m_rot_rows = (gs.m_rot_rows > 0 && gs.m_rot_rows % 256 == 0 && gs.m_rot_rows < M) ? gs.m_rot_rows : 0;
  for (int i = 0; i < 8; ++i)
    p.scatter_base[i] = i < static_cast<int>(gs.scatter_ptrs.size())
                            ? reinterpret_cast<__nv_bfloat16*>(gs.scatter_ptrs[i])
                            : nullptr;
  p.scatter_rows = gs.scatter_rows;

  const int out_cols = swiglu ? bn / 2 : bn;
  if (use_pair) {
    // fp32 output: TMA store / reduce-add map over D, 32x32 boxes with 128-byte swizzle
    CUtensorMap td = out_f32 ? make_tmap_2d(D.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, N, M,
                                            D.stride(0), 32, 32, true)
                             : ta;  // unused for bf16 outputs
    const int pair_tiles = ((M + 255) / 256) * ((N + out_cols - 1) / out_cols);  // out_cols = bn (or bn/2)
    if (!a_mn && !b_mn) (bn == 256 ? launch_pair<false, false, 256>(ta, tb, td, p, pair_tiles, stream) : launch_pair<false, false, 128>(ta, tb, td, p, pair_tiles, stream));
    else if (!a_mn && b_mn) (bn == 256 ? launch_pair<false, true, 256>(ta, tb, td, p, pair_tiles, stream) : launch_pair<false, true, 128>(ta, tb, td, p, pair_tiles, stream));
    else if (a_mn && b_mn) (bn == 256 ? launch_pair<true, true, 256>(ta, tb, td, p, pair_tiles, stream) : launch_pair<true, true, 128>(ta, tb, td, p, pair_tiles, stream));
    else (bn == 256 ? launch_pair<true, false, 256>(ta, tb, td, p, pair_tiles, stream) : launch_pair<true, false, 128>(ta, tb, td, p, pair_tiles, stream));
    return;
  }
  const int num_tiles = ((M + BM - 1) / BM) * ((N + out_cols - 1) / out_cols);
  if (!a_mn && !b_mn) dispatch_bn<false, false>(bn, ta, tb, p, num_tiles, stream);
  else if (!a_mn && b_mn) dispatch_bn<false, true>(bn, ta, tb, p, num_tiles, stream);
  else if (a_mn && b_mn) dispatch_bn<true, true>(bn, ta, tb, p, num_tiles, stream);
  else dispatch_bn<true, false>(bn, ta, tb, p, num_tiles, stream);
}

}  // namespace ft

// Attention over whole sequences whose rows each see one interval of keys, with capped scores or a bias
// of distance, forward and backward, on tcgen05 (sm_100a).
//
//     x_ij = scale q_i k_j,   capped: x = c tanh(x / c),   with slopes: x -= slope_h |i - j|
//     p_ij = exp(x_ij - lse_i) for lo_i <= j < hi_i, else 0;      o_i = sum_j p_ij v_j
//     dv = p^T do,  dp = do v^T,  ds = p (dp - rowsum(do o)) (1 - tanh^2),  dq = scale ds k,  dk = scale ds^T q
//
// Every mask that is served here (documents packed in a row, padding, a sliding window, a prefix that is
// seen from both sides, causal or not) leaves a row i one interval [lo_i, hi_i) that holds i itself, or
// nothing.  A mask is two integers per row, made by one kernel, and four per tile of 128 rows (least and
// largest lo and hi): which tiles meet, and which of those need no test of single elements, is read off them.
//
// Layout: q, k, v [batch, tokens, heads, d] with any strides that TMA takes, d a multiple of 8 up to 128.
// TMA maps have d, heads, tokens and batch as dimensions of their own, so odd lengths and head sizes end
// in zeros instead of in a neighbour.  Row statistics are padded to whole tiles.
//
// No sum depends on the order of atomics: dq comes from a kernel of its own (7 products instead of the
// 5 of one that adds dq up in memory), and the query heads of a group are added up inside the tile of their
// keys.  The results of a call are the same bits every time.
//
// Padding (rows that see nothing) may hold anything, NaN included: where a tile holds such rows, they are
// zeroed in shared memory before a product sums over them.
//
// masked_attn_host.cpp: the entry points; masked_attn.cu: the mask and the forward pass; masked_attn_dq.cu and
// masked_attn_dkv.cu: the backward pass; masked_attn.cuh: what the kernels share.  Only the entry points see
// torch (its headers take nvcc minutes), the kernels are launched through the functions below.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ft {
namespace ma {

constexpr int TILE = 128;
constexpr int HEAD = 128;  // values of a head that a tile has room for
constexpr int STEP = 64;   // keys (or, for dk and dv, queries) that a step of a kernel takes
constexpr int NTHREADS = 320;  // of the backward kernels: 8 compute warps, 1 TMA warp, 1 MMA warp
constexpr int PRODUCER_WARP = 8, MMA_WARP = 9, COMPUTE_WARPS = 8;
constexpr int MAX_TILES = 2048;  // 262144 tokens: the tiles that meet a tile are listed in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNever = 0x7fffffff;  // lo of a row that sees nothing; its hi is 0

// ------------------------------------------------------------------------------ arguments
struct MaskArgs {
  const void* docs;        // [B, S] int32 or int64, or null
  const bool* marks;       // [B, S], or null
  int64_t docs_stride, marks_stride;
  int2* rows;              // [B, padded] (lo, hi)
  int4* tiles;             // [B, ntiles] (least lo, largest lo, least hi, largest hi)
  int* order;              // [B, ntiles]: key tiles, the one that the most query tiles look at first
  int S, padded, window;   // window: 0x40000000 for none
  bool causal, docs64;
};

struct Common {
  int B, S, padded, ntiles, nq, nkv, group, ksteps, d;
  const int2* rows;       // mask, and 0 or padded (ntiles) per batch
  const int4* tiles;
  int64_t rows_stride, tiles_stride;
  const int* order;       // strides as tiles
  const float* slopes;
  float scale, scale_log2;
  float cap_in, cap_out;  // exp2(s cap_in) = exp(2 scale s / c); c log2(e)
  float cap_small;        // products up to this take the polynomial
  float cap_poly[5];      // tanh(scale s / c) = s (cap_poly[0] + cap_poly[1] s^2 + ...)
  float* neg_lse2;        // [B, nq, padded], minus the log-sum-exp in log2 units; -inf where a row sees nothing
  int* err;
};

struct Out {  // a [batch, tokens, heads, d] tensor of bf16, strides in elements
  void* p;
  int64_t batch, token, head;
};

struct FwdParams : Common {
  bool rest;               // write what o's rounding to bf16 left out, in bf16
};

struct BwdParams : Common {
  Out o;
  const void* low;         // what o's rounding to bf16 left out, in bf16 and laid out like o
  float* neg_delta;        // [B, nq, padded], -rowsum(do o)
  Out dk, dv;
  int split;               // blocks that share the query heads of a group, and with more than one
  float* part;             // [split][2 (dv, dk)][B, nkv, padded][d]: their sums, joined in order
};

// Each returns what cudaGetLastError() says.  launch_delta comes before the other two of the
// backward pass.
cudaError_t launch_mask(const MaskArgs& a, int batch, cudaStream_t st);
cudaError_t launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,
                       const CUtensorMap& tlow, const FwdParams& p, bool cap, bool bias, cudaStream_t st);
cudaError_t launch_delta(const BwdParams& p, const Out& dout, cudaStream_t st);
cudaError_t launch_dq(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                      const CUtensorMap& tdq, const BwdParams& p, bool cap, bool bias, cudaStream_t st);
cudaError_t launch_dkv(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                       const CUtensorMap& tdk, const CUtensorMap& tdv, const BwdParams& p, bool cap, bool bias, cudaStream_t st);
cudaError_t launch_join(const BwdParams& p, cudaStream_t st);  // of the shares of dk and dv, where p.split > 1

}  // namespace ma
}  // namespace ft

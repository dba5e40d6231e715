// Softmax cross entropy of a linear head, x = h W^T, without the logits in memory (sm_100a).
//
//   lse_t = log sum_j exp x_tj,   loss_t = lse_t - x_t,label     (0 where the label is ignored)
//   d_tj  = g_t (exp(x_tj - lse_t) - [j = label_t]),   dh = d W,   dW = d^T h
//
// Forward: the tcgen05 GEMM of gemm_core.cuh whose epilogue reduces each 256-column tile of
// fp32 logits to (max, sum of exponentials) per row; a second kernel joins the tiles of a row.
// The logits leave TMEM only as those two numbers and the label's.
// Backward, in pieces of the vocabulary so that the workspace stays bounded: the product again,
// with an epilogue that turns the fp32 logits into d (bf16, [T, piece]), then dW of the
// piece's rows and the piece's share of dh from it.  The fourth product is the price of never
// storing the logits, whether or not they would fit the workspace.
//
// Bound by the tensor cores for batches of a thousand tokens and more (82 to 88 % active in each
// product) and by the power limit: the four products of 4096 tokens, 128256 words, hidden 4096 run at
// 0.89 to 0.95 of the sustained cuBLAS rate (12.8 to 13.7 ms for the loss and both gradients); by the
// reads of w and the write of dw below that.
//
// d is rounded to bf16 because the tensor cores take it as an operand.  It is stored
// without the upstream gradient's common factor, which is applied in fp32 to the products: the
// entry of the label, close to -1, then keeps its leading digits exactly.
// dh is summed over the pieces in fp32.  A product with too few tiles for the GPU (dh of a short
// batch, whose sum runs over the vocabulary) is split over the sum into partial outputs that a
// last kernel adds in a fixed order: no atomics, the same bits on every run.
#include "checks.h"
#include "gemm_core.cuh"

namespace ft {
namespace gemm {

constexpr float kLog2e = 1.4426950408889634f;

// The tensor cores add each 16-deep step into their fp32 accumulator with truncation, which
// draws a sum of n steps towards zero: a step loses a constant share a of the partial sum so far,
// and partial sums that grow evenly (a run of like signs, or a random walk, in the mean) make
// that a n / 2 of the result.  Measured against 64-bit products, a / 2 = 1.2e-8 (H = 64) to 1.54e-8
// (H = 8192), 1.49e-8 = 2^-26 at H = 4096, where the loss was 2.0e-6 too small.  The logits of
// both passes are therefore multiplied by 1 + 2^-26 n, folded into constants of the epilogues.
// A row whose sums do not grow evenly (a dominating channel) is not mended by this, and the loss is a
// difference of logits.  So the label's logit is left out of the tiles' sums and the loss is
//   log(1 + sum over j != label of exp(x_j - t)),
// with t an fp32 sum of the label's products: it cannot be negative, a small loss keeps its digits, and
// an error of one logit, which the sum of many averages out, does not stand alone in it.  The lse of the
// backward is that of the accumulator's logits throughout, the label's too, times the one factor that both
// passes use, so that p - 1 of a certain word vanishes there as well.
__host__ __device__ __forceinline__ float untruncate(int K) {
  return 1.f + 1.4901161e-8f * static_cast<float>((K + 15) / 16);
}

// What the exponentials of a row with the maximum m are taken from: m, or 0 for a row of nothing but
// -inf, whose sum then stays 0.  The difference x - m is taken before the multiplication by log2 e: m
// log2 e, rounded, would be off by 4e-6 for a logit of 64, and the sum with it.
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.f : m; }

// (max, sum exp(x - max)) of a row's logits in this tile without the label's, and the label's.
struct XentStatsEpi {
  struct Args {
    float2* part;   // [T, tiles_n]: before `untruncate`
    int tiles_n;
    const int64_t* labels;
    float* target;  // [T] the label's logit, before `untruncate`; it is not in `part`
    int64_t vstart;
  };
  static constexpr bool kSplitK = false;
  static constexpr bool kScales = false;
  static constexpr bool kBf16Tma = false;
  __device__ __forceinline__ static float f32_scale(const Args&) { return 1.f; }
  template <int BN>
  __device__ __forceinline__ static void tile(const Params& p, const Args& e, uint32_t tmem_acc, int q,
                                              int lane, int row, int n0, int tn, int, bool) {
    const bool row_ok = row < p.M;
    const uint32_t tbase = tmem_acc + (static_cast<uint32_t>(q * 32) << 16);
    float m = -INFINITY, s = 0.f;
    const float unit = kLog2e * untruncate(p.K);
    const int64_t at = row_ok ? e.labels[row] - e.vstart - n0 : -1;
#pragma unroll 1
    for (int c = 0; c < BN / 32; ++c) {
      const int valid = p.N - n0 - c * 32;
      if (valid <= 0) break;  // the same for the whole warp
      uint32_t r[32];
      tmem_ld_32x32b_x32(tbase + c * 32, r);
      tmem_wait_ld();
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
      if (valid < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i >= valid) v[i] = -INFINITY;
      }
      const int64_t off = at - c * 32;
      const bool hit = off >= 0 && off < 32;
      if (__any_sync(0xffffffffu, hit)) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (off == i) {
            t = v[i];
            v[i] = -INFINITY;
          }
        if (hit) e.target[row] = t;
      }
      float m0 = v[0], m1 = v[1], m2 = v[2], m3 = v[3];
#pragma unroll
      for (int i = 4; i < 32; i += 4) {
        m0 = fmaxf(m0, v[i]); m1 = fmaxf(m1, v[i + 1]);
        m2 = fmaxf(m2, v[i + 2]); m3 = fmaxf(m3, v[i + 3]);
      }
      const float nm = fmaxf(m, fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)));
      const float from = finite_base(nm);  // NaN makes the sum NaN
      float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        s0 += ex2_approx((v[i] - from) * unit);
        s1 += ex2_approx((v[i + 1] - from) * unit);
        s2 += ex2_approx((v[i + 2] - from) * unit);
        s3 += ex2_approx((v[i + 3] - from) * unit);
      }
      s = s * ex2_approx((m - from) * unit) + ((s0 + s1) + (s2 + s3));
      m = nm;
    }
    if (row_ok) e.part[(int64_t)row * e.tiles_n + tn] = make_float2(m, s);
  }
};

// d (without the common factor) of this tile in bf16.
struct XentGradEpi {
  struct Args {
    const int64_t* labels;
    const float* lse;      // [T]
    const float* weight;   // [T] relative row weights, or null: 1, and 0 where ignored
    int64_t vstart;        // of this piece
    int64_t ignore_index;
  };
  static constexpr bool kSplitK = false;
  static constexpr bool kScales = false;
  static constexpr bool kBf16Tma = true;
  __device__ __forceinline__ static float f32_scale(const Args&) { return 1.f; }

  // What turns the logits of a row into its d: p = 2^(x unit - base), less 1 at column `at`, times g.
  struct Row {
    int64_t at = -1;
    float unit, base = 0.f, g = 0.f;
    __device__ __forceinline__ Row(const Params& p, const Args& e, int row, int n0)
        : unit(kLog2e * untruncate(p.K)) {
      if (row >= p.M) return;
      const int64_t lab = e.labels[row];
      at = lab - e.vstart - n0;
      g = lab == e.ignore_index ? 0.f : (e.weight ? e.weight[row] : 1.f);
      base = e.lse[row] * kLog2e;
    }
    template <int N>
    __device__ __forceinline__ void apply(int col, float (&v)[N]) const {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = ex2_approx(fmaf(v[i], unit, -base));
      const int64_t off = at - col;
      const bool hit = off >= 0 && off < N;
      if (__any_sync(0xffffffffu, hit)) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (hit && off == i) v[i] -= 1.f;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = g == 0.f ? 0.f : v[i] * g;  // an ignored row's NaN stays out
    }
  };

  template <int BN>
  __device__ __forceinline__ static void tile(const Params& p, const Args& e, uint32_t tmem_acc, int q,
                                              int lane, int row, int n0, int, int, bool) {
    const uint32_t tbase = tmem_acc + (static_cast<uint32_t>(q * 32) << 16);
    const Row turn(p, e, row, n0);
#pragma unroll 1
    for (int c = 0; c < BN / 32; ++c) {
      if (n0 + c * 32 >= p.N) break;
      uint32_t r[32];
      tmem_ld_32x32b_x32(tbase + c * 32, r);
      tmem_wait_ld();
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
      turn.apply(c * 32, v);
      // rows of D are padded to whole 32-column chunks
      if (row < p.M)
        store_bf16x32(reinterpret_cast<__nv_bfloat16*>(p.D) + (int64_t)row * p.ldd + n0 + c * 32, v, 32);
    }
  }
  template <int BN>
  __device__ __forceinline__ static void tile_bf16_tma(const Params& p, const Args& e, const CUtensorMap* tma_d,
                                                       float (*box)[32 * 32], uint32_t tmem_acc, int q, int lane,
                                                       int row0, int n0, int& buf) {
    const Row turn(p, e, row0 + lane, n0);
    epilogue_tile_bf16_tma<BN>(p, tma_d, box, tmem_acc, q, lane, row0, n0, buf,
                               [&](int col, float (&v)[64]) { turn.apply(col, v); });
  }
};

// The products with d: scaled by the common factor a[0] * b[0], optionally split over K.
struct XentProductEpi {
  struct Args {
    const float* a;  // null: no factor
    const float* b;
    int ksplit;
  };
  static constexpr bool kSplitK = true;
  static constexpr bool kScales = true;
  static constexpr bool kBf16Tma = true;  // split K is for fp32 outputs only
  template <int BN>
  __device__ __forceinline__ static void tile_bf16_tma(const Params& p, const Args& e, const CUtensorMap* tma_d,
                                                       float (*box)[32 * 32], uint32_t tmem_acc, int q, int lane,
                                                       int row0, int n0, int& buf) {
    const float scale = f32_scale(e);
    epilogue_tile_bf16_tma<BN>(p, tma_d, box, tmem_acc, q, lane, row0, n0, buf, [&](int, float (&v)[64]) {
#pragma unroll
      for (int i = 0; i < 64; ++i) v[i] *= scale;
    });
  }
  __device__ __forceinline__ static float f32_scale(const Args& e) {
    return e.a ? e.a[0] * e.b[0] : 1.f;
  }
  template <int BN>
  __device__ __forceinline__ static void tile(const Params& p, const Args& e, uint32_t tmem_acc, int q,
                                              int lane, int row, int n0, int, int split, bool) {
    const bool row_ok = row < p.M;
    const uint32_t tbase = tmem_acc + (static_cast<uint32_t>(q * 32) << 16);
    const float scale = f32_scale(e);
    const int64_t at = ((int64_t)split * p.split_rows + row) * p.ldd;
#pragma unroll 1
    for (int c = 0; c < BN / 32; ++c) {
      const int col0 = n0 + c * 32;
      const int valid = min(32, p.N - col0);
      if (valid <= 0) break;
      uint32_t r[32];
      tmem_ld_32x32b_x32(tbase + c * 32, r);
      tmem_wait_ld();
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * scale;
      if (!row_ok) {
      } else if (p.mode == EPI_STORE_BF16 || p.mode == EPI_ACC_BF16) {
        __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(p.D) + at + col0;
        if (p.mode == EPI_ACC_BF16) {
          float o[32];
          load_bf16x32(d, o, valid);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += o[i];
        }
        store_bf16x32(d, v, valid);
      } else {
        float4* d4 = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.D) + at + col0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j * 4 < valid) {
            float4 x = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            if (p.mode == EPI_ACC_F32) {
              const float4 o = d4[j];
              x.x += o.x; x.y += o.y; x.z += o.z; x.w += o.w;
            }
            d4[j] = x;
          }
        }
      }
    }
  }
};

// ------------------------------------------------------------------ few tokens
// The forward for one or two tokens that no backward follows: one read of w, and nothing for the tensor
// cores to win (a 128-row tile would be nearly empty).  Over 32000 words of 4096: 44.9 us for one token (5.8 TB/s)
// and 51.5 us for two, where the GEMM takes 51 to 58 us up to 128 tokens; three took 71 us here.  A warp takes two vocabulary rows at a time, 2 x 4
// packs of E values in flight per lane; h lies in shared memory in fp32, one plane per 4 of a
// pack's E values, so that the lanes of a 16-byte read touch neighbouring words.  Every warp keeps a
// running (max, sum) per token; a block leaves one pair per token, like a tile of the GEMM.
constexpr int kFewTokens = 2;
constexpr int kFewThreads = 256;

template <int TOK, int E>  // E: 16 values per pack where rows lie on 32-byte boundaries, else 8
__global__ void __launch_bounds__(kFewThreads, 2)
    xent_few_kernel(const __nv_bfloat16* __restrict__ h, int64_t ldh, const __nv_bfloat16* __restrict__ w, int64_t ldw,
                    const int64_t* __restrict__ labels, float2* __restrict__ part, float* __restrict__ target, int T,
                    int V, int H, int64_t vstart) {
  extern __shared__ __align__(16) float hs[];  // [TOK][E / 4][packs][4]
  __shared__ float2 red[kFewThreads / 32][TOK];
  constexpr int U = 4;
  const int packs = H / E, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < TOK * H; i += kFewThreads) {
    const int t = i / H, k = i - t * H, g = k / E, r = k - g * E;
    hs[((t * (E / 4) + r / 4) * packs + g) * 4 + r % 4] =
        t < T ? __bfloat162float(h[t * ldh + k]) : 0.f;
  }
  __syncthreads();
  float m[TOK], s[TOK];
#pragma unroll
  for (int t = 0; t < TOK; ++t) { m[t] = -INFINITY; s[t] = 0.f; }
  const int warps = gridDim.x * (kFewThreads / 32);
  for (int row = 2 * (blockIdx.x * (kFewThreads / 32) + threadIdx.x / 32); row < V; row += 2 * warps) {
    const __nv_bfloat16* wr[2] = {w + row * ldw, w + min(row + 1, V - 1) * ldw};
    float acc[2][TOK];
#pragma unroll
    for (int t = 0; t < TOK; ++t) acc[0][t] = acc[1][t] = 0.f;
    for (int g0 = lane; g0 < packs; g0 += 32 * U) {
      uint32_t x[2][U][E / 2];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int g = g0 + 32 * u;
          const __nv_bfloat16* at = wr[j] + g * E;
#pragma unroll
          for (int i = 0; i < E / 2; ++i) x[j][u][i] = 0;
          if (g < packs) {
            if constexpr (E == 16)
              asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                           : "=r"(x[j][u][0]), "=r"(x[j][u][1]), "=r"(x[j][u][2]), "=r"(x[j][u][3]), "=r"(x[j][u][4]),
                             "=r"(x[j][u][5]), "=r"(x[j][u][6]), "=r"(x[j][u][7])
                           : "l"(__cvta_generic_to_global(at)));
            else {
              const uint4 q = *reinterpret_cast<const uint4*>(at);
              x[j][u][0] = q.x; x[j][u][1] = q.y; x[j][u][2] = q.z; x[j][u][3] = q.w;
            }
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int g = min(g0 + 32 * u, packs - 1);  // past the end x is 0
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          float4 hv[TOK];
#pragma unroll
          for (int t = 0; t < TOK; ++t)
            hv[t] = *reinterpret_cast<const float4*>(hs + ((t * (E / 4) + q) * packs + g) * 4);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t a = x[j][u][2 * q], b = x[j][u][2 * q + 1];
            const float a0 = __uint_as_float(a << 16), a1 = __uint_as_float(a & 0xffff0000u);
            const float b0 = __uint_as_float(b << 16), b1 = __uint_as_float(b & 0xffff0000u);
#pragma unroll
            for (int t = 0; t < TOK; ++t)
              acc[j][t] = fmaf(b1, hv[t].w, fmaf(b0, hv[t].z, fmaf(a1, hv[t].y, fmaf(a0, hv[t].x, acc[j][t]))));
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (row + j >= V) break;  // the same for the whole warp
#pragma unroll
      for (int t = 0; t < TOK; ++t) {
        const float x = warp_sum(acc[j][t]);
        if (t < T && labels[t] == vstart + row + j) {  // the same for the whole warp
          if (lane == 0) target[t] = x;
          continue;
        }
        const float nm = fmaxf(m[t], x);
        const float from = finite_base(nm);
        s[t] = s[t] * ex2_approx((m[t] - from) * kLog2e) + ex2_approx((x - from) * kLog2e);
        m[t] = nm;
      }
    }
  }
  if (lane == 0) {
#pragma unroll
    for (int t = 0; t < TOK; ++t) red[threadIdx.x / 32][t] = make_float2(m[t], s[t]);
  }
  __syncthreads();
  if (threadIdx.x < T) {
    float2 v = red[0][threadIdx.x];
    for (int i = 1; i < kFewThreads / 32; ++i) {
      const float2 o = red[i][threadIdx.x];
      const float nm = fmaxf(v.x, o.x);
      const float from = finite_base(nm);
      v.y = v.y * ex2_approx((v.x - from) * kLog2e) + o.y * ex2_approx((o.x - from) * kLog2e);
      v.x = nm;
    }
    part[threadIdx.x * gridDim.x + blockIdx.x] = v;
  }
}

// ------------------------------------------------------------------ small kernels
// One warp per row joins the tiles' (max, sum), logits times `fix`, and sums the label's products in
// fp32 (no h: `target` holds that sum already).  stats[row] = (max, sum, t, label's logit of the
// accumulator), the first two without the label, the last two 0 and -inf where the label is not here.
__global__ void __launch_bounds__(256) xent_join_kernel(const float2* __restrict__ part,
                                                        const float* __restrict__ target,
                                                        const int64_t* __restrict__ labels,
                                                        const __nv_bfloat16* __restrict__ h, int64_t ldh,
                                                        const __nv_bfloat16* __restrict__ w, int64_t ldw, int H,
                                                        float4* __restrict__ stats, float* __restrict__ lse,
                                                        float* __restrict__ losses, int T, int tiles_n,
                                                        int64_t vstart, int64_t V, int64_t ignore_index,
                                                        float fix) {
  const int row = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (row >= T) return;
  const float2* p = part + (int64_t)row * tiles_n;
  const int64_t lab = labels[row], local = lab - vstart;
  const bool has = local >= 0 && local < V;
  float t = 0.f;
  if (has && h) {
    const uint4* a = reinterpret_cast<const uint4*>(h + row * ldh);
    const uint4* b = reinterpret_cast<const uint4*>(w + local * ldw);
    float t0 = 0.f, t1 = 0.f;
    constexpr int U = 4;  // reads of each row in flight: the wait for them is most of this kernel
    for (int i0 = lane; i0 < H / 8; i0 += 32 * U) {
      uint4 x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + 32 * u, H / 8 - 1);
        x[u] = a[i];
        y[u] = b[i];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t p4[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, q4[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
        if (i0 + 32 * u < H / 8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf16x2(p4[j]), g = unpack_bf16x2(q4[j]);
            t0 = fmaf(f.x, g.x, t0);
            t1 = fmaf(f.y, g.y, t1);
          }
        }
      }
    }
    t = warp_sum(t0 + t1);
  }
  const float unit = kLog2e * fix;
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < tiles_n; i += 32) {
    const float2 v = p[i];
    const float nm = fmaxf(m, v.x);
    const float from = finite_base(nm);
    s = s * exp2f((m - from) * unit) + v.y * exp2f((v.x - from) * unit);
    m = nm;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    const float nm = fmaxf(m, om);
    const float from = finite_base(nm);
    s = s * exp2f((m - from) * unit) + os * exp2f((om - from) * unit);
    m = nm;
  }
  if (lane == 0) {
    const float top = m * fix, log_s = logf(s);
    const float at = has ? target[row] * fix : -INFINITY;
    if (has && !h) t = target[row];
    stats[row] = make_float4(top, s, t, at);
    // lse = log(exp(others) + exp(at))
    const float others = top + log_s;
    lse[row] = fmaxf(others, at) + log1pf(expf(-fabsf(others - at)));
    const float z = (top - t) + log_s;
    const float loss = fmaxf(z, 0.f) + log1pf(expf(-fabsf(z)));
    // a label that no column answers to has no probability: its loss is not a number (nor is an
    // infinite logit's)
    losses[row] = lab == ignore_index ? 0.f : has && t < INFINITY ? loss : __int_as_float(0x7fffffff);
  }
}

// out = {sum of losses (divided by the number of rows that count, for `mean`), the factor of
// its gradient: 1, or 1 / that number (0 for none)}: one block, a fixed order.
__global__ void __launch_bounds__(1024) xent_total_kernel(const float* __restrict__ losses,
                                                          const int64_t* __restrict__ labels,
                                                          float* __restrict__ out, int T,
                                                          int64_t ignore_index, int mean) {
  __shared__ float ls[32];
  __shared__ int ns[32];
  float s = 0.f;
  int n = 0;
  for (int i = threadIdx.x; i < T; i += 1024) {
    s += losses[i];
    n += labels[i] != ignore_index;
  }
  s = warp_sum(s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (threadIdx.x % 32 == 0) { ls[threadIdx.x / 32] = s; ns[threadIdx.x / 32] = n; }
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(ls[threadIdx.x]);
    n = ns[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (threadIdx.x == 0) {
      out[0] = mean ? s / n : s;  // none that counts: 0 / 0, as the mean of nothing
      out[1] = !mean ? 1.f : n ? 1.f / n : 0.f;
    }
  }
}

// Row gradients -> their largest magnitude (the common factor) and weights relative to it.  An ignored
// row's gradient counts as 0, whatever it holds.
// Magnitudes are compared as bit patterns, so that NaN wins.  Where the largest is NaN or infinite
// the factor is 1 and the weights are the gradients themselves: what is not finite stays in its own row.
__global__ void __launch_bounds__(1024) xent_weights_kernel(const float* __restrict__ g,
                                                            const int64_t* __restrict__ labels,
                                                            float* __restrict__ weight, float* __restrict__ factor,
                                                            int T, int64_t ignore_index) {
  __shared__ uint32_t red[32];
  uint32_t top = 0;
  for (int i = threadIdx.x; i < T; i += 1024)
    if (labels[i] != ignore_index) top = max(top, __float_as_uint(g[i]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, red[threadIdx.x % 32]);
  const float m = top > 0 && top < 0x7f800000u ? __uint_as_float(top) : 1.f;
  for (int i = threadIdx.x; i < T; i += 1024) weight[i] = labels[i] != ignore_index ? g[i] / m : 0.f;
  if (threadIdx.x == 0) { factor[0] = m; factor[1] = 1.f; }
}

// dh = factor * sum of the partial products, in order.
__global__ void __launch_bounds__(256) xent_dh_kernel(const float* __restrict__ part, __nv_bfloat16* __restrict__ dh,
                                                      const float* __restrict__ a, const float* __restrict__ b,
                                                      int64_t quads, int64_t stride, int splits, int H4,
                                                      int64_t lddh) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const float f = a[0] * b[0];
  float4 s = reinterpret_cast<const float4*>(part)[i];
  for (int k = 1; k < splits; ++k) {
    const float4 v = reinterpret_cast<const float4*>(part + k * stride)[i];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  const int64_t row = i / H4;
  const int c = static_cast<int>(i - row * H4) * 4;
  *reinterpret_cast<uint2*>(dh + row * lddh + c) =
      make_uint2(pack_bf16x2(s.x * f, s.y * f), pack_bf16x2(s.z * f, s.w * f));
}

// ------------------------------------------------------------------ host side
constexpr auto kBF16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;

// Where the k-blocks of a tile are over before four warps have drained the one before it, eight
// epilogue warps (and four operand stages in place of six, to make room for their boxes) win.
// Weight gradient of 32000 x 4096: 68.8 instead of 75.6 us for 64 tokens, 82.3 instead of 91.1 for
// 256, but 116 instead of 112 for 512 and 262 instead of 235 for 1021 (of 5120).  d of 4096 tokens
// over 32000 words: 101 instead of 117 us at a hidden size of 256, 125 instead of 140 at 512, 364
// instead of 340 at 2048.
constexpr int kFewKProduct = 256, kFewKLogits = 512;

static Params base_params(int M, int N, int K, torch::Tensor& err) {
  Params p{};
  p.M = M; p.N = N; p.K = K;
  p.group_m = 8;
  p.err = err.data_ptr<int>();
  p.gate_row_elems = p.gate_chunk_elems = 1;
  return p;
}

// x = h W^T into an epilogue (W: rows [v0, v0 + N) of the head).
template <class Epi>
static void logits_gemm(const torch::Tensor& h, const torch::Tensor& w, int64_t v0, int N, Params p,
                        typename Epi::Args e, int bn, cudaStream_t st) {
  const int T = h.size(0), H = h.size(1);
  const bool pair = T > 128;
  const auto* wp = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()) + v0 * w.stride(0);
  CUtensorMap ta = make_tmap_2d(h.data_ptr(), kBF16, 2, H, T, h.stride(0), 64, 128, true);
  CUtensorMap tb = make_tmap_2d(wp, kBF16, 2, H, N, w.stride(0), 64, pair ? bn / 2 : bn, true);
  const int tiles = (T + (pair ? 255 : 127)) / (pair ? 256 : 128) * ((N + bn - 1) / bn);
  CUtensorMap td = ta;
  if (pair && Epi::kBf16Tma) td = make_tmap_2d(p.D, kBF16, 2, N, T, p.ldd, 64, 32, true);
  if (pair && Epi::kBf16Tma && H <= kFewKLogits)
    launch_pair<false, false, 256, Epi, Epi::kBf16Tma ? 8 : 4>(ta, tb, td, p, tiles, st, e);
  else if (pair) launch_pair<false, false, 256, Epi>(ta, tb, td, p, tiles, st, e);
  else if (bn == 256) launch<false, false, 256, 4, Epi>(ta, tb, p, tiles, st, e);
  else launch<false, false, 128, 6, Epi>(ta, tb, p, tiles, st, e);
}

static int logits_bn(int T, int N) { return T > 128 ? 256 : (N > 128 * num_sms() ? 256 : 128); }

// D = d W (a_mn false, D fp32 partials) or d^T h (a_mn true).
template <bool A_MN>
static void product(const void* A, int64_t lda, const void* B, int64_t ldb, int M, int N, int K, void* D,
                    int64_t ldd, int mode, int ksplit, int split_rows, const float* fa, const float* fb,
                    torch::Tensor& err, cudaStream_t st) {
  Params p = base_params(M, N, K, err);
  p.D = D;
  p.ldd = ldd;
  p.mode = mode;
  p.split_rows = split_rows;
  XentProductEpi::Args e{fa, fb, ksplit};
  const bool pair = M > 128 && N > 128;
  const bool f32 = mode == EPI_STORE_F32 || mode == EPI_ACC_F32;
  int bn = N > 128 ? 256 : 128;
  const long units = pair ? num_sms() / 2 : num_sms(), tm = (M + (pair ? 255 : 127)) / (pair ? 256 : 128);
  if (bn == 256 && ksplit == 1) {  // the narrow tile where it fills the last wave better
    const long kb = (K + BK - 1) / BK;
    const long c256 = (tm * ((N + 255) / 256) + units - 1) / units * (256 * kb + 2048);
    const long c128 = (tm * ((N + 127) / 128) + units - 1) / units * (128 * kb + 2048);
    if (c128 * 105 < c256 * 100) bn = 128;
  }
  CUtensorMap ta = A_MN ? make_tmap_2d(A, kBF16, 2, M, K, lda, 64, 64, true)
                        : make_tmap_2d(A, kBF16, 2, K, M, lda, 64, 128, true);
  CUtensorMap tb = make_tmap_2d(B, kBF16, 2, N, K, ldb, 64, 64, true);
  const int tiles = static_cast<int>(tm) * ((N + bn - 1) / bn) * ksplit;
  if (pair) {
    const bool few_k = bn == 256 && ksplit == 1 && K <= kFewKProduct;
    CUtensorMap td = f32 ? make_tmap_2d(D, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, N,
                                        ksplit == 1 ? M : (uint64_t)ksplit * split_rows, ldd, 32, 32, true)
                         : make_tmap_2d(D, kBF16, 2, N, M, ldd, 64, 32, true);
    if (few_k) launch_pair<A_MN, true, 256, XentProductEpi, 8>(ta, tb, td, p, tiles, st, e);
    else if (bn == 256) launch_pair<A_MN, true, 256, XentProductEpi>(ta, tb, td, p, tiles, st, e);
    else launch_pair<A_MN, true, 128, XentProductEpi>(ta, tb, td, p, tiles, st, e);
  } else if (bn == 256) {
    launch<A_MN, true, 256, 4, XentProductEpi>(ta, tb, p, tiles, st, e);
  } else {
    launch<A_MN, true, 128, 6, XentProductEpi>(ta, tb, p, tiles, st, e);
  }
}

static void check_operands(const torch::Tensor& h, const torch::Tensor& w, const torch::Tensor& labels,
                           const torch::Tensor& err) {
  check_one_device("linear_xent", h, w, labels, err);
  TORCH_CHECK(h.dim() == 2 && w.dim() == 2, "linear_xent: h and w must be matrices");
  TORCH_CHECK(h.size(1) == w.size(1) && h.size(1) >= 8 && h.size(1) % 8 == 0,
              "linear_xent: h and w must agree in a hidden size that is a multiple of 8, got ", h.size(1), " and ",
              w.size(1));
  for (const torch::Tensor* t : {&h, &w})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kBFloat16 && t->stride(1) == 1 &&
                    t->stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "linear_xent: h and w must be bf16 CUDA matrices with 16-byte aligned rows");
  TORCH_CHECK(labels.is_cuda() && labels.scalar_type() == at::kLong && labels.dim() == 1 && labels.is_contiguous() &&
                  labels.size(0) == h.size(0),
              "linear_xent: labels must be one int64 per row of h");
  TORCH_CHECK(h.size(0) >= 1 && h.size(0) < (int64_t(1) << 30) && w.size(0) >= 1 && w.size(0) < (int64_t(1) << 30),
              "linear_xent: rows out of range");
  TORCH_CHECK(err.is_cuda() && err.scalar_type() == at::kInt);
}

}  // namespace gemm

// {stats [T, 4] (see xent_join_kernel), lse [T], losses [T]} and, for reduce 1 (sum) or 2 (mean), {the
// loss, the factor of its gradient (1, or 1 / rows that count)} as 0-d tensors.  `graded`: a
// backward will use lse.
std::vector<torch::Tensor> linear_xent_fwd(const torch::Tensor& h, const torch::Tensor& w,
                                           const torch::Tensor& labels, int64_t vstart, int64_t ignore_index,
                                           int64_t reduce, bool graded, torch::Tensor& err) {
  using namespace gemm;
  check_operands(h, w, labels, err);
  const c10::cuda::CUDAGuard guard(h.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int T = h.size(0), V = w.size(0), H = h.size(1);
  // few tokens: a read of w by plain loads (see xent_few_kernel), while h fits beside two blocks.  Its
  // logits are fp32 sums; a backward needs lse from the accumulators that it will see itself
  const int tok = T <= 1 ? 1 : 2;
  const int few_bytes = tok * H * 4;
  const bool few = !graded && T <= kFewTokens && few_bytes <= 96 * 1024;
  const int bn = logits_bn(T, V);
  const int tiles_n = few ? std::min((V + 15) / 16, 2 * num_sms()) : (V + bn - 1) / bn;
  const auto f32 = h.options().dtype(at::kFloat);
  // one buffer: the tiles' pairs, then the labels' logits
  torch::Tensor part = torch::empty({(int64_t)T * tiles_n * 2 + T}, f32);
  float* target = part.data_ptr<float>() + (int64_t)T * tiles_n * 2;
  torch::Tensor stats = torch::empty({T, 4}, f32), lse_t = torch::empty({T}, f32), losses = torch::empty({T}, f32);
  if (few) {
    const bool wide = H % 16 == 0 && w.stride(0) % 16 == 0 && reinterpret_cast<uintptr_t>(w.data_ptr()) % 32 == 0;
    auto kern = tok == 1 ? (wide ? xent_few_kernel<1, 16> : xent_few_kernel<1, 8>)
                         : (wide ? xent_few_kernel<2, 16> : xent_few_kernel<2, 8>);
    static unsigned long long done[4] = {0, 0, 0, 0};
    smem_attr_once(kern, 96 * 1024, done[2 * (tok - 1) + wide]);
    kern<<<tiles_n, kFewThreads, few_bytes, st>>>(
        reinterpret_cast<const __nv_bfloat16*>(h.data_ptr()), h.stride(0),
        reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()), w.stride(0), labels.data_ptr<int64_t>(),
        reinterpret_cast<float2*>(part.data_ptr<float>()), target, T, V, H, vstart);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  } else {
    Params p = base_params(T, V, H, err);
    XentStatsEpi::Args e{reinterpret_cast<float2*>(part.data_ptr<float>()), tiles_n, labels.data_ptr<int64_t>(), target,
                         vstart};
    logits_gemm<XentStatsEpi>(h, w, 0, V, p, e, bn, st);
  }
  xent_join_kernel<<<(T + 7) / 8, 256, 0, st>>>(
      reinterpret_cast<const float2*>(part.data_ptr<float>()), target, labels.data_ptr<int64_t>(),
      few ? nullptr : reinterpret_cast<const __nv_bfloat16*>(h.data_ptr()), h.stride(0),
      reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()), w.stride(0), H,
      reinterpret_cast<float4*>(stats.data_ptr<float>()), lse_t.data_ptr<float>(), losses.data_ptr<float>(), T, tiles_n,
      vstart, V, ignore_index, few ? 1.f : untruncate(H));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (reduce == 0) return {stats, lse_t, losses};
  torch::Tensor total = torch::empty({2}, f32);
  xent_total_kernel<<<1, 1024, 0, st>>>(losses.data_ptr<float>(), labels.data_ptr<int64_t>(), total.data_ptr<float>(),
                                        T, ignore_index, reduce == 2);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {stats, lse_t, losses, total.select(0, 0), total.select(0, 1)};
}

// grad: fp32, one value (times factor: the gradient of a sum or mean) or one per row.
// dh: bf16 [T, H] or none; dw: [V, H] bf16 or fp32 or none, stored or accumulated.
// Holds d and all shares of the hidden gradient but one within workspace_bytes (or 256 columns of d,
// where that is more), and one fp32 [T, H] sum beside them (T rounded up to 256 above 128).
// Returns the number of kernels launched.
int64_t linear_xent_bwd(const torch::Tensor& h, const torch::Tensor& w, const torch::Tensor& labels,
                        const torch::Tensor& lse, const torch::Tensor& grad, const torch::Tensor& factor,
                        const c10::optional<torch::Tensor>& dh, const c10::optional<torch::Tensor>& dw,
                        bool accumulate, int64_t vstart, int64_t ignore_index, int64_t workspace_bytes,
                        torch::Tensor& err) {
  using namespace gemm;
  check_one_device("linear_xent_bwd", h, lse, grad, factor);
  if (dh.has_value()) check_one_device("linear_xent_bwd", h, *dh);
  if (dw.has_value()) check_one_device("linear_xent_bwd", h, *dw);
  check_operands(h, w, labels, err);
  const int T = h.size(0), H = h.size(1), V = w.size(0);
  TORCH_CHECK(lse.is_cuda() && lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.numel() == T);
  TORCH_CHECK(grad.is_cuda() && grad.scalar_type() == at::kFloat && grad.is_contiguous() &&
                  (grad.dim() == 0 || grad.numel() == T),
              "linear_xent_bwd: grad must be one fp32 value or one per row");
  TORCH_CHECK(factor.is_cuda() && factor.scalar_type() == at::kFloat && (grad.dim() > 0 || factor.numel() == 1));
  if (dh.has_value())
    TORCH_CHECK(dh->is_cuda() && dh->scalar_type() == at::kBFloat16 && dh->is_contiguous() && dh->dim() == 2 &&
                dh->size(0) == T && dh->size(1) == H);
  int dw_mode = 0;
  if (dw.has_value()) {
    const bool f32 = dw->scalar_type() == at::kFloat;
    TORCH_CHECK(dw->is_cuda() && (f32 || dw->scalar_type() == at::kBFloat16) && dw->dim() == 2 && dw->size(0) == V &&
                    dw->size(1) == H && dw->stride(1) == 1 && dw->stride(0) % (f32 ? 4 : 8) == 0 &&
                    reinterpret_cast<uintptr_t>(dw->data_ptr()) % 16 == 0,
                "linear_xent_bwd: dw must be [V, H] bf16 or fp32 with 16-byte aligned rows");
    dw_mode = f32 ? (accumulate ? EPI_ACC_F32 : EPI_STORE_F32) : (accumulate ? EPI_ACC_BF16 : EPI_STORE_BF16);
  }
  if (!dh.has_value() && !dw.has_value()) return 0;
  const c10::cuda::CUDAGuard guard(h.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const auto f32 = h.options().dtype(at::kFloat);
  int64_t launches = 0;

  // common factor and row weights
  const float *fa = grad.data_ptr<float>(), *fb = factor.data_ptr<float>(), *weight = nullptr;
  torch::Tensor weights;
  if (grad.dim() > 0) {
    weights = torch::empty({T + 2}, f32);
    xent_weights_kernel<<<1, 1024, 0, st>>>(fa, labels.data_ptr<int64_t>(), weights.data_ptr<float>() + 2,
                                            weights.data_ptr<float>(), T, ignore_index);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    fa = weights.data_ptr<float>();
    fb = fa + 1;
    weight = fa + 2;
    ++launches;
  }

  // Pieces of the vocabulary, whole 256-column tiles and as even as they go, and shares of the dh
  // product, by the time that a model of them takes: whole waves of tiles at 20 TFLOP/s per unit (a pair
  // of SMs, or half of it), the sums of the pieces and the last kernel's read of the shares at 6.5
  // TB/s.  All shares but the first, which the sum over the pieces needs anyway, come out of what d
  // leaves of the workspace, so up to twice the fewest pieces are looked at.
  // 1021 tokens of 5120, 32003 words: 80 tiles for 74 pairs, so unsplit the second wave is nearly empty:
  // 422 us by the model, 262 us in 7 shares (measured: 264 in 12).
  const bool pair = T > 128 && H > 128;
  const int64_t units = pair ? num_sms() / 2 : num_sms(), tile_m = pair ? 256 : 128;
  const auto ceil_div = [](int64_t n, int64_t by) { return (n + by - 1) / by; };
  const auto tile_s = [&](double K) { return 2 * tile_m * 256 * K / (pair ? 20e12 : 10e12); };
  const int64_t tm = ceil_div(T, tile_m), th = ceil_div(H, 256);
  // the pair kernel stores whole tiles of 256 rows into a share
  const int64_t split_rows = pair ? ceil_div(T, 256) * 256 : T;
  const int64_t fewest = ceil_div(V, std::max<int64_t>(256, workspace_bytes / (2 * (int64_t)T) / 256 * 256));
  int64_t piece = 0, ldd = 0, ksplit = 1;
  double best = 1e30;
  for (int64_t pieces = fewest; pieces <= (pair && dh.has_value() ? 2 * fewest : fewest); ++pieces) {
    const int64_t cols = ceil_div(ceil_div(V, pieces), 256) * 256, count = ceil_div(V, cols);
    const int64_t pitch = std::min<int64_t>(cols, (V + 31) / 32 * 32);
    const int64_t n_tiles = ceil_div(std::min<int64_t>(cols, V), 256);
    double cost = count * (ceil_div(tm * n_tiles, units) * tile_s(H) + 6e-6);
    if (dw.has_value()) cost += count * ceil_div(n_tiles * th, units) * tile_s(T);
    int64_t shares = 1;
    if (dh.has_value()) {
      const int64_t left = std::max<int64_t>(0, workspace_bytes - 2 * T * pitch);
      const int64_t most = std::min<int64_t>({32, std::max<int64_t>(1, ceil_div(std::min<int64_t>(cols, V), BK) / 8),
                                              1 + left / (4 * split_rows * H)});
      double least = 1e30;
      for (int64_t k = 1; k <= most; ++k) {
        const double c = double(ceil_div(tm * th * k, units)) / k * tile_s(V) + k * (8.0 * count - 4) * T * H / 6.5e12;
        if (c < least * 0.98) { least = c; shares = k; }
      }
      cost += least;
    }
    if (cost < best * 0.98) { best = cost; piece = cols; ldd = pitch; ksplit = shares; }
  }
  torch::Tensor d = torch::empty({T, ldd}, h.options());
  torch::Tensor acc;
  if (dh.has_value()) acc = torch::empty({ksplit * split_rows, H}, f32);

  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int n = static_cast<int>(std::min<int64_t>(piece, V - v0));
    Params p = base_params(T, n, H, err);
    p.D = d.data_ptr();
    p.ldd = ldd;
    XentGradEpi::Args e{labels.data_ptr<int64_t>(), lse.data_ptr<float>(), weight, vstart + v0, ignore_index};
    logits_gemm<XentGradEpi>(h, w, v0, n, p, e, logits_bn(T, n), st);
    ++launches;
    if (dw.has_value()) {
      char* out = reinterpret_cast<char*>(dw->data_ptr()) + v0 * dw->stride(0) * dw->element_size();
      product<true>(d.data_ptr(), ldd, h.data_ptr(), h.stride(0), n, H, T, out, dw->stride(0), dw_mode, 1, 0, fa, fb,
                    err, st);
      ++launches;
    }
    if (dh.has_value()) {
      const auto* wp = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()) + v0 * w.stride(0);
      // every share needs a k-block: a short last piece adds to fewer partial outputs
      const long shares = std::min<long>(ksplit, (n + BK - 1) / BK);
      product<false>(d.data_ptr(), ldd, wp, w.stride(0), T, H, n, acc.data_ptr(), H,
                     v0 == 0 ? EPI_STORE_F32 : EPI_ACC_F32, static_cast<int>(shares), static_cast<int>(split_rows),
                     nullptr, nullptr, err, st);
      ++launches;
    }
  }
  if (dh.has_value()) {
    const int64_t quads = (int64_t)T * (H / 4);
    xent_dh_kernel<<<static_cast<unsigned>((quads + 255) / 256), 256, 0, st>>>(
        acc.data_ptr<float>(), reinterpret_cast<__nv_bfloat16*>(dh->data_ptr()), fa, fb, quads, split_rows * H,
        static_cast<int>(ksplit), H / 4, dh->stride(0));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    ++launches;
  }
  return launches;
}

}  // namespace ft

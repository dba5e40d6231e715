// Attention over a mask of intervals: the mask and the forward pass (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ the mask
// One block per sequence.  A document is a run of equal numbers; it begins at i = 0 and where the number
// changes (negative numbers: padding).  Forward: the running maximum of the beginnings, and of the
// places that are not marked as prefix (a row leads when there is none in its document so far).
// Backward: the running minimum of the places where a document begins or a mark is missing, which ends
// the interval of a leading row.
// The largest v of the threads before this one (`none` for the first), and of all in `total`.
__device__ __forceinline__ int block_scan_max(int v, int none, int* warps, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffff, v, o);
    if (lane >= o) v = max(v, u);
  }
  int before = __shfl_up_sync(0xffffffff, v, 1);
  if (lane == 0) before = none;
  __syncthreads();
  if (lane == 31) warps[w] = v;
  __syncthreads();
  total = none;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
    if (i < w) before = max(before, warps[i]);
    total = max(total, warps[i]);
  }
  return before;
}

__global__ void __launch_bounds__(1024) mask_kernel(const MaskArgs a) {
  __shared__ int warps[32];
  const int b = blockIdx.x, S = a.S;
  int2* rows = a.rows + static_cast<int64_t>(b) * a.padded;
  int4* tiles = a.tiles + static_cast<int64_t>(b) * (a.padded / TILE);
  auto doc = [&](int i) -> int64_t {
    if (!a.docs) return 0;
    const int64_t at = b * a.docs_stride + i;
    return a.docs64 ? static_cast<const int64_t*>(a.docs)[at] : static_cast<const int*>(a.docs)[at];
  };
  auto begins = [&](int i) { return i == 0 || (a.docs && doc(i) != doc(i - 1)); };
  auto marked = [&](int i) { return a.marks && a.marks[b * a.marks_stride + i]; };
  const int chunk = blockDim.x * 4;
  int carry_first = -1, carry_plain = -1;
  for (int c0 = 0; c0 < S; c0 += chunk) {
    const int i0 = c0 + threadIdx.x * 4;
    int first[4], plain[4], f = -1, u = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e;
      if (i < S) {
        if (begins(i)) f = i;
        if (!marked(i)) u = i;
      }
      first[e] = f;
      plain[e] = u;
    }
    int all_f, all_u;
    const int before_f = max(block_scan_max(f, -1, warps, all_f), carry_first);
    const int before_u = max(block_scan_max(u, -1, warps, all_u), carry_plain);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i0 + e < S) {
        const int lo = max(first[e], before_f);
        rows[i0 + e] = make_int2(lo, max(plain[e], before_u) < lo);  // .y: does the row lead
      }
    carry_first = max(carry_first, all_f);
    carry_plain = max(carry_plain, all_u);
  }
  // backward, with the order of rows turned so that the same scan serves: -(place) grows
  int carry = -S;
  const int chunks = (a.padded + chunk - 1) / chunk;
  for (int c = chunks - 1; c >= 0; --c) {
    const int i0 = c * chunk + (static_cast<int>(blockDim.x) - 1 - static_cast<int>(threadIdx.x)) * 4;
    int next[4], n = -kNever, all;  // next[e]: -(first break after row i0 + e) within this thread's rows
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const int i = i0 + e;
      next[e] = n;
      if (i < S && (begins(i) || (a.causal && a.marks && !marked(i)))) n = -i;
    }
    const int before = max(block_scan_max(n, -kNever, warps, all), carry);
    int4 t = make_int4(kNever, 0, kNever, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e;
      if (i >= a.padded) continue;
      int2 r = make_int2(kNever, 0);
      if (i < S && doc(i) >= 0) {
        const int2 got = rows[i];
        const int stop = min(S, -max(next[e], before));
        const int hi = !a.causal || (a.marks && got.y) ? stop : i + 1;
        r = make_int2(max(got.x, i - a.window + 1), min(hi, i + a.window));
      }
      rows[i] = r;
      t = make_int4(min(t.x, r.x), max(t.y, r.x), min(t.z, r.y), max(t.w, r.y));
    }
    // 32 threads of 4 rows each: one tile per warp
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      t.x = min(t.x, __shfl_xor_sync(0xffffffff, t.x, o));
      t.y = max(t.y, __shfl_xor_sync(0xffffffff, t.y, o));
      t.z = min(t.z, __shfl_xor_sync(0xffffffff, t.z, o));
      t.w = max(t.w, __shfl_xor_sync(0xffffffff, t.w, o));
    }
    if ((threadIdx.x & 31) == 31 && i0 < a.padded) tiles[i0 / TILE] = t;
    carry = max(carry, all);
  }
}

// ------------------------------------------------------------------------------ forward
// Two query tiles per block share the key and value tiles of a ring: two heads of a group at the same
// 128 rows where the group has an even number of heads, else 256 rows of one head.  Warps 0-3 and 4-7 each
// run the softmax of one tile, a row per thread that is read once and kept in registers; warp 9 issues the
// products of one tile while the other's softmax runs.  TMEM: S0, S1, O0, O1; the probabilities go over the first half of S as bf16 pairs.
constexpr int KV_STAGES = 4;
// Growth of a row's running maximum (log2 units) below which the sums stay relative to the old one: the
// probabilities stay under 2^8, which bf16 and the fp32 sums hold as well as values under 1.
constexpr float kRescale = 8.0f;

struct FwdSmem {
  __nv_bfloat16 q[2][TILE * HEAD];
  __nv_bfloat16 kv[KV_STAGES][TILE * HEAD];  // K_j, V_j, K_j+1, ...
  uint64_t q_full, kv_full[KV_STAGES], kv_empty[KV_STAGES], clean;
  uint64_t s_full[2], p_half[2], p_full[2], o_done[2], drained;
  uint32_t dead[MAX_TILES / 32];
  uint32_t tmem_base;
};

// Probabilities of 32 keys relative to 2^m from their scores (times `mul`, log2 units), as bf16 pairs; their fp32
// sums in `sums` (of the unrounded values: only p v sees the rounding).  A score of -inf gives 0.
template <bool TEST>
__device__ __forceinline__ void probs32(const uint32_t* sv, float mul, float m, uint64_t& sums, uint32_t (&pk)[16]) {
  const uint64_t mul2_ = pair(mul, mul), m2 = pair(-m, -m);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t x = fma2(pair(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), mul2_, m2);
    const float2 y0 = apart(x);
    float2 y = exp2_of(y0, e);
    if (TEST && on_fma_pipe(e)) y = make_float2(y0.x == -INFINITY ? 0.f : y.x, y0.y == -INFINITY ? 0.f : y.y);
    sums = add2(sums, pair(y.x, y.y));
    pk[e] = pack_bf16x2(y.x, y.y);
  }
}

// The scores of 128 keys from their raw products: transformed (capped, biased), and -inf where they are not
// seen.  TEST: element e is seen when off + e is in [0, width).  Returns the largest.
template <bool CAP, bool ALIBI, bool TEST>
__device__ __forceinline__ float scores128(uint32_t (&sv)[128], const Common& p, float slope2, float far, int off,
                                           int width) {
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < 128; ++e) {
    if (CAP || ALIBI) {
      float keep;
      sv[e] = __float_as_uint(score<CAP, ALIBI>(__uint_as_float(sv[e]), p, slope2, far - e, keep));
    }
    if (TEST && static_cast<uint32_t>(off + e) >= static_cast<uint32_t>(width)) sv[e] = __float_as_uint(-INFINITY);
  }
#pragma unroll
  for (int e = 0; e < 128; e += 2)
    asm("max.f32 %0, %0, %1, %2;"
        : "+f"(m4[(e >> 1) & 3])
        : "f"(__uint_as_float(sv[e])), "f"(__uint_as_float(sv[e + 1])));
  return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
}

template <bool CAP, bool ALIBI>
__global__ void __launch_bounds__(NTHREADS, 1)
    fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FwdParams p) {
  using Sm = FwdSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has
  const uint32_t tile_bytes = chunks * TILE * 64 * 2;

  // late query tiles (the longest rows of a causal mask) first
  const int per = p.pair_heads ? p.nq / 2 : p.nq;
  const int b = blockIdx.x / per, hx = blockIdx.x % per;
  const int yr = static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y);
  const int head[2] = {p.pair_heads ? 2 * hx : hx, p.pair_heads ? 2 * hx + 1 : hx};
  const int qt[2] = {p.pair_heads ? yr : 2 * yr, p.pair_heads ? yr : 2 * yr + 1};
  const int kvh = head[0] / p.group;
  const int2* rows = p.rows + b * p.rows_stride;
  const int4* tiles = p.tiles + b * p.tiles_stride;
  int first[2], end[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    first[t] = end[t] = 0;
    if (qt[t] < p.ntiles) {
      const int4 u = tiles[qt[t]];
      if (u.w > 0) first[t] = u.x / TILE, end[t] = (u.w + TILE - 1) / TILE;
    }
  }
  const int j0 = first[0] == end[0] ? first[1] : first[1] == end[1] ? first[0] : min(first[0], first[1]);
  const int j1 = max(end[0], end[1]);  // no keys at all: both 0

  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < KV_STAGES; ++i) {
      mbar_init(&s.kv_full[i], 1);
      mbar_init(&s.kv_empty[i], 1);
    }
    mbar_init(&s.clean, 1);
    mbar_init(&s.drained, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s.s_full[t], 1);
      mbar_init(&s.p_half[t], 4);
      mbar_init(&s.p_full[t], 4);
      mbar_init(&s.o_done[t], 1);
    }
    fence_barrier_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  note_dead(s.dead, tiles, j0, j1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // where an allocation of all 512 columns begins
  auto tS = [](int t) -> uint32_t { return tmem + static_cast<uint32_t>(t) * 128u; };
  auto tO = [](int t) -> uint32_t { return tmem + 256u + static_cast<uint32_t>(t) * 128u; };

  if (warp < COMPUTE_WARPS) {
    more_registers<FwdRegisters::compute>();
    // ------------------------------------------------------------ softmax warps 0..7
    const int t = warp >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    // (chosen, not indexed: an array that is indexed at run time lies in local memory)
    const int tile = t ? qt[1] : qt[0], h = t ? head[1] : head[0], begin = t ? first[1] : first[0];
    const bool real = tile < p.ntiles;
    const int row = tile * TILE + r;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int n = (t ? end[1] : end[0]) - begin;
    float m_used = -INFINITY, l_run = 0.f;
    bool ok = true;
    int lo = 0, width = 0;
    int4 sum = make_int4(0, 0, 0, 0);
    float slope2 = 0.f;
    if (n > 0) {
      const int2 lh = rows[row];
      if (lh.y > lh.x) lo = lh.x, width = lh.y - lh.x;
      sum = tiles[tile];
      if (ALIBI) slope2 = p.slopes[h] * kLog2e;
    }
    for (int c = 0; c < n && ok; ++c) {
      const int k0 = (begin + c) * TILE;
      ok = wait_warp(&s.s_full[t], c & 1, p.err, 319);
      if (!ok) break;
      tc_fence_after();
      const bool test = k0 < sum.y || k0 + TILE > sum.z;
      const int off = k0 - lo;                 // element e is seen when off + e is in [0, width)
      const float far = static_cast<float>(row - k0);
      uint32_t sv[128];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        tmem_ld_32x32b_x32(tS(t) + lane_off + q * 32, *reinterpret_cast<uint32_t(*)[32]>(sv + q * 32));
      tmem_wait_ld();
      constexpr bool RAW = !CAP && !ALIBI;  // scores without the scale, which then goes into the exponent's FMA
      const float mul = RAW ? p.scale_log2 : 1.f;
      const float mx = mul * (test ? scores128<CAP, ALIBI, true>(sv, p, slope2, far, off, width)
                                   : scores128<CAP, ALIBI, false>(sv, p, slope2, far, off, width));
      const bool need = mx - m_used > kRescale || m_used == -INFINITY;
      const float m_new = need ? fmaxf(m_used, mx) : m_used;
      // S of this block was committed behind the last product into O, which is complete by now
      if (c > 0 && __any_sync(0xffffffffu, need)) {
        const float alpha = m_used == -INFINITY ? 0.f : ex2_approx(m_used - m_new);
        l_run *= alpha;
        for (int cc = 0; cc < p.ksteps; ++cc) {
          uint32_t ov[16];
          const uint32_t ta = tO(t) + lane_off + cc * 16;
          tmem_ld_32x32b_x16(ta, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st_32x32b_x16(ta, ov);
        }
      }
      m_used = m_new;
      const float m = m_used == -INFINITY ? 0.f : m_used;  // a row that has seen nothing yet
      uint64_t sums = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t pk[16];
        if (test) probs32<true>(sv + q * 32, mul, m, sums, pk);
        else probs32<false>(sv + q * 32, mul, m, sums, pk);
        tmem_st_32x32b_x16(tS(t) + lane_off + q * 16, pk);
        if (q == 1) {  // keys 0..63 are stored: their half of the product may start
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.p_half[t]);
        }
      }
      tmem_wait_st();
      const float2 two = apart(sums);
      l_run += two.x + two.y;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full[t]);
    }
    if (n > 0 && ok) ok = wait_warp(&s.o_done[t], 0, p.err, 321);
    if (real && ok) {
      tc_fence_after();
      const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
      __nv_bfloat16* out = at(p.o, b, row, h);
      for (int c = 0; c < p.ksteps; ++c) {
        uint32_t ov[16];
        if (n > 0) {
          tmem_ld_32x32b_x16(tO(t) + lane_off + c * 16, ov);
          tmem_wait_ld();
        }
        if (row < p.S) {
          // a sum of NaN stays one (l is NaN then, not 0)
          if (n == 0 || l_run == 0.f) zero16(out + c * 16, p.d - c * 16);
          else store16(out + c * 16, ov, l_run == l_run ? inv : l_run, p.d - c * 16);
          if (p.low) {
            __nv_bfloat16* low = static_cast<__nv_bfloat16*>(p.low) + (out - static_cast<__nv_bfloat16*>(p.o.p)) + c * 16;
            if (n == 0 || l_run == 0.f) {
              zero16(low, p.d - c * 16);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float v = __uint_as_float(ov[i]) * inv;
                ov[i] = __float_as_uint(v - __bfloat162float(__float2bfloat16_rn(v)));
              }
              store16(low, ov, 1.f, p.d - c * 16);
            }
          }
        }
      }
      if (p.neg_lse2)
        p.neg_lse2[(static_cast<int64_t>(b) * p.nq + h) * p.padded + row] =
            l_run == 0.f ? -INFINITY : -(m_used + log2f(l_run));
    }
  } else {
    fewer_registers<FwdRegisters::other>();
    if (warp == PRODUCER_WARP) {
      // ------------------------------------------------------------ TMA producer
      if (j0 < j1) {
        if (lane == 0) {
          const bool two = qt[1] < p.ntiles;
          mbar_arrive_expect_tx(&s.q_full, two ? 2 * tile_bytes : tile_bytes);
          for (int t = 0; t < (two ? 2 : 1); ++t)
            for (int c = 0; c < chunks; ++c)
              tma_load_4d(s.q[t] + c * 128 * 64, &tm_q, &s.q_full, c * 64, head[t], qt[t] * TILE, b);
        }
        int item = 0;
        bool ok = true;
        for (int j = j0; j < j1 && ok; ++j) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++item) {
            const int st = item % KV_STAGES;
            ok = ok && wait_warp(&s.kv_empty[st], ((item / KV_STAGES) & 1) ^ 1, p.err, 311);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&s.kv_full[st], tile_bytes);
              for (int c = 0; c < chunks; ++c)
                tma_load_4d(s.kv[st] + c * 128 * 64, kv ? &tm_v : &tm_k, &s.kv_full[st], c * 64, kvh, j * TILE, b);
            }
            __syncwarp();
            if (kv && is_dead(s.dead, j)) {
              ok = wait_warp(&s.kv_full[st], (item / KV_STAGES) & 1, p.err, 312);
              zero_dead_rows(s.kv[st], chunks, rows + j * TILE, lane);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s.clean);
            }
          }
        }
        // the copies have landed before the block may leave, also after a wait that ran out
        wait_phase(&s.q_full, 0, p.err, 313);
        for (int i = max(0, item - KV_STAGES); i < item; ++i)
          wait_phase(&s.kv_full[i % KV_STAGES], (i / KV_STAGES) & 1, p.err, 313);
      }
    } else if (warp == MMA_WARP) {
      // ------------------------------------------------------------ MMA issuer
      if (j0 < j1) {
        // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
        const uint32_t leader = elect_one();
        const uint32_t idS = make_idesc_bf16(128, TILE, false, false);           // Q (K-major) x K (K-major)
        const uint32_t idO = make_idesc_bf16(128, p.ksteps * 16, false, true);   // P (TMEM) x V (MN-major)
        int cleaned = j0 - 1, n_clean = 0;
        auto kv_wait = [&](int item) -> bool {
          return wait_warp(&s.kv_full[item % KV_STAGES], (item / KV_STAGES) & 1, p.err, 314);
        };
        // S_t may go over P_t of the block before: that product was issued earlier by this thread
        auto issue_s = [&](int t, int j) {
          tc_fence_after();
          const uint32_t qa = smem_u32(s.q[t]), ka = smem_u32(s.kv[(2 * (j - j0)) % KV_STAGES]);
          mma_tiles(tS(t), qa, ka, idS, p.ksteps, leader);
          commit(&s.s_full[t], leader);
        };
        auto issue_pv = [&](int t, int j) -> bool {
          const int item = 2 * (j - j0) + 1;
          if (!kv_wait(item)) return false;
          if (is_dead(s.dead, j) && cleaned < j) {
            if (!wait_warp(&s.clean, n_clean++ & 1, p.err, 315)) return false;
            cleaned = j;
          }
          const uint32_t va = smem_u32(s.kv[item % KV_STAGES]);
          const int c = j - first[t];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (!wait_warp(half ? &s.p_full[t] : &s.p_half[t], c & 1, p.err, 316)) return false;
            tc_fence_after();
#pragma unroll
            for (int kk = half * 4; kk < half * 4 + 4; ++kk)
              mma_ts(tO(t), tS(t) + kk * 8, make_sw128_desc(va + kk * 2048, 128 * 128, 1024), idO,
                          (c > 0 || kk > 0) ? 1u : 0u, leader);
          }
          commit(&s.o_done[t], j + 1 == end[t] ? leader : 0u);
          return true;
        };
        bool ok = wait_warp(&s.q_full, 0, p.err, 317) && kv_wait(0);
        if (ok) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (first[t] == j0 && j0 < end[t]) issue_s(t, j0);
          commit(&s.kv_empty[0], leader);
        }
        for (int j = j0; ok && j < j1; ++j) {
          const int iv = 2 * (j - j0) + 1, ik = iv + 1;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok) break;
            if (first[t] <= j && j < end[t]) ok = issue_pv(t, j);
            if (ok && first[t] <= j + 1 && j + 1 < end[t]) {
              ok = kv_wait(ik);
              if (ok) issue_s(t, j + 1);
            }
          }
          if (!ok) break;
          commit(&s.kv_empty[iv % KV_STAGES], leader);
          if (j + 1 < j1) commit(&s.kv_empty[ik % KV_STAGES], leader);
        }
        if (!ok) {
          commit(&s.drained, leader);
          wait_warp(&s.drained, 0, p.err, 318);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(s.tmem_base, 512);
  }
}

cudaError_t launch_mask(const MaskArgs& a, int batch, cudaStream_t st) {
  mask_kernel<<<batch, 1024, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const FwdParams& p, bool cap,
                       bool bias, cudaStream_t st) {
  static_assert(sizeof(FwdSmem) + 1024 <= 232448, "shared memory");
  const dim3 grid(p.B * (p.pair_heads ? p.nq / 2 : p.nq), p.pair_heads ? p.ntiles : (p.ntiles + 1) / 2);
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = fwd_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(FwdSmem) + 1024, cfg);
    kernel<<<grid, NTHREADS, sizeof(FwdSmem) + 1024, st>>>(tq, tk, tv, p);
  });
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

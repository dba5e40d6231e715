// Attention over a mask of intervals: the gradient of the queries and the row sums before it (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ backward: rowsum(do o)
// 16 lanes per (row, head), 8 values each, four rows in flight; 0 for rows that see nothing and behind the last
// token.  o comes with what its rounding left out: where a row sees few keys, that rounding is as large as the
// one of ds and dq and dk would be off by 1.7 roundings instead of 1.4.  Bound by HBM: 202 MB (8192 tokens, 32 heads of 128) in
// 39 us, 0.79 of the copy rate.  Inside the dq kernel, whose blocks have o and do at hand or could, it cost more (214 -> 300 us).
constexpr int DELTA_UNITS = 4;

__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ BwdParams p, const Out dout) {
  const int part = threadIdx.x & 15, b = blockIdx.y;
  const uint32_t total = static_cast<uint32_t>(p.padded) * p.nq;  // of one sequence: 32-bit divisions
  const uint32_t u0 = blockIdx.x * 16 + threadIdx.x / 16, step = gridDim.x * 16;  // (blocks times threads may pass 32 bits)
  uint4 x[DELTA_UNITS], l[DELTA_UNITS], y[DELTA_UNITS];
  int64_t stat[DELTA_UNITS];
  bool live[DELTA_UNITS];
#pragma unroll
  for (int k = 0; k < DELTA_UNITS; ++k) {
    const uint32_t unit = u0 + k * step, h = unit % p.nq;
    const int i = static_cast<int>(unit / p.nq);
    stat[k] = unit < total ? (static_cast<int64_t>(b) * p.nq + h) * p.padded + i : -1;
    // loaded wherever there is a row, whether it sees anything or not: nothing waits for the mask
    const bool in = unit < total && i < p.S;
    live[k] = in && p.rows[b * p.rows_stride + i].y > 0;
    x[k] = l[k] = y[k] = make_uint4(0, 0, 0, 0);
    if (in && part * 8 < p.d) {
      const __nv_bfloat16* o = at(p.o, b, i, h) + part * 8;
      x[k] = __ldg(reinterpret_cast<const uint4*>(o));
      l[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.low) +
                                                  (o - static_cast<const __nv_bfloat16*>(p.o.p))));
      y[k] = __ldg(reinterpret_cast<const uint4*>(at(dout, b, i, h) + part * 8));
    }
  }
#pragma unroll
  for (int k = 0; k < DELTA_UNITS; ++k) {
    float acc = 0.f;
    {
      const uint32_t xs[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, ls[4] = {l[k].x, l[k].y, l[k].z, l[k].w},
                     ys[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = unpack_bf16x2(xs[e]), w = unpack_bf16x2(ls[e]), v = unpack_bf16x2(ys[e]);
        acc = fmaf(u.x + w.x, v.x, fmaf(u.y + w.y, v.y, acc));
      }
    }
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) acc += __shfl_xor_sync(0xffffffff, acc, w);
    if (part == 0 && stat[k] >= 0) p.neg_delta[stat[k]] = live[k] ? -acc : 0.f;
  }
}

// ------------------------------------------------------------------------------ backward: dq
// One block per 128 queries of a head; the keys go past, 64 at a time.  S = Q K^T and dP = dO V^T come from shared
// memory, ds goes over S in TMEM as bf16 pairs (rows are queries there, as the product ds K wants its left
// operand), so no tile of scores touches shared memory.  S and dP have two buffers each: those of step j+2 are issued
// behind dq of step j, while the compute warps work on step j+1.
// Measured (32 heads over 8, d = 128): 8192 tokens in documents 194 us, 16384 tokens with 8 heads over 1 590 us (three products:
// 0.85 of the GEMM rate).  Bound by the reads of shared memory of products with 64 columns; 8192 tokens also by a block's
// way in and out.  Q and dO in TMEM (197 instead of 199 us, ragged 176 instead of 170), K and V in rings of their own (206) and
// more steps per wait were no better.
constexpr int DQ_STAGES = 4;

struct DqSmem {
  __nv_bfloat16 q[TILE * HEAD], dout[TILE * HEAD], k[DQ_STAGES][STEP * HEAD], v[DQ_STAGES][STEP * HEAD];
  uint64_t q_full, full[DQ_STAGES], empty[DQ_STAGES], landed;
  uint64_t sp_full[2], ds_full[2], done, drained;
  uint32_t tmem_base;
};

template <bool CAP, bool ALIBI>
__global__ void __launch_bounds__(NTHREADS, 1)
    dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
              const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ BwdParams p) {
  using Sm = DqSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has
  const int b = blockIdx.x / p.nq, h = blockIdx.x % p.nq, kvh = h / p.group;
  const int qt = static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y);
  const int2* rows = p.rows + b * p.rows_stride;
  const int4* tiles = p.tiles + b * p.tiles_stride;
  if (threadIdx.x == PRODUCER_WARP * 32) {
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < DQ_STAGES; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s.sp_full[i], 1), mbar_init(&s.ds_full[i], COMPUTE_WARPS);
    mbar_init(&s.landed, 1);
    mbar_init(&s.done, 1);
    mbar_init(&s.drained, 1);
    fence_barrier_init();
    // on their way before it is known whether the queries see anything
    mbar_arrive_expect_tx(&s.q_full, 2 * chunks * PIECE);
    for (int c = 0; c < chunks; ++c) {
      tma_load_4d(s.q + c * TILE * 64, &tm_q, &s.q_full, c * 64, h, qt * TILE, b);
      tma_load_4d(s.dout + c * TILE * 64, &tm_do, &s.q_full, c * 64, h, qt * TILE, b);
    }
    prefetch(tm_k), prefetch(tm_v), prefetch(tm_dq);
  }
  DeadTiles dead_rows(warp == PRODUCER_WARP, tiles, qt - 30, p.ntiles);
  const int4 sum = tiles[qt];
  const int j0 = uniform(sum.w > 0 ? sum.x / STEP : 0);
  const int n = uniform(sum.w > 0 ? (sum.w + STEP - 1) / STEP - j0 : 0);

  if (warp == MMA_WARP) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // where an allocation of all 512 columns begins
  auto tS = [](int buf) -> uint32_t { return tmem + static_cast<uint32_t>(buf) * 64u; };
  auto tdP = [](int buf) -> uint32_t { return tmem + 128u + static_cast<uint32_t>(buf) * 64u; };
  constexpr uint32_t tdQ = tmem + 384;

  if (warp < COMPUTE_WARPS) {
    // two warps per TMEM lane quadrant (32 queries), 32 of the 64 keys each
    const int quad = warp & 3, half = warp >> 2;
    const int row = qt * TILE + quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int64_t stat = (static_cast<int64_t>(b) * p.nq + h) * p.padded + row;
    int lo = 0, width = 0;
    const int2 lh = rows[row];
    if (lh.y > lh.x) lo = lh.x, width = lh.y - lh.x;
    const float neg_lse2 = p.neg_lse2[stat], neg_delta = p.neg_delta[stat];
    const float slope2 = ALIBI ? p.slopes[h] * kLog2e : 0.f;
    const uint64_t mul = pair(unit<CAP>(p), unit<CAP>(p)), m = pair(neg_lse2, neg_lse2), nd = pair(neg_delta, neg_delta);
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const int buf = it & 1, k0 = (j0 + it) * STEP;
      const bool test = k0 < sum.y || k0 + STEP > sum.z;
      const uint32_t ts = tS(buf) + lane_off + half * 32;
      const int off = k0 + half * 32 - lo;
      const float far = static_cast<float>(row - k0 - half * 32);
      ok = wait_warp(&s.sp_full[buf], (it >> 1) & 1, p.err, 341);
      if (!ok) break;
      tc_fence_after();
      uint32_t sv[32], dv[32], pk[16];
      tmem_ld_32x32b_x32(ts, sv);
      tmem_ld_32x32b_x32(tdP(buf) + lane_off + half * 32, dv);
      tmem_wait_ld();
      float keep[CAP ? 32 : 1];
      cap_scores<CAP, CAP>(sv, keep, p);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const uint64_t x = pair(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
        float2 y = apart(fma2(x, mul, m));
        if (ALIBI) y.x = fmaf(-slope2, fabsf(far - e), y.x), y.y = fmaf(-slope2, fabsf(far - (e + 1)), y.y);
        y = exp2_of<CAP>(y, e / 2);
        if (CAP) y.x *= keep[CAP ? e : 0], y.y *= keep[CAP ? e + 1 : 0];
        const float2 g = apart(mul2(pair(y.x, y.y), add2(pair(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1])), nd)));
        sv[e] = __float_as_uint(g.x);
        sv[e + 1] = __float_as_uint(g.y);
      }
      if (test) {  // replaced, not multiplied: the product may be NaN in a masked place
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (static_cast<uint32_t>(off + e) >= static_cast<uint32_t>(width)) sv[e] = 0u;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1]));
      tmem_st_32x32b_x16(ts, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.ds_full[buf]);
    }
    // (dq takes the place of the queries on its way out: without keys they may still be arriving)
    if (ok) ok = n > 0 ? wait_warp(&s.done, 0, p.err, 343) : wait_warp(&s.q_full, 0, p.err, 344);
    if (!ok) {
      asm volatile("bar.sync 1, 256;" ::: "memory");
    } else {
      tc_fence_after();
      for (int c = half; c < p.ksteps; c += 2) {
        uint32_t v[16] = {};
        if (n > 0) {
          tmem_ld_32x32b_x16(tdQ + lane_off + c * 16, v);
          tmem_wait_ld();
        }
        if (width == 0) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = 0u;
        }
        stage16(s.q, quad * 32 + lane, c, v, p.scale);
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the compute warps
      if (threadIdx.x == 0) {
        tma_store_tile(&tm_dq, s.q, chunks, h, qt * TILE, b);
        tma_store_wait_read();
      }
    }
  } else if (warp == PRODUCER_WARP) {
    if (n > 0) {
      bool ok = true;
      int got = 0, n_dead = 0;
      for (int it = 0; it < n && ok; ++it) {
        const int st = it % DQ_STAGES, ph = (it / DQ_STAGES) & 1, k0 = (j0 + it) * STEP;
        ok = wait_warp(&s.empty[st], ph ^ 1, p.err, 331);
        if (!ok) break;
        // keys of rows that see nothing are zeroed before the products may have them
        const bool dead = dead_rows(tiles, (j0 + it) / 2, p.ntiles);
        uint64_t* bar = dead ? &s.landed : &s.full[st];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, 2 * chunks * STEP_PIECE);
          for (int c = 0; c < chunks; ++c) {
            tma_load_4d(s.k[st] + c * STEP * 64, &tm_k, bar, c * 64, kvh, k0, b);
            tma_load_4d(s.v[st] + c * STEP * 64, &tm_v, bar, c * 64, kvh, k0, b);
          }
        }
        ++got;
        __syncwarp();
        if (dead) {
          ok = wait_warp(&s.landed, n_dead++ & 1, p.err, 332);
          zero_dead_rows(s.k[st], chunks, rows + k0, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.full[st]);
        }
      }
      for (int i = max(0, got - DQ_STAGES); i < got; ++i) wait_phase(&s.full[i % DQ_STAGES], (i / DQ_STAGES) & 1, p.err, 334);
    }
    // (all copies have landed before the block may leave, also after a wait that ran out)
    wait_phase(&s.q_full, 0, p.err, 334);
  } else if (n > 0) {
    // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
    const uint32_t leader = elect_one();
    const uint32_t idQ = make_idesc_bf16(TILE, p.ksteps * 16, false, true);
    const uint32_t qa = desc_low(smem_u32(s.q), 16), da = desc_low(smem_u32(s.dout), 16);
    const uint32_t ka = desc_low(smem_u32(s.k[0]), 16), va = desc_low(smem_u32(s.v[0]), 16);
    const uint32_t kt = desc_low(smem_u32(s.k[0]), STEP_PIECE);
    constexpr uint32_t stage = STEP * HEAD * 2 >> 4;
    auto issue = [&](int it) -> bool {
      const int st = it % DQ_STAGES, buf = it & 1;
      if (!wait_warp(&s.full[st], (it / DQ_STAGES) & 1, p.err, 335)) return false;
      tc_fence_after();
      mma_scores(tS(buf), qa, ka + st * stage, p.ksteps, leader);
      mma_scores(tdP(buf), da, va + st * stage, p.ksteps, leader);
      commit(&s.sp_full[buf], leader);
      return true;
    };
    bool ok = wait_warp(&s.q_full, 0, p.err, 338) && issue(0) && (n < 2 || issue(1));
    for (int it = 0; ok && it < n; ++it) {
      const int st = it % DQ_STAGES, buf = it & 1;
      ok = wait_warp(&s.ds_full[buf], (it >> 1) & 1, p.err, 339);
      if (!ok) break;
      tc_fence_after();
      // ds: keys 0..31 in columns 0..15 of the buffer, 32..63 in 32..47
      mma_values(tdQ, tS(buf), 32, kt + st * stage, idQ, it > 0, leader);
      commit(&s.empty[st], leader);
      if (it + 2 < n) ok = issue(it + 2);
    }
    commit(ok ? &s.done : &s.drained, leader);
    if (!ok) wait_warp(&s.drained, 0, p.err, 340);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(s.tmem_base, 512);
  }
  // what follows on the stream waits for this kernel, so one of its blocks waits for the one before (launch_dq)
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

cudaError_t launch_delta(const BwdParams& p, const Out& dout, cudaStream_t st) {
  const int64_t per = 16 * DELTA_UNITS, total = static_cast<int64_t>(p.padded) * p.nq;
  delta_kernel<<<dim3(static_cast<unsigned>((total + per - 1) / per), p.B), 256, 0, st>>>(p, dout);
  return cudaGetLastError();
}

cudaError_t launch_dq(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                      const CUtensorMap& tdq, const BwdParams& p, bool cap, bool bias, cudaStream_t st) {
  static_assert(sizeof(DqSmem) + 1024 <= 232448, "shared memory");
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = dq_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long set = 0;
    smem_attr_once(kernel, sizeof(DqSmem) + 1024, set);
    // Launched behind dk and dv, of which it reads nothing: its blocks may start as soon as all of theirs have, so that they
    // fill the SMs on which the last of those are through (both passes: 8192 tokens in documents 640 -> 626 us, 2 x 4096 in windows of
    // 1024 with a cap 826 -> 811).
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.B * p.nq, p.ntiles);
    cfg.blockDim = dim3(NTHREADS);
    cfg.dynamicSmemBytes = sizeof(DqSmem) + 1024;
    cfg.stream = st;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, tq, tk, tv, td, tdq, p);
  });
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

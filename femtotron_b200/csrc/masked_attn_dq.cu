// Attention over a mask of intervals: the gradient of the queries and the row sums before it (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ backward: rowsum(do o)
// 16 lanes per (row, head), 8 values each, four rows in flight; 0 for rows that see nothing and behind the last
// token.  o comes with what its rounding left out: where a row sees few keys, that rounding is as large as the
// one of ds and dq and dk would be off by 1.7 roundings instead of 1.4.  Bound by HBM.
constexpr int DELTA_UNITS = 4;

__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ BwdParams p, const Out dout) {
  const int part = threadIdx.x & 15;
  const int64_t total = static_cast<int64_t>(p.B) * p.padded * p.nq;
  const int64_t u0 = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  uint4 x[DELTA_UNITS], l[DELTA_UNITS], y[DELTA_UNITS];
  int64_t stat[DELTA_UNITS];
  bool live[DELTA_UNITS];
#pragma unroll
  for (int k = 0; k < DELTA_UNITS; ++k) {
    const int64_t unit = u0 + k * step;
    const int h = static_cast<int>(unit % p.nq);
    const int64_t tok = unit / p.nq;
    const int b = static_cast<int>(tok / p.padded), i = static_cast<int>(tok % p.padded);
    stat[k] = unit < total ? (static_cast<int64_t>(b) * p.nq + h) * p.padded + i : -1;
    live[k] = unit < total && i < p.S && part * 8 < p.d && p.rows[b * p.rows_stride + i].y > 0;
    if (live[k]) {
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
    if (live[k]) {
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
    if (part == 0 && stat[k] >= 0) p.neg_delta[stat[k]] = -acc;
  }
}

// ------------------------------------------------------------------------------ backward: dq
// One block per 128 queries of a head; the keys go past.  S = Q K^T and dP = dO V^T come from shared
// memory, ds goes over S in TMEM as bf16 pairs (rows are queries there, as the product ds K wants its left
// operand), so no tile of scores touches shared memory.  S has two buffers: S of block j+2 is issued behind
// dq of block j, two steps ahead of the warps that read it.  Three key stages, since K_j is held from S_j to
// dq_j, and two value stages fill the shared memory.
struct DqSmem {
  __nv_bfloat16 q[TILE * HEAD], dout[TILE * HEAD], k[3][TILE * HEAD], v[2][TILE * HEAD];
  uint64_t q_full, k_full[3], k_empty[3], v_full[2], v_empty[2], clean;
  uint64_t s_full[2], dp_full, ds_full, done, drained;
  uint32_t dead[MAX_TILES / 32];
  uint32_t tmem_base;
};

template <bool CAP, bool ALIBI>
__global__ void __launch_bounds__(NTHREADS, 1)
    dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
              const __grid_constant__ BwdParams p) {
  using Sm = DqSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has
  const uint32_t tile_bytes = chunks * TILE * 64 * 2;
  const int b = blockIdx.x / p.nq, h = blockIdx.x % p.nq, kvh = h / p.group;
  const int qt = static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y);
  const int2* rows = p.rows + b * p.rows_stride;
  const int4* tiles = p.tiles + b * p.tiles_stride;
  const int4 sum = tiles[qt];
  const int j0 = sum.w > 0 ? sum.x / TILE : 0, n = sum.w > 0 ? (sum.w + TILE - 1) / TILE - j0 : 0;

  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&s.k_full[i], 1), mbar_init(&s.k_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.s_full[i], 1);
    }
    mbar_init(&s.clean, 1);
    mbar_init(&s.dp_full, 1);
    mbar_init(&s.ds_full, 8);
    mbar_init(&s.done, 1);
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  note_dead(s.dead, tiles, j0, j0 + n);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // where an allocation of all 512 columns begins
  auto tS = [](int st) -> uint32_t { return tmem + static_cast<uint32_t>(st) * 128u; };
  const uint32_t tdP = tmem + 256, tdQ = tmem + 384;

  if (warp < COMPUTE_WARPS) {
    more_registers<BwdRegisters::compute>();
    // two warps per TMEM lane quadrant (32 queries), 64 of the 128 keys each
    const int quad = warp & 3, half = warp >> 2;
    const int row = qt * TILE + quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int64_t stat = (static_cast<int64_t>(b) * p.nq + h) * p.padded + row;
    int lo = 0, width = 0;
    const int2 lh = rows[row];
    if (lh.y > lh.x) lo = lh.x, width = lh.y - lh.x;
    const float neg_lse2 = p.neg_lse2[stat], neg_delta = p.neg_delta[stat];
    const float slope2 = ALIBI ? p.slopes[h] * kLog2e : 0.f;
    bool ok = true;
    for (int it = 0; it < n && ok; ++it) {
      const int k0 = (j0 + it) * TILE;
      const bool test = k0 < sum.y || k0 + TILE > sum.z;
      const uint32_t ts = tS(it & 1) + lane_off + half * 64;
      const int off = k0 + half * 64 - lo;
      const float far = static_cast<float>(row - k0 - half * 64);
      ok = wait_warp(&s.s_full[it & 1], (it >> 1) & 1, p.err, 341);
      if (!ok) break;
      tc_fence_after();
      float pv[64];
      {
        uint32_t sv[64];
        tmem_ld_32x32b_x32(ts, *reinterpret_cast<uint32_t(*)[32]>(sv));
        tmem_ld_32x32b_x32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
        tmem_wait_ld();
        const uint64_t mul = pair(p.scale_log2, p.scale_log2), m = pair(neg_lse2, neg_lse2);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          float2 y, keep = make_float2(1.f, 1.f);
          if (!CAP && !ALIBI) {
            y = apart(fma2(pair(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), mul, m));
          } else {
            y.x = score<CAP, ALIBI>(__uint_as_float(sv[e]), p, slope2, far - e, keep.x) + neg_lse2;
            y.y = score<CAP, ALIBI>(__uint_as_float(sv[e + 1]), p, slope2, far - (e + 1), keep.y) + neg_lse2;
          }
          y = exp2_of(y, e / 2);
          pv[e] = CAP ? y.x * keep.x : y.x;
          pv[e + 1] = CAP ? y.y * keep.y : y.y;
        }
      }
      ok = wait_warp(&s.dp_full, it & 1, p.err, 342);
      if (!ok) break;
      tc_fence_after();
      uint32_t dv[64];
      tmem_ld_32x32b_x32(tdP + lane_off + half * 64, *reinterpret_cast<uint32_t(*)[32]>(dv));
      tmem_ld_32x32b_x32(tdP + lane_off + half * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(dv + 32));
      tmem_wait_ld();
      const uint64_t nd = pair(neg_delta, neg_delta);
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const float2 g = apart(mul2(pair(pv[e], pv[e + 1]), add2(pair(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1])), nd)));
        pv[e] = g.x;
        pv[e + 1] = g.y;
      }
      if (test) {  // replaced, not multiplied: the product may be NaN in a masked place
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (static_cast<uint32_t>(off + e) >= static_cast<uint32_t>(width)) pv[e] = 0.f;
      }
#pragma unroll
      for (int h32 = 0; h32 < 2; ++h32) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(pv[h32 * 32 + 2 * i], pv[h32 * 32 + 2 * i + 1]);
        tmem_st_32x32b_x16(ts + h32 * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.ds_full);
    }
    if (n > 0 && ok) ok = wait_warp(&s.done, 0, p.err, 343);
    if (ok) {
      tc_fence_after();
      __nv_bfloat16* out = at(p.dq, b, row, h);
      for (int c = half; c < p.ksteps; c += 2) {
        uint32_t v[16];
        if (n > 0) {
          tmem_ld_32x32b_x16(tdQ + lane_off + c * 16, v);
          tmem_wait_ld();
        }
        if (row < p.S) {
          if (width == 0) zero16(out + c * 16, p.d - c * 16);
          else store16(out + c * 16, v, p.scale, p.d - c * 16);
        }
      }
    }
  } else {
    fewer_registers<BwdRegisters::other>();
    if (warp == PRODUCER_WARP) {
      if (n > 0) {
        auto load = [&](__nv_bfloat16* dst, const CUtensorMap* tm, uint64_t* bar, int head, int tile) {
          for (int c = 0; c < chunks; ++c) tma_load_4d(dst + c * 128 * 64, tm, bar, c * 64, head, tile * TILE, b);
        };
        if (lane == 0) {
          mbar_arrive_expect_tx(&s.q_full, 2 * tile_bytes);
          load(s.q, &tm_q, &s.q_full, h, qt);
          load(s.dout, &tm_do, &s.q_full, h, qt);
        }
        bool ok = true;
        int nk = 0, nv = 0;
        for (int it = 0; it < n && ok; ++it) {
          const int ks = it % 3, vs = it & 1;
          ok = wait_warp(&s.k_empty[ks], ((it / 3) & 1) ^ 1, p.err, 331);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&s.k_full[ks], tile_bytes);
            load(s.k[ks], &tm_k, &s.k_full[ks], kvh, j0 + it);
          }
          ++nk;
          __syncwarp();
          if (is_dead(s.dead, j0 + it)) {
            ok = wait_warp(&s.k_full[ks], (it / 3) & 1, p.err, 332);
            zero_dead_rows(s.k[ks], chunks, rows + (j0 + it) * TILE, lane);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.clean);
          }
          ok = ok && wait_warp(&s.v_empty[vs], ((it >> 1) & 1) ^ 1, p.err, 333);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&s.v_full[vs], tile_bytes);
            load(s.v[vs], &tm_v, &s.v_full[vs], kvh, j0 + it);
          }
          ++nv;
          __syncwarp();
        }
        // the copies have landed before the block may leave, also after a wait that ran out
        wait_phase(&s.q_full, 0, p.err, 334);
        for (int i = max(0, nk - 3); i < nk; ++i) wait_phase(&s.k_full[i % 3], (i / 3) & 1, p.err, 334);
        for (int i = max(0, nv - 2); i < nv; ++i) wait_phase(&s.v_full[i & 1], (i >> 1) & 1, p.err, 334);
      }
    } else if (warp == MMA_WARP) {
      if (n > 0) {
        // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
        const uint32_t leader = elect_one();
        const uint32_t idS = make_idesc_bf16(128, TILE, false, false);
        const uint32_t idQ = make_idesc_bf16(128, p.ksteps * 16, false, true);
        int n_clean = 0;
        auto issue_s = [&](int it) -> bool {
          if (!wait_warp(&s.k_full[it % 3], (it / 3) & 1, p.err, 335)) return false;
          if (is_dead(s.dead, j0 + it) && !wait_warp(&s.clean, n_clean++ & 1, p.err, 336)) return false;
          tc_fence_after();
          mma_tiles(tS(it & 1), smem_u32(s.q), smem_u32(s.k[it % 3]), idS, p.ksteps, leader);
          commit(&s.s_full[it & 1], leader);
          return true;
        };
        auto issue_dp = [&](int it) -> bool {
          if (!wait_warp(&s.v_full[it & 1], (it >> 1) & 1, p.err, 337)) return false;
          tc_fence_after();
          mma_tiles(tdP, smem_u32(s.dout), smem_u32(s.v[it & 1]), idS, p.ksteps, leader);
          commit(&s.dp_full, leader);
          commit(&s.v_empty[it & 1], leader);
          return true;
        };
        bool ok = wait_warp(&s.q_full, 0, p.err, 338) && issue_s(0) && issue_dp(0) && (n < 2 || issue_s(1));
        for (int it = 0; ok && it < n; ++it) {
          ok = wait_warp(&s.ds_full, it & 1, p.err, 339);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ka = smem_u32(s.k[it % 3]);
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)  // ds: keys 0..63 in columns 0..31, 64..127 in 64..95
            mma_ts(tdQ, tS(it & 1) + (kk >> 2) * 64 + (kk & 3) * 8, make_sw128_desc(ka + kk * 2048, 128 * 128, 1024),
                        idQ, (it > 0 || kk > 0) ? 1u : 0u, leader);
          commit(&s.k_empty[it % 3], leader);
          ok = (it + 1 >= n || issue_dp(it + 1)) && (it + 2 >= n || issue_s(it + 2));
        }
        commit(ok ? &s.done : &s.drained, leader);
        if (!ok) wait_warp(&s.drained, 0, p.err, 340);
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

cudaError_t launch_delta(const BwdParams& p, const Out& dout, cudaStream_t st) {
  const int64_t per = 16 * DELTA_UNITS, total = static_cast<int64_t>(p.B) * p.padded * p.nq;
  delta_kernel<<<static_cast<unsigned>((total + per - 1) / per), 256, 0, st>>>(p, dout);
  return cudaGetLastError();
}

cudaError_t launch_dq(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                      const BwdParams& p, bool cap, bool bias, cudaStream_t st) {
  static_assert(sizeof(DqSmem) + 1024 <= 232448, "shared memory");
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = dq_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(DqSmem) + 1024, cfg);
    kernel<<<dim3(p.B * p.nq, p.ntiles), NTHREADS, sizeof(DqSmem) + 1024, st>>>(tq, tk, tv, td, p);
  });
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

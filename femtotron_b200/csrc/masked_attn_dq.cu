// Attention over a mask of intervals: the gradient of the queries (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

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
  const uint32_t tmem = s.tmem_base;
  auto tS = [tmem](int st) -> uint32_t { return tmem + static_cast<uint32_t>(st) * 128u; };
  const uint32_t tdP = tmem + 256, tdQ = tmem + 384;

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
    if (n > 0 && elect_one()) {
      const uint32_t idS = make_idesc_bf16(128, TILE, false, false);
      const uint32_t idQ = make_idesc_bf16(128, p.ksteps * 16, false, true);
      int n_clean = 0;
      auto product = [&](uint32_t dst, uint32_t a, uint32_t bb) {
        for (int kk = 0; kk < p.ksteps; ++kk) {
          const uint32_t off = (kk >> 2) * 128 * 128 + (kk & 3) * 32;
          mma_bf16(dst, make_sw128_desc(a + off, 16, 1024), make_sw128_desc(bb + off, 16, 1024), idS, kk > 0 ? 1u : 0u);
        }
      };
      auto issue_s = [&](int it) -> bool {
        if (!wait_phase(&s.k_full[it % 3], (it / 3) & 1, p.err, 335)) return false;
        if (is_dead(s.dead, j0 + it) && !wait_phase(&s.clean, n_clean++ & 1, p.err, 336)) return false;
        tc_fence_after();
        product(tS(it & 1), smem_u32(s.q), smem_u32(s.k[it % 3]));
        mma_commit(&s.s_full[it & 1]);
        return true;
      };
      auto issue_dp = [&](int it) -> bool {
        if (!wait_phase(&s.v_full[it & 1], (it >> 1) & 1, p.err, 337)) return false;
        tc_fence_after();
        product(tdP, smem_u32(s.dout), smem_u32(s.v[it & 1]));
        mma_commit(&s.dp_full);
        mma_commit(&s.v_empty[it & 1]);
        return true;
      };
      bool ok = wait_phase(&s.q_full, 0, p.err, 338) && issue_s(0) && issue_dp(0) && (n < 2 || issue_s(1));
      for (int it = 0; ok && it < n; ++it) {
        ok = wait_phase(&s.ds_full, it & 1, p.err, 339);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ka = smem_u32(s.k[it % 3]);
#pragma unroll
        for (int kk = 0; kk < TILE / 16; ++kk)  // ds: keys 0..63 in columns 0..31, 64..127 in 64..95
          mma_bf16_ts(tdQ, tS(it & 1) + (kk >> 2) * 64 + (kk & 3) * 8, make_sw128_desc(ka + kk * 2048, 128 * 128, 1024),
                      idQ, (it > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&s.k_empty[it % 3]);
        ok = (it + 1 >= n || issue_dp(it + 1)) && (it + 2 >= n || issue_s(it + 2));
      }
      mma_commit(ok ? &s.done : &s.drained);
      if (!ok) wait_phase(&s.drained, 0, p.err, 340);
    }
  } else {
    // two warps per TMEM lane quadrant (32 queries), 64 of the 128 keys each
    const int quad = warp & 3, half = warp >> 2;
    const int row = qt * TILE + quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int64_t stat = (static_cast<int64_t>(b) * p.nq + h) * p.padded + row;
    int lo = 0, width = 0;
    const int2 lh = rows[row];
    if (lh.y > lh.x) lo = lh.x, width = lh.y - lh.x;
    const float lse2 = p.lse2[stat], delta = p.delta[stat];
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
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          float keep;
          if (!CAP && !ALIBI) pv[e] = ex2_approx(fmaf(__uint_as_float(sv[e]), p.scale_log2, -lse2));
          else {
            pv[e] = ex2_approx(score<CAP, ALIBI>(__uint_as_float(sv[e]), p, slope2, far - e, keep) - lse2);
            if (CAP) pv[e] *= keep;
          }
        }
      }
      ok = wait_warp(&s.dp_full, it & 1, p.err, 342);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int h32 = 0; h32 < 2; ++h32) {
        uint32_t dv[32], pk[16];
        tmem_ld_32x32b_x32(tdP + lane_off + half * 64 + h32 * 32, dv);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) pv[h32 * 32 + e] *= __uint_as_float(dv[e]) - delta;
        if (test) {  // replaced, not multiplied: the product may be NaN in a masked place
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (static_cast<uint32_t>(off + h32 * 32 + e) >= static_cast<uint32_t>(width)) pv[h32 * 32 + e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack_bf16x2(pv[h32 * 32 + 2 * e], pv[h32 * 32 + 2 * e + 1]);
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
  }

  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
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

// Attention over a mask of intervals: the gradients of the keys and values (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ backward: dk, dv
// One block per 128 keys of a key head; the query tiles that see any of them go past, for every query head
// of the group, so dk and dv are complete in TMEM.  S^T = K Q^T and dP^T = V dO^T (rows are keys); P^T and
// dS^T go over them as bf16 pairs and are the left operands of dv += P^T dO and dk += dS^T Q.  The order
// dv_i, S_i+1, dk_i, dP_i+1 lets the exponentials of one tile run under the products of its neighbours.
constexpr int Q_STAGES = 2;

struct DkvSmem {
  __nv_bfloat16 k[TILE * HEAD], v[TILE * HEAD], q[Q_STAGES][TILE * HEAD], dout[Q_STAGES][TILE * HEAD];
  int2 rows[Q_STAGES][TILE];
  float lse2[Q_STAGES][TILE], delta[Q_STAGES][TILE];
  uint64_t kv_full, q_full[Q_STAGES], q_empty[Q_STAGES], do_full[Q_STAGES], do_empty[Q_STAGES], clean;
  uint64_t s_full, dp_full, p_full, ds_full, done, drained;
  uint16_t list[MAX_TILES];  // query tiles that see a key of this block; bit 14: elements need a test, 15: dead rows
  int count;
  uint32_t tmem_base;
};

template <bool CAP, bool ALIBI>
__global__ void __launch_bounds__(NTHREADS, 1)
    dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
               const __grid_constant__ BwdParams p) {
  using Sm = DkvSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has
  const uint32_t tile_bytes = chunks * TILE * 64 * 2;
  // early key tiles (seen by the most rows of a causal mask) first
  const int b = blockIdx.x / p.nkv, kvh = blockIdx.x % p.nkv, jt = blockIdx.y;
  const int k0 = jt * TILE;
  const int2* rows = p.rows + b * p.rows_stride;
  const int4* tiles = p.tiles + b * p.tiles_stride;

  if (threadIdx.x == 0) {
    mbar_init(&s.kv_full, 1);
    for (int i = 0; i < Q_STAGES; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
      mbar_init(&s.do_full[i], 1);
      mbar_init(&s.do_empty[i], 1);
    }
    mbar_init(&s.clean, 1);
    mbar_init(&s.s_full, 1);
    mbar_init(&s.dp_full, 1);
    mbar_init(&s.p_full, 8);
    mbar_init(&s.ds_full, 8);
    mbar_init(&s.done, 1);
    mbar_init(&s.drained, 1);
    fence_barrier_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 0) {
    int count = 0;
    for (int i0 = 0; i0 < p.ntiles; i0 += 32) {
      const int i = i0 + lane;
      int4 u = make_int4(kNever, 0, 0, 0);
      if (i < p.ntiles) u = tiles[i];
      const bool hit = u.w > k0 && u.x < k0 + TILE;
      const uint32_t m = __ballot_sync(0xffffffff, hit);
      if (hit)
        s.list[count + __popc(m & ((1u << lane) - 1))] = static_cast<uint16_t>(
            i | (k0 < u.y || k0 + TILE > u.z ? 0x4000 : 0) | (u.z == 0 ? 0x8000 : 0));
      count += __popc(m);
    }
    if (lane == 0) s.count = count;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  const uint32_t tS = tmem, tdP = tmem + 128, tdV = tmem + 256, tdK = tmem + 384;
  const int count = s.count, n = count * p.group;

  if (warp == PRODUCER_WARP) {
    if (n > 0) {
      auto load = [&](__nv_bfloat16* dst, const CUtensorMap* tm, uint64_t* bar, int head, int tile) {
        for (int c = 0; c < chunks; ++c) tma_load_4d(dst + c * 128 * 64, tm, bar, c * 64, head, tile * TILE, b);
      };
      if (lane == 0) {
        mbar_arrive_expect_tx(&s.kv_full, 2 * tile_bytes);
        load(s.k, &tm_k, &s.kv_full, kvh, jt);
        load(s.v, &tm_v, &s.kv_full, kvh, jt);
      }
      bool ok = true;
      int nq = 0, nd = 0;
      for (int it = 0; it < n && ok; ++it) {
        const int st = it % Q_STAGES, ph = (it / Q_STAGES) & 1;
        const int h = kvh * p.group + it / count, entry = s.list[it % count], i = entry & 0x3fff;
        ok = wait_warp(&s.q_empty[st], ph ^ 1, p.err, 351);
        if (!ok) break;
        if (lane == 0) {
          const int64_t stat = (static_cast<int64_t>(b) * p.nq + h) * p.padded + i * TILE;
          mbar_arrive_expect_tx(&s.q_full[st], tile_bytes + TILE * 16);
          load(s.q[st], &tm_q, &s.q_full[st], h, i);
          bulk_load(s.rows[st], rows + i * TILE, TILE * 8, &s.q_full[st]);
          bulk_load(s.lse2[st], p.lse2 + stat, TILE * 4, &s.q_full[st]);
          bulk_load(s.delta[st], p.delta + stat, TILE * 4, &s.q_full[st]);
        }
        ++nq;
        __syncwarp();
        ok = wait_warp(&s.do_empty[st], ph ^ 1, p.err, 352);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&s.do_full[st], tile_bytes);
          load(s.dout[st], &tm_do, &s.do_full[st], h, i);
        }
        ++nd;
        __syncwarp();
        if (entry & 0x8000) {
          ok = wait_warp(&s.q_full[st], ph, p.err, 353) && wait_warp(&s.do_full[st], ph, p.err, 353);
          zero_dead_rows(s.q[st], chunks, rows + i * TILE, lane);
          zero_dead_rows(s.dout[st], chunks, rows + i * TILE, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.clean);
        }
      }
      // the copies have landed before the block may leave, also after a wait that ran out
      wait_phase(&s.kv_full, 0, p.err, 354);
      for (int i = max(0, nq - Q_STAGES); i < nq; ++i)
        wait_phase(&s.q_full[i % Q_STAGES], (i / Q_STAGES) & 1, p.err, 354);
      for (int i = max(0, nd - Q_STAGES); i < nd; ++i)
        wait_phase(&s.do_full[i % Q_STAGES], (i / Q_STAGES) & 1, p.err, 354);
    }
  } else if (warp == MMA_WARP) {
    if (n > 0 && elect_one()) {
      const uint32_t idS = make_idesc_bf16(128, TILE, false, false);
      const uint32_t idKV = make_idesc_bf16(128, p.ksteps * 16, false, true);
      int n_clean = 0;
      auto product = [&](uint32_t dst, uint32_t a, uint32_t bb) {
        for (int kk = 0; kk < p.ksteps; ++kk) {
          const uint32_t off = (kk >> 2) * 128 * 128 + (kk & 3) * 32;
          mma_bf16(dst, make_sw128_desc(a + off, 16, 1024), make_sw128_desc(bb + off, 16, 1024), idS, kk > 0 ? 1u : 0u);
        }
      };
      auto gather = [&](uint32_t dst, uint32_t a, uint32_t bb, bool more) {  // queries 0..63 in columns 0..31, 64.. in 64..
#pragma unroll
        for (int kk = 0; kk < TILE / 16; ++kk)
          mma_bf16_ts(dst, a + (kk >> 2) * 64 + (kk & 3) * 8, make_sw128_desc(bb + kk * 2048, 128 * 128, 1024), idKV,
                      (more || kk > 0) ? 1u : 0u);
      };
      auto issue_s = [&](int it) -> bool {
        const int st = it % Q_STAGES;
        if (!wait_phase(&s.q_full[st], (it / Q_STAGES) & 1, p.err, 355)) return false;
        if ((s.list[it % count] & 0x8000) && !wait_phase(&s.clean, n_clean++ & 1, p.err, 356)) return false;
        tc_fence_after();
        product(tS, smem_u32(s.k), smem_u32(s.q[st]));
        mma_commit(&s.s_full);
        return true;
      };
      auto issue_dp = [&](int it) -> bool {
        const int st = it % Q_STAGES;
        if (!wait_phase(&s.do_full[st], (it / Q_STAGES) & 1, p.err, 357)) return false;
        tc_fence_after();
        product(tdP, smem_u32(s.v), smem_u32(s.dout[st]));
        mma_commit(&s.dp_full);
        return true;
      };
      bool ok = wait_phase(&s.kv_full, 0, p.err, 358) && issue_s(0) && issue_dp(0);
      for (int it = 0; ok && it < n; ++it) {
        const int st = it % Q_STAGES;
        ok = wait_phase(&s.p_full, it & 1, p.err, 359);
        if (!ok) break;
        tc_fence_after();
        gather(tdV, tS, smem_u32(s.dout[st]), it > 0);
        mma_commit(&s.do_empty[st]);
        if (it + 1 < n) ok = issue_s(it + 1);
        ok = ok && wait_phase(&s.ds_full, it & 1, p.err, 360);
        if (!ok) break;
        tc_fence_after();
        gather(tdK, tdP, smem_u32(s.q[st]), it > 0);
        mma_commit(&s.q_empty[st]);
        if (it + 1 < n) ok = issue_dp(it + 1);
      }
      mma_commit(ok ? &s.done : &s.drained);
      if (!ok) wait_phase(&s.drained, 0, p.err, 361);
    }
  } else {
    // two warps per TMEM lane quadrant (32 keys), 64 of the 128 queries each
    const int quad = warp & 3, half = warp >> 2;
    const int key = k0 + quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t ts = tS + lane_off + half * 64, td = tdP + lane_off + half * 64;
    bool ok = true;
    for (int it = 0; it < n && ok; ++it) {
      const int st = it % Q_STAGES, entry = s.list[it % count], i = entry & 0x3fff;
      const bool test = entry & 0x4000;
      const float slope2 = ALIBI ? p.slopes[kvh * p.group + it / count] * kLog2e : 0.f;
      const float far = static_cast<float>(key - i * TILE - half * 64);
      ok = wait_warp(&s.s_full, it & 1, p.err, 362);
      if (!ok) break;
      tc_fence_after();
      float pv[64];
      {
        uint32_t sv[64];
        tmem_ld_32x32b_x32(ts, *reinterpret_cast<uint32_t(*)[32]>(sv));
        tmem_ld_32x32b_x32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
        tmem_wait_ld();
        // the statistics arrived with the queries (q_full), which S waited for
        const float4* L = reinterpret_cast<const float4*>(s.lse2[st] + half * 64);
        const int4* R = reinterpret_cast<const int4*>(s.rows[st] + half * 64);
#pragma unroll
        for (int h32 = 0; h32 < 2; ++h32) {
          uint32_t pk[16];
          float kp[32];
#pragma unroll
          for (int c4 = 0; c4 < 8; ++c4) {
            const float4 l4 = L[h32 * 8 + c4];
            const float ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int e = h32 * 32 + c4 * 4 + u;
              float keep = 1.f;
              if (!CAP && !ALIBI) pv[e] = ex2_approx(fmaf(__uint_as_float(sv[e]), p.scale_log2, -ls[u]));
              else pv[e] = ex2_approx(score<CAP, ALIBI>(__uint_as_float(sv[e]), p, slope2, far - e, keep) - ls[u]);
              if (CAP) kp[c4 * 4 + u] = keep;
            }
          }
          if (test) {
#pragma unroll
            for (int e2 = 0; e2 < 16; ++e2) {
              const int4 two = R[h32 * 16 + e2];  // rows 2 e2 and 2 e2 + 1: (lo, hi, lo, hi)
              if (key < two.x || key >= two.y) pv[h32 * 32 + 2 * e2] = 0.f;
              if (key < two.z || key >= two.w) pv[h32 * 32 + 2 * e2 + 1] = 0.f;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) pk[e] = pack_bf16x2(pv[h32 * 32 + 2 * e], pv[h32 * 32 + 2 * e + 1]);
          tmem_st_32x32b_x16(ts + h32 * 16, pk);
          if (CAP) {
#pragma unroll
            for (int e = 0; e < 32; ++e) pv[h32 * 32 + e] *= kp[e];
          }
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full);
      ok = wait_warp(&s.dp_full, it & 1, p.err, 363);
      if (!ok) break;
      tc_fence_after();
      const float4* Dl = reinterpret_cast<const float4*>(s.delta[st] + half * 64);
#pragma unroll
      for (int h32 = 0; h32 < 2; ++h32) {
        uint32_t dv[32], pk[16];
        tmem_ld_32x32b_x32(td + h32 * 32, dv);
        tmem_wait_ld();
#pragma unroll
        for (int c4 = 0; c4 < 8; ++c4) {
          const float4 d4 = Dl[h32 * 8 + c4];
          const float ds[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int e = c4 * 4 + u;
            const float w = pv[h32 * 32 + e], g = w * (__uint_as_float(dv[e]) - ds[u]);
            pv[h32 * 32 + e] = test && w == 0.f ? 0.f : g;  // a masked place may hold NaN
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack_bf16x2(pv[h32 * 32 + 2 * e], pv[h32 * 32 + 2 * e + 1]);
        tmem_st_32x32b_x16(td + h32 * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.ds_full);
    }
    if (n > 0 && ok) ok = wait_warp(&s.done, 0, p.err, 364);
    if (ok) {
      tc_fence_after();
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __nv_bfloat16* out = at(which ? p.dk : p.dv, b, key, kvh);
        for (int c = half; c < p.ksteps; c += 2) {
          uint32_t v[16];
          if (n > 0) {
            tmem_ld_32x32b_x16((which ? tdK : tdV) + lane_off + c * 16, v);
            tmem_wait_ld();
          }
          if (key < p.S) {
            if (n == 0) zero16(out + c * 16, p.d - c * 16);
            else store16(out + c * 16, v, which ? p.scale : 1.f, p.d - c * 16);
          }
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

cudaError_t launch_dkv(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                       const BwdParams& p, bool cap, bool bias, cudaStream_t st) {
  static_assert(sizeof(DkvSmem) + 1024 <= 232448, "shared memory");
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = dkv_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(DkvSmem) + 1024, cfg);
    kernel<<<dim3(p.B * p.nkv, p.ntiles), NTHREADS, sizeof(DkvSmem) + 1024, st>>>(tq, tk, tv, td, p);
  });
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

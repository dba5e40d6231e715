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
  float neg_lse2[Q_STAGES][TILE], neg_delta[Q_STAGES][TILE];
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
  const int bk = blockIdx.x / p.split, sp = blockIdx.x % p.split, jt = blockIdx.y;
  const int b = bk / p.nkv, kvh = bk % p.nkv, heads = p.group / p.split, head0 = kvh * p.group + sp * heads;
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
  constexpr uint32_t tmem = 0;  // where an allocation of all 512 columns begins
  const uint32_t tS = tmem, tdP = tmem + 128, tdV = tmem + 256, tdK = tmem + 384;
  const int count = s.count, n = count * heads;

  if (warp < COMPUTE_WARPS) {
    more_registers<BwdRegisters::compute>();
    // two warps per TMEM lane quadrant (32 keys), 64 of the 128 queries each
    const int quad = warp & 3, half = warp >> 2;
    const int key = k0 + quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t ts = tS + lane_off + half * 64, td = tdP + lane_off + half * 64;
    bool ok = true;
    for (int it = 0; it < n && ok; ++it) {
      const int st = it % Q_STAGES, entry = s.list[it % count], i = entry & 0x3fff;
      const bool test = entry & 0x4000;
      const float slope2 = ALIBI ? p.slopes[head0 + it / count] * kLog2e : 0.f;
      const float far = static_cast<float>(key - i * TILE - half * 64);
      // the statistics of the queries come into registers while S is still in work: between the products'
      // operand reads, shared memory answers late
      ok = wait_warp(&s.q_full[st], (it / Q_STAGES) & 1, p.err, 365);
      if (!ok) break;
      float4 L[16], Dl[16];
#pragma unroll
      for (int c4 = 0; c4 < 16; ++c4) L[c4] = reinterpret_cast<const float4*>(s.neg_lse2[st] + half * 64)[c4];
#pragma unroll
      for (int c4 = 0; c4 < 16; ++c4) Dl[c4] = reinterpret_cast<const float4*>(s.neg_delta[st] + half * 64)[c4];
      ok = wait_warp(&s.s_full, it & 1, p.err, 362);
      if (!ok) break;
      tc_fence_after();
      float pv[64];
      {
        uint32_t sv[64];
        tmem_ld_32x32b_x32(ts, *reinterpret_cast<uint32_t(*)[32]>(sv));
        tmem_ld_32x32b_x32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
        tmem_wait_ld();
        const int4* R = reinterpret_cast<const int4*>(s.rows[st] + half * 64);
        const uint64_t mul = pair(p.scale_log2, p.scale_log2);
        float kp[CAP ? 64 : 1];
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 l = e & 2 ? make_float2(L[e / 4].z, L[e / 4].w) : make_float2(L[e / 4].x, L[e / 4].y);
          float2 y, keep = make_float2(1.f, 1.f);
          if (!CAP && !ALIBI) {
            y = apart(fma2(pair(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), mul, pair(l.x, l.y)));
          } else {
            y.x = score<CAP, ALIBI>(__uint_as_float(sv[e]), p, slope2, far - e, keep.x) + l.x;
            y.y = score<CAP, ALIBI>(__uint_as_float(sv[e + 1]), p, slope2, far - (e + 1), keep.y) + l.y;
          }
          y = exp2_of(y, e / 2);
          pv[e] = y.x;
          pv[e + 1] = y.y;
          if (CAP) kp[e] = keep.x, kp[e + 1] = keep.y;
        }
        if (test) {
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            const int4 two = R[e / 2];  // rows e and e + 1: (lo, hi, lo, hi)
            if (key < two.x || key >= two.y) pv[e] = 0.f;
            if (key < two.z || key >= two.w) pv[e + 1] = 0.f;
          }
        }
#pragma unroll
        for (int h32 = 0; h32 < 2; ++h32) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(pv[h32 * 32 + 2 * i], pv[h32 * 32 + 2 * i + 1]);
          tmem_st_32x32b_x16(ts + h32 * 16, pk);
        }
        if (CAP) {
#pragma unroll
          for (int e = 0; e < 64; ++e) pv[e] *= kp[CAP ? e : 0];
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full);
      ok = wait_warp(&s.dp_full, it & 1, p.err, 363);
      if (!ok) break;
      tc_fence_after();
      uint32_t dv[64];
      tmem_ld_32x32b_x32(td, *reinterpret_cast<uint32_t(*)[32]>(dv));
      tmem_ld_32x32b_x32(td + 32, *reinterpret_cast<uint32_t(*)[32]>(dv + 32));
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const uint64_t nd = e & 2 ? pair(Dl[e / 4].z, Dl[e / 4].w) : pair(Dl[e / 4].x, Dl[e / 4].y);
        const float2 g = apart(mul2(pair(pv[e], pv[e + 1]), add2(pair(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1])), nd)));
        dv[e] = __float_as_uint(g.x);
        dv[e + 1] = __float_as_uint(g.y);
      }
      if (test) {  // a masked place may hold NaN
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (pv[e] == 0.f) dv[e] = 0u;
      }
#pragma unroll
      for (int h32 = 0; h32 < 2; ++h32) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          pk[i] = pack_bf16x2(__uint_as_float(dv[h32 * 32 + 2 * i]), __uint_as_float(dv[h32 * 32 + 2 * i + 1]));
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
          if (p.split > 1) {
            float* part = p.part + c * 16 +
                          (((static_cast<int64_t>(sp) * 2 + which) * p.B * p.nkv + bk) * p.padded + key) * p.d;
            const int m = min(16, p.d - c * 16);
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              if (i < m)
                *reinterpret_cast<float4*>(part + i) =
                    n == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                           : make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]),
                                         __uint_as_float(v[i + 3]));
          } else if (key < p.S) {
            if (n == 0) zero16(out + c * 16, p.d - c * 16);
            else store16(out + c * 16, v, which ? p.scale : 1.f, p.d - c * 16);
          }
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
          mbar_arrive_expect_tx(&s.kv_full, 2 * tile_bytes);
          load(s.k, &tm_k, &s.kv_full, kvh, jt);
          load(s.v, &tm_v, &s.kv_full, kvh, jt);
        }
        bool ok = true;
        int nq = 0, nd = 0;
        for (int it = 0; it < n && ok; ++it) {
          const int st = it % Q_STAGES, ph = (it / Q_STAGES) & 1;
          const int h = head0 + it / count, entry = s.list[it % count], i = entry & 0x3fff;
          ok = wait_warp(&s.q_empty[st], ph ^ 1, p.err, 351);
          if (!ok) break;
          if (lane == 0) {
            const int64_t stat = (static_cast<int64_t>(b) * p.nq + h) * p.padded + i * TILE;
            mbar_arrive_expect_tx(&s.q_full[st], tile_bytes + TILE * 16);
            load(s.q[st], &tm_q, &s.q_full[st], h, i);
            bulk_load(s.rows[st], rows + i * TILE, TILE * 8, &s.q_full[st]);
            bulk_load(s.neg_lse2[st], p.neg_lse2 + stat, TILE * 4, &s.q_full[st]);
            bulk_load(s.neg_delta[st], p.neg_delta + stat, TILE * 4, &s.q_full[st]);
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
      if (n > 0) {
        // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
        const uint32_t leader = elect_one();
        const uint32_t idS = make_idesc_bf16(128, TILE, false, false);
        const uint32_t idKV = make_idesc_bf16(128, p.ksteps * 16, false, true);
        int n_clean = 0;
        auto gather = [&](uint32_t dst, uint32_t a, uint32_t bb, bool more) {
          // queries 0..63 in columns 0..31, 64..127 in 64..95
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)
            mma_ts(dst, a + (kk >> 2) * 64 + (kk & 3) * 8, make_sw128_desc(bb + kk * 2048, 128 * 128, 1024), idKV,
                        (more || kk > 0) ? 1u : 0u, leader);
        };
        auto issue_s = [&](int it) -> bool {
          const int st = it % Q_STAGES;
          if (!wait_warp(&s.q_full[st], (it / Q_STAGES) & 1, p.err, 355)) return false;
          if ((s.list[it % count] & 0x8000) && !wait_warp(&s.clean, n_clean++ & 1, p.err, 356)) return false;
          tc_fence_after();
          mma_tiles(tS, smem_u32(s.k), smem_u32(s.q[st]), idS, p.ksteps, leader);
          commit(&s.s_full, leader);
          return true;
        };
        auto issue_dp = [&](int it) -> bool {
          const int st = it % Q_STAGES;
          if (!wait_warp(&s.do_full[st], (it / Q_STAGES) & 1, p.err, 357)) return false;
          tc_fence_after();
          mma_tiles(tdP, smem_u32(s.v), smem_u32(s.dout[st]), idS, p.ksteps, leader);
          commit(&s.dp_full, leader);
          return true;
        };
        bool ok = wait_warp(&s.kv_full, 0, p.err, 358) && issue_s(0) && issue_dp(0);
        for (int it = 0; ok && it < n; ++it) {
          const int st = it % Q_STAGES;
          ok = wait_warp(&s.p_full, it & 1, p.err, 359);
          if (!ok) break;
          tc_fence_after();
          gather(tdV, tS, smem_u32(s.dout[st]), it > 0);
          commit(&s.do_empty[st], leader);
          if (it + 1 < n) ok = issue_s(it + 1);
          ok = ok && wait_warp(&s.ds_full, it & 1, p.err, 360);
          if (!ok) break;
          tc_fence_after();
          gather(tdK, tdP, smem_u32(s.q[st]), it > 0);
          commit(&s.q_empty[st], leader);
          if (it + 1 < n) ok = issue_dp(it + 1);
        }
        commit(ok ? &s.done : &s.drained, leader);
        if (!ok) wait_warp(&s.drained, 0, p.err, 361);
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

// Sums of the blocks that shared a group's heads, in order; 8 values of a row of dv or dk per thread.
__global__ void __launch_bounds__(256) join_kernel(const BwdParams p) {
  const int units = p.d / 8;
  const int64_t per = static_cast<int64_t>(p.B) * p.nkv * p.padded * units;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= 2 * per) return;
  const int which = i >= per;
  const int64_t j = which ? i - per : i;
  const int64_t row = j / units;
  const int key = static_cast<int>(row % p.padded);
  if (key >= p.S) return;
  const int bk = static_cast<int>(row / p.padded), c = static_cast<int>(j % units) * 8;
  uint32_t v[16];
  float acc[8] = {};
  for (int sp = 0; sp < p.split; ++sp) {
    const float4* part = reinterpret_cast<const float4*>(
        p.part + (((static_cast<int64_t>(sp) * 2 + which) * p.B * p.nkv + bk) * p.padded + key) * p.d + c);
    const float4 x = part[0], y = part[1];
    acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
    acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = k < 8 ? __float_as_uint(acc[k]) : 0u;
  store16(at(which ? p.dk : p.dv, bk / p.nkv, key, bk % p.nkv) + c, v, which ? p.scale : 1.f, 8);
}

cudaError_t launch_dkv(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                       const BwdParams& p, bool cap, bool bias, cudaStream_t st) {
  static_assert(sizeof(DkvSmem) + 1024 <= 232448, "shared memory");
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = dkv_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(DkvSmem) + 1024, cfg);
    kernel<<<dim3(p.B * p.nkv * p.split, p.ntiles), NTHREADS, sizeof(DkvSmem) + 1024, st>>>(tq, tk, tv, td, p);
  });
  if (p.split > 1) {
    const int64_t n = static_cast<int64_t>(p.B) * p.nkv * p.padded * (p.d / 8) * 2;
    join_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

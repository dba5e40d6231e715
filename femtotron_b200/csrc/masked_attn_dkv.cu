// Attention over a mask of intervals: the gradients of the keys and values (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ backward: dk, dv
// One block per 128 keys of a key head; the query tiles that see any of them go past, 64 queries at a time, for every
// query head of the group (or the block's share of them), so dk and dv are complete in TMEM.  S^T = K Q^T and
// dP^T = V dO^T (rows are keys); P^T and dS^T go over them as bf16 pairs and are the left operands of dv += P^T dO and
// dk += dS^T Q.  S and dP have two buffers each, so the products of one step run under the exponentials of another:
// with one buffer of 128 queries the two took turns (3320 clocks per 128 x 128 block).
// Measured (32 heads over 8, d = 128): 8192 tokens in documents 224 us, 16384 tokens with 8 heads over 1 in 831 us (four products:
// 0.80 of the GEMM rate).  Bound by the reads of shared memory of products with 64 columns.  10 warps on four schedulers leave 168
// registers each; 146 are used, all with a cap (dp - delta before the exponentials; after
// them the loop spilled, now only where both forms of the cap are worked out).
constexpr int Q_STAGES = 4;

struct DkvSmem {
  __nv_bfloat16 k[TILE * HEAD], v[TILE * HEAD], q[Q_STAGES][STEP * HEAD], dout[Q_STAGES][STEP * HEAD];
  int2 rows[Q_STAGES][STEP];
  float neg_lse2[Q_STAGES][STEP], neg_delta[Q_STAGES][STEP];
  uint64_t kv_full, full[Q_STAGES], empty[Q_STAGES], landed;
  uint64_t sp_full[2], pd_full[2], done, drained;
  uint16_t list[MAX_TILES];  // query tiles that see a key of this block; bit 14: elements need a test, 15: dead rows
  int count;
  uint32_t tmem_base;
};

template <bool CAP, bool ALIBI>
__global__ void __launch_bounds__(NTHREADS, 1)
    dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
               const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
               const __grid_constant__ BwdParams p) {
  asm volatile("griddepcontrol.launch_dependents;");  // dq may begin where this kernel leaves SMs idle
  using Sm = DkvSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has
  const int bk = blockIdx.x / p.split, sp = blockIdx.x % p.split, b = bk / p.nkv;
  // the key tiles that the most queries see first, so that the last blocks are short (8192 tokens in documents, 32 heads over
  // 8, 3.5 blocks per SM: 240 -> 224 us; the other kernels have more and shorter blocks and gain nothing)
  const int jt = uniform(min(max(p.order[b * p.tiles_stride + blockIdx.y], 0), p.ntiles - 1));
  const int kvh = bk % p.nkv, heads = p.group / p.split, head0 = kvh * p.group + sp * heads;
  const int k0 = jt * TILE;
  const int2* rows = p.rows + b * p.rows_stride;
  const int4* tiles = p.tiles + b * p.tiles_stride;

  if (threadIdx.x == 0) {
    mbar_init(&s.kv_full, 1);
    for (int i = 0; i < Q_STAGES; ++i) mbar_init(&s.full[i], 1), mbar_init(&s.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s.sp_full[i], 1), mbar_init(&s.pd_full[i], COMPUTE_WARPS);
    mbar_init(&s.landed, 1);
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
  auto tS = [](int buf) -> uint32_t { return tmem + static_cast<uint32_t>(buf) * 64u; };
  auto tdP = [](int buf) -> uint32_t { return tmem + 128u + static_cast<uint32_t>(buf) * 64u; };
  constexpr uint32_t tdV = tmem + 256, tdK = tmem + 384;
  const int count = uniform(s.count), n = count * heads * (TILE / STEP);  // steps: the halves of the tiles, head by head

  if (warp < COMPUTE_WARPS) {
    // two warps per TMEM lane quadrant (32 keys), 32 of the 64 queries each
    const int quad = warp & 3, half = warp >> 2;
    const int key = k0 + quad * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint64_t mul = pair(unit<CAP>(p), unit<CAP>(p));
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const int st = it % Q_STAGES, buf = it & 1, tile = it / 2, entry = s.list[tile % count];
      const int q0 = (entry & 0x3fff) * TILE + (it & 1) * STEP + half * 32;
      const bool test = entry & 0x4000;
      const float slope2 = ALIBI ? p.slopes[head0 + tile / count] * kLog2e : 0.f;
      const float far = static_cast<float>(key - q0);
      const uint32_t ts = tS(buf) + lane_off + half * 32, td = tdP(buf) + lane_off + half * 32;
      // the statistics of the queries come into registers while S is still in work: between the products'
      // operand reads, shared memory answers late
      ok = wait_warp(&s.full[st], (it / Q_STAGES) & 1, p.err, 365);
      if (!ok) break;
      float4 L[8], Dl[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) L[i] = reinterpret_cast<const float4*>(s.neg_lse2[st] + half * 32)[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) Dl[i] = reinterpret_cast<const float4*>(s.neg_delta[st] + half * 32)[i];
      ok = wait_warp(&s.sp_full[buf], (it >> 1) & 1, p.err, 362);
      if (!ok) break;
      tc_fence_after();
      uint32_t sv[32], dv[32], pk[16];
      tmem_ld_32x32b_x32(ts, sv);
      tmem_ld_32x32b_x32(td, dv);
      tmem_wait_ld();
      float keep[CAP ? 32 : 1];
      cap_scores<CAP, CAP>(sv, keep, p);
      // (dp - delta) and the slope of the cap first: their registers are free before the exponentials
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const uint64_t nd = e & 2 ? pair(Dl[e / 4].z, Dl[e / 4].w) : pair(Dl[e / 4].x, Dl[e / 4].y);
        uint64_t g = add2(pair(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1])), nd);
        if (CAP) g = mul2(g, pair(keep[CAP ? e : 0], keep[CAP ? e + 1 : 0]));
        const float2 y = apart(g);
        dv[e] = __float_as_uint(y.x);
        dv[e + 1] = __float_as_uint(y.y);
      }
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const uint64_t l = e & 2 ? pair(L[e / 4].z, L[e / 4].w) : pair(L[e / 4].x, L[e / 4].y);
        const uint64_t x = pair(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
        float2 y = apart(fma2(x, mul, l));
        if (ALIBI) y.x = fmaf(-slope2, fabsf(far - e), y.x), y.y = fmaf(-slope2, fabsf(far - (e + 1)), y.y);
        y = exp2_of<CAP>(y, e / 2);
        sv[e] = __float_as_uint(y.x);
        sv[e + 1] = __float_as_uint(y.y);
      }
      if (test) {
        const int4* R = reinterpret_cast<const int4*>(s.rows[st] + half * 32);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const int4 two = R[e / 2];  // rows e and e + 1: (lo, hi, lo, hi)
          // a masked place may hold NaN in dP and in the cap's slope too
          if (key < two.x || key >= two.y) sv[e] = 0u, dv[e] = 0u;
          if (key < two.z || key >= two.w) sv[e + 1] = 0u, dv[e + 1] = 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1]));
      tmem_st_32x32b_x16(ts, pk);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 g = apart(mul2(pair(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])),
                                    pair(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1]))));
        pk[e / 2] = pack_bf16x2(g.x, g.y);
      }
      tmem_st_32x32b_x16(td, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.pd_full[buf]);
    }
    if (n > 0 && ok) ok = wait_warp(&s.done, 0, p.err, 364);
    if (ok) {
      tc_fence_after();
      // the keys and values are no longer needed: dk and dv take their places on the way out
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        for (int c = half; c < p.ksteps; c += 2) {
          uint32_t v[16] = {};
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
                *reinterpret_cast<float4*>(part + i) = make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]),
                                                                   __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
          } else {
            stage16(which ? s.k : s.v, quad * 32 + lane, c, v, which ? p.scale : 1.f);
          }
        }
      }
      fence_proxy_async_smem();
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the compute warps, also after a wait that ran out
    if (ok && p.split == 1 && threadIdx.x == 0) {
      tma_store_tile(&tm_dv, s.v, chunks, kvh, k0, b);
      tma_store_tile(&tm_dk, s.k, chunks, kvh, k0, b);
      tma_store_wait_read();
    }
  } else if (warp == PRODUCER_WARP) {
    if (n > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&s.kv_full, 2 * chunks * PIECE);
        for (int c = 0; c < chunks; ++c) {
          tma_load_4d(s.k + c * TILE * 64, &tm_k, &s.kv_full, c * 64, kvh, k0, b);
          tma_load_4d(s.v + c * TILE * 64, &tm_v, &s.kv_full, c * 64, kvh, k0, b);
        }
      }
      bool ok = true;
      int got = 0, n_dead = 0;
      for (int it = 0; it < n && ok; ++it) {
        const int st = it % Q_STAGES, ph = (it / Q_STAGES) & 1, tile = it / 2, entry = s.list[tile % count];
        const int h = head0 + tile / count, q0 = (entry & 0x3fff) * TILE + (it & 1) * STEP;
        ok = wait_warp(&s.empty[st], ph ^ 1, p.err, 351);
        if (!ok) break;
        // rows that see nothing are zeroed before the products sum over them
        const bool dead = entry & 0x8000;
        uint64_t* bar = dead ? &s.landed : &s.full[st];
        if (lane == 0) {
          const int64_t stat = (static_cast<int64_t>(b) * p.nq + h) * p.padded + q0;
          mbar_arrive_expect_tx(bar, 2 * chunks * STEP_PIECE + STEP * 16);
          for (int c = 0; c < chunks; ++c) {
            tma_load_4d(s.q[st] + c * STEP * 64, &tm_q, bar, c * 64, h, q0, b);
            tma_load_4d(s.dout[st] + c * STEP * 64, &tm_do, bar, c * 64, h, q0, b);
          }
          bulk_load(s.rows[st], rows + q0, STEP * 8, bar);
          bulk_load(s.neg_lse2[st], p.neg_lse2 + stat, STEP * 4, bar);
          bulk_load(s.neg_delta[st], p.neg_delta + stat, STEP * 4, bar);
        }
        ++got;
        __syncwarp();
        if (dead) {
          ok = wait_warp(&s.landed, n_dead++ & 1, p.err, 353);
          zero_dead_rows(s.q[st], chunks, rows + q0, lane);
          zero_dead_rows(s.dout[st], chunks, rows + q0, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.full[st]);
        }
      }
      // the copies have landed before the block may leave, also after a wait that ran out
      wait_phase(&s.kv_full, 0, p.err, 354);
      for (int i = max(0, got - Q_STAGES); i < got; ++i) wait_phase(&s.full[i % Q_STAGES], (i / Q_STAGES) & 1, p.err, 354);
    }
  } else if (n > 0) {
    // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
    const uint32_t leader = elect_one();
    const uint32_t idKV = make_idesc_bf16(TILE, p.ksteps * 16, false, true);
    const uint32_t ka = desc_low(smem_u32(s.k), 16), va = desc_low(smem_u32(s.v), 16);
    const uint32_t qa = desc_low(smem_u32(s.q[0]), 16), da = desc_low(smem_u32(s.dout[0]), 16);
    const uint32_t qt = desc_low(smem_u32(s.q[0]), STEP_PIECE), dt = desc_low(smem_u32(s.dout[0]), STEP_PIECE);
    constexpr uint32_t stage = STEP * HEAD * 2 >> 4;
    auto issue = [&](int it) -> bool {
      const int st = it % Q_STAGES, buf = it & 1;
      if (!wait_warp(&s.full[st], (it / Q_STAGES) & 1, p.err, 355)) return false;
      tc_fence_after();
      mma_scores(tS(buf), ka, qa + st * stage, p.ksteps, leader);
      mma_scores(tdP(buf), va, da + st * stage, p.ksteps, leader);
      commit(&s.sp_full[buf], leader);
      return true;
    };
    bool ok = wait_warp(&s.kv_full, 0, p.err, 358) && issue(0) && issue(1);
    for (int it = 0; ok && it < n; ++it) {
      const int st = it % Q_STAGES, buf = it & 1;
      ok = wait_warp(&s.pd_full[buf], (it >> 1) & 1, p.err, 359);
      if (!ok) break;
      tc_fence_after();
      // queries 0..31 in columns 0..15 of the buffer, 32..63 in 32..47
      mma_values(tdV, tS(buf), 32, dt + st * stage, idKV, it > 0, leader);
      mma_values(tdK, tdP(buf), 32, qt + st * stage, idKV, it > 0, leader);
      commit(&s.empty[st], leader);
      if (it + 2 < n) ok = issue(it + 2);
    }
    commit(ok ? &s.done : &s.drained, leader);
    if (!ok) wait_warp(&s.drained, 0, p.err, 361);
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
  float acc[8] = {};
  for (int sp = 0; sp < p.split; ++sp) {
    const float4* part = reinterpret_cast<const float4*>(
        p.part + (((static_cast<int64_t>(sp) * 2 + which) * p.B * p.nkv + bk) * p.padded + key) * p.d + c);
    const float4 x = part[0], y = part[1];
    acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
    acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
  }
  const float f = which ? p.scale : 1.f;
  *reinterpret_cast<uint4*>(at(which ? p.dk : p.dv, bk / p.nkv, key, bk % p.nkv) + c) =
      make_uint4(pack_bf16x2(acc[0] * f, acc[1] * f), pack_bf16x2(acc[2] * f, acc[3] * f),
                 pack_bf16x2(acc[4] * f, acc[5] * f), pack_bf16x2(acc[6] * f, acc[7] * f));
}

cudaError_t launch_dkv(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& td,
                       const CUtensorMap& tdk, const CUtensorMap& tdv, const BwdParams& p, bool cap, bool bias,
                       cudaStream_t st) {
  static_assert(sizeof(DkvSmem) + 1024 <= 232448, "shared memory");
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = dkv_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(DkvSmem) + 1024, cfg);
    kernel<<<dim3(p.B * p.nkv * p.split, p.ntiles), NTHREADS, sizeof(DkvSmem) + 1024, st>>>(tq, tk, tv, td, tdk, tdv, p);
  });
  return cudaGetLastError();
}

cudaError_t launch_join(const BwdParams& p, cudaStream_t st) {
  const int64_t n = static_cast<int64_t>(p.B) * p.nkv * p.padded * (p.d / 8) * 2;
  join_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

// Attention over a mask of intervals: the mask and the forward pass (masked_attn.h).
#include "masked_attn.cuh"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ the mask
// One block per sequence, 8192 tokens at a time, eight neighbours per thread.  A document is a run of equal numbers; it
// begins at i = 0 and where the number changes (negative numbers: padding).  Forward: the running maximum of the
// beginnings, and of the places that are not marked as prefix (a row leads when there is none in its document so
// far).  Backward: the running minimum of the places where a document begins or a mark is missing, which ends the
// interval of a leading row.  Bound by latency: a thread's tokens are loaded together, before anything depends on
// them (8192 tokens: 25 us with a load per question, 12 us so, and 1 us for the order of the tiles; the sequences of a batch
// run beside each other).
constexpr int MASK_THREADS = 1024, PER = 8;

// The largest v of the threads before this one (AFTER: behind it; `none` where there are none), and of all in `total`.
template <bool AFTER>
__device__ __forceinline__ int block_scan_max(int v, int none, int* warps, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto from = [](int x, int o) { return AFTER ? __shfl_down_sync(0xffffffff, x, o) : __shfl_up_sync(0xffffffff, x, o); };
  const int edge = AFTER ? 31 - lane : lane;  // lanes on the side that is looked at
  auto scan = [&](int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = from(x, o);
      if (edge >= o) x = max(x, u);
    }
    return x;
  };
  v = scan(v);
  int beside = from(v, 1);
  if (edge == 0) beside = none;
  __syncthreads();
  if (edge == 31) warps[w] = v;
  __syncthreads();
  // every warp scans the 32 totals by itself
  const int t = scan(warps[lane]);
  total = __shfl_sync(0xffffffff, t, AFTER ? 0 : 31);
  const int ahead = __shfl_sync(0xffffffff, t, AFTER ? min(w + 1, 31) : max(w - 1, 0));
  return (AFTER ? w < 31 : w > 0) ? max(beside, ahead) : beside;
}

// What the rows i0 ... i0 + 7 are: does a document begin, is there no mark, is it padding (bits of the result)
template <typename T>
struct Tokens {
  uint32_t begins, plain, dead;
  __device__ __forceinline__ Tokens(const MaskArgs& a, int b, int i0) {
    T d[PER + 1];
    bool m[PER];
    const T* docs = a.docs ? static_cast<const T*>(a.docs) + b * a.docs_stride : nullptr;
    const bool* marks = a.marks ? a.marks + b * a.marks_stride : nullptr;
#pragma unroll
    for (int e = 0; e <= PER; ++e) d[e] = docs ? docs[min(max(i0 + e - 1, 0), a.S - 1)] : 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) m[e] = marks ? marks[min(i0 + e, a.S - 1)] : false;
    begins = plain = dead = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      begins |= static_cast<uint32_t>(d[e + 1] != d[e] || i0 + e == 0) << e;
      plain |= static_cast<uint32_t>(!m[e]) << e;
      dead |= static_cast<uint32_t>(d[e + 1] < 0 || i0 + e >= a.S) << e;
    }
  }
};

// Eight rows, two per access; padded is a multiple of eight
__device__ __forceinline__ void put_rows(int2* rows, int i0, int padded, const int2 (&r)[PER]) {
  if (i0 >= padded) return;
#pragma unroll
  for (int e = 0; e < PER; e += 2)
    reinterpret_cast<int4*>(rows + i0)[e / 2] = make_int4(r[e].x, r[e].y, r[e + 1].x, r[e + 1].y);
}
__device__ __forceinline__ void get_rows(const int2* rows, int i0, int padded, int2 (&r)[PER]) {
#pragma unroll
  for (int e = 0; e < PER; e += 2) {
    const int4 two = i0 < padded ? reinterpret_cast<const int4*>(rows + i0)[e / 2] : make_int4(0, 0, 0, 0);
    r[e] = make_int2(two.x, two.y);
    r[e + 1] = make_int2(two.z, two.w);
  }
}

template <typename T>
__global__ void __launch_bounds__(MASK_THREADS) mask_kernel(const MaskArgs a) {
  __shared__ int warps[32];
  const int b = blockIdx.x, S = a.S;
  int2* rows = a.rows + static_cast<int64_t>(b) * a.padded;
  int4* tiles = a.tiles + static_cast<int64_t>(b) * (a.padded / TILE);
  constexpr int chunk = MASK_THREADS * PER;
  int carry_first = -1, carry_plain = -1;
  for (int c0 = 0; c0 < S; c0 += chunk) {
    const int i0 = c0 + threadIdx.x * PER;
    const Tokens<T> k(a, b, i0);
    const uint32_t in = i0 >= S ? 0u : i0 + PER <= S ? 0xffu : (1u << (S - i0)) - 1;
    const uint32_t bg = k.begins & in, pl = k.plain & in;
    int all_f, all_u;
    int f = max(block_scan_max<false>(bg ? i0 + 31 - __clz(bg) : -1, -1, warps, all_f), carry_first);
    int u = max(block_scan_max<false>(pl ? i0 + 31 - __clz(pl) : -1, -1, warps, all_u), carry_plain);
    int2 r[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (bg >> e & 1) f = i0 + e;
      if (pl >> e & 1) u = i0 + e;
      r[e] = make_int2(f, u < f);  // .y: does the row lead
    }
    put_rows(rows, i0, a.padded, r);
    carry_first = max(carry_first, all_f);
    carry_plain = max(carry_plain, all_u);
  }
  // backward: the largest of the negative places of the threads behind; each thread reads the rows that it wrote
  int carry = -S;
  for (int c0 = (a.padded - 1) / chunk * chunk; c0 >= 0; c0 -= chunk) {
    const int i0 = c0 + threadIdx.x * PER;
    const Tokens<T> k(a, b, i0);
    int2 r[PER];
    get_rows(rows, i0, a.padded, r);
    const uint32_t in = i0 >= S ? 0u : i0 + PER <= S ? 0xffu : (1u << (S - i0)) - 1;
    const uint32_t stops = (k.begins | (a.causal && a.marks ? k.plain : 0u)) & in;
    int all;
    int next = max(block_scan_max<true>(stops ? -(i0 + __ffs(stops) - 1) : -kNever, -kNever, warps, all), carry);
    int4 t = make_int4(kNever, 0, kNever, 0);
#pragma unroll
    for (int e = PER - 1; e >= 0; --e) {
      const int i = i0 + e, hi = !a.causal || (a.marks && r[e].y) ? min(S, -next) : i + 1;
      r[e] = k.dead >> e & 1 ? make_int2(kNever, 0) : make_int2(max(r[e].x, i - a.window + 1), min(hi, i + a.window));
      t = make_int4(min(t.x, r[e].x), max(t.y, r[e].x), min(t.z, r[e].y), max(t.w, r[e].y));
      if (stops >> e & 1) next = -i;
    }
    put_rows(rows, i0, a.padded, r);
    // 16 threads of 8 rows each: two tiles per warp
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      t.x = min(t.x, __shfl_xor_sync(0xffffffff, t.x, o));
      t.y = max(t.y, __shfl_xor_sync(0xffffffff, t.y, o));
      t.z = min(t.z, __shfl_xor_sync(0xffffffff, t.z, o));
      t.w = max(t.w, __shfl_xor_sync(0xffffffff, t.w, o));
    }
    if ((threadIdx.x & 15) == 0 && i0 < a.padded) tiles[i0 / TILE] = t;
    carry = max(carry, all);
  }
  // The order of the key tiles, by how many query tiles look at them and then by index; 16 threads per tile count, and
  // count the tiles before it.
  __shared__ int2 reach[MAX_TILES];
  __shared__ int work[MAX_TILES];
  const int n = a.padded / TILE, part = threadIdx.x & 15;
  auto each = [&](auto&& count, auto&& put) {
    for (int i0 = 0; i0 < n; i0 += MASK_THREADS / 16) {
      const int i = i0 + threadIdx.x / 16;
      int c = 0;
      if (i < n)
        for (int j = part; j < n; j += 16) c += count(i, j);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffff, c, o);
      if (part == 0 && i < n) put(i, c);
    }
    __syncthreads();
  };
  __syncthreads();  // the tiles are written
  for (int i = threadIdx.x; i < n; i += MASK_THREADS) reach[i] = make_int2(tiles[i].x, tiles[i].w);
  __syncthreads();
  each([&](int i, int j) { return reach[j].y > i * TILE && reach[j].x < (i + 1) * TILE; },
       [&](int i, int c) { work[i] = c * MAX_TILES + MAX_TILES - 1 - i; });
  each([&](int i, int j) { return work[j] > work[i]; },
       [&](int i, int c) { a.order[static_cast<int64_t>(b) * n + c] = i; });
}

// ------------------------------------------------------------------------------ forward
// One block per 128 queries of a head, two blocks per SM: half of TMEM and 97 KB of shared memory each.  While one waits for
// its products, for the softmax, or on its way in or out (where blocks of short documents spend nearly half of their time:
// 16 000 clocks of 36 000), the other one works.  Warps 0-3 run the softmax, a row per thread.  TMEM: two S of 64 keys, and O;
// the probabilities go over the first half of their S as bf16 pairs.  S of step j + 2 is issued behind the product of step j,
// so one S waits while the other is worked on.  Keys leave their place with their S, values with their product: two of each do.
// Measured (32 heads over 8, d = 128, us; in brackets one block per SM with two query tiles that shared the keys): 8192 tokens
// in documents 159 (171), 2 x 4096 with windows of 1024 and a cap 221 (241), 16384 tokens with 8 heads over 1 448 (497), 0.75
// of the GEMM rate.  What bounds it: the softmax's instructions, 880 clocks per step and tile at 642 of products.  There, 128
// keys per step in halves, all waits before the products and the first keys before the block has met had been slower.
constexpr int FWD_THREADS = 192, FWD_PRODUCER = 4, FWD_MMA = 5;
constexpr int KV_STAGES = 2;  // as many as S: a place for keys is free when the S of its buffer is there
// Growth of a row's running maximum (log2 units) below which the sums stay relative to the old one: the
// probabilities stay under 2^8, which bf16 and the fp32 sums hold as well as values under 1.
constexpr float kRescale = 8.0f;

struct FwdSmem {
  __nv_bfloat16 q[TILE * HEAD], k[KV_STAGES][STEP * HEAD], v[KV_STAGES][STEP * HEAD];
  uint64_t q_full, k_full[KV_STAGES], v_full[KV_STAGES], v_empty[KV_STAGES], landed;
  uint64_t s_full[2], p_full[2], o_done, done, drained;
  uint32_t tmem_base;
};

// Probabilities of 32 keys relative to 2^m from their scores (times `mul`, log2 units), as bf16 pairs; their fp32 sums
// before and after that rounding in `sums` and `used`.  The first are the softmax's (and the backward's); the values'
// weighted sum is divided by the second, so that its weights add up to 1: what rounding does to a weight then counts against
// v_j - o instead of v_j, which where a row has one or two large weights is the difference between an exact and a rounded
// o, and, by way of rowsum(do o), dq.  A score of -inf gives 0.
template <bool CAP, bool TEST>
__device__ __forceinline__ void probs32(const uint32_t* sv, float mul, float m, uint64_t& sums, uint64_t& used,
                                        uint32_t (&pk)[16]) {
  const uint64_t mul2_ = pair(mul, mul), m2 = pair(-m, -m);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t x = fma2(pair(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), mul2_, m2);
    const float2 y0 = apart(x);
    float2 y = exp2_of<CAP>(y0, e);
    if (TEST && on_fma_pipe<CAP>(e)) y = make_float2(y0.x == -INFINITY ? 0.f : y.x, y0.y == -INFINITY ? 0.f : y.y);
    sums = add2(sums, pair(y.x, y.y));
    pk[e] = pack_bf16x2(y.x, y.y);
    used = add2(used, pair(__uint_as_float(pk[e] << 16), __uint_as_float(pk[e] & 0xffff0000u)));
  }
}

// What `mul` times makes the scores of STEP keys, from their raw products (capped, biased), and -inf where they are
// not seen.  TEST: element e is seen when off + e is in [0, width).  Returns the largest.
template <bool CAP, bool ALIBI, bool TEST>
__device__ __forceinline__ float scores(uint32_t (&sv)[STEP], const Common& p, float slope2, float far, int off, int width) {
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  float none[1];
  cap_scores<CAP, false>(sv, none, p);
#pragma unroll
  for (int e = 0; e < STEP; ++e) {
    if (ALIBI) sv[e] = __float_as_uint(fmaf(-slope2, fabsf(far - e), __uint_as_float(sv[e]) * unit<CAP>(p)));
    if (TEST && static_cast<uint32_t>(off + e) >= static_cast<uint32_t>(width)) sv[e] = __float_as_uint(-INFINITY);
  }
#pragma unroll
  for (int e = 0; e < STEP; e += 2)
    asm("max.f32 %0, %0, %1, %2;"
        : "+f"(m4[(e >> 1) & 3])
        : "f"(__uint_as_float(sv[e])), "f"(__uint_as_float(sv[e + 1])));
  return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
}

template <bool CAP, bool ALIBI>
__global__ void __launch_bounds__(FWD_THREADS, 2)
    fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
               const __grid_constant__ CUtensorMap tm_low, const __grid_constant__ FwdParams p) {
  using Sm = FwdSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has

  // late query tiles (the longest rows of a causal mask) first
  const int b = blockIdx.x / p.nq, h = blockIdx.x % p.nq, kvh = h / p.group;
  const int tile = static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y);
  const int2* rows = p.rows + b * p.rows_stride;
  const int4* tiles = p.tiles + b * p.tiles_stride;
  if (threadIdx.x == FWD_PRODUCER * 32) {
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < KV_STAGES; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
    }
    mbar_init(&s.landed, 1);
    mbar_init(&s.o_done, 1);
    mbar_init(&s.done, 1);
    mbar_init(&s.drained, 1);
    fence_barrier_init();
    // the queries are on their way before it is known whether they see anything
    mbar_arrive_expect_tx(&s.q_full, chunks * PIECE);
    for (int c = 0; c < chunks; ++c) tma_load_4d(s.q + c * TILE * 64, &tm_q, &s.q_full, c * 64, h, tile * TILE, b);
    prefetch(tm_k), prefetch(tm_v), prefetch(tm_o);
    if (p.rest) prefetch(tm_low);
  }
  DeadTiles dead_rows(warp == FWD_PRODUCER, tiles, tile - 30, p.ntiles);
  const int4 sum = tiles[tile];
  const int j0 = uniform(sum.w > 0 ? sum.x / STEP : 0);
  const int n = uniform(sum.w > 0 ? (sum.w + STEP - 1) / STEP - j0 : 0);  // steps of 64 keys

  if (warp == FWD_MMA) {
    tmem_alloc(&s.tmem_base, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(s.tmem_base);
  auto tS = [&](int buf) -> uint32_t { return tmem + static_cast<uint32_t>(buf) * 64u; };
  const uint32_t tO = tmem + 128u;

  if (warp < 4) {
    // ------------------------------------------------------------ softmax warps
    const int r = warp * 32 + lane, row = tile * TILE + r;
    const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
    float m_used = -INFINITY, l_run = 0.f, l_used = 0.f;
    bool ok = true;
    int lo = 0, width = 0;
    const int2 lh = rows[row];
    if (lh.y > lh.x) lo = lh.x, width = lh.y - lh.x;
    const float slope2 = ALIBI ? p.slopes[h] * kLog2e : 0.f;
    const float mul = ALIBI ? 1.f : unit<CAP>(p);  // goes into the exponent's FMA
    for (int c = 0; c < n; ++c) {
      const int k0 = (j0 + c) * STEP, buf = c & 1;
      const uint32_t ts = tS(buf) + lane_off;
      ok = wait_warp(&s.s_full[buf], (c >> 1) & 1, p.err, 319);
      if (!ok) break;
      tc_fence_after();
      const bool test = k0 < sum.y || k0 + STEP > sum.z;
      const int off = k0 - lo;                 // element e is seen when off + e is in [0, width)
      const float far = static_cast<float>(row - k0);
      uint32_t sv[STEP];
      tmem_ld_32x32b_x32(ts, *reinterpret_cast<uint32_t(*)[32]>(sv));
      tmem_ld_32x32b_x32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
      tmem_wait_ld();
      const float mx = mul * (test ? scores<CAP, ALIBI, true>(sv, p, slope2, far, off, width)
                                   : scores<CAP, ALIBI, false>(sv, p, slope2, far, off, width));
      const bool need = mx - m_used > kRescale || m_used == -INFINITY;
      const float m_new = need ? fmaxf(m_used, mx) : m_used;
      if (c > 0 && __any_sync(0xffffffffu, need)) {
        // O holds still: the product of the step before is done, the next one waits for this warp.  (S of this step was
        // committed behind the product of step c - 2, so the barrier is at most one phase behind.)
        ok = wait_warp(&s.o_done, (c - 1) & 1, p.err, 320);
        if (!ok) break;
        tc_fence_after();
        const float alpha = m_used == -INFINITY ? 0.f : ex2_approx(m_used - m_new);
        l_run *= alpha;
        l_used *= alpha;
        for (int cc = 0; cc < p.ksteps; ++cc) {
          uint32_t ov[16];
          const uint32_t ta = tO + lane_off + cc * 16;
          tmem_ld_32x32b_x16(ta, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st_32x32b_x16(ta, ov);
        }
      }
      m_used = m_new;
      const float m = m_used == -INFINITY ? 0.f : m_used;  // a row that has seen nothing yet
      uint64_t sums = 0, used = 0;
#pragma unroll
      for (int q = 0; q < STEP / 32; ++q) {
        uint32_t pk[16];
        if (test) probs32<CAP, true>(sv + q * 32, mul, m, sums, used, pk);
        else probs32<CAP, false>(sv + q * 32, mul, m, sums, used, pk);
        tmem_st_32x32b_x16(ts + q * 16, pk);
      }
      tmem_wait_st();
      const float2 two = apart(sums), rounded = apart(used);
      l_run += two.x + two.y;
      l_used += rounded.x + rounded.y;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_full[buf]);
    }
    // o takes the place of the queries (without keys they may still be arriving) and what its rounding leaves out that of
    // the keys
    if (ok) ok = n > 0 ? wait_warp(&s.done, 0, p.err, 321) : wait_warp(&s.q_full, 0, p.err, 322);
    tc_fence_after();
    const bool none = n == 0 || l_run == 0.f;
    const float inv = none ? 0.f : 1.f / l_used;
    if (p.neg_lse2 && ok)
      p.neg_lse2[(static_cast<int64_t>(b) * p.nq + h) * p.padded + row] =
          l_run == 0.f ? -INFINITY : -(m_used + log2f(l_run)) + 0.f * l_used;  // NaN where a score was
    // (the barrier is met also after a wait that ran out)
    const int parts = (p.ksteps + 1) / 2;  // of 32 values
    uint32_t ov[2][32] = {};
    if (n > 0 && ok) tmem_ld_32x32b_x32(tO + lane_off, ov[0]);
#pragma unroll
    for (int c = 0; c < HEAD / 32; ++c) {
      if (c >= parts || !ok) break;
      if (n > 0) {
        tmem_wait_ld();
        if (c + 1 < parts) tmem_ld_32x32b_x32(tO + lane_off + (c + 1) * 32, ov[(c + 1) & 1]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t w[4], rest[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // a sum that is NaN stays one
          const float x = none ? 0.f : __uint_as_float(ov[c & 1][u * 8 + i * 2]) * inv;
          const float y = none ? 0.f : __uint_as_float(ov[c & 1][u * 8 + i * 2 + 1]) * inv;
          w[i] = pack_bf16x2(x, y);
          const float2 r2 = unpack_bf16x2(w[i]);
          rest[i] = pack_bf16x2(x - r2.x, y - r2.y);
        }
        stage8(s.q, r, c * 4 + u, make_uint4(w[0], w[1], w[2], w[3]));
        if (p.rest) stage8(s.k[0], r, c * 4 + u, make_uint4(rest[0], rest[1], rest[2], rest[3]));
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the four warps
    if (ok && threadIdx.x == 0) {
      tma_store_tile(&tm_o, s.q, chunks, h, tile * TILE, b);
      if (p.rest) tma_store_tile(&tm_low, s.k[0], chunks, h, tile * TILE, b);
      tma_store_wait_read();
    }
  } else if (warp == FWD_PRODUCER) {
    // ------------------------------------------------------------ TMA producer
    bool ok = true;
    int got_k = 0, got_v = 0, n_dead = 0;
    for (int c = 0; c < n && ok; ++c) {
      const int st = c % KV_STAGES, ph = (c / KV_STAGES) & 1, k0 = (j0 + c) * STEP;
      // a place for keys is free when their S is done
      if (c >= KV_STAGES) ok = wait_warp(&s.s_full[st], ph ^ 1, p.err, 310);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&s.k_full[st], chunks * STEP_PIECE);
        for (int i = 0; i < chunks; ++i) tma_load_4d(s.k[st] + i * STEP * 64, &tm_k, &s.k_full[st], i * 64, kvh, k0, b);
      }
      ++got_k;
      __syncwarp();
      ok = wait_warp(&s.v_empty[st], ph ^ 1, p.err, 311);
      if (!ok) break;
      // values of rows that see nothing are zeroed before the products may have them
      const bool dead = dead_rows(tiles, (j0 + c) / 2, p.ntiles);
      uint64_t* bar = dead ? &s.landed : &s.v_full[st];
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, chunks * STEP_PIECE);
        for (int i = 0; i < chunks; ++i) tma_load_4d(s.v[st] + i * STEP * 64, &tm_v, bar, i * 64, kvh, k0, b);
      }
      ++got_v;
      __syncwarp();
      if (dead) {
        ok = wait_warp(&s.landed, n_dead++ & 1, p.err, 312);
        zero_dead_rows(s.v[st], chunks, rows + k0, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.v_full[st]);
      }
    }
    // all copies have landed before the block may leave, also after a wait that ran out
    for (int i = max(0, got_k - KV_STAGES); i < got_k; ++i) wait_phase(&s.k_full[i % KV_STAGES], (i / KV_STAGES) & 1, p.err, 313);
    for (int i = max(0, got_v - KV_STAGES); i < got_v; ++i) wait_phase(&s.v_full[i % KV_STAGES], (i / KV_STAGES) & 1, p.err, 313);
    wait_phase(&s.q_full, 0, p.err, 313);
  } else if (n > 0) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
    const uint32_t leader = elect_one();
    const uint32_t idO = make_idesc_bf16(TILE, p.ksteps * 16, false, true);  // P (TMEM) x V (MN-major)
    const uint32_t qa = desc_low(smem_u32(s.q), 16), ka = desc_low(smem_u32(s.k[0]), 16);
    const uint32_t va = desc_low(smem_u32(s.v[0]), STEP_PIECE);
    constexpr uint32_t stage = STEP * HEAD * 2 >> 4;
    bool ok = wait_warp(&s.q_full, 0, p.err, 317);
    auto issue_s = [&](int c, bool ready) {
      if (!ok || c >= n) return;
      ok = ready || wait_warp(&s.k_full[c % KV_STAGES], (c / KV_STAGES) & 1, p.err, 314);
      if (!ok) return;
      tc_fence_after();
      mma_scores(tS(c & 1), qa, ka + (c % KV_STAGES) * stage, p.ksteps, leader);
      commit(&s.s_full[c & 1], leader);
    };
    issue_s(0, false);
    issue_s(1, false);
    for (int c = 0; ok && c < n; ++c) {
      const int st = c % KV_STAGES, ph = (c / KV_STAGES) & 1, buf = c & 1;
      const uint32_t have = over(&s.p_full[buf], (c >> 1) & 1, &s.v_full[st], ph, &s.k_full[(c + 2) % KV_STAGES],
                                 ((c + 2) / KV_STAGES) & 1);
      ok = (have & 2) || wait_warp(&s.v_full[st], ph, p.err, 315);
      ok = ok && ((have & 1) || wait_warp(&s.p_full[buf], (c >> 1) & 1, p.err, 316));
      if (!ok) break;
      tc_fence_after();
      mma_values(tO, tS(buf), 16, va + st * stage, idO, c > 0, leader);
      commit(&s.o_done, leader);
      commit(&s.v_empty[st], leader);
      if (c + 1 == n) commit(&s.done, leader);
      issue_s(c + 2, have & 4);
    }
    if (!ok) {
      commit(&s.drained, leader);
      wait_warp(&s.drained, 0, p.err, 318);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == FWD_MMA) {
    tc_fence_after();
    tmem_dealloc(s.tmem_base, 256);
  }
}

cudaError_t launch_mask(const MaskArgs& a, int batch, cudaStream_t st) {
  if (a.docs64) mask_kernel<int64_t><<<batch, MASK_THREADS, 0, st>>>(a);
  else mask_kernel<int><<<batch, MASK_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,
                       const CUtensorMap& tlow, const FwdParams& p, bool cap, bool bias, cudaStream_t st) {
  static_assert(2 * (sizeof(FwdSmem) + 2048) <= 233472, "shared memory of two blocks");
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = fwd_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(FwdSmem) + 1024, cfg);
    kernel<<<dim3(p.B * p.nq, p.ntiles), FWD_THREADS, sizeof(FwdSmem) + 1024, st>>>(tq, tk, tv, to, tlow, p);
  });
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

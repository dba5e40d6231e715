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
// Two query tiles per block share the key and value tiles of a ring: two heads of a group at the same
// 128 rows where the group has an even number of heads, else 256 rows of one head.  Warps 0-3 and 4-7 each
// run the softmax of one tile, a row per thread.  TMEM: two S of 64 keys and O for each tile; the probabilities
// go over the first half of their S as bf16 pairs.  S of step j+2 is issued behind the product of step j, so one S
// waits while the other is worked on: with one S of 128 keys a tile's softmax (2100 clocks) and its products (512
// each, and 400 until their result is seen) took turns, 3750 clocks for two tiles of 128 keys.
//
// Measured (32 heads over 8, d = 128): 8192 tokens in documents 170 us, of which a block of 20 000 clocks in its steps (1600 per
// step of two tiles) spends another 16 000 on its way in and out: two loads before the first key tile can be asked for (1900),
// that tile and its S (3600), the last product (1900), results (7500: o and its rest are 128 KB on their way to L2), the
// next block (1300).  16384 tokens, 8 heads over 1: 490 us, 0.68 of the GEMM rate.  What bounds it there: the products of 64
// columns, which read 128 bytes of shared memory per clock (48 clocks where the tensor cores need 32).  128 keys per step in
// two halves (8192: 180 -> 190 us), all waits before the products (180 -> 185), rings of their own for K and V (175 -> 179)
// and the first key tiles before the block has met (173 -> 176) were slower.
constexpr int KV_STAGES = 4;
// Growth of a row's running maximum (log2 units) below which the sums stay relative to the old one: the
// probabilities stay under 2^8, which bf16 and the fp32 sums hold as well as values under 1.
constexpr float kRescale = 8.0f;

struct FwdSmem {
  __nv_bfloat16 q[2][TILE * HEAD], k[KV_STAGES][STEP * HEAD], v[KV_STAGES][STEP * HEAD];
  uint64_t q_full, full[KV_STAGES], empty[KV_STAGES], landed;
  uint64_t s_full[2][2], p_full[2][2], o_done[2], done[2], drained;
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
__global__ void __launch_bounds__(NTHREADS, 1)
    fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
               const __grid_constant__ CUtensorMap tm_low, const __grid_constant__ FwdParams p) {
  using Sm = FwdSmem;
  extern __shared__ uint8_t smem_raw[];
  Sm& s = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = p.d > 64 ? 2 : 1;  // pieces of 64 values that a head has

  // late query tiles (the longest rows of a causal mask) first
  const int per = p.pair_heads ? p.nq / 2 : p.nq;
  const int b = blockIdx.x / per, hx = blockIdx.x % per;
  const int yr = static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y);
  const int head0 = p.pair_heads ? 2 * hx : hx, head1 = p.pair_heads ? 2 * hx + 1 : hx;
  const int tile0 = p.pair_heads ? yr : 2 * yr, tile1 = p.pair_heads ? yr : 2 * yr + 1;
  const int4* tiles = p.tiles + b * p.tiles_stride;
  const int kvh = head0 / p.group;
  const int2* rows = p.rows + b * p.rows_stride;
  if (threadIdx.x == PRODUCER_WARP * 32) {
    mbar_init(&s.q_full, 1);
    for (int i = 0; i < KV_STAGES; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.landed, 1);
    mbar_init(&s.drained, 1);
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s.s_full[t][i], 1);
        mbar_init(&s.p_full[t][i], 4);
      }
      mbar_init(&s.o_done[t], 1);
      mbar_init(&s.done[t], 1);
    }
    fence_barrier_init();
    // the queries are on their way before it is known whether they see anything
    const bool two = tile1 < p.ntiles;
    mbar_arrive_expect_tx(&s.q_full, chunks * PIECE * (two ? 2 : 1));
    for (int c = 0; c < chunks; ++c) {
      tma_load_4d(s.q[0] + c * TILE * 64, &tm_q, &s.q_full, c * 64, head0, tile0 * TILE, b);
      if (two) tma_load_4d(s.q[1] + c * TILE * 64, &tm_q, &s.q_full, c * 64, head1, tile1 * TILE, b);
    }
    prefetch(tm_k), prefetch(tm_v), prefetch(tm_o);
    if (p.rest) prefetch(tm_low);
  }
  DeadTiles dead_rows(warp == PRODUCER_WARP, tiles, tile1 - 30, p.ntiles);
  const int4 u0 = tiles[tile0], u1 = tile1 < p.ntiles ? tiles[tile1] : make_int4(kNever, 0, 0, 0);
  // the steps of 64 keys that each tile takes: none, or a run that holds the tile's own keys, so the two runs meet
  int first0 = 0, end0 = 0, first1 = 0, end1 = 0;
  if (u0.w > 0) first0 = u0.x / STEP, end0 = (u0.w + STEP - 1) / STEP;
  if (u1.w > 0) first1 = u1.x / STEP, end1 = (u1.w + STEP - 1) / STEP;
  first0 = uniform(first0), end0 = uniform(end0), first1 = uniform(first1), end1 = uniform(end1);
  const int j0 = first0 == end0 ? first1 : first1 == end1 ? first0 : min(first0, first1);
  const int j1 = max(end0, end1);  // no keys at all: both 0

  if (warp == MMA_WARP) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // where an allocation of all 512 columns begins
  auto tS = [](int t, int buf) -> uint32_t { return tmem + static_cast<uint32_t>(t) * 128u + static_cast<uint32_t>(buf) * 64u; };
  auto tO = [](int t) -> uint32_t { return tmem + 256u + static_cast<uint32_t>(t) * 128u; };

  if (warp < COMPUTE_WARPS) {
    // ------------------------------------------------------------ softmax warps 0..7
    const int t = warp >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    const int tile = t ? tile1 : tile0, h = t ? head1 : head0, begin = t ? first1 : first0;
    const bool real = tile < p.ntiles;
    const int row = tile * TILE + r;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int n = (t ? end1 : end0) - begin;
    float m_used = -INFINITY, l_run = 0.f, l_used = 0.f;
    bool ok = true;
    int lo = 0, width = 0;
    const int4 sum = t ? u1 : u0;
    float slope2 = 0.f;
    if (n > 0) {
      const int2 lh = rows[row];
      if (lh.y > lh.x) lo = lh.x, width = lh.y - lh.x;
      if (ALIBI) slope2 = p.slopes[h] * kLog2e;
    }
    const float mul = ALIBI ? 1.f : unit<CAP>(p);  // goes into the exponent's FMA
    for (int c = 0; c < n; ++c) {
      const int k0 = (begin + c) * STEP, buf = c & 1;
      const uint32_t ts = tS(t, buf) + lane_off;
      ok = wait_warp(&s.s_full[t][buf], (c >> 1) & 1, p.err, 319);
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
        ok = wait_warp(&s.o_done[t], (c - 1) & 1, p.err, 320);
        if (!ok) break;
        tc_fence_after();
        const float alpha = m_used == -INFINITY ? 0.f : ex2_approx(m_used - m_new);
        l_run *= alpha;
        l_used *= alpha;
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
      if (lane == 0) mbar_arrive(&s.p_full[t][buf]);
    }
    if (n > 0 && ok) ok = wait_warp(&s.done[t], 0, p.err, 321);
    // o takes the place of the queries (a tile without keys may still wait for them) and what its rounding leaves out that of
    // keys, which the other tile has to be done with too.
    if (n == 0) ok = wait_warp(&s.q_full, 0, p.err, 322);
    if (p.rest && ok && (t ? end0 > first0 : end1 > first1)) ok = wait_warp(&s.done[t ^ 1], 0, p.err, 323);
    if (real) {
      tc_fence_after();
      const bool none = n == 0 || l_run == 0.f;
      const float inv = none ? 0.f : 1.f / l_used;
      if (p.neg_lse2 && ok)
        p.neg_lse2[(static_cast<int64_t>(b) * p.nq + h) * p.padded + row] =
            l_run == 0.f ? -INFINITY : -(m_used + log2f(l_run)) + 0.f * l_used;  // NaN where a score was
      // (the barrier is met also after a wait that ran out)
      const int parts = (p.ksteps + 1) / 2;  // of 32 values
      uint32_t ov[2][32] = {};
      if (n > 0 && ok) tmem_ld_32x32b_x32(tO(t) + lane_off, ov[0]);
#pragma unroll
      for (int c = 0; c < HEAD / 32; ++c) {
        if (c >= parts || !ok) break;
        if (n > 0) {
          tmem_wait_ld();
          if (c + 1 < parts) tmem_ld_32x32b_x32(tO(t) + lane_off + (c + 1) * 32, ov[(c + 1) & 1]);
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
          stage8(s.q[t], r, c * 4 + u, make_uint4(w[0], w[1], w[2], w[3]));
          if (p.rest) stage8(s.k[2 * t], r, c * 4 + u, make_uint4(rest[0], rest[1], rest[2], rest[3]));
        }
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");  // the four warps of this tile
      if (ok && quad == 0 && lane == 0) {
        tma_store_tile(&tm_o, s.q[t], chunks, h, tile * TILE, b);
        if (p.rest) tma_store_tile(&tm_low, s.k[2 * t], chunks, h, tile * TILE, b);
        tma_store_wait_read();
      }
    }
  } else if (warp == PRODUCER_WARP) {
    // ------------------------------------------------------------ TMA producer
    if (j0 < j1) {
      bool ok = true;
      int got = 0, n_dead = 0;
      for (int j = j0; j < j1 && ok; ++j) {
        const int st = (j - j0) % KV_STAGES, ph = ((j - j0) / KV_STAGES) & 1;
        ok = wait_warp(&s.empty[st], ph ^ 1, p.err, 311);
        if (!ok) break;
        // values of rows that see nothing are zeroed before the products may have them
        const bool dead = dead_rows(tiles, j / 2, p.ntiles);
        uint64_t* bar = dead ? &s.landed : &s.full[st];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, 2 * chunks * STEP_PIECE);
          for (int c = 0; c < chunks; ++c) {
            tma_load_4d(s.k[st] + c * STEP * 64, &tm_k, bar, c * 64, kvh, j * STEP, b);
            tma_load_4d(s.v[st] + c * STEP * 64, &tm_v, bar, c * 64, kvh, j * STEP, b);
          }
        }
        ++got;
        __syncwarp();
        if (dead) {
          ok = wait_warp(&s.landed, n_dead++ & 1, p.err, 312);
          zero_dead_rows(s.v[st], chunks, rows + j * STEP, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.full[st]);
        }
      }
      for (int i = max(0, got - KV_STAGES); i < got; ++i) wait_phase(&s.full[i % KV_STAGES], (i / KV_STAGES) & 1, p.err, 313);
    }
    // (all copies have landed before the block may leave, also after a wait that ran out)
    wait_phase(&s.q_full, 0, p.err, 313);
  } else if (j0 < j1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp goes through the loop, so that descriptors are made in uniform registers; one lane issues.
    const uint32_t leader = elect_one();
    const uint32_t idO = make_idesc_bf16(TILE, p.ksteps * 16, false, true);  // P (TMEM) x V (MN-major)
    const uint32_t qa = desc_low(smem_u32(s.q[0]), 16), ka = desc_low(smem_u32(s.k[0]), 16);
    const uint32_t va = desc_low(smem_u32(s.v[0]), STEP_PIECE);
    constexpr uint32_t stage = STEP * HEAD * 2 >> 4, tile = TILE * HEAD * 2 >> 4;
    bool ok = wait_warp(&s.q_full, 0, p.err, 317);
    auto issue_s = [&](int j, int t, int first, int end) {
      if (first > j || j >= end) return;
      const int buf = (j - first) & 1;
      mma_scores(tS(t, buf), qa + t * tile, ka + ((j - j0) % KV_STAGES) * stage, p.ksteps, leader);
      commit(&s.s_full[t][buf], leader);
    };
    auto arrived = [&](int j) {
      if (j < j1) ok = ok && wait_warp(&s.full[(j - j0) % KV_STAGES], ((j - j0) / KV_STAGES) & 1, p.err, 314);
    };
    auto issue_o = [&](int j, int t, int first, int end, bool ready) {
      if (first > j || j >= end) return;
      const int c = j - first, buf = c & 1;
      ok = ok && (ready || wait_warp(&s.p_full[t][buf], (c >> 1) & 1, p.err, 316));
      if (!ok) return;
      tc_fence_after();
      mma_values(tO(t), tS(t, buf), 16, va + ((j - j0) % KV_STAGES) * stage, idO, c > 0, leader);
      commit(&s.o_done[t], leader);
      if (j + 1 == end) commit(&s.done[t], leader);
    };
    for (int j = j0; j < j0 + 2; ++j) {
      arrived(j);
      if (!ok) break;
      tc_fence_after();
      issue_s(j, 0, first0, min(end0, j1));
      issue_s(j, 1, first1, min(end1, j1));
    }
    for (int j = j0; ok && j < j1; ++j) {
      const int next = j + 2 - j0, c0 = j - first0, c1 = j - first1;
      const uint32_t have = over(&s.full[next % KV_STAGES], (next / KV_STAGES) & 1, &s.p_full[0][c0 & 1], (c0 >> 1) & 1,
                                 &s.p_full[1][c1 & 1], (c1 >> 1) & 1);
      if (!(have & 1)) arrived(j + 2);
      issue_o(j, 0, first0, end0, have & 2);
      if (!ok) break;
      issue_s(j + 2, 0, first0, end0);
      issue_o(j, 1, first1, end1, have & 4);
      if (!ok) break;
      commit(&s.empty[(j - j0) % KV_STAGES], leader);
      issue_s(j + 2, 1, first1, end1);
    }
    if (!ok) {
      commit(&s.drained, leader);
      wait_warp(&s.drained, 0, p.err, 318);
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
  if (a.docs64) mask_kernel<int64_t><<<batch, MASK_THREADS, 0, st>>>(a);
  else mask_kernel<int><<<batch, MASK_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,
                       const CUtensorMap& tlow, const FwdParams& p, bool cap, bool bias, cudaStream_t st) {
  static_assert(sizeof(FwdSmem) + 1024 <= 232448, "shared memory");
  const dim3 grid(p.B * (p.pair_heads ? p.nq / 2 : p.nq), p.pair_heads ? p.ntiles : (p.ntiles + 1) / 2);
  pick(cap, bias, [&](auto CAP, auto BIAS) {
    constexpr auto kernel = fwd_kernel<decltype(CAP)::value, decltype(BIAS)::value>;
    static unsigned long long cfg = 0;
    smem_attr_once(kernel, sizeof(FwdSmem) + 1024, cfg);
    kernel<<<grid, NTHREADS, sizeof(FwdSmem) + 1024, st>>>(tq, tk, tv, to, tlow, p);
  });
  return cudaGetLastError();
}

}  // namespace ma
}  // namespace ft

// Shared device parts of the kernels of masked_attn.h.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "masked_attn.h"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ shared device parts
// A value that all lanes of the warp share, in a form that the compiler knows to be so: what branches and descriptors are
// made of then stays in uniform registers (without it every product of the MMA warp waited for six moves into them: 110
// clocks where the product takes 32 to 64).
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ uint64_t clock_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Wait for a phase of a barrier, two seconds at most; false after that, with `code` in the status word.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = clock_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (clock_ns() - t0 > 2000000000ull) {
      if (err) atomicExch(err, code);
      return false;
    }
  }
}

// The same for a whole warp: all lanes go on or none does.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, wait_phase(bar, parity, err, code));
}

// tcgen05.mma by the lanes where `on` is not 0 (one of the warp).  Operands in shared memory come as the low word of their
// descriptor (address and leading offset), which grows by a constant from product to product; the high word is the
// same for all tiles here (128-byte swizzle, 1024 bytes between groups of 8 rows).  The predicate is the
// instruction's own.  What stands between two products counts: one of 64 columns takes 32 to 48 clocks.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t leading) {
  return ((addr >> 4) & 0x3FFFu) | ((leading >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%1, %6};\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(on), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(on), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}

// Bytes between the two 64-value pieces of a tile of 128 and of STEP rows
constexpr uint32_t PIECE = TILE * 128, STEP_PIECE = STEP * 128;

// dst = A B^T of a tile of 128 rows and one of STEP rows, 16 values of d at a time; a, b: desc_low(tile, 16)
__device__ __forceinline__ void mma_scores(uint32_t dst, uint32_t a, uint32_t b, int ksteps, uint32_t on) {
  constexpr uint32_t idesc = make_idesc_bf16(TILE, STEP, false, false);
#pragma unroll
  for (int kk = 0; kk < HEAD / 16; ++kk) {
    if (kk >= ksteps) break;
    mma_ss(dst, a + (((kk >> 2) * PIECE + (kk & 3) * 32) >> 4), b + (((kk >> 2) * STEP_PIECE + (kk & 3) * 32) >> 4), idesc,
           kk > 0, on);
  }
}

// dst (+)= A B with A in TMEM (bf16 pairs: 16 values in 8 columns, and `jump` columns from one 32 to the next) and the STEP
// rows of B; b: desc_low(tile, STEP_PIECE)
__device__ __forceinline__ void mma_values(uint32_t dst, uint32_t a, int jump, uint32_t b, uint32_t idesc, bool add,
                                           uint32_t on) {
#pragma unroll
  for (int kk = 0; kk < STEP / 16; ++kk)
    mma_ts(dst, a + (kk >> 1) * jump + (kk & 1) * 8, b + (kk * 2048 >> 4), idesc, (add || kk > 0) ? 1u : 0u, on);
}

// Two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 apart(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The larger value, NaN where one is NaN (fmaxf would drop it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x of two values on the FMA pipe, for x below 127.  Cody and Waite's reduction x = n + f: adding 1.5 2^23 rounds
// to the integer n, which is left in the low bits, and f is in [-1/2, 1/2]; 2^f by the cubic that minimises the largest
// relative error there (7.5e-5, found by linear programming over 4001 points; bf16 rounds by 2e-3), n goes into the exponent.
// Below -125 the result is 2^-125; a NaN gives the largest number there is, which bf16 rounds to infinity.
__device__ __forceinline__ float2 exp2_pair(float a, float b) {
  const uint64_t shift = pair(12582912.f, 12582912.f);
  const uint64_t x = pair(max_nan(a, -125.f), max_nan(b, -125.f));
  const uint64_t t = add2(x, shift);
  const uint64_t f = add2(x, fma2(t, pair(-1.f, -1.f), shift));
  uint64_t q = fma2(pair(0.0551716685f, 0.0551716685f), f, pair(0.2426111251f, 0.2426111251f));
  q = fma2(q, f, pair(0.6932609677f, 0.6932609677f));
  q = fma2(q, f, pair(0.9999280572f, 0.9999280572f));
  const float2 qs = apart(q), ts = apart(t);
  // 1.5 2^23 + n has n in its low bits and nothing else in the low nine
  return make_float2(__uint_as_float(__float_as_uint(qs.x) + (__float_as_uint(ts.x) << 23)),
                     __uint_as_float(__float_as_uint(qs.y) + (__float_as_uint(ts.y) << 23)));
}

// Whether each of three phases is over (bits 0 to 2), for a whole warp, without waiting.  The three answers are under way
// together: where products read all that shared memory gives, each takes its time, and the MMA warp asks for all that its
// step needs at once (forward of 16384 tokens, 8 heads, when a block had two query tiles: 495 -> 489 us; no gain in the two
// backward kernels, which ask singly).
// The phase before the one asked for has to be over already: two phases back has the same parity.
__device__ __forceinline__ uint32_t over(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, uint64_t* c, uint32_t pc) {
  uint32_t x, y, z;
  asm volatile(
      "{\n\t.reg .pred p, q, r;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%3], %4;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q, [%5], %6;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 r, [%7], %8;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "selp.u32 %1, 1, 0, q;\n\t"
      "selp.u32 %2, 1, 0, r;\n\t}"
      : "=r"(x), "=r"(y), "=r"(z)
      : "r"(smem_u32(a)), "r"(pa), "r"(smem_u32(b)), "r"(pb), "r"(smem_u32(c)), "r"(pc)
      : "memory");
  return (__all_sync(0xffffffffu, x) ? 1u : 0u) | (__all_sync(0xffffffffu, y) ? 2u : 0u) |
         (__all_sync(0xffffffffu, z) ? 4u : 0u);
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x of the e-th pair of a row.  Every eighth pair runs on the FMA pipe: the special-function unit takes 8 clocks for one
// exponential of a warp and would set the pace alone, the other form takes nine instructions.  (Forward, and dk and dv, of 16384
// tokens, 8 heads over 1: none 460 and 817 us, every eighth 448 and 808, fourth 451 and 818, third 470 and 841.)  With capped
// scores the FMA pipe sets the pace.
template <bool CAP>
__device__ __forceinline__ constexpr bool on_fma_pipe(int e) { return !CAP && e % 8 == 7; }
template <bool CAP>
__device__ __forceinline__ float2 exp2_of(float2 x, int e) {
  return on_fma_pipe<CAP>(e) ? exp2_pair(x.x, x.y) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
}

// Raw products as what an FMA with `unit(p)` turns into scores in log2 units: with the cap tanh(x) (KEEP: `keep` is
// 1 - tanh^2, the slope of the cap), without it the products themselves.  tanh(x) = 1 - 2 / (1 + exp(2x)) costs two
// special-function instructions of 8 clocks each (tanh.approx would be off by 5e-4 of the cap: whole percents of p).
// Products within 0.7 of the cap, as nearly all are, take a polynomial, off by 2e-7 (the other form by 1e-7).  Which form a
// product takes depends on its own value alone, so that a row's bits do not depend on what it cannot see (padding, other
// documents, later tokens) nor on the rows beside it.  A warp whose products are all small, seen or not, is through with
// that; else it works out both where one of its next eight products is large.  (Two rows of 4096 tokens in windows of 1024, 32
// heads over 8, all small: 213, 273, 293 us for forward, dq, and dk and dv, where the other form alone took 288 forward; every
// fourth product large: 393, 393, 444, where a form chosen by the warp took 288, 337, 357.)
template <bool CAP, bool KEEP, int N>
__device__ __forceinline__ void cap_scores(uint32_t (&sv)[N], float (&keep)[KEEP ? N : 1], const Common& p) {
  if (!CAP) return;
  float m[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < N; ++e) m[e & 1] = fmaxf(m[e & 1], fabsf(__uint_as_float(sv[e])));
  uint64_t c[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) c[i] = pair(p.cap_poly[i], p.cap_poly[i]);
  auto near = [&](int from, int to) {
#pragma unroll
    for (int e = from; e < to; e += 2) {
      const uint64_t s = pair(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), u = mul2(s, s);
      const uint64_t t = mul2(fma2(fma2(fma2(fma2(u, c[4], c[3]), u, c[2]), u, c[1]), u, c[0]), s);
      const float2 y = apart(t);
      sv[e] = __float_as_uint(y.x);
      sv[e + 1] = __float_as_uint(y.y);
      if (KEEP) {
        const float2 k = apart(fma2(mul2(t, pair(-1.f, -1.f)), t, pair(1.f, 1.f)));
        keep[KEEP ? e : 0] = k.x;
        keep[KEEP ? e + 1 : 0] = k.y;
      }
    }
  };
  if (__all_sync(0xffffffffu, fmaxf(m[0], m[1]) <= p.cap_small)) {
    near(0, N);
    return;
  }
  constexpr int G = 8;  // (groups of two: 428, 467, 524 us, of four: 408, 401, 457; of 16 spill more)
#pragma unroll
  for (int g = 0; g < N; g += G) {
    float far[G];
    bool any = false;
#pragma unroll
    for (int e = 0; e < G; ++e) far[e] = __uint_as_float(sv[g + e]), any = any || !(fabsf(far[e]) <= p.cap_small);
    near(g, g + G);
    if (__any_sync(0xffffffffu, any)) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float r = rcp_approx(1.f + ex2_approx(far[e] * p.cap_in));
        if (!(fabsf(far[e]) <= p.cap_small)) {
          sv[g + e] = __float_as_uint(fmaf(-2.f, r, 1.f));
          if (KEEP) keep[KEEP ? g + e : 0] = 4.f * r * (1.f - r);
        }
      }
    }
  }
}
template <bool CAP>
__device__ __forceinline__ float unit(const Common& p) { return CAP ? p.cap_out : p.scale_log2; }

// Zero the rows that see nothing of a tile of STEP rows (`chunks` pieces of 128 bytes a row); one warp.  The swizzle
// permutes within a row's 128 bytes only.
__device__ __forceinline__ void zero_dead_rows(void* tile, int chunks, const int2* rows, int lane) {
  for (int r = lane; r < STEP; r += 32)
    if (rows[r].y == 0)
      for (int c = 0; c < chunks; ++c) {
        uint4* to = reinterpret_cast<uint4*>(static_cast<uint8_t*>(tile) + c * STEP_PIECE + r * 128);
#pragma unroll
        for (int u = 0; u < 8; ++u) to[u] = make_uint4(0, 0, 0, 0);
      }
}

// Which of 32 tiles hold rows that see nothing, for one warp.  The first 32 are asked for before it is known which of them are
// needed (one latency instead of two); what lies elsewhere follows when the walk gets there.
struct DeadTiles {
  int base;
  uint32_t bits;
  __device__ __forceinline__ DeadTiles(bool here, const int4* tiles, int first, int ntiles) : base(0), bits(0) {
    if (here) look(tiles, max(first, 0), ntiles);
  }
  __device__ __forceinline__ void look(const int4* tiles, int first, int ntiles) {
    base = first;
    const int t = first + (threadIdx.x & 31);
    bits = __ballot_sync(0xffffffff, t < ntiles && tiles[t].z == 0);
  }
  __device__ __forceinline__ bool operator()(const int4* tiles, int t, int ntiles) {
    if (t < base || t >= base + 32) look(tiles, t, ntiles);
    return bits >> (t - base) & 1;
  }
};
__device__ __forceinline__ void prefetch(const CUtensorMap& map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
}

// Results leave through shared memory and TMA: a thread has a row of a tile, and 32 rows of 16 bytes each, kilobytes apart, are
// the slowest way to memory (forward pass of 8192 tokens 180 -> 169 us).  The tile is laid
// out as it would have been loaded; rows behind the last token and values behind d are not written.
__device__ __forceinline__ void stage8(void* tile, int r, int unit, uint4 v) {  // values 8 unit ... 8 unit + 7 of row r
  *reinterpret_cast<uint4*>(static_cast<uint8_t*>(tile) + (unit >> 3) * PIECE + r * 128 + (((unit & 7) ^ (r & 7)) * 16)) = v;
}
__device__ __forceinline__ void stage16(void* tile, int r, int c, const uint32_t* v, float f) {
  auto p = [&](int i) { return pack_bf16x2(__uint_as_float(v[i]) * f, __uint_as_float(v[i + 1]) * f); };
  stage8(tile, r, 2 * c, make_uint4(p(0), p(2), p(4), p(6)));
  stage8(tile, r, 2 * c + 1, make_uint4(p(8), p(10), p(12), p(14)));
}
__device__ __forceinline__ void tma_store_tile(const CUtensorMap* map, const void* tile, int chunks, int head, int row, int b) {
  for (int c = 0; c < chunks; ++c)
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(static_cast<const uint8_t*>(tile) + c * PIECE)), "r"(c * 64), "r"(head), "r"(row), "r"(b)
                 : "memory");
  tma_store_commit();
}

__device__ __forceinline__ __nv_bfloat16* at(const Out& x, int b, int s, int h) {
  return static_cast<__nv_bfloat16*>(x.p) + b * x.batch + s * x.token + h * x.head;
}

// The kernel of capped or plain scores, with or without the bias.
template <class F>
void pick(bool cap, bool bias, F&& go) {
  if (cap) bias ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
  else bias ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
}

}  // namespace ma
}  // namespace ft

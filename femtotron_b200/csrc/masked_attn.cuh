// Shared device parts of the kernels of masked_attn.h.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "masked_attn.h"

namespace ft {
namespace ma {

// ------------------------------------------------------------------------------ shared device parts
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

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A raw product s as a score in log2 units.  tanh(x) = 1 - 2 / (1 + exp(2x)): two special-function
// instructions, off by 1e-7 in all (tanh.approx would be 5e-4 of the cap: whole percents of p).
// `keep` is 1 - tanh^2, the slope of the cap.
template <bool CAP, bool ALIBI>
__device__ __forceinline__ float score(float s, const Common& p, float slope2, float dist, float& keep) {
  float y;
  if (CAP) {
    const float r = rcp_approx(1.f + ex2_approx(s * p.cap_in));
    y = fmaf(-2.f * p.cap_out, r, p.cap_out);
    keep = 4.f * r * (1.f - r);
  } else {
    y = s * p.scale_log2;
    keep = 1.f;
  }
  return ALIBI ? fmaf(-slope2, fabsf(dist), y) : y;
}

// Zero the rows of a tile (`chunks` pieces of [128 rows][128 bytes]) that see nothing; one warp.  The
// swizzle permutes within a row's 128 bytes only.
__device__ __forceinline__ void zero_dead_rows(void* tile, int chunks, const int2* rows, int lane) {
  for (int r = lane; r < TILE; r += 32)
    if (rows[r].y == 0)
      for (int c = 0; c < chunks; ++c) {
        uint4* at = reinterpret_cast<uint4*>(static_cast<uint8_t*>(tile) + c * 16384 + r * 128);
#pragma unroll
        for (int u = 0; u < 8; ++u) at[u] = make_uint4(0, 0, 0, 0);
      }
}

// Bits of the tiles in [a, b) that hold rows which see nothing; all warps of the block.
__device__ __forceinline__ void note_dead(uint32_t* words, const int4* tiles, int a, int b) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int w = (a >> 5) + warp; w <= (b - 1) >> 5 && a < b; w += NTHREADS / 32) {
    const int t = w * 32 + lane;
    const uint32_t m = __ballot_sync(0xffffffff, t >= a && t < b && tiles[t].z == 0);
    if (lane == 0) words[w] = m;
  }
}
__device__ __forceinline__ bool is_dead(const uint32_t* words, int t) { return (words[t >> 5] >> (t & 31)) & 1; }

// 16 fp32 TMEM columns times f as bf16 to out[0..16), of which the first n are real (n a multiple of 8)
__device__ __forceinline__ void store16(__nv_bfloat16* out, const uint32_t (&v)[16], float f, int n) {
  auto p = [&](int i) { return pack_bf16x2(__uint_as_float(v[i]) * f, __uint_as_float(v[i + 1]) * f); };
  if (n > 0) *reinterpret_cast<uint4*>(out) = make_uint4(p(0), p(2), p(4), p(6));
  if (n > 8) *reinterpret_cast<uint4*>(out + 8) = make_uint4(p(8), p(10), p(12), p(14));
}
__device__ __forceinline__ void zero16(__nv_bfloat16* out, int n) {
  if (n > 0) *reinterpret_cast<uint4*>(out) = make_uint4(0, 0, 0, 0);
  if (n > 8) *reinterpret_cast<uint4*>(out + 8) = make_uint4(0, 0, 0, 0);
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

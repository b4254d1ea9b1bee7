// Pieces that the two forms of attention over an 8-bit cache share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace pb {
namespace cache8 {

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Row sums. A key's weight is w = 2^(s + ev - m + c), m the running maximum of s + ev (lagging by up to 8) and c a
// constant; the row sum adds w 2^-ev. V's scales 2^ev lie in [2^-100, 2^120], so a key's part of the sum lies between
// 2^(c - 120) for the maximum itself and 2^(c + 8 + 100). Counted in units of 2^13 neither end leaves fp32's normal
// range, for up to 2^25 keys.
constexpr float kSumUnit = 0x1p-13f;
// A block of tiny values (of zeros above all: 2^-100) beside large ones: w itself leaves fp32's range before its part
// of the sum is negligible, so blocks under this scale add exp2(s - m + c) on its own. What is left out then needs
// two blocks of one row whose scales are 2^115 and more apart, the smaller one above this.
constexpr float kTinyScale = 0x1p-60f;

// sum * 2^d for d <= 0: the sum may be as large as 2^-d, so that 2^d alone would be zero too early.
__device__ __forceinline__ float scale_sum(float sum, float d) {
  const float h = exp2_fast(0.5f * d);
  return sum * h * h;
}

// Two e4m3 bytes -> two halves (exact).
__device__ __forceinline__ uint32_t f16x2_of(uint32_t two_bytes) {
  uint32_t d;
  asm("{\n.reg .b16 h;\ncvt.u16.u32 h, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(d) : "r"(two_bytes));
  return d;
}

// The same of a word's upper two bytes.
__device__ __forceinline__ uint32_t f16x2_of_upper(uint32_t w) {
  uint32_t d;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(d) : "r"(w));
  return d;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 bytes of a cache row, past L1: a CTA reads each of them once.
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// 0xff in each byte of `w` that holds an e4m3 NaN (0x7f, 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t m = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (m >> 7) * 255u;
}

// Bit i: byte i of `w` is an e4m3 NaN.
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) {
  return ((nan_bytes(w) & 0x01010101u) * 0x01020408u) >> 24 & 15u;
}

// A query row times the power of two `down` fits f16; `up` undoes it. The row's largest magnitude goes to [2^13, 2^14):
// f16 ends at 2^16 and its least step is 2^-24, so channels down to 2^-30 of the largest keep all their bits (bf16 has
// eight) and smaller ones are off by at most 2^-38 of the largest. Rows of zeros or subnormal numbers and rows with an
// infinity stay as they are; rows under 2^-113 go as far up as `up` stays a normal number.
__device__ __forceinline__ void row_power(float amax, float& down, float& up) {
  const uint32_t ex = (__float_as_uint(amax) >> 23) & 255u;
  const bool plain = ex == 0u || ex == 255u;
  const uint32_t lift = min(13u, ex - 1u);
  down = plain ? 1.f : __uint_as_float((254u - ex + lift) << 23);
  up = plain ? 1.f : __uint_as_float((ex - lift) << 23);
}

// Keys of sequence b in the launch's view (what follows its last token taken off); may be negative.
__device__ __forceinline__ long long keys_of(const CacheAttnParams& p, int b) {
  const long long n = static_cast<long long>(p.lengths[b]) + p.offset;
  return max((n > p.T ? p.T : n) - p.back, -(1LL << 30));
}

// The merge kernel is launched while the main kernel runs, so that its start costs nothing: the main kernel lets
// it once all its CTAs are there, and it waits for the main kernel's end before it reads anything (nine
// sequences of 1 to 100001 tokens: 38.6 -> 36.9 us; five-token chunks of 8 sequences 70.0 -> 68.8).
__device__ __forceinline__ void let_merge_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_pieces() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The workspace's int64 words: [0, grid) hold per CTA the item that its run begins and leaves unfinished:
// sequence, KV head, first row and the number of CTAs that hold its further pieces (0: none).
struct Cut {
  int b, hk, row0, more;
};

__device__ __forceinline__ void put_cut(const CacheAttnParams& p, int cta, const Cut& c) {
  *reinterpret_cast<int4*>(p.plan + 2 * cta) = make_int4(c.b, c.hk, c.row0, c.more);
}
__device__ __forceinline__ Cut get_cut(const CacheAttnParams& p, int cta) {
  const int4 v = *reinterpret_cast<const int4*>(p.plan + 2 * cta);
  return {v.x, v.y, v.z, v.w};
}

}  // namespace cache8
}  // namespace pb

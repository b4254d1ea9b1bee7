// Rotary embedding in every layout the models use, and the append of rotated keys and of
// values to an 8-bit cache.
//
// Rotation. A head's first R channels hold R / 2 pairs (a, c): channels (i, i + R/2) in the
// half-split layout, (2i, 2i + 1) in the interleaved one. With the factors (cos, sin) of the
// token's position the pair becomes
//   a' = a cos - c sin        c' = c cos + a sin
// and channels R..D-1 are copied. Every product and sum is rounded separately in fp32 (no
// FMA), as torch's elementwise operations round them, so both orders give the same bits; the
// result is rounded once to the tensor's type. The factors may carry a length-scaling
// magnitude. The gradient is the same kernel with -sin.
//
// Append. Rows of keys (rotated, still fp32) and values are stored as e4m3 with one scale
// 2^e per (sequence, head, 32 cache rows): e is the least with amax / 2^e <= 448, so dividing
// by the scale is exact and each value is rounded once. A block that already holds rows
// keeps max(e_old, e_new); when e grows its old rows are requantised by the exact factor
// 2^(e_old - e). Values that are not finite are stored as NaN and do not take part in amax.
//
// Both are bound by their bytes: each value is read and written once. Measured (B200, bf16):
//   rotation  8 x 2048 tokens, 32 + 8 heads of 128, 32 turned: 335 MB in 58 us, 5.8 TB/s (a plain copy: 6.5)
//             34 turned (a multiple of 2 alone: one channel per load) 168 us, 36 (two per load) 117 us: bound by the
//             requests in flight, each moving 2 or 4 bytes. The presets turn 32, 64 or 128 channels, so these widths
//             have no form of their own (the torch operations take 885 us).
//   append    4 x 2048 tokens, 32 + 8 heads of 128: 186 MB in 53 us, 3.5 TB/s; one token for 64 sequences 9 us,
//             which is the host's time for the call
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace pb {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

__device__ __forceinline__ void turn(float a, float c, float cs, float sn, float& ya, float& yc) {
  ya = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(c, sn));
  yc = __fadd_rn(__fmul_rn(c, cs), __fmul_rn(a, sn));
}

// Division of n < 2^31 by a number known at launch: floor(n / d) = (umulhi(m, n) + n) >> l with
// l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1 (Granlund and Montgomery 1994).
struct Divider {
  uint32_t mul, shift, by;
  explicit Divider(uint32_t d) : shift(0), by(d) {
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(mul, n) + n) >> shift; }
};

// One thread turns (or copies) a unit: 2 V channels of one head, two vectors of V elements. A head has
// R / (2V) turned ones, then (D - R) / (2V) copied ones. Bound by the bytes in flight: eight blocks per SM
// (32 registers) with one unit per thread move 335 MB in 58 us (5.8 TB/s); two units per thread 72 us, four
// 105 us.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(256, 8) rotary_kernel(RotaryParams p, Divider per_token, Divider per_head, Divider per_seq,
                                                        uint32_t total) {
  const uint32_t w = blockIdx.x * 256u + threadIdx.x;
  if (w >= total) return;
  const int turned = p.R / (2 * V);
  const uint32_t tok = per_token.div(w), r = w - tok * per_token.by;
  const int h = per_head.div(r), u = r - h * per_head.by;
  const uint32_t b = per_seq.div(tok), s = tok - b * per_seq.by;
  const bool is_q = h < p.H;
  const int hh = is_q ? h : h - p.H;
  const T* src = is_q ? static_cast<const T*>(p.q) + b * p.q_sb + s * p.q_ss + hh * p.q_sh
                      : static_cast<const T*>(p.k) + b * p.k_sb + s * p.k_ss + hh * p.k_sh;
  T* dst = is_q ? static_cast<T*>(p.q_out) + (static_cast<long long>(tok) * p.H + hh) * p.D
                : static_cast<T*>(p.k_out) + (static_cast<long long>(tok) * p.Hk + hh) * p.D;
  int e0, e1;  // first channels of the unit's two vectors
  if (u >= turned) {
    e0 = p.R + (u - turned) * 2 * V;
    e1 = e0 + V;
  } else if (INTER) {
    e0 = u * 2 * V;
    e1 = e0 + V;
  } else {
    e0 = u * V;
    e1 = e0 + p.R / 2;
  }
  const Vec<T, V> x0 = *reinterpret_cast<const Vec<T, V>*>(src + e0);
  const Vec<T, V> x1 = *reinterpret_cast<const Vec<T, V>*>(src + e1);
  Vec<T, V> y0 = x0, y1 = x1;
  if (u < turned) {
    const long long at = b * p.f_sb + s * p.f_ss + hh * p.f_sh + u * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float cs = p.cos[at + i], sn = p.sign * p.sin[at + i];
      float ya, yc;
      if (INTER) {
        // pair i of the unit: channels 2i and 2i + 1 of its 2V contiguous ones
        constexpr int W = V;
        const int a = 2 * i, c = 2 * i + 1;
        turn(to_f(a < W ? x0.v[a % W] : x1.v[a % W]), to_f(c < W ? x0.v[c % W] : x1.v[c % W]), cs, sn, ya, yc);
        if (a < W)
          y0.v[a % W] = from_f<T>(ya);
        else
          y1.v[a % W] = from_f<T>(ya);
        if (c < W)
          y0.v[c % W] = from_f<T>(yc);
        else
          y1.v[c % W] = from_f<T>(yc);
      } else {
        turn(to_f(x0.v[i]), to_f(x1.v[i]), cs, sn, ya, yc);
        y0.v[i] = from_f<T>(ya);
        y1.v[i] = from_f<T>(yc);
      }
    }
  }
  *reinterpret_cast<Vec<T, V>*>(dst + e0) = y0;
  *reinterpret_cast<Vec<T, V>*>(dst + e1) = y1;
}

template <typename T, int V>
void launch_rotary_v(const RotaryParams& all, cudaStream_t stream) {
  const uint32_t units = all.D / (2 * V), per_token = (all.H + all.Hk) * units;
  // whole sequences per launch (or part of one, with its own base pointers), so that unit counts stay within 2^30
  const long long most = (1LL << 30) / per_token;
  const long long B = all.tokens / all.S;
  const long long seqs = most / all.S > 0 ? most / all.S : 1;
  const long long toks = seqs * all.S <= most ? all.S : most;
  for (long long b0 = 0; b0 < B; b0 += seqs) {
    for (long long s0 = 0; s0 < all.S; s0 += toks) {
      RotaryParams p = all;
      const long long nb = B - b0 < seqs ? B - b0 : seqs, ns = all.S - s0 < toks ? all.S - s0 : toks;
      p.q = static_cast<const T*>(all.q) + b0 * all.q_sb + s0 * all.q_ss;
      p.k = static_cast<const T*>(all.k) + b0 * all.k_sb + s0 * all.k_ss;
      p.q_out = static_cast<T*>(all.q_out) + (b0 * all.S + s0) * all.H * all.D;
      p.k_out = static_cast<T*>(all.k_out) + (b0 * all.S + s0) * all.Hk * all.D;
      p.cos += b0 * all.f_sb + s0 * all.f_ss;
      p.sin += b0 * all.f_sb + s0 * all.f_ss;
      const uint32_t total = static_cast<uint32_t>(nb * ns * per_token);
      const unsigned grid = (total + 255) / 256;
      const Divider dt(per_token), dh(units), ds(static_cast<uint32_t>(ns));
      if (p.interleave)
        rotary_kernel<T, V, true><<<grid, 256, 0, stream>>>(p, dt, dh, ds, total);
      else
        rotary_kernel<T, V, false><<<grid, 256, 0, stream>>>(p, dt, dh, ds, total);
    }
  }
}

// Widest vector that the channel counts, strides and base addresses all allow. (D is even.)
template <typename T>
void launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  auto fits = [&](int v) {
    const long long bytes = static_cast<long long>(v) * sizeof(T);
    if (p.D % (2 * v) != 0 || p.R % (2 * v) != 0) return false;
    for (const void* a : {p.q, p.k, static_cast<const void*>(p.q_out), static_cast<const void*>(p.k_out)})
      if (reinterpret_cast<uintptr_t>(a) % bytes != 0) return false;
    for (long long st : {p.q_sb, p.q_ss, p.q_sh, p.k_sb, p.k_ss, p.k_sh})
      if (st % v != 0) return false;
    return true;
  };
  constexpr int kWide = 16 / sizeof(T);
  if (fits(kWide))
    launch_rotary_v<T, kWide>(p, stream);
  else if (kWide > 4 && fits(4))
    launch_rotary_v<T, 4>(p, stream);
  else if (fits(2))
    launch_rotary_v<T, 2>(p, stream);
  else
    launch_rotary_v<T, 1>(p, stream);
}

// ------------------------------------------------------------------------------- append
constexpr int kRows = kCacheBlock;  // cache rows per scale
constexpr int kThreads = 128;

// Least power of two s with amax / s <= 448 = 1.75 * 2^8, from amax's exponent and mantissa.
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, kCacheMinExp), kCacheMaxExp);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3_of(float x) {
  const uint32_t u = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  return fabsf(x) < INFINITY ? u : 0x7fu;
}

__device__ __forceinline__ float of_e4m3(uint32_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// max(m, |x|) that a NaN ends in.
__device__ __forceinline__ float max_abs(float m, float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(x)));
  return m;
}

// A lane's N = D / 32 channels of a row, and what turning them takes: each becomes x cs + other sn, with
// `other` its pair's other channel and the sign of sin already in sn (the same products and the same
// sum as `turn`). Channels at or past R keep their value. EASY: pairs lie at the same place of two lanes
// (or in one lane), a lane is turned whole or not at all, and its factors can be read as one vector.
template <int N, bool INTER, bool EASY>
struct Turner {
  float cs[N], sn[N];
  int from;  // half-split layout: the lane that holds the pairs' other channels

  __device__ __forceinline__ void factors(const float* cos, const float* sin, int lane, int R) {
    const int e0 = lane * N, half = R >> 1;
    if (EASY) {
      const bool upper = !INTER && e0 >= half;
      from = (upper ? lane - half / N : lane + half / N) & 31;
      if (e0 >= R) return;
      if (INTER) {
        const Vec<float, N / 2> c = *reinterpret_cast<const Vec<float, N / 2>*>(cos + e0 / 2);
        const Vec<float, N / 2> s = *reinterpret_cast<const Vec<float, N / 2>*>(sin + e0 / 2);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          cs[i] = c.v[i / 2];
          sn[i] = i & 1 ? s.v[i / 2] : -s.v[i / 2];
        }
      } else {
        const int f = upper ? e0 - half : e0;
        const Vec<float, N> c = *reinterpret_cast<const Vec<float, N>*>(cos + f);
        const Vec<float, N> s = *reinterpret_cast<const Vec<float, N>*>(sin + f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          cs[i] = c.v[i];
          sn[i] = upper ? s.v[i] : -s.v[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = e0 + i;
        const bool first = INTER ? (i & 1) == 0 : e < half;
        const int f = INTER ? e >> 1 : (first ? e : e - half);
        cs[i] = e < R ? cos[f] : 1.f;
        sn[i] = e < R ? (first ? -sin[f] : sin[f]) : 0.f;
      }
    }
  }
  // `row` is read again only where the pair's channels lie at different places of their lanes.
  __device__ __forceinline__ void apply(float (&x)[N], const __nv_bfloat16* row, int lane, int R) const {
    float other[N];
    if (INTER) {
#pragma unroll
      for (int i = 0; i < N; ++i) other[i] = x[i ^ 1];
    } else if (EASY) {
#pragma unroll
      for (int i = 0; i < N; ++i) other[i] = __shfl_sync(0xffffffffu, x[i], from);
    } else {
      const int half = R >> 1;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = lane * N + i;
        other[i] = e < R ? to_f(row[e < half ? e + half : e - half]) : 0.f;
      }
    }
    if (EASY) {
      if (lane * N < R) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(other[i], sn[i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (lane * N + i < R) x[i] = __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(other[i], sn[i]));
    }
  }
};

template <int N>
__device__ __forceinline__ Vec<__nv_bfloat16, N> load_row(const __nv_bfloat16* row, int lane) {
  return *reinterpret_cast<const Vec<__nv_bfloat16, N>*>(row + lane * N);
}
template <int N>
__device__ __forceinline__ void widen(const Vec<__nv_bfloat16, N>& raw, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f(raw.v[i]);
}

// CTAs [0, q_blocks) turn the queries, one token each: its factors are read once, its heads go over the
// four warps, eight rows in flight each. The rest take one (sequence, KV head, block of 32 cache rows, K
// or V) each: pass one leaves the rows' values in registers and finds amax, pass two requantises old
// rows if need be and stores. What bounds it is the instructions per value next to 3 bytes of traffic, so
// values are kept in vectors and the rare case (something not finite) in a branch of its own. Seven blocks per
// SM (72 registers) against the four of an unbounded build (93): more rows in flight. Blocks of 256 threads
// were slower: the two barriers then hold up twice the rows.
template <int D, bool INTER, bool EASY>
__global__ void __launch_bounds__(kThreads, 7) rotary_append_kernel(AppendParams p) {
  constexpr int N = D / 32;
  constexpr int kWarps = kThreads / 32;
  constexpr int kWarpRows = kRows / kWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long blk = blockIdx.x;
  if (blk < p.q_blocks) {
    const int b = static_cast<int>(blk / p.s);
    const int i = static_cast<int>(blk - static_cast<long long>(b) * p.s);
    const __nv_bfloat16* src = p.q + b * p.q_sb + i * p.q_ss;
    __nv_bfloat16* dst = p.q_out + blk * p.H * D;
    const long long pos = min(max(static_cast<long long>(p.lengths[b]) + i, 0LL), p.table_rows - 1);
    Turner<N, INTER, EASY> turner;
    turner.factors(p.cos + pos * (p.R >> 1), p.sin + pos * (p.R >> 1), lane, p.R);
    for (int h0 = warp; h0 < p.H; h0 += 8 * kWarps) {
      Vec<__nv_bfloat16, N> raw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (h0 + j * kWarps < p.H) raw[j] = load_row<N>(src + (h0 + j * kWarps) * p.q_sh, lane);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int h = h0 + j * kWarps;
        if (h >= p.H) break;
        float x[N];
        widen<N>(raw[j], x);
        turner.apply(x, src + h * p.q_sh, lane, p.R);
        Vec<__nv_bfloat16, N> y;
#pragma unroll
        for (int e = 0; e < N; ++e) y.v[e] = from_f<__nv_bfloat16>(x[e]);
        *reinterpret_cast<Vec<__nv_bfloat16, N>*>(dst + h * D + lane * N) = y;
      }
    }
    return;
  }
  unsigned rest = static_cast<unsigned>(blk - p.q_blocks);
  const bool is_v = rest & 1;
  rest >>= 1;
  const int nth = static_cast<int>(rest % p.blocks_per_seq);
  rest /= p.blocks_per_seq;
  const int hk = static_cast<int>(rest % p.Hkv);
  const int b = static_cast<int>(rest / p.Hkv);
  const int start = p.lengths[b];                      // first appended row
  if (start < 0 || start >= p.T) return;
  const int end = static_cast<int>(min(static_cast<long long>(start) + p.s, static_cast<long long>(p.T)));
  if (start / kRows + static_cast<long long>(nth) > (end - 1) / kRows) return;
  const int cb = start / kRows + nth;                  // cache block
  const int row0 = cb * kRows;
  const int lo = max(start - row0, 0);                 // appended rows of the block: [lo, hi)
  const int hi = min(end - row0, kRows);
  if (hi <= lo) return;

  const __nv_bfloat16* x0 =
      (is_v ? p.v + b * p.v_sb + hk * p.v_sh : p.k + b * p.k_sb + hk * p.k_sh) + (row0 - start) * (is_v ? p.v_ss : p.k_ss);
  const long long x_ss = is_v ? p.v_ss : p.k_ss;
  uint8_t* cache = (is_v ? p.v_cache + b * p.vc_sb + hk * p.vc_sh : p.k_cache + b * p.kc_sb + hk * p.kc_sh) +
                   static_cast<long long>(row0) * D + lane * N;
  float* scale = (is_v ? p.v_scale + b * p.vs_sb + hk * p.vs_sh : p.k_scale + b * p.ks_sb + hk * p.ks_sh) + cb;
  const float held = lo > 0 ? *scale : 0.f;  // read before the barrier below, written after it

  Vec<__nv_bfloat16, N> raw[kWarpRows];
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j) {
    const int r = warp + j * kWarps;
    if (r >= lo && r < hi) raw[j] = load_row<N>(x0 + r * x_ss, lane);
  }
  float x[kWarpRows][N];
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j) {
    const int r = warp + j * kWarps;
    if (r >= lo && r < hi) {
      widen<N>(raw[j], x[j]);
      if (!is_v && p.cos != nullptr) {
        const long long at = min(static_cast<long long>(row0 + r), p.table_rows - 1) * (p.R >> 1);
        Turner<N, INTER, EASY> turner;
        turner.factors(p.cos + at, p.sin + at, lane, p.R);
        turner.apply(x[j], x0 + r * x_ss, lane, p.R);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) amax = max_abs(amax, x[j][i]);
    }
  }
  // (a block with something that is not finite in it finds its scale again, without that)
  if (__syncthreads_or(!(amax < INFINITY))) {
    amax = 0.f;
#pragma unroll
    for (int j = 0; j < kWarpRows; ++j) {
      const int r = warp + j * kWarps;
      if (r >= lo && r < hi) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (fabsf(x[j][i]) < INFINITY) amax = fmaxf(amax, fabsf(x[j][i]));
          else x[j][i] = NAN;
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  __shared__ float red[kWarps];
  if (lane == 0) red[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) amax = fmaxf(amax, red[w]);
  const float now = fmaxf(block_scale(amax), held);
  const float inv = 1.f / now;
  if (threadIdx.x == 0) *scale = now;
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j) {
    const int r = warp + j * kWarps;
    if (r >= lo && r < hi) {
      // (NaN converts to NaN; everything else is within +-448 now)
      Vec<uint16_t, N / 2> y;
#pragma unroll
      for (int i = 0; i < N; i += 2)
        y.v[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(x[j][i] * inv, x[j][i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<Vec<uint16_t, N / 2>*>(cache + r * D) = y;
    } else if (r < lo && now > held) {
      Vec<uint8_t, N>* at = reinterpret_cast<Vec<uint8_t, N>*>(cache + r * D);
      Vec<uint8_t, N> y = *at;
      const float f = held * inv;
#pragma unroll
      for (int i = 0; i < N; ++i) y.v[i] = static_cast<uint8_t>(e4m3_of(of_e4m3(y.v[i]) * f));
      *at = y;
    }
  }
}

}  // namespace

void rotary(const RotaryParams& p, int dtype, cudaStream_t stream) {
  if (dtype == 0)
    launch_rotary<__nv_bfloat16>(p, stream);
  else if (dtype == 1)
    launch_rotary<float>(p, stream);
  else
    launch_rotary<__half>(p, stream);
}

void rotary_append(AppendParams p, int D, bool interleave, cudaStream_t stream) {
  p.q_blocks = p.cos != nullptr ? static_cast<long long>(p.B) * p.s : 0;
  p.blocks_per_seq = p.s == 1 ? 1 : (p.s - 1 + kRows - 1) / kRows + 1;
  const long long blocks = p.q_blocks + 2LL * p.B * p.Hkv * p.blocks_per_seq;
  const unsigned grid = static_cast<unsigned>(blocks);
  const int N = D / 32, half = p.R >> 1;
  const bool aligned = reinterpret_cast<uintptr_t>(p.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sin) % 16 == 0;
  const bool easy = aligned && (interleave ? p.R % N == 0 && (half * 2) % N == 0 : half % N == 0);
  auto run = [&](auto kern) { kern<<<grid, kThreads, 0, stream>>>(p); };
  if (D == 64) {
    if (interleave)
      easy ? run(rotary_append_kernel<64, true, true>) : run(rotary_append_kernel<64, true, false>);
    else
      easy ? run(rotary_append_kernel<64, false, true>) : run(rotary_append_kernel<64, false, false>);
  } else {
    if (interleave)
      easy ? run(rotary_append_kernel<128, true, true>) : run(rotary_append_kernel<128, true, false>);
    else
      easy ? run(rotary_append_kernel<128, false, true>) : run(rotary_append_kernel<128, false, false>);
  }
}

}  // namespace pb

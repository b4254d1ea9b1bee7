// Attention of a few query rows per KV head over an 8-bit cache (one-token decode above all).
//
//   o_r = sum_t softmax_t(scale q_r . K_t) V_t,   K_t = 2^ek k_t,  V_t = 2^ev v_t
//
// with e4m3 rows k_t, v_t and one scale per 32 cache rows and head. A row r is one (token, query
// head of the KV head's group); it sees the keys at or before its token's position.
//
// Bound: 2 D + 1/4 bytes per visible key and KV head, read once, against group x 4 D flops: HBM.
// Per SM that is about 23 cached values per clock, each needing `group` multiply-adds and a
// conversion, which the fp32 pipes cannot do at group 4 and up. So the products run on the
// tensor cores as m16n8k16 f16 products with keys (then channels) on M and query rows on N: the
// e4m3 operand converts exactly to f16 in registers. tcgen05 would need the converted tile in shared
// memory and 128 rows of M per product; here 8 or 16 rows are useful and the pipes idle anyway. Each warp
// copies its own 32-key steps (cp.async, two or three steps ahead), so no barrier of the CTA stands between
// the memory and the products.
//
// Measured (B200, 32 query and 8 KV heads): 64 sequences of 8192 tokens, heads of 128, 1.08 GB, in 175 us,
// 6.15 TB/s (a plain copy: 6.5), while the SMs run at 1965 MHz, and 197 us once the power cap has them at 1700;
// one sequence of 1000 tokens, heads of 64, 14 us, of which the kernels take 8. What is left is the latency of
// a 32-key step that three CTAs per SM do not quite hide. Other forms: the bytes loaded straight into
// registers 196 us where this took 193 and, at 16 rows, 41 us where this took 38.6 (nine sequences of 1 to 100001
// tokens; 36.6 us now, with the merge launched early); a
// ring whose lanes copy only what they read themselves (half lines of K) 240 us when direct loads took 214;
// four CTAs per SM 226 us (registers spill); a second wave of short runs for the SMs that finish first (equal
// runs end 25 % apart) 208 us, its CTAs' starts costing more than they even out.
//
// Up to 16 rows per KV head come here, in one or two tiles of 8; more go to the tensor-memory form
// (cache_attention_tc.cu). Both sides, 20 rows per KV head, 8 sequences of up to 16384 tokens: two passes
// over the cache here 134 us, four tiles in one pass 118 us (255 registers and spills), there 70 us.
//
//   S^T = K Q^T    A: K rows (lane g holds rows g, g + 8), B: Q.  The contraction index d is
//                  permuted so that a lane's 16 consecutive bytes of a row are four k-steps.
//   O^T = V^T P^T  A: V^T.  A lane holds 16 (D = 64: 8) consecutive channels of 4 keys; bytes of
//                  neighbouring keys are interleaved (prmt) into the k-pairs of the fragment.
//                  B: P^T from S^T by an 8 x 8 transpose (movmatrix).
// One scale belongs to one 32-key step: K's multiplies the scores; V's goes into the weights,
// w = 2^(s + ev - m), m the running maximum of s + ev, while the row sum adds w 2^-ev. So the weights
// fit f16 whatever the scales. Query rows are normalised by a power of two to fit f16 (exact down to 2^-30
// of the row's largest channel, see row_power; the factor goes to the scores). Weights are rounded to f16 as
// 2^10 w: half a step is 2^-11 relative down to w = 2^-24, less than the 2^-8 that half a step of bf16 is of the
// output, and far tails stay above zero.
//
// Work split: the key blocks of all (sequence, KV head, row group) items form one list, cut into
// equal runs over the grid on the device from the lengths, so ragged batches load all SMs alike
// and nothing depends on the host knowing a length. A run's piece of an item is written as an
// unnormalised partial (slot 2 CTA + 1 where the item begins in the run, 2 CTA where it began before);
// an item inside one run is finished at once. A second kernel merges the partials in CTA order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cache_attention_common.cuh"

namespace pb {
namespace {

using namespace cache8;

constexpr int kWarps = 4;
constexpr int kMaxSeqs = 1024;  // sequences per launch (prefix table in shared memory)
// An item's start and end cost a CTA about as much as this many key blocks (nine sequences of 1 to 100001
// tokens: 43 us without it, 39 with it).
constexpr int kItemCost = 4;
constexpr int kMinRun = kItemCost + 4;  // list entries per CTA at least: an item's cost and a block per warp

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Keys of sequence b (0 .. T) and its visible key blocks.
__device__ __forceinline__ int seq_blocks(const CacheAttnParams& p, int b, long long& n, int& first) {
  n = max(keys_of(p, b), 0LL);
  long long lo = 0;
  if (p.window >= 0) {
    lo = n - p.s - p.window;
    lo = lo < 0 ? 0 : lo;
  }
  first = static_cast<int>(lo / kCacheBlock);
  return static_cast<int>((n + kCacheBlock - 1) / kCacheBlock) - first;
}

// Shared memory of a CTA: per warp a ring of kStages 32-key steps: K rows, V rows, the step's two scales.
// Copies take whole 128-byte lines; a row's 16-byte chunks are permuted so that the fragment reads below
// meet no bank twice. The warps' results are merged over the ring's memory at an item's end.
template <int D, int RT>
struct Cfg {
  static constexpr int kStages = D == 128 && RT == 1 ? 2 : 3;
  static constexpr int kRows = kCacheBlock * D;      // bytes of K or V in a step
  static constexpr int kStage = 2 * kRows + 16;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kRed = kWarps * RT * 8 * (D + 2) * 4;
  static constexpr int kBytes = kRing > kRed ? kRing : kRed;
  static constexpr int kCtas = RT == 1 ? 3 : 2;      // per SM, what the registers allow
};

// Where chunk c (16 bytes) of row r of a step lies. D = 128: c ^ (r & 7) within the row; D = 64: two rows
// make a line of eight chunks, and the line's number moves them by pairs.
template <int D>
__device__ __forceinline__ int chunk_at(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (((r >> 1) & 3) << 1)) << 4);
}
// The key (of eight) that row g of an S^T tile stands for. At D = 128 rows 2i and 2i + 1 have to differ in
// bit 2 for K's reads, and rows 2t (and 2t + 1) in their upper bits for V's: 0 5 2 7 4 1 6 3.
template <int D>
__device__ __forceinline__ int key_of(int g) {
  return D == 128 ? (g & 1 ? (g + 4) & 7 : g) : g;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t* src, bool real) {
  const int n = real ? BYTES : 0;  // the rest is zero-filled
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Starts the copies of the step at key row `base` (keys past n are zero-filled).
template <int D>
__device__ __forceinline__ void start_step(uint32_t stage, const uint8_t* k, const uint8_t* v, const float* ks,
                                           const float* vs, int base, int n, int lane) {
  constexpr int PR = D / 16;  // chunks per row
  const int c = lane % PR, r0 = lane / PR;
  const long long off = static_cast<long long>(base) * D + lane * 16;
#pragma unroll
  for (int i = 0; i < PR; ++i) {
    const int r = r0 + i * (32 / PR);
    const bool real = base + r < n;
    const uint32_t dst = stage + chunk_at<D>(r, c);
    copy_async<16>(dst, k + (real ? off + i * 512 : 0), real);
    copy_async<16>(dst + kCacheBlock * D, v + (real ? off + i * 512 : 0), real);
  }
  if (lane < 2)
    copy_async<4>(stage + 2 * kCacheBlock * D + 4 * lane,
                  reinterpret_cast<const uint8_t*>((lane ? vs : ks) + base / kCacheBlock), true);
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}

template <int D, int RT>
__global__ void __launch_bounds__(kWarps * 32, (Cfg<D, RT>::kCtas)) cache_attn_kernel(const CacheAttnParams p) {
  constexpr int R = RT * 8;         // query rows per item
  constexpr int KS = D / 16;        // k-steps of the score product = m-tiles of the value product
  __shared__ long long prefix[kMaxSeqs + 1];
  __shared__ long long warp_sum[kWarps];
  using C = Cfg<D, RT>;
  extern __shared__ __align__(16) uint8_t ring_smem[];
  float(*red)[R][D + 2] = reinterpret_cast<float(*)[R][D + 2]>(ring_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  let_merge_start();
  const uint32_t ring = smem_u32(ring_smem) + warp * C::kStages * C::kStage;

  // ------------------------------------------------ the block list: prefix per sequence, this CTA's run
  const long long heads = p.mult;  // (KV head, row group) items per sequence
  long long base = 0;
  for (int b0 = 0; b0 < p.B; b0 += kWarps * 32) {
    const int b = b0 + tid;
    long long n;
    int first;
    long long x = 0;
    if (b < p.B) {
      const int blocks = seq_blocks(p, b, n, first);
      x = blocks > 0 ? (blocks + kItemCost) * heads : 0;
    }
    const long long own = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    long long before = base;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    for (int w = 0; w < kWarps; ++w) base += warp_sum[w];
    if (b < p.B) prefix[b] = before + x - own;
    __syncthreads();
  }
  const long long total = base;
  if (tid == 0) prefix[p.B] = total;
  __syncthreads();
  long long run = (total + gridDim.x - 1) / gridDim.x;
  run = run < kMinRun ? kMinRun : run;
  // sequences without a visible key: zeros
  for (int e = blockIdx.x; e < p.B; e += gridDim.x) {
    if (prefix[e + 1] != prefix[e]) continue;
    uint4* dst = reinterpret_cast<uint4*>(p.out + e * p.o_sb);
    for (int i = tid; i < p.s * p.H * (D / 8); i += kWarps * 32) dst[i] = make_uint4(0, 0, 0, 0);
  }
  long long pos = blockIdx.x * run;
  const long long end = min(pos + run, total);
  if (pos >= end) {
    if (tid == 0) put_cut(p, blockIdx.x, {0, 0, 0, 0});
    return;
  }
  Cut cut = {0, 0, 0, 0};
  int b = 0;
  {
    int hi = p.B;  // last sequence with prefix <= pos (empty ones share a prefix with their follower)
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (prefix[mid] <= pos) b = mid;
      else hi = mid;
    }
  }

  while (pos < end) {
    while (prefix[b + 1] <= pos) ++b;
    long long n64;
    int first;
    const int nb = seq_blocks(p, b, n64, first);
    const int n = static_cast<int>(n64);
    const long long rel = pos - prefix[b];
    const int len = nb + kItemCost;             // the item's length in the list: its cost, then its blocks
    const int hr = static_cast<int>(rel / len);  // (KV head, row group)
    const int v0 = static_cast<int>(rel - static_cast<long long>(hr) * len);
    const int v1 = static_cast<int>(min(static_cast<long long>(len), v0 + (end - pos)));
    const int j0 = max(v0 - kItemCost, 0), j1 = max(v1 - kItemCost, 0);
    pos += v1 - v0;
    if (j1 == j0) continue;  // the run ends inside the cost: the blocks are all the next CTA's
    const int hk = hr / p.tiles;
    const int row0 = (hr - hk * p.tiles) * R;
    const int rows = p.s * p.group;

    // ---------------------------------------------- query rows: B fragments and row factors
    uint32_t q[RT][KS][2];
    float rf[RT][2];            // factor of rows 2t, 2t + 1: softmax scale, log2(e), the row's power of two
    int kmax[RT][2], kmin[RT][2];
    int lo_max = INT_MAX;        // lowest kmax and highest kmin of the item's rows: steps between need no mask
    int hi_min = 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 8 + g;
      float x[D / 4];
      float amax = 0.f;
      if (r < rows) {
        const int i = r / p.group;
        const __nv_bfloat16* src = p.q + b * p.q_sb + i * p.q_ss + (hk * p.group + r - i * p.group) * p.q_sh;
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint4 raw = *reinterpret_cast<const uint4*>(src + hf * 64 + t * 16 + w * 8);
            const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float lo = __uint_as_float(u[e] << 16), hi = __uint_as_float(u[e] & 0xffff0000u);
              x[hf * 16 + w * 8 + 2 * e] = lo;
              x[hf * 16 + w * 8 + 2 * e + 1] = hi;
              amax = fmaxf(amax, fmaxf(fabsf(lo), fabsf(hi)));
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < D / 4; ++e) x[e] = 0.f;
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      float down, up;
      row_power(amax, down, up);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        q[rt][ks][0] = pack_f16(x[4 * ks] * down, x[4 * ks + 1] * down);
        q[rt][ks][1] = pack_f16(x[4 * ks + 2] * down, x[4 * ks + 3] * down);
      }
      const float f = up * p.scale_log2;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        rf[rt][e] = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4);
        const int rr = row0 + rt * 8 + 2 * t + e;
        const int at = n - p.s + rr / p.group;  // the row's position
        kmax[rt][e] = rr < rows ? at : -1;
        kmin[rt][e] = p.window >= 0 ? max(at - p.window, 0) : 0;
        if (rr < rows) {
          lo_max = min(lo_max, at);
          hi_min = max(hi_min, kmin[rt][e]);
        }
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      lo_max = min(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, off));
      hi_min = max(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, off));
    }

    const uint8_t* kp = p.k + b * p.k_sb + hk * p.k_sh;
    const uint8_t* vp = p.v + b * p.v_sb + hk * p.v_sh;
    const float* ksp = p.k_scale + b * p.ks_sb + hk * p.ks_sh;
    const float* vsp = p.v_scale + b * p.vs_sb + hk * p.vs_sh;

    float m[RT][2], l[RT][2], o[RT][KS][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[rt][e] = -INFINITY;
        l[rt][e] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < KS; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[rt][mt][e] = 0.f;
    }

#pragma unroll
    for (int i = 0; i < C::kStages; ++i) {
      const int ji = j0 + warp + i * kWarps;
      if (ji < j1) start_step<D>(ring + i * C::kStage, kp, vp, ksp, vsp, (first + ji) * kCacheBlock, n, lane);
      copy_commit();
    }
    int slot = 0;
    for (int j = j0 + warp; j < j1; j += kWarps) {
      const int base_row = (first + j) * kCacheBlock;
      const uint32_t stage = ring + slot * C::kStage;
      slot = slot + 1 == C::kStages ? 0 : slot + 1;
      copy_wait<C::kStages - 1>();
      __syncwarp();  // every lane's copies are there for all
      float ks_now, vs_now;
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ks_now), "=f"(vs_now) : "r"(stage + 2 * C::kRows) : "memory");
      // ------------------------------------------ S^T = K Q^T
      float s[RT][2][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[rt][mt][e] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
          const int r = mt * 16 + key_of<D>(g);
          const uint4 ra = lds16(stage + chunk_at<D>(r, hf * 4 + t)), rb = lds16(stage + chunk_at<D>(r + 8, hf * 4 + t));
          const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = f16x2_of(wa[w]), a2 = f16x2_of(wa[w] >> 16);
            const uint32_t a1 = f16x2_of(wb[w]), a3 = f16x2_of(wb[w] >> 16);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma_f16(s[rt][mt], a0, a1, a2, a3, q[rt][hf * 4 + w][0], q[rt][hf * 4 + w][1]);
          }
        }
      }
      uint32_t vr[8][D / 32];  // keys of S^T's rows 2t, 2t+1, 2t+8, 2t+9 (+16); D / 8 bytes at channel g * D / 8
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = (i >> 2) * 16 + ((i >> 1) & 1) * 8 + key_of<D>(2 * t + (i & 1));
        const uint32_t at = stage + C::kRows + (D == 128 ? chunk_at<D>(r, g) : chunk_at<D>(r, g >> 1) + (g & 1) * 8);
        if (D == 128) {
          const uint4 r = lds16(at);
          vr[i][0] = r.x;
          vr[i][1] = r.y;
          vr[i][D / 32 - 2] = r.z;
          vr[i][D / 32 - 1] = r.w;
        } else {
          const uint2 r = lds8(at);
          vr[i][0] = r.x;
          vr[i][1] = r.y;
        }
      }
      const bool edge = base_row + kCacheBlock - 1 > lo_max || base_row < hi_min;
      if (edge) {
        // A value row may hold NaN where only some rows see it: its bytes become zero, and the channel becomes
        // NaN in the rows that do see it (elsewhere the products see to that).
        uint32_t bad[8];  // bit c: channel g * D / 8 + c of key i of vr
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          bad[i] = 0;
#pragma unroll
          for (int w = 0; w < D / 32; ++w) bad[i] |= nan_bits(vr[i][w]) << (4 * w);
          any |= bad[i];
        }
        if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int w = 0; w < D / 32; ++w) vr[i][w] &= ~nan_bytes(vr[i][w]);
#pragma unroll 1
            for (int src = 0; src < 4; ++src) {  // the lane of this quad's channels that holds the key's bytes
              const uint32_t m = __shfl_sync(0xffffffffu, bad[i], (lane & ~3) | src);
              const int key = base_row + (i >> 2) * 16 + ((i >> 1) & 1) * 8 + key_of<D>(2 * src + (i & 1));
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (m != 0 && key <= kmax[rt][e] && key >= kmin[rt][e]) {
#pragma unroll
                    for (int c = 0; c < D / 8; ++c)
                      if (m >> c & 1) o[rt][c >> 1][e + 2 * (c & 1)] = NAN;
                  }
            }
          }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = base_row + mt * 16 + (e >> 1) * 8 + key_of<D>(g);
              if (key > kmax[rt][e & 1] || key < kmin[rt][e & 1]) s[rt][mt][e] = -INFINITY;
            }
      }
      // ------------------------------------------ weights 2^(s + ev - m + 10)
      // m follows the maximum of s + ev when that has grown by 2^4: weights stay under 2^14, and most
      // steps need no exchange between lanes and leave O as it is.
      const float ev = __log2f(vs_now), vi = kSumUnit / vs_now;
      bool grow = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = rf[rt][e] * ks_now;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            float& x0 = s[rt][mt][e];
            float& x1 = s[rt][mt][e + 2];
            if (edge) {  // a hidden key stays -inf whatever the factor's sign or size
              x0 = x0 == -INFINITY ? x0 : fmaf(x0, f, ev);
              x1 = x1 == -INFINITY ? x1 : fmaf(x1, f, ev);
            } else {
              x0 = fmaf(x0, f, ev);
              x1 = fmaf(x1, f, ev);
            }
          }
          grow |= fmaxf(fmaxf(s[rt][0][e], s[rt][0][e + 2]), fmaxf(s[rt][1][e], s[rt][1][e + 2])) > m[rt][e] + 4.f;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float corr[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(s[rt][0][e], s[rt][0][e + 2]), fmaxf(s[rt][1][e], s[rt][1][e + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = mx > m[rt][e] + 4.f ? mx : m[rt][e];
            const float d = m[rt][e] == mn ? 0.f : m[rt][e] - mn;
            corr[e] = exp2_fast(d);
            m[rt][e] = mn;
            l[rt][e] = scale_sum(l[rt][e], d);
          }
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[rt][mt][e] *= corr[e & 1];
        }
      }
      const bool tiny = vs_now < kTinyScale;
      uint32_t pf[RT][2][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ref = m[rt][e] == -INFINITY ? 0.f : m[rt][e] - 10.f;
          float add = 0.f;
          if (tiny) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int hh = 0; hh < 4; hh += 2) l[rt][e] = fmaf(exp2_fast(s[rt][mt][e + hh] - (ref + ev)), kSumUnit, l[rt][e]);
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int hh = 0; hh < 4; hh += 2) {
              const float x = exp2_fast(s[rt][mt][e + hh] - ref);
              s[rt][mt][e + hh] = x;
              add += x;
            }
          // (a row that sees nothing of the step adds nothing, whatever the block's scale holds)
          if (!tiny && add != 0.f) l[rt][e] = fmaf(add, vi, l[rt][e]);
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          pf[rt][mt][0] = transpose8x8(pack_f16(s[rt][mt][0], s[rt][mt][1]));
          pf[rt][mt][1] = transpose8x8(pack_f16(s[rt][mt][2], s[rt][mt][3]));
        }
      }
      // ------------------------------------------ O^T += V^T P^T, two m-tiles of channels per word
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const uint32_t r0 = vr[4 * ks][w], r1 = vr[4 * ks + 1][w], r2 = vr[4 * ks + 2][w], r3 = vr[4 * ks + 3][w];
          const uint32_t lo01 = __byte_perm(r0, r1, 0x5140), hi01 = __byte_perm(r0, r1, 0x7362);
          const uint32_t lo23 = __byte_perm(r2, r3, 0x5140), hi23 = __byte_perm(r2, r3, 0x7362);
          {
            const uint32_t a0 = f16x2_of(lo01), a1 = f16x2_of(lo01 >> 16), a2 = f16x2_of(lo23), a3 = f16x2_of(lo23 >> 16);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma_f16(o[rt][2 * w], a0, a1, a2, a3, pf[rt][ks][0], pf[rt][ks][1]);
          }
          {
            const uint32_t a0 = f16x2_of(hi01), a1 = f16x2_of(hi01 >> 16), a2 = f16x2_of(hi23), a3 = f16x2_of(hi23 >> 16);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma_f16(o[rt][2 * w + 1], a0, a1, a2, a3, pf[rt][ks][0], pf[rt][ks][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (j + C::kStages * kWarps < j1)
        start_step<D>(stage, kp, vp, ksp, vsp, base_row + C::kStages * kWarps * kCacheBlock, n, lane);
      copy_commit();
    }

    // ---------------------------------------------- merge the warps (over the ring: all copies have landed)
    copy_wait<0>();
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[rt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        float* dst = red[warp][rt * 8 + 2 * t + e];
        // fragment (m-tile mt, half e2) of lane g is channel g * D / 8 + 2 mt + e2
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          dst[g * (D / 8) + 2 * mt] = o[rt][mt][e];
          dst[g * (D / 8) + 2 * mt + 1] = o[rt][mt][e + 2];
        }
        if (g == 0) {
          dst[D] = m[rt][e];
          dst[D + 1] = x;
        }
      }
    __syncthreads();
    const bool whole = j0 == 0 && j1 == nb;
    if (j0 == 0 && j1 < nb) cut = {b, hk, row0, static_cast<int>((nb - j1 + run - 1) / run)};
    float* part = p.part + (2LL * blockIdx.x + (j0 == 0)) * R * (D + 2);
    for (int w = tid; w < R * (D / 4); w += kWarps * 32) {
      const int r = w / (D / 4), c = (w - r * (D / 4)) * 4;
      if (row0 + r >= rows) continue;
      float M = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) M = fmaxf(M, red[x][r][D]);
      float L = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float mw = red[x][r][D];
        const float d = M == -INFINITY ? 0.f : mw - M, f = exp2_fast(d);
        L += scale_sum(red[x][r][D + 1], d);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += red[x][r][c + e] * f;
      }
      if (whole) {
        const int rr = row0 + r, i = rr / p.group;
        const float inv = L == 0.f ? 0.f : kSumUnit / L;
        const uint2 y = make_uint2(pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv));
        __nv_bfloat16* dst =
            p.out + b * p.o_sb + (static_cast<long long>(i) * p.H + hk * p.group + rr - i * p.group) * D + c;
        *reinterpret_cast<uint2*>(dst) = y;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) part[r * (D + 2) + c + e] = a[e];
        if (c == 0) {
          part[r * (D + 2) + D] = M;
          part[r * (D + 2) + D + 1] = L;
        }
      }
    }
    __syncthreads();  // red is written again for the next item
  }
  if (tid == 0) put_cut(p, blockIdx.x, cut);
}

// Merges the pieces of the item that CTA blockIdx.x of the main kernel began and did not finish. Few
// pieces: a warp per row. Many (one long sequence spread over the grid): a CTA per row, its warps
// taking every eighth piece. Either way the order of the sums is fixed by the pieces' order.
constexpr int kMergeWarps = 8;

template <int D>
__device__ __forceinline__ void store_row(const CacheAttnParams& p, const Cut& cut, int r, int c, float x0, float x1) {
  const int rr = cut.row0 + r, i = rr / p.group, h = cut.hk * p.group + rr - i * p.group;
  __nv_bfloat16* dst = p.out + cut.b * p.o_sb + (static_cast<long long>(i) * p.H + h) * D + c;
  *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(x0, x1);
}

template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) cache_attn_merge_kernel(const CacheAttnParams p) {
  constexpr int N = D / 32;
  wait_for_pieces();
  const Cut cut = get_cut(p, blockIdx.x);
  if (cut.more == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float red[kMergeWarps][D + 2];
  const int rows = min(p.item_rows, p.s * p.group - cut.row0);
  const long long step = static_cast<long long>(p.item_rows) * (D + 2);
  const bool few = cut.more < kMergeWarps;
  const int first = few ? 0 : warp, by = few ? 1 : kMergeWarps;  // this warp's pieces
  const int r0 = few ? blockIdx.y * kMergeWarps + warp : blockIdx.y, r_step = few ? gridDim.y * kMergeWarps : gridDim.y;
  for (int r = r0; r < rows; r += r_step) {
    const float* part = p.part + 2LL * blockIdx.x * step + r * (D + 2);
    auto slot = [&](int c) { return part + (2 * c + (c == 0)) * step; };
    float M = -INFINITY, L = 0.f, a[N];
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] = 0.f;
    for (int c = first + lane * by; c <= cut.more; c += 32 * by) M = fmaxf(M, slot(c)[D]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
#pragma unroll 8
    for (int c = first; c <= cut.more; c += by) {
      const float* x = slot(c);
      const float d = M == -INFINITY ? 0.f : x[D] - M, f = exp2_fast(d);
      L += scale_sum(x[D + 1], d);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float2 y = *reinterpret_cast<const float2*>(x + lane * N + e);
        a[e] = fmaf(y.x, f, a[e]);
        a[e + 1] = fmaf(y.y, f, a[e + 1]);
      }
    }
    if (few) {
      const float inv = L == 0.f ? 0.f : kSumUnit / L;
#pragma unroll
      for (int e = 0; e < N; e += 2) store_row<D>(p, cut, r, lane * N + e, a[e] * inv, a[e + 1] * inv);
      continue;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) red[warp][lane * N + e] = a[e];
    if (lane == 0) {
      red[warp][D] = M;
      red[warp][D + 1] = L;
    }
    __syncthreads();
    if (threadIdx.x < D / 2) {
      float mx = -INFINITY, l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
      for (int w = 0; w < kMergeWarps; ++w) mx = fmaxf(mx, red[w][D]);
#pragma unroll
      for (int w = 0; w < kMergeWarps; ++w) {
        const float d = mx == -INFINITY ? 0.f : red[w][D] - mx, f = exp2_fast(d);
        l += scale_sum(red[w][D + 1], d);
        x0 = fmaf(red[w][2 * threadIdx.x], f, x0);
        x1 = fmaf(red[w][2 * threadIdx.x + 1], f, x1);
      }
      const float inv = l == 0.f ? 0.f : kSumUnit / l;
      store_row<D>(p, cut, r, 2 * threadIdx.x, x0 * inv, x1 * inv);
    }
    __syncthreads();
  }
}

template <int D, int RT>
int ctas_per_sm() {
  static const int n = [] {  // (threads that come here first together wait for one of them)
    cudaFuncSetAttribute(cache_attn_kernel<D, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, RT>::kBytes);
    int found = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&found, cache_attn_kernel<D, RT>, kWarps * 32, Cfg<D, RT>::kBytes);
    return found < 1 ? 1 : found;
  }();
  return n;
}

template <int D, int RT>
void launch(const CacheAttnParams& p, cudaStream_t stream) {
  cudaFuncSetAttribute(cache_attn_kernel<D, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, RT>::kBytes);
  cache_attn_kernel<D, RT><<<p.grid, kWarps * 32, Cfg<D, RT>::kBytes, stream>>>(p);
}

int row_groups_of_8(const CacheAttnParams& p) { return p.s * p.group <= 8 ? 1 : 2; }

}  // namespace

bool cache_attn_many_rows(const CacheAttnParams& p) { return static_cast<long long>(p.s) * p.group > 16; }

void cache_attn_limits(const CacheAttnParams& p, int* seqs, int* tokens) {
  *seqs = kMaxSeqs;
  *tokens = p.s;
  if (cache_attn_many_rows(p)) {
    // entries of one sequence: its row tiles; whole tokens, so that a launch's rows are a chunk again
    const int most = kCacheTcEntries * kCacheTcRows / p.group;
    *tokens = p.s < most ? p.s : (most < 1 ? 1 : most);
    const int tiles = static_cast<int>((static_cast<long long>(*tokens) * p.group + kCacheTcRows - 1) / kCacheTcRows);
    *seqs = kCacheTcEntries / tiles < 1 ? 1 : kCacheTcEntries / tiles;
  }
}

void cache_attn_plan(CacheAttnParams& p, int D, long long* part_floats, long long* plan_words) {
  const long long rows = static_cast<long long>(p.s) * p.group;
  if (cache_attn_many_rows(p)) {
    p.item_rows = kCacheTcRows;
    p.tiles = static_cast<int>((rows + kCacheTcRows - 1) / kCacheTcRows);
    p.entries_per_seq = p.tiles;
    p.mult = p.Hkv;
    p.grid = device_sm_count();
  } else {
    const int rt = row_groups_of_8(p);
    p.item_rows = rt * 8;
    p.tiles = static_cast<int>((rows + p.item_rows - 1) / p.item_rows);
    p.entries_per_seq = 1;
    p.mult = p.Hkv * p.tiles;
    const int per_sm = D == 64 ? (rt == 1 ? ctas_per_sm<64, 1>() : ctas_per_sm<64, 2>())
                               : (rt == 1 ? ctas_per_sm<128, 1>() : ctas_per_sm<128, 2>());
    // key blocks if all caches were full
    const long long most = static_cast<long long>(p.B) * p.mult * ((p.T + kCacheBlock - 1) / kCacheBlock + kItemCost);
    const long long want = (most + kMinRun - 1) / kMinRun;
    const long long full = static_cast<long long>(device_sm_count()) * per_sm;
    p.grid = static_cast<int>(want < 1 ? 1 : (want < full ? want : full));
  }
  *part_floats = 2LL * p.grid * p.item_rows * (D + 2);
  *plan_words = 2LL * p.grid;
}

void cache_attn(const CacheAttnParams& p, int D, cudaStream_t stream) {
  const bool one = p.item_rows == 8;
  if (cache_attn_many_rows(p))
    cache_attn_tc(p, D, stream);
  else if (D == 64)
    one ? launch<64, 1>(p, stream) : launch<64, 2>(p, stream);
  else
    one ? launch<128, 1>(p, stream) : launch<128, 2>(p, stream);
  const dim3 merge(p.grid, p.item_rows < 32 ? p.item_rows : 32);
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = merge, cfg.blockDim = dim3(kMergeWarps * 32), cfg.stream = stream, cfg.attrs = &early, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, D == 64 ? cache_attn_merge_kernel<64> : cache_attn_merge_kernel<128>, p);
}

}  // namespace pb

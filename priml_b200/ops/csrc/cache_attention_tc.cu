// Attention of many query rows per KV head over an 8-bit cache (a prompt's chunk, a few tokens of a
// large group): tcgen05, rows on M.
//
// The mathematics is cache_attention.cu's. A work item is (sequence, 256-row tile, KV head), its rows
// being (token, query head of the group); the key tiles of all items form one list that is cut into
// equal runs over one persistent CTA per SM (lengths and causality are read on the device, so ragged
// batches and causal items of different length load all SMs alike).
//
// What bounds it: 4 D flops per (row, visible key) on the tensor cores, and one exp2 per pair on the
// 16-per-clock special-function units: at D = 128 both take 2048 clocks per SM for 256 rows x 128 keys.
// Feeding the MMA: kind::f16 needs both operands in 16 bits, so four warps convert each e4m3 tile to
// f16 (exact, half an instruction per value) on its way from global to swizzled shared memory, once
// per 256 rows. The block scales never touch the tiles: K's multiplies the scores of its 32 keys as
// part of the exponent's multiply-add; V's goes into the weights, w = 2^(s + ev - M), M being the
// running maximum of s + ev, so that w is within f16 whatever the scales, and the row sum adds
// w 2^-ev. Queries are normalised by a power of two per row to fit f16.
//
//   warps 0-3, 4-7  softmax of row tiles 0 and 1 (one row per thread); they also load their Q rows
//   warps 8-11      K and V tiles: load 16 bytes a lane a tile ahead, convert, store swizzled
//   warp 12         MMA issue: S_t = Q_t K^T, O_t += P_t V with P_t read from TMEM
// While one group's softmax runs the tensor cores work for the other. Items of at most 128 rows use
// both groups on the same rows: group t takes every other key tile, and the two results are merged.
// TMEM: S_0 [0, 128) S_1 [128, 256) O_0 [256, 256 + D) O_1; P_t lies over S_t's first 64 columns.
#include <cuda_fp16.h>

#include "attention_common.cuh"

namespace pb {
namespace {

using namespace attn;

constexpr int kKeys = 128;  // keys per tile
constexpr int kSoftmaxWarps = 8;
constexpr int kConvertWarps = 4;
constexpr int kThreads = 32 * (kSoftmaxWarps + kConvertWarps + 1);  // threads that work
constexpr int kLaunch = 512;  // launched: whole warpgroups, so that the register split below is theirs
// Registers per thread after the split; 512 threads are launched with 128 each (65,536).
constexpr int kRegsSoftmax = 176, kRegsConvert = 96, kRegsMma = 56;
static_assert(256 * kRegsSoftmax + 128 * kRegsConvert + 128 * kRegsMma <= kLaunch * 128, "register split");
constexpr int kAllBarrier = 1;   // named barriers: every thread; the two softmax groups
constexpr int kMergeBarrier = 2;
constexpr float kShift = 7.f;    // weights are up to 2^(threshold + shift) = 2^15, within f16

template <int D>
struct Cfg {
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kQTile = (D / 64) * kChunkBytes;  // [128 rows][D] f16 in 64-column chunks
  static constexpr int kOffK = 2 * kQTile;
  static constexpr int kOffV = kOffK + kStages * kQTile;
  static constexpr int kOffPrefix = kOffV + kStages * kQTile;
  static constexpr int kOffBars = kOffPrefix + (kCacheTcEntries + 2) * 8;
  static constexpr int kBytes = kOffBars + 512 + 1024;
  static constexpr int kMergeStride = D + 4;  // floats per row of the group merge (over the K and V stages)
  static_assert(128 * kMergeStride * 4 <= 2 * kStages * kQTile, "the merge rows must fit the K and V stages");
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

// Instruction descriptor: f16 A and B, fp32 accumulation.
constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t f16x2_of(uint32_t two_bytes) {  // two e4m3 bytes, exact
  uint32_t d;
  asm("{\n.reg .b16 h;\ncvt.u16.u32 h, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(d) : "r"(two_bytes));
  return d;
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {  // 0xff where a byte is an e4m3 NaN
  const uint32_t m = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (m >> 7) * 255u;
}

__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

template <int N>
__device__ __forceinline__ void bar_sync(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// Positions of a row tile's first and last rows, its visible key tiles and their count.
struct Span {
  int n;            // keys of the sequence in the launch's view (back already taken off)
  int pos0, pos1;   // positions of the tile's first and last token
  int first;        // first visible key tile
  int count;        // visible key tiles
};

__device__ __forceinline__ Span span_of(const CacheAttnParams& p, int b, int r0, int nrows) {
  Span s;
  long long n = static_cast<long long>(p.lengths[b]) + p.offset;
  n = (n > p.T ? p.T : n) - p.back;
  s.n = n < 0 ? 0 : static_cast<int>(n);
  // positions from the unclamped count: a sequence shorter than the chunk has queries before its start
  const int base = static_cast<int>(n < -(1LL << 30) ? -(1LL << 30) : n) - p.s;
  const int rows = p.s * p.group;
  const int r1 = min(r0 + nrows, rows) - 1;
  s.pos0 = base + r0 / p.group;
  s.pos1 = base + r1 / p.group;
  const int lo = p.window >= 0 ? max(s.pos0 - p.window, 0) : 0;
  s.first = lo / kKeys;
  s.count = s.pos1 < 0 || r1 < r0 ? 0 : s.pos1 / kKeys - s.first + 1;
  return s;
}

struct Piece {
  int b, tile, hk;
  Span sp;
  int j0, j1;      // key tiles of the item in this CTA's run
  bool both;       // at most 128 rows: the groups share them
};

// Walks a CTA's run of the list.
struct Walk {
  const CacheAttnParams& p;
  const long long* prefix;
  long long pos, end;
  int entry;
  __device__ Walk(const CacheAttnParams& p_, const long long* prefix_, long long pos_, long long end_)
      : p(p_), prefix(prefix_), pos(pos_), end(end_), entry(0) {
    int hi = p.B * p.entries_per_seq;
    while (hi - entry > 1) {
      const int mid = (entry + hi) >> 1;
      if (prefix[mid] <= pos) entry = mid;
      else hi = mid;
    }
  }
  __device__ bool next(Piece& x) {
    if (pos >= end) return false;
    while (prefix[entry + 1] <= pos) ++entry;
    x.b = entry / p.entries_per_seq;
    x.tile = entry - x.b * p.entries_per_seq;
    x.sp = span_of(p, x.b, x.tile * kCacheTcRows, kCacheTcRows);
    const long long rel = pos - prefix[entry];
    x.hk = static_cast<int>(rel / x.sp.count);
    x.j0 = static_cast<int>(rel - static_cast<long long>(x.hk) * x.sp.count);
    x.j1 = static_cast<int>(min(static_cast<long long>(x.sp.count), x.j0 + (end - pos)));
    x.both = p.s * p.group - x.tile * kCacheTcRows <= 128;
    pos += x.j1 - x.j0;
    return true;
  }
};

template <int D>
__global__ void __launch_bounds__(kLaunch, 1) cache_attn_tc_kernel(const CacheAttnParams p) {
  using C = Cfg<D>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::kOffK;
  uint8_t* sV = smem + C::kOffV;
  long long* prefix = reinterpret_cast<long long*>(smem + C::kOffPrefix);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
  uint64_t* k_full = bars;             // [NS] four converting warps
  uint64_t* k_empty = k_full + NS;     // [NS]
  uint64_t* v_full = k_empty + NS;     // [NS]
  uint64_t* v_empty = v_full + NS;     // [NS]
  uint64_t* s_full = v_empty + NS;     // [2]
  uint64_t* p_ready = s_full + 2;      // [2] four softmax warps
  uint64_t* o_final = p_ready + 2;     // [2]
  uint64_t* drain = o_final + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ long long warp_sum[kLaunch / 32];
  __shared__ uint32_t v_bad[NS][kConvertWarps][4];  // keys of an edge tile whose values hold a NaN

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], kConvertWarps);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], kConvertWarps);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_ready[t], 4);
      mbar_init(&o_final[t], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kSoftmaxWarps + kConvertWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }

  // -------------------------------------------------- the list of key tiles and this CTA's run of it
  const int entries = p.B * p.entries_per_seq;
  long long total = 0;
  for (int e0 = 0; e0 < entries; e0 += kLaunch) {
    const int e = e0 + tid;
    long long x = 0;
    if (e < entries) {
      const int b = e / p.entries_per_seq;
      x = static_cast<long long>(span_of(p, b, (e - b * p.entries_per_seq) * kCacheTcRows, kCacheTcRows).count) * p.mult;
    }
    const long long own = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    long long before = total;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    for (int w = 0; w < kLaunch / 32; ++w) total += warp_sum[w];
    if (e < entries) prefix[e] = before + x - own;
    __syncthreads();
  }
  if (tid == 0) prefix[entries] = total;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  long long run = (total + gridDim.x - 1) / gridDim.x;
  run = run < 2 ? 2 : run;
  if (blockIdx.x == 0) {
    for (int e = tid; e <= entries; e += kLaunch) p.plan[e] = prefix[e];
    if (tid == 0) p.plan[entries + 1] = run;
  }
  const long long from = min(blockIdx.x * run, total);
  Walk walk(p, prefix, from, min(from + run, total));
  Piece x;

  if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------------ softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int t = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * kKeys + lane_off;
    const uint32_t tO = tmem + 2 * kKeys + t * D + lane_off;
    uint32_t tiles_before = 0, n_s = 0, n_seg = 0;
    while (walk.next(x)) {
      const int rows = p.s * p.group;
      const int rr = x.tile * kCacheTcRows + (x.both ? r : t * 128 + r);  // row of the KV head
      const bool row_ok = rr < rows;
      const int tok = rr / p.group;
      const int head = x.hk * p.group + rr - tok * p.group;
      // ------------------------------ Q row: power of two, f16, swizzled tile
      float factor;
      {
        const __nv_bfloat16* src = p.q + x.b * p.q_sb + (row_ok ? tok * p.q_ss + head * p.q_sh : 0);
        float amax = 0.f;
        if (row_ok) {
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 raw = *reinterpret_cast<const uint4*>(src + c * 8);
            const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(u[e] << 16)), fabsf(__uint_as_float(u[e] & 0xffff0000u))));
          }
        }
        const uint32_t ex = (__float_as_uint(amax) >> 23) & 255u;
        const bool plain = ex < 2u || ex > 252u;  // zero or not finite: as it is
        float down = plain ? 1.f : __uint_as_float((254u - ex) << 23);
        factor = (plain ? 1.f : __uint_as_float(ex << 23)) * fabsf(p.scale_log2);
        if (p.scale_log2 < 0.f) down = -down;
        if (!x.both || t == 0) {
          uint8_t* tile = sQ + t * C::kQTile + r * 128;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            uint4 y = make_uint4(0, 0, 0, 0);
            if (row_ok) {
              const uint4 raw = *reinterpret_cast<const uint4*>(src + c * 8);
              const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
              uint32_t h[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                h[e] = pack_f16(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
              y = make_uint4(h[0], h[1], h[2], h[3]);
            }
            *reinterpret_cast<uint4*>(tile + (c >> 3) * kChunkBytes + (((c & 7) ^ (r & 7)) << 4)) = y;
          }
        }
      }
      fence_proxy_async_smem();
      bar_sync<kThreads>(kAllBarrier);

      // ------------------------------ key tiles
      const int pos = x.sp.pos0 - (x.tile * kCacheTcRows) / p.group + tok;
      const int kmax = row_ok ? pos : -1;
      const int kmin = p.window >= 0 ? pos - p.window : 0;
      const float* ksp = p.k_scale + x.b * p.ks_sb + x.hk * p.ks_sh;
      const float* vsp = p.v_scale + x.b * p.vs_sb + x.hk * p.vs_sh;
      const Span mine = x.both ? x.sp : span_of(p, x.b, x.tile * kCacheTcRows + t * 128, 128);
      const int blocks = (x.sp.n + kCacheBlock - 1) / kCacheBlock;
      float m = -INFINITY, l = 0.f;  // running maximum of s + ev (may lag by < 2^8), row sum of 2^(s - m + shift)
      bool ok = true;
      int n = 0;
      for (int j = x.j0; j < x.j1 && ok; ++j) {
        const int kt = x.sp.first + j;
        if (x.both ? ((j - x.j0) & 1) != t : (mine.count == 0 || kt < mine.first || kt >= mine.first + mine.count)) continue;
        const int k0 = kt * kKeys;
        float kc[4], ve[4], vi[4];  // score factor, exponent of V's scale and its reciprocal, per 32 keys
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int blk = k0 / kCacheBlock + i;
          const float ks = blk < blocks ? ksp[blk] : 1.f, vs = blk < blocks ? vsp[blk] : 1.f;
          kc[i] = fmaxf(factor * ks, 1e-37f);
          ve[i] = __log2f(vs);
          vi[i] = 1.f / vs;
        }
        if (!mbar_wait_warp_sleep(&s_full[t], n_s & 1, p.status, kTimeoutEpilogue, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t v[kKeys];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * c));
        tmem_wait_ld();
        const bool edge = k0 + kKeys - 1 > x.sp.pos0 || (p.window >= 0 && k0 < x.sp.pos1 - p.window);
        if (edge) {
          const uint32_t tile_no = tiles_before + (j - x.j0);
          const int st = tile_no % NS;
          if (!mbar_wait_warp(&v_full[st], (tile_no / NS) & 1, p.status, kTimeoutEpilogue, abort_flag)) { ok = false; break; }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t bad = 0;
#pragma unroll
            for (int w = 0; w < kConvertWarps; ++w) bad |= v_bad[st][w][c];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int key = k0 + 32 * c + i;
              if (bad >> i & 1) v[32 * c + i] = 0x7fffffffu;
              if (key > kmax || key < kmin) v[32 * c + i] = __float_as_uint(-INFINITY);
            }
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float a = -INFINITY, a2 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            a = fmaxf(a, __uint_as_float(v[32 * c + i]));
            a2 = fmaxf(a2, __uint_as_float(v[32 * c + i + 1]));
          }
          mx = fmaxf(mx, fmaf(fmaxf(a, a2), kc[c], ve[c]));
        }
        const bool grow = mx > m + kRescaleThreshold;
        const bool scale_o = grow && n > 0 && m != -INFINITY;
        if (__any_sync(0xffffffffu, scale_o)) {
          const float f = scale_o ? fast_exp2(m - mx) : 1.f;
          l *= f;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tO + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_32x32b_x16(tO + c * 16, o);
          }
        }
        if (grow) m = mx;
        const float ref = m == -INFINITY ? 0.f : kShift - m;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float add = ref + ve[c];
          const uint64_t mul2 = f2_pack(kc[c], kc[c]), add2 = f2_pack(add, add);
          uint64_t rs = f2_pack(0.f, 0.f);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(v[32 * c + 2 * i]), __uint_as_float(v[32 * c + 2 * i + 1])), mul2, add2),
                      x0, x1);
            const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
            const uint64_t e2 = f2_pack(e0, e1);
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(rs) : "l"(e2));
            pk[i] = pack_f16(e0, e1);
          }
          float r0, r1;
          f2_unpack(rs, r0, r1);
          l = fmaf(r0 + r1, vi[c], l);
          tmem_st_32x32b_x16(tS + 16 * c, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
        ++n_s;
        ++n;
      }
      if (ok) ok = mbar_wait_warp_sleep(&o_final[t], n_seg & 1, p.status, kTimeoutEpilogue, abort_flag);
      tc_fence_after();

      // ------------------------------ epilogue
      const bool whole = x.j0 == 0 && x.j1 == x.sp.count;
      float f_own = 1.f, f_other = 0.f;  // merge of the two groups' results (both == true)
      float* scratch = reinterpret_cast<float*>(sK) + r * C::kMergeStride;
      if (x.both) {
        if (t == 1) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            if (ok && n > 0) {
              tmem_ld_32x32b_x32(tO + c * 32, o);
              tmem_wait_ld();
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(scratch + c * 32 + 4 * i) =
                  make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          scratch[D] = m;
          scratch[D + 1] = l;
        }
        bar_sync<kSoftmaxWarps * 32>(kMergeBarrier);
        if (t == 0) {
          const float m2 = scratch[D], l2 = scratch[D + 1];
          const float mm = fmaxf(m, m2);
          f_own = m == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : fast_exp2(m - mm);
          f_other = m2 == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : fast_exp2(m2 - mm);
          l = l * f_own + l2 * f_other;
          m = mm;
        }
      }
      {
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const bool write = row_ok && (!x.both || t == 0);
        float* part = p.part + ((2LL * blockIdx.x + (x.j0 == 0)) * kCacheTcRows + (x.both ? r : t * 128 + r)) * (D + 2);
        __nv_bfloat16* orow = p.out + x.b * p.o_sb + (static_cast<long long>(write ? tok : 0) * p.H + (write ? head : 0)) * D;
        if (write && !whole) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
        if (!x.both || t == 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            if (ok && n > 0) {
              tmem_ld_32x32b_x32(tO + c * 32, o);
              tmem_wait_ld();
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0u;
            }
            if (write) {
              float y[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(o[i]) * f_own;
              if (x.both) {
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = fmaf(scratch[c * 32 + i], f_other, y[i]);
              }
              if (whole) {
                uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  dst[i] = make_uint4(pack_bf16x2(y[8 * i] * inv, y[8 * i + 1] * inv),
                                      pack_bf16x2(y[8 * i + 2] * inv, y[8 * i + 3] * inv),
                                      pack_bf16x2(y[8 * i + 4] * inv, y[8 * i + 5] * inv),
                                      pack_bf16x2(y[8 * i + 6] * inv, y[8 * i + 7] * inv));
              } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  *reinterpret_cast<float2*>(part + c * 32 + 2 * i) = make_float2(y[2 * i], y[2 * i + 1]);
              }
            }
          }
        }
      }
      tiles_before += x.j1 - x.j0;
      ++n_seg;
      tc_fence_before();
      bar_sync<kThreads>(kAllBarrier);
      if (*abort_flag) break;
    }
  } else if (warp < kSoftmaxWarps + kConvertWarps) {
    // ------------------------------------------------------------------ e4m3 -> f16 tiles
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    constexpr int PR = D / 16;              // 16-byte pieces per row
    constexpr int NP = kKeys * PR / 128;    // pieces per thread and tile
    const int c = tid - kSoftmaxWarps * 32;
    const int piece = c % PR, row_c = c / PR;  // piece i: row row_c + i * (128 / PR)
    uint32_t tile_no = 0;
    while (walk.next(x)) {
      bar_sync<kThreads>(kAllBarrier);
      const uint8_t* kp = p.k + x.b * p.k_sb + x.hk * p.k_sh + piece * 16;
      const uint8_t* vp = p.v + x.b * p.v_sb + x.hk * p.v_sh + piece * 16;
      uint4 kr[NP], vr[NP];
      auto load = [&](uint4(&dst)[NP], const uint8_t* src, int k0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int row = k0 + row_c + i * (128 / PR);
          dst[i] = row < x.sp.n ? load16(src + static_cast<long long>(row) * D) : make_uint4(0, 0, 0, 0);
        }
      };
      auto store = [&](const uint4(&src)[NP], uint8_t* tile) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int row = row_c + i * (128 / PR);
          uint8_t* base = tile + (piece >> 2) * kChunkBytes + row * 128;
          const uint32_t u[4] = {src[i].x, src[i].y, src[i].z, src[i].w};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[2 * e] = f16x2_of(u[e]);
            h[2 * e + 1] = f16x2_of(u[e] >> 16);
          }
          const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
          // the pieces of a row's two 64-channel chunks share banks: the upper chunk's lanes store
          // their halves in the other order
          const int p0 = 2 * (piece & 3);
          const bool swap = piece >= 4;
          *reinterpret_cast<uint4*>(base + (((p0 + swap) ^ (row & 7)) << 4)) = swap ? hi : lo;
          *reinterpret_cast<uint4*>(base + (((p0 + !swap) ^ (row & 7)) << 4)) = swap ? lo : hi;
        }
      };
      int k0 = (x.sp.first + x.j0) * kKeys;
      load(kr, kp, k0);
      load(vr, vp, k0);
      bool ok = true;
      for (int j = x.j0; j < x.j1 && ok; ++j, ++tile_no, k0 += kKeys) {
        const int st = tile_no % NS;
        const uint32_t ph = (tile_no / NS) & 1;
        if (!mbar_wait_warp(&k_empty[st], ph ^ 1u, p.status, kTimeoutProducer, abort_flag)) { ok = false; break; }
        store(kr, sK + st * C::kQTile);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[st]);
        if (j + 1 < x.j1) load(kr, kp, k0 + kKeys);
        if (!mbar_wait_warp(&v_empty[st], ph ^ 1u, p.status, kTimeoutProducer, abort_flag)) { ok = false; break; }
        if (k0 + kKeys - 1 > x.sp.pos0 || (p.window >= 0 && k0 < x.sp.pos1 - p.window)) {
          // an edge tile: values that are NaN become zero, their keys are told to the softmax
          uint32_t bad[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const uint32_t a = nan_bytes(vr[i].x), b2 = nan_bytes(vr[i].y), c2 = nan_bytes(vr[i].z), d2 = nan_bytes(vr[i].w);
            vr[i] = make_uint4(vr[i].x & ~a, vr[i].y & ~b2, vr[i].z & ~c2, vr[i].w & ~d2);
            const int row = row_c + i * (128 / PR);
            if (a | b2 | c2 | d2) bad[(i * (128 / PR)) >> 5] |= 1u << (row & 31);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t all = __reduce_or_sync(0xffffffffu, bad[w]);
            if (lane == 0) v_bad[st][warp - kSoftmaxWarps][w] = all;
          }
        }
        store(vr, sV + st * C::kQTile);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
        if (j + 1 < x.j1) load(vr, vp, k0 + kKeys);
      }
      bar_sync<kThreads>(kAllBarrier);
      if (*abort_flag) break;
    }
  } else {
    // ------------------------------------------------------------------ MMA issuer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
    if (warp > kSoftmaxWarps + kConvertWarps) return;  // fills the warpgroup
    constexpr uint32_t idesc_s = idesc_f16(128, kKeys, false);
    constexpr uint32_t idesc_o = idesc_f16(128, D, true);
    uint32_t tile_no = 0, n_p[2] = {0, 0};
    while (walk.next(x)) {
      bar_sync<kThreads>(kAllBarrier);
      tc_fence_after();
      if (lane == 0) {
        Span sp[2];
        sp[0] = span_of(p, x.b, x.tile * kCacheTcRows, 128);
        sp[1] = span_of(p, x.b, x.tile * kCacheTcRows + 128, 128);
        const int jn = x.j1 - x.j0, kt0 = x.sp.first + x.j0;
        int done[2] = {0, 0};
        bool ok = true;
        auto active = [&](int t, int j) {
          return x.both || (sp[t].count > 0 && kt0 + j >= sp[t].first && kt0 + j < sp[t].first + sp[t].count);
        };
        auto issue_s = [&](int t, int j) -> bool {
          const uint32_t no = tile_no + j, st = no % NS;
          if (!mbar_wait(&k_full[st], (no / NS) & 1, p.status, kTimeoutMma, abort_flag)) return false;
          tc_fence_after();
          if (active(t, j)) {
            const uint32_t q_base = smem_u32(sQ + (x.both ? 0 : t) * C::kQTile);
            const uint32_t k_base = smem_u32(sK + st * C::kQTile);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16(tmem + t * kKeys, kmajor_desc(q_base, kk), kmajor_desc(k_base, kk), idesc_s, kk > 0);
            umma_commit(&s_full[t]);
          }
          return true;
        };
        auto issue_pv = [&](int t, int j) -> bool {
          if (!active(t, j)) return true;
          const uint32_t no = tile_no + j, st = no % NS;
          if (!mbar_wait(&p_ready[t], n_p[t] & 1, p.status, kTimeoutMma, abort_flag)) return false;
          if (!mbar_wait(&v_full[st], (no / NS) & 1, p.status, kTimeoutMma, abort_flag)) return false;
          tc_fence_after();
          const uint32_t v_base = smem_u32(sV + st * C::kQTile);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_f16_tmem_a(tmem + 2 * kKeys + t * D, tmem + t * kKeys + kk * 8, mnmajor_desc(v_base, kk), idesc_o,
                            (done[t] | kk) != 0);
          ++n_p[t];
          ++done[t];
          return true;
        };
        auto k_done = [&](int j) { umma_commit(&k_empty[(tile_no + j) % NS]); };
        auto v_done = [&](int j) { umma_commit(&v_empty[(tile_no + j) % NS]); };
        if (x.both) {
          // one row tile: group t works on key tiles t, t + 2, ...
          ok = issue_s(0, 0);
          if (ok) k_done(0);
          if (ok && jn > 1) {
            ok = issue_s(1, 1);
            if (ok) k_done(1);
          }
          for (int j = 0; j < jn && ok; ++j) {
            const int t = j & 1;
            if (!(ok = issue_pv(t, j))) break;
            v_done(j);
            if (j + 2 < jn) {
              if (!(ok = issue_s(t, j + 2))) break;
              k_done(j + 2);
            }
          }
        } else {
          ok = issue_s(0, 0) && issue_s(1, 0);
          if (ok) k_done(0);
          for (int j = 0; j < jn && ok; ++j) {
            if (!(ok = issue_pv(0, j))) break;
            if (j + 1 < jn && !(ok = issue_s(0, j + 1))) break;
            if (!(ok = issue_pv(1, j))) break;
            v_done(j);
            if (j + 1 < jn) {
              if (!(ok = issue_s(1, j + 1))) break;
              k_done(j + 1);
            }
          }
        }
        umma_commit(&o_final[0]);
        umma_commit(&o_final[1]);
        tile_no += jn;
      }
      __syncwarp();
      bar_sync<kThreads>(kAllBarrier);
      if (*abort_flag) break;
    }
    if (lane == 0) {
      umma_commit(drain);
      mbar_wait(drain, 0, p.status, kTimeoutDrain, nullptr);
    }
    __syncwarp();
  }
  tc_fence_before();
  bar_sync<kThreads>(kAllBarrier);
  tc_fence_after();
  if (warp == kSoftmaxWarps + kConvertWarps) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
void launch(const CacheAttnParams& p, cudaStream_t stream) {
  cudaFuncSetAttribute(cache_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kBytes);
  cache_attn_tc_kernel<D><<<p.grid, kLaunch, Cfg<D>::kBytes, stream>>>(p);
}

}  // namespace

void cache_attn_tc(const CacheAttnParams& p, int D, cudaStream_t stream) {
  if (D == 64)
    launch<64>(p, stream);
  else
    launch<128>(p, stream);
}

}  // namespace pb

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
// Feeding the MMA: kind::f16 needs both operands in 16 bits, so the e4m3 tiles are converted to f16
// (exact, half an instruction per value) on their way to swizzled shared memory, once per 256 rows.
// The block scales never touch the tiles: K's multiplies the scores of its 32 keys as part of the
// exponent's multiply-add; V's goes into the weights, w = 2^(s + ev - M), M being the running maximum
// of s + ev, so that w is within f16 whatever the scales, and the row sum adds w 2^-ev. Queries are
// normalised by a power of two per row to fit f16 (exact down to 2^-30 of the row's largest channel).
//
//   warps 0-3, 4-7   softmax of row tiles 0 and 1 (one row per thread); they also load their Q rows
//   warps 8-11       K tiles, e4m3 -> f16: 16-byte loads a tile ahead, held in registers
//   warps 12-15      V tiles, the same, with the scales of both
//   warps 16, 17     MMA issue for group t: S_t = Q_t K^T, O_t += P_t V with P_t read from TMEM
//   warp 18          walks the run and hands its pieces out
// The softmax goes 64 keys at a time with two score buffers per group: while it works on one, the
// tensor cores fill the other and work for the other group. Items of at most 128 rows use both groups
// on the same rows: group t takes half t of every key tile, and the two results are merged.
// No role waits for the end of a piece but where it must: loads and conversions run ahead into the
// next piece while the softmax warps finish the last.
//
// Measured (B200, D = 128): a 2048-token prompt chunk that ends a cache of 32768, 32 + 8 heads, 1.07 TFLOP in
// 1.22 to 1.24 ms (860 to 872 TFLOP/s under the power cap). The tensor cores wait for the softmax warps'
// chain per 64 keys (score load, exponent, weight store), whose latency two buffers per group hide in part.
// Sixteen softmax warps of 64 registers were slower (1.70 against 1.29 ms: the rows' state spills), as was raw
// e4m3 staged through shared memory by bulk copies. Five tokens each of 8 sequences take 69 us, bound by the
// conversion: about 2000 clocks per tile of K or V and its four warps. Rows copied into the idle lanes of the
// tile, each copy with a part of the keys, halve the softmax's time there and change nothing in all (70 us).
// TMEM: S_0 [0, 64) and [64, 128), S_1 [128, 256), O_0 [256, 256 + D), O_1; P lies over the first half
// of its scores.
#include "attention_common.cuh"
#include "cache_attention_common.cuh"

#include <type_traits>

namespace pb {
namespace {

using namespace attn;
using namespace cache8;

constexpr int kKeys = 128;  // keys per tile
constexpr int kHalf = 64;   // keys per step of the softmax
constexpr int kSoftmaxWarps = 8, kConvertWarps = 4;  // converting warps of K, and as many of V
constexpr int kMmaWarp = kSoftmaxWarps + 2 * kConvertWarps, kWalkWarp = kMmaWarp + 2;
constexpr int kLaunch = 640;  // whole warpgroups, so that the register split below is theirs
// Registers per thread after the split; 640 threads are launched with 96 each.
constexpr int kRegsSoftmax = 136, kRegsConvert = 72, kRegsIssue = 64;
static_assert(256 * kRegsSoftmax + 256 * kRegsConvert + 128 * kRegsIssue <= kLaunch * 96, "register split");
constexpr float kTinyLog2 = -60.f;  // log2 of kTinyScale
constexpr float kShift = 7.f;     // weights are up to 2^(threshold + shift) = 2^15, within f16
// An item's start and end cost a CTA about as much as this many key tiles. Without it CTAs with many short items
// ran long: five tokens each of 8 ragged sequences 116 us (with it 72), four windowed prompts of 1111 tokens, 576
// items, 144 us (109).
constexpr int kItemCost = 3;
constexpr int kPieces = 4;        // work pieces in flight between the walking warp and the others
constexpr int kScratchCols = 32;  // columns that the groups exchange at a time

template <int D>
struct Cfg {
  static constexpr int kStages = 2;
  static constexpr int kQTile = (D / 64) * kChunkBytes;  // [128 rows][D] f16 in 64-column chunks
  static constexpr int kOffK = 2 * kQTile;
  static constexpr int kOffV = kOffK + kStages * kQTile;
  static constexpr int kScratchStride = kScratchCols + 4;  // floats
  static constexpr int kScratch = 128 * kScratchStride * 4;
  // The groups' exchange: query tile 1 is free in the pieces that need it.
  static constexpr int kOffScratch = D == 128 ? kQTile : kOffV + kStages * kQTile;
  static constexpr int kOffPrefix = kOffV + kStages * kQTile + (D == 128 ? 0 : kScratch);
  static constexpr int kOffBars = kOffPrefix + (kCacheTcEntries + 2) * 8;
  static constexpr int kBytes = kOffBars + 512 + 1024;
  static_assert(kBytes <= 227 * 1024 - 1024, "shared memory");
};

// Instruction descriptor: f16 A and B, fp32 accumulation.
constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// TMEM loads together with their wait. The registers hold nothing before the wait, which the compiler
// does not know: with the wait in a statement of its own it may move or spill them in between.
__device__ __forceinline__ void tmem_read_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_read_x32x2(uint32_t taddr, uint32_t (&a)[32], uint32_t (&b)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, "
      "%53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),
        "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(a[16]),
        "=r"(a[17]), "=r"(a[18]), "=r"(a[19]), "=r"(a[20]), "=r"(a[21]), "=r"(a[22]), "=r"(a[23]), "=r"(a[24]),
        "=r"(a[25]), "=r"(a[26]), "=r"(a[27]), "=r"(a[28]), "=r"(a[29]), "=r"(a[30]), "=r"(a[31]), "=r"(b[0]),
        "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]),
        "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15]), "=r"(b[16]), "=r"(b[17]),
        "=r"(b[18]), "=r"(b[19]), "=r"(b[20]), "=r"(b[21]), "=r"(b[22]), "=r"(b[23]), "=r"(b[24]), "=r"(b[25]),
        "=r"(b[26]), "=r"(b[27]), "=r"(b[28]), "=r"(b[29]), "=r"(b[30]), "=r"(b[31])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
}

// Descriptors of 128-byte-swizzled tiles as their low words; all share the high word. The steps of a
// product differ by constants in the low word, so one addition makes the next step's descriptor: the
// issuing warp's few instructions per MMA are what the tensor cores wait for.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // 1024 bytes between 8-row groups
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr, uint32_t lbo_bytes) {
  return (smem_addr >> 4) | ((lbo_bytes >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 b, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}" ::"r"(d),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// x, at least 1e-37 (a hidden key's -inf must stay -inf times this); NaN stays NaN.
__device__ __forceinline__ float positive(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(1e-37f));
  return x;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile(
      "{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(e));
  return e != 0;
}

// A value that all lanes share, told to the compiler as such.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

// Positions of a row tile's first and last rows, its visible key tiles and their count.
struct Span {
  int n;           // keys of the sequence in the launch's view
  int pos0, pos1;  // positions of the tile's first and last token
  int first;       // first visible key tile
  int count;       // visible key tiles
};

__device__ __forceinline__ Span span_of(const CacheAttnParams& p, int b, int r0, int nrows) {
  Span s;
  const int n = static_cast<int>(keys_of(p, b));
  s.n = n < 0 ? 0 : n;
  // positions from the unclamped count: a sequence shorter than the chunk has queries before its start
  const int base = n - p.s;
  const int r1 = min(r0 + nrows, p.s * p.group) - 1;
  s.pos0 = base + r0 / p.group;
  s.pos1 = base + r1 / p.group;
  const int lo = p.window >= 0 ? max(s.pos0 - p.window, 0) : 0;
  s.first = lo / kKeys;
  s.count = s.pos1 < 0 || r1 < r0 ? 0 : s.pos1 / kKeys - s.first + 1;
  return s;
}

// One piece of a CTA's run: key tiles [kt0, kt0 + count) of an item. Lies in shared memory.
struct Piece {
  int b, hk, row0;       // sequence, KV head, first row of the row tile
  int n;                 // keys of the sequence
  int base;              // position of the chunk's first token
  int kt0, count;        // key tiles of this piece (count 0: the run is done)
  int edge_hi, edge_lo;  // a key tile at k0 needs masks if k0 > edge_hi or k0 < edge_lo
  int lo_block;          // first block of 32 keys that any row of the tile sees
  int from[2], to[2];    // tiles of the piece that row tile 0 / 1 sees
  int both;              // at most 128 rows: the groups share them and take half of each tile
  int whole, begins;     // the piece is the whole item; it holds the item's first tile
  int nan;               // an edge tile of the piece holds a value that is NaN (set by V's converting warps)
};

// Walks a CTA's run of the list (one thread; its state lies in shared memory, not in registers).
struct Walk {
  long long pos, end, run;
  int entry;
  Cut cut;
  __device__ void start(const CacheAttnParams& p, const long long* prefix, long long pos_, long long end_,
                        long long run_) {
    pos = pos_;
    end = end_;
    run = run_;
    entry = 0;
    cut = {0, 0, 0, 0};
    int hi = p.B * p.entries_per_seq;
    while (hi - entry > 1) {
      const int mid = (entry + hi) >> 1;
      if (prefix[mid] <= pos) entry = mid;
      else hi = mid;
    }
  }
  __device__ void next(const CacheAttnParams& p, const long long* prefix, Piece& x) {
    int b, tile, hk, j0, j1;
    Span sp;
    do {
      if (pos >= end) {
        x.count = 0;
        return;
      }
      while (prefix[entry + 1] <= pos) ++entry;
      b = entry / p.entries_per_seq;
      tile = entry - b * p.entries_per_seq;
      sp = span_of(p, b, tile * kCacheTcRows, kCacheTcRows);
      const long long rel = pos - prefix[entry];
      const int len = sp.count + kItemCost;  // the item's length in the list: its cost, then its tiles
      hk = static_cast<int>(rel / len);
      const int v0 = static_cast<int>(rel - static_cast<long long>(hk) * len);
      const int v1 = static_cast<int>(min(static_cast<long long>(len), v0 + (end - pos)));
      j0 = max(v0 - kItemCost, 0);
      j1 = max(v1 - kItemCost, 0);
      pos += v1 - v0;
    } while (j1 == j0);  // the run ends inside the cost: the tiles are all the next CTA's
    x.b = b;
    x.hk = hk;
    x.row0 = tile * kCacheTcRows;
    x.n = sp.n;
    x.base = sp.pos0 - x.row0 / p.group;
    x.kt0 = sp.first + j0;
    x.count = j1 - j0;
    x.edge_hi = sp.pos0 - kKeys + 1;
    x.edge_lo = p.window >= 0 ? sp.pos1 - p.window : INT_MIN;
    x.lo_block = p.window >= 0 ? max(sp.pos0 - p.window, 0) / kCacheBlock : 0;
    x.both = p.s * p.group - x.row0 <= 128;
    x.whole = j0 == 0 && j1 == sp.count;
    x.begins = j0 == 0;
    x.nan = 0;
    for (int t = 0; t < 2; ++t) {
      const Span st = span_of(p, b, x.row0 + 128 * t, 128);
      x.from[t] = max(st.first - x.kt0, 0);
      x.to[t] = st.count == 0 ? 0 : min(st.first + st.count - x.kt0, x.count);
    }
    if (j0 == 0 && j1 < sp.count) cut = {b, hk, x.row0, static_cast<int>((sp.count - j1 + run - 1) / run)};
  }
};

// NaNs in the values of a piece's edge tiles are zero in shared memory. This makes their channels NaN in the stored result
// of a row at position `pos` that sees them, reading the cache again (and the piece from shared memory: nothing here
// may live in registers while the softmax runs).
template <int D>
__device__ __forceinline__ void store_nans(const CacheAttnParams& p, const Piece& x, int pos, __nv_bfloat16* out, float* part) {
  const uint8_t* rows = p.v + x.b * p.v_sb + x.hk * p.v_sh;
  const int kmin = p.window >= 0 ? pos - p.window : 0;
#pragma unroll 1
  for (int k0 = x.kt0 * kKeys; k0 < (x.kt0 + x.count) * kKeys; k0 += kKeys) {
    if (k0 <= x.edge_hi && k0 >= x.edge_lo) continue;
#pragma unroll 1
    for (int key = max(k0, kmin); key <= min(k0 + kKeys - 1, pos); ++key) {
      const uint8_t* row = rows + static_cast<long long>(key) * D;
#pragma unroll 1
      for (int c = 0; c < D; ++c) {
        if ((row[c] & 0x7f) != 0x7f) continue;
        if (x.whole) out[c] = __float2bfloat16_rn(NAN);
        else part[c] = NAN;
      }
    }
  }
}

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
  uint64_t* k_full = bars;                      // [NS] four converting warps
  uint64_t* k_empty = k_full + NS;              // [NS]
  uint64_t* v_full = k_empty + NS;              // [NS]
  uint64_t* v_empty = v_full + NS;              // [NS]
  uint64_t* s_full = v_empty + NS;              // [2][2] group, score buffer
  uint64_t* p_ready = s_full + 4;               // [2][2] four softmax warps
  uint64_t* pv_done = p_ready + 4;              // [2]
  uint64_t* o_final = pv_done + 2;              // [2]
  uint64_t* q_full = o_final + 2;               // eight softmax warps
  uint64_t* piece_full = q_full + 1;            // [kPieces]
  uint64_t* piece_empty = piece_full + kPieces; // [kPieces] softmax, converting and MMA warps
  uint64_t* group_bar = piece_empty + kPieces;  // the softmax warps
  uint64_t* drain = group_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ long long warp_sum[kLaunch / 32];
  __shared__ alignas(16) float scales[NS][12];      // per 32 keys: K's scale, log2 of V's, kSumUnit over V's
  __shared__ Piece pieces[kPieces];
  __shared__ Walk walk;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  let_merge_start();
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], kConvertWarps);
      mbar_init(&k_empty[s], 2);  // both MMA warps
      mbar_init(&v_full[s], kConvertWarps);
      mbar_init(&v_empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[2 * t + i], 1);
        mbar_init(&p_ready[2 * t + i], 4);
      }
      mbar_init(&pv_done[t], 1);
      mbar_init(&o_final[t], 1);
    }
    mbar_init(q_full, kSoftmaxWarps);
    for (int s = 0; s < kPieces; ++s) {
      mbar_init(&piece_full[s], 1);
      mbar_init(&piece_empty[s], kSoftmaxWarps + 2 * kConvertWarps + 2);
    }
    mbar_init(group_bar, kSoftmaxWarps);
    mbar_init(drain, 2);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
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
      const int count = span_of(p, b, (e - b * p.entries_per_seq) * kCacheTcRows, kCacheTcRows).count;
      x = count > 0 ? static_cast<long long>(count + kItemCost) * p.mult : 0;
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
  // row tiles without a visible key: zeros
  for (int e = blockIdx.x; e < entries; e += gridDim.x) {
    if (prefix[e + 1] != prefix[e]) continue;
    const int b = e / p.entries_per_seq, r0 = (e - b * p.entries_per_seq) * kCacheTcRows;
    const int rows = min(kCacheTcRows, p.s * p.group - r0);
    for (int i = tid; i < rows * p.Hkv * (D / 8); i += kLaunch) {
      const int c = i % (D / 8), hk = i / (D / 8) % p.Hkv, rr = r0 + i / (D / 8) / p.Hkv;
      const int tok = rr / p.group;
      __nv_bfloat16* dst =
          p.out + b * p.o_sb + (static_cast<long long>(tok) * p.H + hk * p.group + rr - tok * p.group) * D + c * 8;
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    }
  }

  if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------------ softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int t = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * kKeys + lane_off;
    const uint32_t tO = tmem + 2 * kKeys + t * D + lane_off;
    uint32_t tiles_before = 0, n_seg = 0, meetings = 0;
    uint32_t s_phase = 0, n_pv = 0;  // parity of each score buffer's next fill; steps so far
    bool ok = true;
    auto meet = [&]() {  // all softmax warps, with a limit (a named barrier would wait for a warp that gave up)
      __syncwarp();
      if (lane == 0) mbar_arrive(group_bar);
      ok = mbar_wait_warp(group_bar, meetings++ & 1, p.status, kTimeoutEpilogue, abort_flag) && ok;
    };
    for (; ok; ++n_seg) {
      if (!(ok = mbar_wait_warp(&piece_full[n_seg % kPieces], (n_seg / kPieces) & 1, p.status, kTimeoutEpilogue, abort_flag))) break;
      const Piece& x = pieces[n_seg % kPieces];
      const int count = x.count;
      if (count == 0) break;
      const bool both = x.both;
      const int rr = x.row0 + (both ? r : t * 128 + r);  // row of the KV head
      const bool row_ok = rr < p.s * p.group;
      const int tok = rr / p.group;
      const int head = x.hk * p.group + rr - tok * p.group;
      // ------------------------------ Q row: power of two, f16, swizzled tile
      // (every MMA of the last piece is done: this thread saw o_final)
      float factor;
      {
        const __nv_bfloat16* src = p.q + x.b * p.q_sb + (row_ok ? tok * p.q_ss + head * p.q_sh : 0);
        float amax = 0.f;
        uint4 raw[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          raw[c] = row_ok ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(u[e] << 16)), fabsf(__uint_as_float(u[e] & 0xffff0000u))));
        }
        float down, up;
        row_power(amax, down, up);
        factor = up * fabsf(p.scale_log2);
        if (p.scale_log2 < 0.f) down = -down;
        if (!both || t == 0) {
          uint8_t* tile = sQ + t * C::kQTile + r * 128;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              h[e] = pack_f16(__uint_as_float(u[e] << 16) * down, __uint_as_float(u[e] & 0xffff0000u) * down);
            *reinterpret_cast<uint4*>(tile + (c >> 3) * kChunkBytes + (((c & 7) ^ (r & 7)) << 4)) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      // ------------------------------ key tiles
      const int pos = x.base + tok;
      const int kmax = row_ok ? pos : -1;
      const int kmin = p.window >= 0 ? pos - p.window : 0;
      const int edge_hi = x.edge_hi, edge_lo = x.edge_lo, kt0 = x.kt0;
      // Step u of the group: 64 keys, half u & 1 of tile u / 2, or half t of tile u where the groups share the rows.
      const int u_end = both ? count : 2 * x.to[t];
      float m = -INFINITY, l = 0.f;  // running maximum of s + ev (may lag by < 2^8), row sum of 2^(s - m + shift)
      int n = 0;
      for (int u = both ? 0 : 2 * x.from[t]; u < u_end; ++u) {
        const int j = both ? u : u >> 1, half = both ? t : u & 1, buf = u & 1;
        const int k0 = (kt0 + j) * kKeys;
        const uint32_t tB = tS + buf * kHalf;
        if (!(ok = mbar_wait_warp(&s_full[2 * t + buf], s_phase >> buf & 1, p.status, kTimeoutEpilogue, abort_flag))) break;
        s_phase ^= 1u << buf;
        tc_fence_after();
        // the tile's scales come with its values
        const uint32_t tile_no = tiles_before + j;
        const int st = tile_no % NS;
        if (!(ok = mbar_wait_warp(&v_full[st], (tile_no / NS) & 1, p.status, kTimeoutEpilogue, abort_flag))) break;
        const float2 ks2 = *reinterpret_cast<const float2*>(&scales[st][2 * half]);
        const float2 ve2 = *reinterpret_cast<const float2*>(&scales[st][4 + 2 * half]);
        const float2 vi2 = *reinterpret_cast<const float2*>(&scales[st][8 + 2 * half]);
        float kc[2] = {positive(factor * ks2.x), positive(factor * ks2.y)};
        float ve[2] = {ve2.x, ve2.y};
        float vi[2] = {vi2.x, vi2.y};
        uint32_t va[32], vb[32];
        tmem_read_x32x2(tB, va, vb);
        if (k0 > edge_hi || k0 < edge_lo) {
          auto mask = [&](uint32_t(&v)[32], int c) {  // scores of keys 32c .. 32c + 31 of the tile
            // bit i: the row sees key i of these
            const int hi = kmax - k0 - 32 * c, lo = kmin - k0 - 32 * c;
            const uint32_t sees = (hi < 0 ? 0u : hi > 30 ? ~0u : (2u << hi) - 1u) & (lo <= 0 ? ~0u : lo > 31 ? 0u : ~0u << lo);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(sees >> i & 1)) v[i] = __float_as_uint(-INFINITY);
            if (sees == 0) {  // the row's weights are zero whatever the block's scales hold
              kc[c & 1] = 1.f;
              ve[c & 1] = vi[c & 1] = 0.f;
            }
          };
          mask(va, 2 * half);
          mask(vb, 2 * half + 1);
        }
        float a0 = -INFINITY, a1 = -INFINITY, b0 = -INFINITY, b1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {  // three-operand maxima in four chains
          a0 = fmaxf(fmaxf(a0, __uint_as_float(va[i])), __uint_as_float(va[i + 1]));
          b0 = fmaxf(fmaxf(b0, __uint_as_float(vb[i])), __uint_as_float(vb[i + 1]));
          a1 = fmaxf(fmaxf(a1, __uint_as_float(va[i + 2])), __uint_as_float(va[i + 3]));
          b1 = fmaxf(fmaxf(b1, __uint_as_float(vb[i + 2])), __uint_as_float(vb[i + 3]));
        }
        const float mx = fmaxf(fmaf(fmaxf(a0, a1), kc[0], ve[0]), fmaf(fmaxf(b0, b1), kc[1], ve[1]));
        const bool grow = mx > m + kRescaleThreshold;
        const bool scale_o = grow && n > 0 && m != -INFINITY;
        if (__any_sync(0xffffffffu, scale_o)) {
          // the last step's product must be in O; the one after it waits for this step's weights
          if (!(ok = mbar_wait_warp(&pv_done[t], (n_pv - 1) & 1, p.status, kTimeoutEpilogue, abort_flag))) break;
          tc_fence_after();
          const float d = scale_o ? m - mx : 0.f, f = fast_exp2(d);
          l = scale_sum(l, d);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_read_x16(tO + c * 16, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_32x32b_x16(tO + c * 16, o);
          }
        }
        if (grow) m = mx;
        const float ref = m == -INFINITY ? 0.f : kShift - m;
        // (one branch ahead of both halves: within them it cost 3 % of a long chunk's time)
        if (__builtin_expect(fminf(ve[0], ve[1]) < kTinyLog2, 0)) {
          auto sum_alone = [&](const uint32_t(&v)[32], int c) {
            if (!(ve[c] < kTinyLog2)) return;
            vi[c] = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) l = fmaf(fast_exp2(fmaf(__uint_as_float(v[i]), kc[c], ref)), kSumUnit, l);
          };
          sum_alone(va, 0);
          sum_alone(vb, 1);
        }
        auto weigh = [&](const uint32_t(&v)[32], int c) {
          const float add = ref + ve[c];
          const uint64_t mul2 = f2_pack(kc[c], kc[c]), add2 = f2_pack(add, add);
          uint64_t rs = f2_pack(0.f, 0.f);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), mul2, add2);
            float x0, x1;
            f2_unpack(x2, x0, x1);
            const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);  // (0 for a hidden key, in the sum as in P)
            const uint64_t e2 = f2_pack(e0, e1);
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(rs) : "l"(e2));
            pk[i] = pack_f16(e0, e1);
          }
          float r0, r1;
          f2_unpack(rs, r0, r1);
          l = fmaf(r0 + r1, vi[c], l);
          tmem_st_32x32b_x16(tB + 16 * c, pk);
        };
        weigh(va, 0);
        weigh(vb, 1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * t + buf]);
        ++n_pv;
        ++n;
      }
      if (!ok || !(ok = mbar_wait_warp(&o_final[t], n_seg & 1, p.status, kTimeoutEpilogue, abort_flag))) break;
      tc_fence_after();

      // ------------------------------ epilogue
      const bool whole = x.whole;
      const bool write = row_ok && (!both || t == 0);
      float f_own = 1.f, f_other = 0.f;  // merge of the two groups' results
      float* scratch = reinterpret_cast<float*>(smem + C::kOffScratch) + r * C::kScratchStride;
      if (both) {
        if (t == 1) {
          scratch[0] = m;
          scratch[1] = l;
        }
        meet();
        if (t == 0) {
          const float m2 = scratch[0], l2 = scratch[1];
          const float mm = fmaxf(m, m2);
          const float d = mm == -INFINITY ? 0.f : m - mm, d2 = mm == -INFINITY ? 0.f : m2 - mm;
          f_own = fast_exp2(d);
          f_other = fast_exp2(d2);
          l = scale_sum(l, d) + scale_sum(l2, d2);
          m = mm;
        }
        meet();
      }
      const float inv = l == 0.f ? 0.f : kSumUnit / l;
      float* part = p.part + ((2LL * blockIdx.x + x.begins) * kCacheTcRows + (both ? r : t * 128 + r)) * (D + 2);
      __nv_bfloat16* orow = p.out + x.b * p.o_sb + (static_cast<long long>(write ? tok : 0) * p.H + (write ? head : 0)) * D;
      if (write && !whole) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_read_x32(tO + c * 32, o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        float y[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(o[i]) * f_own;
        if (both) {
          if (t == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float4*>(scratch + 4 * i) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          }
          meet();
          if (t == 0 && ok) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 z = *reinterpret_cast<const float4*>(scratch + 4 * i);
              y[4 * i] = fmaf(z.x, f_other, y[4 * i]);
              y[4 * i + 1] = fmaf(z.y, f_other, y[4 * i + 1]);
              y[4 * i + 2] = fmaf(z.z, f_other, y[4 * i + 2]);
              y[4 * i + 3] = fmaf(z.w, f_other, y[4 * i + 3]);
            }
          }
          meet();
        }
        if (write && whole) {
          uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(pack_bf16x2(y[8 * i] * inv, y[8 * i + 1] * inv),
                                pack_bf16x2(y[8 * i + 2] * inv, y[8 * i + 3] * inv),
                                pack_bf16x2(y[8 * i + 4] * inv, y[8 * i + 5] * inv),
                                pack_bf16x2(y[8 * i + 6] * inv, y[8 * i + 7] * inv));
        } else if (write) {
#pragma unroll
          for (int i = 0; i < 16; ++i) *reinterpret_cast<float2*>(part + c * 32 + 2 * i) = make_float2(y[2 * i], y[2 * i + 1]);
        }
      }
      if (write && x.nan) store_nans<D>(p, x, x.base + tok, orow, part);
      if (!ok) break;
      tiles_before += count;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[n_seg % kPieces]);
    }
  } else if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ e4m3 -> f16 tiles
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    constexpr int PR = D / 16;              // 16-byte pieces per row
    constexpr int NP = kKeys * PR / 128;    // pieces per thread and tile, in two batches
    const bool is_v = warp >= kSoftmaxWarps + kConvertWarps;
    const int c = (tid - kSoftmaxWarps * 32) & 127;
    const int piece = c % PR, row_c = c / PR;  // piece i: row row_c + i * (128 / PR)
    uint8_t* tiles = is_v ? sV : sK;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    // The tile behind the next one is brought into L2 where several row tiles read it (a 2048-token chunk over
    // 32768 tokens: 1256 us without, 1228 with it); read once, it only costs the asking (five tokens each of 8
    // sequences: 69 us without, 71 with it).
    const bool far_ahead = p.tiles > 1 && c == 0;
    uint32_t tile_no = 0;
    bool ok = true;
    for (uint32_t seg = 0; ok; ++seg) {
      if (!(ok = mbar_wait_warp(&piece_full[seg % kPieces], (seg / kPieces) & 1, p.status, kTimeoutProducer, abort_flag))) break;
      Piece& x = pieces[seg % kPieces];
      const int count = x.count;
      if (count == 0) break;
      const int n_keys = x.n, edge_hi = x.edge_hi, edge_lo = x.edge_lo;
      const uint8_t* src = (is_v ? p.v + x.b * p.v_sb + x.hk * p.v_sh : p.k + x.b * p.k_sb + x.hk * p.k_sh) + piece * 16;
      // lanes 0-3 of the first V warp bring K's scales of the tile's blocks, lanes 4-7 V's
      const bool brings = is_v && c < 8;
      const float* scale = c < 4 ? p.k_scale + x.b * p.ks_sb + x.hk * p.ks_sh : p.v_scale + x.b * p.vs_sb + x.hk * p.vs_sh;
      // (blocks of the tile that no row sees may hold anything: their scales are not read)
      const int blocks = (n_keys + kCacheBlock - 1) / kCacheBlock, lo_block = x.lo_block;
      auto scale_at = [&](int k0) {
        const int blk = k0 / kCacheBlock + (c & 3);
        return brings && blk >= lo_block && blk < blocks ? scale[blk] : 1.f;
      };
      int k0 = x.kt0 * kKeys;
      uint4 raw[NP];
      auto load = [&](int from, int to, int base) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (i < from || i >= to) continue;
          const int row = base + row_c + i * (128 / PR);
          raw[i] = row < n_keys ? load16(src + static_cast<long long>(row) * D) : make_uint4(0, 0, 0, 0);
        }
      };
      load(0, NP, k0);
      float sc = scale_at(k0);
      for (int j = 0; j < count; ++j, ++tile_no, k0 += kKeys) {
        const int st = tile_no % NS;
        if (!(ok = mbar_wait_warp(&empty[st], ((tile_no / NS) & 1) ^ 1u, p.status, kTimeoutProducer, abort_flag))) break;
        if (brings) {
          scales[st][c] = c < 4 ? sc : __log2f(sc);
          if (c >= 4) scales[st][4 + c] = kSumUnit / sc;
          if (j + 1 < count) sc = scale_at(k0 + kKeys);
        }
        if (is_v && (k0 > edge_hi || k0 < edge_lo)) {
          // an edge tile: values that are NaN become zero here, and the rows' ends are told to look for them
          uint32_t any = 0;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const uint32_t a = nan_bytes(raw[i].x), b2 = nan_bytes(raw[i].y), c2 = nan_bytes(raw[i].z), d2 = nan_bytes(raw[i].w);
            raw[i] = make_uint4(raw[i].x & ~a, raw[i].y & ~b2, raw[i].z & ~c2, raw[i].w & ~d2);
            any |= a | b2 | c2 | d2;
          }
          if (any != 0) x.nan = 1;
        }
        uint8_t* tile = tiles + st * C::kQTile;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int i = half * NP / 2; i < (half + 1) * NP / 2; ++i) {
            const int row = row_c + i * (128 / PR);
            uint8_t* base = tile + (piece >> 2) * kChunkBytes + row * 128;
            // the pieces of a row's two 64-channel chunks share banks: the upper chunk's lanes store
            // their halves in the other order
            const int p0 = 2 * (piece & 3);
            const bool swap = piece >= 4;
            const uint32_t u[4] = {swap ? raw[i].z : raw[i].x, swap ? raw[i].w : raw[i].y, swap ? raw[i].x : raw[i].z,
                                   swap ? raw[i].y : raw[i].w};
            uint32_t f[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[2 * e] = f16x2_of(u[e]);
              f[2 * e + 1] = f16x2_of_upper(u[e]);
            }
            *reinterpret_cast<uint4*>(base + (((p0 + swap) ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<uint4*>(base + (((p0 + !swap) ^ (row & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
          }
          if (j + 1 < count) load(half * NP / 2, (half + 1) * NP / 2, k0 + kKeys);
          if (far_ahead && half == 0 && j + 2 < count) {
            const int ahead = k0 + 2 * kKeys, bytes = min(kKeys, n_keys - ahead) * D;
            if (bytes > 0)
              asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src + static_cast<long long>(ahead) * D), "r"(bytes));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[seg % kPieces]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == kWalkWarp && lane == 0) {
      // ---------------------------------------------------------------- the run's pieces
      const long long run = max((total + gridDim.x - 1) / gridDim.x, 2LL + kItemCost);
      const long long from = min(blockIdx.x * run, total);
      walk.start(p, prefix, from, min(from + run, total), run);
      for (uint32_t seg = 0;; ++seg) {
        Piece& x = pieces[seg % kPieces];
        if (!mbar_wait(&piece_empty[seg % kPieces], ((seg / kPieces) & 1) ^ 1u, p.status, kTimeoutProducer, abort_flag)) break;
        walk.next(p, prefix, x);
        mbar_arrive(&piece_full[seg % kPieces]);
        if (x.count == 0) break;
      }
      put_cut(p, blockIdx.x, walk.cut);
    } else if (warp < kMmaWarp + 2) {
      // ---------------------------------------------------------------- MMA issuers
      // One warp per group: neither group's next product waits in program order for the other's weights.
      // The whole warp walks along, so that its scalars stay in uniform registers.
      constexpr uint32_t idesc_s = idesc_f16(128, kHalf, false);
      constexpr uint32_t idesc_o = idesc_f16(128, D, true);
      const bool leader = elect_one();
      const uint32_t t = uniform(static_cast<uint32_t>(warp - kMmaWarp));
      const uint32_t t_s = uniform(tmem) + t * kKeys, t_o = uniform(tmem) + 2 * kKeys + t * D;
      const uint32_t q0_low = uniform(desc_low(smem_u32(sQ), 16));
      const uint32_t k0_low = uniform(desc_low(smem_u32(sK), 16)), v0_low = uniform(desc_low(smem_u32(sV), kChunkBytes));
      uint32_t tile_no = 0, p_phase = 0;
      bool ok = true;
      for (uint32_t seg = 0; ok; ++seg) {
        if (!(ok = mbar_wait_warp(&piece_full[seg % kPieces], (seg / kPieces) & 1, p.status, kTimeoutMma, abort_flag))) break;
        const Piece& x = pieces[seg % kPieces];
        const int jn = uniform(x.count);
        if (jn == 0) break;
        if (!(ok = mbar_wait_warp(q_full, seg & 1, p.status, kTimeoutMma, abort_flag))) break;
        tc_fence_after();
        const bool both = uniform(x.both);
        const int steps = both ? jn : 2 * jn;
        const int from = both ? 0 : 2 * uniform(x.from[t]), to = both ? jn : 2 * uniform(x.to[t]);
        __syncwarp();
        if (leader) mbar_arrive(&piece_empty[seg % kPieces]);
        const uint32_t q_low = q0_low + (both ? 0 : t * (C::kQTile / 16));
        uint32_t more = 0;  // whether O_t holds products of this piece
        for (int u = -2; u < steps; ++u) {
          if (u >= 0) {  // O_t += P_t V of step u
            const uint32_t no = tile_no + (both ? u : u >> 1), st = no % NS, half = both ? t : u & 1, buf = u & 1;
            // A group that does not see the tile waits for it all the same: releasing tiles ahead of their
            // being filled, it would stand in for the other group's release.
            if (!(ok = mbar_wait_warp(&v_full[st], (no / NS) & 1, p.status, kTimeoutMma, abort_flag))) break;
            if (u >= from && u < to) {
              if (!(ok = mbar_wait_warp(&p_ready[2 * t + buf], p_phase >> buf & 1, p.status, kTimeoutMma, abort_flag))) break;
              p_phase ^= 1u << buf;
              tc_fence_after();
              const uint32_t v_low = v0_low + (st * C::kQTile + half * (kHalf * 128)) / 16, pw = t_s + buf * kHalf;
              if (leader) {
#pragma unroll
                for (int kk = 0; kk < kHalf / 16; ++kk)
                  mma_ts(t_o, pw + kk * 8, v_low + kk * (2048 / 16), idesc_o, kk > 0 ? 1 : more);
                umma_commit(&pv_done[t]);
              }
              more = 1;
            }
            if ((both || half == 1) && leader) umma_commit(&v_empty[st]);
          }
          if (u + 2 < steps) {  // S_t of the step after the next, into the buffer that step u left
            const uint32_t w = u + 2, no = tile_no + (both ? w : w >> 1), st = no % NS, half = both ? t : w & 1, buf = w & 1;
            if (!(ok = mbar_wait_warp(&k_full[st], (no / NS) & 1, p.status, kTimeoutMma, abort_flag))) break;
            if (static_cast<int>(w) >= from && static_cast<int>(w) < to) {
              tc_fence_after();
              const uint32_t k_low = k0_low + (st * C::kQTile + half * (kHalf * 128)) / 16, d = t_s + buf * kHalf;
              if (leader) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                  const uint32_t step = ((kk >> 2) * kChunkBytes + (kk & 3) * 32) / 16;
                  mma_ss(d, q_low + step, k_low + step, idesc_s, kk > 0);
                }
                umma_commit(&s_full[2 * t + buf]);
              }
            }
            if ((both || half == 1) && leader) umma_commit(&k_empty[st]);
          }
        }
        if (leader) umma_commit(&o_final[t]);
        tile_no += jn;
      }
      if (leader) {
        umma_commit(drain);
        mbar_wait(drain, 0, p.status, kTimeoutDrain, nullptr);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) {
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

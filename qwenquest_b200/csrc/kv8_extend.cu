// Causal attention of an extend batch over the 8-bit block cache on the
// fifth-generation tensor cores (bf16 queries, head_dim 128, any group).
//
// Bound by the two products and the exponentials, so the codes are widened
// to fp16 once per tile (exact: e4m3 has 4 significant bits and no exponent
// outside fp16's) by warps of their own, and both products run at fp16's
// rate.  fp16 also holds the operands of the other side better than bf16
// would: a query row is scaled by a power of two to at most 256 (exact down
// to 2^-25 of its largest element), the weights carry 11 bits.
//
// Rows: the new tokens of an entry times the query heads of one KV head,
// token-major; a CTA takes 256 of them (two M tiles of 128) against key tiles
// of 128, so short chunks fill the tiles with heads and every key tile
// serves 256 rows.  Where the last units leave SMs idle their keys are cut into
// stretches whose (M, l, O) records kv8_extend_join_kernel merges.
// Scales: as in the one-token kernel a score is S ks / up, the weight into
// the V product 2^(s + lg - M) with lg = log2(vs), and the sum takes that
// times 2^(-lg - kTop): constants of a group of 16 keys (no block is shorter).
// Warps: 0-7 softmax (thread = row = TMEM lane; 0-3 tile 0, 4-7 tile 1),
// 8-11 widen K and V, 12-13 MMA issue (one per M tile), 14 scales.
// Tensor memory: per M tile S (128 fp32 columns, overlaid by P in fp16 once
// read) and O (128).  The order per tile is S(j) P(j) O(j) S(j + 1): while
// one tile's softmax runs the tensor cores work for the other.
// The weights' reference is raised only past kRaiseAt; O is rescaled then.
// Every wait is bounded; see the one-token kernel.

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include <cuda_fp16.h>

#include "kv8_tma.cuh"

namespace qq {
namespace kv8 {
namespace {

using namespace tc;

constexpr int kM = 128, kN = 128;            // rows and keys per tile
constexpr int kUnitRows = 2 * kM;                // query rows per CTA
constexpr int kTileBytes = 128 * kTcDim * 2; // 32 KiB: 128 rows of fp16, two 64-column blocks
constexpr int kHalf = kTileBytes / 2;
constexpr int kStages = 2;                   // K tiles and V tiles in shared memory
constexpr int kMeta = 4;
constexpr int kGroups = kN / 16;               // groups of 16 keys at most in a tile
constexpr int kWidenWarp = 8, kMmaWarp = 12, kScaleWarp = 14;
constexpr int kThreads = 16 * 32;  // four warpgroups
// Registers per thread: 128 at launch (all 65,536 over 512 threads), then by role.
constexpr int kRegsSoft = 152, kRegsWiden = 120, kRegsRest = 88;
static_assert(128 * (2 * kRegsSoft + kRegsWiden + kRegsRest) <= kThreads * 128, "the launch's registers");
constexpr int kOffQ = 0, kOffK = 2 * kTileBytes, kOffV = kOffK + kStages * kTileBytes;
constexpr int kDynSmem = kOffV + kStages * kTileBytes + 1024;
constexpr uint32_t kTmemCols = 512;
// Where the weights lie in fp16 (2^-24 to 2^16): the largest key of the first tile gets 2^kTop.  A half tile's sum past
// kRaiseAt raises the reference until it is 2^kTop again, one past kMost is made again.  So the steps are 2^-31 of some
// half tile's weights, together.  Rows whose sums have passed kAlong are raised with another row of their warp: 579 us
// for the 8,192 tokens of a prompt where each row on its own took 590 and no kTop 571 (chunks: 154, 158, 151).
constexpr float kTop = 7.f, kRaiseAt = 16384.f, kMost = 60000.f, kAlong = 256.f;

enum : int {
  kBarQ = 0,                          // [2] queries of a tile written
  kBarK = kBarQ + 2,                  // [stages] keys written
  kBarKFree = kBarK + kStages,        // [stages] read by both tiles' MMAs
  kBarV = kBarKFree + kStages,
  kBarVFree = kBarV + kStages,
  kBarMeta = kBarVFree + kStages,     // [kMeta] scales written
  kBarMetaFree = kBarMeta + kMeta,
  kBarS = kBarMetaFree + kMeta,       // [2] scores made
  kBarP = kBarS + 2,                  // [2][2] weights of a tile's first and second 64 keys written
  kBarO = kBarP + 4,                  // [2] the product of a tile's first 64 keys made
  kBarDone = kBarO + 2,               // [2] the tile's last MMA has finished
  kBarLag = kBarDone + 2,             // [2] the first tile's softmax is at it (key tiles in turn)
  kNumBars = kBarLag + 2
};

struct ExtendArgs {
  AttnArgs a;
  int tiles;   // units of a KV head at most
  int sms;
  int most;    // stretches of a unit at most
};

// A stretch's record of a unit: (M, l) of 256 rows, then O [256][128].
constexpr int64_t kRecord = kUnitRows * (2 + (int64_t)kTcDim);

// fp16 operands, fp32 accumulator.
constexpr uint32_t kIdS = (1u << 4) | ((kN >> 3) << 17) | ((kM >> 4) << 24);
constexpr uint32_t kIdO = (1u << 4) | (1u << 16) | ((kTcDim >> 3) << 17) | ((kM >> 4) << 24);

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four e4m3 codes as two fp16 pairs (exact).
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
// acc = 0 h + acc in every half: NaN once one of h is (on the FMA pipe, which has room).
__device__ __forceinline__ void nan_of(uint32_t& acc, const uint4& h) {
  asm("fma.rn.f16x2 %0, %1, %5, %0;\n\tfma.rn.f16x2 %0, %2, %5, %0;\n\t"
      "fma.rn.f16x2 %0, %3, %5, %0;\n\tfma.rn.f16x2 %0, %4, %5, %0;"
      : "+r"(acc)
      : "r"(h.x), "r"(h.y), "r"(h.z), "r"(h.w), "r"(0));
}
// Loads under a predicate that leave their registers alone until they land (a
// select behind a load would wait for it on the spot).
__device__ __forceinline__ uint2 load8_or_zero(const void* p, bool there) {
  uint2 r;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
      "@p ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];\n\t}\n"
      : "=&r"(r.x), "=&r"(r.y)
      : "l"(p), "r"((int)there));
  return r;
}
__device__ __forceinline__ uint4 load16_or_zero(const void* p, bool there) {
  uint4 r;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\t"
      "mov.u32 %3, 0;\n\t@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}\n"
      : "=&r"(r.x), "=&r"(r.y), "=&r"(r.z), "=&r"(r.w)
      : "l"(p), "r"((int)there));
  return r;
}
__device__ __forceinline__ int32_t load_or(const int32_t* p, bool there, int32_t other) {
  int32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.u32 %0, %3;\n\t@p ld.global.nc.u32 %0, [%1];\n\t}\n"
      : "=&r"(r)
      : "l"(p), "r"((int)there), "r"(other));
  return r;
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Two fp32 numbers in a register pair: one instruction of the fp32 pipe for both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 both_of(f32x2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 x, f32x2 y, f32x2 z) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 x, f32x2 y) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
// The units of the batch, the ones with the most keys first: entries and their
// tiles from the last to the first, KV heads innermost.  SMs take a unit each at
// a time, so the last units, which would leave SMs idle, are cut into `splits`
// stretches of the keys, each of at least four key tiles (188 units of 35 to 47
// key tiles on 148 SMs: 148 + 40 x 3 CTAs in 150 us; all whole 182, all cut in
// two 175).  A batch with fewer units than SMs is cut throughout.
struct Units {
  int tiles, whole, splits;
};

// A unit or a stretch of one (all within 32 bits: at most 65535 tiles of 256
// rows, and positions of a table of less than 2^31 tokens).
struct Unit {
  int entry;               // -1: none
  int kvh;
  int q_row;               // the entry's first query row
  int prefix;
  int row0, rows;          // rows [row0, row0 + rows) of the entry's n * group
  int splits;              // stretches of the unit, 1: this is all of it
  int key_begin, key_end;
  int tiles;
  const int32_t* table;    // the request's blocks
};
// The unit that choose(units, index, split) names; called by one whole warp.  A
// batch of up to 32 entries is read once.
template <typename Choose>
__device__ __forceinline__ Unit find_unit(const ExtendArgs& g, uint32_t* err, Choose choose) {
  const AttnArgs& a = g.a;
  const int lane = threadIdx.x & 31;
  int64_t row0 = 0, pre = 0;
  auto tiles_of = [&](int e, int& n, uint32_t* report) {
    n = (int)extend_entry(a, e, row0, pre, report);
    return (n * a.group + kUnitRows - 1) / kUnitRows;
  };
  int n, mine = tiles_of(lane, n, err), all = mine;
  for (int e = lane + 32; e < a.bs; e += 32) {
    int other;
    all += tiles_of(e, other, err);
  }
  all = __reduce_add_sync(0xffffffffu, all);
  if (all > g.tiles) raise_error(err, QQ_DEV_ERR_BOUNDS);  // entries share query rows
  Units units;
  units.tiles = min(all, g.tiles);
  const int total = units.tiles * a.c.kv_heads, rest = total % g.sms;
  units.splits = rest == 0 ? 1 : min(g.most, g.sms / rest);
  units.whole = units.splits == 1 ? total : total - rest;
  int index = 0, split = 0;
  choose(units, index, split);
  Unit u{};
  u.entry = -1;
  const int back = index / a.c.kv_heads, tile = units.tiles - 1 - back;
  if (tile < 0) return u;
  int before = 0;
  for (int e0 = 0; e0 < a.bs; e0 += 32) {
    if (a.bs > 32) mine = tiles_of(e0 + lane, n, nullptr);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const int excl = before + incl - mine;
    const uint32_t m = __ballot_sync(0xffffffffu, tile >= excl && tile < excl + mine);
    if (m == 0) {
      before += __shfl_sync(0xffffffffu, incl, 31);
      continue;
    }
    const int src = __ffs(m) - 1, entry = e0 + src;
    u.kvh = index - back * a.c.kv_heads;
    u.q_row = (int)__shfl_sync(0xffffffffu, row0, src);
    u.prefix = (int)__shfl_sync(0xffffffffu, pre, src);
    u.row0 = (tile - __shfl_sync(0xffffffffu, excl, src)) * kUnitRows;
    u.rows = min(kUnitRows, __shfl_sync(0xffffffffu, n, src) * a.group - u.row0);
    u.table = a.table + a.reqs[entry] * a.table_stride;
    const int keys = u.prefix + (u.row0 + u.rows - 1) / a.group + 1;  // what its last row sees
    const int key_tiles = (keys + kN - 1) / kN;
    const int cuts = index < units.whole ? 1 : min(units.splits, (key_tiles + 3) / 4), each = (key_tiles + cuts - 1) / cuts;
    u.splits = (key_tiles + each - 1) / each;
    if (split >= u.splits) return u;
    u.entry = entry;
    u.key_begin = split * each * kN;
    u.key_end = min(keys, u.key_begin + each * kN);
    u.tiles = (u.key_end - u.key_begin + kN - 1) / kN;
    return u;
  }
  return u;
}

// kGroup: keys that share their scales, 16, or 64 where blocks are that long.
template <int kGroup>
__global__ void __launch_bounds__(kThreads, 1) kv8_extend_kernel(ExtendArgs g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kNumBars];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Unit s_unit;
  __shared__ int s_record;  // of a stretch
  __shared__ float s_up[kUnitRows];                                   // scale_log2 / up of each row
  __shared__ __align__(16) float4 s_scale[kMeta][kGroups];        // ks, lg, 2^(-lg - kTop) of 16 keys
  const AttnArgs& a = g.a;
  const Cache& c = a.c;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  // the same in all lanes, and known to be
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  volatile int* abort_flag = &s_abort;
  auto wait = [&](int i, uint32_t parity) { return mbar_wait<8>(bar(i), parity, abort_flag, a.err); };
  wait_prior_grid();

  if (warp == 0) {
    int cut = 0;
    const Unit u = find_unit(g, blockIdx.x == 0 ? a.err : nullptr, [&](const Units& units, int& index, int& split) {
      cut = max(0, (int)blockIdx.x - units.whole);
      index = min((int)blockIdx.x, units.whole) + cut / units.splits;
      split = cut % units.splits;
    });
    if (lane == 0) s_unit = u, s_record = cut;
  }
  if (threadIdx.x == 32) {
    s_abort = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kBarQ + i), 4);
      mbar_init(bar(kBarS + i), 1);
      mbar_init(bar(kBarP + 2 * i), 4);
      mbar_init(bar(kBarP + 2 * i + 1), 4);
      mbar_init(bar(kBarO + i), 1);
      mbar_init(bar(kBarDone + i), 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar(kBarK + i), 4);
      mbar_init(bar(kBarV + i), 4);
      mbar_init(bar(kBarKFree + i), 2);
      mbar_init(bar(kBarVFree + i), 2);
    }
    for (int i = 0; i < kMeta; ++i) {
      mbar_init(bar(kBarMeta + i), 1);
      mbar_init(bar(kBarMetaFree + i), 8);
    }
    mbar_init(bar(kBarLag), 4);
    mbar_init(bar(kBarLag + 1), 4);
    mbar_init_fence();
  }
  if (warp == kMmaWarp) tmem_alloc(smem_u32(&s_tmem), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  allow_next_grid();  // not before the tensor memory is this CTA's
  const Unit& u = s_unit;
  const int kvh = u.kvh;
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  if (u.entry < 0) {  // past the last unit, uniform
    if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  const int tiles = __shfl_sync(0xffffffffu, u.tiles, 0);

  if (warp < kWidenWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
    // ================================================================ softmax (warps 0-7)
    const int h = warp >> 2, r = threadIdx.x;      // row of the CTA's 256
    const int token = (u.row0 + r) / a.group;
    // ---- this warp's 32 query rows to fp16: four lanes per row, 32 channels
    // each, all of it asked for at once
    uint4 ask[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = warp * 32 + i * 8 + (lane >> 2);
      const int t = (u.row0 + rr) / a.group, hd = kvh * a.group + u.row0 + rr - t * a.group;
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) +
                                                      (int64_t)(u.q_row + t) * a.q_stride + (int64_t)hd * kTcDim +
                                                      (lane & 3) * 32);
#pragma unroll
      for (int k = 0; k < 4; ++k) ask[i][k] = load16_or_zero(q + k, rr < u.rows);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = warp * 32 + i * 8 + (lane >> 2);
      uint32_t w[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[4 * k] = ask[i][k].x, w[4 * k + 1] = ask[i][k].y, w[4 * k + 2] = ask[i][k].z, w[4 * k + 3] = ask[i][k].w;
      // magnitudes compare as integers
      auto largest = [&]() {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) top = __vmaxu2(top, w[k] & 0x7FFF7FFFu);
        return max(top & 0xFFFF0000u, top << 16);
      };
      uint32_t most = largest();
      if (most >= 0x7F800000u) {
        // an infinite query has no scores either: NaN, and left out of the maximum
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          uint32_t fine = w[k] & 0x7FFF7FFFu;
          if ((w[k] & 0x7F80u) == 0x7F80u) w[k] |= 0x7FFFu, fine &= 0xFFFF0000u;
          if ((w[k] & 0x7F800000u) == 0x7F800000u) w[k] |= 0x7FFF0000u, fine &= 0xFFFFu;
          top = __vmaxu2(top, fine);
        }
        most = max(top & 0xFFFF0000u, top << 16);
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int k2 = max(-120, fit_exponent(__uint_as_float(most)) - 1);  // at most 224
      const float up = a.scale_log2 < 0.f ? -exp2_int(k2) : exp2_int(k2);
      uint8_t* dst = smem + kOffQ + h * kTileBytes + (lane & 2) / 2 * kHalf + (rr & 127) * 128;
      auto scaled = [&](uint32_t x) { return pack_f16(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xFFFF0000u) * up); };
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint4*>(dst + ((((lane & 1) * 4 + k) ^ (rr & 7)) << 4)) =
            make_uint4(scaled(w[4 * k]), scaled(w[4 * k + 1]), scaled(w[4 * k + 2]), scaled(w[4 * k + 3]));
      if ((lane & 3) == 0) s_up[rr] = fabsf(a.scale_log2) * exp2_int(-k2);
    }
    fence_async_shared();
    mbar_arrive_warp(bar(kBarQ + h));
    __syncwarp();
    const float inv_up = s_up[r];

    const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + h * 256, tO = tS + 128;
    const int reach = u.prefix + token - u.key_begin;  // the last key this row sees, in its stretch
    // The weights' reference m need not be the running maximum, only near
    // enough for fp16 and fp32: it starts kTop below the maximum of the first
    // tile with a key, and is raised where a half tile's sum passes kRaiseAt,
    // for the tiles to come.  So the scores are read once; a half whose sum
    // passes kMost (a weight might not fit fp16) is made again from the tile's
    // maximum.  Without kTop (the largest key a weight of 1) a long tail would
    // lose its bits behind one key with most of the mass: 131,072 even keys
    // behind one of 99 % and a small value were off by 21 % of the result.
    float m = -INFINITY, l = 0.f, alpha = 1.f;  // O still has to be multiplied by alpha
    bool ok = true;
    const int sees = __reduce_min_sync(0xffffffffu, reach);  // the last key that all of the warp's rows see
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int meta = j % kMeta;
      ok = __all_sync(0xffffffffu, wait(kBarMeta + meta, (j / kMeta) & 1) && wait(kBarS + h, j & 1));
      if (!ok) break;
      tc_fence_after();
      // columns c <= lim are seen by this row
      const int lim = max(-1, min(kN - 1, reach - j * kN));
      const bool full = sees - j * kN >= kN - 1;
      uint32_t v[2][32];  // scores in chunks of 32 columns, the next one always on its way
      float part, sum;    // of the half in hand: what l takes, and the plain sum
      float most = 0.f;   // the larger of the halves' sums
      uint32_t pk[32];
      // The maximum (with its scales) over the chunks from k0 on; the two buffers are free afterwards.
      auto highest = [&](int k0) {
        float mb = -INFINITY;
#pragma unroll 1
        for (int k = k0; k < 4; ++k) {
          tmem_ld32(tS + k * 32, v[0]);
          tmem_wait_ld32(v[0]);
#pragma unroll
          for (int q = 0; q < 32; q += kGroup) {
            const float4 f = s_scale[meta][(k * 32 + q) / kGroup];
            float y = -INFINITY;
#pragma unroll
            for (int e = 0; e < (kGroup < 32 ? kGroup : 32); ++e)
              y = fmaxf(y, k * 32 + q + e <= lim ? __uint_as_float(v[0][q + e]) : -INFINITY);
            // a masked group (-inf) stays -inf also where its scale is 0
            mb = fmaxf(mb, y == -INFINITY ? y : fmaf(y, inv_up * f.x, f.y));
          }
        }
        return mb;
      };
      // O times alpha: no product is under way (S(j) was committed behind O(j - 1))
      auto rescale = [&]() {
#pragma unroll 1
        for (int k = 0; k < kTcDim / 32; ++k) {
          tmem_ld32(tO + k * 32, v[0]);
          tmem_wait_ld32(v[0]);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[0][e] = __float_as_uint(__uint_as_float(v[0][e]) * alpha);
          tmem_st32(tO + k * 32, v[0]);
        }
        tmem_st_wait();
        alpha = 1.f;
      };
      if (__any_sync(0xffffffffu, m == -INFINITY)) {
        const float mb = highest(0);
        if (m == -INFINITY) m = mb - kTop;
      }
      if (__any_sync(0xffffffffu, alpha != 1.f)) rescale();  // after a tile, so O is there
      tmem_ld32(tS, v[0]);
      if (h == 0) mbar_arrive_warp(bar(kBarLag + (j & 1)));

      // P of chunk k (v[k & 1]) into pk, its sums into part and sum
      auto chunk = [&](int k, auto is_full) {
        const uint32_t(&x)[32] = v[k & 1];
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int q = 0; q < 32; q += kGroup) {
          const float4 f = s_scale[meta][(k * 32 + q) / kGroup];
          const float mul = inv_up * f.x, add = f.y - ref;
          const f32x2 mul_2 = pair(mul, mul), add_2 = pair(add, add);
          f32x2 s[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < (kGroup < 32 ? kGroup : 32); e += 2) {
            const f32x2 y = fma2(pair(__uint_as_float(x[q + e]), __uint_as_float(x[q + e + 1])), mul_2, add_2);
            const float2 t = both_of(y);
            float2 w = make_float2(ex2(t.x), ex2(t.y));
            if (!is_full.value) {
              w.x = k * 32 + q + e <= lim ? w.x : 0.f;
              w.y = k * 32 + q + e + 1 <= lim ? w.y : 0.f;
            }
            s[(e >> 1) & 1] = add2(s[(e >> 1) & 1], pair(w.x, w.y));
            pk[(k & 1) * 16 + (q + e) / 2] = pack_f16(w.x, w.y);
          }
          const float2 s2 = both_of(add2(s[0], s[1]));
          part = fmaf(s2.x + s2.y, f.z, part);
          sum += s2.x + s2.y;
        }
      };
      // 64 keys: weights, sums, P, and word to the MMA warp.  P goes over columns
      // whose scores have been read; the product of the first half runs while
      // the second half's exponentials do.
      auto half = [&](int hf, auto is_full) {
        for (int tries = 0;; ++tries) {
          part = 0.f, sum = 0.f;
          tmem_wait_ld32(v[0]);
          tmem_ld32(tS + hf * 64 + 32, v[1]);
          chunk(2 * hf, is_full);
          tmem_wait_ld32(v[1]);
          if (hf == 0) tmem_ld32(tS + 64, v[0]);
          chunk(2 * hf + 1, is_full);
          const bool over = sum > kMost;
          if (tries == 1 || !__any_sync(0xffffffffu, over)) break;
          if (hf == 0) tmem_wait_ld32(v[0]);
          const float mb = highest(2 * hf);  // P of the first half lies over its scores by now
          if (over) {
            alpha = ex2(m - (mb - kTop));
            l *= alpha;
            most *= alpha;
            m = mb - kTop;
          }
          if (hf == 1) ok = __all_sync(0xffffffffu, ok && wait(kBarO + h, j & 1));
          tc_fence_after();
          if (ok && (hf == 1 || j > 0)) rescale();
          alpha = 1.f;
          tmem_ld32(tS + hf * 64, v[0]);
        }
        l += part;
        tmem_st32(tS + hf * 32, pk);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive_warp(bar(kBarP + 2 * h + hf));
        most = fmaxf(most, sum);
      };
      if (full) {
        half(0, std::true_type{});
        half(1, std::true_type{});
      } else {
        half(0, std::false_type{});
        half(1, std::false_type{});
      }
      // for the tiles to come; a warp's rows together, since one that raises holds up all
      if (__any_sync(0xffffffffu, most > kRaiseAt) && most > kAlong) {
        const float up = __log2f(most) - kTop;
        m += up;
        alpha = ex2(-up);
        l *= alpha;
      }
      mbar_arrive_warp(bar(kBarMetaFree + meta));
    }
    // ---- O / l, or this stretch's record.  The rows go through this warp's part
    // of Q's memory (the products are done with it), so that 16 lanes write a
    // row's 256 bytes together.
    ok = __all_sync(0xffffffffu, ok && (tiles == 0 || wait(kBarDone + h, 0)));
    tc_fence_after();
    const bool record = u.splits > 1;
    const float to_l = alpha * exp2f(-kTop), f = record ? to_l : (l == 0.f ? 0.f : to_l / l);
    float* rec = a.part + (int64_t)s_record * kRecord;
    if (record && ok && r < u.rows) rec[2 * r] = m, rec[2 * r + 1] = l;
    const int rows = ok ? u.rows : 0;
    uint8_t* const stage = smem + kOffQ + warp * (kTileBytes / 4);  // 32 rows of 256 bytes, 16-byte pieces swizzled by the row
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {  // 64 channels: a row of the record's half, or half a row of bf16
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t o[32] = {};
        if (tiles > 0 && ok) {
          tmem_ld32(tO + part * 64 + k * 32, o);
          tmem_wait_ld32(o);
        }
        if (record) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stage + lane * 256 + (((k * 8 + e) ^ (lane & 15)) << 4)) =
                make_float4(__uint_as_float(o[4 * e]) * f, __uint_as_float(o[4 * e + 1]) * f,
                            __uint_as_float(o[4 * e + 2]) * f, __uint_as_float(o[4 * e + 3]) * f);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(stage + lane * 256 + (((part * 8 + k * 4 + e) ^ (lane & 15)) << 4)) =
                make_uint4(pack_bf16(__uint_as_float(o[8 * e + 0]) * f, __uint_as_float(o[8 * e + 1]) * f),
                           pack_bf16(__uint_as_float(o[8 * e + 2]) * f, __uint_as_float(o[8 * e + 3]) * f),
                           pack_bf16(__uint_as_float(o[8 * e + 4]) * f, __uint_as_float(o[8 * e + 5]) * f),
                           pack_bf16(__uint_as_float(o[8 * e + 6]) * f, __uint_as_float(o[8 * e + 7]) * f));
        }
      }
      if (!record && part == 0) continue;
      __syncwarp();
      const int first = u.row0 + warp * 32 + (lane >> 4);
      int t = first / a.group, hd = first - t * a.group;  // of the row at hand
#pragma unroll 4
      for (int k = 0; k < 16; ++k) {  // two rows at a time
        const int row = 2 * k + (lane >> 4), rr = warp * 32 + row;
        if (rr >= rows) break;
        const uint4 w = *reinterpret_cast<const uint4*>(stage + row * 256 + (((lane & 15) ^ (row & 15)) << 4));
        if (record) {
          *reinterpret_cast<uint4*>(rec + 2 * kUnitRows + (int64_t)rr * kTcDim + part * 64 + (lane & 15) * 4) = w;
        } else {
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (int64_t)(u.q_row + t) * a.out_stride +
                                    (int64_t)(kvh * a.group + hd) * kTcDim + (lane & 15) * 8) = w;
          for (hd += 2; hd >= a.group; hd -= a.group) ++t;
        }
      }
      __syncwarp();
    }
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsWiden));
    // ================================================================ K and V to fp16
    // Sixteen lanes per key row, 8 codes each; a warp's 32 rows in sixteen steps.
    // The codes of the next tile are on their way while one is widened.
    const int ww = warp - kWidenWarp, hr = lane >> 4, ch = lane & 15;
    // lane L looks after key ww * 32 + L of a tile: its block (-1 past the end), loaded two tiles ahead, ...
    const int key0 = u.key_begin + ww * 32 + lane, key_end = u.key_end;
    const int32_t* const table = u.table;
    auto key_block = [&](int j) -> int32_t {
      const int p = key0 + j * kN;
      return load_or(table + (p >> c.shift), p < key_end, -1);
    };
    // ... and its row of the pool; -1: zeros
    auto key_row = [&](int j, int32_t b) -> int32_t {
      const int p = key0 + j * kN;
      if (b >= 0 && b < c.num_blocks) return (b * c.kv_heads + kvh) * c.block + (p & (c.block - 1));
      if (kvh == 0 && p < key_end) raise_error(a.err, QQ_DEV_ERR_BOUNDS);
      return -1;
    };
    uint2 wk[16], wv[16];
    auto load = [&](int32_t rows) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int32_t r = __shfl_sync(0xffffffffu, rows, 2 * i + hr);
        const int64_t at = (int64_t)r * kTcDim + ch * 8;
        wk[i] = load8_or_zero(c.k + at, r >= 0);
        wv[i] = load8_or_zero(c.v + at, r >= 0);
      }
    };
    // 8 codes are one 16-byte piece in fp16, swizzled by the row; steps i and i + 4 share a swizzle
    uint32_t at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      at[k] = base + (ch >> 3) * kHalf + (ww * 32 + hr) * 128 + (((ch & 7) ^ (2 * k + hr)) << 4);
    uint32_t nan;  // fp16 pair, NaN once a code of V was
    auto store = [&](uint32_t off, const uint2 (&w)[16], auto look) {
      nan = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        uint4 h;
        widen4(w[i].x, h.x, h.y);
        widen4(w[i].y, h.z, h.w);
        if (look.value) nan_of(nan, h);
        st_shared16(at[i & 3] + off + i * 256, h);
      }
    };
    // A weight of zero does not hide a NaN of V from the rows that may not see
    // its key.  So a key with one gets zeros for V and NaN for K: the rows that
    // see it become NaN, the scores of the others are masked.
    auto hide_nan = [&](uint32_t off) {
      if (!__any_sync(0xffffffffu, (nan & 0x7FFFu) > 0x7C00u || (nan & 0x7FFF0000u) > 0x7C000000u)) return;
      auto nan4 = [](uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; };  // codes 0x7F and 0xFF
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t m = __ballot_sync(0xffffffffu, (nan4(wv[i].x) | nan4(wv[i].y)) != 0);
        if (m >> (lane & 16) & 0xFFFFu) {
          st_shared16(at[i & 3] + off + i * 256, make_uint4(0, 0, 0, 0));
          wk[i] = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
        }
      }
    };
    int32_t ahead = key_block(1);
    load(key_row(0, key_block(0)));
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int st = j % kStages;
      const uint32_t turn = ((j / kStages) - 1) & 1;
      const int32_t next = key_row(j + 1, ahead);
      ahead = key_block(j + 2);
      if (j >= kStages && !__all_sync(0xffffffffu, wait(kBarVFree + st, turn))) break;
      store(kOffV + st * kTileBytes, wv, std::true_type{});
      hide_nan(kOffV + st * kTileBytes);
      mbar_arrive_warp(bar(kBarV + st));
      if (j >= kStages && !__all_sync(0xffffffffu, wait(kBarKFree + st, turn))) break;
      store(kOffK + st * kTileBytes, wk, std::false_type{});
      mbar_arrive_warp(bar(kBarK + st));
      load(next);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
    if (warp == kScaleWarp) {
    // ================================================================ scales
    for (int j = 0; j < tiles; ++j) {
      const int m = j % kMeta;
      float4 f = make_float4(0.f, -INFINITY, 0.f, 0.f);
      const int p = u.key_begin + j * kN + lane * kGroup;
      if (lane < kN / kGroup && p < u.key_end) {
        const int32_t b = u.table[p >> c.shift];
        if (b >= 0 && b < c.num_blocks) {
          const int bh = b * c.kv_heads + kvh;
          f.x = c.k_scale[bh];
          // 2^-lg stays a normal number; times 2^-kTop, or l of 2^20 keys of blocks of zeros would not be finite
          f.y = fminf(fmaxf(log2f(c.v_scale[bh]), -100.f), 126.f);
          if (isnan(c.v_scale[bh])) f.y = c.v_scale[bh];
          f.z = exp2f(-f.y - kTop);
        }
      }
      if (j >= kMeta && !__all_sync(0xffffffffu, wait(kBarMetaFree + m, ((j / kMeta) - 1) & 1))) break;
      if (lane < kN / kGroup) s_scale[m][lane] = f;
      mbar_arrive_warp(bar(kBarMeta + m));
    }
    } else if (warp < kScaleWarp) {
    // ================================================================ MMA issue, one warp per M tile
    if (tiles > 0) {
      const int h = warp - kMmaWarp;
      const uint32_t tS = tmem + h * 256, tO = tS + 128;
      const uint64_t dq = desc_k(base + kOffQ + h * kTileBytes);
      auto all = [&](int i, uint32_t parity) { return __all_sync(0xffffffffu, wait(i, parity)); };
      bool ok = all(kBarQ + h, 0);
      auto scores = [&](int j) {
        const int st = j % kStages;
        // The second tile's scores wait for the first one's softmax, so that one's
        // exponentials meet the other's products (in step, both wait for the
        // tensor cores, then both for the exponentials: 627 us where this takes 571).
        ok = ok && (h == 0 || all(kBarLag + (j & 1), (j >> 1) & 1)) && all(kBarK + st, (j / kStages) & 1);
        if (!ok) return;
        // the widened tiles reach the tensor cores through this thread's fence
        fence_async_shared();
        tc_fence_after();
        const uint64_t dk = desc_k(base + kOffK + st * kTileBytes);
        umma_f16_x4_warp(tS, dq, dk, 2, 2, kIdS, 0u);
        umma_f16_x4_warp(tS, dq + (kHalf >> 4), dk + (kHalf >> 4), 2, 2, kIdS, 1u);
        umma_commit_warp(bar(kBarS + h));
        umma_commit_warp(bar(kBarKFree + st));
      };
      scores(0);
#pragma unroll 1
      for (int j = 0; j < tiles && ok; ++j) {
        const int st = j % kStages;
        ok = all(kBarV + st, (j / kStages) & 1) && all(kBarP + 2 * h, j & 1);
        if (!ok) break;
        fence_async_shared();
        tc_fence_after();
        const uint64_t dv = desc_mn(base + kOffV + st * kTileBytes, kHalf);
        umma_f16_ts_x4_warp(tO, tS, dv, 8, (16 * 128) >> 4, kIdO, j > 0 ? 1u : 0u);
        umma_commit_warp(bar(kBarO + h));
        ok = all(kBarP + 2 * h + 1, j & 1);
        if (!ok) break;
        tc_fence_after();
        umma_f16_ts_x4_warp(tO, tS + 32, dv + ((64 * 128) >> 4), 8, (16 * 128) >> 4, kIdO, 1u);
        umma_commit_warp(bar(kBarVFree + st));
        if (j + 1 < tiles) scores(j + 1);
      }
      umma_commit_warp(bar(kBarDone + h));
      mbar_wait(bar(kBarDone + h), 0, abort_flag, a.err, true);
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Merges the records of the units that were cut: a warp per query row, four
// channels per lane.  Launched always (how many units there are is known on the
// device alone), and done at once where none was cut.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) kv8_extend_join_kernel(ExtendArgs g) {
  __shared__ Unit s_unit;
  __shared__ int s_record;
  const AttnArgs& a = g.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    int record = 0;
    const Unit u = find_unit(g, nullptr, [&](const Units& units, int& index, int&) {
      record = blockIdx.x * units.splits;
      index = units.whole + blockIdx.x;  // past the last one where none was cut
    });
    if (lane == 0) s_unit = u, s_record = record;
  }
  __syncthreads();
  wait_prior_grid();
  allow_next_grid();
  const Unit& u = s_unit;
  if (u.entry < 0 || u.splits == 1) return;
  const int splits = u.splits;
  for (int r = blockIdx.y * kJoinWarps + warp; r < u.rows; r += gridDim.y * kJoinWarps) {
    const float* rec = a.part + (int64_t)s_record * kRecord;
    float M = -INFINITY;
    for (int s = lane; s < splits; s += 32) M = fmaxf(M, rec[s * kRecord + 2 * r]);
    M = warp_max(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float* p = rec + s * kRecord;
      const float f = ex2(p[2 * r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(p + 2 * kUnitRows + (int64_t)r * kTcDim + lane * 4);
      l = fmaf(f, p[2 * r + 1], l);
      o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int token = (u.row0 + r) / a.group, head = u.kvh * a.group + u.row0 + r - token * a.group;
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (int64_t)(u.q_row + token) * a.out_stride +
                              (int64_t)head * kTcDim + lane * 4) =
        make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  }
}

// Tiles of a KV head at most: a ragged end per entry.
int64_t unit_tiles(int bs, int group, int64_t tokens) { return (tokens * group + kUnitRows - 1) / kUnitRows + bs; }

// Stretches of a unit at most: none below four key tiles.
int64_t most_splits(int64_t max_keys) {
  return std::min<int64_t>(device_sm_count(), std::max<int64_t>(1, (max_keys + 4 * kN - 1) / (4 * kN)));
}

}  // namespace

bool extend_tc_fits(const AttnArgs& a, int dtype) {
  const int64_t tiles = unit_tiles(a.bs, a.group, a.tokens);
  return dtype == QQ_BF16 && a.c.dim == kTcDim && (a.q_stride * 2) % 16 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0 &&
         (a.out_stride * 2) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && tiles <= 65535 &&
         tiles * a.c.kv_heads <= INT_MAX / 2;
}

// The stretches' records: at most one per SM.
size_t extend_tc_workspace(int bs, int kv_heads, int group, int64_t tokens, int64_t max_keys) {
  const int64_t most = most_splits(max_keys), units = unit_tiles(bs, group, tokens) * kv_heads;
  return most == 1 ? 0 : sizeof(float) * (size_t)(std::min<int64_t>(device_sm_count(), units * most) * kRecord);
}

int run_extend_tc(const AttnArgs& a, int64_t max_keys, size_t ws_bytes, cudaStream_t s) {
  ExtendArgs g{};
  g.a = a;
  g.tiles = (int)unit_tiles(a.bs, a.group, a.tokens);
  g.sms = device_sm_count();
  g.most = (int)most_splits(max_keys);
  if (g.most > 1 && (a.part == nullptr || ws_bytes < extend_tc_workspace(a.bs, a.c.kv_heads, a.group, a.tokens, max_keys)))
    return QQ_ERR_WORKSPACE;
  static SmemLimit limit16, limit64;
  int rc = limit16.ensure((const void*)kv8_extend_kernel<16>, kDynSmem);
  if (rc == QQ_OK) rc = limit64.ensure((const void*)kv8_extend_kernel<64>, kDynSmem);
  if (rc != QQ_OK) return rc;
  const int units = g.tiles * a.c.kv_heads;
  const unsigned grid = (unsigned)(units + (g.most > 1 ? g.sms : 0));
  rc = a.c.block >= 64 ? launch_pdl(kv8_extend_kernel<64>, dim3(grid), dim3(kThreads), kDynSmem, s, g)
                       : launch_pdl(kv8_extend_kernel<16>, dim3(grid), dim3(kThreads), kDynSmem, s, g);
  if (rc != QQ_OK || g.most == 1) return rc;
  // as many CTAs to a unit as there may be room for
  const int cut = std::min(units, g.sms - 1), y = std::max(4, std::min(kUnitRows / kJoinWarps, 8 * g.sms / std::max(1, cut)));
  return launch_pdl(kv8_extend_join_kernel, dim3(std::max(1, cut), y), dim3(kJoinWarps * 32), 0, s, g);
}

}  // namespace kv8
}  // namespace qq

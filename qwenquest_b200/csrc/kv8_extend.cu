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
// serves 256 rows.  With few CTAs the keys are cut into `splits` stretches
// whose (M, l, O) records kv8_extend_join_kernel merges.
// Scales: as in the one-token kernel a score is S ks / up, the weight into
// the V product 2^(s + lg - M) with lg = log2(vs), and the sum takes that
// times 2^-lg: constants of a group of 16 keys (no block is shorter).
// Warps: 0-7 softmax (thread = row = TMEM lane; 0-3 tile 0, 4-7 tile 1),
// 8-11 widen K and V, 12-13 MMA issue (one per M tile), 14 scales.
// Tensor memory: per M tile S (128 fp32 columns, overlaid by P in fp16 once
// read) and O (128).  The order per tile is S(j) P(j) O(j) S(j + 1): while
// one tile's softmax runs the tensor cores work for the other.
// The running maximum is raised only past a factor of 2^8; O is rescaled then.
// Every wait is bounded; see the one-token kernel.

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
constexpr int kGroups = kN / 16;
constexpr int kWidenWarp = 8, kMmaWarp = 12, kScaleWarp = 14;
constexpr int kThreads = 15 * 32;
constexpr int kOffQ = 0, kOffK = 2 * kTileBytes, kOffV = kOffK + kStages * kTileBytes;
constexpr int kDynSmem = kOffV + kStages * kTileBytes + 1024;
constexpr uint32_t kTmemCols = 512;
constexpr float kRaise = 8.f;

enum : int {
  kBarQ = 0,                          // [2] queries of a tile written
  kBarK = kBarQ + 2,                  // [stages] keys written
  kBarKFree = kBarK + kStages,        // [stages] read by both tiles' MMAs
  kBarV = kBarKFree + kStages,
  kBarVFree = kBarV + kStages,
  kBarMeta = kBarVFree + kStages,     // [kMeta] scales written
  kBarMetaFree = kBarMeta + kMeta,
  kBarS = kBarMetaFree + kMeta,       // [2] scores made
  kBarP = kBarS + 2,                  // [2] weights written
  kBarO = kBarP + 2,                  // [2] a product made
  kBarDone = kBarO + 2,               // [2] the tile's last MMA has finished
  kNumBars = kBarDone + 2
};

struct ExtendArgs {
  AttnArgs a;
  int splits;
};

// A split's record of a unit: (M, l) of 256 rows, then O [256][128].
constexpr int64_t kRecord = kUnitRows * (2 + (int64_t)kTcDim);

// fp16 operands, fp32 accumulator.
constexpr uint32_t kIdS = (1u << 4) | ((kN >> 3) << 17) | ((kM >> 4) << 24);
constexpr uint32_t kIdO = (1u << 4) | (1u << 16) | ((kTcDim >> 3) << 17) | ((kM >> 4) << 24);

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t widen2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// The CTA's rows and keys.
struct Unit {
  ExtendEntry x;
  int64_t row0, rows;      // rows [row0, row0 + rows) of the entry's n * group
  int64_t req;
  int64_t key_begin, key_end;
  int tiles;
};
__device__ __forceinline__ Unit unit_of(const ExtendArgs& g, int64_t tile, int split, uint32_t* err) {
  const AttnArgs& a = g.a;
  Unit u{};
  u.x = extend_tile(a, tile, kUnitRows, a.group, err);
  if (u.x.entry < 0) return u;
  u.row0 = u.x.tile * kUnitRows;
  u.rows = min((int64_t)kUnitRows, u.x.n * a.group - u.row0);
  u.req = a.reqs[u.x.entry];
  const int64_t keys = u.x.prefix + (u.row0 + u.rows - 1) / a.group + 1;  // what its last row sees
  const int64_t all = (keys + kN - 1) / kN, each = (all + g.splits - 1) / g.splits;
  u.key_begin = min(all, split * each) * kN;
  u.key_end = min(keys, u.key_begin + each * kN);
  u.tiles = u.key_end > u.key_begin ? (int)((u.key_end - u.key_begin + kN - 1) / kN) : 0;
  return u;
}

__global__ void __launch_bounds__(kThreads, 1) kv8_extend_kernel(ExtendArgs g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kNumBars];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Unit s_unit;
  __shared__ float s_up[kUnitRows];                                   // scale_log2 / up of each row
  __shared__ __align__(16) float4 s_scale[kMeta][kGroups];        // ks, lg, 2^-lg of 16 keys
  const AttnArgs& a = g.a;
  const Cache& c = a.c;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  volatile int* abort_flag = &s_abort;
  auto wait = [&](int i, uint32_t parity) { return mbar_wait(bar(i), parity, abort_flag, a.err); };
  const int kvh = blockIdx.x;
  // the last tiles of an entry see the most keys: they start first
  const int64_t tile = gridDim.y - 1 - blockIdx.y;

  if (warp == 0) {
    const Unit u = unit_of(g, tile, blockIdx.z, blockIdx.x == 0 && tile == 0 && blockIdx.z == 0 ? a.err : nullptr);
    if (lane == 0) s_unit = u;
  }
  if (threadIdx.x == 32) {
    s_abort = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kBarQ + i), kM);
      mbar_init(bar(kBarS + i), 1);
      mbar_init(bar(kBarP + i), kM);
      mbar_init(bar(kBarO + i), 1);
      mbar_init(bar(kBarDone + i), 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(bar(kBarK + i), 128);
      mbar_init(bar(kBarV + i), 128);
      mbar_init(bar(kBarKFree + i), 2);
      mbar_init(bar(kBarVFree + i), 2);
    }
    for (int i = 0; i < kMeta; ++i) {
      mbar_init(bar(kBarMeta + i), 32);
      mbar_init(bar(kBarMetaFree + i), kUnitRows);
    }
    mbar_init_fence();
  }
  __syncthreads();
  const Unit& u = s_unit;
  if (u.x.entry < 0) return;  // past the last tile, uniform
  if (warp == kMmaWarp) tmem_alloc(smem_u32(&s_tmem), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int tiles = u.tiles;

  if (warp >= kWidenWarp && warp < kMmaWarp) {
    // ================================================================ K and V to fp16
    // Eight lanes per key row, 16 codes each; a warp's 32 rows in eight steps.
    // The codes of the next tile are on their way while one is widened.
    const int ww = warp - kWidenWarp, ch = lane & 7;
    // lane L holds the pool row of key ww * 32 + L of a tile; -1: zeros
    auto key_row = [&](int j) -> int32_t {
      const int64_t p = u.key_begin + (int64_t)j * kN + ww * 32 + lane;
      if (p >= u.key_end) return -1;
      const int64_t s = key_slot<kTable>(a, u.x.entry, u.req, p, kvh == 0 ? a.err : nullptr);
      return s < 0 ? -1 : (int32_t)(((s >> c.shift) * c.kv_heads + kvh) * c.block + (s & (c.block - 1)));
    };
    auto load = [&](const uint8_t* pool, int32_t rows, uint4 (&w)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int32_t r = __shfl_sync(0xffffffffu, rows, i * 4 + (lane >> 3));
        w[i] = r < 0 ? make_uint4(0, 0, 0, 0)
                     : __ldg(reinterpret_cast<const uint4*>(pool + (int64_t)r * kTcDim + ch * 16));
      }
    };
    auto store = [&](uint32_t off, const uint4 (&w)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = ww * 32 + i * 4 + (lane >> 3);
        const uint4 lo = make_uint4(widen2(w[i].x), widen2(w[i].x >> 16), widen2(w[i].y), widen2(w[i].y >> 16));
        const uint4 hi = make_uint4(widen2(w[i].z), widen2(w[i].z >> 16), widen2(w[i].w), widen2(w[i].w >> 16));
        // 16-byte pieces 2 ch and 2 ch + 1 of the row's 16; the two blocks of a
        // row share their banks, so the lanes of the second one start with the odd piece
        uint8_t* row = smem + off + (ch >> 2) * kHalf + r * 128;
        const int p0 = (((2 * ch) & 7) ^ (r & 7)) << 4, p1 = (((2 * ch + 1) & 7) ^ (r & 7)) << 4;
        const bool odd = ch >= 4;
        *reinterpret_cast<uint4*>(row + (odd ? p1 : p0)) = odd ? hi : lo;
        *reinterpret_cast<uint4*>(row + (odd ? p0 : p1)) = odd ? lo : hi;
      }
      fence_async_shared();
    };
    // A weight of zero does not hide a NaN of V from the rows that may not see
    // its key.  So a key with one gets zeros for V and NaN for K: the rows that
    // see it become NaN, the scores of the others are masked.
    auto hide_nan = [&](uint4 (&k)[8], uint4 (&v)[8]) {
      auto nan4 = [](uint32_t w) { return (w & 0x7F7F7F7Fu) + 0x01010101u; };  // top bits: codes 0x7F and 0xFF
      auto nan16 = [&](const uint4& w) { return (nan4(w.x) | nan4(w.y) | nan4(w.z) | nan4(w.w)) & 0x80808080u; };
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) any |= nan16(v[i]);
      if (!__any_sync(0xffffffffu, any != 0)) return;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t m = __ballot_sync(0xffffffffu, nan16(v[i]) != 0);
        if (m >> (lane & 24) & 255u) {
          v[i] = make_uint4(0, 0, 0, 0);
          k[i] = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
        }
      }
    };
    uint4 wk[8], wv[8];
    int32_t next = tiles > 0 ? key_row(0) : -1;
    if (tiles > 0) {
      load(c.k, next, wk);
      load(c.v, next, wv);
    }
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int st = j % kStages;
      const uint32_t turn = ((j / kStages) - 1) & 1;
      if (j + 1 < tiles) next = key_row(j + 1);
      hide_nan(wk, wv);
      if (j >= kStages && !__all_sync(0xffffffffu, wait(kBarKFree + st, turn))) break;
      store(kOffK + st * kTileBytes, wk);
      mbar_arrive(bar(kBarK + st));
      if (j + 1 < tiles) load(c.k, next, wk);
      if (j >= kStages && !__all_sync(0xffffffffu, wait(kBarVFree + st, turn))) break;
      store(kOffV + st * kTileBytes, wv);
      mbar_arrive(bar(kBarV + st));
      if (j + 1 < tiles) load(c.v, next, wv);
    }
  } else if (warp == kScaleWarp) {
    // ================================================================ scales
    for (int j = 0; j < tiles; ++j) {
      const int m = j % kMeta;
      float4 f = make_float4(0.f, -INFINITY, 0.f, 0.f);
      const int64_t p = u.key_begin + (int64_t)j * kN + lane * 16;
      if (lane < kGroups && p < u.key_end) {
        const int64_t s = key_slot<kTable>(a, u.x.entry, u.req, p, nullptr);
        if (s >= 0) {
          const int64_t bh = (s >> c.shift) * c.kv_heads + kvh;
          f.x = c.k_scale[bh];
          // 2^-lg stays a normal number
          f.y = fminf(fmaxf(log2f(c.v_scale[bh]), -100.f), 126.f);
          if (isnan(c.v_scale[bh])) f.y = c.v_scale[bh];
          f.z = exp2f(-f.y);
        }
      }
      if (j >= kMeta && !__all_sync(0xffffffffu, wait(kBarMetaFree + m, ((j / kMeta) - 1) & 1))) break;
      if (lane < kGroups) s_scale[m][lane] = f;
      mbar_arrive(bar(kBarMeta + m));
    }
  } else if (warp >= kMmaWarp) {
    // ================================================================ MMA issue, one warp per M tile
    if (lane == 0 && tiles > 0) {
      const int h = warp - kMmaWarp;
      const uint32_t tS = tmem + h * 256, tO = tS + 128;
      const uint64_t dq = desc_k(base + kOffQ + h * kTileBytes);
      bool ok = wait(kBarQ + h, 0);
      auto scores = [&](int j) {
        const int st = j % kStages;
        ok = ok && wait(kBarK + st, (j / kStages) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint64_t dk = desc_k(base + kOffK + st * kTileBytes);
        umma_bf16_x4(tS, dq, dk, 2, 2, kIdS, 0u);
        umma_bf16_x4(tS, dq + (kHalf >> 4), dk + (kHalf >> 4), 2, 2, kIdS, 1u);
        umma_commit(bar(kBarS + h));
        umma_commit(bar(kBarKFree + st));
      };
      scores(0);
#pragma unroll 1
      for (int j = 0; j < tiles && ok; ++j) {
        const int st = j % kStages;
        ok = wait(kBarV + st, (j / kStages) & 1) && wait(kBarP + h, j & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dv = desc_mn(base + kOffV + st * kTileBytes, kHalf);
        umma_bf16_ts_x4(tO, tS, dv, 8, (16 * 128) >> 4, kIdO, j > 0 ? 1u : 0u);
        umma_bf16_ts_x4(tO, tS + 32, dv + ((64 * 128) >> 4), 8, (16 * 128) >> 4, kIdO, 1u);
        umma_commit(bar(kBarO + h));
        umma_commit(bar(kBarVFree + st));
        if (j + 1 < tiles) scores(j + 1);
      }
      umma_commit(bar(kBarDone + h));
      mbar_wait(bar(kBarDone + h), 0, abort_flag, a.err, true);
    }
    __syncwarp();
  } else {
    // ================================================================ softmax (warps 0-7)
    const int h = warp >> 2, r = threadIdx.x;      // row of the CTA's 256
    const int64_t row = u.row0 + r;
    const int64_t token = row / a.group;
    const int head = kvh * a.group + (int)(row - token * a.group);
    // ---- this warp's 32 query rows to fp16: four lanes per row, 32 channels each
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 8) {
      const int rr = warp * 32 + r0 + (lane >> 2), col = (lane & 3) * 32;
      float x[32] = {};
      if (rr < u.rows) {
        const int64_t t = (u.row0 + rr) / a.group;
        const int hd = kvh * a.group + (int)(u.row0 + rr - t * a.group);
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) +
                                                        (u.x.row0 + t) * a.q_stride + (int64_t)hd * kTcDim + col);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 w = q[k];
          const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int b = 0; b < 4; ++b)
            x[8 * k + 2 * b] = __uint_as_float(v[b] << 16), x[8 * k + 2 * b + 1] = __uint_as_float(v[b] & 0xFFFF0000u);
        }
      }
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const bool finite = fabsf(x[k]) <= 3.402823466e38f;
        if (finite) most = fmaxf(most, fabsf(x[k]));
        else x[k] = __uint_as_float(0x7FFFFFFFu);  // an infinite query has no scores either
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int k2 = max(-120, fit_exponent(most) - 1);  // at most 224
      const float up = a.scale_log2 < 0.f ? -exp2_int(k2) : exp2_int(k2);
      uint8_t* dst = smem + kOffQ + h * kTileBytes + (lane & 2) / 2 * kHalf + (rr & 127) * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int piece = (lane & 1) * 4 + k;
        const float* y = x + 8 * k;
        *reinterpret_cast<uint4*>(dst + ((piece ^ (rr & 7)) << 4)) =
            make_uint4(pack_f16(y[0] * up, y[1] * up), pack_f16(y[2] * up, y[3] * up),
                       pack_f16(y[4] * up, y[5] * up), pack_f16(y[6] * up, y[7] * up));
      }
      if ((lane & 3) == 0) s_up[rr] = fabsf(a.scale_log2) * exp2_int(-k2);
    }
    fence_async_shared();
    mbar_arrive(bar(kBarQ + h));
    __syncwarp();
    const float inv_up = s_up[r];

    const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + h * 256, tO = tS + 128;
    const int64_t qpos = u.x.prefix + token;
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int m = j % kMeta;
      ok = __all_sync(0xffffffffu, wait(kBarMeta + m, (j / kMeta) & 1) && wait(kBarS + h, j & 1));
      if (!ok) break;
      tc_fence_after();
      // columns c <= lim are seen by this row
      const int64_t lim64 = qpos - u.key_begin - (int64_t)j * kN;
      const int lim = lim64 > kN - 1 ? kN - 1 : (lim64 < -1 ? -1 : (int)lim64);
      const bool full = __all_sync(0xffffffffu, lim == kN - 1);
      float v[64];
      auto half = [&](int hf) {
        tmem_ld32(tS + hf * 64, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld32(tS + hf * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tmem_ld_wait();
        if (!full) {
#pragma unroll
          for (int e = 0; e < 64; ++e) v[e] = hf * 64 + e <= lim ? v[e] : -INFINITY;
        }
      };
      float mb = -INFINITY;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        half(hf);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 f = s_scale[m][hf * 4 + q];
          const float* w = v + q * 16;
          float x = max3(max3(w[0], w[1], w[2]), w[3], w[4]), y = max3(max3(w[5], w[6], w[7]), w[8], w[9]);
          x = max3(x, w[10], w[11]), y = max3(y, w[12], w[13]);
          x = max3(x, w[14], w[15]);
          x = fmaxf(x, y);
          // a masked group (-inf) stays -inf also where its scale is 0
          mb = fmaxf(mb, x == -INFINITY ? x : fmaf(x, inv_up * f.x, f.y));
        }
      }
      const bool raise = mb > m_used + kRaise;
      float alpha = 1.f;
      if (raise) {
        alpha = ex2(m_used - mb);
        m_used = mb;
        l *= alpha;
      }
      if (j > 0 && __any_sync(0xffffffffu, raise)) {
        ok = __all_sync(0xffffffffu, wait(kBarO + h, (j - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        uint32_t o[32];
#pragma unroll 1
        for (int k = 0; k < kTcDim / 32; ++k) {
          tmem_ld32(tO + k * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(tO + k * 32, o);
        }
        tmem_st_wait();
      }
      // the second half is still in registers; P of the first half goes over columns the first half has left
      const float ref = m_used == -INFINITY ? 0.f : m_used;
      uint32_t pk[32];
      auto weights = [&](int hf, auto is_full) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 f = s_scale[m][hf * 4 + q];
          const float mul = inv_up * f.x, add = f.y - ref;
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float p0 = ex2(fmaf(v[q * 16 + e], mul, add)), p1 = ex2(fmaf(v[q * 16 + e + 1], mul, add));
            if (!is_full.value) {
              p0 = hf * 64 + q * 16 + e <= lim ? p0 : 0.f;
              p1 = hf * 64 + q * 16 + e + 1 <= lim ? p1 : 0.f;
            }
            s0 += p0;
            s1 += p1;
            pk[(q * 16 + e) / 2] = pack_f16(p0, p1);
          }
          l = fmaf(s0 + s1, f.z, l);
        }
      };
      uint32_t pk1[32];
      auto both = [&](auto is_full) {
        weights(1, is_full);
#pragma unroll
        for (int e = 0; e < 32; ++e) pk1[e] = pk[e];
        half(0);
        weights(0, is_full);
      };
      if (full) both(std::true_type{});
      else both(std::false_type{});
      tmem_st32(tS, pk);
      tmem_st32(tS + 32, pk1);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar(kBarP + h));
      mbar_arrive(bar(kBarMetaFree + m));
    }
    // ---- O / l, or this stretch's record
    ok = __all_sync(0xffffffffu, ok && (tiles == 0 || wait(kBarDone + h, 0)));
    tc_fence_after();
    const bool valid = ok && r < u.rows;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float* rec = a.part + (((int64_t)tile * c.kv_heads + kvh) * g.splits + blockIdx.z) * kRecord;
    if (g.splits > 1 && valid) rec[2 * r] = m_used, rec[2 * r + 1] = l;
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (u.x.row0 + token) * a.out_stride + (int64_t)head * kTcDim;
#pragma unroll 1
    for (int k = 0; k < kTcDim / 32; ++k) {
      uint32_t o[32] = {};
      if (tiles > 0 && ok) {
        tmem_ld32(tO + k * 32, o);
        tmem_ld_wait();
      }
      if (!valid) continue;
      if (g.splits > 1) {
        float4* w = reinterpret_cast<float4*>(rec + 2 * kUnitRows + (int64_t)r * kTcDim + k * 32);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                             __uint_as_float(o[4 * e + 3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint4 w;
          w.x = pack_bf16(__uint_as_float(o[8 * e + 0]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
          w.y = pack_bf16(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
          w.z = pack_bf16(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
          w.w = pack_bf16(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
          *reinterpret_cast<uint4*>(dst + k * 32 + e * 8) = w;
        }
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

// Merges the records of a unit's stretches: a warp per query row, four channels per lane.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) kv8_extend_join_kernel(ExtendArgs g) {
  __shared__ Unit s_unit;
  const AttnArgs& a = g.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y;
  if (warp == 0) {
    const Unit u = unit_of(g, blockIdx.x, 0, nullptr);
    if (lane == 0) s_unit = u;
  }
  __syncthreads();
  wait_prior_grid();
  const Unit& u = s_unit;
  const int r = blockIdx.z * kJoinWarps + warp;
  if (u.x.entry < 0 || r >= u.rows) return;
  const float* rec = a.part + ((int64_t)blockIdx.x * a.c.kv_heads + kvh) * g.splits * kRecord;
  float M = -INFINITY;
  for (int s = lane; s < g.splits; s += 32) M = fmaxf(M, rec[s * kRecord + 2 * r]);
  M = warp_max(M);
  const float ref = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < g.splits; ++s) {
    const float* p = rec + s * kRecord;
    const float f = ex2(p[2 * r] - ref);
    const float4 v = *reinterpret_cast<const float4*>(p + 2 * kUnitRows + (int64_t)r * kTcDim + lane * 4);
    l = fmaf(f, p[2 * r + 1], l);
    o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t row = u.row0 + r, token = row / a.group;
  const int head = kvh * a.group + (int)(row - token * a.group);
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (u.x.row0 + token) * a.out_stride +
                            (int64_t)head * kTcDim + lane * 4) =
      make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

int64_t unit_tiles(int bs, int group, int64_t tokens) { return (tokens * group + kUnitRows - 1) / kUnitRows + bs; }

// Stretches of the keys: one CTA per SM at a time, no stretch below four key tiles.
int extend_splits(int bs, int kv_heads, int group, int64_t tokens, int64_t max_keys) {
  // about as many units as there are full tiles (the bound counts a ragged end per entry)
  const int64_t units = unit_tiles(bs, group, tokens) * kv_heads;
  int64_t s = device_sm_count() / units;
  const int64_t most = (max_keys + 4 * kN - 1) / (4 * kN);
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s);
}

}  // namespace

bool extend_tc_fits(const AttnArgs& a, int dtype) {
  return dtype == QQ_BF16 && a.c.dim == kTcDim && a.c.kv_heads <= 65535 && (a.q_stride * 2) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && (a.out_stride * 2) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && unit_tiles(a.bs, a.group, a.tokens) <= 65535;
}

size_t extend_tc_workspace(int bs, int kv_heads, int group, int64_t tokens, int64_t max_keys) {
  const int s = extend_splits(bs, kv_heads, group, tokens, max_keys);
  return s <= 1 ? 0 : sizeof(float) * (size_t)(unit_tiles(bs, group, tokens) * kv_heads * s * kRecord);
}

int run_extend_tc(const AttnArgs& a, int64_t max_keys, size_t ws_bytes, cudaStream_t s) {
  ExtendArgs g{};
  g.a = a;
  g.splits = extend_splits(a.bs, a.c.kv_heads, a.group, a.tokens, max_keys);
  if (g.splits > 1 &&
      (a.part == nullptr || ws_bytes < extend_tc_workspace(a.bs, a.c.kv_heads, a.group, a.tokens, max_keys)))
    return QQ_ERR_WORKSPACE;
  static SmemLimit limit;
  int rc = limit.ensure((const void*)kv8_extend_kernel, kDynSmem);
  if (rc != QQ_OK) return rc;
  const unsigned tiles = (unsigned)unit_tiles(a.bs, a.group, a.tokens);
  kv8_extend_kernel<<<dim3(a.c.kv_heads, tiles, g.splits), kThreads, kDynSmem, s>>>(g);
  if ((rc = launch_status()) != QQ_OK || g.splits == 1) return rc;
  return launch_pdl(kv8_extend_join_kernel, dim3(tiles, a.c.kv_heads, kUnitRows / kJoinWarps), dim3(kJoinWarps * 32), 0, s, g);
}

}  // namespace kv8
}  // namespace qq

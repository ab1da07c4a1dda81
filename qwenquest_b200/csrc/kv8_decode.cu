// One query token per request over the 8-bit block cache on the
// fifth-generation tensor cores (bf16 queries, head_dim 128, up to 16 query
// heads per KV head): the whole sequence through the block table, or listed rows.
//
// Bound by the bytes of the codes (2 x 128 per token and KV head), so the
// codes go from HBM to shared memory (TMA) to the tensor cores without a
// conversion: both products have an operand of the other side in e4m3, held
// to bf16's precision by a pair hi + lo / 16 in two columns of one MMA.
//   S^T [128 tokens x NC] = K [128 x 128] . Q^T      NC = 2 x 8 (or 2 x 16)
//   O^T [128 dims x NC]   = V^T [128 x 128] . P      columns: heads hi, heads lo
// A tile of 128 tokens is a row per thread in both, so each thread has one
// token's scores of all heads, and later one channel of all heads.
//
// Scales: a token's score is S ks q^-1 log2(e) scaling; its weight into the V
// product is 2^(s - M) vs.  With vs = vm 2^ev the running maximum M is that of
// s + ev, so what enters the product, vm 2^(s + ev - M), is at most 2 whatever
// the blocks' scales are, and the sum l takes 2^(s + ev - M) 2^-ev.
//
// Work: the tiles of all (request, KV head) pairs in a row, cut into equal
// shares, one per CTA (two CTAs per SM); a pair cut by a share's edge leaves
// (M, l, O) records that kv8_decode_join_kernel merges.
// Warps: 0-3 softmax, 4 TMA, 5 MMA issue, 6 queries, 7 scales.  The MMAs go
// S(0) S(1) O(0) S(2) O(1) ...: the softmax of a tile runs while the next
// tile's scores are made, and a tile's O is added in registers one tile later.
// Every wait is bounded (kWaitLimitNs); on expiry the CTA reports
// QQ_DEV_ERR_TIMEOUT, waits for its own copies and MMAs and returns.

#include <climits>
#include <cmath>

#include <cuda_fp16.h>

#include "kv8_tma.cuh"

namespace qq {
namespace kv8 {
namespace {

using namespace tc;

constexpr int kTile = 128;                     // tokens
constexpr int kSlotBytes = kTile * kTcDim;     // 16 KiB: K or V codes of a tile
constexpr int kSoft = 128;                     // softmax threads
constexpr int kThreads = 256;
constexpr int kMeta = 4;                       // tiles of scales in flight
constexpr int kMaxSlots = 12;
constexpr uint32_t kMasked = 0xFFFFFFFFu;      // a V scale's bits where the token takes no part
constexpr float kLo = 16.f;
constexpr float kPScale = 128.f;               // weights (at most 2) times this are e4m3's upper binades

// mbarriers
enum : int {
  kBarFull = 0,                      // [slots] codes have landed
  kBarEmpty = kBarFull + kMaxSlots,  // [slots] codes have been read
  kBarQ = kBarEmpty + kMaxSlots,     // [2] queries written
  kBarQFree = kBarQ + 2,             // [2] queries read
  kBarMeta = kBarQFree + 2,          // [kMeta] scales written
  kBarMetaFree = kBarMeta + kMeta,   // [kMeta] scales read
  kBarS = kBarMetaFree + kMeta,      // [2] scores made
  kBarP = kBarS + 2,                 // [2] weights written
  kBarO = kBarP + 2,                 // [2] product made
  kBarDone = kBarO + 2,              // the last MMA has finished
  kNumBars = kBarDone + 1
};

// Tile lo of share c of `ctas`.
__host__ __device__ __forceinline__ int64_t share_lo(int64_t total, int64_t c, int64_t ctas) { return total * c / ctas; }

// Steps through a share's tiles: entry e, head h, tile t of the entry's T.  The next entry's length is loaded one
// entry ahead.
template <int KEYS>
struct Walk {
  const AttnArgs& a;
  int e, h, t, T;
  int64_t n, n1;
  __device__ Walk(const AttnArgs& args, int entry, int head, int tile) : a(args), e(entry), h(head), t(tile) {
    n = entry_keys<KEYS>(a, e, nullptr);
    T = (int)((n + kTile - 1) / kTile);
    n1 = e + 1 < a.bs ? entry_keys<KEYS>(a, e + 1, nullptr) : 0;
  }
  __device__ __forceinline__ bool last() const { return t + 1 == T; }
  __device__ __forceinline__ void next() {
    if (++t < T) return;
    t = 0;
    if (++h < a.c.kv_heads) return;
    h = 0;
    do {
      ++e;
      n = n1;
      n1 = e + 1 < a.bs ? entry_keys<KEYS>(a, e + 1, nullptr) : 0;
    } while (n == 0 && e < a.bs);
    T = (int)((n + kTile - 1) / kTile);
  }
};

struct DecodeArgs {
  AttnArgs a;
  int slots;  // 16 KiB slots of the code ring
};

__host__ __device__ constexpr int64_t record_floats(int heads) { return heads * (2 + (int64_t)kTcDim); }

// The tiles of all entries before this thread's and in all; every thread of the block calls it.
template <int KEYS, int THREADS>
__device__ __forceinline__ void sum_tiles(const AttnArgs& a, int per, int64_t& before, int64_t& total, uint32_t* err) {
  __shared__ int64_t s_sum[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t mine = 0;
  for (int j = 0; j < per; ++j) {
    const int e = threadIdx.x * per + j;
    if (e < a.bs) mine += (entry_keys<KEYS>(a, e, err) + kTile - 1) / kTile;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  before = incl - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
}

template <int KEYS, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS == 8 ? 2 : 1)
    kv8_decode_kernel(const DecodeArgs g, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  constexpr int NC = 2 * HEADS;               // columns: hi, lo
  constexpr int kColBytes = NC * 128;         // Q or P in shared memory
  constexpr uint32_t kTmemCols = 4 * NC;      // S[2], O[2]
  constexpr int kPages = kTile / 16;          // block-table pages of a tile at most
  constexpr int kMetaN = KEYS == kRows ? kTile : kPages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kNumBars];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_start[3];
  __shared__ float s_ks[kMeta][kMetaN], s_vs[kMeta][kMetaN];
  __shared__ float s_qinv[4][HEADS];  // a pair's stay until the softmax has passed it: two more pairs on
  __shared__ __align__(16) float s_max[2][4][HEADS];
  __shared__ float s_sum[4][HEADS];
  const AttnArgs& a = g.a;
  const Cache& c = a.c;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t off_q = g.slots * kSlotBytes, off_p = off_q + 2 * kColBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  volatile int* abort_flag = &s_abort;
  auto wait = [&](int i, uint32_t parity) { return mbar_wait(bar(i), parity, abort_flag, a.err); };

  // ---- this CTA's share and where it begins
  const int per = (a.bs + kThreads - 1) / kThreads;
  int64_t before, tiles;
  sum_tiles<KEYS, kThreads>(a, per, before, tiles, blockIdx.x == 0 ? a.err : nullptr);
  const int64_t total = tiles * c.kv_heads;
  const int64_t ctas = min((int64_t)gridDim.x, total);  // no share is empty
  allow_next_grid();
  if (blockIdx.x >= ctas) return;  // uniform over the CTA
  const int64_t lo = share_lo(total, blockIdx.x, ctas), hi = share_lo(total, blockIdx.x + 1, ctas);
  {
    int64_t at = before * c.kv_heads;
    for (int j = 0; j < per; ++j) {
      const int e = threadIdx.x * per + j;
      if (e >= a.bs || at > lo) break;
      const int64_t T = (entry_keys<KEYS>(a, e, nullptr) + kTile - 1) / kTile;
      if (lo < at + T * c.kv_heads) {
        const int64_t r = lo - at;
        s_start[0] = e;
        s_start[1] = (int)(r / T);
        s_start[2] = (int)(r % T);
      }
      at += T * c.kv_heads;
    }
  }
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < g.slots; ++i) {
      mbar_init(bar(kBarFull + i), 1);
      mbar_init(bar(kBarEmpty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kBarQ + i), 32);
      mbar_init(bar(kBarQFree + i), 1);
      mbar_init(bar(kBarS + i), 1);
      mbar_init(bar(kBarP + i), kSoft);
      mbar_init(bar(kBarO + i), 1);
    }
    for (int i = 0; i < kMeta; ++i) {
      mbar_init(bar(kBarMeta + i), 32);
      mbar_init(bar(kBarMetaFree + i), kSoft);
    }
    mbar_init(bar(kBarDone), 1);
    mbar_init_fence();
  }
  if (warp == 5) tmem_alloc(smem_u32(&s_tmem), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int count = (int)(hi - lo);
  Walk<KEYS> w(a, s_start[0], s_start[1], s_start[2]);
  const int64_t pool_rows = (int64_t)c.num_blocks * c.kv_heads * c.block;

  if (warp == 4) {
    // ================================================================ codes
    const int pages = kTile >> c.shift;
    int issued = 0;
    for (int i = 0; i < count; ++i, w.next()) {
      int4 row;
      uint32_t mask = 0xffffffffu;
      if (KEYS == kTable) {
        const int64_t j = (int64_t)w.t * kTile + ((int64_t)lane << c.shift);
        int32_t b = -1;
        if (lane < pages && j < w.n) b = a.table[a.reqs[w.e] * a.table_stride + (j >> c.shift)];
        const bool in = b >= 0 && b < c.num_blocks;
        mask = __ballot_sync(0xffffffffu, in);
        row.x = in ? (b * c.kv_heads + w.h) * c.block : 0;
      } else {
        const int64_t j = (int64_t)w.t * kTile + lane * 4;
        const int32_t* p = a.rows + (int64_t)w.e * a.rows_stride + j;
        int32_t r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          r[u] = j + u < w.n ? p[u] : -1;
          const bool in = r[u] >= 0 && (r[u] >> c.shift) < c.num_blocks;
          r[u] = in ? ((r[u] >> c.shift) * c.kv_heads + w.h) * c.block + (r[u] & (c.block - 1)) : (int32_t)pool_rows;
        }
        row = make_int4(r[0], r[1], r[2], r[3]);
      }
      bool ok = true;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int s = issued % g.slots, turn = issued / g.slots;
        ok = turn == 0 || wait(kBarEmpty + s, (turn - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t full = bar(kBarFull + s), dst = base + s * kSlotBytes;
        if (lane == 0)
          mbar_arrive_expect(full, KEYS == kTable ? (uint32_t)__popc(mask) << (c.shift + 7) : (uint32_t)kSlotBytes);
        __syncwarp();
        if (KEYS == kTable) {
          if (mask >> lane & 1) tma_load_rows(dst + (lane << (c.shift + 7)), v ? &map_v : &map_k, row.x, full);
        } else {
          tma_gather_rows(dst + lane * 512, v ? &map_v : &map_k, row, full);
        }
        ++issued;
      }
      if (!ok) break;
    }
    // every copy has landed before the CTA's memory is given up
    for (int i = max(0, issued - g.slots); i < issued; ++i)
      mbar_wait(bar(kBarFull + i % g.slots), (i / g.slots) & 1, abort_flag, a.err, true);
  } else if (warp == 5) {
    // ================================================================ MMA issue
    if (lane == 0) {
      constexpr uint32_t kIdS = instr_desc_e4m3(0, 0, kTile, NC), kIdO = instr_desc_e4m3(1, 0, kTcDim, NC);
      bool ok = true;
      int pair = 0;  // (entry, head) segments so far
      bool first = true;
      auto scores = [&](int i) {
        const int s = (2 * i) % g.slots, qb = pair & 1;
        ok = ok && (!first || wait(kBarQ + qb, (pair >> 1) & 1)) && wait(kBarFull + s, ((2 * i) / g.slots) & 1);
        if (!ok) return;
        tc_fence_after();
        umma_e4m3_x4(tmem + (i & 1) * NC, desc_k(base + s * kSlotBytes), desc_k(base + off_q + qb * kColBytes), 2, 2,
                     kIdS, 0u);
        umma_commit(bar(kBarS + (i & 1)));
        umma_commit(bar(kBarEmpty + s));
        first = w.last();
        if (first) {
          umma_commit(bar(kBarQFree + qb));
          ++pair;
        }
        w.next();
      };
      scores(0);
      if (count > 1) scores(1);
      for (int i = 0; i < count && ok; ++i) {
        const int s = (2 * i + 1) % g.slots;
        ok = wait(kBarFull + s, ((2 * i + 1) / g.slots) & 1) && wait(kBarP + (i & 1), (i >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        umma_e4m3_x4(tmem + 2 * NC + (i & 1) * NC, desc_mn(base + s * kSlotBytes, kSlotBytes),
                     desc_k(base + off_p + (i & 1) * kColBytes), 256, 2, kIdO, 0u);
        umma_commit(bar(kBarO + (i & 1)));
        umma_commit(bar(kBarEmpty + s));
        if (i + 2 < count) scores(i + 2);
      }
      // the tensor memory is freed after the last MMA that was issued
      umma_commit(bar(kBarDone));
      mbar_wait(bar(kBarDone), 0, abort_flag, a.err, true);
    }
    __syncwarp();
  } else if (warp == 6) {
    // ================================================================ queries
    int pair = 0;
    bool first = true;
    for (int i = 0; i < count; ++i, w.next()) {
      if (!first) {
        first = w.last();
        continue;
      }
      const int qb = pair & 1;
      if (pair >= 2 && !__all_sync(0xffffffffu, wait(kBarQFree + qb, ((pair >> 1) - 1) & 1))) break;
      uint8_t* dst = smem + off_q + qb * kColBytes;
#pragma unroll
      for (int r = 0; r < HEADS; ++r) {
        float x[4] = {};
        if (r < a.group) {
          const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.q) + w.e * a.q_stride +
                                                          (int64_t)(w.h * a.group + r) * kTcDim + lane * 4);
          x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xFFFF0000u);
          x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xFFFF0000u);
        }
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool finite = fabsf(x[k]) <= 3.402823466e38f;
          if (finite) most = fmaxf(most, fabsf(x[k]));
          else x[k] = __uint_as_float(0x7FFFFFFFu);  // an infinite query has no scores either
        }
        const int k2 = fit_exponent(warp_max(most));
        const float up = exp2_int(k2);
        uint32_t h0, l0, h1, l1;
        split_e4m3x2(x[0] * up, x[1] * up, kLo, h0, l0);
        split_e4m3x2(x[2] * up, x[3] * up, kLo, h1, l1);
        *reinterpret_cast<uint32_t*>(dst + swz(r, lane * 4)) = h0 | (h1 << 16);
        *reinterpret_cast<uint32_t*>(dst + swz(HEADS + r, lane * 4)) = l0 | (l1 << 16);
        if (lane == 0) s_qinv[pair & 3][r] = a.scale_log2 * exp2_int(-k2);
      }
      fence_async_shared();
      mbar_arrive(bar(kBarQ + qb));
      ++pair;
      first = w.last();
    }
  } else if (warp == 7) {
    // ================================================================ scales
    for (int i = 0; i < count; ++i, w.next()) {
      const int m = i % kMeta;
      constexpr int N = (kMetaN + 31) / 32;
      float ks[N], vs[N];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int k = u * 32 + lane;
        const int64_t j = KEYS == kRows ? (int64_t)w.t * kTile + k : (int64_t)w.t * kTile + ((int64_t)k << c.shift);
        int64_t slot = -1;
        if (k < (KEYS == kRows ? kTile : kTile >> c.shift) && j < w.n)
          slot = key_slot<KEYS>(a, w.e, KEYS == kRows ? 0 : a.reqs[w.e], j, w.h == 0 ? a.err : nullptr);
        const int64_t bh = slot < 0 ? 0 : (slot >> c.shift) * c.kv_heads + w.h;
        ks[u] = slot < 0 ? 0.f : c.k_scale[bh];
        vs[u] = slot < 0 ? __uint_as_float(kMasked) : c.v_scale[bh];
      }
      if (i >= kMeta && !__all_sync(0xffffffffu, wait(kBarMetaFree + m, ((i / kMeta) - 1) & 1))) break;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int k = u * 32 + lane;
        if (k < kMetaN) s_ks[m][k] = ks[u], s_vs[m][k] = vs[u];
      }
      mbar_arrive(bar(kBarMeta + m));
    }
  } else {
    // ================================================================ softmax (warps 0-3)
    // Once a wait has run out (ok false) the warps still walk to the end, for
    // the barrier they share, but touch no tensor memory and write nothing.
    const int tok = threadIdx.x;  // token of the tile, and channel of the output
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    float M[HEADS], l[HEADS], corr[HEADS], O[HEADS];
    int pair = 0;
    bool first = true, ok = true;
    auto columns = [&](uint32_t col, uint32_t (&v)[NC]) {
#pragma unroll
      for (int k = 0; k < NC; k += 16) tmem_ld16(lane_base + col + k, *reinterpret_cast<uint32_t(*)[16]>(&v[k]));
      tmem_ld_wait();
    };
    auto add_product = [&](int i, const float (&by)[HEADS]) {  // O = O by + product of tile i
      ok = __all_sync(0xffffffffu, ok && wait(kBarO + (i & 1), (i >> 1) & 1));
      if (!ok) return;
      tc_fence_after();
      uint32_t v[NC];
      columns(2 * NC + (i & 1) * NC, v);
#pragma unroll
      for (int r = 0; r < HEADS; ++r)
        O[r] = fmaf(O[r], by[r], fmaf(__uint_as_float(v[HEADS + r]), 1.f / kLo, __uint_as_float(v[r])));
    };
    for (int i = 0; i < count; ++i, w.next()) {
      const int b = i & 1, m = i % kMeta;
      if (first) {
#pragma unroll
        for (int r = 0; r < HEADS; ++r) M[r] = -INFINITY, l[r] = 0.f, O[r] = 0.f, corr[r] = 0.f;
        ok = ok && wait(kBarQ + (pair & 1), (pair >> 1) & 1);
      }
      ok = ok && wait(kBarMeta + m, (i / kMeta) & 1);
      const int mk = KEYS == kRows ? tok : tok >> c.shift;
      const float ks = s_ks[m][mk], vs = s_vs[m][mk];
      const bool seen = (int64_t)w.t * kTile + tok < w.n && __float_as_uint(vs) != kMasked;
      ok = __all_sync(0xffffffffu, ok && wait(kBarS + b, (i >> 1) & 1));
      mbar_arrive(bar(kBarMetaFree + m));
      uint32_t v[NC] = {};
      if (ok) {
        tc_fence_after();
        columns(b * NC, v);
      }
      // vs = vm 2^ev; ev stays where 2^-ev and the sums of it are normal numbers
      const int ev = seen ? min(126, max(-100, (int)((__float_as_uint(vs) >> 23) & 255) - 127)) : 0;
      const float back = seen ? exp2_int(-ev) : 0.f;
      const float vm = seen ? vs * back * kPScale : 0.f;
      float u[HEADS];
#pragma unroll
      for (int r = 0; r < HEADS; ++r) {
        const float s = fmaf(__uint_as_float(v[HEADS + r]), 1.f / kLo, __uint_as_float(v[r])) * (s_qinv[pair & 3][r] * ks);
        u[r] = seen ? s + (float)ev : -INFINITY;
        const float most = warp_max(u[r]);
        if (lane == r) s_max[b][warp][r] = most;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float before_corr[HEADS];
      uint32_t hi8[HEADS / 2], lo8[HEADS / 2];
#pragma unroll
      for (int r = 0; r < HEADS; r += 2) {
        float wgt[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int q = r + k;
          const float mn =
              fmaxf(fmaxf(fmaxf(s_max[b][0][q], s_max[b][1][q]), fmaxf(s_max[b][2][q], s_max[b][3][q])), M[q]);
          const float ref = mn == -INFINITY ? 0.f : mn;
          before_corr[q] = corr[q];
          corr[q] = ex2(M[q] - ref);
          M[q] = mn;
          const float p = ex2(u[q] - ref);
          l[q] = fmaf(l[q], corr[q], p * back);
          wgt[k] = p * vm;
        }
        split_e4m3x2(wgt[0], wgt[1], kLo, hi8[r / 2], lo8[r / 2]);
      }
      uint8_t* P = smem + off_p + b * kColBytes;
#pragma unroll
      for (int r = 0; r < HEADS; ++r) {
        P[swz(r, tok)] = (uint8_t)(hi8[r / 2] >> (8 * (r & 1)));
        P[swz(HEADS + r, tok)] = (uint8_t)(lo8[r / 2] >> (8 * (r & 1)));
      }
      // what a masked token's row of V holds (stale codes, maybe NaN) must not meet its zero weight
      if (!__all_sync(0xffffffffu, seen)) {
        const int s = (2 * i + 1) % g.slots;
        ok = __all_sync(0xffffffffu, ok && wait(kBarFull + s, ((2 * i + 1) / g.slots) & 1));
        if (ok && !seen) {
          uint4* row = reinterpret_cast<uint4*>(smem + s * kSlotBytes + tok * 128);
#pragma unroll
          for (int k = 0; k < 8; ++k) row[k] = make_uint4(0, 0, 0, 0);
        }
      }
      fence_async_shared();
      tc_fence_before();
      mbar_arrive(bar(kBarP + b));
      if (!first) add_product(i - 1, before_corr);
      first = w.last();
      if (!first && i + 1 < count) continue;

      // ---- the end of the pair, or of the share: the result, or a record of this part
      add_product(i, corr);
#pragma unroll
      for (int r = 0; r < HEADS; ++r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        if (lane == 0) s_sum[warp][r] = l[r];
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (ok) {
        const bool whole = i >= w.t && first;  // all of the pair's tiles are this CTA's
        float* rec = a.part + ((int64_t)blockIdx.x * 2 + (pair > 0)) * record_floats(HEADS);
#pragma unroll
        for (int r = 0; r < HEADS; ++r) {
          const float sum = (s_sum[0][r] + s_sum[1][r]) + (s_sum[2][r] + s_sum[3][r]);
          const float o = O[r] * (1.f / kPScale);
          if (whole) {
            if (r < a.group)
              static_cast<__nv_bfloat16*>(a.out)[w.e * a.out_stride + (int64_t)(w.h * a.group + r) * kTcDim + tok] =
                  __float2bfloat16_rn(sum == 0.f ? 0.f : o / sum);
          } else {
            if (tok == 0) rec[r] = M[r], rec[HEADS + r] = sum;
            rec[2 * HEADS + r * kTcDim + tok] = o;
          }
        }
      }
      ++pair;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the records of entry blockIdx.x, KV head blockIdx.y where its tiles
// lay in several shares; an entry without keys gets zeros.  A warp per query
// head, four channels per lane; the records' weights first, a lane each.
constexpr int kJoinThreads = 256;
template <int KEYS, int HEADS>
__global__ void __launch_bounds__(kJoinThreads) kv8_decode_join_kernel(const DecodeArgs g, int64_t ctas) {
  __shared__ int64_t s_before;
  const AttnArgs& a = g.a;
  const int e = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (a.bs + kJoinThreads - 1) / kJoinThreads;
  int64_t before, tiles;
  sum_tiles<KEYS, kJoinThreads>(a, per, before, tiles, nullptr);
  if (threadIdx.x == e / per) {
    for (int i = e / per * per; i < e; ++i) before += (entry_keys<KEYS>(a, i, nullptr) + kTile - 1) / kTile;
    s_before = before;
  }
  __syncthreads();
  const int64_t total = tiles * a.c.kv_heads;
  const int64_t T = (entry_keys<KEYS>(a, e, nullptr) + kTile - 1) / kTile;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + e * a.out_stride + (int64_t)h * a.group * kTcDim;
  wait_prior_grid();
  if (T == 0) {
    for (int i = threadIdx.x; i < a.group * kTcDim; i += kJoinThreads) out[i] = __float2bfloat16_rn(0.f);
    return;
  }
  ctas = min(ctas, total);
  const int64_t first = s_before * a.c.kv_heads + h * T, last = first + T - 1;
  auto owner = [&](int64_t x) {
    int64_t c = x * ctas / total;
    while (share_lo(total, c + 1, ctas) <= x) ++c;
    while (share_lo(total, c, ctas) > x) --c;
    return c;
  };
  const int64_t c0 = owner(first), c1 = owner(last);
  if (c0 == c1) return;  // written by its CTA
  const int parts = (int)(c1 - c0 + 1);
  const int skip = first > share_lo(total, c0, ctas) ? 1 : 0;  // the first CTA's record lies behind another pair's
  auto record = [&](int k) { return a.part + ((c0 + k) * 2 + (k == 0 ? skip : 0)) * record_floats(HEADS); };
  for (int r = warp; r < a.group; r += kJoinThreads / 32) {
    float M = -INFINITY;
    for (int k = lane; k < parts; k += 32) M = fmaxf(M, record(k)[r]);
    M = warp_max(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float sum = 0.f, o[4] = {};
    for (int k0 = 0; k0 < parts; k0 += 32) {
      float wgt = 0.f;
      if (k0 + lane < parts) {
        const float* p = record(k0 + lane);
        wgt = ex2(p[r] - ref);
        sum = fmaf(wgt, p[HEADS + r], sum);
      }
      const int n = min(32, parts - k0);
#pragma unroll 8
      for (int k = 0; k < n; ++k) {
        const float f = __shfl_sync(0xffffffffu, wgt, k);
        const float4 v = *reinterpret_cast<const float4*>(record(k0 + k) + 2 * HEADS + r * kTcDim + lane * 4);
        o[0] = fmaf(f, v.x, o[0]), o[1] = fmaf(f, v.y, o[1]), o[2] = fmaf(f, v.z, o[2]), o[3] = fmaf(f, v.w, o[3]);
      }
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(out + r * kTcDim + lane * 4) =
        make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
  }
}


template <int KEYS, int HEADS>
int launch(DecodeArgs g, int64_t ctas, cudaStream_t s) {
  constexpr int fixed = 1024 + 4 * 2 * HEADS * 128;
  constexpr int slots = HEADS == 8 ? 6 : 10;  // two CTAs per SM of the 16-column kernel share its 228 KiB
  static_assert(slots >= 4 && slots <= kMaxSlots, "ring");
  g.slots = slots;
  const size_t smem = fixed + slots * kSlotBytes;
  static SmemLimit limit;
  int rc = limit.ensure((const void*)kv8_decode_kernel<KEYS, HEADS>, smem);
  if (rc != QQ_OK) return rc;
  CUtensorMap mk, mv;
  const int64_t rows = (int64_t)g.a.c.num_blocks * g.a.c.kv_heads * g.a.c.block;
  const int box = KEYS == kTable ? g.a.c.block : 1;
  if ((rc = encode_rows(&mk, g.a.c.k, rows, box)) != QQ_OK) return rc;
  if ((rc = encode_rows(&mv, g.a.c.v, rows, box)) != QQ_OK) return rc;
  kv8_decode_kernel<KEYS, HEADS><<<(unsigned)ctas, kThreads, smem, s>>>(g, mk, mv);
  if ((rc = launch_status()) != QQ_OK) return rc;
  return launch_pdl(kv8_decode_join_kernel<KEYS, HEADS>, dim3(g.a.bs, g.a.c.kv_heads), dim3(kJoinThreads), 0, s, g, ctas);
}

int64_t decode_ctas(int bs, int kv_heads, int group, int64_t max_keys) {
  const int64_t most = (int64_t)bs * kv_heads * ((max_keys + kTile - 1) / kTile);
  const int64_t ctas = (int64_t)device_sm_count() * (group <= 8 ? 2 : 1);
  return most < ctas ? most : ctas;
}

}  // namespace

bool decode_tc_fits(const AttnArgs& a, int dtype) {
  return dtype == QQ_BF16 && a.c.dim == kTcDim && a.group <= 16 && (a.q_stride * 2) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && (a.out_stride * 2) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(a.out) % 8 == 0;
}

size_t decode_tc_workspace(int bs, int kv_heads, int group, int64_t max_keys) {
  return sizeof(float) * (size_t)(decode_ctas(bs, kv_heads, group, max_keys) * 2 * record_floats(group <= 8 ? 8 : 16));
}

int run_decode_tc(const AttnArgs& a, int keys, int64_t max_keys, size_t ws_bytes, cudaStream_t s) {
  if (a.part == nullptr || ws_bytes < decode_tc_workspace(a.bs, a.c.kv_heads, a.group, max_keys)) return QQ_ERR_WORKSPACE;
  DecodeArgs g{};
  g.a = a;
  const int64_t ctas = decode_ctas(a.bs, a.c.kv_heads, a.group, max_keys);
  if (a.group <= 8) return keys == kTable ? launch<kTable, 8>(g, ctas, s) : launch<kRows, 8>(g, ctas, s);
  return keys == kTable ? launch<kTable, 16>(g, ctas, s) : launch<kRows, 16>(g, ctas, s);
}

}  // namespace kv8
}  // namespace qq

// One query token per request over the 8-bit block cache on the
// fifth-generation tensor cores (bf16 queries, head_dim 128, up to 16 query
// heads per KV head): the whole sequence through the block table, or listed rows.
//
// Bound by the bytes of the codes (2 x 128 per token and KV head), so the
// codes go from HBM to shared memory (TMA) to the tensor cores without a
// conversion: both products have an operand of the other side in e4m3, held
// by a pair hi + lo / 16 (queries) or hi + lo / 32 (weights) in two columns of
// one MMA: 8 significant bits, bf16's, down to a fixed part of the largest.
//   S^T [128 tokens x NC] = K [128 x 128] . Q^T      NC = 2 x 8 (or 2 x 16)
//   O^T [128 dims x NC]   = V^T [128 x 128] . P      columns: heads hi, heads lo
// A tile of 128 tokens is a row per thread in both, so each thread has one
// token's scores of all heads, and later one channel of all heads.
//
// Scales: a token's score is S ks q^-1 log2(e) scaling; its weight into the V
// product is 2^(s - R) vs.  With vs = vm 2^ev the reference R is a maximum of
// s + ev, so what enters the product, vm 2^(s + ev - R), is at most 2 whatever
// the blocks' scales are, and the sum l takes 2^(s + ev - R) 2^-ev.
// R is the tile's own maximum, or 2^-kFall of the largest so far where that is
// more: O and l are multiplied by 2^(R before - R), which may be above 1, when a
// tile is added.  A weight in the product is a multiple of 2^-21 of 2^R, with 8
// bits down to 2^-13 of it.  Against the running maximum the tail of a row
// would lose those bits to one key with most of the mass, as attention sinks
// have it, while l kept them: 131,072 equal keys behind one of 95 % of the mass
// and a small value were off by 98 % of the result, and are by 0.1 %.
//
// Work: the tiles of all (request, KV head) pairs in a row, cut into equal
// shares, one per CTA (two CTAs per SM); a pair cut by a share's edge leaves
// (M, l, O) records that kv8_decode_join_kernel merges.
// Few pairs of moderate length (a lone request, a selection) take the other
// form: a cluster of 16, 8 or 4 CTAs to a pair, which joins its records through the
// CTAs' shared memory and so needs no second launch.
// Warps: 0-3 softmax, 4 TMA, 5 MMA issue, 6 queries, 7 scales.  The MMAs go
// S(0) S(1) O(0) S(2) O(1) ...: the softmax of a tile runs while the next
// tile's scores are made, and a tile's O is added in registers one tile later.
// Every wait is bounded (kWaitLimitNs); on expiry the CTA reports
// QQ_DEV_ERR_TIMEOUT, waits for its own copies and MMAs and returns.

#include <algorithm>
#include <atomic>
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
constexpr int kClusterTiles = 4;              // tiles of each of them at most
constexpr int kInv = 4;                        // pairs of which the softmax may not have seen the queries' scales
constexpr uint32_t kMasked = 0xFFFFFFFFu;      // a V scale's bits where the token takes no part
constexpr float kLo = 16.f;                    // queries: up to 448, whose rest is at most 16
constexpr float kPScale = 128.f;               // weights (at most 2) times this are e4m3's upper binades
constexpr float kPLo = 32.f;                   // their rest is at most 8
constexpr float kNone = -3.402823466e38f;      // the maximum of no keys: finite, so that differences are numbers
// How far the reference may lie below the largest score: keys that much lighter share steps of 2^-33 of the heaviest.
// A key of a block of zeros (scale 2^-126) adds up to 2^-kLeastEv to l, 2^kFall more once the reference has fallen:
// finite over 2^24 such keys.
constexpr float kFall = 12.f;
constexpr int kLeastEv = -90;

// mbarriers
enum : int {
  kBarFull = 0,                      // [slots] codes have landed
  kBarEmpty = kBarFull + kMaxSlots,  // [slots] codes have been read
  kBarQ = kBarEmpty + kMaxSlots,     // [2] queries written
  kBarQFree = kBarQ + 2,             // [2] queries read
  kBarInv = kBarQFree + 2,           // [kInv] the same for the softmax, which may be up to three pairs behind
  kBarMeta = kBarInv + kInv,          // [kMeta] scales written
  kBarMetaFree = kBarMeta + kMeta,   // [kMeta] scales read
  kBarS = kBarMetaFree + kMeta,      // [2] scores made
  kBarP = kBarS + 2,                 // [2] weights written
  kBarO = kBarP + 2,                 // [2] product made
  kBarDone = kBarO + 2,              // the last MMA has finished
  kNumBars = kBarDone + 1
};

// The tiles in equal shares: the first `more` shares have one tile more.
struct Shares {
  int64_t ctas, each, more;
  bool narrow;  // 32 bits hold all of it: a 64-bit division takes four times as long
  __device__ __forceinline__ Shares(int64_t total, int64_t grid) {
    ctas = min(grid, total);  // no share is empty
    narrow = total <= UINT32_MAX;
    each = ratio(total, max((int64_t)1, ctas));
    more = total - each * ctas;
  }
  __device__ __forceinline__ int64_t ratio(int64_t x, int64_t y) const {
    return narrow ? (uint32_t)x / (uint32_t)y : x / y;
  }
  __device__ __forceinline__ int64_t lo(int64_t c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int64_t owner(int64_t tile) const {  // the share that tile lies in
    const int64_t cut = more * (each + 1);
    return tile < cut ? ratio(tile, each + 1) : more + ratio(tile - cut, each);
  }
};

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

// N values per lane reduced over the warp's lanes (N 8 or 16): lanes hold halves
// of the values in turn, so lane L ends with value L / (32 / N) in N + 1 shuffles.
template <int N, typename Op>
__device__ __forceinline__ float reduce_lanes(float (&x)[N], int lane, Op op) {
  int m = 16;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, m >>= 1) {
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const bool up = (lane & m) != 0;
      const float send = up ? x[i] : x[i + n / 2], keep = up ? x[i + n / 2] : x[i];
      x[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, m));
    }
  }
#pragma unroll
  for (; m > 0; m >>= 1) x[0] = op(x[0], __shfl_xor_sync(0xffffffffu, x[0], m));
  return x[0];
}

struct DecodeArgs {
  AttnArgs a;
  int slots;        // 16 KiB slots of the code ring
  int64_t* before;  // [bs + 1] tiles of the entries before each, left by CTA 0 for the join
};

__host__ __device__ constexpr int64_t record_floats(int heads) { return heads * (2 + (int64_t)kTcDim); }

// The tiles of this thread's first entry, of all entries before it, and in all; every thread of the block calls it.
template <int KEYS, int THREADS>
__device__ __forceinline__ void sum_tiles(const AttnArgs& a, int per, int64_t& own, int64_t& before, int64_t& total,
                                          uint32_t* err) {
  __shared__ int64_t s_sum[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t mine = 0;
  own = 0;
  for (int j = 0; j < per; ++j) {
    const int e = threadIdx.x * per + j;
    if (e < a.bs) mine += (entry_keys<KEYS>(a, e, err) + kTile - 1) / kTile;
    if (j == 0) own = mine;
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

// CH channels from `col` on of query head r of (entry, KV head) (zeros past the group) as hi and lo columns of Q;
// called by all lanes of the warps that hold the head's 128 / CH pieces side by side.
template <int HEADS, int CH>
__device__ __forceinline__ void write_query(const AttnArgs& a, int e, int h, int r, int col, uint8_t* dst, float* qinv) {
  float x[CH] = {};
  if (r < a.group) {
    const uint2* q = reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.q) + e * a.q_stride +
                                                    (int64_t)(h * a.group + r) * kTcDim + col);
#pragma unroll
    for (int k = 0; k < CH / 4; ++k) {
      const uint2 u = q[k];
      x[4 * k] = __uint_as_float(u.x << 16), x[4 * k + 1] = __uint_as_float(u.x & 0xFFFF0000u);
      x[4 * k + 2] = __uint_as_float(u.y << 16), x[4 * k + 3] = __uint_as_float(u.y & 0xFFFF0000u);
    }
  }
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const bool finite = fabsf(x[k]) <= 3.402823466e38f;
    if (finite) most = fmaxf(most, fabsf(x[k]));
    else x[k] = __uint_as_float(0x7FFFFFFFu);  // an infinite query has no scores either
  }
#pragma unroll
  for (int o = 1; o < kTcDim / CH; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const int k2 = fit_exponent(most);
  const float up = exp2_int(k2);
#pragma unroll
  for (int k = 0; k < CH; k += 8) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) split_e4m3x2(x[k + 2 * u] * up, x[k + 2 * u + 1] * up, kLo, hi[u], lo[u]);
    *reinterpret_cast<uint2*>(dst + swz(r, col + k)) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
    *reinterpret_cast<uint2*>(dst + swz(HEADS + r, col + k)) = make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
  }
  if (col == 0) qinv[r] = a.scale_log2 * exp2_int(-k2);
}

// CLUSTER: a cluster of that many CTAs takes a pair and joins it itself.
template <int KEYS, int HEADS, int CLUSTER>
__global__ void __launch_bounds__(kThreads, HEADS == 8 ? 2 : 1)
    kv8_decode_kernel(const DecodeArgs g, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap row_k,
                      const __grid_constant__ CUtensorMap row_v) {
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
  __shared__ float s_qinv[kInv][HEADS];
  __shared__ __align__(16) float s_max[2][HEADS][4];
  __shared__ __align__(16) float s_sum[HEADS][4];
  const AttnArgs& a = g.a;
  const Cache& c = a.c;
  if (threadIdx.x < (KEYS == kRows ? 4 : 2))
    prefetch_map(threadIdx.x == 0 ? &map_k : threadIdx.x == 1 ? &map_v : threadIdx.x == 2 ? &row_k : &row_v);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t off_q = g.slots * kSlotBytes, off_p = off_q + 2 * kColBytes;
  // the same in all lanes, and known to be
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  volatile int* abort_flag = &s_abort;
  auto wait = [&](int i, uint32_t parity) { return mbar_wait<8>(bar(i), parity, abort_flag, a.err); };

  // ---- barriers and tensor memory, then this CTA's share and where it begins
  if (threadIdx.x == kThreads - 1) {
    s_abort = 0;
    for (int i = 0; i < g.slots; ++i) {
      mbar_init(bar(kBarFull + i), 1);
      mbar_init(bar(kBarEmpty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kBarQ + i), 1);
      mbar_init(bar(kBarQFree + i), 1);
      mbar_init(bar(kBarS + i), 1);
      mbar_init(bar(kBarP + i), kSoft / 32);
      mbar_init(bar(kBarO + i), 1);
    }
    for (int i = 0; i < kInv; ++i) mbar_init(bar(kBarInv + i), 1);
    for (int i = 0; i < kMeta; ++i) {
      mbar_init(bar(kBarMeta + i), 1);
      mbar_init(bar(kBarMetaFree + i), kSoft / 32);
    }
    mbar_init(bar(kBarDone), 1);
    mbar_init_fence();
  }
  if (warp == 5) tmem_alloc(smem_u32(&s_tmem), kTmemCols);
  wait_prior_grid();
  bool any = true;  // this CTA has tiles, `count` of them from s_start on
  int count;
  if constexpr (CLUSTER > 0) {
    const int pair = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER, e = pair / c.kv_heads, h = pair - e * c.kv_heads;
    const int64_t n = entry_keys<KEYS>(a, e, rank == 0 && h == 0 && threadIdx.x == 0 ? a.err : nullptr);
    const int T = (int)((n + kTile - 1) / kTile), each = T / CLUSTER, more = T % CLUSTER;
    count = each + (rank < more ? 1 : 0);
    if (threadIdx.x == 0) s_start[0] = e, s_start[1] = h, s_start[2] = rank * each + min(rank, more);
  } else {
    const int per = (a.bs + kThreads - 1) / kThreads;
    int64_t own, before, tiles;
    sum_tiles<KEYS, kThreads>(a, per, own, before, tiles, blockIdx.x == 0 ? a.err : nullptr);
    auto entry_tiles = [&](int j) {  // of this thread's entry j
      return j == 0 ? own : (entry_keys<KEYS>(a, threadIdx.x * per + j, nullptr) + kTile - 1) / kTile;
    };
    const Shares shares(tiles * c.kv_heads, gridDim.x);
    allow_next_grid();
    if (blockIdx.x == 0) {
      int64_t at = before;
      for (int j = 0; j < per; ++j) {
        const int e = threadIdx.x * per + j;
        if (e >= a.bs) break;
        g.before[e] = at;
        at += entry_tiles(j);
      }
      if (threadIdx.x == 0) g.before[a.bs] = tiles;
    }
    any = blockIdx.x < shares.ctas;
    const int64_t lo = shares.lo(blockIdx.x);
    count = any ? (int)(shares.lo(blockIdx.x + 1) - lo) : 0;
    {
      int64_t at = before * c.kv_heads;
      for (int j = 0; any && j < per; ++j) {
        const int e = threadIdx.x * per + j;
        if (e >= a.bs || at > lo) break;
        const int T = (int)entry_tiles(j);
        if (lo < at + (int64_t)T * c.kv_heads) {
          int r = (int)(lo - at), h = 0;
          if (r >= T) h = r / T, r -= h * T;
          s_start[0] = e;
          s_start[1] = h;
          s_start[2] = r;
        }
        at += (int64_t)T * c.kv_heads;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (CLUSTER > 0) allow_next_grid();
  if (!any) {  // uniform over the CTA
    if (warp == 5) tmem_dealloc(s_tmem, kTmemCols);
    return;
  }
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  count = __shfl_sync(0xffffffffu, count, 0);
  Walk<KEYS> w(a, s_start[0], s_start[1], s_start[2]);
  const int64_t pool_rows = (int64_t)c.num_blocks * c.kv_heads * c.block;

  if (CLUSTER > 0 && count == 0) {
    if (threadIdx.x < HEADS) {
      reinterpret_cast<float*>(smem)[threadIdx.x] = -INFINITY;
      reinterpret_cast<float*>(smem)[HEADS + threadIdx.x] = 0.f;
    }
  } else if (warp == 4) {
    // ================================================================ codes
    // the table entries or rows of a tile are loaded one tile ahead
    const int pages = kTile >> c.shift;
    int issued = 0;
    auto fetch = [&](const Walk<KEYS>& x, int32_t (&r)[4]) {
      r[0] = r[1] = r[2] = r[3] = -1;
      if (KEYS == kTable) {
        const int64_t j = (int64_t)x.t * kTile + ((int64_t)lane << c.shift);
        if (lane < pages && j < x.n) r[0] = a.table[a.reqs[x.e] * a.table_stride + (j >> c.shift)];
      } else {
        const int64_t j = (int64_t)x.t * kTile + lane * 4;
        const int32_t* p = a.rows + (int64_t)x.e * a.rows_stride + j;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (j + u < x.n) r[u] = p[u];
      }
    };
    Walk<KEYS> ahead = w;
    int32_t next[4];
    fetch(ahead, next);
    for (int i = 0; i < count; ++i, w.next()) {
      int32_t r[4] = {next[0], next[1], next[2], next[3]};
      if (i + 1 < count) {
        ahead.next();
        fetch(ahead, next);
      }
      int4 row;
      uint32_t mask, bytes;  // the lanes that copy a box; all bytes of the copies
      bool single = false;   // this lane copies single rows
      if (KEYS == kTable) {
        const int32_t b = r[0];
        const bool in = b >= 0 && b < c.num_blocks;
        mask = __ballot_sync(0xffffffffu, in);
        bytes = (uint32_t)__popc(mask) << (c.shift + 7);
        row.x = in ? (b * c.kv_heads + w.h) * c.block : 0;
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool in = r[u] >= 0 && (r[u] >> c.shift) < c.num_blocks;
          r[u] = in ? ((r[u] >> c.shift) * c.kv_heads + w.h) * c.block + (r[u] & (c.block - 1)) : (int32_t)pool_rows;
        }
        row = make_int4(r[0], r[1], r[2], r[3]);
        // 16 listed rows that follow one another (a page selection's do) are one box of the pool, the others
        // go four at a time: the copy engine takes a row of a gather as long as several rows of a box
        const int32_t lead = __shfl_sync(0xffffffffu, r[0], lane & ~3);
        const bool follow = r[3] < pool_rows && r[0] == lead + 4 * (lane & 3) && r[1] == r[0] + 1 && r[2] == r[0] + 2 &&
                            r[3] == r[0] + 3;
        const uint32_t f = __ballot_sync(0xffffffffu, follow);
        const bool box = (f >> (lane & ~3) & 15u) == 15u;
        mask = __ballot_sync(0xffffffffu, box && (lane & 3) == 0);
        single = !box && (r[0] < pool_rows || r[1] < pool_rows || r[2] < pool_rows || r[3] < pool_rows);
        bytes = (uint32_t)__popc(mask) * 2048u + (uint32_t)__popc(__ballot_sync(0xffffffffu, single)) * 512u;
      }
      bool ok = true;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int s = issued % g.slots, turn = issued / g.slots;
        ok = turn == 0 || wait(kBarEmpty + s, (turn - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t full = bar(kBarFull + s), dst = base + s * kSlotBytes;
        if (lane == 0) mbar_arrive_expect(full, bytes);
        __syncwarp();
        if (mask >> lane & 1)
          tma_load_rows(dst + (KEYS == kTable ? lane << (c.shift + 7) : lane * 512), v ? &map_v : &map_k, row.x, full);
        if (KEYS == kRows && single) tma_gather_rows(dst + lane * 512, v ? &row_v : &row_k, row, full);
        ++issued;
      }
      if (!ok) break;
    }
    // every copy has landed before the CTA's memory is given up
    for (int i = max(0, issued - g.slots); i < issued; ++i)
      mbar_wait(bar(kBarFull + i % g.slots), (i / g.slots) & 1, abort_flag, a.err, true);
  } else if (warp == 5) {
    // ================================================================ MMA issue
    constexpr uint32_t kIdS = instr_desc_e4m3(0, 0, kTile, NC), kIdO = instr_desc_e4m3(1, 0, kTcDim, NC);
    auto all = [&](int i, uint32_t parity) { return __all_sync(0xffffffffu, wait(i, parity)); };
    bool ok = true;
    int pair = 0;  // (entry, head) segments so far
    bool first = true;
    auto scores = [&](int i) {
      const int s = (2 * i) % g.slots, qb = pair & 1;
      ok = ok && (!first || all(kBarQ + qb, (pair >> 1) & 1)) && all(kBarFull + s, ((2 * i) / g.slots) & 1);
      if (!ok) return;
      tc_fence_after();
      umma_e4m3_x4_warp(tmem + (i & 1) * NC, desc_k(base + s * kSlotBytes), desc_k(base + off_q + qb * kColBytes), 2, 2,
                        kIdS, 0u);
      umma_commit_warp(bar(kBarS + (i & 1)));
      umma_commit_warp(bar(kBarEmpty + s));
      first = w.last();
      if (first) {
        umma_commit_warp(bar(kBarQFree + qb));
        ++pair;
      }
      w.next();
    };
    scores(0);
    if (count > 1) scores(1);
    for (int i = 0; i < count && ok; ++i) {
      const int s = (2 * i + 1) % g.slots;
      ok = all(kBarFull + s, ((2 * i + 1) / g.slots) & 1) && all(kBarP + (i & 1), (i >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      umma_e4m3_x4_warp(tmem + 2 * NC + (i & 1) * NC, desc_mn(base + s * kSlotBytes, kSlotBytes),
                        desc_k(base + off_p + (i & 1) * kColBytes), 256, 2, kIdO, 0u);
      umma_commit_warp(bar(kBarO + (i & 1)));
      umma_commit_warp(bar(kBarEmpty + s));
      if (i + 2 < count) scores(i + 2);
    }
    // the tensor memory is freed after the last MMA that was issued
    umma_commit_warp(bar(kBarDone));
    mbar_wait(bar(kBarDone), 0, abort_flag, a.err, true);
  } else if (warp == 6) {
    // ================================================================ queries
    int pair = 0;
    bool first = true;
    for (int i = 0; i < count; ++i, w.next()) {
      const bool begins = first;
      first = w.last();
      if (!begins) continue;
      const int p = pair++, qb = p & 1;
      if (p == 0) continue;  // the softmax warps write that one
      if (p >= 2 && !__all_sync(0xffffffffu, wait(kBarQFree + qb, ((p >> 1) - 1) & 1))) break;
#pragma unroll
      for (int r0 = 0; r0 < HEADS; r0 += 8)  // four lanes per head, 32 channels each
        write_query<HEADS, 32>(a, w.e, w.h, r0 + (lane >> 2), (lane & 3) * 32, smem + off_q + qb * kColBytes,
                               s_qinv[p % kInv]);
      fence_async_shared();
      mbar_arrive_warp(bar(kBarQ + qb));
      mbar_arrive_warp(bar(kBarInv + p % kInv));
    }
  } else if (warp == 7) {
    // ================================================================ scales
    // the slots of a tile's tokens are found one tile ahead
    constexpr int N = (kMetaN + 31) / 32;
    auto find = [&](const Walk<KEYS>& x, int32_t (&slot)[N]) {
      const int64_t req = KEYS == kRows ? 0 : a.reqs[x.e];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int k = u * 32 + lane;
        const int64_t j = (int64_t)x.t * kTile + (KEYS == kRows ? k : (int64_t)k << c.shift);
        slot[u] = -1;
        if (k < (KEYS == kRows ? kTile : kTile >> c.shift) && j < x.n)
          slot[u] = (int32_t)key_slot<KEYS>(a, x.e, req, j, x.h == 0 ? a.err : nullptr);
      }
    };
    Walk<KEYS> ahead = w;
    int32_t next[N];
    find(ahead, next);
    for (int i = 0; i < count; ++i, w.next()) {
      const int m = i % kMeta;
      float ks[N], vs[N];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const bool in = next[u] >= 0;
        const int64_t bh = in ? (int64_t)(next[u] >> c.shift) * c.kv_heads + w.h : 0;
        ks[u] = in ? c.k_scale[bh] : 0.f;
        vs[u] = in ? c.v_scale[bh] : __uint_as_float(kMasked);
      }
      if (i + 1 < count) {
        ahead.next();
        find(ahead, next);
      }
      if (i >= kMeta && !__all_sync(0xffffffffu, wait(kBarMetaFree + m, ((i / kMeta) - 1) & 1))) break;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int k = u * 32 + lane;
        if (k < kMetaN) s_ks[m][k] = ks[u], s_vs[m][k] = vs[u];
      }
      mbar_arrive_warp(bar(kBarMeta + m));
    }
  } else {
    // ================================================================ softmax (warps 0-3)
    // Once a wait has run out (ok false) the warps still walk to the end, for
    // the barrier they share, but touch no tensor memory and write nothing.
    const int tok = threadIdx.x;  // token of the tile, and channel of the output
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    float M[HEADS], R[HEADS], l[HEADS], step[HEADS], O[HEADS];  // largest score, reference, sum, 2^(R before - R), output
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
        O[r] = fmaf(O[r], by[r], fmaf(__uint_as_float(v[HEADS + r]), 1.f / kPLo, __uint_as_float(v[r])));
    };
    // the first queries by all four warps: nothing else can go on before them (1.8 us with one warp)
    constexpr int kCh = kTcDim * HEADS / kSoft;
    write_query<HEADS, kCh>(a, w.e, w.h, tok / (kTcDim / kCh), tok % (kTcDim / kCh) * kCh, smem + off_q, s_qinv[0]);
    fence_async_shared();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (warp == 0) {
      mbar_arrive_warp(bar(kBarQ));
      mbar_arrive_warp(bar(kBarInv));
    }
    for (int i = 0; i < count; ++i, w.next()) {
      const int b = i & 1, m = i % kMeta;
      if (first) {
#pragma unroll
        for (int r = 0; r < HEADS; ++r) M[r] = R[r] = kNone, l[r] = 0.f, O[r] = 0.f, step[r] = 0.f;
        // Q's own barrier may be two phases on by now: with a tile to a pair the
        // scores run two pairs ahead of this, and the queries two more.  The
        // scales of pair p + kInv are written after S(p + 2), so after P(p).
        ok = ok && wait(kBarInv + pair % kInv, (pair / kInv) & 1);
      }
      ok = ok && wait(kBarMeta + m, (i / kMeta) & 1);
      const int mk = KEYS == kRows ? tok : tok >> c.shift;
      const float ks = s_ks[m][mk], vs = s_vs[m][mk];
      const bool seen = (int64_t)w.t * kTile + tok < w.n && __float_as_uint(vs) != kMasked;
      ok = __all_sync(0xffffffffu, ok && wait(kBarS + b, (i >> 1) & 1));
      mbar_arrive_warp(bar(kBarMetaFree + m));
      uint32_t v[NC] = {};
      if (ok) {
        tc_fence_after();
        columns(b * NC, v);
      }
      // vs = vm 2^ev; ev stays where 2^-ev and the sums of it are normal numbers
      const int ev = seen ? min(126, max(kLeastEv, (int)((__float_as_uint(vs) >> 23) & 255) - 127)) : 0;
      const float back = seen ? exp2_int(-ev) : 0.f;
      const float vm = seen ? vs * back * kPScale : 0.f;
      float u[HEADS], most[HEADS];
#pragma unroll
      for (int r = 0; r < HEADS; ++r) {
        const float s = fmaf(__uint_as_float(v[HEADS + r]), 1.f / kLo, __uint_as_float(v[r])) * (s_qinv[pair % kInv][r] * ks);
        u[r] = seen ? s + (float)ev : -INFINITY;
        most[r] = u[r];
      }
      const float top = reduce_lanes(most, lane, [](float x, float y) { return fmaxf(x, y); });
      if (lane % (32 / HEADS) == 0) s_max[b][lane / (32 / HEADS)][warp] = top;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      float before[HEADS];
      uint32_t hi8[HEADS / 2], lo8[HEADS / 2];
#pragma unroll
      for (int r = 0; r < HEADS; r += 2) {
        float wgt[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int q = r + k;
          const float4 m4 = *reinterpret_cast<const float4*>(s_max[b][q]);
          const float m = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
          M[q] = fmaxf(m, M[q]);
          const float ref = fmaxf(m, M[q] - kFall);
          before[q] = step[q];
          step[q] = ex2(R[q] - ref);
          R[q] = ref;
          const float p = ex2(u[q] - ref);
          l[q] = fmaf(l[q], step[q], p * back);
          wgt[k] = p * vm;
        }
        split_e4m3x2(wgt[0], wgt[1], kPLo, hi8[r / 2], lo8[r / 2]);
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
      mbar_arrive_warp(bar(kBarP + b));
      if (!first) add_product(i - 1, before);
      first = w.last();
      if (!first && i + 1 < count) continue;

      // ---- the end of the pair, or of the share: the result, or a record of this part
      add_product(i, step);
      const float part = reduce_lanes(l, lane, [](float x, float y) { return x + y; });
      if (lane % (32 / HEADS) == 0) s_sum[lane / (32 / HEADS)][warp] = part;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (ok) {
        const bool whole = CLUSTER == 0 && i >= w.t && first;  // all of the pair's tiles are this CTA's
        // in a cluster over the first codes: all copies and products are done
        float* rec = CLUSTER > 0 ? reinterpret_cast<float*>(smem)
                             : a.part + ((int64_t)blockIdx.x * 2 + (pair > 0)) * record_floats(HEADS);
#pragma unroll
        for (int r = 0; r < HEADS; ++r) {
          const float4 l4 = *reinterpret_cast<const float4*>(s_sum[r]);
          const float sum = (l4.x + l4.y) + (l4.z + l4.w);
          const float o = O[r] * (1.f / kPScale);
          if (whole) {
            if (r < a.group)
              static_cast<__nv_bfloat16*>(a.out)[w.e * a.out_stride + (int64_t)(w.h * a.group + r) * kTcDim + tok] =
                  __float2bfloat16_rn(sum == 0.f ? 0.f : o * __frcp_rn(sum));
          } else {
            if (tok == 0) rec[r] = R[r], rec[HEADS + r] = sum;
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
  if constexpr (CLUSTER > 0) {
    // ---- the pair's outputs in equal parts, four threads per output, each with its part of the records
    constexpr int kOuts = HEADS * kTcDim / CLUSTER, kRecords = CLUSTER / 4;
    cluster_sync();
    const int rank = blockIdx.x % CLUSTER, part = threadIdx.x & 3;
#pragma unroll
    for (int it = 0; it < kOuts / (kThreads / 4); ++it) {
      const int i = rank * kOuts + it * (kThreads / 4) + (threadIdx.x >> 2), r = i / kTcDim, ch = i % kTcDim;
      float m[kRecords], l[kRecords], o[kRecords];
#pragma unroll
      for (int k = 0; k < kRecords; ++k) {
        m[k] = ld_cluster(base + r * 4, part * kRecords + k);
        l[k] = ld_cluster(base + (HEADS + r) * 4, part * kRecords + k);
        o[k] = ld_cluster(base + (2 * HEADS + r * kTcDim + ch) * 4, part * kRecords + k);
      }
      float mn = m[0];
#pragma unroll
      for (int k = 1; k < kRecords; ++k) mn = fmaxf(mn, m[k]);
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
      const float ref = mn == -INFINITY ? 0.f : mn;
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int k = 0; k < kRecords; ++k) {
        const float f = ex2(m[k] - ref);
        sum = fmaf(f, l[k], sum);
        if (m[k] != -INFINITY) x = fmaf(f, o[k], x);  // a CTA without tiles left no outputs
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        x += __shfl_xor_sync(0xffffffffu, x, d);
      }
      if (part == 0 && r < a.group)
        static_cast<__nv_bfloat16*>(a.out)[(int64_t)s_start[0] * a.out_stride + (int64_t)(s_start[1] * a.group + r) * kTcDim + ch] =
            __float2bfloat16_rn(sum == 0.f ? 0.f : x / sum);
    }
    cluster_sync();  // the records stay until all have read them
  }
}

// Joins the records of a pair whose tiles lay in several shares; an entry
// without keys gets zeros.  Lanes hold four channels.  SPLIT: a CTA per query
// head, its warps take the records in turn (few pairs, many records each);
// else a CTA per pair and a warp per query head (a pair has two or three
// records: 2048 CTAs of the other kind took 15 us where 256 of this take 7).
// A record's outputs are asked for together with the maxima, so the chain is
// one load long.
constexpr int join_warps(bool split) { return split ? 16 : 8; }
template <int HEADS, bool SPLIT>
__global__ void __launch_bounds__(32 * join_warps(SPLIT)) kv8_decode_join_kernel(const DecodeArgs g, int64_t ctas) {
  constexpr int kJoinWarps = SPLIT ? 16 : 8, kJoinThreads = 32 * kJoinWarps;
  constexpr int kJoinAhead = SPLIT ? 5 : 4;  // records in flight per warp (80 of a pair: its part of 148 x 2 CTAs)
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
  __shared__ __align__(16) float s_o[kJoinWarps][kTcDim];
  const AttnArgs& a = g.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int e = blockIdx.x, h = SPLIT ? blockIdx.y / a.group : blockIdx.y;
  wait_prior_grid();
  allow_next_grid();
  const int64_t total = g.before[a.bs] * a.c.kv_heads, T = g.before[e + 1] - g.before[e];
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + e * a.out_stride;
  if (T == 0) {
    out += (int64_t)(SPLIT ? blockIdx.y : h * a.group) * kTcDim;
    for (int i = threadIdx.x; i < (SPLIT ? 1 : a.group) * kTcDim; i += kJoinThreads) out[i] = __float2bfloat16_rn(0.f);
    return;
  }
  const Shares shares(total, ctas);
  const int64_t first = g.before[e] * a.c.kv_heads + h * T, last = first + T - 1;
  const int64_t c0 = shares.owner(first), c1 = shares.owner(last);
  if (c0 == c1) return;  // written by its CTA
  const int parts = (int)(c1 - c0 + 1);
  const int skip = first > shares.lo(c0) ? 1 : 0;  // the first CTA's record lies behind another pair's
  auto record = [&](int k) { return a.part + ((c0 + k) * 2 + (k == 0 ? skip : 0)) * record_floats(HEADS); };
  for (int r = SPLIT ? blockIdx.y - h * a.group : warp; r < a.group; r += kJoinWarps) {
    const int step = SPLIT ? kJoinWarps : 1;
    float M = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = SPLIT ? warp : 0; k0 < parts; k0 += step * kJoinAhead) {
      float m[kJoinAhead], s[kJoinAhead];
      float4 v[kJoinAhead];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        const float* p = record(min(k0 + k * step, parts - 1));
        m[k] = k0 + k * step < parts ? p[r] : -INFINITY;
        s[k] = p[HEADS + r];
        v[k] = *reinterpret_cast<const float4*>(p + 2 * HEADS + r * kTcDim + lane * 4);
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) mn = fmaxf(mn, m[k]);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float f0 = ex2(M - ref);
      l *= f0, o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        if (k0 + k * step >= parts) break;
        const float f = ex2(m[k] - ref);
        l = fmaf(f, s[k], l);
        o.x = fmaf(f, v[k].x, o.x), o.y = fmaf(f, v[k].y, o.y), o.z = fmaf(f, v[k].z, o.z), o.w = fmaf(f, v[k].w, o.w);
      }
      M = mn;
    }
    if (!SPLIT) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      *reinterpret_cast<uint2*>(out + (int64_t)(h * a.group + r) * kTcDim + lane * 4) =
          make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
      continue;
    }
    if (lane == 0) s_m[warp] = M, s_l[warp] = l;
    *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = o;
    __syncthreads();
    if (threadIdx.x < kTcDim) {
      float mn = -INFINITY;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) mn = fmaxf(mn, s_m[w]);
      const float ref = mn == -INFINITY ? 0.f : mn;
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float f = ex2(s_m[w] - ref);
        sum = fmaf(f, s_l[w], sum);
        x = fmaf(f, s_o[w][threadIdx.x], x);
      }
      out[(int64_t)blockIdx.y * kTcDim + threadIdx.x] = __float2bfloat16_rn(sum == 0.f ? 0.f : x / sum);
    }
    break;
  }
}

template <int KEYS, int HEADS>
constexpr int ring_slots() {
  return HEADS == 8 ? 6 : 10;  // two CTAs per SM of the 16-column kernel share its 228 KiB
}
template <int KEYS, int HEADS>
constexpr size_t decode_smem() {
  return 1024 + 4 * 2 * HEADS * 128 + ring_slots<KEYS, HEADS>() * kSlotBytes;
}

struct Maps {
  CUtensorMap mk, mv, rk, rv;
};
template <int KEYS>
int encode_maps(const Cache& c, Maps& m) {
  const int64_t rows = (int64_t)c.num_blocks * c.kv_heads * c.block;
  const int box = KEYS == kTable ? c.block : 16;
  int rc;
  if ((rc = encode_rows(&m.mk, c.k, rows, box)) != QQ_OK) return rc;
  if ((rc = encode_rows(&m.mv, c.v, rows, box)) != QQ_OK) return rc;
  if (KEYS == kRows) {
    if ((rc = encode_rows(&m.rk, c.k, rows, 1)) != QQ_OK) return rc;
    return encode_rows(&m.rv, c.v, rows, 1);
  }
  m.rk = m.mk, m.rv = m.mv;  // not read
  return QQ_OK;
}

template <int KEYS, int HEADS>
int launch(DecodeArgs g, int64_t ctas, cudaStream_t s) {
  static_assert(ring_slots<KEYS, HEADS>() >= 4 && ring_slots<KEYS, HEADS>() <= kMaxSlots, "ring");
  g.slots = ring_slots<KEYS, HEADS>();
  constexpr size_t smem = decode_smem<KEYS, HEADS>();
  static SmemLimit limit;
  int rc = limit.ensure((const void*)kv8_decode_kernel<KEYS, HEADS, 0>, smem);
  if (rc != QQ_OK) return rc;
  Maps m;
  if ((rc = encode_maps<KEYS>(g.a.c, m)) != QQ_OK) return rc;
  rc = launch_pdl(kv8_decode_kernel<KEYS, HEADS, 0>, dim3((unsigned)ctas), dim3(kThreads), smem, s, g, m.mk, m.mv, m.rk,
                  m.rv);
  if (rc != QQ_OK) return rc;
  const int pairs = g.a.bs * g.a.c.kv_heads;
  if (ctas >= 4 * (int64_t)pairs)
    return launch_pdl(kv8_decode_join_kernel<HEADS, true>, dim3(g.a.bs, g.a.heads), dim3(32 * join_warps(true)), 0, s, g,
                      ctas);
  return launch_pdl(kv8_decode_join_kernel<HEADS, false>, dim3(g.a.bs, g.a.c.kv_heads), dim3(32 * join_warps(false)), 0, s,
                    g, ctas);
}

template <int KEYS, int HEADS, int CLUSTER>
int resident_clusters() {
  static ResidentClusters known;
  constexpr size_t smem = decode_smem<KEYS, HEADS>();
  return known.ask((const void*)kv8_decode_kernel<KEYS, HEADS, CLUSTER>, dim3(CLUSTER), kThreads, smem, smem);
}

template <int KEYS, int HEADS, int CLUSTER>
int launch_clusters(DecodeArgs g, cudaStream_t s) {
  g.slots = ring_slots<KEYS, HEADS>();
  Maps m;
  const int rc = encode_maps<KEYS>(g.a.c, m);
  if (rc != QQ_OK) return rc;
  ClusterLaunch l(dim3(g.a.bs * g.a.c.kv_heads * CLUSTER), dim3(CLUSTER), kThreads, decode_smem<KEYS, HEADS>(), s);
  return cudaLaunchKernelEx(&l.cfg, kv8_decode_kernel<KEYS, HEADS, CLUSTER>, g, m.mk, m.mv, m.rk, m.rv) == cudaSuccess
             ? QQ_OK
             : QQ_ERR_CUDA;
}

// The cluster a call goes by, 0: shares and a join.  All clusters run at a
// time, and no CTA has more than kClusterTiles tiles.  On the device (group 8,
// 4 KV heads) 1 x 2,048 keys take 7.7 us where shares and a join take 9.4, 1 x
// 8,192 10.6 and 11.9, 3 x 2,048 9.1 and 11.0, 8 x 2,048 12.2 and 12.9; with
// eight tiles to a CTA 2 x 8,192 would take 13.8 and 13.3.
template <int CLUSTER>
bool cluster_fits(int64_t pairs, int group, int64_t max_keys) {
  if (max_keys > (int64_t)CLUSTER * kClusterTiles * kTile) return false;
  return pairs <= (group <= 8 ? std::min(resident_clusters<kTable, 8, CLUSTER>(), resident_clusters<kRows, 8, CLUSTER>())
                              : std::min(resident_clusters<kTable, 16, CLUSTER>(), resident_clusters<kRows, 16, CLUSTER>()));
}
int cluster_of(int bs, int kv_heads, int group, int64_t max_keys) {
  const int64_t pairs = (int64_t)bs * kv_heads;
  if (pairs > device_sm_count()) return 0;
  return cluster_fits<16>(pairs, group, max_keys)  ? 16
         : cluster_fits<8>(pairs, group, max_keys) ? 8
         : cluster_fits<4>(pairs, group, max_keys) ? 4
                                                   : 0;
}
template <int CLUSTER>
int run_clusters(const DecodeArgs& g, int keys, cudaStream_t s) {
  if (g.a.group <= 8) return keys == kTable ? launch_clusters<kTable, 8, CLUSTER>(g, s) : launch_clusters<kRows, 8, CLUSTER>(g, s);
  return keys == kTable ? launch_clusters<kTable, 16, CLUSTER>(g, s) : launch_clusters<kRows, 16, CLUSTER>(g, s);
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
  if (cluster_of(bs, kv_heads, group, max_keys) > 0) return 0;
  return sizeof(float) * (size_t)(decode_ctas(bs, kv_heads, group, max_keys) * 2 * record_floats(group <= 8 ? 8 : 16)) +
         sizeof(int64_t) * (size_t)(bs + 1);
}

int run_decode_tc(const AttnArgs& a, int keys, int64_t max_keys, size_t ws_bytes, cudaStream_t s) {
  // a share's place among the tiles of its entry's heads is held in 32 bits
  if ((max_keys + kTile - 1) / kTile * a.c.kv_heads > INT32_MAX) return QQ_ERR_UNSUPPORTED;
  DecodeArgs g{};
  g.a = a;
  const int cluster = cluster_of(a.bs, a.c.kv_heads, a.group, max_keys);
  if (cluster > 0) return cluster == 16 ? run_clusters<16>(g, keys, s) : cluster == 8 ? run_clusters<8>(g, keys, s) : run_clusters<4>(g, keys, s);
  if (a.part == nullptr || ws_bytes < decode_tc_workspace(a.bs, a.c.kv_heads, a.group, max_keys)) return QQ_ERR_WORKSPACE;
  const int64_t ctas = decode_ctas(a.bs, a.c.kv_heads, a.group, max_keys);
  g.before = reinterpret_cast<int64_t*>(a.part + ctas * 2 * record_floats(a.group <= 8 ? 8 : 16));
  if (a.group <= 8) return keys == kTable ? launch<kTable, 8>(g, ctas, s) : launch<kRows, 8>(g, ctas, s);
  return keys == kTable ? launch<kTable, 16>(g, ctas, s) : launch<kRows, 16>(g, ctas, s);
}

}  // namespace kv8
}  // namespace qq

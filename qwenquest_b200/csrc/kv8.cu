// The 8-bit block KV cache: its tables and slots, made on the GPU from request
// lengths, and the quantising write with its read-back.
//
// Tables.  Request r holds held[r] blocks, block_table[r][0 .. held[r]); free
// blocks wait in a ring (taken at its head, given back at its tail), so which
// block a request gets depends on the order of calls alone.  A step's batch
// grows requests (qq_block_plan) or shrinks them (qq_block_trim) without a
// host round trip, so both can be captured in a graph.
//
// Quantisation.  Per block and KV head a power of two s = 2^k, k the smallest
// with amax <= 448 * 2^k over the finite values written; a value is stored as
// e4m3(x / s), to nearest even.  A power of two costs no accuracy in a
// floating-point code (the significand is kept; values below 2^-6 s lose bits,
// at most one binade earlier than with amax / 448) and makes growth exact:
// when a later token needs a larger scale, the codes the block holds are
// multiplied by s_old / s_new, which changes their exponents only and rounds
// none but those that fall below 2^-6 of the new scale.

#include <climits>

#include <cuda_fp16.h>

#include "kv8.cuh"

namespace qq {
namespace {

using namespace kv8;

// ------------------------------------------------------------------ tables

struct TableArgs {
  int32_t* table;
  int64_t stride;
  int32_t* held;
  int32_t* claim;
  int32_t* free_blocks;
  int64_t* ring;
  int capacity, max_reqs, max_blocks, shift;
  const int64_t* reqs;
  const int64_t* seq;     // plan: lengths with the new tokens; trim: tokens to keep (null: none)
  const int64_t* prefix;  // plan: lengths before them
  int bs;
  int64_t* slots;
  int64_t num_slots;
  int64_t* offsets;
  int32_t* map;
  int64_t map_stride, map_rows;
  uint32_t* err;
};

constexpr int kTableThreads = 1024;
constexpr int kTablePer = QQ_MAX_BS / kTableThreads;  // batch entries per thread at most

// Shared arrays of bs entries each (plus one for the two prefix sums).
struct TableSmem {
  int64_t* off;   // [bs + 1] new tokens before entry i
  int32_t* sum;   // [bs + 1] blocks moved before entry i
  int32_t* req;   // -1: nothing to do for this entry
  int32_t* held;
  int64_t* pre;
};
__host__ __device__ inline size_t table_smem_bytes(int bs) { return (size_t)(bs + 1) * 12 + (size_t)bs * 16 + 16; }
__device__ inline TableSmem table_smem(void* p, int bs) {
  TableSmem s;
  s.off = static_cast<int64_t*>(p);
  s.pre = s.off + bs + 1;
  s.sum = reinterpret_cast<int32_t*>(s.pre + bs);
  s.req = s.sum + bs + 1;
  s.held = s.req + bs;
  return s;
}

// Counts of blocks, which stop at INT_MAX: 4,096 entries may ask for more than 2^31 between them.
__device__ __forceinline__ int32_t add_counts(int32_t x, int32_t y) {
  return (int32_t)min((uint32_t)x + (uint32_t)y, (uint32_t)INT_MAX);
}

// Exclusive sums over the block of one (int64, count of blocks) pair per thread; totals to all threads.
__device__ void block_scan(int64_t& a, int32_t& b, int64_t& a_total, int32_t& b_total) {
  __shared__ int64_t sa[32];
  __shared__ int32_t sb[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t ia = a;
  int32_t ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ua = __shfl_up_sync(0xffffffffu, ia, o);
    const int32_t ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) ia += ua, ib = add_counts(ib, ub);
  }
  if (lane == 31) sa[warp] = ia, sb[warp] = ib;
  const int32_t before = __shfl_up_sync(0xffffffffu, ib, 1);
  __syncthreads();
  if (warp == 0) {
    int64_t wa = sa[lane];
    int32_t wb = sb[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t ua = __shfl_up_sync(0xffffffffu, wa, o);
      const int32_t ub = __shfl_up_sync(0xffffffffu, wb, o);
      if (lane >= o) wa += ua, wb = add_counts(wb, ub);
    }
    sa[lane] = wa, sb[lane] = wb;
  }
  __syncthreads();
  a_total = sa[31], b_total = sb[31];
  a = ia - a + (warp ? sa[warp - 1] : 0);
  b = add_counts(lane ? before : 0, warp ? sb[warp - 1] : 0);
}

// The last i in [0, n) with sums[i] <= x (sums ascending, sums[0] <= x).
template <typename V>
__device__ __forceinline__ int last_at_most(const V* sums, int n, V x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A request that the batch names twice is served for its first entry only: the
// claim word of a request takes the largest bs - i (0 between launches).  An
// entry whose `lens` is 0 is padding and claims nothing (null: none is).
__device__ __forceinline__ void claim_requests(const TableArgs& a, const int64_t* lens) {
  for (int i = threadIdx.x; i < a.bs; i += kTableThreads) {
    const int64_t r = a.reqs[i];
    if (r >= 0 && r < a.max_reqs && (lens == nullptr || lens[i] != 0)) atomicMax(a.claim + r, a.bs - i);
  }
  __syncthreads();
}
__device__ __forceinline__ void release_claims(const TableArgs& a) {
  for (int i = threadIdx.x; i < a.bs; i += kTableThreads) {
    const int64_t r = a.reqs[i];
    if (r >= 0 && r < a.max_reqs) a.claim[r] = 0;
  }
}

// Latency-bound: a step's batch is a few thousand integers.  kState: this CTA
// updates the tables (one CTA); kSlots: the grid writes the slots.  Every CTA
// reads the lengths and sums them itself, so the slots need no second pass
// over the tables: a page the request does not hold yet is found in the ring.
template <bool kState, bool kSlots>
__global__ void __launch_bounds__(kTableThreads) block_plan_kernel(TableArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ int s_taken;
  const TableSmem s = table_smem(smem_raw, a.bs);
  const int tid = threadIdx.x;
  const int block = 1 << a.shift;
  if (tid == 0) s_taken = 0;
  wait_prior_grid();
  allow_next_grid();
  claim_requests(a, a.seq);
  const int64_t head = a.ring[0], free_count = min(a.ring[1] - head, (int64_t)INT_MAX - 1);

  // ---- this thread's entries: new tokens and blocks to take
  int64_t toks[kTablePer], my_toks = 0;
  int32_t need[kTablePer], my_need = 0;
  const int per = (a.bs + kTableThreads - 1) / kTableThreads;
#pragma unroll
  for (int j = 0; j < kTablePer; ++j) {
    const int i = tid * per + j;
    toks[j] = 0, need[j] = 0;
    if (j >= per || i >= a.bs) continue;
    const int64_t r = a.reqs[i], seq = a.seq[i], pre = a.prefix[i];
    int32_t req = -1, held = 0;
    if (seq != 0) {  // 0: a padding entry
      bool good = pre >= 0 && seq >= pre;
      if (good) toks[j] = seq - pre;
      good = good && r >= 0 && r < a.max_reqs && seq <= ((int64_t)a.max_blocks << a.shift);
      if (good) good = ld_volatile_s32(a.claim + r) == a.bs - i;
      if (good) {
        req = (int32_t)r;
        held = a.held[r];
        good = held >= 0 && held <= a.max_blocks;
      }
      if (good) need[j] = max(0, (int32_t)((seq + block - 1) >> a.shift) - held);
      else req = -1;
      if (!good) raise_error(a.err, QQ_DEV_ERR_BOUNDS);
    }
    s.req[i] = req;
    s.held[i] = held;
    s.pre[i] = pre;
    my_toks += toks[j];
    my_need = add_counts(my_need, need[j]);
  }
  int64_t tok_at = my_toks, tok_total;
  int32_t need_at = my_need, need_total;
  block_scan(tok_at, need_at, tok_total, need_total);
#pragma unroll
  for (int j = 0; j < kTablePer; ++j) {
    const int i = tid * per + j;
    if (j >= per || i >= a.bs) continue;
    s.off[i] = tok_at;
    s.sum[i] = need_at;
    tok_at += toks[j];
    need_at = add_counts(need_at, need[j]);
    if (need[j] > 0) {
      if (need_at <= free_count) {
        atomicMax(&s_taken, need_at);
      } else {  // the ring runs out: this request stays as it was
        s.req[i] = -1;
        raise_error(a.err, QQ_DEV_ERR_CAPACITY);
      }
    }
  }
  if (tid == 0) {
    s.off[a.bs] = tok_total;
    s.sum[a.bs] = need_total;
    if (tok_total > a.num_slots) raise_error(a.err, QQ_DEV_ERR_BOUNDS);
  }
  __syncthreads();

  if (kSlots) {
    if (blockIdx.x == 0)
      for (int i = tid; i <= a.bs; i += kTableThreads) a.offsets[i] = s.off[i];
    for (int64_t t = (int64_t)blockIdx.x * kTableThreads + tid; t < a.num_slots; t += (int64_t)gridDim.x * kTableThreads) {
      int64_t slot = -1;
      if (t < tok_total) {
        const int e = last_at_most(s.off, a.bs, t);
        const int32_t req = s.req[e];
        if (req >= 0) {
          const int64_t pos = s.pre[e] + t - s.off[e];
          const int32_t page = (int32_t)(pos >> a.shift);
          const int32_t b = page < s.held[e]
                                ? a.table[req * a.stride + page]
                                : a.free_blocks[(head + s.sum[e] + page - s.held[e]) % a.capacity];
          if (b >= 0) {
            slot = ((int64_t)b << a.shift) | (pos & (block - 1));
            if (a.map != nullptr) {
              if (req < a.map_rows && pos < a.map_stride && slot <= INT_MAX) a.map[req * a.map_stride + pos] = (int32_t)slot;
              else raise_error(a.err, QQ_DEV_ERR_BOUNDS);
            }
          } else {
            raise_error(a.err, QQ_DEV_ERR_BOUNDS);
          }
        }
      }
      a.slots[t] = slot;
    }
  }
  if (kState) {
    __syncthreads();  // the slots above read the tables as they were
    for (int o = tid; o < s_taken; o += kTableThreads) {
      const int e = last_at_most(s.sum, a.bs, o);
      a.table[s.req[e] * a.stride + s.held[e] + o - s.sum[e]] = a.free_blocks[(head + o) % a.capacity];
    }
    for (int i = tid; i < a.bs; i += kTableThreads) {
      if (s.req[i] >= 0) a.held[s.req[i]] = s.held[i] + s.sum[i + 1] - s.sum[i];
    }
    release_claims(a);
    if (tid == 0) a.ring[0] = head + s_taken;
  }
}

__global__ void __launch_bounds__(kTableThreads) block_trim_kernel(TableArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const TableSmem s = table_smem(smem_raw, a.bs);
  const int tid = threadIdx.x;
  const int block = 1 << a.shift;
  wait_prior_grid();
  allow_next_grid();
  claim_requests(a, nullptr);
  const int64_t tail = a.ring[1], room = min(a.capacity - (tail - a.ring[0]), (int64_t)INT_MAX - 1);
  int32_t back[kTablePer], my_back = 0;
  const int per = (a.bs + kTableThreads - 1) / kTableThreads;
#pragma unroll
  for (int j = 0; j < kTablePer; ++j) {
    const int i = tid * per + j;
    back[j] = 0;
    if (j >= per || i >= a.bs) continue;
    const int64_t r = a.reqs[i], keep = a.seq == nullptr ? 0 : a.seq[i];
    int32_t req = -1, held = 0;
    if (r != -1) {  // -1: a padding entry
      bool good = r >= 0 && r < a.max_reqs && keep >= 0;
      if (good) good = ld_volatile_s32(a.claim + r) == a.bs - i;
      if (good) {
        req = (int32_t)r;
        held = a.held[r];
        good = held >= 0 && held <= a.max_blocks;
      }
      if (good && keep < ((int64_t)held << a.shift)) back[j] = held - (int32_t)((keep + block - 1) >> a.shift);
      if (!good) req = -1, raise_error(a.err, QQ_DEV_ERR_BOUNDS);
    }
    s.req[i] = req;
    s.held[i] = held;
    my_back = add_counts(my_back, back[j]);
  }
  int64_t none = 0, none_total;
  int32_t at = my_back, total;
  block_scan(none, at, none_total, total);
#pragma unroll
  for (int j = 0; j < kTablePer; ++j) {
    const int i = tid * per + j;
    if (j >= per || i >= a.bs) continue;
    s.sum[i] = at;
    at = add_counts(at, back[j]);
  }
  if (tid == 0) s.sum[a.bs] = total;
  __syncthreads();
  if (total > room) {  // more blocks than the ring was made for: a table that names blocks it does not own
    if (tid == 0) raise_error(a.err, QQ_DEV_ERR_BOUNDS);
  } else {
    for (int o = tid; o < total; o += kTableThreads) {
      const int e = last_at_most(s.sum, a.bs, o);
      // entry e gives back pages [held - back, held), ascending
      const int32_t page = s.held[e] - (s.sum[e + 1] - s.sum[e]) + o - s.sum[e];
      int32_t* p = a.table + s.req[e] * a.stride + page;
      a.free_blocks[(tail + o) % a.capacity] = *p;
      *p = -1;
    }
    for (int i = tid; i < a.bs; i += kTableThreads)
      if (s.req[i] >= 0) a.held[s.req[i]] = s.held[i] - (s.sum[i + 1] - s.sum[i]);
    if (tid == 0) a.ring[1] = tail + total;
  }
  release_claims(a);
}

// ------------------------------------------------------------------ append

struct AppendArgs {
  Cache c;
  const void* k;
  const void* v;
  int64_t k_stride, v_stride;  // elements between tokens
  const int64_t* slots;
  int64_t n;
  int window;  // tokens whose runs a CTA takes
  bool claimed;  // kv8_claim_kernel has run
  uint32_t* err;
};

constexpr int kMaxWindow = 64;
constexpr int kAppendThreads = 128;
// `state`: 64 bits whose upper half counts the calls, then a claim word per
// block, K or V and head, 0 between calls.
constexpr int kClaims = QQ_KV8_STATE_WORDS;
// Up to this many tokens a window is one token and a run looks for its block
// among the tokens before it; a call with more claims the blocks in a launch of
// its own (64 tokens: 3.3 us by looking, 5.6 by claims; 256: 7.5 and 9.0; 512:
// 12.6 and 13.4).
constexpr int64_t kLookTokens = 512;

__device__ __forceinline__ bool run_head(const Cache& c, int64_t slot, int64_t before) {
  return slot >= 0 && ((slot & (c.block - 1)) == 0 || before != slot - 1);
}

// The claims of a call: a block's word takes n - t for the first token t of a
// run in it, the largest of them (so the first run has it).
constexpr int kClaimThreads = 128;
__global__ void __launch_bounds__(kClaimThreads) kv8_claim_kernel(Cache c, const int64_t* slots, int64_t n) {
  wait_prior_grid();
  allow_next_grid();
  const int64_t t = (int64_t)blockIdx.x * kClaimThreads + threadIdx.x, total = (int64_t)c.num_blocks << c.shift;
  if (t >= n) return;
  const int64_t slot = slots[t];
  if (slot >= total || !run_head(c, slot, t > 0 ? slots[t - 1] : -1)) return;
  uint32_t* claims = c.state + kClaims + (slot >> c.shift) * 2 * c.kv_heads;
  for (int i = 0; i < 2 * c.kv_heads; ++i) atomicMax(claims + i, (uint32_t)(n - t));
}

// A run is a stretch of tokens whose slots ascend by one inside a block; the
// CTAs of its first token quantise it, one per K or V and head (blockIdx.y).
// A lane holds up to kHeld pieces of 8 elements in registers between the pass
// for the maximum and the one that stores the codes: a block of 64 x 128 bf16
// is read once, and all of it at once (longer runs are read again, from L2).
// Bound by the values' bytes for a prefill and by the chain slots -> values ->
// maximum -> codes for a decode step.
// Two runs of one call that meet in a block would race: the first one is
// written, the others are skipped and reported.  Which is the first is found
// from the call's own slots, so calls of other streams, which write other
// blocks, and captured calls have no part in it: either by looking at the tokens
// before the run, or from the block's claim, which the run that made it takes
// back (no other run of the call finds its own number there, before or after).
template <typename T, int DIM>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 2 ? 8 : 4) kv8_append_kernel(AppendArgs a) {
  constexpr int kHeld = 8;
  constexpr int kWords = sizeof(T) == 2 ? 1 : 2;  // 16-byte loads per piece
  __shared__ int64_t s_slots[kMaxWindow + kMaxBlock + 1];
  __shared__ uint32_t s_heads[kMaxWindow / 32];
  __shared__ float s_most[2][kAppendThreads / 32];
  const Cache& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int dim = DIM > 0 ? DIM : c.dim;
  const int chunks = dim >> 3;  // 8-element pieces of a row
  const bool is_v = blockIdx.y >= c.kv_heads;
  const int h = is_v ? blockIdx.y - c.kv_heads : blockIdx.y;
  const int64_t stride = is_v ? a.v_stride : a.k_stride;
  const int64_t w0 = (int64_t)blockIdx.x * a.window;
  const int64_t total = (int64_t)c.num_blocks << c.shift;
  wait_prior_grid();
  allow_next_grid();
  // s_slots[i] is the slot of token w0 - 1 + i (-1 outside the batch)
  for (int i = tid; i < a.window + c.block + 1; i += kAppendThreads) {
    const int64_t t = w0 - 1 + i;
    s_slots[i] = t >= 0 && t < a.n ? a.slots[t] : -1;
  }
  __syncthreads();
  // the window's run heads, one bit each
  if (tid < kMaxWindow) {
    bool head = false;
    if (tid < a.window && w0 + tid < a.n) {
      const int64_t slot = s_slots[tid + 1];
      head = run_head(c, slot, s_slots[tid]);
      if (slot >= total || slot < -1) {
        raise_error(a.err, QQ_DEV_ERR_BOUNDS);
        head = false;
      }
    }
    const uint32_t m = __ballot_sync(0xffffffffu, head);
    if (lane == 0) s_heads[warp] = m;
  }
  __syncthreads();
  uint64_t heads = s_heads[0] | (uint64_t)s_heads[1] << 32;
  for (int turn = 0; heads != 0; heads &= heads - 1, turn ^= 1) {
    const int u = __ffsll(heads) - 1;
    const int64_t slot = s_slots[u + 1];
    const int off = (int)(slot & (c.block - 1));
    const int32_t b = (int32_t)(slot >> c.shift);
    int n = 0;  // the run's tokens
    for (int base = 0; base < c.block; base += 32) {
      const int i = base + lane;
      const bool in = off + i < c.block && s_slots[u + 1 + i] == slot + i;
      const uint32_t m = __ballot_sync(0xffffffffu, in);
      if (m != 0xffffffffu) {
        n = base + __ffs(~m) - 1;
        break;
      }
      n = base + 32;
    }
    // whether the block has an earlier run
    auto look = [&]() {
      bool met = false;
      if (!a.claimed) {
        for (int64_t i = tid; i < w0 + u; i += kAppendThreads) {
          const int64_t other = a.slots[i];
          met |= other >= 0 && other >> c.shift == b;
        }
      } else if (tid == 0) {
        uint32_t* claim = c.state + kClaims + (int64_t)b * 2 * c.kv_heads + blockIdx.y;
        met = ld_volatile_u32(claim) != (uint32_t)(a.n - (w0 + u));
        if (!met) *claim = 0;
      }
      return met;
    };
    bool met;
    const T* src = static_cast<const T*>(is_v ? a.v : a.k) + (w0 + u) * stride + (int64_t)h * dim;
    const int64_t bh = (int64_t)b * c.kv_heads + h;
    uint8_t* codes = (is_v ? c.v : c.k) + bh * c.block * dim;
    float* scale = (is_v ? c.v_scale : c.k_scale) + bh;
    const int items = n * chunks;
    const bool held = items <= kAppendThreads * kHeld;
    auto piece = [&](int i) {
      const int r = i / chunks;
      return reinterpret_cast<const uint4*>(src + r * stride + (i - r * chunks) * 8);
    };
    auto unpack = [&](const uint4* w, float (&x)[8]) {
      const uint32_t lo[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
      if (kWords == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[2 * e] = __uint_as_float(lo[e] << 16), x[2 * e + 1] = __uint_as_float(lo[e] & 0xFFFF0000u);
      } else {
        const uint4& v = w[kWords - 1];
        const uint32_t hi[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(lo[e]), x[4 + e] = __uint_as_float(hi[e]);
      }
    };
    float most = 0.f;
    auto raise_most = [&](const float (&x)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float m = fabsf(x[e]);
        if (m <= 3.402823466e38f) most = fmaxf(most, m);  // infinities and NaN set no scale
      }
    };
    const float old = off == 0 ? 0.f : *scale;
    uint4 raw[kHeld * kWords];
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int i = tid + k * kAppendThreads;
#pragma unroll
        for (int w = 0; w < kWords; ++w) raw[k * kWords + w] = i < items ? __ldg(piece(i) + w) : make_uint4(0, 0, 0, 0);
      }
      met = look();  // while the values are on their way
      // magnitudes compare as integers; only a run with an infinity or a NaN is looked at element by element
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < kHeld * kWords; ++k) {
        if (sizeof(T) == 2) {
          top = __vmaxu2(top, __vmaxu2(raw[k].x & 0x7FFF7FFFu, raw[k].y & 0x7FFF7FFFu));
          top = __vmaxu2(top, __vmaxu2(raw[k].z & 0x7FFF7FFFu, raw[k].w & 0x7FFF7FFFu));
        } else {
          top = max(top, max(raw[k].x & 0x7FFFFFFFu, raw[k].y & 0x7FFFFFFFu));
          top = max(top, max(raw[k].z & 0x7FFFFFFFu, raw[k].w & 0x7FFFFFFFu));
        }
      }
      most = __uint_as_float(sizeof(T) == 2 ? max(top & 0xFFFF0000u, top << 16) : top);
      if (!(most <= 3.402823466e38f)) {
        most = 0.f;
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
          float x[8];
          unpack(raw + k * kWords, x);
          raise_most(x);
        }
      }
    } else {
      met = look();
#pragma unroll 2
      for (int i = tid; i < items; i += kAppendThreads) {
        float x[8];
        load8(reinterpret_cast<const T*>(piece(i)), x);
        raise_most(x);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) s_most[turn][warp] = most;
    if (__syncthreads_or(met)) {  // also: all have read the old scale
      if (tid == 0) raise_error(a.err, QQ_DEV_ERR_BOUNDS);
      continue;
    }
    most = fmaxf(fmaxf(s_most[turn][0], s_most[turn][1]), fmaxf(s_most[turn][2], s_most[turn][3]));
    // most = 1.m * 2^E <= 1.75 * 2^8 * 2^k
    const uint32_t bits = __float_as_uint(most);
    const int e2 = max((int)(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7), -126);
    const float now = fmaxf(old, __uint_as_float((uint32_t)(e2 + 127) << 23));
    if (off != 0 && now != old) {  // the codes already here, in steps of the larger scale
      const float ratio = __fdiv_rn(old, now);
      for (int i = tid; i < c.block * chunks; i += kAppendThreads) {
        const int r = i / chunks;
        if (r >= off && r < off + n) continue;
        uint2* p8 = reinterpret_cast<uint2*>(codes + (int64_t)i * 8);
        float x[8];
        from_e4m3x8(*p8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= ratio;
        *p8 = make_uint2(e4m3x2(x[0], x[1]) | (e4m3x2(x[2], x[3]) << 16),
                         e4m3x2(x[4], x[5]) | (e4m3x2(x[6], x[7]) << 16));
      }
    }
    // dividing by a power of two is multiplying by its inverse; a scale the caller brought may be any number
    const uint32_t nb = __float_as_uint(now);
    const bool pow2 = (nb & 0x7FFFFFu) == 0 && nb != 0;
    const float inv = __fdiv_rn(1.f, now);
    uint8_t* dst = codes + (int64_t)off * dim;
    auto put = [&](int i, const float (&x)[8]) {
      *reinterpret_cast<uint2*>(dst + (int64_t)i * 8) = make_uint2(
          e4m3x2(x[0], x[1]) | (e4m3x2(x[2], x[3]) << 16), e4m3x2(x[4], x[5]) | (e4m3x2(x[6], x[7]) << 16));
    };
    if (held && pow2) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int i = tid + k * kAppendThreads;
        if (i >= items) break;
        float x[8];
        unpack(raw + k * kWords, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inv;
        put(i, x);
      }
    } else {
#pragma unroll 1
      for (int i = tid; i < items; i += kAppendThreads) {
        float x[8];
        load8(reinterpret_cast<const T*>(piece(i)), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = pow2 ? x[e] * inv : __fdiv_rn(x[e], now);
        put(i, x);
      }
    }
    if (tid == 0) *scale = now;
  }
  if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicAdd(c.state + 1, 1u);
}

// ------------------------------------------------------------------ gather

// out[i] = the values of slot slots[i] (code times scale): a warp per token, so
// the slot's place is found once for its row of K and of V, 8 elements of each
// per lane and step.  Bound by the bytes (22.8K tokens of 4 x 128: 12.5 us
// cold; a thread per piece took 17.3, three quarters of the issue slots for its
// divisions).  A slot of -1 gives zeros.
constexpr int kGatherWarps = 4;
template <typename T, int DIM>
__global__ void __launch_bounds__(32 * kGatherWarps) kv8_gather_kernel(Cache c, const int64_t* slots, int64_t n, T* k_out,
                                                                       T* v_out, uint32_t* err) {
  wait_prior_grid();
  allow_next_grid();
  const int dim = DIM > 0 ? DIM : c.dim, lane = threadIdx.x & 31;
  const int chunks = dim >> 3, row = c.kv_heads * chunks;
  const int64_t total = (int64_t)c.num_blocks << c.shift;
  for (int64_t t = (int64_t)blockIdx.x * kGatherWarps + (threadIdx.x >> 5); t < n; t += (int64_t)gridDim.x * kGatherWarps) {
    const int64_t slot = slots[t];
    const bool in = slot >= 0 && slot < total;
    if (!in && slot != -1 && lane == 0) raise_error(err, QQ_DEV_ERR_BOUNDS);
    const int64_t bh0 = in ? (slot >> c.shift) * c.kv_heads : 0;
    const int64_t at0 = (bh0 * c.block + (slot & (c.block - 1))) * dim;
#pragma unroll 1
    for (int w = lane; w < row; w += 32) {
      float kx[8] = {}, vx[8] = {};
      if (in) {
        const int h = w / chunks;
        const int64_t at = at0 + ((int64_t)h * c.block * chunks + (w - h * chunks)) * 8;
        const uint2 kc = *reinterpret_cast<const uint2*>(c.k + at), vc = *reinterpret_cast<const uint2*>(c.v + at);
        const float ks = c.k_scale[bh0 + h], vs = c.v_scale[bh0 + h];
        from_e4m3x8(kc, kx);
        from_e4m3x8(vc, vx);
#pragma unroll
        for (int e = 0; e < 8; ++e) kx[e] *= ks, vx[e] *= vs;
      }
      store8(k_out + (t * row + w) * 8, kx);
      store8(v_out + (t * row + w) * 8, vx);
    }
  }
}

template <typename T>
int launch_gather(const Cache& c, const int64_t* slots, int64_t n, void* k_out, void* v_out, uint32_t* err,
                  cudaStream_t s) {
  const int64_t most = (int64_t)device_sm_count() * 32, ctas = (n + kGatherWarps - 1) / kGatherWarps;
  const dim3 grid((unsigned)(ctas < most ? ctas : most)), block(32 * kGatherWarps);
  T *k = static_cast<T*>(k_out), *v = static_cast<T*>(v_out);
  return c.dim == 128 ? launch_pdl(kv8_gather_kernel<T, 128>, grid, block, 0, s, c, slots, n, k, v, err)
                      : launch_pdl(kv8_gather_kernel<T, 0>, grid, block, 0, s, c, slots, n, k, v, err);
}

int check_tables(const qq_block_tables* t, int bs, const int64_t* reqs) {
  if (t == nullptr || t->block_table == nullptr || t->held == nullptr || t->claim == nullptr ||
      t->free_blocks == nullptr || t->ring == nullptr || t->capacity <= 0 || t->max_reqs <= 0 || t->max_blocks <= 0 ||
      t->table_stride < t->max_blocks || bs < 0 || (bs > 0 && reqs == nullptr))
    return QQ_ERR_INVALID;
  if (bs > QQ_MAX_BS ||
      (t->block_size != 16 && t->block_size != 32 && t->block_size != 64 && t->block_size != 128))
    return QQ_ERR_UNSUPPORTED;
  return QQ_OK;
}

TableArgs table_args(const qq_block_tables& t, const int64_t* reqs, int bs, uint32_t* err) {
  TableArgs a{};
  a.table = t.block_table;
  a.stride = t.table_stride;
  a.held = t.held;
  a.claim = t.claim;
  a.free_blocks = t.free_blocks;
  a.ring = t.ring;
  a.capacity = t.capacity;
  a.max_reqs = t.max_reqs;
  a.max_blocks = t.max_blocks;
  while ((1 << a.shift) < t.block_size) ++a.shift;
  a.reqs = reqs;
  a.bs = bs;
  a.err = err;
  return a;
}

// Up to this many slots one CTA makes the whole plan; past it the slots take a grid of their own.
constexpr int64_t kOneCtaSlots = 4096;

}  // namespace
}  // namespace qq

extern "C" int qq_block_plan(const qq_block_tables* tables, const int64_t* req_pool_indices, const int64_t* seq_lens,
                             const int64_t* prefix_lens, int bs, int64_t* slots, int64_t num_slots,
                             int64_t* token_offsets, int32_t* req_to_token, int64_t map_stride, int64_t map_rows,
                             uint32_t* err, void* stream) {
  using namespace qq;
  int rc = check_tables(tables, bs, req_pool_indices);
  if (rc != QQ_OK) return rc;
  if (token_offsets == nullptr || num_slots < 0 || (num_slots > 0 && slots == nullptr) ||
      (bs > 0 && (seq_lens == nullptr || prefix_lens == nullptr)) ||
      (req_to_token != nullptr && (map_stride <= 0 || map_rows <= 0)))
    return QQ_ERR_INVALID;
  TableArgs a = table_args(*tables, req_pool_indices, bs, err);
  a.seq = seq_lens;
  a.prefix = prefix_lens;
  a.slots = slots;
  a.num_slots = num_slots;
  a.offsets = token_offsets;
  a.map = req_to_token;
  a.map_stride = map_stride;
  a.map_rows = map_rows;
  static SmemLimit one, wide, state;
  const size_t smem = table_smem_bytes(bs);
  cudaStream_t s = as_stream(stream);
  if (num_slots <= kOneCtaSlots) {
    if ((rc = one.ensure((const void*)block_plan_kernel<true, true>, smem + kStaticSmem)) != QQ_OK) return rc;
    return launch_pdl(block_plan_kernel<true, true>, dim3(1), dim3(kTableThreads), smem, s, a);
  }
  if ((rc = wide.ensure((const void*)block_plan_kernel<false, true>, smem + kStaticSmem)) != QQ_OK) return rc;
  if ((rc = state.ensure((const void*)block_plan_kernel<true, false>, smem + kStaticSmem)) != QQ_OK) return rc;
  const int64_t ctas = (num_slots + kTableThreads - 1) / kTableThreads;
  const int most = device_sm_count();
  rc = launch_pdl(block_plan_kernel<false, true>, dim3((unsigned)(ctas < most ? ctas : most)), dim3(kTableThreads), smem, s, a);
  if (rc != QQ_OK) return rc;
  a.err = nullptr;  // what is wrong has been reported
  return launch_pdl(block_plan_kernel<true, false>, dim3(1), dim3(kTableThreads), smem, s, a);
}

extern "C" int qq_block_trim(const qq_block_tables* tables, const int64_t* req_pool_indices, const int64_t* keep_lens,
                             int bs, uint32_t* err, void* stream) {
  using namespace qq;
  int rc = check_tables(tables, bs, req_pool_indices);
  if (rc != QQ_OK || bs == 0) return rc;
  TableArgs a = table_args(*tables, req_pool_indices, bs, err);
  a.seq = keep_lens;
  static SmemLimit limit;
  const size_t smem = table_smem_bytes(bs);
  if ((rc = limit.ensure((const void*)block_trim_kernel, smem + kStaticSmem)) != QQ_OK) return rc;
  return launch_pdl(block_trim_kernel, dim3(1), dim3(kTableThreads), smem, as_stream(stream), a);
}

extern "C" int qq_kv8_append(const qq_kv8_cache* cache, const void* k, const void* v, int dtype, int64_t k_stride,
                             int64_t v_stride, const int64_t* slots, int64_t num_tokens, uint32_t* err, void* stream) {
  using namespace qq;
  int rc = kv8::check(cache);
  if (rc != QQ_OK) return rc;
  if (num_tokens < 0 || cache->state == nullptr || (dtype != QQ_BF16 && dtype != QQ_F32)) return QQ_ERR_INVALID;
  if (num_tokens == 0) return QQ_OK;
  const int64_t row = (int64_t)cache->kv_heads * cache->head_dim;
  if (k == nullptr || v == nullptr || slots == nullptr || k_stride < row || v_stride < row) return QQ_ERR_INVALID;
  const int size = dtype == QQ_BF16 ? 2 : 4;
  if ((k_stride * size) % 16 != 0 || (v_stride * size) % 16 != 0 || reinterpret_cast<uintptr_t>(k) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(v) % 16 != 0 || reinterpret_cast<uintptr_t>(cache->state) % 8 != 0)
    return QQ_ERR_UNSUPPORTED;
  AppendArgs a{};
  a.c = kv8::view(*cache);
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.slots = slots;
  a.n = num_tokens;
  a.err = err;
  // A token per CTA column while there are few (each may be its own run), wider
  // windows for a prefill, whose runs are whole blocks: about kLookTokens columns.
  a.window = 1;
  while (a.window < kMaxWindow && num_tokens > kLookTokens * a.window) a.window *= 2;
  a.claimed = num_tokens > kLookTokens;
  const int64_t ctas = (num_tokens + a.window - 1) / a.window;
  const int pairs = 2 * cache->kv_heads;
  if (num_tokens > INT32_MAX || pairs > 65535) return QQ_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)ctas, pairs);
  const bool d128 = cache->head_dim == 128;
  cudaStream_t s = as_stream(stream);
  if (a.claimed) {
    const dim3 claim_grid((unsigned)((num_tokens + kClaimThreads - 1) / kClaimThreads));
    rc = launch_pdl(kv8_claim_kernel, claim_grid, dim3(kClaimThreads), 0, s, a.c, slots, num_tokens);
    if (rc != QQ_OK) return rc;
  }
  if (dtype == QQ_BF16)
    return d128 ? launch_pdl(kv8_append_kernel<__nv_bfloat16, 128>, dim3(grid), dim3(kAppendThreads), 0, s, a)
                : launch_pdl(kv8_append_kernel<__nv_bfloat16, 0>, dim3(grid), dim3(kAppendThreads), 0, s, a);
  return d128 ? launch_pdl(kv8_append_kernel<float, 128>, dim3(grid), dim3(kAppendThreads), 0, s, a)
              : launch_pdl(kv8_append_kernel<float, 0>, dim3(grid), dim3(kAppendThreads), 0, s, a);
}

extern "C" int qq_kv8_gather(const qq_kv8_cache* cache, const int64_t* slots, int64_t num_tokens, void* k_out,
                             void* v_out, int dtype, uint32_t* err, void* stream) {
  using namespace qq;
  const int rc = kv8::check(cache);
  if (rc != QQ_OK) return rc;
  if (num_tokens < 0 || (dtype != QQ_BF16 && dtype != QQ_F32)) return QQ_ERR_INVALID;
  if (num_tokens == 0) return QQ_OK;
  if (slots == nullptr || k_out == nullptr || v_out == nullptr) return QQ_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(k_out) % 16 != 0 || reinterpret_cast<uintptr_t>(v_out) % 16 != 0)
    return QQ_ERR_UNSUPPORTED;
  const kv8::Cache c = kv8::view(*cache);
  cudaStream_t s = as_stream(stream);
  return dtype == QQ_BF16 ? launch_gather<__nv_bfloat16>(c, slots, num_tokens, k_out, v_out, err, s)
                          : launch_gather<float>(c, slots, num_tokens, k_out, v_out, err, s);
}

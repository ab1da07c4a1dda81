// Attention over the 8-bit block KV cache: the entry points, and the kernel
// that takes every geometry (any head_dim that is a multiple of 8, any group
// of query heads, bf16 or fp32, with fp32 products and sums throughout).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale_log2 q.k_j - m)
//
// One CTA takes up to 4, 8 or 16 query rows that share a KV head (the heads of a
// group, and for an extend batch several new tokens: 16 rows) and one of
// `splits` equal stretches of their keys; tiles of 64 keys are dequantised to
// fp32 in shared memory once for all rows.  The maximum m and the sum run along
// with the tiles; split stretches leave (m, sum, O) records that a second
// kernel joins, or are a cluster that joins them itself.  One token per request is bound by the chain of a tile (table,
// codes, scores, weights, product), so stretches go down to a tile and K and V
// are asked for together (5 x up to 2500 keys of 2 heads of 64 for 8 query
// heads: 13.5 us; 53 with 16 rows always, one tile in hand and stretches of four).
// An extend batch is bound by the fp32 FMAs and their shared-memory operands.

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include <cuda_fp16.h>

#include "kv8_attn.cuh"

namespace qq {
namespace {

using namespace kv8;

constexpr int kMostRows = 16;
constexpr int kTileKeys = 64;
constexpr int kAnyThreads = 128;
constexpr int kMostSplits = 256;
constexpr int64_t kSparePositions = 1 << 17;  // of an extend batch: 128 for each stretch of a row and the two tiles ahead

struct AnyArgs {
  AttnArgs a;
  int rows;         // query rows per CTA at most: 4, 8 or 16
  int head_chunk;   // query heads per CTA
  int chunks;       // CTAs per KV head along its group
  int tile_tokens;  // query tokens per CTA
  int key_groups;   // the product's threads: key groups x channels
  int splits;
  int cluster;      // CTAs of a cluster that take a unit's splits and join them, 0: records and a join
};

// Records of a unit (row tile, KV head, head chunk) and split: rows x (m, l), then rows x dim.
__host__ __device__ inline int64_t any_record(int rows, int dim) { return rows * (2 + (int64_t)dim); }

// K and V of a tile at once, but for 16 rows, whose CTAs would no longer be four to an SM.
__host__ __device__ constexpr bool any_both(int rows) { return rows < 16; }
inline int any_tile_floats(int rows, int dim, int key_groups) {
  const int tile = kTileKeys * (dim + 4) * (any_both(rows) ? 2 : 1), sums = key_groups * rows * dim;
  return tile > sums ? tile : sums;
}
inline size_t any_smem(const AnyArgs& g) {
  const int dim = g.a.c.dim;
  return sizeof(float) * (g.rows * dim + any_tile_floats(g.rows, dim, g.key_groups) + g.rows * kTileKeys);
}

// The keys of a stretch when `tiles` tiles are cut into at most `splits`.
__device__ __forceinline__ int64_t stretch_keys(int64_t keys, int splits) {
  return ((keys + kTileKeys - 1) / kTileKeys + splits - 1) / splits * kTileKeys;
}

// CLUSTER: the splits of a unit are a cluster, which joins them itself.
template <typename T, int KEYS, int ROWS, bool CLUSTER>
__global__ void __launch_bounds__(kAnyThreads) kv8_attn_any_kernel(AnyArgs g) {
  constexpr bool kBoth = any_both(ROWS);
  extern __shared__ __align__(16) float s_buf[];
  __shared__ float s_m[ROWS], s_l[ROWS], s_corr[ROWS];
  __shared__ int64_t s_slot[kTileKeys];
  __shared__ float s_ks[kTileKeys], s_vs[kTileKeys];
  const AttnArgs& a = g.a;
  const Cache& c = a.c;
  const int dim = c.dim, pitch = dim + 4, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* s_q = s_buf;                      // [ROWS][dim], times scale_log2
  float* s_p = s_q + ROWS * dim;           // [ROWS][64]
  float* s_k = s_p + ROWS * kTileKeys;     // [64][pitch]
  float* s_v = kBoth ? s_k + kTileKeys * pitch : s_k;
  wait_prior_grid();
  allow_next_grid();

  const int kvh = blockIdx.y / g.chunks, chunk = blockIdx.y - kvh * g.chunks;
  const int h0 = kvh * a.group + chunk * g.head_chunk;
  const int nh = min(g.head_chunk, a.group - chunk * g.head_chunk);
  // errors of the entries are reported once
  uint32_t* err = blockIdx.y == 0 && blockIdx.z == 0 ? a.err : nullptr;
  int e = blockIdx.x;
  int64_t row0 = e, tokens = 1, seen0;  // query rows row0 .., the first sees keys [0, seen0), each next one more
  if (KEYS == kExtend) {
    const ExtendEntry x = extend_tile(a, blockIdx.x, g.tile_tokens, 1, blockIdx.x == 0 ? err : nullptr);
    if (blockIdx.x == 0 && extend_tiles(a, g.tile_tokens, 1, nullptr) > gridDim.x)
      raise_error(err, QQ_DEV_ERR_BOUNDS);  // entries share query rows
    if (x.entry < 0) return;  // past the last tile
    e = x.entry;
    row0 = x.row0 + x.tile * g.tile_tokens;
    tokens = min((int64_t)g.tile_tokens, x.n - x.tile * g.tile_tokens);
    seen0 = x.prefix + x.tile * g.tile_tokens + 1;
  } else {
    seen0 = entry_keys<KEYS>(a, e, tid == 0 ? err : nullptr);
  }
  const int R = (int)tokens * nh;
  const int64_t L = seen0 > 0 ? seen0 + tokens - 1 : 0;
  const int64_t req = KEYS == kRows ? 0 : (L > 0 ? a.reqs[e] : 0);
  const int64_t stretch = stretch_keys(L, g.splits);
  const int64_t k0 = blockIdx.z * stretch, k1 = min(L, k0 + stretch);
  if (!CLUSTER && k0 >= k1 && blockIdx.z > 0) return;  // nothing left for this one, uniform

  for (int i = tid; i < R * dim; i += kAnyThreads) {
    const int r = i / dim, d = i - r * dim;
    const T* q = static_cast<const T*>(a.q) + (row0 + r / nh) * a.q_stride + (int64_t)(h0 + r % nh) * dim;
    s_q[i] = Elem<T>::load(q + d) * a.scale_log2;
  }
  for (int i = R * dim + tid; i < ROWS * dim; i += kAnyThreads) s_q[i] = 0.f;
  if (tid < ROWS) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float acc[2][ROWS] = {};
  const int lanes = kAnyThreads / g.key_groups, group = tid / lanes, d0 = tid - group * lanes;
  uint32_t* kerr = blockIdx.y == 0 ? a.err : nullptr;

  // codes of a tile to fp32, K or V or both; whether V held a NaN
  auto load_tile = [&](auto keys, auto values) {
    const int per = dim >> 3;
    int nan = 0;
#pragma unroll 4
    for (int i = tid; i < kTileKeys * per; i += kAnyThreads) {
      const int j = i / per, ch = i - j * per;
      const int64_t slot = s_slot[j];
      uint2 ck = make_uint2(0, 0), cv = make_uint2(0, 0);
      if (slot >= 0) {
        const int64_t at = (((slot >> c.shift) * c.kv_heads + kvh) * c.block + (slot & (c.block - 1))) * dim + ch * 8;
        if (keys.value) ck = __ldg(reinterpret_cast<const uint2*>(c.k + at));
        if (values.value) cv = __ldg(reinterpret_cast<const uint2*>(c.v + at));
      }
      float x[8];
      if (keys.value) {
        from_e4m3x8(ck, x);
        const float f = s_ks[j];
        float4* d = reinterpret_cast<float4*>(s_k + j * pitch + ch * 8);
        d[0] = make_float4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
        d[1] = make_float4(x[4] * f, x[5] * f, x[6] * f, x[7] * f);
      }
      if (values.value) {
        from_e4m3x8(cv, x);
        const float f = s_vs[j];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          x[u] *= f;
          nan |= isnan(x[u]);
        }
        float4* d = reinterpret_cast<float4*>(s_v + j * pitch + ch * 8);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
    return nan;
  };

  // the places and scales of a tile are asked for while the one before is at work
  int64_t slot = -1;
  float ks = 0.f, vs = 0.f;
  auto place = [&](int64_t j0) {
    slot = -1, ks = 0.f, vs = 0.f;
    if (tid >= kTileKeys || j0 + tid >= k1) return;
    slot = key_slot<KEYS>(a, e, req, j0 + tid, kerr);
    if (slot < 0) return;
    const int64_t bh = (slot >> c.shift) * c.kv_heads + kvh;
    ks = c.k_scale[bh];
    vs = c.v_scale[bh];
  };
  place(k0);
  for (int64_t j0 = k0; j0 < k1; j0 += kTileKeys) {
    __syncthreads();
    if (tid < kTileKeys) s_slot[tid] = slot, s_ks[tid] = ks, s_vs[tid] = vs;
    __syncthreads();
    int nan = load_tile(std::true_type{}, std::bool_constant<kBoth>{});
    place(j0 + kTileKeys);
    __syncthreads();
    {  // scores: thread = key x half of the rows
      constexpr int kHalf = ROWS / 2;
      const int j = tid & 63, r0 = (tid >> 6) * kHalf;
      float s[kHalf] = {};
      const float* kp = s_k + j * pitch;
      for (int d = 0; d < dim; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(kp + d);
#pragma unroll
        for (int r = 0; r < kHalf; ++r) {
          const float4 q4 = *reinterpret_cast<const float4*>(s_q + (r0 + r) * dim + d);
          s[r] += fmaf(k4.x, q4.x, fmaf(k4.y, q4.y, fmaf(k4.z, q4.z, k4.w * q4.w)));
        }
      }
      const bool there = s_slot[j] >= 0;
#pragma unroll
      for (int r = 0; r < kHalf; ++r) {
        const bool seen = there && r0 + r < R && j0 + j < seen0 + (KEYS == kExtend ? (r0 + r) / nh : 0);
        s_p[(r0 + r) * kTileKeys + j] = seen ? s[r] : -INFINITY;
      }
    }
    __syncthreads();
    if (!kBoth) nan = load_tile(std::false_type{}, std::true_type{});
#pragma unroll
    for (int r = warp * (ROWS / 4); r < (warp + 1) * (ROWS / 4); ++r) {  // softmax: a warp's rows
      const float x0 = s_p[r * kTileKeys + lane], x1 = s_p[r * kTileKeys + lane + 32];
      // the maximum drops NaN: a NaN score must reach the sum through its weight
      const float mo = s_m[r], mn = fmaxf(mo, warp_max(fmaxf(x0, x1))), base = mn == -INFINITY ? 0.f : mn;
      const float p0 = exp2f(x0 - base), p1 = exp2f(x1 - base);
      float l = p0 + p1;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      s_p[r * kTileKeys + lane] = p0;
      s_p[r * kTileKeys + lane + 32] = p1;
      __syncwarp();
      if (lane == 0) {
        const float corr = exp2f(mo - base);
        s_corr[r] = corr;
        s_m[r] = mn;
        s_l[r] = s_l[r] * corr + l;
      }
    }
    const int any_nan = __syncthreads_or(nan);
    auto product = [&](auto guard) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int d = d0 + u * kAnyThreads;
        if (d >= dim) break;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) acc[u][r] *= s_corr[r];
        // a NaN stays with the rows that see its key
        auto behind = [&](float p, float v) { return guard.value && p == 0.f ? 0.f : v; };
        const int keys = kTileKeys / g.key_groups;
        for (int j = group * keys; j < (group + 1) * keys; j += 4) {
          const float v0 = s_v[j * pitch + d], v1 = s_v[(j + 1) * pitch + d];
          const float v2 = s_v[(j + 2) * pitch + d], v3 = s_v[(j + 3) * pitch + d];
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float4 p = *reinterpret_cast<const float4*>(s_p + r * kTileKeys + j);
            acc[u][r] += fmaf(p.x, behind(p.x, v0), fmaf(p.y, behind(p.y, v1),
                                                        fmaf(p.z, behind(p.z, v2), p.w * behind(p.w, v3))));
          }
        }
      }
    };
    if (any_nan) product(std::true_type{});
    else product(std::false_type{});
  }
  __syncthreads();
  float* rec = a.part + (((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * g.splits + blockIdx.z) * any_record(ROWS, dim);
  const bool whole = !CLUSTER && stretch >= L;  // all keys are in this stretch
  if (!CLUSTER && !whole && tid < R) rec[2 * tid] = s_m[tid], rec[2 * tid + 1] = s_l[tid];
  if (g.key_groups > 1) {  // the groups' sums meet in the first one's threads
    if (d0 < dim)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) s_k[(group * ROWS + r) * dim + d0] = acc[0][r];
    __syncthreads();
    if (!CLUSTER && (group > 0 || d0 >= dim)) return;
#pragma unroll
    for (int r = 0; r < ROWS && d0 < dim; ++r)
      for (int k = 1; k < g.key_groups; ++k) acc[0][r] += s_k[(k * ROWS + r) * dim + d0];
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int d = d0 + u * kAnyThreads;
    if (d >= dim || group > 0) break;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r >= R) break;
      if (CLUSTER) {
        s_q[r * dim + d] = acc[u][r];  // the queries have done their work
      } else if (whole) {
        T* o = static_cast<T*>(a.out) + (row0 + r / nh) * a.out_stride + (int64_t)(h0 + r % nh) * dim;
        const float l = s_l[r];
        Elem<T>::store(o + d, l == 0.f ? 0.f : acc[u][r] / l);
      } else {
        rec[2 * ROWS + r * dim + d] = acc[u][r];
      }
    }
  }
  if constexpr (CLUSTER) {
    // ---- four threads per output, each with its part of the records
    __syncthreads();
    cluster_sync();
    const int outs = R * dim, part = tid & 3;
    for (int i0 = blockIdx.z * (kAnyThreads / 4); i0 < outs; i0 += g.cluster * (kAnyThreads / 4)) {
      const int i = min(i0 + (tid >> 2), outs - 1), r = i / dim;
      float m[4], l[4], o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int rank = part + 4 * k;
        m[k] = -INFINITY, l[k] = 0.f, o[k] = 0.f;
        if (rank >= g.cluster) continue;
        m[k] = ld_cluster(smem_u32(s_m + r), rank);
        l[k] = ld_cluster(smem_u32(s_l + r), rank);
        o[k] = ld_cluster(smem_u32(s_q + i), rank);
      }
      float mn = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
      const float ref = mn == -INFINITY ? 0.f : mn;
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = exp2f(m[k] - ref);
        sum = fmaf(f, l[k], sum);
        x = fmaf(f, o[k], x);
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        x += __shfl_xor_sync(0xffffffffu, x, d);
      }
      if (part == 0 && i0 + (tid >> 2) < outs)
        Elem<T>::store(static_cast<T*>(a.out) + (row0 + r / nh) * a.out_stride + (int64_t)(h0 + r % nh) * dim + i - r * dim,
                       sum == 0.f ? 0.f : x / sum);
    }
    cluster_sync();  // the records stay until all have read them
  }
}

// Joins the splits of unit (blockIdx.x, blockIdx.y), the CTAs of blockIdx.z
// taking its rows in turn: a thread per split for the weights, then four
// channels per thread and the splits over groups of threads, so that a row is
// a few loads long (a warp per row: 14 us for 40 splits, this 8).
constexpr int kAnyJoinThreads = 128;
template <typename T, int KEYS>
__global__ void __launch_bounds__(kAnyJoinThreads) kv8_attn_join_kernel(AnyArgs g) {
  __shared__ float s_w[kMostSplits], s_m[kAnyJoinThreads / 32], s_l[kAnyJoinThreads / 32];
  __shared__ float4 s_o[kAnyJoinThreads];
  const AttnArgs& a = g.a;
  const int dim = a.c.dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.y / g.chunks, chunk = blockIdx.y - kvh * g.chunks;
  const int h0 = kvh * a.group + chunk * g.head_chunk;
  const int nh = min(g.head_chunk, a.group - chunk * g.head_chunk);
  wait_prior_grid();
  allow_next_grid();
  int64_t row0 = blockIdx.x, tokens = 1, seen0;
  if (KEYS == kExtend) {
    const ExtendEntry x = extend_tile(a, blockIdx.x, g.tile_tokens, 1, nullptr);
    if (x.entry < 0) return;
    row0 = x.row0 + x.tile * g.tile_tokens;
    tokens = min((int64_t)g.tile_tokens, x.n - x.tile * g.tile_tokens);
    seen0 = x.prefix + x.tile * g.tile_tokens + 1;
  } else {
    seen0 = entry_keys<KEYS>(a, blockIdx.x, nullptr);
  }
  const int64_t L = seen0 > 0 ? seen0 + tokens - 1 : 0, stretch = stretch_keys(L, g.splits);
  if (stretch >= L) return;  // written by its CTA
  const int splits = (int)((L + stretch - 1) / stretch);
  const int64_t record = any_record(g.rows, dim);
  const float* rec = a.part + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * g.splits * record;
  int pieces = 2;  // of four channels, to a power of two
  while (pieces * 4 < dim) pieces *= 2;
  const int piece = tid & (pieces - 1), group = tid / pieces, groups = kAnyJoinThreads / pieces;
  for (int r = blockIdx.z; r < (int)tokens * nh; r += gridDim.z) {
    float m = -INFINITY, l = 0.f;
    for (int s = tid; s < splits; s += kAnyJoinThreads) m = fmaxf(m, rec[s * record + 2 * r]);
    m = warp_max(m);
    if (lane == 0) s_m[warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const float base = m == -INFINITY ? 0.f : m;
    for (int s = tid; s < splits; s += kAnyJoinThreads) {
      const float w = exp2f(rec[s * record + 2 * r] - base);
      s_w[s] = w;
      l = fmaf(w, rec[s * record + 2 * r + 1], l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (piece * 4 < dim) {
      const float* p = rec + 2 * g.rows + r * dim + piece * 4;
#pragma unroll 8
      for (int s = group; s < splits; s += groups) {
        const float4 v = *reinterpret_cast<const float4*>(p + s * record);
        const float w = s_w[s];
        o.x = fmaf(w, v.x, o.x), o.y = fmaf(w, v.y, o.y), o.z = fmaf(w, v.z, o.z), o.w = fmaf(w, v.w, o.w);
      }
    }
    s_o[tid] = o;
    __syncthreads();
    if (group == 0 && piece * 4 < dim) {
      for (int k = 1; k < groups; ++k) {
        const float4 v = s_o[k * pieces + piece];
        o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
      }
      const float sum = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]), x[4] = {o.x, o.y, o.z, o.w};
      T* out = static_cast<T*>(a.out) + (row0 + r / nh) * a.out_stride + (int64_t)(h0 + r % nh) * dim + piece * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) Elem<T>::store(out + e, sum == 0.f ? 0.f : x[e] / sum);
    }
    __syncthreads();  // the next row's numbers go to the same places
  }
}

AnyArgs any_shape(const AttnArgs& a, int keys) {
  AnyArgs g{};
  g.a = a;
  g.head_chunk = a.group < kMostRows ? a.group : kMostRows;
  g.chunks = (a.group + g.head_chunk - 1) / g.head_chunk;
  g.tile_tokens = keys == kExtend ? kMostRows / g.head_chunk : 1;
  g.rows = keys == kExtend || g.head_chunk > 8 ? 16 : g.head_chunk > 4 ? 8 : 4;
  g.key_groups = 1;
  while (g.key_groups < 8 && 2 * g.key_groups * a.c.dim <= kAnyThreads) g.key_groups *= 2;
  return g;
}
int64_t any_tiles(const AnyArgs& g, int keys, int bs, int64_t tokens) {
  return keys == kExtend ? (tokens + g.tile_tokens - 1) / g.tile_tokens + bs : bs;
}
// Stretches of the keys: about four CTAs per SM over the whole launch.
int any_splits(const AnyArgs& g, int64_t tiles, int kv_heads, int64_t max_keys) {
  const int64_t units = tiles * kv_heads * g.chunks;
  int64_t s = units > 0 ? (4 * (int64_t)device_sm_count() + units - 1) / units : 1;
  const int64_t most = (max_keys + kTileKeys - 1) / kTileKeys;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : (s > kMostSplits ? kMostSplits : s));
}
int64_t any_workspace(const AnyArgs& g, int64_t tiles) {
  return g.splits == 1 || g.cluster > 0 ? 0 : (int64_t)sizeof(float) * tiles * g.a.c.kv_heads * g.chunks * g.splits * any_record(g.rows, g.a.c.dim);
}

template <typename T, int KEYS, int ROWS>
int launch_any(const AnyArgs& g, int64_t tiles, cudaStream_t s) {
  const size_t smem = any_smem(g);
  const dim3 grid((unsigned)tiles, g.a.c.kv_heads * g.chunks, g.splits);
  if constexpr (KEYS != kExtend) {
    if (g.cluster > 0) {
      ClusterLaunch l(grid, dim3(1, 1, g.cluster), kAnyThreads, smem, s);
      return cudaLaunchKernelEx(&l.cfg, kv8_attn_any_kernel<T, KEYS, ROWS, true>, g) == cudaSuccess ? QQ_OK : QQ_ERR_CUDA;
    }
  }
  static SmemLimit limit;
  int rc = limit.ensure((const void*)kv8_attn_any_kernel<T, KEYS, ROWS, false>, smem + kStaticSmem);
  if (rc != QQ_OK) return rc;
  rc = launch_pdl(kv8_attn_any_kernel<T, KEYS, ROWS, false>, grid, dim3(kAnyThreads), smem, s, g);
  if (rc != QQ_OK || g.splits == 1) return rc;
  const int64_t units = tiles * grid.y, per = 4 * (int64_t)device_sm_count() / units;  // CTAs to a unit
  const unsigned z = (unsigned)std::max<int64_t>(1, std::min<int64_t>(per, g.rows));
  return launch_pdl(kv8_attn_join_kernel<T, KEYS>, dim3(grid.x, grid.y, z), dim3(kAnyJoinThreads), 0, s, g);
}
template <typename T>
int launch_any(const AnyArgs& g, int keys, int64_t tiles, cudaStream_t s) {
  if (keys == kExtend) return launch_any<T, kExtend, 16>(g, tiles, s);
  if (keys == kTable)
    return g.rows == 4   ? launch_any<T, kTable, 4>(g, tiles, s)
           : g.rows == 8 ? launch_any<T, kTable, 8>(g, tiles, s)
                         : launch_any<T, kTable, 16>(g, tiles, s);
  return g.rows == 4   ? launch_any<T, kRows, 4>(g, tiles, s)
         : g.rows == 8 ? launch_any<T, kRows, 8>(g, tiles, s)
                       : launch_any<T, kRows, 16>(g, tiles, s);
}

// Shared memory of `rows` rows of up to `dim` channels.
size_t smem_up_to(int rows, int dim) {
  AnyArgs g{};
  g.a.c.dim = dim;
  g.rows = rows;
  g.key_groups = 1;
  return any_smem(g);
}
template <typename T, int KEYS, int ROWS>
int resident_any(int dim, int cluster) {
  static ResidentClusters known[3][3];  // by cluster, by head_dim up to 64, 128 and 256
  const int c = cluster == 16 ? 0 : cluster == 8 ? 1 : 2, d = dim <= 64 ? 0 : dim <= 128 ? 1 : 2;
  return known[c][d].ask((const void*)kv8_attn_any_kernel<T, KEYS, ROWS, true>, dim3(1, 1, cluster), kAnyThreads,
                         smem_up_to(ROWS, 64 << d), smem_up_to(ROWS, kMaxDim));
}
template <typename T, int KEYS>
int resident_any(const AnyArgs& g, int cluster) {
  return g.rows == 4   ? resident_any<T, KEYS, 4>(g.a.c.dim, cluster)
         : g.rows == 8 ? resident_any<T, KEYS, 8>(g.a.c.dim, cluster)
                       : resident_any<T, KEYS, 16>(g.a.c.dim, cluster);
}
// One token per entry: the cluster that takes a unit, 0 for records and a join.
// All clusters run at a time, and no CTA has more than two tiles: 5 x 1,024 keys
// of 2 heads of 64 (a tile to a CTA) take 9.3 us on the device where records and
// a join take 11.5, 10 x 500 (two) 11.8 and 11.3 but 3 us less on the host; with
// three to a CTA 1 x 2,500 would take 15.6 and 11.7.
int any_cluster(const AnyArgs& g, int dtype, int64_t units, int64_t max_keys) {
  if (max_keys <= kTileKeys || units > device_sm_count()) return 0;
  for (int c = 16; c >= 4; c /= 2) {
    if (max_keys > c * 2 * kTileKeys) return 0;
    const int most = dtype == QQ_BF16
                         ? std::min(resident_any<__nv_bfloat16, kTable>(g, c), resident_any<__nv_bfloat16, kRows>(g, c))
                         : std::min(resident_any<float, kTable>(g, c), resident_any<float, kRows>(g, c));
    if (units <= most) return c;
  }
  return 0;
}
// Splits and cluster of a call.
void any_plan(AnyArgs& g, int keys, int dtype, int64_t tiles, int64_t max_keys) {
  g.splits = any_splits(g, tiles, g.a.c.kv_heads, max_keys);
  if (keys == kExtend || g.splits == 1) return;
  g.cluster = any_cluster(g, dtype, tiles * g.a.c.kv_heads * g.chunks, max_keys);
  if (g.cluster > 0) g.splits = g.cluster;
}

int run(const AttnArgs& a, int keys, int dtype, int64_t max_keys, size_t ws_bytes, cudaStream_t s) {
  if (keys != kExtend && decode_tc_fits(a, dtype)) return run_decode_tc(a, keys, max_keys, ws_bytes, s);
  if (keys == kExtend && extend_tc_fits(a, dtype)) return run_extend_tc(a, max_keys, ws_bytes, s);
  AnyArgs g = any_shape(a, keys);
  const int64_t tiles = any_tiles(g, keys, a.bs, a.tokens);
  if (tiles > INT32_MAX || (int64_t)a.c.kv_heads * g.chunks > 65535) return QQ_ERR_UNSUPPORTED;
  any_plan(g, keys, dtype, tiles, max_keys);
  if (any_workspace(g, tiles) > 0 && (a.part == nullptr || ws_bytes < (size_t)any_workspace(g, tiles))) return QQ_ERR_WORKSPACE;
  return dtype == QQ_BF16 ? launch_any<__nv_bfloat16>(g, keys, tiles, s) : launch_any<float>(g, keys, tiles, s);
}

// Checks the arguments the three entries share and fills them in.
int common_args(const qq_kv8_cache* cache, const void* q, int dtype, int q_heads, int64_t q_stride, float scaling,
                void* out, int64_t out_stride, void* workspace, uint32_t* err, AttnArgs& a) {
  const int rc = check(cache);
  if (rc != QQ_OK) return rc;
  if (q == nullptr || out == nullptr || (dtype != QQ_BF16 && dtype != QQ_F32) || q_heads <= 0 ||
      q_heads % cache->kv_heads != 0 || q_stride < (int64_t)q_heads * cache->head_dim ||
      out_stride < (int64_t)q_heads * cache->head_dim)
    return QQ_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return QQ_ERR_UNSUPPORTED;
  a.c = view(*cache);
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.heads = q_heads;
  a.group = q_heads / cache->kv_heads;
  a.scale_log2 = scaling * 1.4426950408889634f;
  a.part = static_cast<float*>(workspace);
  a.err = err;
  return QQ_OK;
}

}  // namespace
}  // namespace qq

extern "C" size_t qq_kv8_workspace_bytes(const qq_kv8_cache* cache, int q_heads, int dtype, int bs, int64_t num_tokens,
                                         int64_t max_keys, int extend) {
  using namespace qq;
  if (kv8::check(cache) != QQ_OK || q_heads <= 0 || q_heads % cache->kv_heads != 0 || bs <= 0) return 0;
  AttnArgs a{};
  a.c = kv8::view(*cache);
  a.group = q_heads / cache->kv_heads;
  const int keys = extend ? kExtend : kTable;
  AnyArgs g = any_shape(a, keys);
  const int64_t tiles = any_tiles(g, keys, bs, num_tokens);
  any_plan(g, keys, dtype, tiles, max_keys);
  size_t need = (size_t)any_workspace(g, tiles);
  // enough for either kernel: which one runs depends on the pointers' alignment too
  if (keys != kExtend && decode_tc_fits(a, dtype)) {
    const size_t tc = decode_tc_workspace(bs, a.c.kv_heads, a.group, max_keys);
    if (tc > need) need = tc;
  }
  a.bs = bs;
  a.tokens = num_tokens;
  if (keys == kExtend && extend_tc_fits(a, dtype)) {
    const size_t tc = extend_tc_workspace(bs, a.c.kv_heads, a.group, num_tokens, max_keys);
    if (tc > need) need = tc;
  }
  return need;
}

extern "C" int qq_kv8_decode_attention(const qq_kv8_cache* cache, const qq_batch* batch, const int32_t* block_table,
                                       int64_t table_stride, int64_t table_rows, const void* q, int dtype, int q_heads,
                                       int64_t q_stride, float scaling, void* out, int64_t out_stride, uint32_t* err,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  using namespace qq;
  if (batch == nullptr || batch->bs < 0) return QQ_ERR_INVALID;
  if (batch->bs == 0) return kv8::check(cache);
  AttnArgs a{};
  const int rc = common_args(cache, q, dtype, q_heads, q_stride, scaling, out, out_stride, workspace, err, a);
  if (rc != QQ_OK) return rc;
  if (batch->req_pool_indices == nullptr || batch->seq_lens == nullptr || block_table == nullptr || table_stride <= 0 ||
      table_rows <= 0)
    return QQ_ERR_INVALID;
  if (batch->bs > QQ_MAX_BS || table_stride > INT32_MAX / kv8::kMaxBlock) return QQ_ERR_UNSUPPORTED;
  a.bs = batch->bs;
  a.reqs = batch->req_pool_indices;
  a.seq = batch->seq_lens;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_rows = table_rows;
  a.tokens = a.bs;
  return run(a, kTable, dtype, table_stride << a.c.shift, workspace_bytes, as_stream(stream));
}

extern "C" int qq_kv8_sparse_attention(const qq_kv8_cache* cache, int bs, const int32_t* rows, int64_t rows_stride,
                                       int top_k, const int32_t* lens, const void* q, int dtype, int q_heads,
                                       int64_t q_stride, float scaling, void* out, int64_t out_stride, uint32_t* err,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  using namespace qq;
  if (bs < 0) return QQ_ERR_INVALID;
  if (bs == 0) return kv8::check(cache);
  AttnArgs a{};
  const int rc = common_args(cache, q, dtype, q_heads, q_stride, scaling, out, out_stride, workspace, err, a);
  if (rc != QQ_OK) return rc;
  if (rows == nullptr || lens == nullptr || top_k <= 0 || rows_stride < top_k) return QQ_ERR_INVALID;
  if (bs > QQ_MAX_BS) return QQ_ERR_UNSUPPORTED;
  a.bs = bs;
  a.rows = rows;
  a.rows_stride = rows_stride;
  a.lens = lens;
  a.top = top_k;
  a.tokens = bs;
  return run(a, kRows, dtype, top_k, workspace_bytes, as_stream(stream));
}

extern "C" int qq_kv8_extend_attention(const qq_kv8_cache* cache, const qq_extend_batch* batch,
                                       const int32_t* block_table, int64_t table_stride, int64_t table_rows,
                                       const void* q, int dtype, int q_heads, int64_t q_stride, float scaling,
                                       void* out, int64_t out_stride, uint32_t* err, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  using namespace qq;
  if (batch == nullptr || batch->bs < 0 || batch->num_tokens < 0) return QQ_ERR_INVALID;
  if (batch->bs == 0 || batch->num_tokens == 0) return kv8::check(cache);
  AttnArgs a{};
  const int rc = common_args(cache, q, dtype, q_heads, q_stride, scaling, out, out_stride, workspace, err, a);
  if (rc != QQ_OK) return rc;
  if (batch->req_pool_indices == nullptr || batch->seq_lens == nullptr || batch->prefix_lens == nullptr ||
      batch->token_offsets == nullptr || block_table == nullptr || table_stride <= 0 || table_rows <= 0)
    return QQ_ERR_INVALID;
  // positions, and those of the key tiles asked for ahead or cut off behind the last one, are held in 32 bits
  if (batch->bs > QQ_MAX_BS || table_stride > INT32_MAX / kv8::kMaxBlock ||
      table_stride << a.c.shift > INT32_MAX - kSparePositions)
    return QQ_ERR_UNSUPPORTED;
  a.bs = batch->bs;
  a.reqs = batch->req_pool_indices;
  a.seq = batch->seq_lens;
  a.prefix = batch->prefix_lens;
  a.offsets = batch->token_offsets;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_rows = table_rows;
  a.tokens = batch->num_tokens;
  return run(a, kExtend, dtype, table_stride << a.c.shift, workspace_bytes, as_stream(stream));
}

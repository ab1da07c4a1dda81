// Attention over the 8-bit block KV cache: the entry points, and the kernel
// that takes every geometry (any head_dim that is a multiple of 8, any group
// of query heads, bf16 or fp32, with fp32 products and sums throughout).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale_log2 q.k_j - m)
//
// One CTA takes up to 16 query rows that share a KV head (the heads of a
// group, and for an extend batch several new tokens) and one of `splits`
// equal stretches of their keys; tiles of 64 keys are dequantised to fp32 in
// shared memory once for all rows.  The maximum m and the sum run along with
// the tiles; split stretches leave (m, sum, O) records that a second kernel
// joins.  Bound by the fp32 FMAs and their shared-memory operands.

#include <climits>
#include <cmath>
#include <type_traits>

#include <cuda_fp16.h>

#include "kv8_attn.cuh"

namespace qq {
namespace {

using namespace kv8;

constexpr int kRowsPerCta = 16;
constexpr int kTileKeys = 64;
constexpr int kAnyThreads = 128;

struct AnyArgs {
  AttnArgs a;
  int head_chunk;   // query heads per CTA
  int chunks;       // CTAs per KV head along its group
  int tile_tokens;  // query tokens per CTA
  int splits;
};

// Records of a unit (row tile, KV head, head chunk) and split: 16 x (m, l), then 16 x dim.
__host__ __device__ inline int64_t any_record(int dim) { return kRowsPerCta * (2 + (int64_t)dim); }

inline size_t any_smem(int dim) {
  return sizeof(float) * (kRowsPerCta * dim + kTileKeys * (dim + 4) + kRowsPerCta * kTileKeys);
}

template <typename T, int KEYS>
__global__ void __launch_bounds__(kAnyThreads) kv8_attn_any_kernel(AnyArgs g) {
  extern __shared__ __align__(16) float s_buf[];
  __shared__ float s_m[kRowsPerCta], s_l[kRowsPerCta], s_corr[kRowsPerCta];
  __shared__ int64_t s_slot[kTileKeys];
  __shared__ float s_ks[kTileKeys], s_vs[kTileKeys];
  const AttnArgs& a = g.a;
  const Cache& c = a.c;
  const int dim = c.dim, pitch = dim + 4, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* s_q = s_buf;                      // [16][dim], times scale_log2
  float* s_kv = s_q + kRowsPerCta * dim;   // [64][pitch]
  float* s_p = s_kv + kTileKeys * pitch;   // [16][64]

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
  const int64_t stretch = ((L + kTileKeys - 1) / kTileKeys + g.splits - 1) / g.splits * kTileKeys;
  const int64_t k0 = blockIdx.z * stretch, k1 = min(L, k0 + stretch);

  for (int i = tid; i < R * dim; i += kAnyThreads) {
    const int r = i / dim, d = i - r * dim;
    const T* q = static_cast<const T*>(a.q) + (row0 + r / nh) * a.q_stride + (int64_t)(h0 + r % nh) * dim;
    s_q[i] = Elem<T>::load(q + d) * a.scale_log2;
  }
  for (int i = R * dim + tid; i < kRowsPerCta * dim; i += kAnyThreads) s_q[i] = 0.f;
  if (tid < kRowsPerCta) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float acc[2][kRowsPerCta] = {};
  uint32_t* kerr = blockIdx.y == 0 ? a.err : nullptr;

  auto load_tile = [&](const uint8_t* codes, const float* s_scale) {
    const int per = dim >> 3;
    int nan = 0;
    for (int i = tid; i < kTileKeys * per; i += kAnyThreads) {
      const int j = i / per, ch = i - j * per;
      const int64_t slot = s_slot[j];
      float x[8] = {};
      if (slot >= 0) {
        const int64_t at = (((slot >> c.shift) * c.kv_heads + kvh) * c.block + (slot & (c.block - 1))) * dim;
        from_e4m3x8(*reinterpret_cast<const uint2*>(codes + at + ch * 8), x);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          x[u] *= s_scale[j];
          nan |= isnan(x[u]);
        }
      }
      float4* d = reinterpret_cast<float4*>(s_kv + j * pitch + ch * 8);
      d[0] = make_float4(x[0], x[1], x[2], x[3]);
      d[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
    return nan;
  };

  for (int64_t j0 = k0; j0 < k1; j0 += kTileKeys) {
    __syncthreads();
    if (tid < kTileKeys) {
      int64_t slot = -1;
      if (j0 + tid < k1) slot = key_slot<KEYS>(a, e, req, j0 + tid, kerr);
      s_slot[tid] = slot;
      const int64_t bh = slot < 0 ? 0 : (slot >> c.shift) * c.kv_heads + kvh;
      s_ks[tid] = slot < 0 ? 0.f : c.k_scale[bh];
      s_vs[tid] = slot < 0 ? 0.f : c.v_scale[bh];
    }
    __syncthreads();
    load_tile(c.k, s_ks);
    __syncthreads();
    {  // scores: thread = key x half of the rows
      const int j = tid & 63, r0 = (tid >> 6) * 8;
      float s[8] = {};
      const float* kp = s_kv + j * pitch;
      for (int d = 0; d < dim; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4*>(kp + d);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float4 q4 = *reinterpret_cast<const float4*>(s_q + (r0 + r) * dim + d);
          s[r] += fmaf(k4.x, q4.x, fmaf(k4.y, q4.y, fmaf(k4.z, q4.z, k4.w * q4.w)));
        }
      }
      const bool there = s_slot[j] >= 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const bool seen = there && r0 + r < R && j0 + j < seen0 + (KEYS == kExtend ? (r0 + r) / nh : 0);
        s_p[(r0 + r) * kTileKeys + j] = seen ? s[r] : -INFINITY;
      }
    }
    __syncthreads();
    const int nan = load_tile(c.v, s_vs);
    for (int r = warp * 4; r < warp * 4 + 4; ++r) {  // softmax: a warp's four rows
      const float x0 = s_p[r * kTileKeys + lane], x1 = s_p[r * kTileKeys + lane + 32];
      // fmaxf drops NaN: a NaN score must reach the sum through its weight
      float m = fmaxf(x0, x1);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float mo = s_m[r], mn = fmaxf(mo, m), base = mn == -INFINITY ? 0.f : mn;
      const float p0 = exp2f(x0 - base), p1 = exp2f(x1 - base);
      float l = p0 + p1;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      s_p[r * kTileKeys + lane] = p0;
      s_p[r * kTileKeys + lane + 32] = p1;
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
        const int d = tid + u * kAnyThreads;
        if (d >= dim) break;
#pragma unroll
        for (int r = 0; r < kRowsPerCta; ++r) acc[u][r] *= s_corr[r];
        // a NaN stays with the rows that see its key
        auto behind = [&](float p, float v) { return guard.value && p == 0.f ? 0.f : v; };
        for (int j = 0; j < kTileKeys; j += 4) {
          const float v0 = s_kv[j * pitch + d], v1 = s_kv[(j + 1) * pitch + d];
          const float v2 = s_kv[(j + 2) * pitch + d], v3 = s_kv[(j + 3) * pitch + d];
#pragma unroll
          for (int r = 0; r < kRowsPerCta; ++r) {
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
  if (g.splits == 1) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int d = tid + u * kAnyThreads;
      if (d >= dim) break;
#pragma unroll
      for (int r = 0; r < kRowsPerCta; ++r) {
        if (r >= R) break;
        T* o = static_cast<T*>(a.out) + (row0 + r / nh) * a.out_stride + (int64_t)(h0 + r % nh) * dim;
        const float l = s_l[r];
        Elem<T>::store(o + d, l == 0.f ? 0.f : acc[u][r] / l);
      }
    }
    return;
  }
  float* rec = a.part + (((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * g.splits + blockIdx.z) * any_record(dim);
  if (tid < kRowsPerCta) {
    rec[2 * tid] = s_m[tid];
    rec[2 * tid + 1] = s_l[tid];
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int d = tid + u * kAnyThreads;
    if (d >= dim) break;
#pragma unroll
    for (int r = 0; r < kRowsPerCta; ++r)
      if (r < R) rec[2 * kRowsPerCta + r * dim + d] = acc[u][r];
  }
}

// Joins the splits of unit (blockIdx.x, blockIdx.y): thread = channel, the rows in turn.
template <typename T, int KEYS>
__global__ void __launch_bounds__(kMaxDim) kv8_attn_join_kernel(AnyArgs g) {
  const AttnArgs& a = g.a;
  const int dim = a.c.dim, d = threadIdx.x;
  const int kvh = blockIdx.y / g.chunks, chunk = blockIdx.y - kvh * g.chunks;
  const int h0 = kvh * a.group + chunk * g.head_chunk;
  const int nh = min(g.head_chunk, a.group - chunk * g.head_chunk);
  int64_t row0 = blockIdx.x, tokens = 1;
  if (KEYS == kExtend) {
    const ExtendEntry x = extend_tile(a, blockIdx.x, g.tile_tokens, 1, nullptr);
    if (x.entry < 0) return;
    row0 = x.row0 + x.tile * g.tile_tokens;
    tokens = min((int64_t)g.tile_tokens, x.n - x.tile * g.tile_tokens);
  }
  const float* rec = a.part + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * g.splits * any_record(dim);
  for (int r = 0; r < (int)tokens * nh; ++r) {
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int s = 0; s < g.splits; ++s) m = fmaxf(m, rec[s * any_record(dim) + 2 * r]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int s = 0; s < g.splits; ++s) {
      const float* p = rec + s * any_record(dim);
      const float w = exp2f(p[2 * r] - base);
      l = fmaf(w, p[2 * r + 1], l);
      if (d < dim) o = fmaf(w, p[2 * kRowsPerCta + r * dim + d], o);
    }
    if (d < dim) {
      T* out = static_cast<T*>(a.out) + (row0 + r / nh) * a.out_stride + (int64_t)(h0 + r % nh) * dim;
      Elem<T>::store(out + d, l == 0.f ? 0.f : o / l);
    }
  }
}

AnyArgs any_shape(const AttnArgs& a, int keys) {
  AnyArgs g{};
  g.a = a;
  g.head_chunk = a.group < kRowsPerCta ? a.group : kRowsPerCta;
  g.chunks = (a.group + g.head_chunk - 1) / g.head_chunk;
  g.tile_tokens = keys == kExtend ? kRowsPerCta / g.head_chunk : 1;
  return g;
}
int64_t any_tiles(const AnyArgs& g, int keys, int bs, int64_t tokens) {
  return keys == kExtend ? (tokens + g.tile_tokens - 1) / g.tile_tokens + bs : bs;
}
// Stretches of the keys: about four CTAs per SM over the whole launch.
int any_splits(const AnyArgs& g, int64_t tiles, int kv_heads, int64_t max_keys) {
  const int64_t units = tiles * kv_heads * g.chunks;
  int64_t s = units > 0 ? (4 * (int64_t)device_sm_count() + units - 1) / units : 1;
  const int64_t most = (max_keys + 4 * kTileKeys - 1) / (4 * kTileKeys);  // no stretch below four tiles
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

template <typename T, int KEYS>
int launch_any(AnyArgs g, int64_t tiles, cudaStream_t s) {
  static SmemLimit limit;
  const size_t smem = any_smem(g.a.c.dim);
  const int rc = limit.ensure((const void*)kv8_attn_any_kernel<T, KEYS>, smem);
  if (rc != QQ_OK) return rc;
  const dim3 grid((unsigned)tiles, g.a.c.kv_heads * g.chunks, g.splits);
  kv8_attn_any_kernel<T, KEYS><<<grid, kAnyThreads, smem, s>>>(g);
  if (g.splits > 1)
    kv8_attn_join_kernel<T, KEYS><<<dim3(grid.x, grid.y), (g.a.c.dim + 31) / 32 * 32, 0, s>>>(g);
  return launch_status();
}

int run(const AttnArgs& a, int keys, int dtype, int64_t max_keys, size_t ws_bytes, cudaStream_t s) {
  if (keys != kExtend && decode_tc_fits(a, dtype)) return run_decode_tc(a, keys, max_keys, ws_bytes, s);
  if (keys == kExtend && extend_tc_fits(a, dtype)) return run_extend_tc(a, max_keys, ws_bytes, s);
  AnyArgs g = any_shape(a, keys);
  const int64_t tiles = any_tiles(g, keys, a.bs, a.tokens);
  if (tiles > INT32_MAX || (int64_t)a.c.kv_heads * g.chunks > 65535) return QQ_ERR_UNSUPPORTED;
  g.splits = any_splits(g, tiles, a.c.kv_heads, max_keys);
  if (g.splits > 1) {
    const size_t need =
        sizeof(float) * (size_t)(tiles * a.c.kv_heads * g.chunks * g.splits * any_record(a.c.dim));
    if (a.part == nullptr || ws_bytes < need) return QQ_ERR_WORKSPACE;
  }
  if (dtype == QQ_BF16)
    return keys == kTable  ? launch_any<__nv_bfloat16, kTable>(g, tiles, s)
           : keys == kRows ? launch_any<__nv_bfloat16, kRows>(g, tiles, s)
                           : launch_any<__nv_bfloat16, kExtend>(g, tiles, s);
  return keys == kTable  ? launch_any<float, kTable>(g, tiles, s)
         : keys == kRows ? launch_any<float, kRows>(g, tiles, s)
                         : launch_any<float, kExtend>(g, tiles, s);
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
  g.splits = any_splits(g, tiles, a.c.kv_heads, max_keys);
  size_t need = 0;
  if (g.splits > 1)
    need = sizeof(float) * (size_t)(tiles * a.c.kv_heads * g.chunks * g.splits * any_record(a.c.dim));
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
  if (batch->bs > QQ_MAX_BS || table_stride > INT32_MAX / kv8::kMaxBlock) return QQ_ERR_UNSUPPORTED;
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

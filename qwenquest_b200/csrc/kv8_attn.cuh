// What the attention kernels over the 8-bit block cache share: their
// arguments, and how a key's place and a row's output are found.
#pragma once

#include <atomic>

#include "kv8.cuh"

namespace qq {
namespace kv8 {

// Which keys a batch entry attends to.
enum Keys : int {
  kTable = 0,   // one query token per entry, positions [0, seq) through the block table
  kRows = 1,    // one query token per entry, the listed rows
  kExtend = 2,  // an entry's new tokens, causal, through the block table
};

struct AttnArgs {
  Cache c;
  int bs;
  const int64_t* reqs;     // kTable, kExtend
  const int64_t* seq;      // kTable, kExtend: keys of the entry
  const int64_t* prefix;   // kExtend: keys before the new tokens
  const int64_t* offsets;  // kExtend: first query row of each entry
  const int32_t* table;    // [table_rows][table_stride]
  int64_t table_stride, table_rows;
  const int32_t* rows;     // kRows: [bs][rows_stride]
  int64_t rows_stride;
  const int32_t* lens;     // kRows
  int top;                 // kRows: listed rows per entry at most
  int64_t tokens;          // query rows
  const void* q;
  int64_t q_stride;        // elements between query rows
  void* out;
  int64_t out_stride;
  int heads, group;
  float scale_log2;        // scaling * log2(e)
  float* part;             // split partials
  uint32_t* err;
};

__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// The keys of one-token entry `e`; 0 when there is nothing to attend to (a
// bad entry is reported by the caller that passes err and attends to nothing).
template <int KEYS>
__device__ __forceinline__ int64_t entry_keys(const AttnArgs& a, int e, uint32_t* err) {
  if (KEYS == kRows) {
    const int32_t n = a.lens[e];
    if (n >= 0 && n <= a.top) return n;
    raise_error(err, QQ_DEV_ERR_BOUNDS);
    return 0;
  }
  const int64_t n = a.seq[e], r = a.reqs[e];
  if (n == 0) return 0;  // a padding entry
  if (n > 0 && n <= a.table_stride << a.c.shift && r >= 0 && r < a.table_rows) return n;
  raise_error(err, QQ_DEV_ERR_BOUNDS);
  return 0;
}

// An extend entry's query tile: `n` new tokens at rows `row0`, keys before them `prefix`.
struct ExtendEntry {
  int entry;      // -1: no such tile
  int64_t tile;   // which tile of the entry
  int64_t row0, n, prefix;
};

// Entry `e` of an extend batch: its new tokens (0: a padding or a bad entry, which is reported), its first query row
// and the keys before it.
__device__ __forceinline__ int64_t extend_entry(const AttnArgs& a, int e, int64_t& row0, int64_t& pre, uint32_t* err) {
  if (e >= a.bs) return 0;
  const int64_t seq = a.seq[e], req = a.reqs[e];
  row0 = a.offsets[e];
  pre = a.prefix[e];
  if (seq == 0) return 0;
  const int64_t n = seq - pre;
  if (pre >= 0 && n >= 0 && row0 >= 0 && row0 <= a.tokens && n <= a.tokens - row0 && seq <= a.table_stride << a.c.shift &&
      req >= 0 && req < a.table_rows)
    return n;
  raise_error(err, QQ_DEV_ERR_BOUNDS);
  return 0;
}

// The batch's tiles of `rows` rows each, `per` rows to a new token; called by one whole warp.
__device__ __forceinline__ int64_t extend_tiles(const AttnArgs& a, int rows, int per, uint32_t* err) {
  int64_t sum = 0, row0, pre;
#pragma unroll 2
  for (int e = threadIdx.x & 31; e < a.bs; e += 32) sum += (extend_entry(a, e, row0, pre, err) * per + rows - 1) / rows;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// Tile `x` of those; called by one whole warp, the same in every lane.
__device__ __forceinline__ ExtendEntry extend_tile(const AttnArgs& a, int64_t x, int rows, int per, uint32_t* err) {
  ExtendEntry r{-1, 0, 0, 0, 0};
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int e0 = 0; e0 < a.bs; e0 += 32) {
    int64_t row0 = 0, pre = 0;
    const int64_t n = extend_entry(a, e0 + lane, row0, pre, err);
    const int64_t tiles = (n * per + rows - 1) / rows;
    int64_t incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const int64_t excl = before + incl - tiles;
    const uint32_t m = __ballot_sync(0xffffffffu, x >= excl && x < excl + tiles);
    if (m != 0) {
      const int src = __ffs(m) - 1;
      r.entry = e0 + src;
      r.tile = x - __shfl_sync(0xffffffffu, excl, src);
      r.row0 = __shfl_sync(0xffffffffu, row0, src);
      r.n = __shfl_sync(0xffffffffu, n, src);
      r.prefix = __shfl_sync(0xffffffffu, pre, src);
      return r;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

// The slot of key `j` of entry `e`, -1 when it takes no part (a bad block or row is reported).
template <int KEYS>
__device__ __forceinline__ int64_t key_slot(const AttnArgs& a, int e, int64_t req, int64_t j, uint32_t* err) {
  if (KEYS == kRows) {
    const int32_t r = a.rows[(int64_t)e * a.rows_stride + j];
    if (r < 0) return -1;  // a padding row
    if (r < (int64_t)a.c.num_blocks << a.c.shift) return r;
  } else {
    const int32_t b = a.table[req * a.table_stride + (j >> a.c.shift)];
    if (b >= 0 && b < a.c.num_blocks) return ((int64_t)b << a.c.shift) | (j & (a.c.block - 1));
  }
  raise_error(err, QQ_DEV_ERR_BOUNDS);
  return -1;
}

// ---------------------------------------------------------------- clusters

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Word `addr` of the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float ld_cluster(uint32_t addr, int rank) {
  float x;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}\n"
               : "=f"(x)
               : "r"(addr), "r"(rank)
               : "memory");
  return x;
}

// A launch by clusters of `cluster` CTAs.
struct ClusterLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  ClusterLaunch(dim3 grid, dim3 cluster, int threads, size_t smem, cudaStream_t s) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster.x;
    attr[0].val.clusterDim.y = cluster.y;
    attr[0].val.clusterDim.z = cluster.z;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
  }
};

// How many clusters of a kernel the current device holds at a time (0: none),
// asked once per device, with `smem` bytes each; `most` is what any launch of it uses.
class ResidentClusters {
 public:
  int ask(const void* kernel, dim3 cluster, int threads, size_t smem, size_t most) {
    const int d = current_device();
    if (d < 0 || d >= kMaxDevices) return 0;
    int n = known_[d].load(std::memory_order_acquire);
    if (n > 0) return n - 1;
    n = 0;
    ClusterLaunch l(cluster, cluster, threads, smem, nullptr);
    l.cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &l.cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    known_[d].store(n + 1, std::memory_order_release);
    return n;
  }

 private:
  std::atomic<int> known_[kMaxDevices] = {};  // one more than the number
};

// The tensor-core kernel for one query token per entry (kTable, kRows): whether
// it takes these arguments, the scratch it needs, and its launch.
bool decode_tc_fits(const AttnArgs& a, int dtype);
size_t decode_tc_workspace(int bs, int kv_heads, int group, int64_t max_keys);
int run_decode_tc(const AttnArgs& a, int keys, int64_t max_keys, size_t ws_bytes, cudaStream_t s);
// The same for an extend batch.
bool extend_tc_fits(const AttnArgs& a, int dtype);
size_t extend_tc_workspace(int bs, int kv_heads, int group, int64_t tokens, int64_t max_keys);
int run_extend_tc(const AttnArgs& a, int64_t max_keys, size_t ws_bytes, cudaStream_t s);

}  // namespace kv8
}  // namespace qq

// Tensor maps over the codes of an 8-bit block cache, and the split of an
// operand into two e4m3 numbers.
#pragma once

#include "kv8_attn.cuh"
#include "tcgen05.cuh"

namespace qq {
namespace kv8 {

constexpr int kTcDim = 128;  // head_dim of the tensor-core kernels: one 128-byte row per token and head

// The codes as rows of 128 bytes ([block][head][token]), copied `box_rows` rows
// at a time into the 128-byte-swizzled layout the matrix descriptors name.
// The encoder is a function of the driver, looked up once.
inline int encode_rows(CUtensorMap* map, const void* codes, int64_t rows, int box_rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> cached{nullptr};
  Encode encode = cached.load(std::memory_order_acquire);
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) !=
            cudaSuccess ||
        fn == nullptr)
      return QQ_ERR_CUDA;
    encode = reinterpret_cast<Encode>(fn);
    cached.store(encode, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {kTcDim, (cuuint64_t)rows}, strides[1] = {kTcDim};
  const cuuint32_t box[2] = {kTcDim, (cuuint32_t)box_rows}, steps[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? QQ_OK
             : QQ_ERR_CUDA;
}

// Byte `col` (0..127) of row `r` of a tile of 128-byte rows in the 128-byte-swizzled layout.
__device__ __forceinline__ uint32_t swz(int r, int col) {
  return (uint32_t)(r * 128 + (((col >> 4) ^ (r & 7)) << 4) + (col & 15));
}

// Two fp32 values as pairs hi + lo / kLo of e4m3 numbers (each result holds
// two codes).  e4m3 has 4 significant bits, so hi + lo carries 8, as many as
// bf16: off by half a step of half a step, 2^-8 of the value, or 2^-10 / kLo
// where lo leaves the type's normal range.
__device__ __forceinline__ void split_e4m3x2(float x0, float x1, float lo_scale, uint32_t& hi, uint32_t& lo) {
  hi = e4m3x2(x0, x1);
  const float2 h = from_e4m3x2(hi);
  lo = e4m3x2((x0 - h.x) * lo_scale, (x1 - h.y) * lo_scale);
}

// 2^k, the largest power of two that keeps amax * 2^k <= 448 and k within +-120 (amax 0: 2^120).
__device__ __forceinline__ int fit_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7);
  return max(-120, min(120, -e));
}
__device__ __forceinline__ float exp2_int(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

}  // namespace kv8
}  // namespace qq

// Shared pieces of the 8-bit block KV cache (e4m3 codes, a scale per block of
// tokens and KV head): conversions, and the views its kernels take.
#pragma once

#include "common.cuh"

namespace qq {
namespace kv8 {

constexpr int kMaxBlock = 128;   // tokens per block: 16, 32, 64 or 128
constexpr int kMaxDim = 256;     // head_dim: a multiple of 8

// The views a launch takes by value.
struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  uint32_t* state;
  int num_blocks;
  int kv_heads;
  int dim;
  int block;
  int shift;  // log2(block)
};

// The default limit of 48 KiB counts a kernel's own shared arrays too, so the
// launches ask for this much more than their dynamic part.
constexpr size_t kStaticSmem = 4096;

inline Cache view(const qq_kv8_cache& c) {
  int shift = 0;
  while ((1 << shift) < c.block_size) ++shift;
  return Cache{c.k, c.v, c.k_scale, c.v_scale, c.state, c.num_blocks, c.kv_heads, c.head_dim, c.block_size, shift};
}

// QQ_OK, or what is wrong with a cache's description.
inline int check(const qq_kv8_cache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr ||
      c->num_blocks <= 0 || c->kv_heads <= 0 || c->head_dim <= 0)
    return QQ_ERR_INVALID;
  if ((c->block_size != 16 && c->block_size != 32 && c->block_size != 64 && c->block_size != 128) ||
      c->head_dim % 8 != 0 || c->head_dim > kMaxDim || c->kv_heads > 65535 ||
      (int64_t)c->num_blocks * c->block_size > INT32_MAX ||
      (int64_t)c->num_blocks * c->kv_heads * c->block_size > INT32_MAX ||
      reinterpret_cast<uintptr_t>(c->k) % 16 != 0 || reinterpret_cast<uintptr_t>(c->v) % 16 != 0)
    return QQ_ERR_UNSUPPORTED;
  return QQ_OK;
}

// Two fp32 values as e4m3 codes (lo in the lower byte), to nearest even; past +-448 the largest value, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 codes as fp32 values (exact).
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ void from_e4m3x8(uint2 w, float (&x)[8]) {
  const uint32_t h[4] = {w.x & 0xFFFFu, w.x >> 16, w.y & 0xFFFFu, w.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = from_e4m3x2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Eight consecutive elements of a row (16-byte aligned for bf16, 32 for fp32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
  *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ int32_t ld_volatile_s32(const int32_t* p) {
  return (int32_t)ld_volatile_u32(reinterpret_cast<const uint32_t*>(p));
}

}  // namespace kv8
}  // namespace qq

// kvpool.cuh — slot plans and the fused norm / rotation / store of queries and
// keys (see kvpool.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gsec {

// 16 bytes of T as floats and back (rounded to nearest once).
template <typename T>
struct Vec16;
template <>
struct Vec16<__nv_bfloat16> {
  static constexpr bool bf16 = true;
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bf16 is the high half of its float
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
  }
};
template <>
struct Vec16<__half> {
  static constexpr bool bf16 = false;
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
  }
};
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Most requests of one slot plan: three int32 per request in shared memory.
constexpr int kPlanMaxBatch = 16384;

struct SlotPlanArgs {
  const int32_t* lens;      // tokens of request i already in the pool
  const int32_t* fresh;     // new tokens of request i
  int batch;
  int32_t* table;           // [batch, width] pages, row pitch in elements
  int64_t table_pitch;
  int width;
  const int32_t* free_pages;
  int64_t nfree;
  const int32_t* cursor;    // pages of the free list already taken
  int page;
  FastDiv page_div;
  int32_t base;             // added to every position
  int64_t* slots;           // [capacity]
  int32_t* positions;       // [capacity]
  int64_t capacity;
  int32_t* cu;              // [batch + 1]
  int32_t* lens_out;        // [batch]
  int32_t* cursor_out;      // [1]
};

struct QkStoreArgs {
  const char* qkv;          // [tokens, (hq + 2 hk) * dim], row pitch in bytes
  int64_t qkv_pitch;
  int64_t tokens;
  int hq, hk, dim;
  char* q_out;              // [tokens, hq, dim]
  char* pool;               // slot records: pitch bytes, V at + plane
  int64_t pitch, plane, pool_rows;
  const void* slots;        // int32 or int64
  const void* positions;
  int slot_bytes, position_bytes;
  const float* cos;         // [max_pos, rot / 2]
  const float* sin;
  int rot;
  int64_t max_pos;
  const void* q_weight;     // [dim] or null
  const void* k_weight;
  float eps;
  int interleaved;
  FastDiv part_div;         // groups of heads per token
  float inv_dim;
};

int slots_plan(const SlotPlanArgs& a, cudaStream_t s);
int qk_norm_rope_store(const QkStoreArgs& a, int dtype, cudaStream_t s);
// Status bits of this file's kernels, at their place in the layout byte.
unsigned kvpool_device_status(bool clear);

}  // namespace gsec

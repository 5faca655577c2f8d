// Rows of logits over a vocabulary: addressing, element access, the order of entries, sums over a CTA.
#pragma once
#include "gdn_common.cuh"
#include "rowio.cuh"

namespace gdn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename Args>
__device__ __forceinline__ int64_t row_offset(const Args& a, int64_t r) {
  return (r / a.inner) * a.stride_outer + (r % a.inner) * a.stride_inner;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// an index as int32 or int64; whatever lies outside [0, V) is -1
__device__ __forceinline__ int load_index(const void* p, int64_t i, int bytes, int V) {
  const int64_t v = bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
  return v >= 0 && v < V ? (int)v : -1;
}

// Entries in the order of top_ids as integers: the larger value first (NaN above infinity, the zeros equal), then the lower index.
// 0 is below every entry's key.
__device__ __forceinline__ uint64_t entry_key(float x, int index) {
  uint32_t b = __float_as_uint(x);
  if (x != x) b = 0x7fc00000u;
  if (x == 0.f) b = 0u;
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((uint64_t)b << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct SumOf {
  template <typename T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct MaxOf {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
// the whole CTA's value, to every thread; `scratch` has a place for each warp and is free again on return
template <int NT, typename T, typename Op>
__device__ __forceinline__ T cta_reduce(T v, T* scratch, Op op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = scratch[lane % (NT / 32)];
#pragma unroll
  for (int o = NT / 64; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  return v;
}

}  // namespace gdn

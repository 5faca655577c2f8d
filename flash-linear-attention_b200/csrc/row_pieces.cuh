// Rows of any width in pieces of N elements a thread: loads and stores as wide as a piece, arithmetic by fp32 pairs, parameters in the
// caller's type, sums over the threads that share a row.
#pragma once
#include "gdn_common.cuh"
#include "rowio.cuh"

namespace gdn {

// ---- pieces of N elements ------------------------------------------------------------------------------------------------
template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// Arithmetic goes by fp32 pairs (f32x2: two operations in one instruction).  A piece of one element is a pair whose second half is zero
// and stays zero: what is spread over a pair is zero there too.
constexpr int pairs(int n) { return (n + 1) / 2; }
template <int N>
__device__ __forceinline__ uint64_t spread(float x) { return pack2(x, N == 1 ? 0.f : x); }
__device__ __forceinline__ float both(uint64_t x) {
  const float2 f = unpack2(x);
  return f.x + f.y;
}

template <typename T, int N>
struct Vec {
  typename Raw<sizeof(T) * N>::type u;
  __device__ __forceinline__ void load(const void* base, int64_t at) { u = *reinterpret_cast<const decltype(u)*>(static_cast<const T*>(base) + at); }
  __device__ __forceinline__ void store(void* base, int64_t at) const { *reinterpret_cast<decltype(u)*>(static_cast<T*>(base) + at) = u; }
  __device__ __forceinline__ void again() {   // what was made of it is not kept
    if constexpr (sizeof(u) == 16) asm volatile("" : "+r"(u.x), "+r"(u.y), "+r"(u.z), "+r"(u.w));
  }
  __device__ __forceinline__ uint64_t pair(int i) const {
    if constexpr (N == 1) {
      return pack2((float)*reinterpret_cast<const T*>(&u), 0.f);
    } else if constexpr (sizeof(T) == 2) {
      return widen2<T>(reinterpret_cast<const uint32_t*>(&u)[i]);
    } else {
      const float* f = reinterpret_cast<const float*>(&u);
      return pack2(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set(int i, uint64_t x) {
    const float2 f = unpack2(x);
    if constexpr (N == 1) {
      *reinterpret_cast<T*>(&u) = static_cast<T>(f.x);
    } else if constexpr (sizeof(T) == 2) {
      reinterpret_cast<uint32_t*>(&u)[i] = narrow2<T>(x);
    } else {
      reinterpret_cast<float*>(&u)[2 * i] = f.x;
      reinterpret_cast<float*>(&u)[2 * i + 1] = f.y;
    }
  }
};

// N parameters from column d on; `absent` where there are none
template <int N>
__device__ __forceinline__ void load_params(const void* p, int dtype, int d, float absent, uint64_t (&x)[pairs(N)]) {
  auto take = [&](auto v) {
    v.load(p, d);
#pragma unroll
    for (int i = 0; i < pairs(N); ++i) x[i] = v.pair(i);
  };
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < pairs(N); ++i) x[i] = spread<N>(absent);
  } else if (dtype == B200GDN_F32) {
    if constexpr (N == 8) {
      Vec<float, 4> lo, hi;
      lo.load(p, d);
      hi.load(p, d + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = i < 2 ? lo.pair(i) : hi.pair(i - 2);
    } else {
      take(Vec<float, N>());
    }
  } else if (dtype == B200GDN_BF16) {
    take(Vec<__nv_bfloat16, N>());
  } else {
    take(Vec<__half, N>());
  }
}

template <int WIDTH, int COUNT>
__device__ __forceinline__ void shuffle_sums(float (&v)[COUNT]) {   // over WIDTH neighbouring lanes, to all of them
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}
// The sums over the TPR threads that share a row, to all of them.  `scratch`: [COUNT][TPR / 32], not to be written again before everyone
// has passed the next call's barrier.
template <int TPR, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], float* scratch) {
  shuffle_sums<(TPR < 32 ? TPR : 32)>(v);
  if constexpr (TPR > 32) {
    constexpr int NW = TPR / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < COUNT; ++i) scratch[i * NW + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = scratch[i * NW + (lane & (NW - 1))];
    shuffle_sums<NW>(v);
  }
}

}  // namespace gdn

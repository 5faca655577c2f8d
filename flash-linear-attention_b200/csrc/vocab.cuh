// Rows of logits over a vocabulary: addressing, element access, the order of entries, sums over a CTA.
#pragma once
#include "gdn_common.cuh"
#include "rowio.cuh"

namespace gdn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename Args>
__device__ __forceinline__ int64_t row_offset(const Args& a, int64_t r) {
  if (r < a.inner) return r * a.stride_inner;   // the usual case, without a division
  return (r / a.inner) * a.stride_outer + (r % a.inner) * a.stride_inner;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Exponents of two: 2^u is an entry's weight beside m, the largest entry of some part of its row, c = scale log2(e).  The difference
// first: it is exact for what counts, is 0 at m, and leaves fp32's range only where the weight is zero.  m = -infinity (nothing above
// it yet) counts as 0.
__device__ __forceinline__ float exponent(float x, float m, float c) { return (x - (m == -INFINITY ? 0.f : m)) * c; }

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

// ---- running maximum and sums ----------------------------------------------------------------------------------------
// m: the largest entry (-infinity: none yet);  s = sum 2^u, t = sum u 2^u with the exponents u beside m
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ Sums moved(Sums a, float m, float c) {   // the same sums beside another, larger m
  if (a.m == -INFINITY) return {m, a.s, a.t};   // of no entries above -infinity: zeros, or NaN with NaN among them
  const float d = (a.m - m) * c, f = exp2_approx(d);
  return {m, a.s * f, f == 0.f ? 0.f : f * (a.t + d * a.s)};
}
__device__ __forceinline__ float warp_max(float x) {   // (NaN is left out)
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(y) : "f"(x));
  return y;
}
template <bool WITH_T>
__device__ __forceinline__ Sums warp_sums(Sums a, float c) {
  a = moved(a, warp_max(a.m), c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if constexpr (WITH_T) a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  return a;
}

// the larger of two words' elements, pair by pair (what is NaN is left out), and the largest of a word of pairs
template <typename T>
__device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}
template <typename T>
__device__ __forceinline__ float max_of_word(uint32_t a) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(a);
  else {
    const float2 f = unpack2(widen2<T>(a));
    return fmaxf(f.x, f.y);
  }
}
template <typename T>
constexpr uint32_t kMinusInfWord = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;

// elements 2 i, 2 i + 1 of a 16-byte word as an fp32 pair
template <typename T>
__device__ __forceinline__ uint64_t pair_of(const uint4& w, int i) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (sizeof(T) == 2) return widen2<T>(u[i]);
  else return pack2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
}

// the largest entries of a 16-byte word, as max_words leaves them
template <typename T>
__device__ __forceinline__ uint32_t largest_of(const uint4& w) {
  if constexpr (sizeof(T) == 4) {
    float m;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(m) : "f"(__uint_as_float(w.x)), "f"(__uint_as_float(w.y)), "f"(__uint_as_float(w.z)));
    return __float_as_uint(fmaxf(m, __uint_as_float(w.w)));
  } else {
    return max_words<T>(max_words<T>(w.x, w.y), max_words<T>(w.z, w.w));
  }
}

// One thread's running sums.  A group of words at a time: their largest entry first, so that the sums are moved seldom.  Per pair of
// 16-bit entries the arithmetic is one operation for the largest, two to widen, two for the exponents, two exponentials, one to add and one
// more for the entropy; with moves, loads and the joining of lanes the kernel was counted at 8.0 instructions an entry.  (At the memory's
// rate an SM gets 11.7 entries of 16 bits a clock, for which it can issue 128 instructions; the exponentials' unit takes 16.)
// BOUNDED: u is at least -2^10, of entries whose 2^u is zero long before: 0 x -infinity is no number.
template <typename T, bool WITH_T>
struct PieceSums {
  static constexpr int PAIRS = sizeof(T) == 2 ? 4 : 2;
  Sums a{-INFINITY, 0.f, 0.f};
  uint64_t s2 = 0ull, t2 = 0ull, s3 = 0ull, t3 = 0ull, m2 = 0ull;   // two running sums each, of pairs; minus the largest

  __device__ __forceinline__ void flush() {
    const float2 s = unpack2(add2(s2, s3)), t = unpack2(add2(t2, t3));
    a.s = s.x + s.y;
    a.t = t.x + t.y;
  }
  template <bool BOUNDED, int N>
  __device__ __forceinline__ void add(const uint4 (&w)[N], float c) {
    uint32_t top = largest_of<T>(w[0]);
#pragma unroll
    for (int g = 1; g < N; ++g) top = max_words<T>(top, largest_of<T>(w[g]));
    const float m = max_of_word<T>(top);
    if (m > a.m) {
      flush();
      a = moved(a, m, c);
      s2 = pack2(a.s, 0.f);
      t2 = pack2(a.t, 0.f);
      s3 = t3 = 0ull;
      m2 = pack2(-m, -m);
    }
    if (!(BOUNDED && WITH_T)) {
      const uint64_t c2 = pack2(c, c);
#pragma unroll
      for (int g = 0; g < N; ++g)
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const uint64_t u2 = mul2(add2(pair_of<T>(w[g], i), m2), c2);
          const float2 u = unpack2(u2);
          const uint64_t e2 = pack2(exp2_approx(u.x), exp2_approx(u.y));
          if (i & 1) s3 = add2(s3, e2);
          else s2 = add2(s2, e2);
          if constexpr (WITH_T) {
            if (i & 1) t3 = fma2(e2, u2, t3);
            else t2 = fma2(e2, u2, t2);
          }
        }
    } else {
#pragma unroll 1
      for (int g = 0; g < N; ++g) {
        uint4 q = w[0];
#pragma unroll
        for (int o = 1; o < N; ++o)
          if (g == o) q = w[o];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const float2 x = unpack2(pair_of<T>(q, i));
          const float u0 = exponent(x.x, a.m, c), u1 = exponent(x.y, a.m, c), e0 = exp2_approx(u0), e1 = exp2_approx(u1);
          s2 = add2(s2, pack2(e0, e1));
          if constexpr (WITH_T) t2 = fma2(pack2(e0, e1), pack2(fmaxf(u0, -1024.f), fmaxf(u1, -1024.f)), t2);
        }
      }
    }
  }
};

// ---- spans -------------------------------------------------------------------------------------------------------------
constexpr int kSpanWarps = 4;

// How rows are cut: `w` words a lane, for as many words of 16 bytes as a row has at most (off a word's boundary it has one more).  By the
// width alone: a row's results are the same bits whatever rows it comes with.
struct Spans {
  int w, per_row;   // w: a power of two
  __device__ __forceinline__ int shift() const { return 31 - __clz(w); }
  __host__ __device__ int groups() const { return 32 * per_row; }
};
inline Spans spans_of(int V, int size) {
  const int64_t words = ((int64_t)V * size + 15) / 16 + 1;
  int w = 8;
  while (w > 1 && words <= 16 * w) w >>= 1;   // short rows: no more lanes without words than have to be
  return Spans{w, (int)((words + 32 * w - 1) / (32 * w))};
}

// A row by words: word j holds the entries from first + j EPW on; the first and the last may hold something else beside (every word that is
// read holds an entry of the row, so no read leaves the 16 bytes that hold one).
template <typename T>
struct Words {
  static constexpr int EPW = 16 / sizeof(T);
  const uint4* at;
  int first, n;
  __device__ __forceinline__ Words(const T* row, int V) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(row);
    const int shift = (int)(b & 15) / (int)sizeof(T);
    at = reinterpret_cast<const uint4*>(b & ~(uintptr_t)15);
    first = -shift;
    n = (shift + V + EPW - 1) / EPW;
  }
  // word j with minus infinity for what is not of the row
  __device__ __forceinline__ uint4 edge(int j, int V) const {
    uint4 q = at[j];
    T* x = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int e = 0; e < EPW; ++e) {
      const int i = first + j * EPW + e;
      if (i < 0 || i >= V) x[e] = static_cast<T>(-INFINITY);
    }
    return q;
  }
};

// A span's words in a warp's registers: word i of lane l is word (32 W span) + 32 i + l of the row; minus infinity for what is not of it.
template <typename T, int W>
struct SpanWords {
  uint4 q[W];
  int j0;       // of this lane
  bool inner;   // nothing but entries
  __device__ __forceinline__ SpanWords(const Words<T>& x, int V, int span, int lane) {
    j0 = span * 32 * W + lane;
    inner = (span > 0 || x.first == 0) && ((span + 1) * 32 * W < x.n || ((span + 1) * 32 * W == x.n && x.first + x.n * Words<T>::EPW == V));
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int j = j0 + 32 * i;
      if (inner) q[i] = x.at[j];
      else if (j < x.n) q[i] = x.edge(j, V);
      else q[i] = make_uint4(kMinusInfWord<T>, kMinusInfWord<T>, kMinusInfWord<T>, kMinusInfWord<T>);
    }
  }
  // this lane's sums
  template <bool WITH_T>
  __device__ __forceinline__ Sums sums(float c) const {
    PieceSums<T, WITH_T> p;
    constexpr int G = W < 4 ? W : 4;
    bool bounded = !inner;
    if (inner) {
#pragma unroll
      for (int i = 0; i < W; i += G) {
        uint4 w[G];
#pragma unroll
        for (int g = 0; g < G; ++g) w[g] = q[i + g];
        p.template add<false>(w, c);
      }
      p.flush();
      // entries of minus infinity: once more, with bounded exponents
      bounded = WITH_T && p.a.t != p.a.t && p.a.s == p.a.s;
    }
    if (bounded) {
      p = PieceSums<T, WITH_T>();
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint4 w[1] = {q[i]};
        p.template add<true>(w, c);
      }
      p.flush();
    }
    return p.a;
  }
};

// A row's spans joined; a whole warp.
__device__ __forceinline__ Sums joined_spans(const float4* part, int n, float c, int lane) {
  Sums v{-INFINITY, 0.f, 0.f};
  for (int i = lane; i < n; i += 32) {
    const float4 f = part[i];
    const Sums o{f.x, f.y, f.z};
    const float m = fmaxf(v.m, o.m);
    const Sums p = moved(o, m, c);
    v = moved(v, m, c);
    v.s += p.s;
    v.t += p.t;
  }
  return warp_sums<true>(v, c);
}

// ---- gradients: a span of dlogits ----------------------------------------------------------------------------------------
// Words of dlogits, each written by one lane: f(x) of the entry's logit.  Where a row of dlogits lies in its words as the row of logits does,
// logits are read by words as well, else entry by entry.
template <typename T, int W>
struct GradientSpan {
  static constexpr int EPW = Words<T>::EPW;
  uint4 q[W];
  // (as SpanWords: word i of lane l is word (32 W span) + 32 i + l)
  __device__ __forceinline__ void load(const T* row, const T* out, int V, int span, int lane) {
    const Words<T> y(out, V);
    const bool alike = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int j = span * 32 * W + lane + 32 * i;
      if (j >= y.n) continue;
      if (alike) {
        q[i] = src[j];
      } else {
        T* x = reinterpret_cast<T*>(&q[i]);
#pragma unroll
        for (int e = 0; e < EPW; ++e) {
          const int at = y.first + j * EPW + e;
          x[e] = at >= 0 && at < V ? row[at] : static_cast<T>(0.f);
        }
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void store(T* out, int V, int span, int lane, F f) const {
    const Words<T> y(out, V);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int j = span * 32 * W + lane + 32 * i, at = y.first + j * EPW;
      if (j >= y.n) continue;
      uint32_t g[4];
#pragma unroll
      for (int e = 0; e < EPW / 2; ++e) {
        const uint64_t d = f(pair_of<T>(q[i], e));
        if constexpr (sizeof(T) == 2) {
          g[e] = narrow2<T>(d);
        } else {
          const float2 p = unpack2(d);
          g[2 * e] = __float_as_uint(p.x);
          g[2 * e + 1] = __float_as_uint(p.y);
        }
      }
      const uint4 w = make_uint4(g[0], g[1], g[2], g[3]);
      if (at >= 0 && at + EPW <= V) {
        __stcs(const_cast<uint4*>(y.at) + j, w);
      } else {
        const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int e = 0; e < EPW; ++e)
          if (at + e >= 0 && at + e < V) out[at + e] = x[e];
      }
    }
  }
};
template <typename T, int W>
__device__ __forceinline__ void zero_span(T* out, int V, int span, int lane) {
  GradientSpan<T, W> z;
#pragma unroll
  for (int i = 0; i < W; ++i) z.q[i] = make_uint4(0u, 0u, 0u, 0u);
  z.store(out, V, span, lane, [](uint64_t x) { return x; });
}
// the entries that the words of a span of dlogits hold
template <typename T, int W>
__device__ __forceinline__ bool in_span(const T* out, int span, int j) {
  constexpr int EPW = Words<T>::EPW;
  const int word = (j + (int)(reinterpret_cast<uintptr_t>(out) & 15) / (int)sizeof(T)) / EPW;
  return j >= 0 && word / (32 * W) == span;
}

}  // namespace gdn

// Layer norm over rows of any width with the residual sum, forward and backward.
//     z = x + residual (rounded: what is handed on is what is normalised);  n = (z - mean) rstd;  y = n w + b
//     h = dy w;  dx = rstd (h - mean(h) - n mean(h n)) + dz;  dw = sum of dy n;  db = sum of dy
// HBM streaming: a row is read once into the registers of TPR threads, NV pieces each of N elements (16 bytes where width and addresses
// allow it, else two elements or one).  CTAs stay and walk the rows, so that a thread's columns stay its own: dw and db are sums in
// registers.  The next rows are on their way while the present ones are worked on.  What a row's threads have to agree on takes one
// barrier, forward as well: a warp's mean and the squares about it are joined to the row's, which loses nothing.  Each CTA of the
// backward pass leaves one partial row of dw and db, which a second kernel adds in a fixed order.
// What held the first forms back was instructions, not bytes: 24 an element with conversions one by one, scalar arithmetic, divisions
// and parameters converted row after row.
// Measured: 65536 x 4096 bf16 forward 180 us (164 at copy rate), backward 292 (246); 16384 x 2048 with a residual 50 (41) forward;
// 65536 x 1024 fp32 with a residual backward 173 (164); 32768 x 1001 bf16, two bytes at a time, 51 to 56 and 75 (20 and 30).  Beyond the
// registers, in several looks: 16384 x 8192 fp32 backward 880 (246), 8192 x 16384 bf16 954 (123).  Forward rows of 16-bit elements from
// 8193 on are held at the cost of spills: 8192 x 16384 155 (82), with a residual 346 (164).
#include "gdn_common.cuh"
#include "layer_norm_pieces.h"
#include "row_pieces.cuh"

namespace gdn {
namespace {

constexpr int threads_of(int tpr) { return tpr > 32 ? tpr : 128; }   // rows of several warps have a CTA to themselves
// forward, an SM's: by the registers of the rows on their way (NV pieces, with a residual twice that) and at work.  One or two pieces a thread:
// 7, with a residual 5, since at 8 rows spill (65536 x 256 bf16 with a residual 25 us at 5, 28 at 6, 36 at 8; 131072 x 100 fp32 without 25 at 7, 28 at 8)
// (with a residual there is more to move for the same arithmetic: the cache does: 16384 rows of 8192, 169 us, 192 with shared memory)
constexpr bool shares_params(int nv, int n, bool res) { return !res && n >= 4 && nv * n > 8 && nv <= 4; }
constexpr int fwd_ctas(int tpr, int nv, bool res) {
  return tpr > 32 ? 512 / threads_of(tpr) : nv >= 16 ? (res ? 2 : 3) : nv == 8 ? (res ? 3 : 4) : nv == 4 ? (res ? 5 : 6) : res ? 5 : 7;
}
constexpr int bwd_ctas(int tpr) { return tpr <= 32 ? 4 : tpr == 64 ? 8 : tpr == 128 ? 4 : tpr == 256 ? 2 : 1; }
constexpr int rows_at_once(int nv, int n) { return nv * n <= 4 ? 4 : nv == 1 ? 2 : 1; }   // of a group of TPR threads

// ---- forward -------------------------------------------------------------------------------------------------------------
template <typename T, int N, int TPR, int NV, bool RES>
__global__ void __launch_bounds__(threads_of(TPR), fwd_ctas(TPR, NV, RES)) layer_norm_fwd_kernel(const b200gdn_layer_norm_args a) {
  constexpr int RPC = threads_of(TPR) / TPR, R = rows_at_once(NV, N), NW = TPR > 32 ? TPR / 32 : 1;
  __shared__ float scratch[2][2 * R * NW];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR, lane = threadIdx.x & 31;
  // down: a power of two, down^2 in [1 / 4 D, 1 / D].  Products with it are exact, so one fused operation is (z - mean) down with one
  // rounding, and the sum of its squares is within range wherever the variance is; times `up` it is the variance.
  const float inv = 1.f / a.D, down = __int_as_float((127 - (33 - __clz(a.D - 1)) / 2) << 23), up = inv / (down * down);
  // Weight and bias as fp32 pairs: in registers where a thread has few columns, else in shared memory, where row after row finds them
  // without conversions (and without a bank conflict: 16 bytes a thread side by side); of very wide rows from the first-level cache.
  constexpr int P = pairs(N);
  constexpr bool HELD = NV * N <= (N <= 2 ? 16 : 8), SHARED = shares_params(NV, N, RES);
  constexpr bool LARGE = R * NV * N > 16;   // widened anew at each step; kept wide the rows would not fit the registers
  extern __shared__ __align__(16) ulonglong2 shared_params[];   // [2][P / 2][TPR NV]
  uint64_t w[HELD ? NV : 1][P], b[HELD ? NV : 1][P];
  if constexpr (HELD) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
#pragma unroll
      for (int i = 0; i < P; ++i) w[v][i] = b[v][i] = 0ull;
      if (d < a.D) {
        load_params<N>(a.weight, a.param_dtype, d, 1.f, w[v]);
        load_params<N>(a.bias, a.param_dtype, d, 0.f, b[v]);
      }
    }
  } else if constexpr (SHARED) {
    for (int q = threadIdx.x; q * N < a.D; q += threads_of(TPR)) {
      load_params<N>(a.weight, a.param_dtype, q * N, 1.f, w[0]);
      load_params<N>(a.bias, a.param_dtype, q * N, 0.f, b[0]);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        shared_params[i * TPR * NV + q] = make_ulonglong2(w[0][2 * i], w[0][2 * i + 1]);
        shared_params[(P / 2 + i) * TPR * NV + q] = make_ulonglong2(b[0][2 * i], b[0][2 * i + 1]);
      }
    }
    __syncthreads();
  }
  // elements that a warp holds of a row (for lane l: of warp l modulo NW)
  float held = a.D;
  if constexpr (TPR > 32) {
    int n = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) n += min(max(a.D - (v * TPR + (lane & (NW - 1)) * 32) * N, 0), 32 * N);
    held = n;
  }
  const float per_held = held > 0.f ? 1.f / held : 0.f, per_held_here = TPR > 32 ? __shfl_sync(0xffffffffu, per_held, threadIdx.x >> 5) : per_held;
  Vec<T, N> x[R][NV], res[RES ? R : 1][NV];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = r0 + r * RPC + group;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int d = (v * TPR + sub) * N;
        x[r][v].u = decltype(x[r][v].u){};
        if constexpr (RES) res[r][v].u = decltype(x[r][v].u){};
        if (row < a.rows && d < a.D) {
          x[r][v].load(a.x, row * a.D + d);
          if constexpr (RES) res[r][v].load(a.residual, row * a.D + d);
        }
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPC * R;
  int64_t r0 = (int64_t)blockIdx.x * RPC * R;
  fetch(r0);
  for (int turn = 0; r0 < a.rows; turn ^= 1) {
    const int64_t now = r0;
    Vec<T, N> z[R][NV];
    float s[R], q[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t sum = 0ull;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if constexpr (RES) {
#pragma unroll
          for (int i = 0; i < P; ++i) z[r][v].set(i, add2(x[r][v].pair(i), res[r][v].pair(i)));
        } else {
          z[r][v] = x[r][v];
        }
#pragma unroll
        for (int i = 0; i < P; ++i) sum = add2(sum, z[r][v].pair(i));   // (zeros beyond the row)
      }
      s[r] = both(sum);
    }
    r0 += step;
    fetch(r0);
    // the mean of what a warp (a row's lanes) holds, the squares about it, then the row's
    shuffle_sums<(TPR < 32 ? TPR : 32)>(s);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mean = s[r] * per_held_here;
      const uint64_t by = spread<N>(down), off = spread<N>(-mean * down);
      uint64_t sum = 0ull;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if ((v * TPR + sub) * N >= a.D) continue;
        if (LARGE) z[r][v].again();
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const uint64_t c = fma2(z[r][v].pair(i), by, off);
          sum = fma2(c, c, sum);
        }
      }
      q[r] = both(sum) * up;
    }
    shuffle_sums<(TPR < 32 ? TPR : 32)>(q);
    if constexpr (TPR > 32) {
      if (lane == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          scratch[turn][2 * r * NW + (threadIdx.x >> 5)] = s[r];
          scratch[turn][(2 * r + 1) * NW + (threadIdx.x >> 5)] = q[r];
        }
      __syncthreads();
      float of[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[r] = scratch[turn][2 * r * NW + (lane & (NW - 1))];
        q[r] = scratch[turn][(2 * r + 1) * NW + (lane & (NW - 1))];
        of[r] = s[r] * per_held;
      }
      shuffle_sums<NW>(s);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float c = of[r] - s[r] * inv;
        q[r] = fmaf(c, c * (held * inv), q[r]);
      }
      shuffle_sums<NW>(q);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = now + r * RPC + group;
      if (row >= a.rows) continue;
      const float mean = s[r] * inv, rstd = __frsqrt_rn(q[r] + a.eps);
      // (the difference first: z rstd - mean rstd in one operation would leave the rounding of mean rstd where z is the mean)
      const uint64_t by = spread<N>(rstd), off = spread<N>(-mean);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int d = (v * TPR + sub) * N;
        if (d >= a.D) continue;
        if (RES && a.z) z[r][v].store(a.z, row * a.D + d);
        if (LARGE) z[r][v].again();
        if constexpr (SHARED) {
#pragma unroll
          for (int i = 0; i < P / 2; ++i) {
            const ulonglong2 p = shared_params[i * TPR * NV + v * TPR + sub], q = shared_params[(P / 2 + i) * TPR * NV + v * TPR + sub];
            w[0][2 * i] = p.x, w[0][2 * i + 1] = p.y;
            b[0][2 * i] = q.x, b[0][2 * i + 1] = q.y;
          }
        } else if constexpr (!HELD) {
          load_params<N>(a.weight, a.param_dtype, d, 1.f, w[0]);
          load_params<N>(a.bias, a.param_dtype, d, 0.f, b[0]);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) z[r][v].set(i, fma2(mul2(add2(z[r][v].pair(i), off), by), w[HELD ? v : 0][i], b[HELD ? v : 0][i]));
        z[r][v].store(a.y, row * a.D + d);
      }
      if (sub == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------------
template <typename T, int N, int TPR, int NV, bool DZ>
__global__ void __launch_bounds__(threads_of(TPR), bwd_ctas(TPR)) layer_norm_bwd_kernel(const b200gdn_layer_norm_args a) {
  constexpr int RPC = threads_of(TPR) / TPR, R = rows_at_once(NV, N);
  __shared__ float scratch[2][2 * R * (TPR > 32 ? TPR / 32 : 1)];
  __shared__ float part[RPC > 1 ? RPC * 2 * TPR * NV * N : 1];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const float inv = 1.f / a.D;
  constexpr int P = pairs(N);
  uint64_t w[NV][P], dw[NV][P], db[NV][P];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int d = (v * TPR + sub) * N;
#pragma unroll
    for (int i = 0; i < P; ++i) w[v][i] = dw[v][i] = db[v][i] = 0ull;
    if (d < a.D) load_params<N>(a.weight, a.param_dtype, d, 1.f, w[v]);
  }
  struct Rows {
    Vec<T, N> z[R][NV], dy[R][NV], dz[DZ ? R : 1][NV];
    float mean[R], rstd[R];
  };
  Rows next;
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = r0 + r * RPC + group;
      const bool live = row < a.rows;   // (a row past the end adds zeros to every sum)
      next.mean[r] = live ? a.mean[row] : 0.f;
      next.rstd[r] = live ? a.rstd[row] : 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int d = (v * TPR + sub) * N;
        next.z[r][v].u = next.dy[r][v].u = decltype(next.z[r][v].u){};
        if constexpr (DZ) next.dz[r][v].u = decltype(next.z[r][v].u){};
        if (live && d < a.D) {
          next.z[r][v].load(a.z, row * a.D + d);
          next.dy[r][v].load(a.dy, row * a.D + d);
          if constexpr (DZ) next.dz[r][v].load(a.dz, row * a.D + d);
        }
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPC * R;
  int64_t r0 = (int64_t)blockIdx.x * RPC * R;
  fetch(r0);
  for (int turn = 0; r0 < a.rows; turn ^= 1) {
    const int64_t now = r0;
    Rows cur = next;
    r0 += step;
    fetch(r0);
    float s[2 * R];   // of h and of h n
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint64_t by = spread<N>(cur.rstd[r]), off = spread<N>(-cur.mean[r]);
      uint64_t s1 = 0ull, s2 = 0ull;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const uint64_t c = add2(cur.z[r][v].pair(i), off), g = cur.dy[r][v].pair(i), h = mul2(g, w[v][i]);   // c = n / rstd
          s1 = add2(s1, h);
          s2 = fma2(h, c, s2);
          dw[v][i] = fma2(mul2(g, by), c, dw[v][i]);
          db[v][i] = add2(db[v][i], g);
        }
      s[2 * r] = both(s1);
      s[2 * r + 1] = both(s2) * cur.rstd[r];
    }
    row_sums<TPR>(s, scratch[turn]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = now + r * RPC + group;
      if (row >= a.rows) continue;
      const uint64_t by = spread<N>(cur.rstd[r]), off = spread<N>(-cur.mean[r]);
      const uint64_t h_mean = spread<N>(-s[2 * r] * inv), hn_mean = spread<N>(-s[2 * r + 1] * inv * cur.rstd[r]);   // (of z - mean)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int d = (v * TPR + sub) * N;
        if (d >= a.D) continue;
        cur.z[r][v].again();   // widened anew: kept wide over the barrier, the rows would not fit the registers
        cur.dy[r][v].again();
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const uint64_t e = fma2(add2(cur.z[r][v].pair(i), off), hn_mean, fma2(cur.dy[r][v].pair(i), w[v][i], h_mean));
          if constexpr (DZ) cur.z[r][v].set(i, fma2(e, by, cur.dz[r][v].pair(i)));
          else cur.z[r][v].set(i, mul2(e, by));
        }
        cur.z[r][v].store(a.dx, row * a.D + d);
      }
    }
  }
  if (a.partials == nullptr) return;
  constexpr int C = TPR * NV * N;
  auto leave = [&](int which, int d, uint64_t x) {   // a pair of columns
    const float2 f = unpack2(x);
    if constexpr (RPC == 1) {
      float* at = a.partials + ((int64_t)blockIdx.x * 2 + which) * a.D;
      if (d < a.D) at[d] = f.x;
      if (N > 1 && d + 1 < a.D) at[d + 1] = f.y;
    } else {
      part[(group * 2 + which) * C + d] = f.x;
      if (N > 1) part[(group * 2 + which) * C + d + 1] = f.y;
    }
  };
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < P; ++i) {
      leave(0, (v * TPR + sub) * N + 2 * i, dw[v][i]);
      leave(1, (v * TPR + sub) * N + 2 * i, db[v][i]);
    }
  if constexpr (RPC > 1) {   // the groups' sums in their order
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * C; i += threads_of(TPR)) {
      const int which = i / C, d = i % C;
      if (d >= a.D) continue;
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < RPC; ++g) s += part[(g * 2 + which) * C + d];
      a.partials[((int64_t)blockIdx.x * 2 + which) * a.D + d] = s;
    }
  }
}

// dw / db = sums of the CTAs' partial rows in a fixed order: warp q adds rows q, q + 32, ... for 32 columns, then the 32 sums are added in
// warp order
__global__ void __launch_bounds__(1024) layer_norm_reduce_kernel(const b200gdn_layer_norm_args a, int n) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  wait_for_predecessor();
  float s4[4] = {0.f, 0.f, 0.f, 0.f};   // four interleaved running sums, so that the loads overlap
  if (i < 2 * a.D) {
    int c = q;
    for (; c + 96 < n; c += 128)
#pragma unroll
      for (int e = 0; e < 4; ++e) s4[e] += a.partials[(int64_t)(c + e * 32) * 2 * a.D + i];
    for (; c < n; c += 32) s4[0] += a.partials[(int64_t)c * 2 * a.D + i];
  }
  part[q][lane] = (s4[0] + s4[1]) + (s4[2] + s4[3]);
  __syncthreads();
  if (q != 0 || i >= 2 * a.D) return;
  float s = part[0][lane];
#pragma unroll
  for (int r = 1; r < 32; ++r) s += part[r][lane];
  void* out = i < a.D ? a.dweight : a.dbias;
  if (out) st_param(out, i < a.D ? i : i - a.D, a.param_dtype, s);
}

// ---- rows wider than a CTA's registers: several passes over the row, and over the columns ---------------------------------
constexpr int NT = 256;
template <int COUNT>
__device__ __forceinline__ void cta_sums(float (&v)[COUNT], float* scratch) {
  __syncthreads();
  row_sums<NT>(v, scratch);
}

template <typename T>
__global__ void __launch_bounds__(NT) layer_norm_wide_fwd_kernel(const b200gdn_layer_norm_args a) {
  __shared__ float scratch[NT / 32];
  const int64_t row = (int64_t)blockIdx.x * a.D;
  auto z = [&](int d) {
    const float x = Io<T>::ld(a.x, row + d);
    return a.residual ? (float)static_cast<T>(x + Io<T>::ld(a.residual, row + d)) : x;
  };
  const float inv = 1.f / a.D;
  float s[1] = {0.f};
  for (int d = threadIdx.x; d < a.D; d += NT) s[0] += z(d);
  cta_sums(s, scratch);
  const float mean = s[0] * inv;
  s[0] = 0.f;
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const float c = z(d) - mean;
    s[0] += c * (c * inv);
  }
  cta_sums(s, scratch);
  const float rstd = 1.f / sqrtf(s[0] + a.eps);
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const float v = z(d);
    if (a.z) Io<T>::st(a.z, row + d, v);
    Io<T>::st(a.y, row + d, fmaf((v - mean) * rstd, a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f, a.bias ? ld_param(a.bias, d, a.param_dtype) : 0.f));
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = rstd;
  }
}

template <typename T>
__global__ void __launch_bounds__(NT) layer_norm_wide_bwd_kernel(const b200gdn_layer_norm_args a) {
  __shared__ float scratch[2 * NT / 32];
  const int64_t row = (int64_t)blockIdx.x * a.D;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x], inv = 1.f / a.D;
  auto h = [&](int d) { return Io<T>::ld(a.dy, row + d) * (a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f); };
  auto n = [&](int d) { return (Io<T>::ld(a.z, row + d) - mean) * rstd; };
  float s[2] = {0.f, 0.f};
  for (int d = threadIdx.x; d < a.D; d += NT) {
    s[0] += h(d);
    s[1] += h(d) * n(d);
  }
  cta_sums(s, scratch);
  for (int d = threadIdx.x; d < a.D; d += NT)
    Io<T>::st(a.dx, row + d, fmaf(rstd, h(d) - s[0] * inv - n(d) * (s[1] * inv), a.dz ? Io<T>::ld(a.dz, row + d) : 0.f));
}

template <typename T>
__global__ void __launch_bounds__(NT) layer_norm_wide_columns_kernel(const b200gdn_layer_norm_args a) {
  const int d = blockIdx.y * NT + threadIdx.x;
  if (d >= a.D) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float dy = Io<T>::ld(a.dy, r * a.D + d);
    dw = fmaf(dy, (Io<T>::ld(a.z, r * a.D + d) - a.mean[r]) * a.rstd[r], dw);
    db += dy;
  }
  a.partials[(int64_t)blockIdx.x * 2 * a.D + d] = dw;
  a.partials[((int64_t)blockIdx.x * 2 + 1) * a.D + d] = db;
}

// ---- launches ------------------------------------------------------------------------------------------------------------
int most_ctas() { return 8 * sm_count(); }   // more than any backward kernel's

int reduce_partials(const b200gdn_layer_norm_args& a, int n, cudaStream_t st) {
  launch_overlapped(true, layer_norm_reduce_kernel, dim3((2 * a.D + 31) / 32), 1024, 0, st, a, n);
  return check_launch("layer_norm_reduce");
}

int grid_of(int64_t rows, int each, int per_sm) {   // CTAs that take `each` rows at a time
  const int64_t want = (rows + each - 1) / each, most = (int64_t)per_sm * sm_count();
  return (int)(want < most ? want : most);
}
template <typename T, int N, int TPR, int NV>
int launch_fwd(const b200gdn_layer_norm_args& a, cudaStream_t st) {
  const int n = grid_of(a.rows, threads_of(TPR) / TPR * rows_at_once(NV, N), fwd_ctas(TPR, NV, a.residual != nullptr));
  auto go = [&](auto kern, bool shared) {
    const size_t smem = shared ? 2 * sizeof(float) * TPR * NV * N : 0;
    if (smem > 48 * 1024)
      if (int e = ensure_smem(kern, smem)) return e;
    kern<<<n, threads_of(TPR), smem, st>>>(a);
    return check_launch("layer_norm_fwd");
  };
  return a.residual ? go(layer_norm_fwd_kernel<T, N, TPR, NV, true>, shares_params(NV, N, true))
                    : go(layer_norm_fwd_kernel<T, N, TPR, NV, false>, shares_params(NV, N, false));
}
template <typename T, int N, int TPR, int NV>
int launch_bwd(const b200gdn_layer_norm_args& a, cudaStream_t st) {
  const int n = grid_of(a.rows, threads_of(TPR) / TPR * rows_at_once(NV, N), bwd_ctas(TPR));
  if (a.dz) layer_norm_bwd_kernel<T, N, TPR, NV, true><<<n, threads_of(TPR), 0, st>>>(a);
  else layer_norm_bwd_kernel<T, N, TPR, NV, false><<<n, threads_of(TPR), 0, st>>>(a);
  if (int e = check_launch("layer_norm_bwd")) return e;
  return a.partials ? reduce_partials(a, n, st) : 0;
}

template <typename T>
int launch_wide(const b200gdn_layer_norm_args& a, cudaStream_t st, bool bwd) {
  if (!bwd) {
    layer_norm_wide_fwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
    return check_launch("layer_norm_wide_fwd");
  }
  layer_norm_wide_bwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
  if (int e = check_launch("layer_norm_wide_bwd")) return e;
  if (a.partials == nullptr) return 0;
  const int n = layer_norm_grid(a.rows);
  layer_norm_wide_columns_kernel<T><<<dim3(n, (a.D + NT - 1) / NT), NT, 0, st>>>(a);
  if (int e = check_launch("layer_norm_wide_columns")) return e;
  return reduce_partials(a, n, st);
}

// Pieces of a row, of 16 bytes.  Forward four a thread, from 2048 16-bit elements on by several warps (65536 rows of 4096, with parameters from
// the cache: 217 us with four pieces a thread, 232 with two, 226 with one, 318 with sixteen, a warp a row; from shared memory 180).  Backward, beside the sums: one a thread as far
// as 512 go.  Smaller pieces (odd widths): up to eight a thread first (8191 rows of 1003 fp32, forward: 17 us with eight, 29 with four).
template <typename T, int N>
int launch_n(const b200gdn_layer_norm_args& a, cudaStream_t st, bool bwd) {
  const int pieces = a.D / N;
  constexpr bool full = sizeof(T) * N == 16;
  if (!bwd) {
    if (pieces <= 8) return launch_fwd<T, N, 8, 1>(a, st);
    if (pieces <= 16) return launch_fwd<T, N, 16, 1>(a, st);
    if (pieces <= 32) return launch_fwd<T, N, 32, 1>(a, st);
    if (pieces <= 64) return launch_fwd<T, N, 32, 2>(a, st);
    if (pieces <= 128) return launch_fwd<T, N, 32, 4>(a, st);
    if constexpr (full) {
      if (pieces <= 256) return launch_fwd<T, N, 64, 4>(a, st);
      if (pieces <= 512) return launch_fwd<T, N, 128, 4>(a, st);
      if (pieces <= 1024) return launch_fwd<T, N, 256, 4>(a, st);
    } else {
      if (pieces <= 256) return launch_fwd<T, N, 32, 8>(a, st);
      if (pieces <= 512) return launch_fwd<T, N, 64, 8>(a, st);
      if (pieces <= 1024) return launch_fwd<T, N, 128, 8>(a, st);
    }
    if (pieces <= 2048) return launch_fwd<T, N, 256, 8>(a, st);
    if (pieces <= 4096) return launch_fwd<T, N, 512, 8>(a, st);
    if constexpr (N == 1)
      if (pieces <= 8192) return launch_fwd<T, N, 512, 16>(a, st);
  } else if constexpr (full) {
    if (pieces <= 8) return launch_bwd<T, N, 8, 1>(a, st);
    if (pieces <= 16) return launch_bwd<T, N, 16, 1>(a, st);
    if (pieces <= 32) return launch_bwd<T, N, 32, 1>(a, st);
    if (pieces <= 64) return launch_bwd<T, N, 64, 1>(a, st);
    if (pieces <= 128) return launch_bwd<T, N, 128, 1>(a, st);
    if (pieces <= 256) return launch_bwd<T, N, 256, 1>(a, st);
    if (pieces <= 512) return launch_bwd<T, N, 512, 1>(a, st);
    if (pieces <= 1024) return launch_bwd<T, N, 512, 2>(a, st);
  } else {
    if (pieces <= 32) return launch_bwd<T, N, 32, 1>(a, st);
    if (pieces <= 64) return launch_bwd<T, N, 32, 2>(a, st);
    if (pieces <= 128) return launch_bwd<T, N, 32, 4>(a, st);
    if (pieces <= 256) return launch_bwd<T, N, 32, 8>(a, st);
    if (pieces <= 512) return launch_bwd<T, N, 64, 8>(a, st);
    if (pieces <= 1024) return launch_bwd<T, N, 128, 8>(a, st);
    if (pieces <= 2048) return launch_bwd<T, N, 256, 8>(a, st);
    if (pieces <= 4096) return launch_bwd<T, N, 512, 8>(a, st);
    if constexpr (N == 1)
      if (pieces <= 8192) return launch_bwd<T, N, 512, 16>(a, st);
  }
  return launch_wide<T>(a, st, bwd);
}

template <typename T>
int launch_t(const b200gdn_layer_norm_args& a, cudaStream_t st, bool bwd) {
  const int n = layer_norm_piece(a);
  if (n == 16 / sizeof(T)) return launch_n<T, 16 / sizeof(T)>(a, st, bwd);
  if constexpr (sizeof(T) == 2)
    if (n == 2) return launch_n<T, 2>(a, st, bwd);
  return launch_n<T, 1>(a, st, bwd);
}

}  // namespace

int layer_norm_grid(int64_t rows) { return (int)(rows < 1 ? 1 : rows < most_ctas() ? rows : most_ctas()); }

int launch_layer_norm(const b200gdn_layer_norm_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

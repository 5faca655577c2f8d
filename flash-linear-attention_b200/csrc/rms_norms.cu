// The RMS norms either side of a block in one pass, with the block's gate, its residual scale and the residual sum:
//     r1 = 1 / rms(y),  p = y r1 w1  (POST; else p = y);   z = residual + c act(gate) p,  c = alpha scale;   r2 = 1 / rms(z),  out = z r2 w
//     h = dout w;  e = dz + r2 (h - z r2^2 mean(h z)) is the gradient of z and of the residual;
//     dgate = e c p act'(gate);  f = e c act w1;  dy = r1 (f - y r1^2 mean(f y))  (POST; else f);
//     dw = sum of dout z r2;  t = sum of e act y r1:  dw1 = alpha scale t,  dscale = alpha w1 t
// z is normalised as it is summed, in fp32; only what is handed on is rounded.  The backward pass forms z again from the inputs, which it
// reads in any case but for the residual, so that z need not be kept.
// HBM streaming, in the manner of layer_norm.cu: a row lies in the registers of TPR threads in NV pieces of N elements, CTAs walk the rows
// with the next one on its way, a thread's columns stay its own and so the parameters' gradients are sums in registers, which a second
// kernel joins in a fixed order.  The second norm needs what the first one gives: two barriers a row, forward as well as backward.
#include "gdn_common.cuh"
#include "row_pieces.cuh"

namespace gdn {
namespace {

constexpr uint32_t POST = B200GDN_NORMS_POST, SIGMOID = B200GDN_NORMS_SIGMOID, SILU = B200GDN_NORMS_SILU;
constexpr int threads_of(int tpr) { return tpr > 32 ? tpr : 128; }

// down: a power of two, down^2 in [1 / 4 D, 1 / D]: a sum of squares of elements times `down` is within range wherever their mean is, which
// is that sum times `up`
__device__ __forceinline__ float down_of(int D) { return __int_as_float((127 - (33 - __clz(D - 1)) / 2) << 23); }

// act(gate) and, where asked for, act'(gate)
template <bool SLOPE>
__device__ __forceinline__ uint64_t activation(uint64_t g, uint32_t flags, uint64_t& slope) {
  const uint64_t one = pack2(1.f, 1.f);
  if (!(flags & (SIGMOID | SILU))) {
    if (SLOPE) slope = one;
    return g;
  }
  const uint64_t s = fast_sigmoid2(g), ns = mul2(s, pack2(-1.f, -1.f)), rest = add2(one, ns);   // 1 - sigmoid
  if (flags & SIGMOID) {
    if (SLOPE) slope = mul2(s, rest);
    return s;
  }
  if (SLOPE) slope = mul2(s, fma2(g, rest, one));
  return mul2(g, s);
}

// ---- forward -------------------------------------------------------------------------------------------------------------
template <typename T, int N, int TPR, int NV>
__global__ void __launch_bounds__(threads_of(TPR), 512 / threads_of(TPR)) rms_norms_fwd_kernel(const b200gdn_rms_norms_args a) {
  constexpr int RPC = threads_of(TPR) / TPR, NW = TPR > 32 ? TPR / 32 : 1, P = pairs(N);
  constexpr bool HELD = NV * N <= 8;   // the parameters as fp32 pairs in registers; else they come from the cache with every row
  __shared__ float scratch[2][2][NW];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool post = a.flags & POST;
  const float inv = 1.f / a.D, down = down_of(a.D), up = inv / (down * down);
  const uint64_t by = spread<N>(down);
  uint64_t c[HELD ? NV : 1][P], w[HELD ? NV : 1][P];
  auto params = [&](int d, uint64_t (&c)[P], uint64_t (&w)[P]) {   // what p's normalised elements are multiplied with, and z's
    load_params<N>(a.scale, a.param_dtype, d, 1.f, c);
    load_params<N>(post ? a.post_weight : nullptr, a.param_dtype, d, 1.f, w);
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = mul2(mul2(c[i], spread<N>(a.alpha)), w[i]);
    load_params<N>(a.weight, a.param_dtype, d, 1.f, w);
  };
  if constexpr (HELD) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int i = 0; i < P; ++i) c[v][i] = w[v][i] = 0ull;
      if ((v * TPR + sub) * N < a.D) params((v * TPR + sub) * N, c[v], w[v]);
    }
  }
  Vec<T, N> y[NV], res[NV], gate[NV];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      y[v].u = res[v].u = gate[v].u = decltype(y[v].u){};
      if (row < a.rows && d < a.D) {
        y[v].load(a.y, row * a.D + d);
        if (a.residual) res[v].load(a.residual, row * a.D + d);
        if (a.gate) gate[v].load(a.gate, row * a.D + d);
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t row = (int64_t)blockIdx.x * RPC + group;
  fetch(row);
  for (int turn = 0; row - group < a.rows; turn ^= 1, row += step) {
    float s[1] = {0.f}, r1 = 1.f;
    if (post) {
      uint64_t sum = 0ull;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const uint64_t x = mul2(y[v].pair(i), by);
          sum = fma2(x, x, sum);
        }
      s[0] = both(sum);
      row_sums<TPR>(s, scratch[turn][0]);
      r1 = __frsqrt_rn(s[0] * up + a.eps);
    }
    uint64_t z[NV][P], sum = 0ull;
    const uint64_t by_r1 = spread<N>(r1);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      if constexpr (!HELD) {
#pragma unroll
        for (int i = 0; i < P; ++i) c[0][i] = 0ull;
        if (d < a.D) params(d, c[0], w[0]);
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        uint64_t none, k = mul2(c[HELD ? v : 0][i], by_r1);
        if (a.gate) k = mul2(k, activation<false>(gate[v].pair(i), a.flags, none));
        z[v][i] = fma2(y[v].pair(i), k, res[v].pair(i));
        const uint64_t x = mul2(z[v][i], by);
        sum = fma2(x, x, sum);
      }
    }
    fetch(row + step);
    s[0] = both(sum);
    row_sums<TPR>(s, scratch[turn][1]);
    const float r2 = __frsqrt_rn(s[0] * up + a.eps);
    const uint64_t by_r2 = spread<N>(r2);
    if (row >= a.rows) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      if (d >= a.D) continue;
      if constexpr (!HELD) load_params<N>(a.weight, a.param_dtype, d, 1.f, w[0]);
      Vec<T, N> o;
      if (a.z) {
#pragma unroll
        for (int i = 0; i < P; ++i) o.set(i, z[v][i]);
        o.store(a.z, row * a.D + d);
      }
#pragma unroll
      for (int i = 0; i < P; ++i) o.set(i, mul2(mul2(z[v][i], by_r2), w[HELD ? v : 0][i]));
      o.store(a.out, row * a.D + d);
    }
    if (sub == 0 && a.rstd_z) {
      a.rstd_y[row] = r1;
      a.rstd_z[row] = r2;
    }
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------------
constexpr int bwd_ctas(int tpr) { return tpr <= 128 ? 4 : tpr == 256 ? 2 : 1; }

template <typename T, int N, int TPR, int NV>
__global__ void __launch_bounds__(threads_of(TPR), bwd_ctas(TPR)) rms_norms_bwd_kernel(const b200gdn_rms_norms_args a) {
  constexpr int RPC = threads_of(TPR) / TPR, NW = TPR > 32 ? TPR / 32 : 1, P = pairs(N);
  constexpr bool HELD = NV * N <= 8;
  __shared__ float scratch[2][2][NW];
  __shared__ float part[RPC > 1 ? RPC * 2 * TPR * NV * N : 1];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool post = a.flags & POST;
  const float inv = 1.f / a.D;
  uint64_t c[HELD ? NV : 1][P], w1[HELD ? NV : 1][P], w[HELD ? NV : 1][P];
  auto params = [&](int d, uint64_t (&c)[P], uint64_t (&w1)[P], uint64_t (&w)[P]) {   // alpha scale, and the norms' weights
    load_params<N>(a.scale, a.param_dtype, d, 1.f, c);
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = mul2(c[i], spread<N>(a.alpha));
    load_params<N>(post ? a.post_weight : nullptr, a.param_dtype, d, 1.f, w1);
    load_params<N>(a.weight, a.param_dtype, d, 1.f, w);
  };
  uint64_t dw[NV][P], dt[NV][P];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int i = 0; i < P; ++i) dw[v][i] = dt[v][i] = 0ull;
    if constexpr (HELD) {
#pragma unroll
      for (int i = 0; i < P; ++i) c[v][i] = w1[v][i] = w[v][i] = 0ull;
      if ((v * TPR + sub) * N < a.D) params((v * TPR + sub) * N, c[v], w1[v], w[v]);
    }
  }
  struct Row {
    Vec<T, N> y[NV], res[NV], gate[NV], dout[NV], dz[NV];
    float r1, r2;
  };
  Row next;
  auto fetch = [&](int64_t row) {
    const bool live = row < a.rows;   // (a row past the end adds zeros to every sum)
    next.r1 = live ? a.rstd_y[row] : 0.f;
    next.r2 = live ? a.rstd_z[row] : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      next.y[v].u = next.res[v].u = next.gate[v].u = next.dout[v].u = next.dz[v].u = decltype(next.y[v].u){};
      if (live && d < a.D) {
        next.y[v].load(a.y, row * a.D + d);
        if (a.residual) next.res[v].load(a.residual, row * a.D + d);
        if (a.gate) next.gate[v].load(a.gate, row * a.D + d);
        if (a.dout) next.dout[v].load(a.dout, row * a.D + d);
        if (a.dz) next.dz[v].load(a.dz, row * a.D + d);
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t row = (int64_t)blockIdx.x * RPC + group;
  fetch(row);
  for (int turn = 0; row - group < a.rows; turn ^= 1, row += step) {
    Row cur = next;
    fetch(row + step);
    const uint64_t r1 = spread<N>(cur.r1), r2 = spread<N>(cur.r2);
    uint64_t z[NV][P], sum = 0ull;   // z, then e
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      if constexpr (!HELD) {
#pragma unroll
        for (int i = 0; i < P; ++i) c[0][i] = w1[0][i] = w[0][i] = 0ull;
        if (d < a.D) params(d, c[0], w1[0], w[0]);
      }
      const int q = HELD ? v : 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        uint64_t none, k = mul2(mul2(c[q][i], w1[q][i]), r1);
        if (a.gate) k = mul2(k, activation<false>(cur.gate[v].pair(i), a.flags, none));
        z[v][i] = fma2(cur.y[v].pair(i), k, cur.res[v].pair(i));
        const uint64_t g = cur.dout[v].pair(i), n = mul2(z[v][i], r2);
        sum = fma2(mul2(g, w[q][i]), n, sum);
        dw[v][i] = fma2(g, n, dw[v][i]);
      }
    }
    float s[1] = {both(sum)};
    row_sums<TPR>(s, scratch[turn][0]);
    const uint64_t back = spread<N>(-s[0] * inv);   // of n = z r2
    const bool live = row < a.rows;
    sum = 0ull;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      if constexpr (!HELD) {
        if (d < a.D) params(d, c[0], w1[0], w[0]);
        else {
#pragma unroll
          for (int i = 0; i < P; ++i) c[0][i] = w1[0][i] = w[0][i] = 0ull;
        }
      }
      const int q = HELD ? v : 0;
      Vec<T, N> dgate;
      dgate.u = decltype(dgate.u){};
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint64_t h = fma2(mul2(z[v][i], r2), back, mul2(cur.dout[v].pair(i), w[q][i]));
        const uint64_t e = fma2(h, r2, cur.dz[v].pair(i)), n1 = mul2(cur.y[v].pair(i), r1);
        uint64_t slope, act = spread<N>(1.f);
        if (a.gate) {
          act = activation<true>(cur.gate[v].pair(i), a.flags, slope);
          if (a.dgate) dgate.set(i, mul2(mul2(mul2(e, c[q][i]), mul2(n1, w1[q][i])), slope));
        }
        const uint64_t f = mul2(e, act);
        dt[v][i] = fma2(f, n1, dt[v][i]);
        z[v][i] = mul2(f, mul2(c[q][i], w1[q][i]));
        sum = fma2(z[v][i], n1, sum);
        cur.res[v].set(i, e);
      }
      if (live && d < a.D) {
        if (a.dgate) dgate.store(a.dgate, row * a.D + d);
        if (a.dresidual) cur.res[v].store(a.dresidual, row * a.D + d);
      }
    }
    uint64_t mean = 0ull;
    if (post) {
      s[0] = both(sum);
      row_sums<TPR>(s, scratch[turn][1]);
      mean = spread<N>(-s[0] * inv);
    }
    if (!live || !a.dy) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int d = (v * TPR + sub) * N;
      if (d >= a.D) continue;
#pragma unroll
      for (int i = 0; i < P; ++i) cur.y[v].set(i, mul2(fma2(mul2(cur.y[v].pair(i), r1), mean, z[v][i]), r1));   // (r1 is one without the first norm)
      cur.y[v].store(a.dy, row * a.D + d);
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
      leave(1, (v * TPR + sub) * N + 2 * i, dt[v][i]);
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

// the CTAs' partial rows in a fixed order: warp q adds rows q, q + 32, ... for 32 columns, then the 32 sums are added in warp order
__global__ void __launch_bounds__(1024) rms_norms_reduce_kernel(const b200gdn_rms_norms_args a, int n) {
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
  if (i < a.D) {
    if (a.dweight) st_param(a.dweight, i, a.param_dtype, s);
    return;
  }
  const int d = i - a.D;
  s *= a.alpha;
  if (a.dpost_weight) st_param(a.dpost_weight, d, a.param_dtype, a.scale ? s * ld_param(a.scale, d, a.param_dtype) : s);
  if (a.dscale) st_param(a.dscale, d, a.param_dtype, (a.flags & POST) && a.post_weight ? s * ld_param(a.post_weight, d, a.param_dtype) : s);
}

// ---- rows wider than a CTA's registers: several looks at the row, and at the columns ---------------------------------------
constexpr int NT = 512;
template <int COUNT>
__device__ __forceinline__ void cta_sums(float (&v)[COUNT], float* scratch) {
  __syncthreads();
  row_sums<NT>(v, scratch);
}

template <typename T>
struct Element {   // of column d: what the passes over a wide row form again each time
  float y, p, act, slope, c, w1, z;
  __device__ __forceinline__ Element(const b200gdn_rms_norms_args& a, int64_t row, int d, float r1) {
    y = Io<T>::ld(a.y, row + d);
    c = a.alpha * (a.scale ? ld_param(a.scale, d, a.param_dtype) : 1.f);
    w1 = (a.flags & POST) && a.post_weight ? ld_param(a.post_weight, d, a.param_dtype) : 1.f;
    p = y * r1 * w1;
    act = slope = 1.f;
    if (a.gate) {
      const float g = Io<T>::ld(a.gate, row + d);
      uint64_t s;
      act = unpack2(activation<true>(pack2(g, 0.f), a.flags, s)).x;
      slope = unpack2(s).x;
    }
    z = fmaf(p, c * act, a.residual ? Io<T>::ld(a.residual, row + d) : 0.f);
  }
};

template <typename T>
__global__ void __launch_bounds__(NT) rms_norms_wide_fwd_kernel(const b200gdn_rms_norms_args a) {
  __shared__ float scratch[NT / 32];
  const int64_t row = (int64_t)blockIdx.x * a.D;
  const float down = down_of(a.D), up = 1.f / a.D / (down * down);
  float s[1] = {0.f}, r1 = 1.f;
  if (a.flags & POST) {
    for (int d = threadIdx.x; d < a.D; d += NT) {
      const float x = Io<T>::ld(a.y, row + d) * down;
      s[0] = fmaf(x, x, s[0]);
    }
    cta_sums(s, scratch);
    r1 = __frsqrt_rn(s[0] * up + a.eps);
    s[0] = 0.f;
  }
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const float x = Element<T>(a, row, d, r1).z * down;
    s[0] = fmaf(x, x, s[0]);
  }
  cta_sums(s, scratch);
  const float r2 = __frsqrt_rn(s[0] * up + a.eps);
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const float z = Element<T>(a, row, d, r1).z;
    if (a.z) Io<T>::st(a.z, row + d, z);
    Io<T>::st(a.out, row + d, z * r2 * (a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f));
  }
  if (threadIdx.x == 0 && a.rstd_z) {
    a.rstd_y[blockIdx.x] = r1;
    a.rstd_z[blockIdx.x] = r2;
  }
}

// e of column d, with the mean of h n
template <typename T>
__device__ __forceinline__ float stream_gradient(const b200gdn_rms_norms_args& a, int64_t row, int d, float z, float r2, float mean) {
  const float h = a.dout ? Io<T>::ld(a.dout, row + d) * (a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f) : 0.f;
  return fmaf(h - z * r2 * mean, r2, a.dz ? Io<T>::ld(a.dz, row + d) : 0.f);
}

template <typename T>
__global__ void __launch_bounds__(NT) rms_norms_wide_bwd_kernel(const b200gdn_rms_norms_args a) {
  __shared__ float scratch[NT / 32];
  const int64_t row = (int64_t)blockIdx.x * a.D;
  const float r1 = a.rstd_y[blockIdx.x], r2 = a.rstd_z[blockIdx.x], inv = 1.f / a.D;
  float s[1] = {0.f};
  if (a.dout)
    for (int d = threadIdx.x; d < a.D; d += NT)
      s[0] += Io<T>::ld(a.dout, row + d) * (a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f) * (Element<T>(a, row, d, r1).z * r2);
  cta_sums(s, scratch);
  const float mean = s[0] * inv;
  s[0] = 0.f;
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const Element<T> x(a, row, d, r1);
    const float e = stream_gradient<T>(a, row, d, x.z, r2, mean);
    s[0] += e * x.act * (x.c * x.w1) * (x.y * r1);
    if (a.dresidual) Io<T>::st(a.dresidual, row + d, e);
    if (a.dgate) Io<T>::st(a.dgate, row + d, e * x.c * x.p * x.slope);
  }
  cta_sums(s, scratch);
  if (threadIdx.x == 0 && a.partials) a.partials[blockIdx.x] = mean;   // (the columns' kernel reads it)
  const float back = a.flags & POST ? s[0] * inv : 0.f;
  if (a.dy)
    for (int d = threadIdx.x; d < a.D; d += NT) {
      const Element<T> x(a, row, d, r1);
      const float e = stream_gradient<T>(a, row, d, x.z, r2, mean);
      Io<T>::st(a.dy, row + d, r1 * (e * x.act * (x.c * x.w1) - x.y * r1 * back));
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) rms_norms_wide_columns_kernel(const b200gdn_rms_norms_args a, float* sums) {
  const int d = blockIdx.y * NT + threadIdx.x;
  if (d >= a.D) return;
  float dw = 0.f, dt = 0.f;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float r1 = a.rstd_y[r], r2 = a.rstd_z[r];
    const Element<T> x(a, r * a.D, d, r1);
    if (a.dout) dw = fmaf(Io<T>::ld(a.dout, r * a.D + d), x.z * r2, dw);
    dt = fmaf(stream_gradient<T>(a, r * a.D, d, x.z, r2, a.partials[r]) * x.act, x.y * r1, dt);
  }
  sums[(int64_t)blockIdx.x * 2 * a.D + d] = dw;
  sums[((int64_t)blockIdx.x * 2 + 1) * a.D + d] = dt;
}

// ---- launches ------------------------------------------------------------------------------------------------------------
int most_ctas() { return 8 * sm_count(); }   // more than any backward kernel's

int reduce_partials(b200gdn_rms_norms_args a, int n, cudaStream_t st) {
  launch_overlapped(true, rms_norms_reduce_kernel, dim3((2 * a.D + 31) / 32), 1024, 0, st, a, n);
  return check_launch("rms_norms_reduce");
}

int grid_of(int64_t rows, int each, int per_sm) {   // CTAs that take `each` rows at a time
  const int64_t want = (rows + each - 1) / each, most = (int64_t)per_sm * sm_count();
  return (int)(want < most ? want : most);
}
template <typename T, int N, int TPR, int NV>
int launch_fwd(const b200gdn_rms_norms_args& a, cudaStream_t st) {
  rms_norms_fwd_kernel<T, N, TPR, NV><<<grid_of(a.rows, threads_of(TPR) / TPR, 512 / threads_of(TPR)), threads_of(TPR), 0, st>>>(a);
  return check_launch("rms_norms_fwd");
}
template <typename T, int N, int TPR, int NV>
int launch_bwd(const b200gdn_rms_norms_args& a, cudaStream_t st) {
  const int n = grid_of(a.rows, threads_of(TPR) / TPR, bwd_ctas(TPR));
  rms_norms_bwd_kernel<T, N, TPR, NV><<<n, threads_of(TPR), 0, st>>>(a);
  if (int e = check_launch("rms_norms_bwd")) return e;
  return a.partials ? reduce_partials(a, n, st) : 0;
}

template <typename T>
int launch_wide(const b200gdn_rms_norms_args& a, cudaStream_t st, bool bwd) {
  if (!bwd) {
    rms_norms_wide_fwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
    return check_launch("rms_norms_wide_fwd");
  }
  rms_norms_wide_bwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
  if (int e = check_launch("rms_norms_wide_bwd")) return e;
  if (a.partials == nullptr) return 0;
  const int n = rms_norms_grid(a.rows);
  b200gdn_rms_norms_args joined = a;
  joined.partials = a.partials + (a.rows + 3) / 4 * 4;   // behind the rows' means
  rms_norms_wide_columns_kernel<T><<<dim3(n, (a.D + NT - 1) / NT), NT, 0, st>>>(a, joined.partials);
  if (int e = check_launch("rms_norms_wide_columns")) return e;
  return reduce_partials(joined, n, st);
}

// Eight elements a thread and, where that is more threads than a CTA has registers for, more.
template <typename T, int N>
int launch_n(const b200gdn_rms_norms_args& a, cudaStream_t st, bool bwd) {
  const int pieces = (a.D + N - 1) / N;
  constexpr int V = 8 / N;   // pieces that make eight elements
  if (!bwd) {
    if (pieces <= 8) return launch_fwd<T, N, 8, 1>(a, st);
    if (pieces <= 32) return launch_fwd<T, N, 32, 1>(a, st);
    if (pieces <= 32 * V) return launch_fwd<T, N, 32, V>(a, st);
    if (pieces <= 64 * V) return launch_fwd<T, N, 64, V>(a, st);
    if (pieces <= 128 * V) return launch_fwd<T, N, 128, V>(a, st);
    if (pieces <= 256 * V) return launch_fwd<T, N, 128, 2 * V>(a, st);
    if (pieces <= 512 * V) return launch_fwd<T, N, 256, 2 * V>(a, st);
    if (pieces <= 1024 * V) return launch_fwd<T, N, 512, 2 * V>(a, st);
  } else {
    if (pieces <= 8) return launch_bwd<T, N, 8, 1>(a, st);
    if (pieces <= 32) return launch_bwd<T, N, 32, 1>(a, st);
    if (pieces <= 32 * V) return launch_bwd<T, N, 32, V>(a, st);
    if (pieces <= 64 * V) return launch_bwd<T, N, 64, V>(a, st);
    if (pieces <= 128 * V) return launch_bwd<T, N, 128, V>(a, st);
    if (pieces <= 256 * V) return launch_bwd<T, N, 256, V>(a, st);
    if (pieces <= 512 * V) return launch_bwd<T, N, 512, V>(a, st);
    if (pieces <= 1024 * V) return launch_bwd<T, N, 512, 2 * V>(a, st);
  }
  return launch_wide<T>(a, st, bwd);
}

// 16 bytes of the rows' elements, of 16-bit ones else two, else one: what divides the width and what every tensor that is read or written
// so lies on a boundary of (N parameters are read N times their own size at once, 16 bytes at most)
template <typename T>
int piece_of(const b200gdn_rms_norms_args& a) {
  constexpr int size = sizeof(T);
  uintptr_t rows = 0, params = 0;
  for (const void* p : {a.y, a.residual, a.gate, static_cast<const void*>(a.z), static_cast<const void*>(a.out), a.dout, a.dz, static_cast<const void*>(a.dy),
                        static_cast<const void*>(a.dresidual), static_cast<const void*>(a.dgate)})
    rows |= reinterpret_cast<uintptr_t>(p);
  for (const void* p : {a.weight, a.post_weight, a.scale}) params |= reinterpret_cast<uintptr_t>(p);
  const int param_size = a.param_dtype == B200GDN_F32 ? 4 : 2;
  auto fits = [&](int n) { return a.D % n == 0 && rows % (n * size) == 0 && params % (n * param_size < 16 ? n * param_size : 16) == 0; };
  return fits(16 / size) ? 16 / size : size == 2 && fits(2) ? 2 : 1;
}

template <typename T>
int launch_t(const b200gdn_rms_norms_args& a, cudaStream_t st, bool bwd) {
  const int n = piece_of<T>(a);
  if (n == 16 / sizeof(T)) return launch_n<T, 16 / sizeof(T)>(a, st, bwd);
  if constexpr (sizeof(T) == 2)
    if (n == 2) return launch_n<T, 2>(a, st, bwd);
  return launch_n<T, 1>(a, st, bwd);
}

}  // namespace

int rms_norms_grid(int64_t rows) { return (int)(rows < 1 ? 1 : rows < most_ctas() ? rows : most_ctas()); }

int64_t rms_norms_partials(int64_t rows, int D) { return (rows + 3) / 4 * 4 + (int64_t)rms_norms_grid(rows) * 2 * D; }

int launch_rms_norms(const b200gdn_rms_norms_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

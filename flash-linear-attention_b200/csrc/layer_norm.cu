// Layer norm over rows, forward and backward.  The simplest form: one CTA per row; the gradients of weight and bias by a second
// kernel over columns and a third that adds its partial sums in a fixed order.
#include "gdn_common.cuh"
#include "rowio.cuh"
#include "vocab.cuh"

namespace gdn {
namespace {

constexpr int NT = 256;

template <typename T>
__global__ void __launch_bounds__(NT) layer_norm_fwd_kernel(const b200gdn_layer_norm_args a) {
  __shared__ float fs[NT / 32];
  const int64_t row = (int64_t)blockIdx.x * a.D;
  auto z = [&](int d) {
    const float x = Io<T>::ld(a.x, row + d);
    if (a.residual == nullptr) return x;
    return (float)static_cast<T>(x + Io<T>::ld(a.residual, row + d));
  };
  float s = 0.f;
  for (int d = threadIdx.x; d < a.D; d += NT) s += z(d);
  const float inv = 1.f / a.D, mean = cta_reduce<NT>(s, fs, SumOf()) * inv;
  s = 0.f;
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const float c = z(d) - mean;
    s += c * (c * inv);   // divided term by term: the sum is within range wherever the variance is
  }
  const float rstd = 1.f / sqrtf(cta_reduce<NT>(s, fs, SumOf()) + a.eps);
  for (int d = threadIdx.x; d < a.D; d += NT) {
    const float v = z(d);
    if (a.z) Io<T>::st(a.z, row + d, v);
    Io<T>::st(a.y, row + d, (v - mean) * rstd * (a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f) + (a.bias ? ld_param(a.bias, d, a.param_dtype) : 0.f));
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = rstd;
  }
}

template <typename T>
__global__ void __launch_bounds__(NT) layer_norm_bwd_kernel(const b200gdn_layer_norm_args a) {
  __shared__ float fs[NT / 32];
  const int64_t row = (int64_t)blockIdx.x * a.D;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
  auto h = [&](int d) { return Io<T>::ld(a.dy, row + d) * (a.weight ? ld_param(a.weight, d, a.param_dtype) : 1.f); };
  auto n = [&](int d) { return (Io<T>::ld(a.z, row + d) - mean) * rstd; };
  float s = 0.f, t = 0.f;
  for (int d = threadIdx.x; d < a.D; d += NT) {
    s += h(d);
    t += h(d) * n(d);
  }
  s = cta_reduce<NT>(s, fs, SumOf()) / a.D;
  t = cta_reduce<NT>(t, fs, SumOf()) / a.D;
  for (int d = threadIdx.x; d < a.D; d += NT)
    Io<T>::st(a.dx, row + d, rstd * (h(d) - s - n(d) * t) + (a.dz ? Io<T>::ld(a.dz, row + d) : 0.f));
}

template <typename T>
__global__ void __launch_bounds__(NT) layer_norm_columns_kernel(const b200gdn_layer_norm_args a) {
  const int d = blockIdx.y * NT + threadIdx.x;
  if (d >= a.D) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float dy = Io<T>::ld(a.dy, r * a.D + d);
    dw += dy * (Io<T>::ld(a.z, r * a.D + d) - a.mean[r]) * a.rstd[r];
    db += dy;
  }
  a.partials[(int64_t)blockIdx.x * 2 * a.D + d] = dw;
  a.partials[((int64_t)blockIdx.x * 2 + 1) * a.D + d] = db;
}

__global__ void __launch_bounds__(NT) layer_norm_reduce_kernel(const b200gdn_layer_norm_args a, int n) {
  const int i = blockIdx.x * NT + threadIdx.x;
  if (i >= 2 * a.D) return;
  float s = 0.f;
  for (int c = 0; c < n; ++c) s += a.partials[(int64_t)c * 2 * a.D + i];
  void* out = i < a.D ? a.dweight : a.dbias;
  if (out) st_param(out, i < a.D ? i : i - a.D, a.param_dtype, s);
}

template <typename T>
int launch_t(const b200gdn_layer_norm_args& a, cudaStream_t st, bool bwd) {
  if (!bwd) {
    layer_norm_fwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
    return check_launch("layer_norm_fwd");
  }
  layer_norm_bwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
  if (int e = check_launch("layer_norm_bwd")) return e;
  if (a.dweight == nullptr && a.dbias == nullptr) return 0;
  const int n = layer_norm_grid(a.rows, a.D, a.dtype);
  layer_norm_columns_kernel<T><<<dim3(n, (a.D + NT - 1) / NT), NT, 0, st>>>(a);
  if (int e = check_launch("layer_norm_columns")) return e;
  layer_norm_reduce_kernel<<<(2 * a.D + NT - 1) / NT, NT, 0, st>>>(a, n);
  return check_launch("layer_norm_reduce");
}

}  // namespace

int layer_norm_grid(int64_t rows, int, int) { return (int)(rows < 296 ? (rows < 1 ? 1 : rows) : 296); }

int launch_layer_norm(const b200gdn_layer_norm_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

// Log probabilities of given tokens, entropy and the most probable entries of rows of logits, and their gradient.
// The simplest form: one CTA per row, three passes over it (largest entry, sums, and one search for each of the top entries).
#include "vocab.cuh"

namespace gdn {
namespace {

constexpr int NT = 256;

template <typename T>
__global__ void __launch_bounds__(NT) logprob_fwd_kernel(const b200gdn_logprob_args a) {
  __shared__ float fs[NT / 32];
  __shared__ uint64_t ks[NT / 32];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row_offset(a, r);
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.V; j += NT) m = fmaxf(m, Io<T>::ld(x, j));
  m = cta_reduce<NT>(m, fs, MaxOf());
  const float base = m == -INFINITY ? 0.f : m;
  float ss[8] = {}, ts[8] = {};   // eight chains of additions: an eighth of the rounding
  for (int j0 = threadIdx.x; j0 < a.V; j0 += 8 * NT) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = j0 + i * NT;
      if (j >= a.V) break;
      const float u = (Io<T>::ld(x, j) - base) * a.scale, e = exp2_approx(u * kLog2e);
      ss[i] += e;
      if (!(e <= 0.f)) ts[i] += e * u;
    }
  }
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s += ss[i];
    t += ts[i];
  }
  s = cta_reduce<NT>(s, fs, SumOf());
  t = cta_reduce<NT>(t, fs, SumOf());
  const bool empty = s == 0.f;
  const float logs = logf(s);
  auto lp = [&](float v) { return empty ? -INFINITY : (v - base) * a.scale - logs; };
  if (threadIdx.x == 0) {
    if (a.logprobs) {
      const int token = load_index(a.tokens, r, a.token_bytes, a.V);
      a.logprobs[r] = token < 0 ? 0.f : lp(Io<T>::ld(x, token));
    }
    if (a.entropy) a.entropy[r] = empty ? 0.f : logs - t / s;
    if (a.stats) {
      a.stats[2 * r] = base;
      a.stats[2 * r + 1] = logs;
    }
  }
  uint64_t below = ~0ull;
  for (int i = 0; i < a.top_k; ++i) {
    uint64_t best = 0;
    for (int j = threadIdx.x; j < a.V; j += NT) {
      const uint64_t k = entry_key(Io<T>::ld(x, j), j);
      if (k < below && k > best) best = k;
    }
    below = cta_reduce<NT>(best, ks, MaxOf());
    if (threadIdx.x == 0) {
      a.top_ids[r * a.top_k + i] = key_index(below);
      a.top_logprobs[r * a.top_k + i] = lp(key_value(below));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(NT) logprob_bwd_kernel(const b200gdn_logprob_args a) {
  __shared__ float fs[NT / 32];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row_offset(a, r);
  const int64_t out = r * a.V;
  const float base = a.stats[2 * r], logs = a.stats[2 * r + 1];
  if (logs == -INFINITY) {   // nothing in this row
    for (int j = threadIdx.x; j < a.V; j += NT) Io<T>::st(a.dlogits, out + j, 0.f);
    return;
  }
  const int token = a.dlogprobs ? load_index(a.tokens, r, a.token_bytes, a.V) : -1;
  const float dlp = token < 0 ? 0.f : a.dlogprobs[r], dh = a.dentropy ? a.dentropy[r] : 0.f, h = a.dentropy ? a.entropy[r] : 0.f;
  const int k = a.dtop_logprobs ? a.top_k : 0;
  float all = 0.f;
  for (int i = threadIdx.x; i < k; i += NT) all += a.dtop_logprobs[r * k + i];
  all = cta_reduce<NT>(all, fs, SumOf()) + dlp;
  auto grad = [&](int j) {
    const float lp = (Io<T>::ld(x, j) - base) * a.scale - logs, p = exp2_approx(lp * kLog2e);
    return p == 0.f ? 0.f : -p * (all + dh * (lp + h));
  };
  for (int j = threadIdx.x; j < a.V; j += NT) Io<T>::st(a.dlogits, out + j, grad(j) * a.scale);
  __syncthreads();
  bool listed = false;
  for (int i = 0; i < k; ++i) listed |= (int)a.top_ids[r * k + i] == token;
  for (int i = threadIdx.x; i < k; i += NT) {
    const int j = (int)a.top_ids[r * k + i];
    Io<T>::st(a.dlogits, out + j, (grad(j) + a.dtop_logprobs[r * k + i] + (j == token ? dlp : 0.f)) * a.scale);
  }
  if (threadIdx.x == 0 && token >= 0 && !listed) Io<T>::st(a.dlogits, out + token, (grad(token) + dlp) * a.scale);
}

template <typename T>
int launch_t(const b200gdn_logprob_args& a, cudaStream_t st, bool bwd) {
  if (bwd) logprob_bwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
  else logprob_fwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
  return check_launch(bwd ? "logprob_bwd" : "logprob_fwd");
}

}  // namespace

int launch_logprob(const b200gdn_logprob_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

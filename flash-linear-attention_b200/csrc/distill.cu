// Divergence of a student's rows of logits from a teacher's entries, and its gradient.
// The simplest form: one CTA per row; the gradient of sum or mean in the same launch, from a second look at the row.
#include "vocab.cuh"

namespace gdn {
namespace {

constexpr int NT = 256;
static_assert(NT >= B200GDN_MAX_LIST, "a thread for each entry of a list");

// less than this is what rounding leaves of a sum of one, and counts as nothing (a list may hold the whole vocabulary)
constexpr float kRestFrom = 1e-6f;

// A row's list in shared memory: thread i < K holds entry i.
struct List {
  int id[B200GDN_MAX_LIST];
  float q[B200GDN_MAX_LIST];   // 0 for absent entries
};

struct RowList {
  int id;             // of this thread's entry, -1 absent
  float l, q;         // log q and q
  float total, rest;  // sum of q; what is left of one (bucket)
  bool counted;
};

__device__ __forceinline__ bool entry_of(const b200gdn_distill_args& a, int64_t at, int& id, float& l) {
  id = load_index(a.ids, at, a.id_bytes, a.V);
  l = ld_param(a.teacher, at, a.teacher_dtype);
  if (l == -INFINITY) id = -1;
  return id >= 0;
}

template <int N>
__device__ __forceinline__ RowList load_list(const b200gdn_distill_args& a, int64_t r, List& list, float* fs) {
  RowList o;
  o.id = -1;
  o.l = -INFINITY;
  if (threadIdx.x < a.K) entry_of(a, r * a.K + threadIdx.x, o.id, o.l);
  o.counted = __syncthreads_or(o.id >= 0);
  float shift = 0.f;
  if (!(a.flags & B200GDN_DISTILL_BUCKET)) {
    const float m = cta_reduce<N>(o.id >= 0 ? o.l : -INFINITY, fs, MaxOf());
    const float s = cta_reduce<N>(o.id >= 0 ? expf(o.l - m) : 0.f, fs, SumOf());
    shift = m + logf(s);
  }
  o.l = o.id >= 0 ? o.l - shift : 0.f;
  o.q = o.id >= 0 ? expf(o.l) : 0.f;
  o.total = cta_reduce<N>(o.q, fs, SumOf());
  o.rest = a.flags & B200GDN_DISTILL_BUCKET ? 1.f - o.total : 0.f;
  if (o.rest < kRestFrom) o.rest = 0.f;
  if (threadIdx.x < a.K) {
    list.id[threadIdx.x] = o.id;
    list.q[threadIdx.x] = o.q;
  }
  __syncthreads();
  return o;
}

__device__ __forceinline__ bool on_list(const List& list, int K, int j) {
  bool on = false;
  for (int i = 0; i < K; ++i) on |= list.id[i] == j;
  return on;
}

// stats of a row: m, log of the sum, what an entry off the list has as the factor of its probability, and as the entries on it
template <typename T>
__device__ __forceinline__ void write_gradient(const b200gdn_distill_args& a, int64_t r, const T* x, const List& list, float base, float logs,
                                               float off, float on, float weight) {
  const int64_t out = r * a.V;
  const bool nothing = logs == -INFINITY || (off == 0.f && on == 0.f);
  for (int j = threadIdx.x; j < a.V; j += NT) {
    const float p = exp2_approx(((Io<T>::ld(x, j) - base) * a.scale - logs) * kLog2e);
    Io<T>::st(a.dlogits, out + j, nothing ? 0.f : p * off * weight);
  }
  __syncthreads();
  if (nothing || threadIdx.x >= a.K || list.id[threadIdx.x] < 0) return;
  const int j = list.id[threadIdx.x];
  float q = 0.f;
  for (int i = 0; i < a.K; ++i)
    if (list.id[i] == j) q += list.q[i];
  const float p = exp2_approx(((Io<T>::ld(x, j) - base) * a.scale - logs) * kLog2e);
  Io<T>::st(a.dlogits, out + j, (p * on - q) * weight);
}

__global__ void __launch_bounds__(1024) distill_count_kernel(const b200gdn_distill_args a) {
  int n = 0;
  for (int64_t r = threadIdx.x; r < a.rows; r += 1024) {
    bool any = false;
    for (int i = 0; i < a.K && !any; ++i) {
      int id;
      float l;
      any = entry_of(a, r * a.K + i, id, l);
    }
    n += any;
  }
  __shared__ int ns[32];
  n = cta_reduce<1024>(n, ns, SumOf());
  if (threadIdx.x == 0) a.counters[0] = n > 0 ? n : 1;
}

__global__ void __launch_bounds__(1024) distill_sum_kernel(const b200gdn_distill_args a) {
  __shared__ float fs[32];
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < a.rows; r += 1024) s += a.row_loss[r];
  s = cta_reduce<1024>(s, fs, SumOf());
  if (threadIdx.x == 0) *a.loss = a.flags & B200GDN_DISTILL_MEAN ? s / (float)a.counters[0] : s;
}

template <typename T>
__global__ void __launch_bounds__(NT) distill_fwd_kernel(const b200gdn_distill_args a) {
  __shared__ List list;
  __shared__ float fs[NT / 32];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row_offset(a, r);
  const RowList mine = load_list<NT>(a, r, list, fs);
  const bool bucket = a.flags & B200GDN_DISTILL_BUCKET;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < a.V; j += NT) m = fmaxf(m, Io<T>::ld(x, j));
  m = cta_reduce<NT>(m, fs, MaxOf());
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, s_off = 0.f;
  for (int j = threadIdx.x; j < a.V; j += NT) {
    const float e = exp2_approx((Io<T>::ld(x, j) - base) * a.scale * kLog2e);
    s += e;
    if (bucket && !on_list(list, a.K, j)) s_off += e;
  }
  s = cta_reduce<NT>(s, fs, SumOf());
  s_off = cta_reduce<NT>(s_off, fs, SumOf());
  const float logs = logf(s);
  float loss = 0.f;
  if (mine.id >= 0 && mine.q != 0.f) loss = s == 0.f ? INFINITY : mine.q * (mine.l - ((Io<T>::ld(x, mine.id) - base) * a.scale - logs));
  loss = cta_reduce<NT>(loss, fs, SumOf());
  float off = mine.total + mine.rest, on = off;
  if (bucket && mine.rest != 0.f) {
    loss += mine.rest * (logf(mine.rest) - (logf(s_off) - logs));
    off = s_off == 0.f ? 0.f : off - mine.rest * (s / s_off);
  }
  if (!mine.counted) loss = off = on = 0.f;
  if (threadIdx.x == 0) {
    a.row_loss[r] = loss;
    if (a.stats) {
      a.stats[4 * r] = base;
      a.stats[4 * r + 1] = logs;
      a.stats[4 * r + 2] = off;
      a.stats[4 * r + 3] = on;
    }
  }
  if (a.dlogits) write_gradient(a, r, x, list, base, logs, off, on, a.scale / (a.flags & B200GDN_DISTILL_MEAN ? (float)a.counters[0] : 1.f));
}

template <typename T>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(const b200gdn_distill_args a) {
  __shared__ List list;
  __shared__ float fs[NT / 32];
  const int64_t r = blockIdx.x;
  float weight;
  if (a.flags & B200GDN_DISTILL_SCALAR) {
    weight = *a.dloss;
    if ((a.flags & B200GDN_DISTILL_SKIP_ONE) && weight == 1.f) return;
    if (a.flags & B200GDN_DISTILL_MEAN) weight /= (float)a.counters[0];
  } else {
    weight = a.dloss[r];
  }
  const T* x = static_cast<const T*>(a.logits) + row_offset(a, r);
  load_list<NT>(a, r, list, fs);
  const float* st = a.stats + 4 * r;
  write_gradient(a, r, x, list, st[0], st[1], st[2], st[3], weight * a.scale);
}

template <typename T>
int launch_t(const b200gdn_distill_args& a, cudaStream_t st, bool bwd) {
  if (bwd) {
    distill_bwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
    return check_launch("distill_bwd");
  }
  if (a.flags & B200GDN_DISTILL_MEAN) {
    distill_count_kernel<<<1, 1024, 0, st>>>(a);
    if (int e = check_launch("distill_count")) return e;
  }
  distill_fwd_kernel<T><<<(unsigned)a.rows, NT, 0, st>>>(a);
  if (int e = check_launch("distill_fwd")) return e;
  if (a.loss == nullptr) return 0;
  distill_sum_kernel<<<1, 1024, 0, st>>>(a);
  return check_launch("distill_sum");
}

}  // namespace

int launch_distill(const b200gdn_distill_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

// Divergence of a student's rows of logits from a teacher's entries, and its gradient.
//
// The rows go by spans as in logprob.cu: sums of 2^u, or with the rest of the vocabulary as an entry those of the entries off the list.  Warps of
// the same launch prepare the teacher's lists: q, its sum and what is left of one, entries given more than once made one.  A second
// kernel joins both to the row's loss and what its gradient needs, a third writes the gradient.
//
// HBM's: two looks at the logits and one write of the gradient.  4096 x 131072 bf16, 64 entries: 498 us (sums 186 to 207, gradient 312),
// 6.5 TB/s of those three; with the rest of the vocabulary as an entry 572 to 592, since every span looks through its row's list.
#include "vocab.cuh"

namespace gdn {
namespace {

// less than this is what rounding leaves of a sum of one, and counts as nothing (a list may hold the whole vocabulary)
constexpr float kRestFrom = 1e-6f;
constexpr int L = B200GDN_MAX_LIST / 32;   // entries of a lane

// What is kept of a row.  A list's entry: its index and q, all occurrences' together at the first, -1 at the others and at absent ones.
struct Entry {
  int id;
  float q;
};
struct RowList {
  float constant;      // sum q log q, the rest's included
  float total, rest;   // sum q; what is left of one
  int counted;
};
// Largest entry and log2 of the sum, of what the list leaves (renormalised: of the row; log_s -infinity: the gradient is zero) and of the
// whole row.  The gradient is the softmax of what is off the list times `by` there, the softmax of the row times `by`, minus q, on it.
struct __align__(16) RowSums {
  struct __align__(16) Part {
    float m, log_s, by, unused;
  } off, row;
};

// The workspace of a call: kept from the forward pass for the backward pass.
struct Work {
  int* counters;     // [2]: rows that count, CTAs that have joined their rows
  RowList* lists;    // [rows]
  RowSums* sums;     // [rows]
  Entry* entries;    // [rows, K]
  float4* part;      // [rows, spans]
  static int64_t bytes(int64_t rows, int K, int per_row) { return rows * (16 + 32 + 8 * (int64_t)K + 16 * (int64_t)per_row) + 16; }
  Work(void* p, int64_t rows, int K, int per_row) {
    part = static_cast<float4*>(p);
    lists = reinterpret_cast<RowList*>(part + rows * per_row);
    sums = reinterpret_cast<RowSums*>(lists + rows);
    entries = reinterpret_cast<Entry*>(sums + rows);
    counters = reinterpret_cast<int*>(entries + rows * K);
  }
};

// an entry of a list: false where it is absent
__device__ __forceinline__ bool load_entry(const b200gdn_distill_args& a, int64_t at, int& id, float& l) {
  id = load_index(a.ids, at, a.id_bytes, a.V);
  l = ld_param(a.teacher, at, a.teacher_dtype);
  if (l == -INFINITY) id = -1;
  return id >= 0;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// ---- a teacher's lists ---------------------------------------------------------------------------------------------------
// One warp: a row's list.
__device__ __forceinline__ void prepare_list(const b200gdn_distill_args& a, const Work& w, int64_t r, int lane) {
  const bool bucket = a.flags & B200GDN_DISTILL_BUCKET;
  int id[L];
  float l[L], q[L], most = -INFINITY;
  bool any = false;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    id[i] = -1;
    l[i] = -INFINITY;
    if (i * 32 + lane < a.K && load_entry(a, r * a.K + i * 32 + lane, id[i], l[i])) {
      any = true;
      most = fmaxf(most, l[i]);
    }
  }
  any = __any_sync(0xffffffffu, any);
  float shift = 0.f;
  if (!bucket) {
    most = warp_max(most);
    if (most == -INFINITY) most = 0.f;   // (no entry but NaN, or none)
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (id[i] >= 0) s += expf(l[i] - most);
    shift = most + logf(warp_sum(s));
  }
  float total = 0.f, constant = 0.f;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    q[i] = id[i] >= 0 ? expf(l[i] - shift) : 0.f;
    total += q[i];
    if (q[i] != 0.f) constant += q[i] * (l[i] - shift);
  }
  total = warp_sum(total);
  constant = warp_sum(constant);
  float rest = bucket ? 1.f - total : 0.f;
  if (rest < kRestFrom) rest = 0.f;
  if (rest != 0.f) constant += rest * logf(rest);
  // entries given more than once: seldom
  bool twice = false;
#pragma unroll
  for (int i = 0; i < L; ++i)
    if (i * 32 < a.K) {
      const unsigned same = __match_any_sync(0xffffffffu, id[i]);
      twice |= id[i] >= 0 && (same & (same - 1)) != 0;
#pragma unroll
      for (int f = i + 1; f < L; ++f)
        if (f * 32 < a.K)
          for (int o = 0; o < 32; ++o) {
            const int other = __shfl_sync(0xffffffffu, id[f], (lane + o) & 31);
            twice |= id[i] >= 0 && other == id[i];
          }
    }
  if (__any_sync(0xffffffffu, twice)) {
    float sum[L];
    bool first[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      sum[i] = 0.f;
      first[i] = true;
    }
#pragma unroll
    for (int f = 0; f < L; ++f)
      if (f * 32 < a.K)
        for (int from = 0; from < 32; ++from) {
          const int other = __shfl_sync(0xffffffffu, id[f], from);
          const float more = __shfl_sync(0xffffffffu, q[f], from);
#pragma unroll
          for (int i = 0; i < L; ++i)
            if (other == id[i]) {
              sum[i] += more;
              if (f * 32 + from < i * 32 + lane) first[i] = false;
            }
        }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      q[i] = sum[i];
      if (!first[i]) id[i] = -1;
    }
  }
#pragma unroll
  for (int i = 0; i < L; ++i)
    if (i * 32 + lane < a.K) w.entries[r * a.K + i * 32 + lane] = Entry{id[i], q[i]};
  if (lane == 0) w.lists[r] = RowList{constant, total, rest, any};
}

// ---- sums ----------------------------------------------------------------------------------------------------------------
// One span's sums.  With the rest of the vocabulary as an entry, entries on the list count as minus infinity.
template <typename T, int W>
__device__ __forceinline__ void sum_span(const b200gdn_distill_args& a, const Work& w, SpanWords<T, W>& words, int per_row, int64_t r, int span, int lane) {
  const Words<T> x(static_cast<const T*>(a.logits) + row_offset(a, r), a.V);
  const float c = a.scale * kLog2e;
  if (a.flags & B200GDN_DISTILL_BUCKET) {
    const int lo = x.first + span * 32 * W * Words<T>::EPW, hi = lo + 32 * W * Words<T>::EPW;
    for (int i = 0; i < a.K; i += 32) {
      const int64_t entry = r * a.K + i + lane;
      int id = i + lane < a.K ? load_index(a.ids, entry, a.id_bytes, a.V) : -1;
      if (id >= 0 && id >= lo && id < hi && ld_param(a.teacher, entry, a.teacher_dtype) == -INFINITY) id = -1;
      unsigned hits = __ballot_sync(0xffffffffu, id >= 0 && id >= lo && id < hi);
      while (hits != 0) {
        const int at = __shfl_sync(0xffffffffu, id, __ffs(hits) - 1) - lo, word = at / Words<T>::EPW, e = at % Words<T>::EPW;
        hits &= hits - 1;
#pragma unroll
        for (int i2 = 0; i2 < W; ++i2)
          if (word == 32 * i2 + lane) {
            T* p = reinterpret_cast<T*>(&words.q[i2]);
#pragma unroll
            for (int e2 = 0; e2 < Words<T>::EPW; ++e2)
              if (e2 == e) p[e2] = static_cast<T>(-INFINITY);
          }
      }
    }
  }
  const Sums v = warp_sums<false>(words.template sums<false>(c), c);
  if (lane == 0) w.part[r * per_row + span] = make_float4(v.m, v.s, 0.f, 0.f);
}

// A row's sums joined: its loss, and what its gradient needs.  One warp, all spans' sums being there.
template <typename T>
__device__ __forceinline__ void join_row(const b200gdn_distill_args& a, const Work& w, int per_row, int64_t r, int lane) {
  const T* row = static_cast<const T*>(a.logits) + row_offset(a, r);
  const float c = a.scale * kLog2e;
  const RowList list = w.lists[r];
  Sums v = joined_spans(w.part + r * per_row, per_row, c, lane);
  const Sums off = v;
  if (a.flags & B200GDN_DISTILL_BUCKET) {   // the entries on the list
    Sums on{-INFINITY, 0.f, 0.f};
    for (int i = lane; i < a.K; i += 32) {
      const Entry e = w.entries[r * a.K + i];
      if (e.id < 0) continue;
      const float x = Io<T>::ld(row, e.id), m = fmaxf(on.m, x);
      on = moved(on, m, c);
      on.s += exp2_approx(exponent(x, m, c));
    }
    on = warp_sums<false>(on, c);
    const float m = fmaxf(v.m, on.m);
    v = moved(v, m, c);
    on = moved(on, m, c);
    v.s += on.s;
  }
  const float log_s = log2f(v.s), ln_s = log_s * kLn2;
  float loss = 0.f;
  for (int i = lane; i < a.K; i += 32) {
    const Entry e = w.entries[r * a.K + i];
    if (e.id >= 0 && e.q != 0.f) loss -= e.q * (exponent(Io<T>::ld(row, e.id), v.m, a.scale) - ln_s);
  }
  loss = warp_sum(loss) + list.constant;
  // What is off the list keeps its own largest entry: its mass P = sum 2^((x - m) c) / s is zero in 32 bits from 87 / scale below the
  // list on, its logarithm and its softmax w are not.  p_j Q - rest p_j / P = w_j (P Q - rest): nothing in it leaves fp32's range.
  const float all = list.total + list.rest;
  RowSums s{{off.m, 0.f, 0.f, 0.f}, {v.m, log_s, all, 0.f}};
  if (off.s != 0.f) {   // something is
    s.off.log_s = log2f(off.s);
    s.off.by = moved(off, v.m, c).s / v.s * all - list.rest;
  }
  if (list.rest != 0.f) loss -= list.rest * (exponent(off.m, v.m, a.scale) + logf(off.s) - ln_s);
  if (!list.counted || v.s == 0.f) {   // none of a teacher's, or no row
    loss = list.counted ? INFINITY : 0.f;
    s.off.log_s = -INFINITY;
  }
  if (lane == 0) {
    a.row_loss[r] = loss;
    w.sums[r] = s;
  }
}

// ---- gradient ------------------------------------------------------------------------------------------------------------
template <typename T, int W>
__device__ __forceinline__ void gradient_span(const b200gdn_distill_args& a, const Work& w, const GradientSpan<T, W>& g, float weight, int64_t r, int span,
                                              int lane) {
  const T* row = static_cast<const T*>(a.logits) + row_offset(a, r);
  T* out = static_cast<T*>(a.dlogits) + r * a.V;
  const RowSums::Part off = w.sums[r].off;
  if (off.log_s == -INFINITY) {
    zero_span<T, W>(out, a.V, span, lane);
    return;
  }
  const float c = a.scale * kLog2e, off_base = off.m == -INFINITY ? 0.f : off.m, by = off.by * weight;
  const uint64_t m2 = pack2(-off_base, -off_base), c2 = pack2(c, c), s2 = pack2(-off.log_s, -off.log_s), by2 = pack2(by, by);
  g.store(out, a.V, span, lane, [&](uint64_t x) {
    const float2 l = unpack2(add2(mul2(add2(x, m2), c2), s2));
    return mul2(pack2(exp2_approx(l.x), exp2_approx(l.y)), by2);
  });
  __syncwarp();
  const RowSums::Part all = w.sums[r].row;
  const float base = all.m == -INFINITY ? 0.f : all.m;
  for (int i = lane; i < a.K; i += 32) {
    const Entry e = w.entries[r * a.K + i];
    if (!in_span<T, W>(out, span, e.id)) continue;
    const float p = exp2_approx((Io<T>::ld(row, e.id) - base) * c - all.log_s);
    Io<T>::st(out, e.id, (p * all.by - e.q) * weight);
  }
}

__device__ __forceinline__ float mean_factor(const b200gdn_distill_args& a, const Work& w) {
  return a.flags & B200GDN_DISTILL_MEAN ? 1.f / (float)max(1, w.counters[0]) : 1.f;
}

// ---- kernels -------------------------------------------------------------------------------------------------------------
// A span of a row, by its number among all.
struct Task {
  int64_t r;
  int span;
  __device__ __forceinline__ Task(int64_t t, int per_row) {
    r = t <= 0xffffffffll ? (int64_t)((uint32_t)t / (uint32_t)per_row) : t / per_row;
    span = (int)(t - r * per_row);
  }
};
template <typename T>
__device__ __forceinline__ const T* logits_of(const b200gdn_distill_args& a, int64_t r) { return static_cast<const T*>(a.logits) + row_offset(a, r); }
template <typename T>
__device__ __forceinline__ T* dlogits_of(const b200gdn_distill_args& a, int64_t r) { return static_cast<T*>(a.dlogits) + r * a.V; }

// the sums of all spans; the first CTAs prepare the lists
template <typename T, int W>
__global__ void __launch_bounds__(32 * kSpanWarps) distill_spans_kernel(const b200gdn_distill_args a, const Work w, int per_row, unsigned list_ctas) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < list_ctas) {
    const int64_t r = (int64_t)blockIdx.x * kSpanWarps + warp;
    if (r < a.rows) prepare_list(a, w, r, lane);
    if (blockIdx.x == 0 && threadIdx.x < 2) w.counters[threadIdx.x] = 0;
    return;
  }
  const Task t((int64_t)(blockIdx.x - list_ctas) * kSpanWarps + warp, per_row);
  if (t.r >= a.rows) return;
  SpanWords<T, W> words(Words<T>(logits_of<T>(a, t.r), a.V), a.V, t.span, lane);
  sum_span<T, W>(a, w, words, per_row, t.r, t.span, lane);
}

// rows joined, a warp each; the CTA that comes last adds up the losses (each thread's and each warp's in a fixed order)
constexpr int kJoinThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) distill_join_kernel(const b200gdn_distill_args a, const Work w, int per_row) {
  __shared__ int counted, last;
  __shared__ float fs[kJoinThreads / 32];
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5);
  wait_for_predecessor();
  if (threadIdx.x == 0) counted = 0;
  __syncthreads();
  if (r < a.rows) {
    join_row<T>(a, w, per_row, r, lane);
    if (lane == 0 && w.lists[r].counted) atomicAdd(&counted, 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (counted > 0) atomicAdd(w.counters, counted);
    __threadfence();
    last = a.loss != nullptr && atomicAdd(w.counters + 1, 1) == (int)gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  int64_t i = threadIdx.x;
  for (; i + 3 * kJoinThreads < a.rows; i += 4 * kJoinThreads)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += __ldcg(a.row_loss + i + e * kJoinThreads);
  for (; i < a.rows; i += kJoinThreads) s[0] += __ldcg(a.row_loss + i);
  const float sum = cta_reduce<kJoinThreads>((s[0] + s[1]) + (s[2] + s[3]), fs, SumOf());
  if (threadIdx.x == 0) *a.loss = a.flags & B200GDN_DISTILL_MEAN ? sum / (float)max(1, __ldcg(w.counters)) : sum;
}

// The gradient, times an upstream gradient where there is one.  From the last row to the first: behind the sums the last rows are still in
// the second-level cache.
template <typename T, int W, bool MAYBE_NONE>
__global__ void __launch_bounds__(32 * kSpanWarps) distill_bwd_kernel(const b200gdn_distill_args a, const Work w, int per_row) {
  const int lane = threadIdx.x & 31;
  wait_for_predecessor();
  const int64_t tasks = a.rows * per_row;
  auto write = [&](int64_t i, float weight) {
    const Task t(tasks - 1 - i, per_row);
    GradientSpan<T, W> g;
    g.load(logits_of<T>(a, t.r), dlogits_of<T>(a, t.r), a.V, t.span, lane);
    const bool by_row = a.dloss != nullptr && !(a.flags & B200GDN_DISTILL_SCALAR);
    gradient_span<T, W>(a, w, g, a.scale * (by_row ? a.dloss[t.r] : weight * mean_factor(a, w)), t.r, t.span, lane);
  };
  const int64_t i = (int64_t)blockIdx.x * kSpanWarps + (threadIdx.x >> 5);
  if constexpr (MAYBE_NONE) {   // no more CTAs than are resident: 65536 that return at once take 70 us
    const float d = *a.dloss;
    if (d == 1.f) return;
    for (int64_t j = i; j < tasks; j += (int64_t)gridDim.x * kSpanWarps) write(j, d);
  } else if (i < tasks) {
    write(i, a.dloss != nullptr && (a.flags & B200GDN_DISTILL_SCALAR) ? *a.dloss : 1.f);
  }
}

template <typename T, int W>
int launch_w(const b200gdn_distill_args& a, const Spans& spans, cudaStream_t st, bool bwd) {
  const Work w(a.workspace, a.rows, a.K, spans.per_row);
  const unsigned grid = (unsigned)((a.rows * spans.per_row + kSpanWarps - 1) / kSpanWarps), lists = (unsigned)((a.rows + kSpanWarps - 1) / kSpanWarps);
  if (!bwd) {
    distill_spans_kernel<T, W><<<lists + grid, 32 * kSpanWarps, 0, st>>>(a, w, spans.per_row, lists);
    if (int e = check_launch("distill_spans")) return e;
    const unsigned joins = (unsigned)((a.rows + kJoinThreads / 32 - 1) / (kJoinThreads / 32));
    launch_overlapped(true, distill_join_kernel<T>, dim3(joins), kJoinThreads, 0, st, a, w, spans.per_row);
    if (int e = check_launch("distill_join")) return e;
    if (a.dlogits == nullptr) return 0;
  }
  if (a.flags & B200GDN_DISTILL_SKIP_ONE) {
    const unsigned resident = (unsigned)resident_ctas<distill_bwd_kernel<T, W, true>>(32 * kSpanWarps, 0);
    distill_bwd_kernel<T, W, true><<<grid < resident ? grid : resident, 32 * kSpanWarps, 0, st>>>(a, w, spans.per_row);
  } else {
    launch_overlapped(!bwd, distill_bwd_kernel<T, W, false>, dim3(grid), 32 * kSpanWarps, 0, st, a, w, spans.per_row);
  }
  return check_launch("distill_bwd");
}

template <typename T>
int launch_t(const b200gdn_distill_args& a, cudaStream_t st, bool bwd) {
  const Spans spans = spans_of(a.V, sizeof(T));
  if (a.rows * (spans.per_row + 1) > (int64_t)(INT32_MAX - 1) * kSpanWarps) return set_error(B200GDN_ERR_UNSUPPORTED, "distill: more than 2^33 spans");
  return spans.w == 8 ? launch_w<T, 8>(a, spans, st, bwd) : spans.w == 4 ? launch_w<T, 4>(a, spans, st, bwd)
         : spans.w == 2 ? launch_w<T, 2>(a, spans, st, bwd) : launch_w<T, 1>(a, spans, st, bwd);
}

}  // namespace

int64_t distill_workspace(int64_t rows, int V, int dtype, int K) { return Work::bytes(rows, K, spans_of(V, dtype == 2 ? 4 : 2).per_row); }

int launch_distill(const b200gdn_distill_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

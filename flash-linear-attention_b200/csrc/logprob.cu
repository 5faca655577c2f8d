// Log probabilities of given tokens, entropy and the most probable entries of rows of logits, and their gradient.
//
// Forward: one look at each logit, by warps that know nothing of one another.  (A row in one cluster, its pieces joined through shared
// memory, came to 4.0 TB/s at best and less with top entries: what has to be said about a row is a chain of a few thousand clocks.)
// A warp takes a span of 32 W words of 16 bytes of a row into registers, and leaves the span's largest entry m and the sums
// s = sum 2^u, t = sum u 2^u; with top entries also the largest entry of each 128 bytes (a group).  A second kernel joins a row's
// spans: lp_j = (u_j - log2 s) ln 2, entropy = (log2 s - t / s) ln 2.
//
// Top entries: the k-th largest of the groups' largest entries, tau, is a bound that at least k entries reach and few more than k exceed; only
// the groups that reach it are read again (k of 2048 in a row of 131072 16-bit logits), and each of the entries found counts how many
// of them are larger, which is its place.  (Groups of a lane's words, 512 bytes from one another, cost no exchange but ten times
// the bytes when they are read again: 2048 rows of 131072, k = 64, 130 us for 122.)
//
// Measured, 131072 16-bit logits a row: 4096 rows with token and entropy 169 us, 6.4 TB/s (the copy rate is 6.56); 2048 rows 89, with 20 top
// entries 113, with 128 138; backward 4096 rows 376 us, 5.7 TB/s.
#include "vocab.cuh"

namespace gdn {
namespace {

// log probability of an entry x; log_s: the base-2 logarithm of the sum, -infinity where nothing is above -infinity
__device__ __forceinline__ float lp_of(float x, float m, float log_s, float scale) {
  return log_s == -INFINITY ? -INFINITY : exponent(x, m, scale) - log_s * kLn2;
}

// values in order as unsigned integers of 16 or 32 bits; 0 for no value at all.  The zeros are one value.
template <typename T>
__device__ __forceinline__ uint32_t ordered(float x) {
  uint32_t b = __float_as_uint(x + 0.f);
  if constexpr (std::is_same<T, __half>::value) b = (uint32_t)__half_as_ushort(__float2half_rn(x + 0.f));
  else if constexpr (sizeof(T) == 2) b >>= 16;
  constexpr uint32_t sign = sizeof(T) == 2 ? 0x8000u : 0x80000000u, all = sizeof(T) == 2 ? 0xffffu : 0xffffffffu;
  return b & sign ? ~b & all : b | sign;
}
template <typename T> using Order = typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type;
template <typename T>
__device__ __forceinline__ float from_ordered(uint32_t o) {
  constexpr uint32_t sign = sizeof(T) == 2 ? 0x8000u : 0x80000000u, all = sizeof(T) == 2 ? 0xffffu : 0xffffffffu;
  const uint32_t b = o & sign ? o & ~sign : ~o & all;
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)b));
  else return __uint_as_float(sizeof(T) == 2 ? b << 16 : b);
}

// Groups of w neighbouring words, 32 a span: the first word of group g of a row.
__device__ __forceinline__ int first_word(int g, int w) { return (g >> 5) * 32 * w + (g & (w - 1)) * 32 + (g & 31 & ~(w - 1)); }

template <typename T, int W, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(32 * kSpanWarps) logprob_spans_kernel(const b200gdn_logprob_args a, const Spans spans, float4* part, void* largest) {
  const int lane = threadIdx.x & 31;
  const int64_t task = (int64_t)blockIdx.x * kSpanWarps + (threadIdx.x >> 5), r = task / spans.per_row;
  const int span = (int)(task - r * spans.per_row);
  if (r >= a.rows) return;
  const Words<T> x(static_cast<const T*>(a.logits) + row_offset(a, r), a.V);
  const float c = a.scale * kLog2e;
  const SpanWords<T, W> words(x, a.V, span, lane);
  const Sums mine = words.template sums<ENTROPY>(c), v = warp_sums<ENTROPY>(mine, c);
  if (lane == 0) part[task] = make_float4(v.m, v.s, v.t, 0.f);
  if constexpr (TOP) {
    // W neighbouring lanes exchange halves until each has the largest entry of W neighbouring words: lane l of words
    // 32 (l mod W) + l - (l mod W) and on
    uint32_t most[W];
#pragma unroll
    for (int i = 0; i < W; ++i) most[i] = largest_of<T>(words.q[i]);
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const uint32_t keep = lane & o ? most[i + o] : most[i], give = lane & o ? most[i] : most[i + o];
        most[i] = max_words<T>(keep, __shfl_xor_sync(0xffffffffu, give, o));
      }
    // (a group without words is 0)
    static_cast<Order<T>*>(largest)[task * 32 + lane] = (Order<T>)(first_word(span * 32 + lane, W) < x.n ? ordered<T>(max_of_word<T>(most[0])) : 0u);
  }
}

// ---- joining a row's spans ---------------------------------------------------------------------------------------------
constexpr int NT = 128, kRoom = 1024;   // threads of a row with top entries; keys of entries that may be among them
constexpr int kBounds = 4 * NT;         // values that tau is the k-th largest of, at most
static_assert(kBounds >= 4 * B200GDN_MAX_TOP && kBounds < 1 << 10 && kRoom >= 2 * B200GDN_MAX_TOP, "entries above tau and as many equal to it as are wanted");

// one thread
template <typename T>
__device__ __forceinline__ void row_results(const b200gdn_logprob_args& a, int64_t r, const Sums& v, float log_s) {
  if (a.logprobs) {
    const int token = load_index(a.tokens, r, a.token_bytes, a.V);
    a.logprobs[r] = token < 0 ? 0.f : lp_of(Io<T>::ld(static_cast<const T*>(a.logits) + row_offset(a, r), token), v.m, log_s, a.scale);
  }
  if (a.entropy) a.entropy[r] = v.s == 0.f ? 0.f : (log_s - v.t / v.s) * kLn2;
  if (a.stats) {
    a.stats[2 * r] = v.m;
    a.stats[2 * r + 1] = log_s;
  }
}

// without top entries: a warp a row
template <typename T>
__global__ void __launch_bounds__(NT) logprob_join_kernel(const b200gdn_logprob_args a, const Spans spans, const float4* part) {
  wait_for_predecessor();
  const int64_t r = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
  if (r >= a.rows) return;
  const int lane = threadIdx.x & 31;
  const Sums v = joined_spans(part + r * spans.per_row, spans.per_row, a.scale * kLog2e, lane);
  if (lane == 0) row_results<T>(a, r, v, log2f(v.s));
}

// The k-th largest of n <= kBounds values (0 where fewer than k are there), two bits at a time from the highest down; of 32 bits the upper 22,
// which bounds it from below as well as tau needs.  One warp.
template <typename T>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* values, int n, int k, int lane) {
  uint32_t v[kBounds / 32];
#pragma unroll
  for (int i = 0; i < kBounds / 32; ++i) v[i] = i * 32 + lane < n ? values[i * 32 + lane] : 0u;
  uint32_t t = 0;
#pragma unroll 1
  for (int bit = sizeof(T) == 2 ? 14 : 30; bit >= (sizeof(T) == 2 ? 0 : 10); bit -= 2) {
    const uint32_t n1 = t | 1u << bit, n2 = t | 2u << bit, n3 = t | 3u << bit;
    uint32_t c = 0;   // three counts in one sum
#pragma unroll
    for (int i = 0; i < kBounds / 32; ++i)
      if (i * 32 < n) c += (v[i] >= n1 ? 1u : 0u) + (v[i] >= n2 ? 1u << 10 : 0u) + (v[i] >= n3 ? 1u << 20 : 0u);
    c = __reduce_add_sync(0xffffffffu, c);
    t = (c >> 20) >= (uint32_t)k ? n3 : (c >> 10 & 0x3ffu) >= (uint32_t)k ? n2 : (c & 0x3ffu) >= (uint32_t)k ? n1 : t;
  }
  return t == 0 ? 0 : max(t, ordered<T>(-INFINITY));   // (the lower bits left out: below minus infinity there are only NaNs)
}

// Keys of a row's entries in the order of their indices, from `found` on; returns how many there are then (those beyond the room are
// not kept).  Of rows with NaN (above everything): those above tau (with tau 0: all) and the first k equal to it.  Of others
// (`ties`) the first k equal to tau alone, and no further than that.  One warp.
template <typename T>
__device__ __noinline__ int keys_in_order(const Words<T>& x, int V, uint32_t tau_bits, int k, bool ties, uint64_t* keys, int found, int lane) {
  const bool everything = tau_bits == 0;
  const float tau = from_ordered<T>(tau_bits);
  int equal = 0;   // entries equal to tau that were met
  for (int j0 = 0; j0 < x.n && !(ties && equal >= k); j0 += 32) {
    const int j = j0 + lane, at = x.first + j * Words<T>::EPW;
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (j < x.n) q = x.at[j];
    const T* w = reinterpret_cast<const T*>(&q);
    auto above = [&](float v) { return !ties && (everything || !(v <= tau)); };
    uint32_t n = 0;   // above tau, and in the upper half equal to it
#pragma unroll
    for (int e = 0; e < Words<T>::EPW; ++e) {
      const float v = Io<T>::ld(w, e);
      if (j < x.n && at + e >= 0 && at + e < V) n += above(v) ? 1u : v == tau ? 0x10000u : 0u;
    }
    if (!__any_sync(0xffffffffu, n != 0)) continue;
    uint32_t before = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, before, 31);
    before -= n;
    int eq = equal + (int)(before >> 16), to = found + (int)(before & 0xffffu) + min(eq, k) - min(equal, k);
    if (n != 0)
#pragma unroll
      for (int e = 0; e < Words<T>::EPW; ++e) {
        const float v = Io<T>::ld(w, e);
        if (at + e < 0 || at + e >= V) continue;
        if (!above(v) && (v != tau || eq++ >= k)) continue;
        if (to < kRoom) keys[to] = entry_key(v, at + e);
        ++to;
      }
    found += (int)(total & 0xffffu) + min(equal + (int)(total >> 16), k) - min(equal, k);
    equal += (int)(total >> 16);
  }
  return found;
}

// with top entries: a CTA a row
template <typename T>
__global__ void __launch_bounds__(NT, 12) logprob_top_kernel(const b200gdn_logprob_args a, const Spans spans, const float4* part, const void* largest) {
  __shared__ __align__(16) uint64_t keys[kRoom];
  __shared__ uint64_t ks[NT / 32];
  __shared__ uint32_t own[kBounds], bound;
  __shared__ uint16_t list[kRoom];
  __shared__ float stats[4];
  __shared__ int n_list, found;
  wait_for_predecessor();
  const int64_t r = a.rows - 1 - blockIdx.x;   // the last rows are still in the second-level cache
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.top_k, groups = spans.groups();
  const Words<T> x(static_cast<const T*>(a.logits) + row_offset(a, r), a.V);
  const Order<T>* of_groups = static_cast<const Order<T>*>(largest) + r * groups;
  // tau from at least four values for each entry that is wanted (of 2 k it would be exceeded by 1.4 k entries, of 4 k by 1.15 k): the
  // largest of the groups i NT + tid, in one, two or four parts.  With few groups tau would be low, and the row is gone through again:
  // the largest entry of each thread's words.
  const bool by_groups = 2 * groups >= 3 * k && groups <= 65536;
  const int parts = !by_groups || k <= NT / 4 ? 1 : k <= NT / 2 ? 2 : 4;
  uint32_t most[4] = {0, 0, 0, 0};
  if (by_groups) {
#pragma unroll 2
    for (int i = tid; i < groups; i += 4 * NT)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e * NT < groups) most[e] = max(most[e], (uint32_t)of_groups[i + e * NT]);
  } else {
    float m = -INFINITY;
    for (int j = tid; j < x.n; j += NT) m = fmaxf(m, max_of_word<T>(largest_of<T>(x.edge(j, a.V))));
    most[0] = tid < x.n ? ordered<T>(m) : 0u;
  }
  const uint32_t even = max(most[0], most[2]), odd = max(most[1], most[3]), mine = max(even, odd);
  own[tid] = parts == 1 ? mine : parts == 2 ? even : most[0];
  if (parts > 1) own[NT + tid] = parts == 2 ? odd : most[1];
  if (parts > 2) own[2 * NT + tid] = most[2], own[3 * NT + tid] = most[3];
  __syncthreads();
  if (warp == 0) {
    const uint32_t t = kth_largest<T>(own, parts * NT, k, lane);
    if (lane == 0) bound = t;
  } else if (warp == 1) {
    const Sums v = joined_spans(part + r * spans.per_row, spans.per_row, a.scale * kLog2e, lane);
    if (lane == 0) {
      stats[0] = v.m;
      stats[1] = log2f(v.s);
      stats[2] = v.s;
      stats[3] = v.t;
      n_list = found = 0;
    }
  }
  __syncthreads();
  const uint32_t tau = bound;
  const float m = stats[0], log_s = stats[1], least = from_ordered<T>(tau);
  if (tid == NT - 1) row_results<T>(a, r, Sums{m, stats[2], stats[3]}, log_s);
  // The entries that reach tau, of the groups (or threads) whose largest does; `strictly`: that are above it.
  auto look = [&](const uint4& q, int j, bool strictly) {
    if (!(max_of_word<T>(largest_of<T>(q)) >= least)) return;
    unsigned hits = 0;   // seldom more than one
#pragma unroll
    for (int e = 0; e < Words<T>::EPW / 2; ++e) {
      const float2 p = unpack2(pair_of<T>(q, e));
      hits |= ((strictly ? p.x > least : p.x >= least) ? 1u << (2 * e) : 0u) | ((strictly ? p.y > least : p.y >= least) ? 2u << (2 * e) : 0u);
    }
    while (hits != 0) {
      const int e = __ffs(hits) - 1, at = x.first + j * Words<T>::EPW + e;
      hits &= hits - 1;
      if (at < 0 || at >= a.V) continue;
      const int to = atomicAdd(&found, 1);
      if (to < kRoom) keys[to] = entry_key(Io<T>::ld(x.at, (int64_t)j * Words<T>::EPW + e), at);
    }
  };
  auto collect = [&](bool strictly) {   // returns how many there are, more than the room where they are not all kept
    if (by_groups) {
      auto reaches = [&](uint32_t largest) { return strictly ? largest > tau : largest >= tau; };
      if (reaches(mine))
        for (int g = tid; g < groups; g += NT)
          if (reaches(of_groups[g])) {
            const int to = atomicAdd(&n_list, 1);
            if (to < kRoom) list[to] = (uint16_t)g;
          }
      __syncthreads();
      const int n = n_list;
      // (many more groups than entries are wanted: most of them no more than equal to tau)
      if (n > (strictly ? kRoom : 128 + 4 * k)) return kRoom + 1;
      constexpr int U = 4;   // words of a thread on their way at once
      const int shift = spans.shift();
      for (int i = tid; i < n << shift; i += U * NT) {
        uint4 q[U];
        int j[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = i + u * NT, g = at < n << shift ? list[at >> shift] : 0;
          j[u] = at < n << shift ? first_word(g, spans.w) + (at & (spans.w - 1)) : x.n;
          q[u] = j[u] < x.n ? x.at[j[u]] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (j[u] < x.n) look(q[u], j[u], strictly);
      }
    } else if (mine >= tau) {
      for (int j = tid; j < x.n; j += NT) look(x.at[j], j, strictly);
    }
    __syncthreads();
    return found;
  };
  const bool numbers = stats[2] == stats[2];   // no NaN (nor infinity) in the row
  int n = kRoom + 1;
  if (tau != 0 && numbers) {
    n = collect(false);
    if (n > kRoom) {   // masked rows and the like: those above tau, then of those equal to it the first
      __syncthreads();
      if (tid == 0) n_list = found = 0;
      __syncthreads();
      n = collect(true);
    }
    __syncthreads();
    if (n < k) {
      if (warp == 0) {
        const int more = keys_in_order<T>(x, a.V, tau, k - n, true, keys, n, lane);
        if (lane == 0) found = more;
      }
      __syncthreads();
      n = found;
    }
  } else {
    if (warp == 0) {
      const int more = keys_in_order<T>(x, a.V, tau, k, false, keys, 0, lane);
      if (lane == 0) found = more;
    }
    __syncthreads();
    n = found;
  }
  auto result = [&](int place, uint64_t key) {
    a.top_ids[r * k + place] = key_index(key);
    a.top_logprobs[r * k + place] = lp_of(key_value(key), m, log_s, a.scale);
  };
  if (n > kRoom) {   // some thousand entries above tau, all in fewer than k groups: one search through the row for each top entry
    uint64_t below = ~0ull;
    for (int i = 0; i < k; ++i) {
      uint64_t best = 0;
      for (int j = tid; j < a.V; j += NT) {
        const uint64_t key = entry_key(Io<T>::ld(x.at, j - x.first), j);
        if (key < below && key > best) best = key;
      }
      below = cta_reduce<NT>(best, ks, MaxOf());
      if (tid == 0) result(i, below);
    }
    return;
  }
  if (tid == 0 && n % 2 != 0 && n < kRoom) keys[n] = 0;   // (below every entry's)
  __syncthreads();
  const ulonglong2* two = reinterpret_cast<const ulonglong2*>(keys);
  for (int i = tid; i < n; i += NT) {
    const uint64_t key = keys[i];
    int larger = 0;
#pragma unroll 4
    for (int o = 0; o < (n + 1) / 2; ++o) {
      const ulonglong2 p = two[o];
      larger += (p.x > key) + (p.y > key);
    }
    if (larger < k) result(larger, key);
  }
}

template <typename T, int W>
int launch_spans(const b200gdn_logprob_args& a, const Spans& spans, float4* part, void* largest, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.rows * spans.per_row + kSpanWarps - 1) / kSpanWarps);
  auto go = [&](auto kern) { kern<<<grid, 32 * kSpanWarps, 0, st>>>(a, spans, part, largest); };
  if (a.top_k > 0) {
    if (a.entropy) go(logprob_spans_kernel<T, W, true, true>);
    else go(logprob_spans_kernel<T, W, false, true>);
  } else {
    if (a.entropy) go(logprob_spans_kernel<T, W, true, false>);
    else go(logprob_spans_kernel<T, W, false, false>);
  }
  return check_launch("logprob_spans");
}

template <typename T>
int launch_fwd(const b200gdn_logprob_args& a, cudaStream_t st) {
  const Spans spans = spans_of(a.V, sizeof(T));
  if (a.rows * spans.per_row > (int64_t)INT32_MAX * kSpanWarps) return set_error(B200GDN_ERR_UNSUPPORTED, "logprob_fwd: more than 2^33 spans");
  float4* part = static_cast<float4*>(a.workspace);
  void* largest = part + a.rows * spans.per_row;
  int e = spans.w == 8 ? launch_spans<T, 8>(a, spans, part, largest, st) : spans.w == 4 ? launch_spans<T, 4>(a, spans, part, largest, st)
          : spans.w == 2 ? launch_spans<T, 2>(a, spans, part, largest, st) : launch_spans<T, 1>(a, spans, part, largest, st);
  if (e) return e;
  if (a.top_k > 0) launch_overlapped(true, logprob_top_kernel<T>, dim3((unsigned)a.rows), NT, 0, st, a, spans, part, largest);
  else launch_overlapped(true, logprob_join_kernel<T>, dim3((unsigned)((a.rows + NT / 32 - 1) / (NT / 32))), NT, 0, st, a, spans, part);
  return check_launch(a.top_k > 0 ? "logprob_top" : "logprob_join");
}

// ---- gradient ----------------------------------------------------------------------------------------------------------
// dx = scale p (-(A + dH (lp + H))) plus what the given entries get: with l = log2 p,  p (a0 + a1 l).  Two exponent instructions for
// every four bytes moved: HBM's.
template <typename T, int W>
__global__ void __launch_bounds__(32 * kSpanWarps) logprob_bwd_kernel(const b200gdn_logprob_args a, const Spans spans) {
  const int lane = threadIdx.x & 31;
  // from the last row to the first: behind the forward pass the last rows are still in the second-level cache
  const int64_t task = a.rows * spans.per_row - 1 - ((int64_t)blockIdx.x * kSpanWarps + (threadIdx.x >> 5)), r = task / spans.per_row;
  if (task < 0) return;
  const int span = (int)(task - r * spans.per_row);
  const T* row = static_cast<const T*>(a.logits) + row_offset(a, r);
  T* out = static_cast<T*>(a.dlogits) + r * a.V;
  const float m = a.stats[2 * r], log_s = a.stats[2 * r + 1], c = a.scale * kLog2e;
  if (log_s == -INFINITY) {   // nothing in this row
    zero_span<T, W>(out, a.V, span, lane);
    return;
  }
  const int token = a.dlogprobs ? load_index(a.tokens, r, a.token_bytes, a.V) : -1;
  const float dlp = token < 0 ? 0.f : a.dlogprobs[r], dh = a.dentropy ? a.dentropy[r] : 0.f, h = a.dentropy ? a.entropy[r] : 0.f;
  const int k = a.dtop_logprobs ? a.top_k : 0;
  constexpr int L = B200GDN_MAX_TOP / 32;
  int id[L];
  float d[L], all = 0.f;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const bool there = i * 32 + lane < k;
    id[i] = there ? (int)a.top_ids[r * k + i * 32 + lane] : -1;
    d[i] = there ? a.dtop_logprobs[r * k + i * 32 + lane] : 0.f;
    all += d[i];
  }
  if (k > 0)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  all += dlp;
  const float a0 = -(all + dh * h) * a.scale, a1 = -dh * kLn2 * a.scale, base = m == -INFINITY ? 0.f : m;
  const uint64_t m2 = pack2(-base, -base), c2 = pack2(c, c), s2 = pack2(-log_s, -log_s), a02 = pack2(a0, a0), a12 = pack2(a1, a1);
  auto grad = [&](uint64_t x) {   // (of masked entries p is zero, and l bounded)
    const float2 l = unpack2(add2(mul2(add2(x, m2), c2), s2));
    return mul2(pack2(exp2_approx(l.x), exp2_approx(l.y)), fma2(a12, pack2(fmaxf(l.x, -1024.f), fmaxf(l.y, -1024.f)), a02));
  };
  GradientSpan<T, W> g;
  g.load(row, out, a.V, span, lane);
  g.store(out, a.V, span, lane, grad);
  // the given entries again, from the lanes that hold them
  __syncwarp();
  auto again = [&](int j, float more) {
    const float x = Io<T>::ld(row, j);
    Io<T>::st(out, j, unpack2(grad(pack2(x, x))).x + more * a.scale);
  };
  bool listed = false;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    if (id[i] < 0) continue;
    listed |= id[i] == token;
    if (in_span<T, W>(out, span, id[i])) again(id[i], d[i] + (id[i] == token ? dlp : 0.f));
  }
  listed = __any_sync(0xffffffffu, listed);
  if (lane == 0 && token >= 0 && !listed && in_span<T, W>(out, span, token)) again(token, dlp);
}

template <typename T>
int launch_bwd(const b200gdn_logprob_args& a, cudaStream_t st) {
  const Spans spans = spans_of(a.V, sizeof(T));
  if (a.rows * spans.per_row > (int64_t)INT32_MAX * kSpanWarps) return set_error(B200GDN_ERR_UNSUPPORTED, "logprob_bwd: more than 2^33 spans");
  const unsigned grid = (unsigned)((a.rows * spans.per_row + kSpanWarps - 1) / kSpanWarps);
  auto go = [&](auto kern) { kern<<<grid, 32 * kSpanWarps, 0, st>>>(a, spans); };
  if (spans.w == 8) go(logprob_bwd_kernel<T, 8>);
  else if (spans.w == 4) go(logprob_bwd_kernel<T, 4>);
  else if (spans.w == 2) go(logprob_bwd_kernel<T, 2>);
  else go(logprob_bwd_kernel<T, 1>);
  return check_launch("logprob_bwd");
}

template <typename T>
int launch_t(const b200gdn_logprob_args& a, cudaStream_t st, bool bwd) { return bwd ? launch_bwd<T>(a, st) : launch_fwd<T>(a, st); }

}  // namespace

int64_t logprob_workspace(int64_t rows, int V, int dtype, int top_k) {
  const Spans spans = spans_of(V, dtype == 2 ? 4 : 2);
  return rows * spans.per_row * (16 + (top_k > 0 ? 32 * (dtype == 2 ? 4 : 2) : 0));
}

int launch_logprob(const b200gdn_logprob_args& a, cudaStream_t st, bool bwd) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16>(a, st, bwd) : a.dtype == 1 ? launch_t<__half>(a, st, bwd) : launch_t<float>(a, st, bwd);
}

}  // namespace gdn

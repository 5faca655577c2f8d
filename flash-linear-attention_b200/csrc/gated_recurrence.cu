// Gated recurrence, elementwise: h_t = exp(g_t) h_{t-1} + x_t along each sequence, forward and backward.
//     forward   over R tokens of a warp with a = exp(g): h' = their recurrence from 0 and A = their product of a; entered with s they leave
//               A s + h'
//     backward  u_t = a_t (dh_t + u_{t+1}) from the right in the same way; dx_t = dh_t + u_{t+1}, dg_t = dx_t a_t h_{t-1}
// HBM streaming: what counts is that every tensor is read once.  A CTA owns 64 neighbouring channels of a sequence, two a lane, and walks it in
// steps of W R tokens, R for each of its W = 8 warps: each warp joins its own tokens, leaves (A, h') in shared memory, and after one barrier
// a step goes through the warps ahead of it for the state its first token sees, then through its tokens again.  Where there are fewer
// sequences x channel tiles than SMs (or some sequences are much longer than others), CTAs of a cluster share a sequence: step by step each
// takes its turn of W R tokens, and their joined pairs go to one another's shared memory.  Tokens come by TMA, two steps ahead where a step's tiles are
// 32 KB (forward with gates of x's type, backward of 16-bit x with fp32 gates), one where they are 48 (the others); where rows are not a multiple of 16 bytes, to
// registers one step ahead.
// The backward pass does not read h, which is rounded to its type, but forms it again from x in fp32; the forward pass leaves the state
// ahead of every 64 tokens (a 32nd of x's bytes in bf16) so that this needs no pass of its own from the left.
// Bound by instructions where warps are few (39 a row of 64 channels forward, 17 of them the decays), by memory where they are many.  Measured: 16 x 1024 x 8192
// bf16 forward 139 us (123 at copy rate), backward 242 (205); 4 x 4096 x 2048, 128 pieces of work, 52 and 73 (31 and 51); 131072 x 1024 with
// fp32 decays, 16 pieces in clusters of 12, 272 (164); 8191 x 1003 fp32, 16 pieces, 40 and 59 (15 and 25).
#include "gdn_common.cuh"
#include "rowio.cuh"
#include "tc5.cuh"
#include "tma.cuh"

namespace gdn {
namespace {

__device__ int g_recurrence_timeout = 0;

constexpr int MOST_RANKS = 16;   // CTAs of a cluster

// A lane's two channels of a token, as loaded: neighbours in one access (APART 1), or 32 apart where rows do not allow that (APART 32).  `two`:
// there is a second one.
constexpr int WIDTH = 64;   // channels of a CTA
template <int APART>
__device__ __forceinline__ int channel_of(int lane) { return APART == 1 ? 2 * lane : lane; }

template <typename T, int APART>
struct Piece {
  using Raw = std::conditional_t<sizeof(T) == 4, uint2, uint32_t>;
  Raw u;
  __device__ __forceinline__ void zero() { u = Raw{}; }
  __device__ __forceinline__ void load(const T* p, bool two) {
    if constexpr (APART == 1) {
      u = __ldcs(reinterpret_cast<const Raw*>(p));
    } else if constexpr (sizeof(T) == 4) {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
      u.x = __ldcs(q);
      u.y = two ? __ldcs(q + APART) : 0u;
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      const uint32_t lo = __ldcs(q), hi = two ? __ldcs(q + APART) : 0;
      u = lo | hi << 16;
    }
  }
  __device__ __forceinline__ void take(const void* shared) { u = *static_cast<const Raw*>(shared); }   // (neighbours)
  __device__ __forceinline__ uint64_t pair() const {
    if constexpr (sizeof(T) == 2) return widen2<T>(u);
    else return pack2(__uint_as_float(u.x), __uint_as_float(u.y));
  }
  // the pair within [-88, 89]; a NaN stays
  __device__ __forceinline__ uint64_t gate() const {
    if constexpr (sizeof(T) == 4) {
      float2 f = unpack2(pair());
      asm("max.NaN.f32 %0, %0, 0fC2B00000;\n min.NaN.f32 %0, %0, 0f42B20000;" : "+f"(f.x));
      asm("max.NaN.f32 %0, %0, 0fC2B00000;\n min.NaN.f32 %0, %0, 0f42B20000;" : "+f"(f.y));
      return pack2(f.x, f.y);
    } else {
      uint32_t w = u;
      if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;\n min.NaN.f16x2 %0, %0, %2;" : "+r"(w) : "r"(0xD580D580u), "r"(0x55905590u));
      else asm("max.NaN.bf16x2 %0, %0, %1;\n min.NaN.bf16x2 %0, %0, %2;" : "+r"(w) : "r"(0xC2B0C2B0u), "r"(0x42B242B2u));
      return widen2<T>(w);
    }
  }
  static __device__ __forceinline__ void store(T* p, uint64_t x, bool two) {
    if constexpr (APART == 1) {
      if constexpr (sizeof(T) == 2) __stcs(reinterpret_cast<uint32_t*>(p), narrow2<T>(x));
      else __stcs(reinterpret_cast<float2*>(p), unpack2(x));
    } else {
      const float2 f = unpack2(x);
      p[0] = static_cast<T>(f.x);
      if (two) p[APART] = static_cast<T>(f.y);
    }
  }
};

// exp of a pair: 2^n 2^f with n the nearest integer to g log2 e and a polynomial of degree six for 2^f on [-1/2, 1/2] (least squares of the
// relative error: 6e-9 root mean square, 1.6e-8 at most), in pairs of operations.  Off by 1.5 units of 2^-24 at most and 0.1
// on average where |g| < 1 (beyond, log2 e as a float adds |g| / 4).  The average is what counts here: a
// channel that remembers a thousand tokens multiplies as many decays, and ex2.approx, which is 0.4 units too small on average (measured),
// would leave its state off by 2.4e-5.  Below 2^-126.5 the result is zero.
__device__ __forceinline__ uint64_t decay(uint64_t g) {   // of a g in [-88, 89]: there 2^n is zero, infinity
  const uint64_t log2e = pack2(1.4426950408889634f, 1.4426950408889634f), bias = pack2(12582912.f, 12582912.f);
  const uint64_t t = fma2(g, log2e, bias);   // 1.5 2^23 + n: n in the lowest bits
  const uint64_t f = fma2(g, log2e, fma2(t, pack2(-1.f, -1.f), bias));
  auto k = [](float c) { return pack2(c, c); };
  uint64_t p = fma2(k(1.5353350318036973e-4f), f, k(1.3398875016719103e-3f));
  p = fma2(p, f, k(9.618437848985195e-3f));
  p = fma2(p, f, k(5.5503323674201965e-2f));
  p = fma2(p, f, k(0.24022647738456726f));
  p = fma2(p, f, k(0.6931471824645996f));
  p = fma2(p, f, k(1.f));
  const float2 n = unpack2(t);
  const float lo = __uint_as_float((__float_as_uint(n.x) << 23) + 0x3f800000u), hi = __uint_as_float((__float_as_uint(n.y) << 23) + 0x3f800000u);
  return mul2(p, pack2(lo, hi));
}

struct Span {   // the tokens of a sequence, and the index of its first chunk
  int64_t first;
  int len, chunk;
};
__device__ __forceinline__ Span span_of(const b200gdn_gated_recurrence_args& a, int seq) {
  if (a.seq_len > 0) return Span{(int64_t)seq * a.seq_len, a.seq_len, (int)(seq * (int64_t)((a.seq_len + BT - 1) / BT))};
  const int c = a.seq_meta[2 * seq], n = a.seq_meta[2 * seq + 1];
  if (n == 0) return Span{0, 0, 0};
  const ChunkMeta head = load_chunk_meta(a.chunk_meta, c), tail = load_chunk_meta(a.chunk_meta, c + n - 1);
  return Span{head.row, tail.row + tail.len - head.row, c};
}

template <int APART>
__device__ __forceinline__ uint64_t load_state(const float* p, int64_t at, bool there, bool two) {
  if (p == nullptr || !there) return 0ull;
  return pack2(p[at], two ? p[at + APART] : 0.f);
}
template <int APART>
__device__ __forceinline__ void store_state(float* p, int64_t at, uint64_t x, bool two) {
  const float2 f = unpack2(x);
  p[at] = f.x;
  if (two) p[at + APART] = f.y;
}

// [0]: the product of the decays, [1]: what the tokens leave of themselves
struct Joined {
  uint64_t a, h;
};

// A state that is infinite stays so for as long as decays are not zero, but their product over many tokens may leave fp32's range.  Such a product is
// kept as -0, one of decays of which one is zero as +0: a finite state they carry alike (a decay is never negative), and where a joined state
// comes out as NaN it is formed again by `carry`, which tells them apart.
__device__ __forceinline__ bool any_zero(uint64_t a) {
  const float2 f = unpack2(a);
  return f.x == 0.f || f.y == 0.f;
}
__device__ __forceinline__ bool any_nan(uint64_t a) {
  const float2 f = unpack2(a);
  return f.x != f.x || f.y != f.y;
}
__device__ __forceinline__ float carry(float a, float s, float h) {   // a s + h
  return __float_as_uint(a) == 0x80000000u && isinf(s) ? s + h : fmaf(a, s, h);
}
template <int R>
__device__ __forceinline__ uint64_t signed_product(uint64_t product, const uint64_t (&decays)[R]) {
  if (!any_zero(product)) return product;
  float2 least = unpack2(decays[0]);
#pragma unroll
  for (int r = 1; r < R; ++r) {
    const float2 f = unpack2(decays[r]);
    least.x = fminf(least.x, f.x);
    least.y = fminf(least.y, f.y);
  }
  const float2 p = unpack2(product);
  return pack2(p.x == 0.f && least.x > 0.f ? -0.f : p.x, p.y == 0.f && least.y > 0.f ? -0.f : p.y);
}
__device__ __forceinline__ uint64_t carry(uint64_t a, uint64_t s, uint64_t h) {
  const float2 u = unpack2(a), v = unpack2(s), w = unpack2(h);
  return pack2(carry(u.x, v.x, w.x), carry(u.y, v.y, w.y));
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {   // the same place in another CTA of the cluster
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(tc5::smem_addr(p)), "r"(rank));
  return a;
}
// from this CTA's shared memory into another's, counted on its barrier
__device__ __forceinline__ void send(uint32_t to, uint32_t from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(to), "r"(from), "r"(bytes), "r"(bar)
               : "memory");
}

// A wait that has run out is told at the end and not repeated: what follows is invalid, but every thread still comes to the end.  Nothing more is
// loaded then, and at the end the first warp, which loads, waits once more for what is on its way, so that no copy outlives its CTA.
struct Patience {
  int stopped = -1;   // the first step whose tokens were not waited for
  __device__ __forceinline__ bool ok() const { return stopped < 0; }
  __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, int step) {
    if (ok() && !tc5::mbar_wait_warp(bar, parity)) stopped = step;
  }
};

// What the warps of a CTA, and the CTAs of a cluster, leave for one another.  A buffer is written again two steps later: by then every warp has
// passed the barrier of the step between, and so has every CTA of the cluster, whose joined pair of that step has come in.
// Between CTAs 512 bytes go as one copy: stores that count on the other's barrier lane by lane cost 0.28 us a CTA of the cluster, a
// barrier of the whole cluster more, since it waits for every store on its way to memory.
template <int W, bool CLUSTER>
struct Exchange {
  ulonglong2 warps[2][W][32];
  uint64_t carry[2][32];   // what enters the step, and what leaves it, without a cluster
  ulonglong2 ranks[CLUSTER ? 2 : 1][CLUSTER ? MOST_RANKS : 1][32], mine[CLUSTER ? 2 : 1][32];
  uint64_t came[2];        // the joined pairs of all CTAs

  __device__ __forceinline__ void init() {
    if constexpr (CLUSTER) {
      if (threadIdx.x == 0) {
        tc5::mbar_init(&came[0], 1);
        tc5::mbar_init(&came[1], 1);
        tc5::fence_mbar_init();
      }
      __syncthreads();
      cluster_sync();
    }
  }
  __device__ __forceinline__ void enter(uint64_t s) {   // what enters the first step
    if (W > 1 && !CLUSTER && threadIdx.x < 32) carry[0][threadIdx.x] = s;
  }
  __device__ __forceinline__ void leave(int n, bool ok) {   // after n steps; no CTA ends while another one may still send to it
    if constexpr (CLUSTER) {
      if (!ok && threadIdx.x < 32)
        for (int i = n > 2 ? n - 2 : 0; i < n; ++i) (void)tc5::mbar_wait_warp(&came[i & 1], (i >> 1) & 1);
      cluster_sync();
    }
  }
};

// What enters warp `warp` of this CTA at step `i`: W warps of each of the cluster's CTAs, from the first one to the last (REVERSE: from the last to
// the first).  s: what enters the step, then what leaves it (of a CTA without a cluster only the last warp knows, and tells the others at
// the next step).  `meanwhile` runs once all warps have their tokens in registers.
template <int W, bool CLUSTER, bool REVERSE, typename F>
__device__ __forceinline__ uint64_t join(Exchange<W, CLUSTER>& x, int i, int warp, int rank, int n_ranks, Joined own, uint64_t& s, Patience& patience,
                                         F meanwhile) {
  const int lane = threadIdx.x & 31, turn = i & 1, ahead_of = REVERSE ? W - 1 - warp : warp;   // warps ahead of this one
  if constexpr (W == 1) {
    const uint64_t mine = s;
    s = fma2(own.a, s, own.h);
    if (any_nan(s)) s = carry(own.a, mine, own.h);
    return mine;
  } else {
    x.warps[turn][warp][lane] = make_ulonglong2(own.a, own.h);
    __syncthreads();
    meanwhile();
    auto at = [&](int q) { return x.warps[turn][REVERSE ? W - 1 - q : q][lane]; };
    if constexpr (!CLUSTER) {
      uint64_t mine = x.carry[turn][lane];
#pragma unroll
      for (int q = 0; q < W - 1; ++q)
        if (q < ahead_of) {
          const ulonglong2 p = at(q);
          mine = fma2(p.x, mine, p.y);
        }
      s = fma2(own.a, mine, own.h);
      if (any_nan(s)) {
        mine = x.carry[turn][lane];
#pragma unroll 1
        for (int q = 0; q < ahead_of; ++q) mine = carry(at(q).x, mine, at(q).y);
        const ulonglong2 p = at(ahead_of);
        s = carry(p.x, mine, p.y);
      }
      if (ahead_of == W - 1) x.carry[turn ^ 1][lane] = s;
      return mine;
    } else {
      auto ahead_at = [&](int n) {   // what the first n warps come to
        Joined ahead = {pack2(1.f, 1.f), 0ull};
#pragma unroll
        for (int q = 0; q < W; ++q)
          if (q < n) {
            const ulonglong2 p = at(q);
            ahead.h = fma2(p.x, ahead.h, p.y);
            ahead.a = mul2(p.x, ahead.a);
          }
        return ahead;
      };
      auto with_sign = [](uint64_t product, uint32_t least_x, uint32_t least_y) {   // by the least of the factors' bits
        const float2 p = unpack2(product);
        return pack2(p.x == 0.f ? least_x == 0u ? 0.f : -0.f : p.x, p.y == 0.f ? least_y == 0u ? 0.f : -0.f : p.y);
      };
      auto carefully = [&](Joined ahead, int n) {
        uint32_t least_x = ~0u, least_y = ~0u;
        ahead.h = 0ull;
#pragma unroll 1
        for (int q = 0; q < n; ++q) {
          const ulonglong2 p = at(q);
          const float2 f = unpack2(p.x);
          least_x = min(least_x, __float_as_uint(f.x));
          least_y = min(least_y, __float_as_uint(f.y));
          ahead.h = carry(p.x, ahead.h, p.y);
        }
        ahead.a = with_sign(ahead.a, least_x, least_y);
        return ahead;
      };
      // warp 0 joins all of them, to tell the other CTAs
      Joined ahead = ahead_at(warp == 0 ? W : ahead_of);
      if (warp == 0) {
        if (any_nan(ahead.h)) {
          ahead = carefully(ahead, W);
        } else if (any_zero(ahead.a)) {   // (common where channels forget, and on the way from CTA to CTA: no loop)
          uint32_t least_x = ~0u, least_y = ~0u;
#pragma unroll
          for (int q = 0; q < W; ++q) {
            const float2 f = unpack2(at(q).x);
            least_x = min(least_x, __float_as_uint(f.x));
            least_y = min(least_y, __float_as_uint(f.y));
          }
          ahead.a = with_sign(ahead.a, least_x, least_y);
        }
        x.mine[turn][lane] = make_ulonglong2(ahead.a, ahead.h);
        tc5::fence_async_smem();
        if (lane == 0) tc5::mbar_expect_tx(&x.came[turn], n_ranks * 512);
        __syncwarp();
        if (lane < n_ranks) send(at_rank(&x.ranks[turn][rank][0], lane), tc5::smem_addr(&x.mine[turn][0]), 512, at_rank(&x.came[turn], lane));
        // ahead of warp 0: nothing, or (REVERSE) the others
        if constexpr (REVERSE) ahead = ahead_at(W - 1);
        else ahead = {pack2(1.f, 1.f), 0ull};
      }
      patience.wait(&x.came[turn], (i >> 1) & 1, i + 1);
      const uint64_t first = s;
      uint64_t entering = s;
#pragma unroll 4
      for (int q = 0; q < n_ranks; ++q) {
        const int r = REVERSE ? n_ranks - 1 - q : q;
        const ulonglong2 p = x.ranks[turn][r][lane];
        if (r == rank) entering = s;
        s = fma2(p.x, s, p.y);
      }
      uint64_t mine = fma2(ahead.a, entering, ahead.h);
      if (any_nan(add2(s, mine))) {   // (a sum of infinities of both signs too: no harm)
        s = first;
#pragma unroll 1
        for (int q = 0; q < n_ranks; ++q) {
          const int r = REVERSE ? n_ranks - 1 - q : q;
          const ulonglong2 p = x.ranks[turn][r][lane];
          if (r == rank) entering = s;
          s = carry(p.x, s, p.y);
        }
        ahead = carefully(ahead, ahead_of);
        mine = carry(ahead.a, entering, ahead.h);
      }
      return mine;
    }
  }
}
// the warp that knows what leaves the last step
template <int W, bool CLUSTER, bool REVERSE>
__device__ __forceinline__ bool knows_the_end(int n, int warp, int rank) { return rank == 0 && warp == (CLUSTER || REVERSE || n == 0 ? 0 : W - 1); }

struct Place {   // of a CTA: its sequence, the lane's first channel and the tile's
  int seq, channel, tile, rank, n_ranks;
};
template <int APART, bool CLUSTER>
__device__ __forceinline__ Place place_of(const b200gdn_gated_recurrence_args& a) {
  const int tiles = (a.D + WIDTH - 1) / WIDTH;
  const int n = CLUSTER ? (int)cluster_size() : 1;
  const int i = blockIdx.x / n, seq = i / tiles, first = (i % tiles) * WIDTH;
  return Place{a.seq_order ? a.seq_order[seq] : seq, first + channel_of<APART>(threadIdx.x & 31), first, CLUSTER ? (int)cluster_rank() : 0, n};
}

// The tensors that a step reads, in tiles of [W R tokens][64 channels], STAGES steps deep, by TMA: `full` counts a stage's bytes.  Tokens
// past the end of the tensor and channels past its last one arrive as zeros, tokens past the sequence's end are another sequence's.
template <int N, int ROWS, int STAGES>
struct Tiles {
  unsigned char* base;
  uint64_t* full;
  int bytes[N];    // of a row
  int offset[N + 1];   // within a stage

  __device__ __forceinline__ void init(unsigned char* shared, uint64_t* bars, const int (&row_bytes)[N]) {
    base = shared;
    full = bars;
    offset[0] = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      bytes[i] = row_bytes[i];
      offset[i + 1] = offset[i] + row_bytes[i] * ROWS;
    }
    if (threadIdx.x == 0) {
      for (int s = 0; s < STAGES; ++s) tc5::mbar_init(&full[s], 1);
      tc5::fence_mbar_init();
    }
    __syncthreads();
  }
  // one thread
  __device__ __forceinline__ void load(int stage, const CUtensorMap* const (&maps)[N], int channel, int row) const {
    tc5::mbar_expect_tx(&full[stage], offset[N]);
#pragma unroll
    for (int i = 0; i < N; ++i) tma::load_2d(base + stage * offset[N] + offset[i], maps[i], channel, row, &full[stage]);
  }
  // the warp that loads, where a wait has run out: what was loaded of the n steps from `first` on
  __device__ __forceinline__ void land(int first, int n) const {
    for (int i = first; i < first + STAGES && i < n; ++i) (void)tc5::mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1);
  }
  __device__ __forceinline__ const unsigned char* row(int stage, int i, int r) const { return base + stage * offset[N] + offset[i] + r * bytes[i]; }
};
constexpr int stages_of(int stage_bytes, bool cluster) {   // two CTAs an SM
  const int room = (cluster ? 76 : 95) * 1024 / stage_bytes;
  return room >= 2 ? 2 : 1;   // (four are no faster)
}

// ---- forward -------------------------------------------------------------------------------------------------------------
// TMA: the tokens come by way of shared memory, one or two steps ahead; else (odd widths and boundaries) straight to registers, one step ahead.
template <typename T, typename G, int APART, int R, int W, bool CLUSTER, bool TMA>
__global__ void __launch_bounds__(W * 32, W == 1 ? 8 : 2)
    recurrence_fwd_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_g, const b200gdn_gated_recurrence_args a) {
  constexpr int ROWS = W * R, STAGES = stages_of(ROWS * WIDTH * (int)(sizeof(T) + sizeof(G)), CLUSTER);
  __shared__ Exchange<W, CLUSTER> exchange;
  __shared__ uint64_t full[STAGES];
  extern __shared__ __align__(128) unsigned char shared_tiles[];
  const Place at = place_of<APART, CLUSTER>(a);
  const Span seq = span_of(a, at.seq);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, step = at.n_ranks * ROWS;
  const bool live = at.channel < a.D, two = APART == 1 || at.channel + APART < a.D;
  const int n = (seq.len + step - 1) / step, in_step = warp * R;
  int t0 = at.rank * ROWS + in_step;
  Piece<T, APART> x[R];
  Piece<G, APART> g[R];
  Tiles<2, ROWS, STAGES> tiles;
  const CUtensorMap* const maps[2] = {&map_x, &map_g};
  Patience patience;
  auto fetch = [&](int t) {
    const T* px = static_cast<const T*>(a.x) + (seq.first + t) * a.stride_x + at.channel;
    const G* pg = static_cast<const G*>(a.g) + (seq.first + t) * a.stride_g + at.channel;
#pragma unroll
    for (int r = 0; r < R; ++r, px += a.stride_x, pg += a.stride_g) {
      x[r].zero();   // past the end: a decay of one, and nothing added
      g[r].zero();
      if (live && t + r < seq.len) {
        x[r].load(px, two);
        g[r].load(pg, two);
      }
    }
  };
  exchange.init();
  if constexpr (TMA) {
    const int row_bytes[2] = {WIDTH * (int)sizeof(T), WIDTH * (int)sizeof(G)};
    tiles.init(shared_tiles, full, row_bytes);
    if (threadIdx.x == 0)
      for (int i = 0; i < STAGES && i < n; ++i) tiles.load(i, maps, at.tile, (int)seq.first + i * step + at.rank * ROWS);
  } else {
    fetch(t0);
  }
  uint64_t s = load_state<APART>(a.h0, (int64_t)at.seq * a.D + at.channel, live, two);
  exchange.enter(s);
  int stage = 0;
  uint32_t phase = 0;
  uint64_t decays[R];
  Piece<T, APART> now[R];
  // the warp's tokens of step i, from t on: their decays, and the pair that they come to
  auto begin = [&](int i, int t) {
    const int rows = seq.len - t;
    Joined own = {pack2(1.f, 1.f), 0ull};
    if constexpr (TMA) {
      patience.wait(&full[stage], phase, i);
      const unsigned char *px = tiles.row(stage, 0, in_step) + 2 * lane * sizeof(T), *pg = tiles.row(stage, 1, in_step) + 2 * lane * sizeof(G);
      if (rows >= R) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          now[r].take(px + r * WIDTH * sizeof(T));
          g[r].take(pg + r * WIDTH * sizeof(G));
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          now[r].zero();
          g[r].zero();
          if (r < rows) {
            now[r].take(px + r * WIDTH * sizeof(T));
            g[r].take(pg + r * WIDTH * sizeof(G));
          }
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) now[r] = x[r];
    }
    if (rows > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        decays[r] = decay(g[r].gate());
        own.h = fma2(decays[r], own.h, now[r].pair());
        own.a = mul2(decays[r], own.a);
      }
      own.a = signed_product(own.a, decays);
    }
    if (!TMA && i + 1 < n) fetch(t + step);
    return own;
  };
  // once all warps have step i in registers
  auto next = [&](int i) {
    if (TMA && threadIdx.x == 0 && patience.ok() && i + STAGES < n) tiles.load(stage, maps, at.tile, (int)seq.first + (i + STAGES) * step + at.rank * ROWS);
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1u;
    }
  };
  // the tokens from t on, entered with h
  auto finish = [&](int t, uint64_t h) {
    const int rows = seq.len - t;
    if (!live || rows <= 0) return;
    if (a.states && (t & (BT - 1)) == 0) store_state<APART>(a.states, (int64_t)(seq.chunk + t / BT) * a.D + at.channel, h, two);
    T* const to = static_cast<T*>(a.h) + (seq.first + t) * a.D + at.channel;
    if (rows >= R) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        h = fma2(decays[r], h, now[r].pair());
        Piece<T, APART>::store(to + (int64_t)r * a.D, h, two);
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        h = fma2(decays[r], h, now[r].pair());
        if (r < rows) Piece<T, APART>::store(to + (int64_t)r * a.D, h, two);
      }
    }
  };
  for (int i = 0; i < n; ++i, t0 += step) {
    const Joined own = begin(i, t0);
    const uint64_t h = join<W, CLUSTER, false>(exchange, i, warp, at.rank, at.n_ranks, own, s, patience, [&] { next(i); });
    finish(t0, h);
  }
  if (a.ht && live && knows_the_end<W, CLUSTER, false>(n, warp, at.rank)) store_state<APART>(a.ht, (int64_t)at.seq * a.D + at.channel, s, two);
  if (!patience.ok()) {
    if (TMA && warp == 0) tiles.land(patience.stopped, n);
    if (lane == 0) atomicExch(&g_recurrence_timeout, 1);
  }
  exchange.leave(n, patience.ok());
}

// ---- backward ------------------------------------------------------------------------------------------------------------
// A CTA's step is one or more chunks, ahead of which the state is known (or, W = 1, the whole of a sequence of up to R).
template <typename T, typename G, int APART, int R, int W, bool CLUSTER, bool TMA>
__global__ void __launch_bounds__(W * 32, W == 1 ? 8 : 2)
    recurrence_bwd_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_dh,
                          const b200gdn_gated_recurrence_args a) {
  static_assert(W == 1 || (W * R) % BT == 0, "a CTA's step begins where a chunk does");
  constexpr int IN_CHUNK = BT / R;   // warps
  constexpr int ROWS = W * R, STAGES = stages_of(ROWS * WIDTH * (int)(2 * sizeof(T) + sizeof(G)), CLUSTER);
  __shared__ Exchange<W, CLUSTER> exchange;
  __shared__ ulonglong2 left[W > 1 ? 2 : 1][W][32];   // (product of decays, tokens' own state) of the warps, from the left
  __shared__ uint64_t full[STAGES];
  extern __shared__ __align__(128) unsigned char shared_tiles[];
  const Place at = place_of<APART, CLUSTER>(a);
  const Span seq = span_of(a, at.seq);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, step = at.n_ranks * ROWS;
  const bool live = at.channel < a.D, two = APART == 1 || at.channel + APART < a.D;
  const int n = (seq.len + step - 1) / step, in_step = warp * R;
  const int last = (n - 1) * step + at.rank * ROWS;   // where this CTA's last (first to be taken) tokens begin
  int t0 = last + in_step;
  Piece<T, APART> x[R], dh[R];
  Piece<G, APART> g[R];
  Tiles<3, ROWS, STAGES> tiles;
  const CUtensorMap* const maps[3] = {&map_x, &map_g, &map_dh};
  Patience patience;
  uint64_t start = 0ull;
  auto fetch_start = [&](int t) { start = load_state<APART>(a.states, (int64_t)(seq.chunk + t / BT) * a.D + at.channel, live && t < seq.len, two); };
  auto fetch = [&](int t) {
    const T* px = static_cast<const T*>(a.x) + (seq.first + t) * a.stride_x + at.channel;
    const G* pg = static_cast<const G*>(a.g) + (seq.first + t) * a.stride_g + at.channel;
    const T* pd = static_cast<const T*>(a.dh) + (seq.first + t) * a.D + at.channel;
#pragma unroll
    for (int r = 0; r < R; ++r, px += a.stride_x, pg += a.stride_g, pd += a.D) {
      x[r].zero();
      g[r].zero();
      dh[r].zero();
      if (live && t + r < seq.len) {
        x[r].load(px, two);
        g[r].load(pg, two);
        if (a.dh) dh[r].load(pd, two);
      }
    }
  };
  exchange.init();
  if constexpr (TMA) {
    const int row_bytes[3] = {WIDTH * (int)sizeof(T), WIDTH * (int)sizeof(G), WIDTH * (int)sizeof(T)};
    tiles.init(shared_tiles, full, row_bytes);
    if (threadIdx.x == 0)
      for (int i = 0; i < STAGES && i < n; ++i) tiles.load(i, maps, at.tile, (int)seq.first + last - i * step);
  } else if (n > 0) {
    fetch(t0);
  }
  if (n > 0) fetch_start(t0);
  uint64_t s = load_state<APART>(a.dht, (int64_t)at.seq * a.D + at.channel, live, two);
  exchange.enter(s);
  int stage = 0;
  uint32_t phase = 0;
  for (int i = 0; i < n; ++i, t0 -= step) {
    uint64_t decays[R], kept[R];
    Piece<T, APART> up[R];
    uint64_t h = start, own_left = 0ull;
    Joined own = {pack2(1.f, 1.f), 0ull};
    const int rows = seq.len - t0;
    if constexpr (TMA) {
      patience.wait(&full[stage], phase, i);
      const unsigned char *px = tiles.row(stage, 0, in_step) + 2 * lane * sizeof(T), *pg = tiles.row(stage, 1, in_step) + 2 * lane * sizeof(G),
                          *pd = tiles.row(stage, 2, in_step) + 2 * lane * sizeof(T);
      if (rows >= R) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[r].take(px + r * WIDTH * sizeof(T));
          g[r].take(pg + r * WIDTH * sizeof(G));
          up[r].take(pd + r * WIDTH * sizeof(T));
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[r].zero();
          g[r].zero();
          up[r].zero();
          if (r < rows) {
            x[r].take(px + r * WIDTH * sizeof(T));
            g[r].take(pg + r * WIDTH * sizeof(G));
            up[r].take(pd + r * WIDTH * sizeof(T));
          }
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) up[r] = dh[r];
    }
    if (rows > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        decays[r] = decay(g[r].gate());
        kept[r] = x[r].pair();
        own_left = fma2(decays[r], own_left, kept[r]);
        own.a = mul2(decays[r], own.a);
      }
#pragma unroll
      for (int q = R - 1; q >= 0; --q) own.h = mul2(decays[q], add2(up[q].pair(), own.h));
      own.a = signed_product(own.a, decays);
    }
    if (i + 1 < n) {
      if (!TMA) fetch(t0 - step);
      fetch_start(t0 - step);
    }
    if constexpr (W > 1) left[i & 1][warp][lane] = make_ulonglong2(own.a, own_left);
    auto next = [&] {
      if (TMA && threadIdx.x == 0 && patience.ok() && i + STAGES < n) tiles.load(stage, maps, at.tile, (int)seq.first + last - (i + STAGES) * step);
    };
    uint64_t u = join<W, CLUSTER, true>(exchange, i, warp, at.rank, at.n_ranks, own, s, patience, next);
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1u;
    }
    if (!live || rows <= 0) continue;
    if constexpr (W > 1) {
      const int before = warp % IN_CHUNK;
#pragma unroll
      for (int w = 0; w < IN_CHUNK - 1; ++w)
        if (w < before) {
          const ulonglong2 p = left[i & 1][warp - before + w][lane];
          h = fma2(p.x, h, p.y);
        }
      if (any_nan(h)) {
        h = load_state<APART>(a.states, (int64_t)(seq.chunk + t0 / BT) * a.D + at.channel, true, two);
#pragma unroll 1
        for (int w = 0; w < before; ++w) {
          const ulonglong2 p = left[i & 1][warp - before + w][lane];
          h = carry(p.x, h, p.y);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint64_t from_before = mul2(decays[r], h);
      h = fma2(decays[r], h, kept[r]);
      kept[r] = from_before;
    }
    T* const to_dx = static_cast<T*>(a.dx) + (seq.first + t0) * a.D + at.channel;
    G* const to_dg = static_cast<G*>(a.dg) + (seq.first + t0) * a.D + at.channel;
    auto finish = [&](auto full) {
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        const uint64_t d = add2(up[r].pair(), u);
        u = mul2(decays[r], d);
        if (decltype(full)::value || r < rows) {
          Piece<T, APART>::store(to_dx + (int64_t)r * a.D, d, two);
          if (a.dg) Piece<G, APART>::store(to_dg + (int64_t)r * a.D, mul2(d, kept[r]), two);
        }
      }
    };
    if (rows >= R) finish(std::true_type());
    else finish(std::false_type());
  }
  if (a.dh0 && live && knows_the_end<W, CLUSTER, true>(n, warp, at.rank)) store_state<APART>(a.dh0, (int64_t)at.seq * a.D + at.channel, s, two);
  if (!patience.ok()) {
    if (TMA && warp == 0) tiles.land(patience.stopped, n);
    if (lane == 0) atomicExch(&g_recurrence_timeout, 1);
  }
  exchange.leave(n, patience.ok());
}

// ---- one token a sequence ------------------------------------------------------------------------------------------------
template <typename T, typename G, int APART>
__global__ void __launch_bounds__(128) recurrence_step_kernel(const b200gdn_gated_recurrence_args a) {
  const int i = blockIdx.x * 128 + threadIdx.x, d = i / 32 * WIDTH + channel_of<APART>(i & 31);
  if (d >= a.D) return;
  const bool two = APART == 1 || d + APART < a.D;
  for (int seq = blockIdx.y; seq < a.n_seq; seq += gridDim.y) {
    Piece<T, APART> x;
    Piece<G, APART> g;
    x.load(static_cast<const T*>(a.x) + (int64_t)seq * a.stride_x + d, two);
    g.load(static_cast<const G*>(a.g) + (int64_t)seq * a.stride_g + d, two);
    const int64_t at = (int64_t)seq * a.D + d;
    const uint64_t before = load_state<APART>(a.h0, at, true, two), h = fma2(decay(g.gate()), before, x.pair());
    if (a.states) store_state<APART>(a.states, at, before, two);
    Piece<T, APART>::store(static_cast<T*>(a.h) + at, h, two);
    if (a.ht) store_state<APART>(a.ht, at, h, two);
  }
}

// ---- launches ------------------------------------------------------------------------------------------------------------
// clusters of more than eight CTAs have to be asked for, once per thread, kernel and device
template <auto KERN>
int allow_large_clusters() {
  static thread_local uint64_t known = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && (known >> dev & 1)) return 0;
  if (cudaFuncSetAttribute(KERN, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return set_error(B200GDN_ERR_CUDA, "cudaFuncSetAttribute(cluster size): %s", cudaGetErrorString(cudaGetLastError()));
  if (dev < 64) known |= 1ull << dev;
  return 0;
}

// How many clusters of `ranks` CTAs are resident at once: fewer than the SMs suggest, since a cluster lies within one of the chip's parts.
template <auto KERN>
int resident_clusters(cudaLaunchConfig_t cfg, int ranks) {
  static std::atomic<int> known[64][MOST_RANKS + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = known[dev][ranks].load(std::memory_order_relaxed);
  if (n > 0) return n - 1;
  cfg.gridDim = dim3(ranks);
  if (cudaOccupancyMaxActiveClusters(&n, KERN, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  known[dev][ranks].store(n + 1, std::memory_order_relaxed);
  return n;
}

// `ranks`: the most CTAs a cluster may have.  Unless it is wanted `exactly`, as many are taken as let every sequence's cluster work at once (131072 tokens of 1024
// channels, bf16 with fp32 gates: 358 us with 12, 484 with 16, of which 14 clusters are resident where 16 are wanted), in sizes that pack well
// (8191 x 1003 fp32 backward: 62 us with 8, 89 with 9).
template <auto KERN, typename... M>
int launch_walk(const char* what, const b200gdn_gated_recurrence_args& a, cudaStream_t st, int W, int ranks, bool exactly, size_t smem, const M&... maps) {
  const int64_t work = (int64_t)a.n_seq * ((a.D + WIDTH - 1) / WIDTH);
  if (smem > 0)
    if (int e = ensure_smem(KERN, smem)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  if (ranks > 1) {
    if (int e = allow_large_clusters<KERN>()) return e;
    cfg.numAttrs = 1;
    const int most = ranks;
    ranks = 1;
    for (int r : {16, 12, 8, 6, 4, 3, 2}) {
      attr.val.clusterDim.x = r;
      if (r > most || (!exactly && (work * r > 2 * sm_count() || resident_clusters<KERN>(cfg, r) < work))) continue;
      ranks = r;
      break;
    }
    attr.val.clusterDim.x = ranks;
  }
  if (work * ranks > INT32_MAX) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 pieces of work", what);
  cfg.gridDim = dim3((unsigned)(work * ranks));
  (void)cudaLaunchKernelEx(&cfg, KERN, maps..., a);   // (an error is check_launch's to name)
  return check_launch(what);
}

// tokens of a warp at a time
template <typename T, typename G>
constexpr int rows_fwd(bool tma) { return sizeof(T) + sizeof(G) <= (tma ? 6 : 4) ? 16 : 8; }
template <typename T, typename G>
constexpr int rows_bwd(bool tma) { return tma && sizeof(T) + sizeof(G) == 4 ? 16 : 8; }

template <typename T, typename G, int APART, int W, bool CLUSTER, bool TMA>
int launch_pass(const b200gdn_gated_recurrence_args& a, cudaStream_t st, bool bwd, int ranks, bool exactly) {
  constexpr int RB = rows_bwd<T, G>(TMA), RF = rows_fwd<T, G>(TMA);
  CUtensorMap x{}, g{}, dh{};
  const int rows = W * (bwd ? RB : RF), stage = rows * WIDTH * (int)(sizeof(T) * (bwd ? 2 : 1) + sizeof(G));
  if (TMA) {
    bind_context();
    int e = tma::encode_plain_2d(&x, a.x, sizeof(T), a.rows, a.D, a.stride_x, WIDTH, rows);
    if (e == 0) e = tma::encode_plain_2d(&g, a.g, sizeof(G), a.rows, a.D, a.stride_g, WIDTH, rows);
    if (e == 0 && bwd) e = tma::encode_plain_2d(&dh, a.dh, sizeof(T), a.rows, a.D, a.D, WIDTH, rows);
    if (e != 0) return set_error(B200GDN_ERR_CUDA, "gated_recurrence: tensor map (%d)", e);
  }
  const size_t smem = TMA ? (size_t)stage * stages_of(stage, CLUSTER) : 0;
  return bwd ? launch_walk<recurrence_bwd_kernel<T, G, APART, RB, W, CLUSTER, TMA>>("recurrence_bwd", a, st, W, ranks, exactly, smem, x, g, dh)
             : launch_walk<recurrence_fwd_kernel<T, G, APART, RF, W, CLUSTER, TMA>>("recurrence_fwd", a, st, W, ranks, exactly, smem, x, g);
}

template <typename T, typename G, int APART>
int launch_c(const b200gdn_gated_recurrence_args& a, cudaStream_t st, bool bwd, bool tiles) {
  if (!bwd && a.seq_len == 1) {
    const int n = a.n_seq < 65535 ? a.n_seq : 65535;
    recurrence_step_kernel<T, G, APART><<<dim3((a.D + 255) / 256, n), 128, 0, st>>>(a);
    return check_launch("recurrence_step");
  }
  const int64_t tokens = a.seq_len > 0 ? a.seq_len : (int64_t)(a.longest > 0 ? a.longest : a.n_chunks) * BT;   // of a sequence, at most
  if (a.seq_len > 0 && tokens <= (bwd ? rows_bwd<T, G>(false) : rows_fwd<T, G>(false))) return launch_pass<T, G, APART, 1, false, false>(a, st, bwd, 1, false);
  // Alone, a CTA takes a sequence's 64 channels; with fewer of these than SMs (forward, where a step costs less than what CTAs tell one another,
  // than three quarters) clusters share them: 4 x 4096 x 2048 bf16, 128 pieces of work, forward 45 us alone and 51 by twos, backward 106 and 72.
  const int64_t work = (int64_t)a.n_seq * ((a.D + WIDTH - 1) / WIDTH);
  auto go = [&](auto tma) {
    constexpr bool TMA = decltype(tma)::value;
    const int64_t step = 8 * (bwd ? rows_bwd<T, G>(TMA) : rows_fwd<T, G>(TMA)), steps = (tokens + step - 1) / step;
    // packed: as many CTAs a cluster as leave the longest sequence no more steps than all SMs take for all of them
    const int64_t all = (int64_t)a.n_chunks * BT / step * (work / a.n_seq) + 1, wanted = a.longest > 0 ? steps * 2 * sm_count() / all : 0;
    if (steps < 2 || (wanted < 2 && work > (bwd ? 4 : 3) * sm_count() / 4)) return launch_pass<T, G, APART, 8, false, TMA>(a, st, bwd, 1, false);
    const bool enough = wanted > 1 && work > sm_count() / 2;
    const int64_t most = enough ? (wanted < 8 ? wanted : 8) : MOST_RANKS;
    return launch_pass<T, G, APART, 8, true, TMA>(a, st, bwd, (int)(steps < most ? steps : most), enough);
  };
  if constexpr (APART == 1)
    if (tiles) return go(std::true_type());
  return go(std::false_type());
}

// two channels in one access where every row of every tensor allows it; by TMA where rows are a multiple of 16 bytes on such boundaries
template <typename T, typename G>
int launch_tg(const b200gdn_gated_recurrence_args& a, cudaStream_t st, bool bwd) {
  auto bits = [](std::initializer_list<const void*> all) {
    uintptr_t b = 0;
    for (const void* p : all) b |= reinterpret_cast<uintptr_t>(p);
    return b;
  };
  const bool pairs = ((a.D | a.stride_x | a.stride_g) & 1) == 0 && bits({a.x, a.h, a.dh, a.dx}) % (2 * sizeof(T)) == 0 &&
                     bits({a.g, a.dg}) % (2 * sizeof(G)) == 0;
  const bool tiles = (a.D * sizeof(T) | a.stride_x * sizeof(T) | a.stride_g * sizeof(G) | bits({a.x, a.g, a.dh})) % 16 == 0 && (!bwd || a.dh != nullptr);
  return pairs ? launch_c<T, G, 1>(a, st, bwd, tiles) : launch_c<T, G, 32>(a, st, bwd, false);
}

}  // namespace

int launch_gated_recurrence(const b200gdn_gated_recurrence_args& a, cudaStream_t st, bool bwd) {
  const bool wide = a.gate_dtype == 2;
  if (a.dtype == 2) return launch_tg<float, float>(a, st, bwd);
  if (a.dtype == 0) return wide ? launch_tg<__nv_bfloat16, float>(a, st, bwd) : launch_tg<__nv_bfloat16, __nv_bfloat16>(a, st, bwd);
  return wide ? launch_tg<__half, float>(a, st, bwd) : launch_tg<__half, __half>(a, st, bwd);
}

int recurrence_timeout_flag() {
  int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_recurrence_timeout, sizeof(int));
  if (v) cudaMemcpyToSymbol(g_recurrence_timeout, &zero, sizeof(int));
  return v;
}

}  // namespace gdn

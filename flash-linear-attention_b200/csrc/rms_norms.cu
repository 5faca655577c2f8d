// The RMS norms either side of a block in one pass, with the block's gate, its residual scale and the residual sum:
//     r1 = 1 / rms(y),  p = y r1 w1  (POST; else p = y);   z = residual + c act(gate) p,  c = alpha scale;   r2 = 1 / rms(z),  out = z r2 w
//     h = dout w;  e = dz + r2 (h - z r2^2 mean(h z)) is the gradient of z and of the residual;
//     dgate = e c p act'(gate);  f = e c act w1;  dy = r1 (f - y r1^2 mean(f y))  (POST; else f);
//     dw = sum of dout z r2;  t = sum of e act y r1:  dw1 = alpha scale t,  dscale = alpha w1 t
// z is normalised as it is summed, in fp32; only what is handed on is rounded.  The backward pass forms z again from the inputs, which it
// reads in any case but for the residual, so that z need not be kept.
// HBM streaming, in the manner of layer_norm.cu: the threads of a group share a row, E elements each, which are worked on as E / 2 fp32 pairs;
// groups walk the rows, so that a thread's columns stay its own: parameters are read once, their gradients are sums in registers, which a
// second kernel joins in a fixed order.  The second norm needs what the first one gives: two barriers a row, forward as well as backward.
// Rows of more than 256 elements come by bulk copies into a ring of shared memory, two rows ahead (backward in fp32 above 512 columns one); shorter ones, of
// tensors that do not begin on 16 bytes, and backward those whose width is no multiple of 16 bytes, to registers, one row ahead (backward with more than 16 bytes of
// a row a thread, so in fp32, where they are used).
// Measured, bf16: 65536 x 4096 with both norms and a scale forward 330 us (328 at copy rate), backward 525 (492); 16384 x 2048 with a sigmoid gate as
// well 62 (51) and 119 (82), where instructions count: 28 and 57 an element; 8191 x 1003 fp32 37 (25) and 58 (40), 8191 x 1002 bf16 25 and 45 (13 and 20).
// Rows of other widths than multiples of 16 bytes beyond 4096 elements spill backward (260 to 576 bytes a thread); beyond 8192 elements a
// row is looked at several times.
#include "gdn_common.cuh"
#include "row_pieces.cuh"
#include "tc5.cuh"
#include "tma.cuh"

namespace gdn {
namespace {

__device__ int g_norms_timeout = 0;

constexpr uint32_t POST = B200GDN_NORMS_POST, SIGMOID = B200GDN_NORMS_SIGMOID, SILU = B200GDN_NORMS_SILU;
constexpr int threads_of(int tpr) { return tpr > 32 ? tpr : 128; }   // rows of several warps have a CTA to themselves

// down: a power of two, down^2 in [1 / 4 D, 1 / D]: a sum of squares of elements times `down` is within range wherever their mean is, which
// is that sum times `up`
__device__ __forceinline__ float down_of(int D) { return __int_as_float((127 - (33 - __clz(D - 1)) / 2) << 23); }

// A thread's E elements of a row, as loaded: pieces of N neighbouring ones, TPR pieces apart; a pair is two neighbours, or (N = 1) an
// element and the one TPR further on.
template <typename T, int N, int TPR, int E>
struct Part {
  static constexpr int WORDS = E * (int)sizeof(T) / 4, BYTES = N * (int)sizeof(T);
  uint32_t w[WORDS];

  static __device__ __forceinline__ int column(int sub, int e) { return ((e / N) * TPR + sub) * N + e % N; }
  // `row`: in global or shared memory
  __device__ __forceinline__ void load(const T* row, int sub, int D) {
    if constexpr (BYTES == 16) {
#pragma unroll
      for (int v = 0; v < E / N; ++v) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (column(sub, v * N) < D) u = *reinterpret_cast<const uint4*>(row + column(sub, v * N));
        w[4 * v] = u.x, w[4 * v + 1] = u.y, w[4 * v + 2] = u.z, w[4 * v + 3] = u.w;
      }
    } else if constexpr (BYTES == 4) {
#pragma unroll
      for (int v = 0; v < WORDS; ++v) w[v] = column(sub, v * N) < D ? *reinterpret_cast<const uint32_t*>(row + column(sub, v * N)) : 0u;
    } else {
#pragma unroll
      for (int v = 0; v < WORDS; ++v) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
        const uint32_t lo = column(sub, 2 * v) < D ? p[column(sub, 2 * v)] : 0, hi = column(sub, 2 * v + 1) < D ? p[column(sub, 2 * v + 1)] : 0;
        w[v] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int sub, int D) const {
    if constexpr (BYTES == 16) {
#pragma unroll
      for (int v = 0; v < E / N; ++v)
        if (column(sub, v * N) < D) *reinterpret_cast<uint4*>(row + column(sub, v * N)) = make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
    } else if constexpr (BYTES == 4) {
#pragma unroll
      for (int v = 0; v < WORDS; ++v)
        if (column(sub, v * N) < D) *reinterpret_cast<uint32_t*>(row + column(sub, v * N)) = w[v];
    } else {
#pragma unroll
      for (int v = 0; v < WORDS; ++v) {
        uint16_t* p = reinterpret_cast<uint16_t*>(row);
        if (column(sub, 2 * v) < D) p[column(sub, 2 * v)] = (uint16_t)w[v];
        if (column(sub, 2 * v + 1) < D) p[column(sub, 2 * v + 1)] = (uint16_t)(w[v] >> 16);
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int v = 0; v < WORDS; ++v) w[v] = 0u;
  }
  __device__ __forceinline__ uint64_t pair(int i) const {
    if constexpr (sizeof(T) == 2) return widen2<T>(w[i]);
    else return pack2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
  __device__ __forceinline__ void set(int i, uint64_t x) {
    if constexpr (sizeof(T) == 2) {
      w[i] = narrow2<T>(x);
    } else {
      const float2 f = unpack2(x);
      w[2 * i] = __float_as_uint(f.x);
      w[2 * i + 1] = __float_as_uint(f.y);
    }
  }
  // a parameter's pairs; `absent` where there is none, zero past the row's end
  static __device__ __forceinline__ void params(const void* p, int dtype, int sub, int D, float absent, uint64_t (&x)[E / 2]) {
    if constexpr (N == 1) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const int a = column(sub, 2 * i), b = column(sub, 2 * i + 1);
        x[i] = pack2(a < D ? (p ? ld_param(p, a, dtype) : absent) : 0.f, b < D ? (p ? ld_param(p, b, dtype) : absent) : 0.f);
      }
    } else {
#pragma unroll
      for (int v = 0; v < E / N; ++v) {
        uint64_t q[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) q[i] = 0ull;
        if (column(sub, v * N) < D) load_params<N>(p, dtype, column(sub, v * N), absent, q);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) x[v * N / 2 + i] = q[i];
      }
    }
  }
};

// The tensors of a row, those that are there, side by side in a ring of SLOTS rows, as bulk copies; each group has its own.  A copy begins on 16
// bytes: of a row that does not, it begins with the end of the row ahead, and ends with the beginning of the next one.  (The tensors themselves
// begin on 16 bytes, so all rows of a number lie alike.)
__host__ __device__ constexpr int room_of(int row_bytes) { return row_bytes % 16 == 0 ? row_bytes : (row_bytes + 31) / 16 * 16; }
template <int SLOTS>
struct Ring {
  unsigned char* base;
  uint64_t* full;
  int slot = 0;
  uint32_t phase = 0;
  int stopped = -1;   // slot and phase of a wait that has run out

  // one thread of the group
  template <typename T>
  __device__ __forceinline__ void fill(int at, const void* const* tensors, int n, int64_t row, int64_t rows, int row_bytes) const {
    const int ahead = (int)(row * row_bytes & 15), end = ahead + row_bytes;
    int bytes = (end + 15) / 16 * 16;
    unsigned char* to = base + at * n * room_of(row_bytes);
    if (row * row_bytes - ahead + bytes > rows * row_bytes) {   // the tensor ends within the last 16 bytes: what is there comes by itself
      bytes = end / 16 * 16;
      for (int i = 0; i < n; ++i)
        for (int e = bytes; e < end; e += (int)sizeof(T))
          *reinterpret_cast<T*>(to + i * room_of(row_bytes) + e) =
              *reinterpret_cast<const T*>(static_cast<const char*>(tensors[i]) + (row * row_bytes - ahead + e));
    }
    tc5::mbar_expect_tx(&full[at], n * bytes);
    for (int i = 0; i < n; ++i)
      tma::load_1d(to + i * room_of(row_bytes), static_cast<const char*>(tensors[i]) + (row * row_bytes - ahead), bytes, &full[at]);
  }
  template <typename T>
  __device__ __forceinline__ const T* first(int n, int64_t row, int row_bytes) const {   // of the tensors of the row that is there now
    return reinterpret_cast<const T*>(base + slot * n * room_of(row_bytes) + (row * row_bytes & 15));
  }
  // A wait that has run out is not repeated: nothing more is copied, and at the end what is on its way is waited for once more, so that no copy
  // outlives its CTA, and the flag set.
  __device__ __forceinline__ void wait() {
    if (stopped < 0 && !tc5::mbar_wait_warp(&full[slot], phase)) stopped = slot << 1 | (int)phase;
  }
  __device__ __forceinline__ bool ok() const { return stopped < 0; }
  __device__ __forceinline__ void finish() {   // a warp of the group
    if (stopped < 0) return;
    slot = stopped >> 1;
    phase = stopped & 1;
    for (int i = 0; i < SLOTS; ++i, next()) (void)tc5::mbar_wait_warp(&full[slot], phase);
    if ((threadIdx.x & 31) == 0) atomicExch(&g_norms_timeout, 1);
  }
  __device__ __forceinline__ void next() {
    if (++slot == SLOTS) {
      slot = 0;
      phase ^= 1u;
    }
  }
};
// Two rows are enough, and more are worse: reads run so far ahead of the writes that memory changes between them more often (65536 x 4096 bf16
// forward: 330 us with two, 373 with three or four).
constexpr int slots_of(int n_tensors, int tpr, int e, int size) {   // of 54 KB for 128 threads
  return 54 * 1024 * threads_of(tpr) / 128 / (threads_of(tpr) / tpr) / (n_tensors * room_of(tpr * e * size)) > 1 ? 2 : 1;
}

// act(gate) and, where asked for, act'(gate).  What the gate is (NO_GATE, or AS_IT_IS, SIGMOID, SILU) is known where a row's loop begins: a
// question asked pair by pair costs a branch each and moves where its ways meet again.
constexpr uint32_t NO_GATE = ~0u, AS_IT_IS = 0u;
template <uint32_t ACT, bool SLOPE>
__device__ __forceinline__ uint64_t activation(uint64_t g, uint64_t& slope) {
  const uint64_t one = pack2(1.f, 1.f);
  if constexpr (ACT == AS_IT_IS) {
    slope = one;
    return g;
  } else {
    const uint64_t s = fast_sigmoid2(g);
    if constexpr (ACT == SIGMOID) {
      if (SLOPE) slope = fma2(mul2(s, s), pack2(-1.f, -1.f), s);
      return s;
    } else {
      if (SLOPE) slope = mul2(s, fma2(g, fma2(s, pack2(-1.f, -1.f), one), one));
      return mul2(g, s);
    }
  }
}
template <uint32_t V> struct Constant { static constexpr uint32_t value = V; };
enum Gates { WITHOUT, WITH, EITHER };   // of a kernel: large ones that need not look are a twentieth faster
template <Gates GATE, typename F>
__device__ __forceinline__ void with_gate(const b200gdn_rms_norms_args& a, F f) {
  if (GATE == WITHOUT || (GATE == EITHER && !a.gate)) f(Constant<NO_GATE>());
  else if constexpr (GATE == WITHOUT) return;
  else if (a.flags & SIGMOID) f(Constant<SIGMOID>());
  else if (a.flags & SILU) f(Constant<SILU>());
  else f(Constant<AS_IT_IS>());
}

// ---- forward -------------------------------------------------------------------------------------------------------------
template <typename T, int N, int TPR, int E, bool RING, Gates GATE>
__global__ void __launch_bounds__(threads_of(TPR), 512 / threads_of(TPR)) rms_norms_fwd_kernel(const b200gdn_rms_norms_args a) {
  using Row = Part<T, N, TPR, E>;
  constexpr int RPC = threads_of(TPR) / TPR, NW = TPR > 32 ? TPR / 32 : 1, P = E / 2, SLOTS = RING ? slots_of(3, TPR, E, sizeof(T)) : 1;
  __shared__ float scratch[2][2][NW];
  __shared__ uint64_t full[RING ? RPC * SLOTS : 1];
  extern __shared__ __align__(128) unsigned char ring_bytes[];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool post = a.flags & POST;
  const float inv = 1.f / a.D, down = down_of(a.D), up = inv / (down * down);
  const uint64_t by = pack2(down, down);
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t row = (int64_t)blockIdx.x * RPC + group;
  const int row_bytes = a.D * (int)sizeof(T), n_tensors = 1 + (a.residual != nullptr) + (GATE != WITHOUT && a.gate != nullptr);
  const void* tensors[3] = {a.y, a.residual ? a.residual : a.gate, a.gate};
  Ring<SLOTS> ring{ring_bytes + group * SLOTS * n_tensors * room_of(row_bytes), full + group * SLOTS};
  const int room = room_of(row_bytes) / (int)sizeof(T);
  Row y, res, gate;
  auto fetch = [&](int64_t row) {
    y.zero(), res.zero(), gate.zero();
    if (row >= a.rows) return;
    y.load(static_cast<const T*>(a.y) + row * a.D, sub, a.D);
    if (a.residual) res.load(static_cast<const T*>(a.residual) + row * a.D, sub, a.D);
    if (GATE != WITHOUT && a.gate) gate.load(static_cast<const T*>(a.gate) + row * a.D, sub, a.D);
  };
  if constexpr (RING) {
    if (sub == 0) {
      for (int i = 0; i < SLOTS; ++i) tc5::mbar_init(&ring.full[i], 1);
      tc5::fence_mbar_init();
      for (int i = 0; i < SLOTS && row + i * step < a.rows; ++i) ring.template fill<T>(i, tensors, n_tensors, row + i * step, a.rows, row_bytes);
    }
    __syncthreads();
  } else {
    fetch(row);
  }
  uint64_t c[P], w[P];   // what the normalised p is multiplied with, and z
  Row::params(post ? a.post_weight : nullptr, a.param_dtype, sub, a.D, 1.f, c);
  Row::params(a.scale, a.param_dtype, sub, a.D, 1.f, w);
#pragma unroll
  for (int i = 0; i < P; ++i) c[i] = mul2(mul2(w[i], pack2(a.alpha, a.alpha)), c[i]);
  Row::params(a.weight, a.param_dtype, sub, a.D, 1.f, w);
  for (int turn = 0; row - group < a.rows; turn ^= 1, row += step) {
    if constexpr (RING) {
      if (row < a.rows) ring.wait();
      const T* at = ring.template first<T>(n_tensors, row, row_bytes);
      y.load(at, sub, a.D);
      if (a.residual) res.load(at += room, sub, a.D);
      else res.zero();
      if (GATE != WITHOUT && a.gate) gate.load(at += room, sub, a.D);
    }
    float s[1] = {0.f}, r1 = 1.f;
    if (post) {
      uint64_t sum = 0ull;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint64_t x = mul2(y.pair(i), by);
        sum = fma2(x, x, sum);
      }
      s[0] = both(sum);
      row_sums<TPR>(s, scratch[turn][0]);
      r1 = __frsqrt_rn(s[0] * up + a.eps);
    }
    uint64_t z[P], sum = 0ull;
    const uint64_t by_r1 = pack2(r1, r1);
    with_gate<GATE>(a, [&](auto act) {
      constexpr uint32_t ACT = decltype(act)::value;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        uint64_t none, k = mul2(c[i], by_r1);
        if constexpr (ACT != NO_GATE) k = mul2(k, activation<ACT, false>(gate.pair(i), none));
        z[i] = fma2(y.pair(i), k, res.pair(i));
        const uint64_t x = mul2(z[i], by);
        sum = fma2(x, x, sum);
      }
    });
    if constexpr (!RING) fetch(row + step);
    s[0] = both(sum);
    row_sums<TPR>(s, scratch[turn][1]);
    if constexpr (RING) {   // (the whole group has passed: what it read is in registers)
      if (TPR == 32) __syncwarp();
      if (sub == 0 && ring.ok() && row + SLOTS * step < a.rows) ring.template fill<T>(ring.slot, tensors, n_tensors, row + SLOTS * step, a.rows, row_bytes);
      ring.next();
    }
    const float r2 = __frsqrt_rn(s[0] * up + a.eps);
    const uint64_t by_r2 = pack2(r2, r2);
    if (row >= a.rows) continue;
    Row o;
    if (a.z) {
#pragma unroll
      for (int i = 0; i < P; ++i) o.set(i, z[i]);
      o.store(static_cast<T*>(a.z) + row * a.D, sub, a.D);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) o.set(i, mul2(mul2(z[i], by_r2), w[i]));
    o.store(static_cast<T*>(a.out) + row * a.D, sub, a.D);
    if (sub == 0 && a.rstd_z) {
      a.rstd_y[row] = r1;
      a.rstd_z[row] = r2;
    }
  }
  if constexpr (RING) ring.finish();
}

// ---- backward ------------------------------------------------------------------------------------------------------------
template <typename T, int N, int TPR, int E, bool RING, Gates GATE>
__global__ void __launch_bounds__(threads_of(TPR), 512 / threads_of(TPR)) rms_norms_bwd_kernel(const b200gdn_rms_norms_args a) {
  using Row = Part<T, N, TPR, E>;
  constexpr int RPC = threads_of(TPR) / TPR, NW = TPR > 32 ? TPR / 32 : 1, P = E / 2, SLOTS = RING ? slots_of(5, TPR, E, sizeof(T)) : 1;
  constexpr bool AHEAD = !RING && E * sizeof(T) <= 16;   // registers for the next row
  __shared__ float scratch[2][2][NW];
  __shared__ float part[RPC > 1 ? RPC * 2 * TPR * E : 1];
  __shared__ uint64_t full[RING ? RPC * SLOTS : 1];
  extern __shared__ __align__(128) unsigned char ring_bytes[];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool post = a.flags & POST;
  const float inv = 1.f / a.D;
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t row = (int64_t)blockIdx.x * RPC + group;
  const int row_bytes = a.D * (int)sizeof(T);
  const void* tensors[5];
  int n_tensors = 0;
  for (const void* p : {a.y, a.residual, a.gate, a.dout, a.dz})
    if (p) tensors[n_tensors++] = p;
  Ring<SLOTS> ring{ring_bytes + group * SLOTS * n_tensors * room_of(row_bytes), full + group * SLOTS};
  const int room = room_of(row_bytes) / (int)sizeof(T);
  struct Rows {
    Row y, res, gate, dout, dz;
    float r1, r2;
  };
  Rows next;
  auto fetch_sums = [&](int64_t row) {   // (a row past the end adds zeros to every sum)
    next.r1 = row < a.rows ? a.rstd_y[row] : 0.f;
    next.r2 = row < a.rows ? a.rstd_z[row] : 0.f;
  };
  auto fetch = [&](Rows& to, int64_t row) {
    to.y.zero(), to.res.zero(), to.gate.zero(), to.dout.zero(), to.dz.zero();
    if (row >= a.rows) return;
    to.y.load(static_cast<const T*>(a.y) + row * a.D, sub, a.D);
    if (a.residual) to.res.load(static_cast<const T*>(a.residual) + row * a.D, sub, a.D);
    if (GATE != WITHOUT && a.gate) to.gate.load(static_cast<const T*>(a.gate) + row * a.D, sub, a.D);
    if (a.dout) to.dout.load(static_cast<const T*>(a.dout) + row * a.D, sub, a.D);
    if (a.dz) to.dz.load(static_cast<const T*>(a.dz) + row * a.D, sub, a.D);
  };
  if constexpr (RING) {
    if (sub == 0) {
      for (int i = 0; i < SLOTS; ++i) tc5::mbar_init(&ring.full[i], 1);
      tc5::fence_mbar_init();
      for (int i = 0; i < SLOTS && row + i * step < a.rows; ++i) ring.template fill<T>(i, tensors, n_tensors, row + i * step, a.rows, row_bytes);
    }
    __syncthreads();
  } else if constexpr (AHEAD) {
    fetch(next, row);
  }
  fetch_sums(row);
  uint64_t c[P], w[P], dw[P], dt[P];   // alpha scale post_weight, weight; the columns' sums
  Row::params(post ? a.post_weight : nullptr, a.param_dtype, sub, a.D, 1.f, c);
  Row::params(a.scale, a.param_dtype, sub, a.D, 1.f, w);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    c[i] = mul2(mul2(w[i], pack2(a.alpha, a.alpha)), c[i]);
    dw[i] = dt[i] = 0ull;
  }
  Row::params(a.weight, a.param_dtype, sub, a.D, 1.f, w);
  // By chunks: from the ring a chunk is read where it is used, and again after the barrier, rather than held.
  constexpr int CHUNK = N == 1 ? 2 : N, CHUNKS = E / CHUNK, CP = CHUNK / 2;
  using Chunk = Part<T, N, TPR, CHUNK>;
  for (int turn = 0; row - group < a.rows; turn ^= 1, row += step) {
    Rows cur;
    const T *at_y = nullptr, *at_res = nullptr, *at_gate = nullptr, *at_dout = nullptr, *at_dz = nullptr;
    const bool live = row < a.rows;
    const float r1f = next.r1, r2f = next.r2;
    if constexpr (RING) {
      if (live) ring.wait();
      const T* at = ring.template first<T>(n_tensors, row, row_bytes);
      at_y = at;
      if (a.residual) at_res = at += room;
      if (GATE != WITHOUT && a.gate) at_gate = at += room;
      if (a.dout) at_dout = at += room;
      if (a.dz) at_dz = at += room;
    } else if constexpr (AHEAD) {
      cur = next;
      fetch(next, row + step);
    } else {
      fetch(cur, row);
    }
    auto chunk = [&](const T* at, const Row& held, int v) {
      Chunk q;
      if constexpr (RING) {
        if (live && at) q.load(at + v * TPR * CHUNK, sub, a.D - v * TPR * CHUNK);
        else q.zero();
      } else {
#pragma unroll
        for (int i = 0; i < Chunk::WORDS; ++i) q.w[i] = held.w[v * Chunk::WORDS + i];
      }
      return q;
    };
    fetch_sums(row + step);
    const uint64_t r1 = pack2(r1f, r1f), r2 = pack2(r2f, r2f);
    uint64_t z[P], sum = 0ull;   // z r2, then f times what dy has of it
    with_gate<GATE>(a, [&](auto act) {
      constexpr uint32_t ACT = decltype(act)::value;
#pragma unroll
      for (int v = 0; v < CHUNKS; ++v) {
        const Chunk y = chunk(at_y, cur.y, v), res = chunk(at_res, cur.res, v), dout = chunk(at_dout, cur.dout, v);
        Chunk gate;
        if constexpr (ACT != NO_GATE) gate = chunk(at_gate, cur.gate, v);
#pragma unroll
        for (int q = 0; q < CP; ++q) {
          const int i = v * CP + q;
          uint64_t none, k = mul2(c[i], r1);
          if constexpr (ACT != NO_GATE) k = mul2(k, activation<ACT, false>(gate.pair(q), none));
          z[i] = mul2(fma2(y.pair(q), k, res.pair(q)), r2);
          const uint64_t g = dout.pair(q);
          sum = fma2(mul2(g, w[i]), z[i], sum);
          dw[i] = fma2(g, z[i], dw[i]);
        }
      }
    });
    float s[1] = {both(sum)};
    row_sums<TPR>(s, scratch[turn][0]);
    const uint64_t back = pack2(-s[0] * inv, -s[0] * inv);
    sum = 0ull;
    with_gate<GATE>(a, [&](auto act) {
      constexpr uint32_t ACT = decltype(act)::value;
#pragma unroll
      for (int v = 0; v < CHUNKS; ++v) {
        const Chunk y = chunk(at_y, cur.y, v), dout = chunk(at_dout, cur.dout, v), dz = chunk(at_dz, cur.dz, v);
        Chunk gate, dgate, dres;
        if constexpr (ACT != NO_GATE) gate = chunk(at_gate, cur.gate, v);
#pragma unroll
        for (int q = 0; q < CP; ++q) {
          const int i = v * CP + q;
          const uint64_t h = fma2(z[i], back, mul2(dout.pair(q), w[i]));
          const uint64_t e = fma2(h, r2, dz.pair(q)), n1 = mul2(y.pair(q), r1), ec = mul2(e, c[i]);
          dres.set(q, e);
          if constexpr (ACT != NO_GATE) {
            uint64_t slope;
            const uint64_t act = activation<ACT, true>(gate.pair(q), slope);
            dgate.set(q, ACT == AS_IT_IS ? mul2(ec, n1) : mul2(mul2(ec, n1), slope));
            dt[i] = fma2(mul2(e, act), n1, dt[i]);
            z[i] = mul2(ec, act);
          } else {
            dt[i] = fma2(e, n1, dt[i]);
            z[i] = ec;
          }
          sum = fma2(z[i], n1, sum);
        }
        if (live) {
          const int64_t to = row * a.D + v * TPR * CHUNK;
          if (ACT != NO_GATE && a.dgate) dgate.store(static_cast<T*>(a.dgate) + to, sub, a.D - v * TPR * CHUNK);
          if (a.dresidual) dres.store(static_cast<T*>(a.dresidual) + to, sub, a.D - v * TPR * CHUNK);
        }
      }
    });
    uint64_t mean = 0ull;
    Row y;   // the row as it was, before its place in the ring is filled again
#pragma unroll
    for (int v = 0; v < CHUNKS; ++v) {
      const Chunk q = chunk(at_y, cur.y, v);
#pragma unroll
      for (int i = 0; i < Chunk::WORDS; ++i) y.w[v * Chunk::WORDS + i] = q.w[i];
    }
    if (post || RING) {   // (with a ring for its barrier: the row has been read)
      s[0] = both(sum);
      row_sums<TPR>(s, scratch[turn][1]);
      if (post) mean = pack2(-s[0] * inv, -s[0] * inv);
    }
    if constexpr (RING) {
      if (TPR == 32) __syncwarp();
      if (sub == 0 && ring.ok() && row + SLOTS * step < a.rows) ring.template fill<T>(ring.slot, tensors, n_tensors, row + SLOTS * step, a.rows, row_bytes);
      ring.next();
    }
    if (!live || !a.dy) continue;
#pragma unroll
    for (int i = 0; i < P; ++i) y.set(i, mul2(fma2(mul2(y.pair(i), r1), mean, z[i]), r1));   // (r1 is one without the first norm)
    y.store(static_cast<T*>(a.dy) + row * a.D, sub, a.D);
  }
  if constexpr (RING) ring.finish();
  if (a.partials == nullptr) return;
  constexpr int COLUMNS = TPR * E;
  auto leave = [&](int which, int i, uint64_t x) {
    const float2 f = unpack2(x);
    const int at[2] = {Row::column(sub, 2 * i), Row::column(sub, 2 * i + 1)};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float v = q ? f.y : f.x;
      if constexpr (RPC > 1) part[(group * 2 + which) * COLUMNS + at[q]] = v;
      else if (at[q] < a.D) a.partials[((int64_t)blockIdx.x * 2 + which) * a.D + at[q]] = v;
    }
  };
#pragma unroll
  for (int i = 0; i < P; ++i) {
    leave(0, i, dw[i]);
    leave(1, i, dt[i]);
  }
  if constexpr (RPC > 1) {   // the groups' sums in their order
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * COLUMNS; i += threads_of(TPR)) {
      const int which = i / COLUMNS, d = i % COLUMNS;
      if (d >= a.D) continue;
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < RPC; ++g) s += part[(g * 2 + which) * COLUMNS + d];
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
    with_gate<EITHER>(a, [&](auto which) {
      constexpr uint32_t ACT = decltype(which)::value;
      if constexpr (ACT != NO_GATE) {
        uint64_t s;
        act = unpack2(activation<ACT, true>(pack2(Io<T>::ld(a.gate, row + d), 0.f), s)).x;
        slope = unpack2(s).x;
      }
    });
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
template <typename T, int N, int TPR, int E, bool RING, bool BWD>
int launch_rows(const b200gdn_rms_norms_args& a, cudaStream_t st) {
  constexpr int threads = threads_of(TPR), RPC = threads / TPR, MOST = BWD ? 5 : 3;   // tensors of a row
  const int n = grid_of(a.rows, RPC, 512 / threads);
  auto go = [&](auto kern) {
    int tensors = 0;
    for (const void* p : {a.y, a.residual, a.gate, BWD ? a.dout : nullptr, BWD ? a.dz : nullptr}) tensors += p != nullptr;
    const size_t smem = RING ? (size_t)RPC * slots_of(MOST, TPR, E, sizeof(T)) * tensors * room_of(a.D * (int)sizeof(T)) : 0;
    if (RING)   // (what a row may take at most: the limit is set once)
      if (int e = ensure_smem(kern, (size_t)RPC * slots_of(MOST, TPR, E, sizeof(T)) * MOST * (TPR * E * sizeof(T) + 16))) return e;
    kern<<<n, threads, smem, st>>>(a);
    return check_launch(BWD ? "rms_norms_bwd" : "rms_norms_fwd");
  };
  auto pass = [&](auto gates) {
    constexpr Gates GATE = decltype(gates)::value;
    if constexpr (BWD) return go(rms_norms_bwd_kernel<T, N, TPR, E, RING, GATE>);
    else return go(rms_norms_fwd_kernel<T, N, TPR, E, RING, GATE>);
  };
  int e;
  if constexpr (RING && N * sizeof(T) == 16) e = a.gate ? pass(std::integral_constant<Gates, WITH>()) : pass(std::integral_constant<Gates, WITHOUT>());
  else e = pass(std::integral_constant<Gates, EITHER>());
  return e == 0 && BWD && a.partials ? reduce_partials(a, n, st) : e;
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

// Sixteen elements a thread where rows come by the ring, else eight; where that is more threads than a CTA has registers for, sixteen.
// (Backward, sixteen in one warp spill: 16384 x 512 bf16 gated 66 us, 47 with eight in two.)
template <typename T, int N, bool BWD>
int launch_n(const b200gdn_rms_norms_args& a, cudaStream_t st) {
  if (a.D <= 64) return launch_rows<T, N, 8, 8, false, BWD>(a, st);
  if (a.D <= 128) return launch_rows<T, N, 16, 8, false, BWD>(a, st);
  if (a.D <= 256) return launch_rows<T, N, 32, 8, false, BWD>(a, st);
  // by the ring: rows in pieces of 16 bytes, and forward narrower ones too, where the tensors begin on 16 (8191 x 1002 bf16 forward 25 us, 30 by
  // registers; backward 54 and 45, 8191 x 1003 fp32 83 and 58)
  if constexpr (N * sizeof(T) == 16 || !BWD) {
    uintptr_t begin = 0;
    for (const void* p : {a.y, a.residual, a.gate, BWD ? a.dout : nullptr, BWD ? a.dz : nullptr}) begin |= reinterpret_cast<uintptr_t>(p);
    if (begin % 16 == 0) {
      if (a.D <= 512) return launch_rows<T, N, BWD ? 64 : 32, BWD ? 8 : 16, true, BWD>(a, st);
      if (a.D <= 1024) return launch_rows<T, N, 64, 16, true, BWD>(a, st);
      if (a.D <= 2048) return launch_rows<T, N, 128, 16, true, BWD>(a, st);
      if (a.D <= 4096) return launch_rows<T, N, 256, 16, true, BWD>(a, st);
      if (a.D <= 8192) return launch_rows<T, N, 512, 16, true, BWD>(a, st);
    }
  }
  if constexpr (N * sizeof(T) != 16) {
    if (a.D <= 512) return launch_rows<T, N, 64, 8, false, BWD>(a, st);
    if (a.D <= 1024) return launch_rows<T, N, 128, 8, false, BWD>(a, st);
    if (a.D <= 2048) return launch_rows<T, N, 256, 8, false, BWD>(a, st);
    if (a.D <= 4096) return launch_rows<T, N, 512, 8, false, BWD>(a, st);
    if (a.D <= 8192) return launch_rows<T, N, 512, 16, false, BWD>(a, st);
  }
  return launch_wide<T>(a, st, BWD);
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

template <typename T, bool BWD>
int launch_t(const b200gdn_rms_norms_args& a, cudaStream_t st) {
  const int n = piece_of<T>(a);
  if (n == 16 / sizeof(T)) return launch_n<T, 16 / sizeof(T), BWD>(a, st);
  if constexpr (sizeof(T) == 2)
    if (n == 2) return launch_n<T, 2, BWD>(a, st);
  return launch_n<T, 1, BWD>(a, st);
}
template <bool BWD>
int launch(const b200gdn_rms_norms_args& a, cudaStream_t st) {
  return a.dtype == 0 ? launch_t<__nv_bfloat16, BWD>(a, st) : a.dtype == 1 ? launch_t<__half, BWD>(a, st) : launch_t<float, BWD>(a, st);
}

}  // namespace

int rms_norms_grid(int64_t rows) { return (int)(rows < 1 ? 1 : rows < most_ctas() ? rows : most_ctas()); }

int64_t rms_norms_partials(int64_t rows, int D) { return (rows + 3) / 4 * 4 + (int64_t)rms_norms_grid(rows) * 2 * D; }

int launch_rms_norms(const b200gdn_rms_norms_args& a, cudaStream_t st, bool bwd) {
  return bwd ? launch<true>(a, st) : launch<false>(a, st);
}

int norms_timeout_flag() {
  int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_norms_timeout, sizeof(int));
  if (v) cudaMemcpyToSymbol(g_norms_timeout, &zero, sizeof(int));
  return v;
}

}  // namespace gdn

// Projections: y = act(x W^T + b) + residual, and its gradients dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum of dz, in 16-bit types
// with fp32 sums.
//
// All three products run in one persistent kernel on tcgen05 with CTA pairs: a pair forms a 256 x BN tile (128 rows in the tensor memory of
// each CTA), each CTA brings its 128 rows of A and its half of B by TMA, one thread issues M = 256 instructions that read both CTAs' shared
// memory.  A single CTA's 128 x 256 tile would need 96 bytes a clock from L2, more than the 64 an SM gets; the pair's 256 x 256 needs 64 a CTA.
// Two warps load and issue, eight carry finished tiles out of tensor memory while the next tile's sums form in its other half.
// Operands lie either way: an operand whose contraction runs along its rows in memory is staged as [contraction][64 columns] panels and read
// as an MN-major operand, so that W and x are never transposed.
// Few tokens (up to 256): the product is formed the other way round, W's rows as the 256-row side and the tokens as a BN of 32 to 256, so that
// what is read is W and little else.  Where there are fewer tiles than CTA pairs the contraction is split; the parts are left in fp32 and a
// second kernel adds them in order and finishes; so is that of the tiles of the last round, where they leave pairs without work.
// Up to 16 tokens, forward: W passes through registers once, as fast as memory gives it (linear_few_kernel).
// TMA wants rows 16 bytes apart: operands of other widths are first copied to rows that are.
// Bound by the tensor pipe (88 to 92 % of its cycles) and the clock it is left: 16384 x 2048 -> 8192 bf16 with bias and SiLU, z kept, 343 us
// (1.60 PFLOP/s; 1.64 is the library's burst), dx 345, dW 366, dz with db 135 (123 at copy rate).  Small products: 2 us until the first operands are there,
// 0.3 us a step of 64, 2 us for the last epilogue and the end.  4 tokens, 2048 -> 8192: 7.6 us a call (5.1 for W at copy rate).
// Rounded to 16 bits beside the results: dz, since the products read 16 bits (bf16 dx and dW are off by 0.0024 of their size against 64 bits, 0.0017 of it by
// their own rounding), and the z kept for the backward pass, which in 32 would take as many bytes again as y: the slope changes by at most 0.8 of what z does.
#include "gdn_common.cuh"
#include "rowio.cuh"
#include "tc5.cuh"
#include "tma.cuh"

namespace gdn {
namespace {

__device__ int g_linear_timeout = 0;

// ---- activations -----------------------------------------------------------------------------------------------------------
enum { NONE = 0, SILU = B200GDN_LINEAR_SILU, SIGMOID = B200GDN_LINEAR_SIGMOID, GELU = B200GDN_LINEAR_GELU };

// The normal distribution's function of a pair, and e = exp(-v^2 / 2).  Of -|v| it is e t Q(t) with t = 1 / (1 + 0.24 |v|), Q of degree seven by least squares of the
// relative error (4.3e-7; 7.5e-7 with fp32's roundings near zero, and v^2 2^-24 more by the exponent's further down), and of |v| one less that: relative to the
// result everywhere.  (1 + erf loses below -4 what a 16-bit result still shows.)  Where the distribution ends, |v| is held at 32, so that infinities are
// multiplied with zero and one.  16384 x 2048 -> 8192: 409 us, 492 with erfcf, 428 with 1 + erf.
__device__ __forceinline__ uint64_t normal2(uint64_t v, uint64_t& e) {
  auto k = [](float c) { return pack2(c, c); };
  const float2 x = unpack2(v);
  float2 f = {fabsf(x.x), fabsf(x.y)};
  asm("min.NaN.f32 %0, %0, 0f42000000;" : "+f"(f.x));
  asm("min.NaN.f32 %0, %0, 0f42000000;" : "+f"(f.y));
  const uint64_t a = pack2(f.x, f.y);
  f = unpack2(mul2(mul2(a, a), k(-0.72134752044448170f)));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  e = pack2(f.x, f.y);
  f = unpack2(fma2(a, k(0.24f), k(1.f)));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  const uint64_t t = pack2(f.x, f.y);
  uint64_t q = fma2(k(-0.05299046263098717f), t, k(0.1527886837720871f));
  q = fma2(q, t, k(-0.0656936764717102f));
  q = fma2(q, t, k(0.1183803603053093f));
  q = fma2(q, t, k(0.06340166181325912f));
  q = fma2(q, t, k(0.09283752739429474f));
  q = fma2(q, t, k(0.09552229940891266f));
  q = fma2(q, t, k(0.09575378894805908f));
  q = mul2(mul2(q, t), e);
  const float2 below = unpack2(q), above = unpack2(fma2(q, k(-1.f), k(1.f)));
  return pack2(x.x > 0.f ? above.x : below.x, x.y > 0.f ? above.y : below.y);
}
__device__ __forceinline__ uint64_t activate2(uint64_t v, int act) {   // of a pair: two results from one reciprocal each
  uint64_t e;
  if (act == SILU) return mul2(v, fast_sigmoid2(v));
  if (act == SIGMOID) return fast_sigmoid2(v);
  if (act == GELU) return mul2(v, normal2(v, e));
  return v;
}
__device__ __forceinline__ float activate(float v, int act) { return unpack2(activate2(pack2(v, 0.f), act)).x; }
__device__ __forceinline__ void activate2(float& a, float& b, int act) {
  const float2 f = unpack2(activate2(pack2(a, b), act));
  a = f.x, b = f.y;
}
__device__ __forceinline__ uint64_t slope2(uint64_t z, int act) {   // act'(z) of a pair
  const uint64_t one = pack2(1.f, 1.f);
  if (act == GELU) {
    uint64_t e;
    const uint64_t n = normal2(z, e);
    return fma2(mul2(z, pack2(0.39894228040143268f, 0.39894228040143268f)), e, n);
  }
  const uint64_t s = fast_sigmoid2(z), rest = fma2(s, pack2(-1.f, -1.f), one);
  return act == SILU ? mul2(s, fma2(z, rest, one)) : mul2(s, rest);
}

// ---- CTA pairs -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t leaders(const void* p) {   // the address of the same place in the pair's first CTA
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(a) : "r"(tc5::smem_addr(p)));
  return a;
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* slot, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5::smem_addr(slot)), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
}
// a box into this CTA's shared memory; its bytes count on the barrier at `bar` (a cluster address: the pair's first CTA's)
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];\n" ::"r"(
                   tc5::smem_addr(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
               : "memory");
}
// called by a whole converged warp; one lane issues
__device__ __forceinline__ void pair_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// the pair's finished instructions arrive on the barrier at this place in both CTAs
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred e;\n.reg .b16 m;\n"
      "mov.b16 m, 3;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}\n" ::"r"(tc5::smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
}
// tc5::mbar_wait for a whole warp, for arrivals of either CTA
__device__ __forceinline__ bool pair_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = tc5::smem_addr(bar);
  bool done = false;
  for (uint32_t it = 0; it < (1u << 22) && !done; ++it) {
    uint32_t d;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(d)
        : "r"(addr), "r"(parity)
        : "memory");
    done = d;
  }
  return __all_sync(0xffffffffu, done);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {   // 32 columns of the lane's row
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32];\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]),
        "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]),
        "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}

// ---- the product -----------------------------------------------------------------------------------------------------------
// D[i, j] = sum over k of A(i, k) B(j, k).  `out`, `z` and `residual` are [tokens][features]: token i and feature j, or the other way round.
struct Product {
  int rows, cols;             // extents of i and j
  int steps;                  // of 64 along k
  int tiles_i, tiles_j;
  int whole, splits;          // tiles that are formed whole, and the parts along k of each of the others
  int act;
  int features;               // extent of out's rows, which lie as far apart
  int wide;                   // out, z and residual: rows on boundaries of 32 or 16 bytes, else 0
  uint32_t idesc;
  void *out, *z;              // z: what the activation is applied to, or NULL
  const void *bias, *residual;
  float* parts;               // of the tiles that are not formed whole: [tile][part][256 x BN], features side by side
  int64_t tokens;
};

constexpr int BK = 64, A_BYTES = 128 * BK * 2, EPILOGUE = 8, THREADS = 32 * (EPILOGUE + 2);   // warps that carry tiles out, and two more
constexpr int b_bytes(int bn) { return bn / 2 * BK * 2; }
constexpr int stages_of(int bn) { return bn == 256 ? 6 : bn == 128 ? 8 : bn == 64 ? 10 : 11; }
constexpr size_t smem_of(int bn) { return (size_t)stages_of(bn) * (A_BYTES + b_bytes(bn)) + 1024; }

struct Tile {
  int i, j, part, k0, k1;   // part: of the tiles that are not formed whole, else -1
};
// Tiles of eight row blocks, column by column: those at work at one time share their rows of A and B in L2.
__device__ __forceinline__ Tile tile_of(const Product& p, int t) {
  int part = -1, q = 0;
  if (t >= p.whole) {
    part = t - p.whole;
    t = p.whole + part / p.splits;
    q = part % p.splits;
  }
  const int n = part < 0 ? 1 : p.splits, group = t / (8 * p.tiles_j), first = group * 8, height = min(8, p.tiles_i - first);
  t -= group * 8 * p.tiles_j;
  return Tile{first + t % height, t / height, part, (int)((int64_t)p.steps * q / n), (int)((int64_t)p.steps * (q + 1) / n)};
}

__device__ __forceinline__ void store32(void* p, uint4 a, uint4 b) {   // 32 bytes, on such a boundary
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z),
               "r"(b.w)
               : "memory");
}
// 32 neighbouring elements of a row; `wide`: the boundary it lies on
template <typename T>
__device__ __forceinline__ void put_row(T* p, int wide, const float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint4 w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = v[q * 16 + h * 8 + e];
      w[h] = pack8<T>(x);
    }
    if (wide == 32) {
      store32(p + q * 16, w[0], w[1]);
    } else {
      reinterpret_cast<uint4*>(p)[2 * q] = w[0];
      reinterpret_cast<uint4*>(p)[2 * q + 1] = w[1];
    }
  }
}
template <typename T>
__device__ __forceinline__ void add_row(const T* p, float (&v)[32]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float x[8];
    unpack8<T>(reinterpret_cast<const uint4*>(p)[q], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[q * 8 + e] += x[e];
  }
}

// SWAPPED: i are features and j tokens
template <typename T, int BN, bool A_MN, bool B_MN, bool SWAPPED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    linear_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Product p) {
  constexpr int STAGES = stages_of(BN), STAGE = A_BYTES + b_bytes(BN);
  constexpr uint32_t COLUMNS = 2 * BN;   // of tensor memory: two tiles
  extern __shared__ unsigned char raw[];
  unsigned char* tiles = raw + ((1024 - (tc5::smem_addr(raw) & 1023)) & 1023);
  __shared__ uint64_t full[STAGES], empty[STAGES], done[2], taken[2];
  __shared__ uint32_t tmem_slot;
  __shared__ float turned[SWAPPED ? 1 : EPILOGUE][32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cta_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc5::mbar_init(&full[s], 1);
      tc5::mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc5::mbar_init(&done[s], 1);
      tc5::mbar_init(&taken[s], 2 * EPILOGUE);   // the epilogue warps of both CTAs
    }
    tc5::fence_mbar_init();
  }
  wait_for_predecessor();   // (no tensor memory is held meanwhile: a kernel ahead that still has its own to come by would wait for this one)
  if (warp == EPILOGUE + 1) pair_tmem_alloc(&tmem_slot, COLUMNS);
  __syncthreads();
  tc5::fence_before_sync();
  cluster_sync();
  tc5::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const int n_tiles = p.whole + (p.tiles_i * p.tiles_j - p.whole) * p.splits, first = blockIdx.x >> 1, by = gridDim.x >> 1;
  bool ok = true;
  if (warp == EPILOGUE) {
    if (lane == 0) {
      tma::prefetch_map(&map_a);
      tma::prefetch_map(&map_b);
    }
    int s = 0;
    uint32_t phase = 0;
    int issued = 0;
    for (int t = first; t < n_tiles && ok; t += by) {
      const Tile at = tile_of(p, t);
      const int i0 = at.i * 256 + rank * 128, j0 = at.j * BN + rank * (BN / 2);
      for (int k = at.k0; k < at.k1; ++k) {
        ok = pair_wait(&empty[s], phase ^ 1u);
        if (!ok) break;
        if (lane == 0) {
          unsigned char* a = tiles + s * STAGE;
          unsigned char* b = a + A_BYTES;
          const uint32_t bar = leaders(&full[s]);
          if (rank == 0) tc5::mbar_expect_tx(&full[s], 2 * STAGE);
          if constexpr (A_MN) {
            pair_load(a, &map_a, i0, k * BK, bar);
            pair_load(a + A_BYTES / 2, &map_a, i0 + 64, k * BK, bar);
          } else {
            pair_load(a, &map_a, k * BK, i0, bar);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int c = 0; c < BN / 128; ++c) pair_load(b + c * 64 * BK * 2, &map_b, j0 + c * 64, k * BK, bar);
          } else {
            pair_load(b, &map_b, k * BK, j0, bar);
          }
        }
        __syncwarp();
        issued = min(issued + 1, STAGES);
        if (++s == STAGES) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    // its copies have landed before a CTA leaves: what was waited for by the other warps in any case, unless a wait ran out
    if (!ok && rank == 0)
      for (int i = 0; i < issued; ++i) {
        if (--s < 0) {
          s = STAGES - 1;
          phase ^= 1u;
        }
        (void)pair_wait(&full[s], phase);
      }
  } else if (warp == EPILOGUE + 1) {
    if (rank == 0) {
      int s = 0, turn = 0;
      uint32_t phase = 0;
      for (int t = first; t < n_tiles && ok; t += by, ++turn) {
        const Tile at = tile_of(p, t);
        const int half = turn & 1;
        ok = pair_wait(&taken[half], ((turn >> 1) & 1) ^ 1u);
        if (!ok) break;
        tc5::fence_after_sync();
        const uint32_t acc = tmem + half * BN;
        for (int k = at.k0; k < at.k1; ++k) {
          ok = pair_wait(&full[s], phase);
          if (!ok) break;
          tc5::fence_after_sync();
          const uint32_t a = tc5::smem_addr(tiles + s * STAGE), b = a + A_BYTES;
          const uint64_t da = A_MN ? tc5::smem_desc(a, 64 * BK * 2, 1024) : tc5::smem_desc(a, 16, 1024);
          const uint64_t db = B_MN ? tc5::smem_desc(b, 64 * BK * 2, 1024) : tc5::smem_desc(b, 16, 1024);
#pragma unroll
          for (int q = 0; q < BK / 16; ++q)   // 16 of the contraction: 32 bytes along a row, or 16 rows
            pair_mma(acc, da + ((A_MN ? q * 2048 : q * 32) >> 4), db + ((B_MN ? q * 2048 : q * 32) >> 4), p.idesc, k > at.k0 || q > 0);
          pair_commit(&empty[s]);
          if (++s == STAGES) {
            s = 0;
            phase ^= 1u;
          }
        }
        if (ok) pair_commit(&done[half]);
      }
    }
  } else {
    int turn = 0;
    for (int t = first; t < n_tiles && ok; t += by, ++turn) {
      const Tile at = tile_of(p, t);
      const int half = turn & 1;
      ok = pair_wait(&done[half], (turn >> 1) & 1);
      if (!ok) break;
      tc5::fence_after_sync();
      // a warp reads its quarter of the lanes; warps four apart share it column block by column block
      const int local = rank * 128 + (warp & 3) * 32 + lane, i = at.i * 256 + local;
      const bool live = i < p.rows;
#pragma unroll 1
      for (int c = warp / 4 * 32; c < BN; c += EPILOGUE / 4 * 32) {
        const int j = at.j * BN + c;
        if (j >= p.cols) break;   // (the same for all)
        float v[32];
        __syncwarp();
        tmem_ld32(tmem + half * BN + c + ((uint32_t)((warp & 3) * 32) << 16), v);
        tc5::tmem_ld_wait();
        if (at.part >= 0) {
          float* part = p.parts + (int64_t)at.part * 256 * BN;
          if constexpr (!SWAPPED) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              store32(part + local * BN + c + q * 8, *reinterpret_cast<const uint4*>(&v[q * 8]), *reinterpret_cast<const uint4*>(&v[q * 8 + 4]));
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(c + e) * 256 + local] = v[e];
          }
        } else if constexpr (SWAPPED) {
          if (!live) continue;
          const float b = p.bias ? (float)static_cast<const T*>(p.bias)[i] : 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (j + e >= p.cols) break;
            const int64_t to = (int64_t)(j + e) * p.features + i;
            float x = v[e] + b;
            if (p.z) static_cast<T*>(p.z)[to] = static_cast<T>(x);
            x = activate(x, p.act);
            if (p.residual) x += (float)static_cast<const T*>(p.residual)[to];
            static_cast<T*>(p.out)[to] = static_cast<T>(x);
          }
        } else if (p.wide && j + 32 <= p.cols) {   // a lane writes 64 bytes of its row, whole sectors
          if (!live) continue;
          const int64_t to = (int64_t)i * p.features + j;
          if (p.bias) add_row<T>(static_cast<const T*>(p.bias) + j, v);
          if (p.z) put_row<T>(static_cast<T*>(p.z) + to, p.wide, v);
          if (p.act != NONE)
#pragma unroll
            for (int e = 0; e < 32; e += 2) activate2(v[e], v[e + 1], p.act);
          if (p.residual) add_row<T>(static_cast<const T*>(p.residual) + to, v);
          put_row<T>(static_cast<T*>(p.out) + to, p.wide, v);
        } else {   // rows on any boundary: turned round, so that a warp writes a row's 32 columns at a time
          const int col = j + lane, i0 = i - lane, rows = min(32, p.rows - i0);
          const bool here = col < p.cols;
          T res[32];   // (all on their way at once)
#pragma unroll
          for (int r = 0; r < 32; ++r)
            if (p.residual) res[r] = here && r < rows ? static_cast<const T*>(p.residual)[(int64_t)(i0 + r) * p.features + col] : static_cast<T>(0.f);
#pragma unroll
          for (int e = 0; e < 32; ++e) turned[warp][lane][e] = v[e];
          __syncwarp();
          const float b = p.bias && here ? (float)static_cast<const T*>(p.bias)[col] : 0.f;
#pragma unroll
          for (int r = 0; r < 32; ++r) v[r] = turned[warp][r][lane] + b;
          __syncwarp();
          if (!here) continue;
          const int64_t to = (int64_t)i0 * p.features + col;
          if (p.z)
#pragma unroll
            for (int r = 0; r < 32; ++r)
              if (r < rows) static_cast<T*>(p.z)[to + (int64_t)r * p.features] = static_cast<T>(v[r]);
          if (p.act != NONE)
#pragma unroll
            for (int r = 0; r < 32; r += 2) activate2(v[r], v[r + 1], p.act);
#pragma unroll
          for (int r = 0; r < 32; ++r)
            if (r < rows) static_cast<T*>(p.out)[to + (int64_t)r * p.features] = static_cast<T>(p.residual ? v[r] + (float)res[r] : v[r]);
        }
      }
      tc5::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_at(leaders(&taken[half]));
    }
  }
  if (!ok && lane == 0) atomicExch(&g_linear_timeout, 1);
  // neither CTA leaves while the other may still read its tiles or arrive on its barriers
  __syncthreads();
  tc5::fence_before_sync();
  cluster_sync();
  tc5::fence_after_sync();
  if (warp == EPILOGUE + 1) pair_tmem_dealloc(tmem, COLUMNS);
}

// Tiles that were formed in parts: the parts in their order, and what follows the product; four features a thread.
template <typename T, int BN, bool SWAPPED>
__global__ void __launch_bounds__(256) linear_join_kernel(const Product p) {
  constexpr int SIZE = 256 * BN, WIDTH = SWAPPED ? 256 : BN;   // features of a tile
  wait_for_predecessor();
  const int tile = blockIdx.y, at = (blockIdx.x * 256 + threadIdx.x) * 4, f_local = at % WIDTH, t_local = at / WIDTH;
  Product whole = p;
  whole.whole = p.tiles_i * p.tiles_j;
  const Tile where = tile_of(whole, p.whole + tile);
  const int f0 = (SWAPPED ? where.i * 256 : where.j * BN) + f_local, token = (SWAPPED ? where.j * BN : where.i * 256) + t_local;
  if (at >= SIZE || f0 >= p.features || token >= p.tokens) return;
  const float* part = p.parts + (int64_t)tile * p.splits * SIZE + at;
  float4 sum = *reinterpret_cast<const float4*>(part);
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) {
    const float4 q = *reinterpret_cast<const float4*>(part + (int64_t)s * SIZE);
    sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
  }
  const float v4[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int f = f0 + e;
    if (f >= p.features) break;
    const int64_t to = (int64_t)token * p.features + f;
    float v = v4[e];
    if (p.bias) v += (float)static_cast<const T*>(p.bias)[f];
    if (p.z) static_cast<T*>(p.z)[to] = static_cast<T>(v);
    v = activate(v, p.act);
    if (p.residual) v += (float)static_cast<const T*>(p.residual)[to];
    static_cast<T*>(p.out)[to] = static_cast<T>(v);
  }
}

// ---- few tokens, forward -----------------------------------------------------------------------------------------------------
// 16 features a CTA, whose warps share the contraction 256 at a time.  What bounds it is W's bytes, so what counts is loads on their way and
// little else: a lane loads 16 bytes of a row of W, and of x, straight into the registers of mma.sync's operands (which contraction index goes
// where does not matter as long as it is the same in both), four steps of 32 at once; nothing is converted or staged.  tcgen05 would need the
// bytes to pass through shared memory and a split contraction to occupy every SM.
constexpr int FEW_STEPS = 4, FEW_WARPS = 16;
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// eight neighbouring elements of a row from k on; zeros past its end, or where there is no row.  By ordinary loads: the kernel ahead may still
// write x, or W, when this one begins, and only of these is it known that they see what was written before wait_for_predecessor.
template <bool WIDE>
__device__ __forceinline__ uint4 eight(const uint16_t* row, int k, int K, bool there) {
  uint4 u = make_uint4(0, 0, 0, 0);
  if constexpr (WIDE) {
    if (there && k < K) u = *reinterpret_cast<const uint4*>(row + k);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (there && k + e < K) w[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return u;
}
template <typename T, int NT, bool WIDE>   // up to 8 NT tokens
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) linear_few_kernel(const Product p, const uint16_t* x, const uint16_t* w, int K) {
  __shared__ float sums[FEW_WARPS][16][8 * NT];
  constexpr int S = NT > 1 ? FEW_STEPS / 2 : FEW_STEPS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3, f0 = blockIdx.x * 16;
  const int n_tokens = (int)p.tokens;
  const uint16_t* rows[2] = {w + (int64_t)(f0 + g) * K, w + (int64_t)(f0 + g + 8) * K};
  wait_for_predecessor();
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  for (int k0 = warp * S * 32; k0 < K; k0 += warps * S * 32) {
    uint4 a[S][2], b[S][NT];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int k = k0 + s * 32 + t * 8;
      a[s][0] = eight<WIDE>(rows[0], k, K, f0 + g < p.features);
      a[s][1] = eight<WIDE>(rows[1], k, K, f0 + g + 8 < p.features);
#pragma unroll
      for (int n = 0; n < NT; ++n) b[s][n] = eight<WIDE>(x + (int64_t)(n * 8 + g) * K, k, K, n * 8 + g < n_tokens);
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_16816<T>(acc[n], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b[s][n].x, b[s][n].y);
        mma_16816<T>(acc[n], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b[s][n].z, b[s][n].w);
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sums[warp][g][n * 8 + 2 * t] = acc[n][0];
    sums[warp][g][n * 8 + 2 * t + 1] = acc[n][1];
    sums[warp][g + 8][n * 8 + 2 * t] = acc[n][2];
    sums[warp][g + 8][n * 8 + 2 * t + 1] = acc[n][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += blockDim.x) {
    const int f = f0 + (i & 15), token = i >> 4;
    if (f >= p.features || token >= n_tokens) continue;
    float v = 0.f;
    for (int q = 0; q < warps; ++q) v += sums[q][i & 15][token];
    if (p.bias) v += (float)static_cast<const T*>(p.bias)[f];
    const int64_t to = (int64_t)token * p.features + f;
    if (p.z) static_cast<T*>(p.z)[to] = static_cast<T>(v);
    v = activate(v, p.act);
    if (p.residual) v += (float)static_cast<const T*>(p.residual)[to];
    static_cast<T*>(p.out)[to] = static_cast<T>(v);
  }
}

// ---- around the gradient's products ------------------------------------------------------------------------------------------
// rows of `cols` to rows `pitch` apart, of up to two operands; eight elements a thread
struct Copies {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int64_t rows[2];
  int cols[2], pitch[2];
};
__global__ void __launch_bounds__(128) linear_pad_kernel(const Copies c) {
  const int o = blockIdx.z, at = (blockIdx.x * 128 + threadIdx.x) * 8, cols = c.cols[o];
  if (at >= cols) return;
  constexpr int U = 4;   // rows on their way at once
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // (these wait for the whole of it before they touch anything)
  for (int64_t r0 = (int64_t)blockIdx.y * U; r0 < c.rows[o]; r0 += (int64_t)gridDim.y * U) {
    uint4 u[U];
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = eight<false>(c.src[o] + (r0 + i) * cols, at, cols, r0 + i < c.rows[o]);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (r0 + i < c.rows[o]) *reinterpret_cast<uint4*>(c.dst[o] + (r0 + i) * c.pitch[o] + at) = u[i];
  }
}

// Two elements of the kept z within their type's finite values (a NaN stays).  z was rounded to be kept: what left the type's range there is infinite,
// and infinity times the slope's zero would be NaN.  The activation saw the number itself, whose slope is that of the type's largest: 0 or 1.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;\n min.NaN.f16x2 %0, %0, %2;" : "+r"(w) : "r"(0xFBFFFBFFu), "r"(0x7BFF7BFFu));
  else asm("max.NaN.bf16x2 %0, %0, %1;\n min.NaN.bf16x2 %0, %0, %2;" : "+r"(w) : "r"(0xFF7FFF7Fu), "r"(0x7F7F7F7Fu));
  return w;
}

// dz = dy act'(z) (rounded for the products; `dz` NULL: not wanted) and, for db, its sums over the rows of a CTA, unrounded.  Warps take rows in
// turn, lanes E columns each; four rows are on their way at once.
template <typename T, int E>
__global__ void __launch_bounds__(256, 3) linear_dz_kernel(const T* dy, const T* z, T* dz, float* sums, int64_t rows, int cols, int pitch, int act) {
  constexpr int P = (E + 1) / 2, U = 4;
  using Raw = std::conditional_t<E == 8, uint4, std::conditional_t<E == 2, uint32_t, uint16_t>>;
  __shared__ float part[8][32 * E];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = (blockIdx.x * 32 + lane) * E;
  uint64_t total[P];
#pragma unroll
  for (int i = 0; i < P; ++i) total[i] = 0ull;
  auto word = [](const Raw& u, int i) -> uint32_t {   // two elements; of one alone the second is zero
    if constexpr (E > 1) return reinterpret_cast<const uint32_t*>(&u)[i];
    else return u;
  };
  if (c < cols) {
    const int64_t step = (int64_t)gridDim.y * 8;
    for (int64_t r0 = blockIdx.y * 8 + warp; r0 < rows; r0 += step * U) {
      Raw d[U], v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        d[u] = v[u] = Raw{};
        if (r0 + u * step < rows) {
          d[u] = *reinterpret_cast<const Raw*>(dy + (r0 + u * step) * cols + c);
          if (act != NONE) v[u] = *reinterpret_cast<const Raw*>(z + (r0 + u * step) * cols + c);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Raw out;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          uint64_t g = widen2<T>(word(d[u], i));
          if (act != NONE) g = mul2(g, slope2(widen2<T>(finite2<T>(word(v[u], i))), act));
          total[i] = add2(total[i], g);   // (a row past the end adds zeros)
          if constexpr (E > 1) reinterpret_cast<uint32_t*>(&out)[i] = narrow2<T>(g);
          else *reinterpret_cast<T*>(&out) = static_cast<T>(unpack2(g).x);
        }
        if (dz && r0 + u * step < rows) *reinterpret_cast<Raw*>(dz + (r0 + u * step) * pitch + c) = out;
      }
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 f = unpack2(total[i]);
    part[warp][lane * E + 2 * i] = f.x;
    if (E > 1) part[warp][lane * E + 2 * i + 1] = f.y;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * E; i += 256) {
    const int col = blockIdx.x * 32 * E + i;
    if (col >= cols) continue;
    float s = part[0][i];
#pragma unroll
    for (int w = 1; w < 8; ++w) s += part[w][i];
    sums[(int64_t)blockIdx.y * cols + col] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) linear_dbias_kernel(const float* sums, T* dbias, int cols, int n) {
  wait_for_predecessor();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int i = 0; i < n; ++i) s += sums[(int64_t)i * cols + c];
  dbias[c] = static_cast<T>(s);
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
constexpr int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct Plan {
  int bn, whole, splits;
  int64_t parts;   // floats
};
// The column tile, and the parts that the tiles of the last, incomplete round are formed in, with the least time by this model: 0.32 us a step
// of 256 x 256 (0.28 of 128 columns, 0.2 of fewer: what the loads take), 2 us a tile that nothing hides, and 3 us with what the parts move.
// (8192 x 2048 from 16384 tokens, 256 tiles on 74 pairs: 408 us in whole tiles, 362 with the last 34 in two parts each.)
Plan plan_of(int64_t rows, int64_t cols, int64_t depth, bool swapped) {
  const int pairs = sm_count() / 2, steps = (int)((depth + BK - 1) / BK);
  Plan best{256, 0, 1, 0};
  double least = 1e30;
  for (int bn : {256, 128, 64, 32}) {
    if (swapped ? (bn < cols && bn < 256) || bn / 2 >= up(cols, 32) : bn < 128) continue;
    const int64_t tiles = (rows + 255) / 256 * ((cols + bn - 1) / bn), whole = tiles / pairs * pairs, rest = tiles - whole;
    const double step = bn == 256 ? 0.32 : bn == 128 ? 0.28 : 0.2;
    for (int s = 1; s <= 16 && (s == 1 || (rest > 0 && rest * s <= pairs && steps / s >= 4)); ++s) {
      const double moved = s > 1 ? 8.0 * rest * s * 256 * bn : 0;
      const double cost = (double)whole / pairs * (steps * step + 2) + (rest > 0 ? (steps + s - 1) / s * step + 2 : 0) + (s > 1 ? 3 + moved / 6e6 : 0);
      if (cost < least) {
        least = cost;
        best = s > 1 ? Plan{bn, (int)whole, s, rest * s * 256 * bn} : Plan{bn, (int)tiles, 1, 0};
      }
    }
  }
  return best;
}

struct Operand {
  const void* base;
  int64_t rows, cols, pitch;   // as it lies
};
template <typename T, int BN, bool A_MN, bool B_MN, bool SWAPPED>
int launch_tiles(const Operand& a, const Operand& b, Product p, cudaStream_t st) {
  CUtensorMap ma, mb;
  bind_context();
  if (int e = tma::encode_bf16_2d(&ma, a.base, a.rows, a.cols, a.pitch, A_MN ? 64 : 128)) return set_error(B200GDN_ERR_CUDA, "linear: tensor map of A (%d)", e);
  if (int e = tma::encode_bf16_2d(&mb, b.base, b.rows, b.cols, b.pitch, B_MN ? 64 : BN / 2)) return set_error(B200GDN_ERR_CUDA, "linear: tensor map of B (%d)", e);
  p.tiles_i = (p.rows + 255) / 256;
  p.tiles_j = (p.cols + BN - 1) / BN;
  const uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
  p.idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
  auto kern = linear_kernel<T, BN, A_MN, B_MN, SWAPPED>;
  if (int e = ensure_smem(kern, smem_of(BN))) return e;
  // With one round of tiles a good part of the time is the launch, barriers and tensor memory: that begins while the kernel ahead finishes.
  const int rest = p.tiles_i * p.tiles_j - p.whole;   // (checked to be within an int)
  const int64_t tiles = p.whole + (int64_t)rest * p.splits;
  const int pairs = (int)(tiles < sm_count() / 2 ? tiles : sm_count() / 2);
  launch_overlapped(tiles <= pairs, kern, dim3(2 * pairs), THREADS, smem_of(BN), st, ma, mb, p);
  if (int e = check_launch("linear")) return e;
  if (rest == 0) return 0;
  launch_overlapped(true, linear_join_kernel<T, BN, SWAPPED>, dim3(256 * BN / 1024, rest), 256, 0, st, p);
  return check_launch("linear_join");
}

// A and B as D's rows and columns; `swapped`: D's rows are features
template <typename T, bool A_MN, bool B_MN>
int launch_product(const Operand& a, const Operand& b, int64_t depth, Product p, bool swapped, float* parts, cudaStream_t st) {
  const int64_t most = ((int64_t)p.rows + 255) / 256 * (((int64_t)p.cols + 31) / 32);
  if (most > INT32_MAX / 16) return set_error(B200GDN_ERR_UNSUPPORTED, "linear: a result of more than 2^27 tiles");
  const Plan plan = plan_of(p.rows, p.cols, depth, swapped);
  p.whole = plan.whole;
  p.steps = (int)((depth + BK - 1) / BK);
  p.splits = plan.splits;
  p.parts = parts;
  p.tokens = swapped ? p.cols : p.rows;
  p.features = swapped ? p.rows : p.cols;
  uintptr_t bits = reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.z) | reinterpret_cast<uintptr_t>(p.bias) |
                   reinterpret_cast<uintptr_t>(p.residual) | (uintptr_t)p.features * 2;
  p.wide = bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : 0;
  if (!swapped) return plan.bn == 256 ? launch_tiles<T, 256, A_MN, B_MN, false>(a, b, p, st) : launch_tiles<T, 128, A_MN, B_MN, false>(a, b, p, st);
  if constexpr (!B_MN)
    return plan.bn == 256   ? launch_tiles<T, 256, A_MN, false, true>(a, b, p, st)
           : plan.bn == 128 ? launch_tiles<T, 128, A_MN, false, true>(a, b, p, st)
           : plan.bn == 64  ? launch_tiles<T, 64, A_MN, false, true>(a, b, p, st)
                            : launch_tiles<T, 32, A_MN, false, true>(a, b, p, st);
  return B200GDN_ERR_UNSUPPORTED;
}

constexpr int64_t FEW = 16, SWAP = 256;   // tokens up to which W passes through registers, and up to which its rows are the tile's 256

// The workspace, piece by piece on 256-byte boundaries; without a base it only counts.
struct Space {
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += up(bytes, 256);
    return p;
  }
};
bool fits_tma(const void* p, int64_t cols) { return cols % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Two operands, each itself or its copy with rows 16 bytes apart (a base of NULL: no such operand).
int operands_of(Operand& a, Operand& b, Space& space, cudaStream_t st, bool run) {
  Copies c{};
  int n = 0;
  int64_t x = 1, y = 1;
  for (Operand* o : {&a, &b}) {
    if (o->base == nullptr || fits_tma(o->base, o->cols)) continue;
    o->pitch = up(o->cols, 8);
    void* copy = space.take(o->rows * o->pitch * 2);
    c.src[n] = static_cast<const uint16_t*>(o->base);
    c.dst[n] = static_cast<uint16_t*>(copy);
    c.rows[n] = o->rows;
    c.cols[n] = (int)o->cols;
    c.pitch[n] = (int)o->pitch;
    o->base = copy;
    x = x > (o->cols + 1023) / 1024 ? x : (o->cols + 1023) / 1024;
    y = y > o->rows ? y : o->rows;
    ++n;
  }
  if (n == 0 || !run) return 0;
  const int64_t most = 16 * (int64_t)sm_count() / x + 1;
  y = (y + 3) / 4;
  linear_pad_kernel<<<dim3((unsigned)x, (unsigned)(y < most ? y : most), n), 128, 0, st>>>(c);
  return check_launch("linear_pad");
}

template <typename T>
int forward(const b200gdn_linear_args& a, Space& space, cudaStream_t st, bool run) {
  Product p{};
  p.act = a.activation;
  p.out = a.y;
  p.z = a.activation == NONE ? nullptr : a.z;
  p.bias = a.bias;
  p.residual = a.residual;
  if (a.rows <= FEW) {
    if (!run) return 0;
    p.tokens = a.rows;
    p.features = a.N;
    // sixteen warps a CTA where features are few and the contraction long, else eight
    const int grid = (a.N + 15) / 16, warps = grid < 2 * sm_count() && a.K > 2048 ? 16 : 8;
    const bool wide = fits_tma(a.x, a.K) && fits_tma(a.weight, a.K);
    auto go = [&](auto kern) {
      launch_overlapped(true, kern, dim3(grid), warps * 32, 0, st, p, static_cast<const uint16_t*>(a.x), static_cast<const uint16_t*>(a.weight), a.K);
    };
    if (a.rows <= 8) wide ? go(linear_few_kernel<T, 1, true>) : go(linear_few_kernel<T, 1, false>);
    else wide ? go(linear_few_kernel<T, 2, true>) : go(linear_few_kernel<T, 2, false>);
    return check_launch("linear_few");
  }
  Operand x{a.x, a.rows, a.K, a.K}, w{a.weight, a.N, a.K, a.K};
  if (int e = operands_of(x, w, space, st, run)) return e;
  const bool swapped = a.rows <= SWAP;
  p.rows = swapped ? a.N : (int)a.rows;
  p.cols = swapped ? (int)a.rows : a.N;
  float* parts = static_cast<float*>(space.take(plan_of(p.rows, p.cols, a.K, swapped).parts * 4));
  if (!run) return 0;
  return swapped ? launch_product<T, false, false>(w, x, a.K, p, true, parts, st) : launch_product<T, false, false>(x, w, a.K, p, false, parts, st);
}

template <typename T>
int backward(const b200gdn_linear_args& a, Space& space, cudaStream_t st, bool run) {
  // dz with rows that TMA reads: dy itself where it is that and lies so
  const bool apart = (a.dx || a.dweight) && (a.activation != NONE || !fits_tma(a.dy, a.N));
  Operand dz{a.dy, a.rows, a.N, a.N};
  T* made = nullptr;
  if (apart) {
    dz.pitch = up(a.N, 8);
    made = static_cast<T*>(space.take(a.rows * dz.pitch * 2));
    dz.base = made;
  }
  // columns of a thread: 16 bytes of them, two, or one, as width and boundaries allow
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.z) | (uintptr_t)a.N * 2;
  const int each = bits % 16 == 0 ? 8 : bits % 4 == 0 ? 2 : 1, per = 32 * each;
  const int64_t columns = (a.N + per - 1) / per;
  int64_t y = 3 * (int64_t)sm_count() / columns;   // one round of CTAs
  if (y < 1) y = 1;
  if (y > (a.rows + 31) / 32) y = (a.rows + 31) / 32;
  float* sums = a.dbias ? static_cast<float*>(space.take(y * a.N * 4)) : nullptr;
  if (run && (apart || a.dbias)) {
    auto go = [&](auto kern) {
      kern<<<dim3((unsigned)columns, (unsigned)y), 256, 0, st>>>(static_cast<const T*>(a.dy), static_cast<const T*>(a.z), made, sums, a.rows, a.N, (int)dz.pitch,
                                                          a.activation);
    };
    each == 8 ? go(linear_dz_kernel<T, 8>) : each == 2 ? go(linear_dz_kernel<T, 2>) : go(linear_dz_kernel<T, 1>);
    if (int e = check_launch("linear_dz")) return e;
    if (a.dbias) {
      launch_overlapped(true, linear_dbias_kernel<T>, dim3((a.N + 255) / 256), 256, 0, st, (const float*)sums, static_cast<T*>(a.dbias), a.N, (int)y);
      if (int e = check_launch("linear_dbias")) return e;
    }
  }
  Operand x{a.dweight ? a.x : nullptr, a.rows, a.K, a.K}, w{a.dx ? a.weight : nullptr, a.N, a.K, a.K};
  if (int e = operands_of(x, w, space, st, run)) return e;
  if (a.dx) {
    const bool swapped = a.rows <= SWAP;
    Product p{};
    p.out = a.dx;
    p.rows = swapped ? a.K : (int)a.rows;
    p.cols = swapped ? (int)a.rows : a.K;
    float* parts = static_cast<float*>(space.take(plan_of(p.rows, p.cols, a.N, swapped).parts * 4));
    if (run)
      if (int e = swapped ? launch_product<T, true, false>(w, dz, a.N, p, true, parts, st) : launch_product<T, false, true>(dz, w, a.N, p, false, parts, st)) return e;
  }
  if (a.dweight) {
    Product p{};
    p.out = a.dweight;
    p.rows = a.N;
    p.cols = a.K;
    float* parts = static_cast<float*>(space.take(plan_of(p.rows, p.cols, a.rows, false).parts * 4));
    if (run)
      if (int e = launch_product<T, true, true>(dz, x, a.rows, p, false, parts, st)) return e;
  }
  return 0;
}

}  // namespace

int64_t linear_workspace(const b200gdn_linear_args& a, bool bwd) {
  Space space{nullptr};
  (void)(bwd ? backward<__half>(a, space, nullptr, false) : forward<__half>(a, space, nullptr, false));
  return space.used;
}

int launch_linear(const b200gdn_linear_args& a, cudaStream_t st, bool bwd) {
  Space space{static_cast<char*>(a.workspace)};
  if (a.dtype == 0) return bwd ? backward<__nv_bfloat16>(a, space, st, true) : forward<__nv_bfloat16>(a, space, st, true);
  return bwd ? backward<__half>(a, space, st, true) : forward<__half>(a, space, st, true);
}

int linear_timeout_flag() {
  int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_linear_timeout, sizeof(int));
  if (v) cudaMemcpyToSymbol(g_linear_timeout, &zero, sizeof(int));
  return v;
}

}  // namespace gdn

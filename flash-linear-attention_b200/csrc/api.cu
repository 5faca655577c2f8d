// C ABI of the library (declared in include/b200gdn.h): argument checks, stage sequencing, error text.
#include <cstdarg>
#include <cstdio>

#include "gdn_common.cuh"
#include "tc5.cuh"

namespace gdn {

static thread_local char g_err[512] = "";
static thread_local int g_launches = 0;

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

void reset_launch_count() { g_launches = 0; }

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(B200GDN_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  ++g_launches;
  return 0;
}

static int check_chunk_args(const b200gdn_chunk_args* a, const char* who) {
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_chunk_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes,
                     sizeof(b200gdn_chunk_args));
  if (a->rows <= 0 || a->H <= 0 || a->HV <= 0 || a->n_seq <= 0 || a->n_chunks <= 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%d H=%d HV=%d n_seq=%d n_chunks=%d)", who, a->rows,
                     a->H, a->HV, a->n_seq, a->n_chunks);
  if (a->HV % a->H != 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: HV=%d not a multiple of H=%d", who, a->HV, a->H);
  if (a->chunk_meta == nullptr || a->seq_meta == nullptr)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: chunk tables missing", who);
  if (a->HV > 65535 || a->n_seq > 65535)
    return set_error(B200GDN_ERR_UNSUPPORTED, "%s: HV and n_seq are grid y/z dimensions (<= 65535)", who);
  return 0;
}

#define REQUIRE(ptr, who)                                                                  \
  if ((ptr) == nullptr) return gdn::set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: %s is NULL", who, #ptr)

}  // namespace gdn

namespace gdn {
__device__ int g_selftest_timeout = 0;
// One warp waits on an mbarrier that nothing will ever complete, with a short limit: the wait must give up, raise the
// flag and let the kernel end normally (what every wait of the real kernels does when a completion is lost).
__global__ void selftest_wait_expiry_kernel(uint32_t limit) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    tc5::mbar_init(&bar, 1);
    tc5::fence_mbar_init();
  }
  __syncthreads();
  const bool ok = tc5::mbar_wait(&bar, 0, limit);
  if (!ok && threadIdx.x == 0) atomicExch(&g_selftest_timeout, 1);
}
static int selftest_timeout_flag() {
  int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_selftest_timeout, sizeof(int));
  if (v) cudaMemcpyToSymbol(g_selftest_timeout, &zero, sizeof(int));
  return v;
}
}  // namespace gdn

extern "C" {

int b200gdn_chunk_fwd(const b200gdn_chunk_args* a, void* stream) {
  using namespace gdn;
  g_launches = 0;
  if (int e = check_chunk_args(a, "chunk_fwd")) return e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint32_t m = a->stage_mask ? a->stage_mask : (B200GDN_FWD_INTRA | B200GDN_FWD_SCAN | B200GDN_FWD_OUT);
  if (m & B200GDN_FWD_INTRA) {
    REQUIRE(a->k, "chunk_fwd"); REQUIRE(a->v, "chunk_fwd"); REQUIRE(a->g, "chunk_fwd"); REQUIRE(a->beta, "chunk_fwd");
    REQUIRE(a->gamma, "chunk_fwd"); REQUIRE(a->w, "chunk_fwd"); REQUIRE(a->u, "chunk_fwd");
    if (!(a->options & B200GDN_FORWARD_ONLY)) { REQUIRE(a->A, "chunk_fwd"); }
    if (int e = launch_intra_fwd(*a, st)) return e;
  }
  if ((m & B200GDN_FWD_SCAN) && (m & B200GDN_FWD_OUT)) {
    // the scan forms the output itself from the tiles it holds on chip: h and v_new are written for the backward
    // pass only (either may be NULL when no backward pass follows)
    REQUIRE(a->k, "chunk_fwd"); REQUIRE(a->w, "chunk_fwd"); REQUIRE(a->gamma, "chunk_fwd");
    REQUIRE(a->q, "chunk_fwd"); REQUIRE(a->o, "chunk_fwd");
    if (int e = launch_scan_out_fwd(*a, st)) return e;
    return 0;
  }
  if (m & B200GDN_FWD_SCAN) {
    REQUIRE(a->k, "chunk_fwd"); REQUIRE(a->w, "chunk_fwd"); REQUIRE(a->gamma, "chunk_fwd");
    if (int e = launch_scan_fwd(*a, st)) return e;
  }
  if (m & B200GDN_FWD_OUT) {
    if (a->options & B200GDN_PREP_L2NORM)
      return set_error(B200GDN_ERR_UNSUPPORTED, "chunk_fwd: the fused L2 norm needs the scan and the output in one call");
    REQUIRE(a->q, "chunk_fwd"); REQUIRE(a->k, "chunk_fwd"); REQUIRE(a->v_new, "chunk_fwd"); REQUIRE(a->h, "chunk_fwd");
    REQUIRE(a->gamma, "chunk_fwd"); REQUIRE(a->o, "chunk_fwd");
    if (int e = launch_out_fwd(*a, st)) return e;
  }
  return 0;
}

int b200gdn_chunk_bwd(const b200gdn_chunk_args* a, void* stream) {
  using namespace gdn;
  g_launches = 0;
  if (int e = check_chunk_args(a, "chunk_bwd")) return e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint32_t m =
      a->stage_mask ? a->stage_mask : (B200GDN_BWD_DVLOCAL | B200GDN_BWD_SCAN | B200GDN_BWD_DQKWG | B200GDN_BWD_WY);
  if ((m & B200GDN_BWD_DVLOCAL) && (m & B200GDN_BWD_SCAN)) {
    // the reverse scan forms the chunk-local part of dv itself from the tiles it holds on chip; dv2 is an output only
    // (NULL: not stored, e.g. when only dh0 of a shard is wanted)
    REQUIRE(a->q, "chunk_bwd"); REQUIRE(a->k, "chunk_bwd"); REQUIRE(a->w, "chunk_bwd"); REQUIRE(a->gamma, "chunk_bwd");
    REQUIRE(a->d_o, "chunk_bwd");
    if (int e = launch_scan_dvl_bwd(*a, st)) return e;
  } else {
    if (m & B200GDN_BWD_DVLOCAL) {
      REQUIRE(a->q, "chunk_bwd"); REQUIRE(a->k, "chunk_bwd"); REQUIRE(a->gamma, "chunk_bwd"); REQUIRE(a->d_o, "chunk_bwd");
      REQUIRE(a->dv2, "chunk_bwd");
      if (int e = launch_dv_local(*a, st)) return e;
    }
    if (m & B200GDN_BWD_SCAN) {
      REQUIRE(a->k, "chunk_bwd"); REQUIRE(a->w, "chunk_bwd"); REQUIRE(a->gamma, "chunk_bwd");
      if (int e = launch_scan_bwd(*a, st)) return e;
    }
  }
  if ((m & B200GDN_BWD_DQKWG) && (m & B200GDN_BWD_WY)) {
    // both chunk-local stages in one kernel: neither the chunk-local part of dk nor dG leaves the chip
    REQUIRE(a->q, "chunk_bwd"); REQUIRE(a->k, "chunk_bwd"); REQUIRE(a->v, "chunk_bwd"); REQUIRE(a->v_new, "chunk_bwd");
    REQUIRE(a->beta, "chunk_bwd"); REQUIRE(a->gamma, "chunk_bwd"); REQUIRE(a->A, "chunk_bwd"); REQUIRE(a->h, "chunk_bwd");
    REQUIRE(a->dh, "chunk_bwd"); REQUIRE(a->dv2, "chunk_bwd"); REQUIRE(a->d_o, "chunk_bwd"); REQUIRE(a->dq, "chunk_bwd");
    REQUIRE(a->dk, "chunk_bwd"); REQUIRE(a->dv, "chunk_bwd"); REQUIRE(a->dg, "chunk_bwd"); REQUIRE(a->dbeta, "chunk_bwd");
    return launch_bwd_local(*a, st);
  }
  if (m & B200GDN_BWD_DQKWG) {
    REQUIRE(a->q, "chunk_bwd"); REQUIRE(a->k, "chunk_bwd"); REQUIRE(a->v_new, "chunk_bwd"); REQUIRE(a->gamma, "chunk_bwd");
    REQUIRE(a->h, "chunk_bwd"); REQUIRE(a->dh, "chunk_bwd"); REQUIRE(a->dv2, "chunk_bwd"); REQUIRE(a->d_o, "chunk_bwd");
    REQUIRE(a->dq, "chunk_bwd"); REQUIRE(a->dk, "chunk_bwd"); REQUIRE(a->dG, "chunk_bwd");
    if (int e = launch_bwd_dqk(*a, st)) return e;
  }
  if (m & B200GDN_BWD_WY) {
    REQUIRE(a->k, "chunk_bwd"); REQUIRE(a->v, "chunk_bwd"); REQUIRE(a->beta, "chunk_bwd"); REQUIRE(a->gamma, "chunk_bwd");
    REQUIRE(a->A, "chunk_bwd"); REQUIRE(a->h, "chunk_bwd"); REQUIRE(a->dv2, "chunk_bwd");
    REQUIRE(a->dG, "chunk_bwd"); REQUIRE(a->dk, "chunk_bwd"); REQUIRE(a->dv, "chunk_bwd"); REQUIRE(a->dg, "chunk_bwd");
    REQUIRE(a->dbeta, "chunk_bwd");
    if (int e = launch_bwd_wy(*a, st)) return e;
  }
  return 0;
}

int b200gdn_recurrent_fwd(const b200gdn_recurrent_args* a, void* stream) {
  using namespace gdn;
  g_launches = 0;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "recurrent_fwd: args is NULL");
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_recurrent_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "recurrent_fwd: struct_bytes %d != %zu (ABI mismatch)", a->struct_bytes,
                     sizeof(b200gdn_recurrent_args));
  if (a->B <= 0 || a->T <= 0 || a->H <= 0 || a->HV <= 0 || a->n_seq <= 0 || a->HV % a->H != 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "recurrent_fwd: bad sizes B=%d T=%d H=%d HV=%d n_seq=%d", a->B, a->T, a->H,
                     a->HV, a->n_seq);
  if (a->qkv_dtype < 0 || a->qkv_dtype > 2) return set_error(B200GDN_ERR_BAD_ARGUMENT, "recurrent_fwd: qkv_dtype %d", a->qkv_dtype);
  if (a->HV > 65535 || a->n_seq > 65535)
    return set_error(B200GDN_ERR_UNSUPPORTED, "recurrent_fwd: HV and n_seq are grid dimensions (<= 65535)");
  REQUIRE(a->q, "recurrent_fwd"); REQUIRE(a->k, "recurrent_fwd"); REQUIRE(a->v, "recurrent_fwd");
  REQUIRE(a->beta, "recurrent_fwd"); REQUIRE(a->o, "recurrent_fwd");
  return launch_recurrent(*a, static_cast<cudaStream_t>(stream));
}

int b200gdn_affine_apply(const b200gdn_affine_args* a, void* stream) {
  using namespace gdn;
  g_launches = 0;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "affine_apply: args is NULL");
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_affine_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "affine_apply: struct_bytes %d != %zu (ABI mismatch)", a->struct_bytes,
                     sizeof(b200gdn_affine_args));
  if (a->HV <= 0 || a->K <= 0 || a->V <= 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "affine_apply: bad sizes");
  REQUIRE(a->M, "affine_apply"); REQUIRE(a->x, "affine_apply"); REQUIRE(a->out, "affine_apply");
  return launch_affine(*a, static_cast<cudaStream_t>(stream));
}

int b200gdn_cp_fold(const b200gdn_fold_args* a, void* stream) {
  using namespace gdn;
  g_launches = 0;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_fold: args is NULL");
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_fold_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_fold: struct_bytes %d != %zu (ABI mismatch)", a->struct_bytes,
                     sizeof(b200gdn_fold_args));
  if (a->HV <= 0 || a->count < 1 || a->first < 0 || (a->step != 1 && a->step != -1) || a->first + (a->count - 1) * a->step < 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_fold: bad sizes (HV=%d first=%d count=%d step=%d)", a->HV, a->first, a->count, a->step);
  if ((a->K != 64 && a->K != 128 && a->K != 256) || a->V <= 0 || a->V % 32 != 0)
    return set_error(B200GDN_ERR_UNSUPPORTED, "cp_fold: K=%d V=%d (K in {64,128,256}, V a multiple of 32)", a->K, a->V);
  REQUIRE(a->gathered, "cp_fold"); REQUIRE(a->out, "cp_fold");
  return launch_cp_fold(*a, static_cast<cudaStream_t>(stream));
}

int b200gdn_cp_prefix(const b200gdn_prefix_args* a, void* stream) {
  using namespace gdn;
  g_launches = 0;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_prefix: args is NULL");
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_prefix_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_prefix: struct_bytes %d != %zu (ABI mismatch)", a->struct_bytes,
                     sizeof(b200gdn_prefix_args));
  if (a->HV <= 0 || a->n_chains <= 0 || a->HV > 65535 || a->n_chains > 65535)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_prefix: bad sizes (HV=%d n_chains=%d)", a->HV, a->n_chains);
  if ((a->K != 64 && a->K != 128 && a->K != 256) || a->V <= 0 || a->V % 32 != 0)
    return set_error(B200GDN_ERR_UNSUPPORTED, "cp_prefix: K=%d V=%d (K in {64,128,256}, V a multiple of 32)", a->K, a->V);
  REQUIRE(a->table, "cp_prefix"); REQUIRE(a->M, "cp_prefix");
  if (a->out == nullptr && a->last == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "cp_prefix: no output given");
  return launch_cp_prefix(*a, static_cast<cudaStream_t>(stream));
}

int64_t b200gdn_saved_bytes(int32_t rows, int32_t H, int32_t HV, int32_t K, int32_t V, int32_t n_chunks) {
  (void)H;
  int64_t r = rows, hv = HV;
  return (int64_t)n_chunks * hv * 64 * 4  /* gamma */
         + r * hv * 64 * 2 * 2           /* A, qk */
         + r * hv * K * 2                /* w */
         + r * hv * V * 2 * 2            /* u, v_new */
         + (int64_t)n_chunks * hv * K * V * 2; /* h */
}

int64_t b200gdn_bwd_workspace_bytes(int32_t rows, int32_t H, int32_t HV, int32_t K, int32_t V, int32_t n_chunks) {
  int64_t r = rows, hv = HV;
  return (int64_t)n_chunks * hv * K * V * 2 /* dh */
         + r * hv * V * 2                    /* dv2 */
         + r * hv * 4                        /* dG (single stages) */
         + (HV > H ? 2 * r * H * K * 4 : 0); /* dq_acc, dk_part (single stages): fp32 sums over a group of value heads */
}

static int check_prep_args(const b200gdn_prep_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_prep_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes,
                     sizeof(b200gdn_prep_args));
  if (a->rows <= 0 || a->H <= 0 || a->HV <= 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: bad sizes", who);
  if (a->qk_dtype < 0 || a->qk_dtype > 2 || a->gb_dtype < 0 || a->gb_dtype > 2)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype codes are 0 (bf16), 1 (fp16), 2 (fp32)", who);
  if (a->flags & B200GDN_PREP_L2NORM) {
    if (a->K != 64 && a->K != 128 && a->K != 256 && a->K != 512)
      return set_error(B200GDN_ERR_UNSUPPORTED, "%s: K=%d (64, 128, 256 and 512 are built)", who, a->K);
    REQUIRE(a->q, who); REQUIRE(a->k, who); REQUIRE(a->rstd_q, who); REQUIRE(a->rstd_k, who);
    if (!bwd) { REQUIRE(a->qn, who); REQUIRE(a->kn, who); }
    else { REQUIRE(a->dqn, who); REQUIRE(a->dkn, who); REQUIRE(a->dq, who); REQUIRE(a->dk, who); }
  }
  if (a->flags & B200GDN_PREP_GATE) {
    if (a->HV > 256) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: HV=%d (at most 256 value heads)", who, a->HV);
    REQUIRE(a->g, who); REQUIRE(a->A_log, who);
    if (!bwd) { REQUIRE(a->g_out, who); }
    else { REQUIRE(a->dg, who); REQUIRE(a->dg_raw, who); REQUIRE(a->dA_log, who); REQUIRE(a->partials, who); }
  }
  if (a->flags & B200GDN_PREP_BETA_SIGMOID) {
    if (a->HV > 256) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: HV=%d (at most 256 value heads)", who, a->HV);
    REQUIRE(a->beta, who);
    if (!bwd) { REQUIRE(a->beta_out, who); }
    else { REQUIRE(a->dbeta, who); REQUIRE(a->dbeta_raw, who); }
  }
  return 0;
}

int b200gdn_prep_fwd(const b200gdn_prep_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_prep_args(a, "prep_fwd", false)) return e;
  return gdn::launch_prep(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_prep_bwd(const b200gdn_prep_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_prep_args(a, "prep_bwd", true)) return e;
  return gdn::launch_prep(*a, static_cast<cudaStream_t>(stream), true);
}

static int check_conv_args(const b200gdn_conv_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_conv_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes,
                     sizeof(b200gdn_conv_args));
  if (a->rows <= 0 || a->D <= 0 || a->n_seq <= 0 || a->n_tiles <= 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%d D=%d n_seq=%d n_tiles=%d)", who, a->rows, a->D, a->n_seq, a->n_tiles);
  if (a->D % 8 != 0) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: D=%d is not a multiple of 8", who, a->D);
  if (a->W < 2 || a->W > 4) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: kernel size %d (2, 3 and 4 are built)", who, a->W);
  if (a->dtype < 0 || a->dtype > 2) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype code %d", who, a->dtype);
  REQUIRE(a->tile_meta, who); REQUIRE(a->seq_meta, who); REQUIRE(a->x, who); REQUIRE(a->weight, who);
  if (!bwd) { REQUIRE(a->y, who); }
  else {
    REQUIRE(a->dy, who); REQUIRE(a->dx, who);
    if (a->dweight != nullptr) REQUIRE(a->partials, who);
  }
  return 0;
}

int b200gdn_conv_fwd(const b200gdn_conv_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_conv_args(a, "conv_fwd", false)) return e;
  return gdn::launch_conv(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_conv_bwd(const b200gdn_conv_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_conv_args(a, "conv_bwd", true)) return e;
  return gdn::launch_conv(*a, static_cast<cudaStream_t>(stream), true);
}

static int check_norm_gate_args(const b200gdn_norm_gate_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_norm_gate_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes,
                     sizeof(b200gdn_norm_gate_args));
  if (a->rows <= 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem", who);
  if (a->D != 64 && a->D != 128 && a->D != 256 && a->D != 512)
    return set_error(B200GDN_ERR_UNSUPPORTED, "%s: D=%d (64, 128, 256 and 512 are built)", who, a->D);
  if (a->dtype < 0 || a->dtype > 2) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype code %d", who, a->dtype);
  REQUIRE(a->x, who); REQUIRE(a->g, who);
  if (!bwd) { REQUIRE(a->y, who); }   // rstd may be NULL where no backward pass follows
  else { REQUIRE(a->rstd, who); REQUIRE(a->dy, who); REQUIRE(a->dx, who); REQUIRE(a->dg, who); REQUIRE(a->partials, who); }
  return 0;
}

int b200gdn_norm_gate_fwd(const b200gdn_norm_gate_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_norm_gate_args(a, "norm_gate_fwd", false)) return e;
  return gdn::launch_norm_gate(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_norm_gate_bwd(const b200gdn_norm_gate_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_norm_gate_args(a, "norm_gate_bwd", true)) return e;
  return gdn::launch_norm_gate(*a, static_cast<cudaStream_t>(stream), true);
}

int b200gdn_norm_gate_ctas(int64_t rows) { return gdn::norm_gate_grid(rows); }

// any of the addresses off a boundary (NULL is on every one)
static bool off_boundary(uintptr_t boundary, std::initializer_list<const void*> all) {
  for (const void* p : all)
    if (reinterpret_cast<uintptr_t>(p) % boundary != 0) return true;
  return false;
}

static int check_layer_norm_args(const b200gdn_layer_norm_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_layer_norm_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes,
                     sizeof(b200gdn_layer_norm_args));
  if (a->rows <= 0 || a->D <= 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%lld D=%d)", who, (long long)a->rows, a->D);
  if (a->rows > INT32_MAX) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", who);
  if (a->D > (1 << 23)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: D=%d (at most 2^23)", who, a->D);
  if (a->dtype < 0 || a->dtype > 2 || a->param_dtype < 0 || a->param_dtype > 2)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype codes %d, %d", who, a->dtype, a->param_dtype);
  if (!bwd) {
    REQUIRE(a->x, who); REQUIRE(a->y, who);
    if ((a->mean == nullptr) != (a->rstd == nullptr)) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: mean and rstd come together", who);
  } else {
    REQUIRE(a->z, who); REQUIRE(a->mean, who); REQUIRE(a->rstd, who); REQUIRE(a->dy, who); REQUIRE(a->dx, who);
    if (a->dweight != nullptr || a->dbias != nullptr) REQUIRE(a->partials, who);
  }
  const uintptr_t size = a->dtype == 2 ? 4 : 2, param_size = a->param_dtype == B200GDN_F32 ? 4 : 2;
  if (off_boundary(size, {a->x, a->residual, a->z, a->y, a->dy, a->dz, a->dx}) || off_boundary(param_size, {a->weight, a->bias, a->dweight, a->dbias}) ||
      off_boundary(4, {a->mean, a->rstd, a->partials}))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a tensor off its elements' boundary", who);
  return 0;
}

int b200gdn_layer_norm_fwd(const b200gdn_layer_norm_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_layer_norm_args(a, "layer_norm_fwd", false)) return e;
  return gdn::launch_layer_norm(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_layer_norm_bwd(const b200gdn_layer_norm_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_layer_norm_args(a, "layer_norm_bwd", true)) return e;
  return gdn::launch_layer_norm(*a, static_cast<cudaStream_t>(stream), true);
}

int b200gdn_layer_norm_ctas(int64_t rows) { return gdn::layer_norm_grid(rows); }

static int check_gated_recurrence_args(const b200gdn_gated_recurrence_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_gated_recurrence_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes,
                     sizeof(b200gdn_gated_recurrence_args));
  if (a->rows <= 0 || a->D <= 0 || a->n_seq <= 0 || a->seq_len < 0 || (a->seq_len == 0 && (a->n_chunks < 0 || a->longest < 0)))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%lld D=%d n_seq=%d seq_len=%d n_chunks=%d)", who, (long long)a->rows, a->D,
                     a->n_seq, a->seq_len, a->n_chunks);
  if (a->rows > (1 << 30)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^30 rows", who);
  if (a->D > (1 << 23)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: D=%d (at most 2^23)", who, a->D);
  if (a->seq_len > 0 && (int64_t)a->n_seq * a->seq_len > a->rows)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: %d sequences of %d tokens in %lld rows", who, a->n_seq, a->seq_len, (long long)a->rows);
  if (a->seq_len == 0) { REQUIRE(a->chunk_meta, who); REQUIRE(a->seq_meta, who); }
  if (a->dtype < 0 || a->dtype > 2 || (a->gate_dtype != a->dtype && a->gate_dtype != 2))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype codes %d, %d (the gate's is 2 or that of x)", who, a->dtype, a->gate_dtype);
  if (a->stride_x < a->D || a->stride_g < a->D)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: strides %lld, %lld of rows of %d", who, (long long)a->stride_x, (long long)a->stride_g, a->D);
  REQUIRE(a->x, who); REQUIRE(a->g, who);
  if (!bwd) { REQUIRE(a->h, who); }
  else { REQUIRE(a->states, who); REQUIRE(a->dx, who); }
  const uintptr_t size = a->dtype == 2 ? 4 : 2, gate = a->gate_dtype == 2 ? 4 : 2;
  if (off_boundary(size, {a->x, a->h, a->dh, a->dx}) || off_boundary(gate, {a->g, a->dg}) ||
      off_boundary(4, {a->h0, a->ht, a->states, a->dht, a->dh0, a->seq_meta, a->seq_order}) || off_boundary(16, {a->chunk_meta}))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a tensor off its elements' boundary", who);
  return 0;
}

int b200gdn_gated_recurrence_fwd(const b200gdn_gated_recurrence_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_gated_recurrence_args(a, "gated_recurrence_fwd", false)) return e;
  return gdn::launch_gated_recurrence(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_gated_recurrence_bwd(const b200gdn_gated_recurrence_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_gated_recurrence_args(a, "gated_recurrence_bwd", true)) return e;
  return gdn::launch_gated_recurrence(*a, static_cast<cudaStream_t>(stream), true);
}

static int check_rms_norms_args(const b200gdn_rms_norms_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_rms_norms_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes, sizeof(b200gdn_rms_norms_args));
  if (a->rows <= 0 || a->D <= 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%lld D=%d)", who, (long long)a->rows, a->D);
  if (a->rows > (1 << 30)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^30 rows", who);
  if (a->D > (1 << 23)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: D=%d (at most 2^23)", who, a->D);
  if (a->dtype < 0 || a->dtype > 2 || a->param_dtype < 0 || a->param_dtype > 2)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype codes %d, %d", who, a->dtype, a->param_dtype);
  const uint32_t both = B200GDN_NORMS_SIGMOID | B200GDN_NORMS_SILU;
  if ((a->flags & both) == both || (a->flags & ~(both | B200GDN_NORMS_POST)) != 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: flags %u", who, a->flags);
  if (a->post_weight != nullptr && !(a->flags & B200GDN_NORMS_POST))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: post_weight without B200GDN_NORMS_POST", who);
  REQUIRE(a->y, who);
  if ((a->rstd_y == nullptr) != (a->rstd_z == nullptr)) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: rstd_y and rstd_z come together", who);
  if (!bwd) { REQUIRE(a->out, who); }
  else {
    REQUIRE(a->rstd_z, who);
    if (a->dweight != nullptr || a->dpost_weight != nullptr || a->dscale != nullptr) REQUIRE(a->partials, who);
    if (a->dgate != nullptr && a->gate == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dgate without a gate", who);
  }
  const uintptr_t size = a->dtype == 2 ? 4 : 2, param_size = a->param_dtype == B200GDN_F32 ? 4 : 2;
  if (off_boundary(size, {a->y, a->residual, a->gate, a->z, a->out, a->dout, a->dz, a->dy, a->dresidual, a->dgate}) ||
      off_boundary(param_size, {a->weight, a->post_weight, a->scale, a->dweight, a->dpost_weight, a->dscale}) ||
      off_boundary(4, {a->rstd_y, a->rstd_z, a->partials}))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a tensor off its elements' boundary", who);
  return 0;
}

int b200gdn_rms_norms_fwd(const b200gdn_rms_norms_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_rms_norms_args(a, "rms_norms_fwd", false)) return e;
  return gdn::launch_rms_norms(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_rms_norms_bwd(const b200gdn_rms_norms_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_rms_norms_args(a, "rms_norms_bwd", true)) return e;
  return gdn::launch_rms_norms(*a, static_cast<cudaStream_t>(stream), true);
}

int64_t b200gdn_rms_norms_partials(int64_t rows, int32_t D) { return gdn::rms_norms_partials(rows, D); }

static int check_linear_args(const b200gdn_linear_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_linear_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes, sizeof(b200gdn_linear_args));
  if (a->rows <= 0 || a->K <= 0 || a->N <= 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%lld K=%d N=%d)", who, (long long)a->rows, a->K, a->N);
  if (a->rows > (1 << 30)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^30 rows", who);
  if (a->K > (1 << 23) || a->N > (1 << 23)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: K=%d, N=%d (at most 2^23)", who, a->K, a->N);
  if (a->dtype < 0 || a->dtype > 1) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype code %d (0 or 1)", who, a->dtype);
  if (a->activation < 0 || a->activation > B200GDN_LINEAR_GELU) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: activation %d", who, a->activation);
  if (!bwd) { REQUIRE(a->x, who); REQUIRE(a->weight, who); REQUIRE(a->y, who); }
  else {
    REQUIRE(a->dy, who);
    if (a->dx != nullptr) REQUIRE(a->weight, who);
    if (a->dweight != nullptr) REQUIRE(a->x, who);
    if (a->activation != 0) REQUIRE(a->z, who);
  }
  if (off_boundary(2, {a->x, a->weight, a->bias, a->residual, a->y, a->z, a->dy, a->dx, a->dweight, a->dbias}))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a tensor off its elements' boundary", who);
  const int64_t need = linear_workspace(*a, bwd);
  if (need > 0) {
    REQUIRE(a->workspace, who);
    if (a->workspace_bytes < need)
      return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a workspace of %lld bytes where %lld are needed", who, (long long)a->workspace_bytes, (long long)need);
    if (off_boundary(256, {a->workspace})) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: workspace off its boundary of 256", who);
  }
  return 0;
}

int b200gdn_linear_fwd(const b200gdn_linear_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_linear_args(a, "linear_fwd", false)) return e;
  return gdn::launch_linear(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_linear_bwd(const b200gdn_linear_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_linear_args(a, "linear_bwd", true)) return e;
  return gdn::launch_linear(*a, static_cast<cudaStream_t>(stream), true);
}

int64_t b200gdn_linear_workspace_bytes(const b200gdn_linear_args* a, int32_t backward) {
  if (a == nullptr || a->rows <= 0 || a->K <= 0 || a->N <= 0) return 0;
  return gdn::linear_workspace(*a, backward != 0);
}

// what the two operators on rows of logits have in common
static int check_rows_of_logits(const char* who, int64_t rows, int64_t inner, int32_t V, int32_t dtype, float scale, const void* logits,
                                const void* dlogits) {
  using namespace gdn;
  if (rows <= 0 || V <= 0 || inner <= 0)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: empty problem (rows=%lld V=%d inner=%lld)", who, (long long)rows, V, (long long)inner);
  if (rows > (1 << 27)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^27 rows", who);
  if (V > (1 << 30)) return set_error(B200GDN_ERR_UNSUPPORTED, "%s: more than 2^30 entries a row", who);
  if (dtype < 0 || dtype > 2) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: dtype code %d", who, dtype);
  if (!(scale > 0.f) || !(scale <= 1e6f)) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: scale %g (above 0, at most 1e6)", who, scale);
  REQUIRE(logits, who);
  const uintptr_t off = (reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dlogits)) % (dtype == 2 ? 4 : 2);
  if (off != 0) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: logits or dlogits off their elements' boundary", who);
  return 0;
}

static int check_logprob_args(const b200gdn_logprob_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_logprob_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes, sizeof(b200gdn_logprob_args));
  if (int e = check_rows_of_logits(who, a->rows, a->inner, a->V, a->dtype, a->scale, a->logits, a->dlogits)) return e;
  if (a->top_k < 0 || a->top_k > B200GDN_MAX_TOP || a->top_k > a->V)
    return set_error(B200GDN_ERR_UNSUPPORTED, "%s: top_k=%d (0 to %d, at most V=%d)", who, a->top_k, B200GDN_MAX_TOP, a->V);
  if (a->tokens != nullptr && a->token_bytes != 4 && a->token_bytes != 8)
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: token_bytes %d (4 or 8)", who, a->token_bytes);
  if (!bwd) {
    if (a->logprobs != nullptr) REQUIRE(a->tokens, who);
    if (a->top_k > 0) { REQUIRE(a->top_ids, who); REQUIRE(a->top_logprobs, who); }
    REQUIRE(a->workspace, who);
  } else {
    REQUIRE(a->stats, who); REQUIRE(a->dlogits, who);
    if (a->dlogprobs != nullptr) REQUIRE(a->tokens, who);
    if (a->dentropy != nullptr) REQUIRE(a->entropy, who);
    if (a->dtop_logprobs != nullptr) REQUIRE(a->top_ids, who);
  }
  if (off_boundary(4, {a->logprobs, a->entropy, a->top_logprobs, a->stats, a->dlogprobs, a->dentropy, a->dtop_logprobs}) || off_boundary(8, {a->top_ids}) ||
      (a->tokens != nullptr && off_boundary(a->token_bytes, {a->tokens})))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a tensor off its elements' boundary", who);
  if (!bwd && off_boundary(16, {a->workspace})) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: workspace off a 16-byte boundary", who);
  return 0;
}

int b200gdn_logprob_fwd(const b200gdn_logprob_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_logprob_args(a, "logprob_fwd", false)) return e;
  return gdn::launch_logprob(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_logprob_bwd(const b200gdn_logprob_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_logprob_args(a, "logprob_bwd", true)) return e;
  return gdn::launch_logprob(*a, static_cast<cudaStream_t>(stream), true);
}

int64_t b200gdn_logprob_workspace_bytes(int64_t rows, int32_t V, int32_t dtype, int32_t top_k) { return gdn::logprob_workspace(rows, V, dtype, top_k); }

static int check_distill_args(const b200gdn_distill_args* a, const char* who, bool bwd) {
  using namespace gdn;
  if (a == nullptr) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: args is NULL", who);
  if (a->struct_bytes != (int32_t)sizeof(b200gdn_distill_args))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: struct_bytes %d != %zu (ABI mismatch)", who, a->struct_bytes, sizeof(b200gdn_distill_args));
  if (int e = check_rows_of_logits(who, a->rows, a->inner, a->V, a->dtype, a->scale, a->logits, a->dlogits)) return e;
  if (a->K < 1 || a->K > B200GDN_MAX_LIST)
    return set_error(B200GDN_ERR_UNSUPPORTED, "%s: K=%d (1 to %d entries a row)", who, a->K, B200GDN_MAX_LIST);
  if (a->id_bytes != 4 && a->id_bytes != 8) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: id_bytes %d (4 or 8)", who, a->id_bytes);
  if (a->teacher_dtype < 0 || a->teacher_dtype > 2) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: teacher_dtype %d", who, a->teacher_dtype);
  REQUIRE(a->teacher, who); REQUIRE(a->ids, who);
  if (!bwd) { REQUIRE(a->row_loss, who); }
  else { REQUIRE(a->dloss, who); REQUIRE(a->dlogits, who); }
  if ((a->flags & B200GDN_DISTILL_SKIP_ONE) && !(bwd && (a->flags & B200GDN_DISTILL_SCALAR)))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: SKIP_ONE goes with a scalar upstream gradient", who);
  REQUIRE(a->workspace, who);
  if (off_boundary(4, {a->row_loss, a->loss, a->dloss}) || off_boundary(a->id_bytes, {a->ids}) ||
      off_boundary(a->teacher_dtype == B200GDN_F32 ? 4 : 2, {a->teacher}))
    return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: a tensor off its elements' boundary", who);
  if (off_boundary(16, {a->workspace})) return set_error(B200GDN_ERR_BAD_ARGUMENT, "%s: workspace off a 16-byte boundary", who);
  return 0;
}

int64_t b200gdn_distill_workspace_bytes(int64_t rows, int32_t V, int32_t dtype, int32_t K) { return gdn::distill_workspace(rows, V, dtype, K); }

int b200gdn_distill_fwd(const b200gdn_distill_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_distill_args(a, "distill_fwd", false)) return e;
  return gdn::launch_distill(*a, static_cast<cudaStream_t>(stream), false);
}

int b200gdn_distill_bwd(const b200gdn_distill_args* a, void* stream) {
  gdn::g_launches = 0;
  if (int e = check_distill_args(a, "distill_bwd", true)) return e;
  return gdn::launch_distill(*a, static_cast<cudaStream_t>(stream), true);
}

int b200gdn_selftest_wait_expiry(void* stream) {
  gdn::g_launches = 0;
  gdn::selftest_wait_expiry_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(2000u);
  return gdn::check_launch("selftest_wait_expiry");
}

int b200gdn_device_status(void) {
  struct { const char* name; int (*flag)(); } k[] = {
      {"intra_fwd", gdn::intra_fwd_timeout_flag}, {"scan_fwd", gdn::scan_fwd_timeout_flag}, {"out_fwd", gdn::out_fwd_timeout_flag},
      {"dv_local", gdn::dv_local_timeout_flag},   {"scan_bwd", gdn::scan_bwd_timeout_flag}, {"bwd_dqk", gdn::bwd_dqk_timeout_flag},
      {"bwd_wy", gdn::bwd_wy_timeout_flag},       {"bwd_local", gdn::bwd_local_timeout_flag},
            {"selftest", gdn::selftest_timeout_flag},
      {"linear", gdn::linear_timeout_flag},     {"gated_recurrence", gdn::recurrence_timeout_flag}, {"rms_norms", gdn::norms_timeout_flag},
      {"decode_stream", gdn::decode_timeout_flag}};
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return gdn::set_error(B200GDN_ERR_CUDA, "device_status: %s", cudaGetErrorString(e));
  int rc = B200GDN_OK;
  for (auto& x : k)
    if (x.flag()) rc = gdn::set_error(B200GDN_ERR_TIMEOUT, "%s: a bounded device wait expired; its results are invalid", x.name);
  return rc;
}

int b200gdn_last_launch_count(void) { return gdn::g_launches; }
int b200gdn_abi_version(void) { return B200GDN_ABI_VERSION; }
const char* b200gdn_last_error(void) { return gdn::g_err; }

}  // extern "C"

// gemm_conv.hip — the MFMA workhorse of the denoising path: one LDS-tiled kernel that is
// either a dense GEMM  out[M,N] = A[M,K].W[N,K]^T  or a channels-last implicit-GEMM
// convolution (3x3 / 1x1, stride 1|2, optional nearest-upsample gather, optional extra 1x1
// tap over a second tensor = fused ResBlock shortcut), with a fused epilogue
// (bias, per-batch bias = time embedding / collapsed cross-attention, SiLU, GEGLU,
// residual add, fp32|half store).
//
// Reference ops replaced: see include/mimo_hip.h (mimo_gemm / mimo_conv2d).
//
// Tiling (gfx950): block = WM x WN waves; block tile (16*MT*WM) x (16*NR*WN) x 64; each wave owns
// (16*MT) x (16*NR) as MT x NR MFMA 16x16x32 tiles, fp32 accumulators in VGPRs.
// Operands go global -> LDS by DMA (`buffer_load_dwordx4 ... lds`): hardware range checking
// turns padding taps / ragged edges into zero fill, the XOR swizzle that makes the
// ds_read_b128 fragment reads bank-conflict-free is applied on the SOURCE address (the DMA
// writes lane-linear), and an NSTAGE-deep LDS ring keeps NSTAGE-1 K-tiles in flight under
// the MFMAs with ONE barrier and one counted `s_waitcnt vmcnt` per K-tile.  Configurations
// (picked per shape in launch_nr): S 2x2 waves, 128-row tile, 2 blocks/CU; L 4x2, 3-deep ring;
// XL 4x4 = 16 waves 256 x 256 (GEGLU); XL8 2x4 = 8 waves with a 256-register budget,
// (256|192|128) x 320; split-K over gridDim.y for long reductions over few tiles;
// gemm_dense_persist_kernel = the dense case as persistent blocks with cross-tile prefetch.
// The MFMA is issued "swapped" (W fragment as the A operand) so that every lane ends up
// with 4 consecutive output columns of one row -> 16-byte epilogue loads/stores.
#include <stdlib.h>

#include "gemm_core.hip.h"
#include "gemm_stream.hip.h"
#include "thinconv.hip.h"

namespace {

// Tuning knobs.  In the shipped build they are compile-time constants (tune_env folds to its default: the library
// reads no environment and keeps no mutable state).  Only the -DMIMO_TUNE build (libmimo_hip_tune.so, used by
// tools/microbench.py for interleaved A/B timing) reads them from the environment, at every launch:
//   MIMO_GEMM_CFG=1|2|3|4   force tile configuration S|L|XL|XL8
//   MIMO_GEMM_STAGGER=0     all waves issue their DMAs right after the barrier (default 1: staggered)
//   MIMO_CONV_TAP_INNER=0   convolution K order tap-outer / channel-chunk-inner (default 1: tap inner)
//   MIMO_GEMM_BM=256|192|128  force the XL8 tile height (default: picked per shape by wave quantisation)
//   MIMO_GEMM_PERSIST=0     dense GEMMs launch one block per output tile (default 1: persistent blocks, cross-tile prefetch)
//   MIMO_GEMM_SPLITK=0      never split K (default 1; per call: MIMO_EPI_NO_SPLITK)
//   MIMO_GEMM_ABLATE=1|2|3  timing experiments: skip DMA | skip MFMA | skip GELU (results are wrong)
struct Tuning {
  int cfg, ablate, stagger, tap_inner, splitk, bm, persist;
};
inline Tuning tuning() {
  return Tuning{tune_env("MIMO_GEMM_CFG", 0), tune_env("MIMO_GEMM_ABLATE", 0), tune_env("MIMO_GEMM_STAGGER", 1),
                tune_env("MIMO_CONV_TAP_INNER", 1), tune_env("MIMO_GEMM_SPLITK", 1), tune_env("MIMO_GEMM_BM", 0),
                tune_env("MIMO_GEMM_PERSIST", 1)};
}

// CU count of the current device: an immutable fact of the hardware, cached after the first query
inline int cus_() {
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    return n;
  }();
  return cus;
}

#ifdef MIMO_TUNE
inline unsigned long long* trace_buf() {
  static unsigned long long* buf = [] {
    void* p = nullptr;
    if (hipMalloc(&p, 4096 * sizeof(unsigned long long)) != hipSuccess) return (unsigned long long*)nullptr;
    (void)hipMemset(p, 0, 4096 * sizeof(unsigned long long));
    return (unsigned long long*)p;
  }();
  return buf;
}
extern "C" unsigned long long* mimo_tune_trace_buf() { return trace_buf(); }   // (for the other translation units)
// copies the trace of the most recent traced launch to `dst` (n entries <= 4096) and clears the device buffer
extern "C" int mimo_tune_trace(unsigned long long* dst, int n) {
  if (!trace_buf() || n > 4096) return MIMO_EINVAL;
  hipError_t e = hipDeviceSynchronize();
  if (e == hipSuccess) e = hipMemcpy(dst, trace_buf(), (size_t)n * 8, hipMemcpyDeviceToHost);
  if (e == hipSuccess) e = hipMemset(trace_buf(), 0, 4096 * 8);
  return (int)e;
}
#endif

// one-block-per-tile launch of gemm_kernel; dense launches that carry a folded LayerNorm half take the EPI = 2 instantiation
#define MIMO_LAUNCH_GK(WM_, WN_, NS_, MT_, nwg_, thr_)                                                                    \
  do {                                                                                                                    \
    if constexpr (MODE == 0) {                                                                                            \
      if (folded) {                                                                                                       \
        hipLaunchKernelGGL((gemm_kernel<DT, NR, MODE, WM_, WN_, NS_, MT_, 2>), dim3((unsigned)(nwg_)), dim3(thr_), 0, st, g); \
        break;                                                                                                            \
      }                                                                                                                   \
    }                                                                                                                     \
    hipLaunchKernelGGL((gemm_kernel<DT, NR, MODE, WM_, WN_, NS_, MT_>), dim3((unsigned)(nwg_)), dim3(thr_), 0, st, g);      \
  } while (0)

constexpr int GEMM_BM64_DEFAULT = 1;   // (tune build: MIMO_GEMM_BM64)

template <int DT, int MODE, int NR>
int launch_nr(GemmArgs& g, hipStream_t st) {
#ifdef MIMO_TUNE
  g.dbg = tune_env("MIMO_GEMM_TRACE", 0) ? trace_buf() : nullptr;
#endif
  // Tile configurations (WM x WN waves, ring depth):
  //   S  2x2, 2 stages: 128 x 32NR tile, 2 blocks/CU          — small / skinny problems
  //   L  4x2, 3 stages: 256 x 32NR tile, 1 block/CU
  //   XL 4x4, 2 stages: 256 x 64NR tile (N = 320 in ONE tile), 16 waves, 1 block/CU — halves the global->LDS
  //      bytes per MAC; the L2->LDS path (~18 TB/s measured) and not the MFMAs bounds the S tile
  //   XL8 2x4, 2 stages: the XL tile on 8 waves of 128 x 16NR (256-register budget) — every NR = 5 XL problem
  const Tuning tn = tuning();
  const int forced = tn.cfg, ablate = tn.ablate;
  if (ablate == 1) g.flags |= F_ABL_NO_DMA;
  if (ablate == 2) g.flags |= F_ABL_NO_MFMA;
  if (ablate == 3) g.flags |= F_ABL_NO_GELU;
  const int64_t m256 = (g.M + 255) / 256;
  const int tn_s = (g.N + 32 * NR - 1) / (32 * NR), tn_xl = (g.N + 64 * NR - 1) / (64 * NR);
  const bool geglu = g.flags & MIMO_EPI_GEGLU;
  int cfg = forced;
  if (cfg == 0) {
    if (g.N <= 32 * NR) cfg = (m256 * tn_s >= 160) ? 2 : 1;  // one S-width tile covers N: a 64NR-wide XL tile would idle
    else cfg = (m256 * tn_xl >= 160) ? 3 : 1;                 // measured crossover (tools/microbench.py)
  }
  if (tn.stagger) g.flags |= F_STAGGER;
  if (tn.tap_inner && MODE != 0) g.flags |= F_TAP_INNER;
  if (cfg == 3 && NR == 5) cfg = 4;  // 16 waves x 128 registers cannot hold a 64 x 80 accumulator tile plus the epilogue
  if (cfg == 3 && g.colstats) cfg = 4;  // the 16-wave tile has no statistics epilogue
  const bool folded = g.row_half || g.a_row_stats;   // (plain one-block-per-tile launches only)
  if (cfg == 3 && g.row_half) cfg = 4;  // the 16-wave tile has no row-statistics epilogue either
  if (cfg == 2 && folded) cfg = 1;      // the 3-stage ring of the L tile leaves no LDS for the (mean, rstd, colsum) region
  const bool allow_splitk = tn.splitk && !(g.flags & MIMO_EPI_NO_SPLITK) && !g.colstats && !g.ln_out && !folded;
  // fused LayerNorm output: the tile must hold whole rows (N == 320 = the NR = 5 XL8 width), dense only
  if (g.ln_out) {
    if constexpr (MODE == 0 && NR == 5) {
      if (g.N == 640 && !geglu && !g.colstats && (g.K % 32) == 0 && g.M < 0x7fffffffLL * 64) {   // whole rows at N = 640: 64-row tiles
        hipLaunchKernelGGL((gemm_ln640_kernel<DT>), dim3((unsigned)((g.M + 63) / 64)), dim3(512), 0, st, g);
        MIMO_LAUNCH_CHECK();
        return MIMO_OK;
      }
      if (g.N != 64 * NR || geglu || g.colstats) return MIMO_EINVAL;
      g.tiles_n = 1;
      const int64_t nwg = (g.M + 127) / 128;
      if (nwg <= 0 || nwg > 0x7fffffff) return MIMO_EINVAL;
      g.ntiles = (unsigned)nwg;
      hipLaunchKernelGGL((gemm_dense_persist_kernel<DT, NR, 2, 4, 4, 1>), dim3((unsigned)(nwg < cus_() ? nwg : cus_())), dim3(512), 0, st, g);
      MIMO_LAUNCH_CHECK();
      return MIMO_OK;
    } else {
      return MIMO_EINVAL;
    }
  }
  // Split-K: a long reduction over few output tiles (the 8x8-level convolutions: M = 3072, K = 11520) leaves most of
  // the chip idle.  Use XL8 tiles, split K over gridDim.y, and let a second tiny launch reduce the fp32 partials
  // (fixed order) and apply the epilogue.  Needs the caller's workspace.
  const int cus = cus_();
  if (forced == 0 && allow_splitk && !geglu && g.ws && NR == 5) {
    const int64_t nt = m256 * tn_xl;
    int64_t sk = nt > 0 ? cus / nt : 0;
    if (sk > g.nkt / 16) sk = g.nkt / 16;
    if (sk > 8) sk = 8;
    const size_t need = (size_t)sk * (size_t)g.M * (size_t)g.N * sizeof(float);
    if (sk >= 2 && nt * 2 <= cus && need <= g.ws_bytes) {
      GemmArgs gp = g;
      gp.tiles_n = tn_xl;
      gp.out = g.ws; gp.ldo = g.N; gp.bias = nullptr; gp.img_bias = nullptr; gp.res = nullptr; gp.out_scale = 1.f;
      gp.flags = (g.flags & 0xffff0000u) | MIMO_EPI_OUT_F32;
      hipLaunchKernelGGL((gemm_kernel<DT, NR, MODE, 2, 4, 2, 8>), dim3((unsigned)nt, (unsigned)sk), dim3(512), 0, st, gp);
      MIMO_LAUNCH_CHECK();
      int64_t rb = (g.M * (g.N >> 2) + 255) / 256;
      if (rb > 4096) rb = 4096;
      hipLaunchKernelGGL(splitk_reduce_kernel<DT>, dim3((unsigned)rb), dim3(256), 0, st, g, (int)sk);
      MIMO_LAUNCH_CHECK();
      return MIMO_OK;
    }
  }
  if (cfg == 4) {  // XL8: the XL tile on 8 waves (2 x 4), each wave (16 MT) x 16NR with a 256-register budget
    // Tile height 256 | 192 | 128 rows (MT = 8 | 6 | 4): with one block per CU the launch runs in rounds of `cus`
    // tiles, so pick the height that minimises rounds x (rows + per-tile overhead) — e.g. M = 12288, N = 1280 is
    // 192 tiles of 256 rows (75 % of the chip for one round) but exactly 256 tiles of 192 rows.
    g.tiles_n = tn_xl;
    auto cost = [&](int bm) {
      const int64_t nt = ((g.M + bm - 1) / bm) * tn_xl;
      return ((nt + cus - 1) / cus) * (int64_t)(bm + 24);
    };
    int bm = tn.bm;
    if (bm != 256 && bm != 192 && bm != 128) {
      bm = 256;
      if (cost(192) < cost(bm)) bm = 192;
      if (cost(128) < cost(bm)) bm = 128;
    }
    const int64_t nwg = ((g.M + bm - 1) / bm) * tn_xl;
    if (nwg <= 0 || nwg > 0x7fffffff) return MIMO_EINVAL;
    // persistent blocks pay off (measured +2..7 %) for short reductions over many rounds of tiles — the level-0 linears;
    // with 2-3 exactly filled rounds or long K the plain launch is faster (tools/microbench.py --ab MIMO_GEMM_PERSIST=0)
    if (MODE == 0 && tn.persist && !g.colstats && !folded && bm == 256 && nwg >= 3 * (int64_t)cus && g.nkt >= 2 && g.nkt <= 20) {
      g.ntiles = (unsigned)nwg;
      hipLaunchKernelGGL((gemm_dense_persist_kernel<DT, NR, 2, 4, 8>), dim3((unsigned)cus), dim3(512), 0, st, g);
      MIMO_LAUNCH_CHECK();
      return MIMO_OK;
    }
    if (bm == 256) MIMO_LAUNCH_GK(2, 4, 2, 8, nwg, 512);
    else if (bm == 192) MIMO_LAUNCH_GK(2, 4, 2, 6, nwg, 512);
    else MIMO_LAUNCH_GK(2, 4, 2, 4, nwg, 512);
  } else if (cfg == 3) {
    g.tiles_n = tn_xl;
    const int64_t nwg = m256 * tn_xl;
    if (nwg <= 0 || nwg > 0x7fffffff) return MIMO_EINVAL;
    if constexpr (NR == 4) {
      if (MODE == 0 && tn.persist && !folded && nwg >= 3 * (int64_t)cus && g.nkt >= 2) {  // GEGLU: +6 % at every level
        g.ntiles = (unsigned)nwg;
        hipLaunchKernelGGL((gemm_dense_persist_kernel<DT, NR, 4, 4, 4>), dim3((unsigned)cus), dim3(1024), 0, st, g);
      } else {
        MIMO_LAUNCH_GK(4, 4, 2, 4, nwg, 1024);
      }
    }
  } else if (cfg == 2) {
    g.tiles_n = tn_s;
    const int64_t nwg = m256 * tn_s;
    if (nwg <= 0 || nwg > 0x7fffffff) return MIMO_EINVAL;
    hipLaunchKernelGGL((gemm_kernel<DT, NR, MODE, 4, 2, 3, 4>), dim3((unsigned)nwg), dim3(512), 0, st, g);
  } else {
    g.tiles_n = tn_s;
    const int64_t nwg = ((g.M + 127) / 128) * tn_s;
    if (nwg <= 0 || nwg > 0x7fffffff) return MIMO_EINVAL;
    // Small-M dense launches (the 8 x 8 level: M = 3072, N = 1280 -> 192 blocks of 128 x 160, one per CU on three quarters of
    // the chip, each a serial chain of K / 64 round trips): 64-row tiles double the blocks (two per CU: 57 KB of LDS each), i.e.
    // the bytes in flight per CU, which is what a latency-bound launch is short of.  A function of (M, N) only; the K order of
    // every output element is unchanged, so the result is bit-identical to the 128-row tile's.
    if constexpr (MODE == 0) {
      if (tune_env("MIMO_GEMM_BM64", GEMM_BM64_DEFAULT) && nwg <= cus && !geglu) {
        const int64_t nwg64 = ((g.M + 63) / 64) * tn_s;
        MIMO_LAUNCH_GK(2, 2, 2, 2, nwg64, 256);
        MIMO_LAUNCH_CHECK();
        return MIMO_OK;
      }
    }
    MIMO_LAUNCH_GK(2, 2, 2, 4, nwg, 256);
  }
  (void)geglu;
  MIMO_LAUNCH_CHECK();
  return MIMO_OK;
}

// MIMO_GEMM_8P (tune build; the shipped default is the constant below): 1 = dense GEMMs with an even number of K-tiles
// and enough 256 x 256 tiles take the 8-phase kernel
constexpr int GEMM_8P_DEFAULT = 1;

// Column-slot width of mimo_epilogue_ext.row_stats = the 16 NR columns one wave owns in the kernel family a producer of
// width N runs on — chosen from N alone (never from M), so a row's partial sums do not depend on the batch:
// 64 (gemm8_kernel, or the NR = 4 tiles when the row count is too small for it) where 256-wide tiles fit N, else 80 (NR = 5).
int row_slot_width(int N) {
  const int tn8 = (N + 255) / 256;
  if (tn8 * 256 - N <= N / 12 && N % 64 == 0) return 64;
  if (N % 160 == 0) return 80;
  return N % 64 == 0 ? 64 : 0;
}

// Slots per row of a folded LayerNorm of width N, or 0 where the fold does not apply: the producer's row-side epilogue has no
// column mask, so N must be a whole number of the WIDEST tile its kernel family uses (4 slots: 256 columns for the 64-wide
// slots, 320 for the 80-wide ones — 480 / 800 / 960 / 1920 would let a wave past column N write into the next row); the
// consumer holds at most 2 * ROW_STAT_LOADS slots (N = 2560 has 40).
int row_stat_slots_of(int N) {
  const int w = N > 0 ? row_slot_width(N) : 0;
  if (!w || N % (4 * w) != 0) return 0;
  const int slots = N / w;
  return (slots & 1) == 0 && slots <= 2 * ROW_STAT_LOADS ? slots : 0;
}

template <int DT, int MODE>
int launch(const GemmArgs& g0, hipStream_t st) {
  GemmArgs g = g0;
  const bool geglu = g.flags & MIMO_EPI_GEGLU;
  if constexpr (MODE == 0) {
    const int p8 = tune_env("MIMO_GEMM_8P", GEMM_8P_DEFAULT);
    const int64_t tn8 = (g.N + 255) / 256, nt8 = ((g.M + 255) / 256) * tn8;
    // (N = 640 is 2.5 tiles of 256: a sixth of the columns would be padding — those shapes keep the 320-wide tiles)
    const bool n_fits = tn8 * 256 - g.N <= g.N / 12;
    if (p8 && !g.colstats && !g.ln_out && (g.K % 128) == 0 && n_fits && nt8 >= 128 && nt8 <= 0x7fffffff && g.M < 0x7fffffff) {
      g.tiles_n = (int)tn8;
      g.ntiles = (unsigned)tune_env("MIMO_G8_GM", G8_GM);
      if (g.row_half || g.a_row_stats) hipLaunchKernelGGL((gemm8_kernel<DT, 2>), dim3((unsigned)nt8), dim3(512), 0, st, g);
      else hipLaunchKernelGGL((gemm8_kernel<DT>), dim3((unsigned)nt8), dim3(512), 0, st, g);
      MIMO_LAUNCH_CHECK();
      return MIMO_OK;
    }
  }
  if (g.row_half) return row_slot_width(g.N) == 80 ? launch_nr<DT, MODE, 5>(g, st) : launch_nr<DT, MODE, 4>(g, st);
  // NR = 5 (BN = 160) divides every SD1.5 width (320/640/960/1280/1920/2560); NR = 4 otherwise
  if (!geglu && (g.N % 160 == 0)) return launch_nr<DT, MODE, 5>(g, st);
  return launch_nr<DT, MODE, 4>(g, st);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

static int check_ext(const mimo_epilogue_ext* e, GemmArgs& g, int64_t M, int N, int K, unsigned flags) {
  g.colstats = nullptr; g.ln_gamma = g.ln_beta = g.ln_pe = nullptr; g.ln_out = nullptr;
  g.ln_eps = 0.f; g.ln_rows_per_frame = 1; g.ln_pe_frames = 1;
  g.row_half = nullptr; g.row_stats = nullptr; g.a_row_stats = nullptr; g.a_colsum = nullptr; g.a_slots = 0; g.a_eps = 0.f;
  if (!e) return MIMO_OK;
  if (e->row_half || e->row_stats) {   // producer half of a folded LayerNorm: fp32 result + half copy + row statistics
    if (!e->row_half || !e->row_stats || e->colstats || e->ln_out || !(flags & MIMO_EPI_OUT_F32) ||
        (flags & (MIMO_EPI_SILU | MIMO_EPI_GEGLU)) || row_stat_slots_of(N) == 0 || M >= 0x7fffffffLL / ((int64_t)N * 2) ||
        !aligned16(e->row_half) || !aligned16(e->row_stats))
      return MIMO_EINVAL;
    g.row_half = e->row_half; g.row_stats = e->row_stats;
  }
  if (e->a_row_stats || e->a_colsum) {  // consumer half
    // (a_slots must be the producer's slot count for THIS K: statistics of another width would be read misaligned)
    if (!e->a_row_stats || !e->a_colsum || e->a_slots <= 0 || e->a_slots != row_stat_slots_of(K) || e->colstats || e->ln_out ||
        M >= 0x7fffffffLL / ((int64_t)e->a_slots * 8) || !aligned16(e->a_row_stats) || !aligned16(e->a_colsum))
      return MIMO_EINVAL;
    g.a_row_stats = e->a_row_stats; g.a_colsum = e->a_colsum; g.a_slots = e->a_slots; g.a_eps = e->a_eps;
  }
  if (e->colstats) {
    if ((M & 31) || (N & 3) || (flags & MIMO_EPI_GEGLU) || !aligned16(e->colstats)) return MIMO_EINVAL;
    g.colstats = e->colstats;
  }
  if (e->ln_out) {
    if (!e->ln_gamma || !e->ln_beta || e->colstats || !aligned16(e->ln_out)) return MIMO_EINVAL;
    if (e->ln_pe && (e->ln_rows_per_frame <= 0 || e->ln_pe_frames <= 0 || (e->ln_rows_per_frame % 128))) return MIMO_EINVAL;
    g.ln_gamma = e->ln_gamma; g.ln_beta = e->ln_beta; g.ln_pe = e->ln_pe; g.ln_out = e->ln_out;
    g.ln_eps = e->ln_eps;
    g.ln_rows_per_frame = e->ln_pe ? e->ln_rows_per_frame : 1;
    g.ln_pe_frames = e->ln_pe ? e->ln_pe_frames : 1;
  }
  return MIMO_OK;
}

extern "C" int mimo_gemm_ext(int dtype, const void* A, int64_t lda, const void* W, void* out, int64_t ldo,
                             int64_t M, int N, int K, const float* bias, const float* img_bias,
                             int64_t img_bias_ld, int64_t rows_per_img, const void* residual, int64_t ldr,
                             float out_scale, unsigned flags, void* workspace, size_t workspace_bytes,
                             const mimo_epilogue_ext* ext, void* stream) {
  if (!A || !W || !out || M <= 0 || N <= 0 || K <= 0) return MIMO_EINVAL;
  if ((K & 7) || (lda & 7) || (N & 3) || (ldo & 3) || !aligned16(A) || !aligned16(W) || !aligned16(out))
    return MIMO_EINVAL;
  if ((flags & MIMO_EPI_GEGLU) && (N & 31)) return MIMO_EINVAL;
  if (flags & ~(MIMO_EPI_SILU | MIMO_EPI_GEGLU | MIMO_EPI_OUT_F32 | MIMO_EPI_RES_F32 | MIMO_EPI_NO_SPLITK)) return MIMO_EINVAL;
  if (residual && (ldr & 3)) return MIMO_EINVAL;
  if (img_bias && (rows_per_img <= 0 || (img_bias_ld & 3))) return MIMO_EINVAL;
  GemmArgs g{};
  g.A = (const uint16_t*)A; g.A2 = nullptr; g.W = (const uint16_t*)W; g.out = out;
  g.bias = bias; g.img_bias = img_bias; g.res = residual;
  g.lda = lda; g.ldw = K; g.ldo = ldo; g.ldr = ldr; g.M = M; g.rows_per_img = rows_per_img > 0 ? rows_per_img : 1;
  g.ldib = img_bias_ld > 0 ? img_bias_ld : N;
  g.N = N; g.K = K; g.out_scale = out_scale; g.flags = flags;
  g.ws = aligned16(workspace) ? workspace : nullptr; g.ws_bytes = workspace_bytes;
  g.nkt = (K + BK - 1) / BK;
  if (int rc = check_ext(ext, g, M, N, K, flags)) return rc;
  if (g.ln_out && ((flags & (MIMO_EPI_SILU | MIMO_EPI_GEGLU)) || ldo != N || (residual && ldr != N))) return MIMO_EINVAL;
  const int64_t ab = ((M - 1) * lda + K) * 2, wb = (int64_t)N * K * 2;
  if (ab >= 0x80000000LL || wb >= 0x80000000LL) return MIMO_EINVAL;  // 32-bit offsets; 2 GiB keeps OOBA + soffset out of range
  g.a_bytes = (unsigned)ab; g.a2_bytes = 0; g.w_bytes = (unsigned)wb;
  hipStream_t st = (hipStream_t)stream;
  // level-0 token linears (K = 320, plain half output or GEGLU): A in registers, W streamed (gemm_stream.hip)
#ifndef MIMO_NO_STREAM
#define MIMO_NO_STREAM 0
#endif
  if (!MIMO_NO_STREAM && tune_env("MIMO_GEMM_STREAM", 1) && mimo_stream::supported(M, N, K, (flags & MIMO_EPI_NO_SPLITK) != 0) && !residual && !img_bias && !g.colstats && !g.ln_out && !g.row_half && !g.a_row_stats &&
      !(flags & (MIMO_EPI_SILU | MIMO_EPI_OUT_F32)) && out_scale == 1.f && (lda & 7) == 0 && (ldo & 3) == 0 &&
      aligned16(A) && aligned16(W) && (reinterpret_cast<uintptr_t>(out) & 7u) == 0) {
    mimo_stream::Args a{};
    a.A = g.A; a.W = g.W; a.out = out; a.bias = bias; a.lda = lda; a.ldo = ldo; a.M = M; a.N = N;
    a.geglu = (flags & MIMO_EPI_GEGLU) ? 1 : 0;
#ifdef MIMO_TUNE
    a.dbg = tune_env("MIMO_GEMM_TRACE", 0) ? trace_buf() : nullptr;
    a.ablate = tune_env("MIMO_STREAM_ABLATE", 0);
#endif
    return mimo_stream::launch(dtype, a, cus_(), st);
  }
  if (dtype == MIMO_F16) return launch<MIMO_F16, 0>(g, st);
  if (dtype == MIMO_BF16) return launch<MIMO_BF16, 0>(g, st);
  return MIMO_EDTYPE;
}

extern "C" int mimo_gemm(int dtype, const void* A, int64_t lda, const void* W, void* out, int64_t ldo,
                         int64_t M, int N, int K, const float* bias, const float* img_bias,
                         int64_t img_bias_ld, int64_t rows_per_img, const void* residual, int64_t ldr,
                         float out_scale, unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
  return mimo_gemm_ext(dtype, A, lda, W, out, ldo, M, N, K, bias, img_bias, img_bias_ld, rows_per_img, residual, ldr,
                       out_scale, flags, workspace, workspace_bytes, nullptr, stream);
}

extern "C" int mimo_conv2d_ext(int dtype, const void* in, const void* in2, const void* W, void* out,
                               const mimo_conv_params* p, const float* bias, const float* img_bias,
                               const void* residual, float out_scale, unsigned flags, void* workspace,
                               size_t workspace_bytes, const mimo_epilogue_ext* ext, void* stream) {
  if (!in || !W || !out || !p) return MIMO_EINVAL;
  if (p->n <= 0 || p->Cin <= 0 || (p->Cin & 7) || (p->Cout & 3) || p->Cout <= 0) return MIMO_EINVAL;
  if (!(p->ksize == 1 || p->ksize == 3) || !(p->stride == 1 || p->stride == 2)) return MIMO_EINVAL;
  if (p->Cin2 < 0 || (p->Cin2 & 7) || (p->Cin2 > 0 && !in2)) return MIMO_EINVAL;
  if ((p->Hup > 0) != (p->Wup > 0)) return MIMO_EINVAL;
  if (flags & ~(MIMO_EPI_SILU | MIMO_EPI_OUT_F32 | MIMO_EPI_RES_F32 | MIMO_EPI_NO_SPLITK)) return MIMO_EINVAL;
  if (!aligned16(in) || !aligned16(W) || !aligned16(out) || (in2 && !aligned16(in2))) return MIMO_EINVAL;
  if (ext && (ext->ln_out || ext->row_half || ext->row_stats || ext->a_row_stats || ext->a_colsum))
    return MIMO_EINVAL;  // the LayerNorm side outputs / folded LayerNorm exist for dense GEMMs only
  // thin-input layers (pose guider, VAE conv_in): direct convolution, see thinconv.hip
  if (tune_env("MIMO_THIN_CONV", 1) && !in2 && p->Cin2 == 0 && !img_bias && !residual && !(ext && ext->colstats) && p->Hup == 0 &&
      !(flags & ~(MIMO_EPI_SILU | MIMO_EPI_OUT_F32 | MIMO_EPI_NO_SPLITK))) {
    const int64_t ib = (int64_t)p->n * p->Hin * p->Win * p->Cin * 2;
    const int64_t ob = (int64_t)p->n * p->Hout * p->Wout * p->Cout * ((flags & MIMO_EPI_OUT_F32) ? 4 : 2);
    if (mimo_thin::supported(p->Cin, p->Cout, p->ksize, p->stride, ib, ob) && (p->ksize == 3 || (p->pad_t == 0 && p->pad_l == 0))) {
      mimo_thin::Args a{};
      a.in = (const uint16_t*)in; a.W = (const uint16_t*)W; a.out = out; a.bias = bias;
      a.n = p->n; a.Hin = p->Hin; a.Win = p->Win; a.Cin = p->Cin; a.Hout = p->Hout; a.Wout = p->Wout; a.Cout = p->Cout;
      a.ksize = p->ksize; a.stride = p->stride; a.pad_t = p->pad_t; a.pad_l = p->pad_l; a.ldw = (int64_t)p->ksize * p->ksize * p->Cin;
      a.out_scale = out_scale; a.flags = flags & (MIMO_EPI_SILU | MIMO_EPI_OUT_F32);
      a.in_bytes = (unsigned)ib; a.w_bytes = (unsigned)((int64_t)p->Cout * a.ldw * 2); a.out_bytes = (unsigned)ob;
      return mimo_thin::launch(dtype, a, cus_(), (hipStream_t)stream);
    }
  }
  GemmArgs g{};
  g.A = (const uint16_t*)in; g.A2 = (const uint16_t*)in2; g.W = (const uint16_t*)W; g.out = out;
  g.bias = bias; g.img_bias = img_bias; g.res = residual;
  g.N = p->Cout; g.K = p->ksize * p->ksize * p->Cin + p->Cin2;
  g.ldw = g.K; g.ldo = p->Cout; g.ldr = p->Cout; g.lda = 0;
  g.M = (int64_t)p->n * p->Hout * p->Wout;
  g.rows_per_img = (int64_t)p->Hout * p->Wout * (p->imgs_per_bias_row > 0 ? p->imgs_per_bias_row : 1);
  g.ldib = p->img_bias_ld > 0 ? p->img_bias_ld : p->Cout;
  if (g.ldib & 3) return MIMO_EINVAL;
  g.out_scale = out_scale; g.flags = flags;
  g.ws = aligned16(workspace) ? workspace : nullptr; g.ws_bytes = workspace_bytes;
  g.Hin = p->Hin; g.Win = p->Win; g.Cin = p->Cin; g.Hout = p->Hout; g.Wout = p->Wout;
  g.ks = p->ksize; g.stride = p->stride; g.pad_t = p->pad_t; g.pad_l = p->pad_l;
  g.Hup = p->Hup; g.Wup = p->Wup; g.Cin2 = p->Cin2;
  g.sh = p->Hup > 0 ? (float)p->Hin / (float)p->Hup : 1.f;
  g.sw = p->Wup > 0 ? (float)p->Win / (float)p->Wup : 1.f;
  g.chunks1 = (p->Cin + BK - 1) / BK;
  g.chunks2 = (p->Cin2 + BK - 1) / BK;
  g.nkt = p->ksize * p->ksize * g.chunks1 + g.chunks2;
  if (int rc = check_ext(ext, g, g.M, g.N, g.K, flags)) return rc;
  {
    const int64_t ab = (int64_t)p->n * p->Hin * p->Win * p->Cin * 2, a2b = g.M * p->Cin2 * 2, wb = (int64_t)g.N * g.K * 2;
    if (ab >= 0x80000000LL || a2b >= 0x80000000LL || wb >= 0x80000000LL) return MIMO_EINVAL;  // see OOBA
    g.a_bytes = (unsigned)ab; g.a2_bytes = (unsigned)a2b; g.w_bytes = (unsigned)wb;
  }
  const bool ups = p->Hup > 0;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MIMO_F16) return ups ? launch<MIMO_F16, 2>(g, st) : launch<MIMO_F16, 1>(g, st);
  if (dtype == MIMO_BF16) return ups ? launch<MIMO_BF16, 2>(g, st) : launch<MIMO_BF16, 1>(g, st);
  return MIMO_EDTYPE;
}

extern "C" int mimo_conv2d(int dtype, const void* in, const void* in2, const void* W, void* out,
                           const mimo_conv_params* p, const float* bias, const float* img_bias,
                           const void* residual, float out_scale, unsigned flags, void* workspace,
                           size_t workspace_bytes, void* stream) {
  return mimo_conv2d_ext(dtype, in, in2, W, out, p, bias, img_bias, residual, out_scale, flags, workspace,
                         workspace_bytes, nullptr, stream);
}

extern "C" int mimo_row_stat_slots(int N) { return row_stat_slots_of(N); }

extern "C" int mimo_version(void) { return 5; }

extern "C" size_t mimo_workspace_bytes(void) { return (size_t)8 * ((size_t)1 << 22) * sizeof(float); }

// Kept for tools/microbench.py: the tune build re-reads its knobs at every launch, the shipped build has none.
extern "C" int mimo_reload_tuning(void) { return MIMO_OK; }

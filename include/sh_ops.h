/* softhier-ops for MI355X (gfx950): the C ABI.
 *
 * This header re-exports the hot-path subset of the reference's operator library header
 * (runwangdl/softhier-mlir runtime/sh_ops.h) with the same names, argument order, types and error codes,
 * so the same op sequence (emitted programs, C test drivers, ctypes callers) runs unchanged. Each
 * declaration cites the reference line it replaces.
 *
 * Execution model (differs from the reference's SPMD model, same observable results):
 *  - One host thread calls each op once. The op validates its arguments on the host, then enqueues HIP
 *    kernels on the library stream (sh_set_stream; default: the legacy null stream, which is ordered with
 *    PyTorch's default stream). Ops are stream-ordered and asynchronous; sh_barrier_global() drains them.
 *  - Tensors are fp16 row-major in GPU memory, addressed by 64-bit byte addresses (device pointers:
 *    a torch tensor's data_ptr(), sh_hbm_addr() or sh_hbm_malloc()). Leading dimensions are in elements.
 *  - `cluster` is accepted for source compatibility and ignored: the op always runs on the whole GPU.
 *    sh_cluster_id() == 0, sh_is_first_core() == 1 and sh_num_clusters() == 1, so guards such as
 *    `if (sh_cluster_id() == 0 && sh_is_first_core())` in emitted code fire exactly once.
 *  - Constraint checks mirror the reference (same conditions, same return codes, same budgets: the
 *    reference's 1 MiB cluster TCDM, reported by sh_l1_size()), so a call fails here exactly when it
 *    fails there. The additive entry points at the end carry no TCDM budget.
 *  - A HIP runtime failure makes an int op return SH_EHIP (-3, additive) and records the message
 *    (sh_last_error / sh_last_error_str); void ops record it the same way.
 *  - Not re-entrant across host threads.
 */
#ifndef SH_OPS_H
#define SH_OPS_H
#include <stdint.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- runtime wrappers (reference runtime/sh_ops.h:19-37, runtime/sh_rt.inc.c:2-29) ---------------------- */
void     sh_init(void);                 /* sh_ops.h:20   picks up the current HIP device; idempotent */
void     sh_barrier_global(void);       /* sh_ops.h:21   drains the library stream */
void     sh_barrier_cluster(void);      /* sh_ops.h:22   same as sh_barrier_global */
uint32_t sh_cluster_id(void);           /* sh_ops.h:23   0 */
uint32_t sh_core_id(void);              /* sh_ops.h:24   0 */
int      sh_is_first_core(void);        /* sh_ops.h:25   1 */
int      sh_is_dm_core(void);           /* sh_ops.h:26   1 */
uint32_t sh_num_clusters(void);         /* sh_ops.h:27   1: the GPU is one cluster */
void     sh_timer_start(void);          /* sh_ops.h:28   HIP event on the library stream */
void     sh_timer_end(void);            /* sh_ops.h:29   prints "[Performance Counter]: Execution period is N ns", restarts */
void     sh_eoc(uint32_t val);          /* sh_ops.h:30   drains the stream, flushes stdout, records val */
uint32_t sh_cycles(void);               /* sh_ops.h:31   ns since sh_init (1 GHz equivalence), read after the stream drains */
void     sh_printf(const char *fmt, ...);                /* sh_ops.h:32 */
uint64_t sh_hbm_addr(uint64_t byte_offset);             /* sh_ops.h:33   arena base + offset (arena: SH_HBM_ARENA_BYTES, default 1 GiB, lazy) */
uint64_t sh_hbm_malloc(uint32_t bytes);                 /* sh_ops.h:34   separate device allocation, 256 B aligned */
uint32_t sh_l1_size(void);                              /* sh_ops.h:35   the reference cluster's TCDM bytes (0x100000) */
void     sh_preload_wait(uint64_t sentinel);            /* sh_ops.h:36   drains the stream (data is resident) */
/* Additive: copy the PT_LOAD segments of a preload image (ELF32, softhier_mlir/sim/preload.py:38-78: segment at
 * physical address SH_PRELOAD_HBM_BASE + offset) into the sh_hbm_addr arena at those offsets. Returns the number of
 * segments copied, -1 for an unreadable / malformed image or a segment beyond the arena, SH_EHIP on a HIP failure. */
#define SH_PRELOAD_HBM_BASE 0xC0000000u
int      sh_preload_load(const char *path);
void     sh_call_on_core_stack(void (*fn)(void), uint32_t bytes_per_core);   /* sh_ops.h:48   calls fn() */

#define SH_ALL 0xFFFFFFFFu                              /* sh_ops.h:39 */
#define SH_CORE_STACK_BYTES 40960u                      /* sh_ops.h:47 */
#define SH_SELF (sh_cluster_id())                       /* sh_ops.h:308 */

/* ---- formats (sh_ops.h:51) -------------------------------------------------------------------------- */
enum sh_fmt { SH_FP16 = 0, SH_FP8 = 1, SH_INT16 = 2, SH_INT8 = 3 };

/* ---- GEMM: Z[M,N] (+)= X[M,K] . W[K,N] (sh_ops.h:53-88, runtime/sh_gemm.inc.c:12-189) ------------------
 * fp16 operands, fp32 accumulation on MFMA, fp16 result (RNE). tm/tn/tk are the caller's tile hints: they set
 * the divisibility rule exactly as in the reference (0 -> 256); the GPU tile is chosen by the library. */
typedef struct {
    uint32_t tm, tn, tk;     /* tile; 0 -> 256 */
    uint32_t pipeline;       /* accepted (the GPU kernels always double-buffer) */
    uint32_t accumulate;     /* 1: Z += X.W (Z read first); 0: Z = X.W */
    uint32_t fmt;            /* enum sh_fmt; only SH_FP16 computes (others: -1) */
    uint32_t l1_base;        /* counts towards the TCDM budget exactly as in the reference */
} sh_gemm_cfg;               /* sh_ops.h:54-60 */

/* sh_ops.h:66-67 (sh_gemm.inc.c:53-117): -1 when M%tm, N%tn or K%tk != 0 (or fmt != SH_FP16, or a NULL
 * address), -2 when sh_gemm_l1_bytes() exceeds the reference TCDM, SH_EHIP on a HIP failure, else 0. */
int sh_gemm(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
            uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg, uint32_t cluster);

/* sh_ops.h:72-73 (sh_gemm.inc.c:127-189): SUMMA mode over a virtual SH_MESH_P x SH_MESH_P mesh of output
 * tiles (the reference's 4 x 4 cluster mesh). Same constraints and codes: tm == tn, M == N == P * tm,
 * K % tk == 0 (-1), TCDM budget (-2). The launch is the tiled GEMM with its XCD-aware tile order (each XCD
 * walks a contiguous band of output tile rows, so an X row panel is fetched into one XCD's L2 and re-read there
 * by the whole band); there is no separate mesh schedule and no broadcast step on one GPU. */
#define SH_MESH_P 4u
int sh_gemm_mesh(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                 uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg);

/* sh_ops.h:88 (sh_gemm.inc.c:24-30): l1_base + (pipeline ? 2 : 1) * (tm*tk + tk*tn) * 2 + tm*tn*2. */
uint32_t sh_gemm_l1_bytes(uint32_t M, uint32_t N, uint32_t K, const sh_gemm_cfg *cfg);

/* Small-M GEMM (sh_ops.h:74-85): Z = X.W (+= with cfg->accumulate) with the reference's plan checks. cfg fields
 * are "0 = auto" here: tm = rows per block (must divide M), tn = column granule (4), tk = K panel. Returns 0, -1
 * (tm does not divide M / NULL), -2 (no plan fits the reference's scratch limit 0x90000 from l1_base), -3 (fmt). */
enum { SH_XM_AUTO = 0, SH_XM_PANEL = 1, SH_XM_WHOLE = 2 };                                   /* sh_ops.h:79 */
int sh_gemm_xmcast(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                   uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg);        /* sh_ops.h:80-81 */
int sh_gemm_xmcast_ex(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                      uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg, uint32_t mode);  /* sh_ops.h:82-83 */
uint32_t sh_gemm_xmcast_l1_bytes(uint32_t M, uint32_t N, uint32_t K, const sh_gemm_cfg *cfg, uint32_t mode);  /* sh_ops.h:84, ~0u: no plan */

/* ---- row-wise / elementwise ops (sh_ops.h:90-100, runtime/sh_rowops.inc.c:383-465) -------------------
 * fp16 in/out, one pass over HBM. Parameter rows (gamma, beta, bias) are fp16 rows. LayerNorm, softmax and
 * scale compute in fp32; add / add_bias use packed fp16 adds (which round exactly as the fp32 sum rounded to
 * fp16); GELU is the tanh form evaluated on packed fp16 (a few fp16 ulps from the fp32 form). */
void sh_layernorm(uint64_t y, uint64_t x, uint64_t gamma, uint64_t beta, uint32_t rows, uint32_t cols, uint32_t ld, float eps, uint32_t cluster);  /* sh_ops.h:94 */
void sh_softmax_rows(uint64_t y, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ld, float scale, uint32_t cluster);  /* sh_ops.h:95 */
void sh_gelu(uint64_t y, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t cluster);                     /* sh_ops.h:96 tanh form */
void sh_add(uint64_t y, uint64_t a, uint64_t b, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t cluster);          /* sh_ops.h:97 */
void sh_add_bias(uint64_t y, uint64_t x, uint64_t bias_row, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t cluster); /* sh_ops.h:98 */
void sh_scale(uint64_t y, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ld, float s, uint32_t cluster);           /* sh_ops.h:99 */
void sh_transpose(uint64_t dst, uint64_t src, uint32_t rows, uint32_t cols, uint32_t ld_src, uint32_t ld_dst, uint32_t cluster); /* sh_ops.h:100 bit-exact */
/* No counterpart in the reference (LayerNorm folded into the next GEMM, sh_gemm_epi.ln_stats): per row of x, the
 * mean and 1 / sqrt(biased variance + eps) as fp32 pairs into stats [rows][2], the statistics sh_layernorm
 * computes (two passes over the row in fp32). */
void sh_row_stats(uint64_t stats, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ld, float eps);
/* No counterpart in the reference: the weight side of the fold for z = LN(x) . W + b, W [K, N] (ldw):
 * wp = r16(gamma_k W[k][n]) (fp16, leading dim ldwp), c[n] = sum_k wp[k][n] (fp32), d[n] = sum_k beta_k W[k][n]
 * + b[n] (fp32; bias = 0: none). gamma, beta, bias: fp16 rows. Run once per weight. */
void sh_ln_fold(uint64_t wp, uint64_t c, uint64_t d, uint64_t w, uint64_t gamma, uint64_t beta, uint64_t bias,
                uint32_t K, uint32_t N, uint32_t ldw, uint32_t ldwp);
/* sh_ops.h:218 (sh_l1.inc.c:58-61): 1-D copy of `bytes` from src to dst in HBM (non-overlapping), enqueued on the
 * library stream (the reference's call is synchronous on its DM core; here it is ordered like every other op). */
void sh_dma_copy(uint64_t dst, uint64_t src, uint32_t bytes);
/* No counterpart in the reference: read [addr, addr + bytes) through the GPU's caches (L2 and the 256 MB Infinity
 * Cache) on the library stream, writing nothing, so that a kernel launched later finds those bytes cached instead of
 * in HBM. For callers that know which weights come next: the encoder stack issues it on a second stream for a
 * layer's remaining weights while its attention runs. 0, -1 for a NULL address, SH_EHIP for a launch failure. */
int sh_prefetch(uint64_t addr, uint64_t bytes);

/* ---- fused attention (sh_ops.h:102-127, runtime/sh_attention.inc.c:55-243) ----------------------------
 * o = softmax(scale * q k^T) v per head; head h = columns [h*dh, (h+1)*dh). Flash-style on the GPU (online
 * softmax over key blocks, scores never leave the CU), so sq only has to satisfy the reference's rules. */
int sh_attention_head(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t S, uint32_t dh,
                      uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale, uint32_t cluster);   /* sh_ops.h:109-110 */
int sh_attention_q(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t S, uint32_t D, uint32_t H,
                   uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale, uint32_t cluster, uint32_t sq); /* sh_ops.h:114-115 */
int sh_attention(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t S, uint32_t D, uint32_t H,
                 uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale, uint32_t cluster);      /* sh_ops.h:116-117 */
uint32_t sh_attention_l1_bytes_q(uint32_t S, uint32_t dh, uint32_t sq);   /* sh_ops.h:118 */
uint32_t sh_attention_l1_bytes(uint32_t S, uint32_t dh);                  /* sh_ops.h:119 */
uint32_t sh_attention_q_block(uint32_t S, uint32_t dh, uint32_t H, uint32_t P);   /* sh_ops.h:123 same rule */
/* sh_ops.h:127: ns stamps of the last attention call's last workgroup, from its first workgroup's start (phase 7
 * = 0): 0 start, 1-2 operands staged, 3-4 first key block's scores / row maximum known, 5 every key block done,
 * 6 stored (the kernels without stamps report only 6, the launch's event time; all 0 when that call was
 * sh_attention_batched or made under stream capture, which carry no stamps). */
uint32_t sh_attention_profile(uint32_t S, uint32_t dh, uint32_t phase);

/* ---- Llama-style decoder ops (sh_ops.h:277-307, runtime/sh_llm.inc.c) -----------------------------------
 * Token masks: tok[j] (uint16, one per position) is the cumulative attention-block id of position j, SH_LLM_PAD
 * for padding; query i attends key j iff tok[j] <= tok[i] (unsigned). A padding query row (or one with no allowed
 * key) is uniform. Row ops need cols % 4 == 0 (and cols <= 8192 here); violations set sh_last_error and return. */
#define SH_LLM_PAD 0xFFFFu                                                                         /* sh_ops.h:283 */
void sh_rmsnorm(uint64_t y, uint64_t x, uint64_t gamma, uint32_t rows, uint32_t cols, uint32_t ld, float eps, uint32_t cluster);  /* sh_ops.h:284 */
void sh_rope(uint64_t y, uint64_t x, uint64_t cos_sin, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t ld_table, uint32_t dh,
             uint32_t cluster);                                                                    /* sh_ops.h:288, rotate-half */
void sh_silu_mul(uint64_t y, uint64_t a, uint64_t b, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t cluster);  /* sh_ops.h:289 */
void sh_softmax_masked(uint64_t y, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ld, float scale, uint64_t tok_q,
                       uint64_t tok_k, uint32_t cluster);                                          /* sh_ops.h:292, scale > 0 */
int sh_attention_head_masked(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t S, uint32_t dh, uint32_t ldq,
                             uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale, uint64_t tok, uint32_t cluster);  /* sh_ops.h:294-295 */
int sh_attention_gqa(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t S, uint32_t D, uint32_t H, uint32_t Hkv,
                     uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale, uint64_t tok, uint32_t cluster);  /* sh_ops.h:299-300 */
void sh_pixel_shuffle(uint64_t dst, uint64_t src, uint32_t grid, uint32_t D, uint32_t s, uint32_t cluster);  /* sh_ops.h:303, bit-exact */

/* ---- test helpers (sh_ops.h:220-240, runtime/sh_test.inc.c, runtime/sh_rt.inc.c:31-59) ----------------
 * Fills run as GPU kernels (LCG jump-ahead per element, identical values to the sequential loop); dumps
 * gather on the GPU and print on the host in the reference's "<tag> r c hex" format. */
void sh_test_fill_int_fp16(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed, int lo, int hi);              /* sh_ops.h:223 */
void sh_test_fill_fp16(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed, int lo, int hi, float scale);     /* sh_ops.h:224 */
void sh_test_dump_samples(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed, uint32_t nsamples, const char *tag); /* sh_ops.h:226 */
void sh_test_dump_samples_idx(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t seed, uint32_t nsamples, const char *tag, uint32_t idx); /* sh_ops.h:227 */
uint32_t sh_test_check_gemm(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                            uint32_t ldx, uint32_t ldw, uint32_t ldz, uint32_t nsamples, float tol,
                            float z0, const char *tag);                                                                        /* sh_ops.h:230-232 */
void     sh_test_fill_const_fp16(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t bits);                        /* sh_ops.h:234 */
void     sh_test_fill_colparity_fp16(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t even, uint32_t odd);      /* sh_ops.h:235 */
uint32_t sh_test_check_const_fp16(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, uint32_t bits, uint32_t tol, const char *tag); /* sh_ops.h:236 */
void sh_test_dump_all(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, const char *tag);                                  /* sh_ops.h:183 */
void sh_test_dump_all_idx(uint64_t a, uint32_t rows, uint32_t cols, uint32_t ld, const char *tag, uint32_t idx);                /* sh_ops.h:184 */
float    sh_fp16_to_f32(uint16_t h);    /* sh_ops.h:239 IEEE binary16 -> binary32, exact */
uint16_t sh_f32_to_fp16(float f);       /* sh_ops.h:240 RNE; overflow -> Inf; NaN -> 0x7E00 | sign */

/* sh_ops.h:249-258 hardware register conversions: portable equivalents on the host (low 16 bits used). */
static inline float    sh_h2f(uint32_t h) { return sh_fp16_to_f32((uint16_t)(h & 0xFFFFu)); }
static inline uint32_t sh_f2h(float f)    { return 0xFFFF0000u | sh_f32_to_fp16(f); }

/* ====================================================================================================
 * Additive entry points (no counterpart in the reference's ABI; existing layouts are unchanged).
 * ==================================================================================================== */
#define SH_EHIP (-3)                     /* an int op's return code for a HIP runtime failure */

int         sh_last_error(void);         /* 0, or the code of the last failure (-1 args, SH_EHIP HIP); cleared on read */
const char *sh_last_error_str(void);     /* message of the last failure ("" if none) */
void        sh_set_stream(uint64_t stream);   /* hipStream_t to enqueue on (0 = legacy null stream) */
uint64_t    sh_get_stream(void);
/* Split-K calls keep an fp32 partials workspace per stream they ran on (at least 64 MiB each, grown geometrically,
 * outgrown buffers kept because graphs captured earlier may address them), so a caller that creates and destroys
 * streams would otherwise hold that memory until exit. sh_stream_release(stream) waits for the stream, then frees
 * everything the library holds for it (0, or SH_EHIP); the next split-K call on that stream allocates again. Call
 * it only when no graph captured on that stream will be replayed. sh_stream_workspace_bytes: the live workspace
 * of a stream (0 if none). */
int         sh_stream_release(uint64_t stream);
uint64_t    sh_stream_workspace_bytes(uint64_t stream);
double      sh_timer_last_ns(void);      /* the period sh_timer_end() printed last */
/* Text capture for in-process callers: while on, everything the library prints (sh_printf, sample dumps,
 * timer lines) is appended to an internal buffer instead of stdout. sh_captured copies it out (NUL
 * terminated, truncated to cap - 1) and returns its full length; turning capture on clears it. */
void        sh_capture(int on);
uint64_t    sh_captured(char *buf, uint64_t cap);

/* Split-K GEMM: K is cut into `splits` contiguous ranges computed by separate workgroups into an fp32
 * workspace owned by the library, then reduced in a fixed order (deterministic) and rounded once to fp16.
 * Two equal ranges (K % 128 == 0) run in one workgroup per tile instead, whose two halves add their fp32 sums
 * in that same order: the same bits, no workspace, no reduction launch.
 * Shape/tile checks as sh_gemm (-1/-2); splits == 0 lets the library choose. */
int sh_gemm_splitk(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                   uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg, uint32_t splits, uint32_t cluster);

/* No counterpart in the reference: sh_gemm_splitk for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). Same arguments, checks and results
 * (the same kernels and summation order, so the same bits); the fp32 partials live in a fixed 16 MiB array of
 * the library's code object on each GPU, so the call makes no hipMalloc / hipFree and skips the one-time tile
 * timing. Returns -1 (before any GPU work) when a launch that writes partials needs more than 16 MiB of them
 * (splits x M x N x 4 bytes); a request of two equal K ranges (K % 128 == 0, 16-byte aligned operands) runs both
 * ranges in one workgroup and writes none, at any size. All calls on one GPU share that array: calls that overlap
 * on one GPU race. */
int sh_gemm_splitk_noalloc(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                           uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg, uint32_t splits, uint32_t cluster);

/* Fused GEMM epilogue: z = act(X.W [+ z_old if cfg->accumulate] + bias) rounded to fp16, then
 * [+ residual, rounded again]. bias: 0 or an fp16 (SH_BIAS_FP16) / fp32 (SH_BIAS_FP32) row of N values.
 * residual: 0 or an fp16 [M,N] tensor with leading dim ldr (may alias z). No tile-divisibility rule and no
 * TCDM budget; M, N, K >= 1. splits: as sh_gemm_splitk (1 = no split, 0 = library choice). */
enum { SH_ACT_NONE = 0, SH_ACT_GELU = 1 };
enum { SH_BIAS_FP16 = 0, SH_BIAS_FP32 = 1 };
typedef struct {
    uint64_t bias;        /* 0: none */
    uint32_t bias_fmt;    /* SH_BIAS_FP16 | SH_BIAS_FP32 */
    uint32_t act;         /* SH_ACT_NONE | SH_ACT_GELU (tanh form, as sh_gelu) */
    uint64_t residual;    /* 0: none */
    uint32_t ldr;         /* leading dim of residual (elements) */
    uint32_t splits;      /* 1: none; 0: library choice */
    /* LayerNorm folded into the GEMM (0: off). With X the raw rows and W' = diag(gamma) W, c = 1^T W' and
     * d = beta^T W + b from sh_ln_fold, the product p = X . W' becomes z = r p - r mu c + d before the rest of the
     * chain (act, residual), which is LN(X) . W + b; ln_stats: fp32 [M][2] (mu, r) rows from sh_row_stats (8-byte
     * aligned, else -1), ln_c: fp32 row of N, and the bias must then be the fp32 row d (SH_BIAS_FP32). Rounded once
     * to fp16. */
    uint64_t ln_stats;
    uint64_t ln_c;
    /* Row partials (0: off): the GEMM also writes, for each stored row of Z and each 32 columns of it, the fp32 pair
     * (sum s, M2 = sum (z - s / 32)^2) of the stored fp16 values to stats_out [M][N / 32] (N % 32 == 0, 16-byte
     * aligned operands): the statistics the next GEMM's LayerNorm fold needs, without a pass over Z. That GEMM
     * takes them with ln_stats = stats_out, ln_parts = N / 32 (its K / 32) and ln_eps, and forms mean and
     * variance with Chan's pairwise combination; ln_parts = 0: ln_stats holds (mean, r) rows of sh_row_stats. */
    uint64_t stats_out;
    uint32_t ln_parts;
    float ln_eps;
} sh_gemm_epi;
int sh_gemm_ex(uint64_t x, uint64_t w, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
               uint32_t ldx, uint32_t ldw, uint32_t ldz, const sh_gemm_cfg *cfg, const sh_gemm_epi *epi);

/* No counterpart in the reference: sh_gemm_ex with the weight given transposed, wt = W^T as an [N, K] row-major
 * tensor with leading dim ldwt >= K (z = X . W, W[k][n] = wt[n * ldwt + k]). For callers that keep their weights
 * transposed once (the encoder layer): both operands are then rows of k, which lets the GPU use larger tiles and
 * plain LDS reads. Same epilogue, checks and codes as sh_gemm_ex (-1 also for ldwt < K). */
int sh_gemm_ex_wt(uint64_t x, uint64_t wt, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                  uint32_t ldx, uint32_t ldwt, uint32_t ldz, const sh_gemm_cfg *cfg, const sh_gemm_epi *epi);

/* Additive (no counterpart in the reference): the GEMM cost model's plan for an (M, N, K) problem with
 * 16-byte-aligned operands and a split request (0 = library choice): out[0] tile configuration, out[1] /
 * out[2] its tile rows / columns, out[3] the split count. A large problem's first call may still replace the
 * configuration by its one-time timing, and a problem of few tiles runs on smaller tiles instead, which with splits = 0 may
 * sum K in up to eight ranges inside a workgroup (fp32, in range order; deterministic). Runs no GPU work. 0, or -1 for an
 * empty problem / NULL out. */
int sh_gemm_plan(uint32_t M, uint32_t N, uint32_t K, uint32_t splits, uint32_t *out);

/* Additive (no counterpart in the reference): the GEMM tile table that sh_gemm_plan indexes and SH_GEMM_CFG forces.
 * sh_gemm_tile_count: its entries. sh_gemm_tile_info(i, out): out[0] / out[1] tile rows / columns, out[2] kernel
 * family (1 register-staged: any alignment and K; 2 direct-to-LDS with a partial last k-slice variant; 5
 * direct-to-LDS, register epilogue; 6 direct-to-LDS for the W^T operand), out[3] threads per workgroup, out[4] W^T
 * operand, out[5] register epilogue (LayerNorm fold and row partials without fp32 partials), out[6] in-workgroup
 * split of two equal K ranges, out[7] partial-k-slice variant. Unsplit direct-to-LDS configurations (families 2, 5
 * and 6) store the same bits; the register-staged ones (1) store the same bits among themselves. 0, or -1 for i out
 * of range / NULL out. No GPU work. */
int sh_gemm_tile_count(void);
int sh_gemm_tile_info(uint32_t i, uint32_t *out);

/* Batched multi-head attention (the reference has no batch dimension): sequence b uses q + b*bsq*2 bytes,
 * likewise k/v/o with their own batch strides in elements (e.g. S*ld for rows stacked as [B*S, ld]).
 * Constraints as sh_attention_q except the TCDM budget; sq == 0 -> the library's choice. */
int sh_attention_batched(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t B, uint32_t S, uint32_t D, uint32_t H,
                         uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo,
                         uint64_t bsq, uint64_t bsk, uint64_t bsv, uint64_t bso, float scale, uint32_t sq);
/* No counterpart in the reference: sh_attention_batched that also reads two ranges [pfN, pfN + pfN_bytes) (bytes 0:
 * none) into the GPU's caches (L2 and the Infinity Cache) while it runs, writing nothing there: the same outputs, bit
 * for bit. For callers that know which weights the next kernels read (the encoder stack: a layer's out-proj and FFN
 * weights and the next layer's QKV weight, which do not all stay in the cache next to the activations); attention
 * leaves memory bandwidth and room on every CU, so the reads cost it little and no second stream or event is
 * needed. A head the one-pass kernel does not take reads the ranges after its kernel instead (sh_prefetch). -1 also
 * for a NULL range with bytes > 0. */
int sh_attention_batched_prefetch(uint64_t q, uint64_t k, uint64_t v, uint64_t o, uint32_t B, uint32_t S, uint32_t D, uint32_t H,
                                  uint32_t ldq, uint32_t ldk, uint32_t ldv, uint32_t ldo,
                                  uint64_t bsq, uint64_t bsk, uint64_t bsv, uint64_t bso, float scale, uint32_t sq,
                                  uint64_t pf0, uint64_t pf0_bytes, uint64_t pf1, uint64_t pf1_bytes);

/* ---- 8-bit paged key / value cache (no counterpart in the reference) -----------------------------------------------
 * Keys and values of many requests in pages of `bs` tokens, 8-bit codes with one fp32 scale for each page and head:
 * value = code x scale. A request's tokens 0, 1, ... lie in the pages its row of the block table names, bs to a page.
 * SH_INT8: two's complement, -127 .. 127. SH_FP8: OCP e4m3 (finite, largest 448). Values are stored with the tokens of a
 * page consecutive, as the product with the probabilities reads them.
 * A serving step: sh_kv_slots (where the new tokens go), the projections, sh_kv_append_rope (queries and keys turned by their positions), sh_attention_kv;
 * or, with a table of the caller's own, sh_rope and sh_kv_append. (sh_rope takes a
 * cos / sin row for each row and no positions: the caller gathers its table's rows at `pos`, any row where that is -1.) The
 * calls need no device memory of the library's own and no host synchronisation, so a step captures into a HIP graph whose replays
 * read the lengths of that moment. */
typedef struct {
    uint64_t k;           /* codes: pages of [hkv][bs][dh], 16-byte aligned */
    uint64_t v;           /* codes: pages of [hkv][dh][bs], 16-byte aligned */
    uint64_t ks, vs;      /* fp32 scales, finite and >= 0: pages of [hkv] */
    uint64_t pgk, pgv;    /* bytes from a page to the next, multiples of 16 and >= hkv bs dh; 0: hkv bs dh */
    uint32_t pgs;         /* floats from a page's scales to the next page's, >= hkv; 0: hkv */
    uint32_t pages;       /* pages of the cache, pages x bs < 2^31 */
    uint32_t hkv;         /* key / value heads, 1 .. 1024 */
    uint32_t dh;          /* head width: a multiple of 16, 16 .. 256 */
    uint32_t bs;          /* tokens of a page: 16, 32 or 64 */
    uint32_t fmt;         /* SH_INT8 | SH_FP8 */
} sh_kv_cache;

/* Block table, slots and lengths of a step, on the GPU. All arrays int32 in GPU memory, written in place:
 *   table [B][ld]     page of each bs tokens of a request (in / out: the new pages' entries are written)
 *   lens [B]          tokens each request holds; lens_out [B] (may be lens): with the new ones
 *   add [B]           tokens each adds (0: none), or < 0: the request has ended, its pages go back
 *   pool [pages]      ring of free page numbers; state {head, count, -}: its first entry and how many there are (to begin:
 *                     pool[i] = i, state = {0, pages, 0}); state_out (may be state) {head, count, requests refused}
 *   row_start [B + 1] first row of each request among the step's new rows, in order, and their total
 *   slots, pos [rows] of each new row: page x bs + offset, and position in its request; -1 for the rows of a refused
 *                     request and behind the last row
 *   kv_len [B]        keys that a request's rows see with themselves (lens + add); 0 for an ended or refused request
 * Requests take pages in order. One that needs more than are left, whose rows end behind `rows` or whose tokens exceed
 * ld x bs is refused: its length and table stay, and those after it that need pages are served only if the pages that
 * it and they ask for together are there. Pages of ended requests can be taken from the next call on: all of its table row's, so a
 * page is in one row only. Rows that share pages (a common prefix) are not for this call: the caller keeps table, lengths
 * and pages of such requests itself, and sh_attention_kv reads them like others. The sum of `add` stays
 * below 2^31. B x ld and pages x bs below 2^31, B <= 65536. 0, -1 for bad arguments, SH_EHIP. */
int sh_kv_slots(uint64_t table, uint32_t ld, uint64_t lens, uint64_t lens_out, uint64_t add, uint64_t pool, uint64_t state, uint64_t state_out,
                uint64_t row_start, uint64_t slots, uint64_t pos, uint64_t kv_len, uint32_t B, uint32_t bs, uint32_t pages, uint32_t rows);

/* New key and value rows (fp16, [rows][hkv dh], leading dims ldk / ldv) into the cache at slots[row] (int32; rows with a
 * slot outside the cache are skipped). The scale of a page and head is the smallest power of two s >= 2^-32 with
 * |x| <= 127 s (448 s for SH_FP8) for its tokens, and never smaller than the one its older tokens have; where it grows, they are
 * rounded to it again. Codes round to nearest even. NaN is stored as 0, infinities as +-65504. A request's new tokens are
 * consecutive rows and, within a page, consecutive slots, and a page that is written belongs to one request: rows that put two
 * requests, one slot twice, or slots with others (or skipped rows) between them into one page leave that page undefined. A first token at offset 0 starts a
 * page anew; other codes of the page are left as they are. 0, -1, SH_EHIP. */
int sh_kv_append(const sh_kv_cache *c, uint64_t k, uint64_t v, uint32_t ldk, uint32_t ldv, uint64_t slots, uint32_t rows);

/* Causal attention of new rows over the cache: o = softmax(scale q k^T) v per head, scale > 0, fp32 sums. Request b's rows are
 * row_start[b] .. row_start[b + 1] - 1 of q / o (fp16, [rows][H dh]; row_start, which does not decrease; 0: row b), its keys the first kv_len[b]
 * tokens of its table row, and its last row sees all of them, each earlier row one key less. window > 0: a row sees
 * only its last `window` keys; pages wholly before every row's window are not read. Head h reads key / value head h / (H / hkv). Keys
 * in pages outside the cache (table entries < 0 or >= pages) are left out. A row that sees no key gets zeros; rows of no
 * request are left as they are, as are a request's rows beyond its first max_q. max_q: an upper bound of a request's rows. ws: scratch
 * of at least sh_attention_kv_ws_bytes(c, B, rows, max_q, H, ld_table) bytes, 16-byte aligned, that no call running at the same
 * time uses (another stream, or a graph replayed beside this one, needs its own); what it holds need not be kept, and what is
 * enough for some B, rows, max_q and ld_table is enough for smaller ones.
 * B x (ld_table bs / 64 + 1) x hkv x ceil(max_q (H / hkv) / 16) below 2^32, for chunks (rows H / 128 + B hkv) below 2^24.
 * Scores, scale q k, stay within fp32. A row of q with an infinity or a NaN in a head gives NaN there wherever it sees a key.
 * max_q chooses the kernel for the whole call: single tokens beside chunks (max_q (H / hkv) > 64) are best a call of their own, over the same
 * rows: the requests of few rows first, then table, kv_len and row_start from the first chunk on (row_start's values stay as they are).
 * A probability is held to 22 bits where max_q (H / hkv) <= 8. With more rows it may be held in fp16: off by up to 2^-11 of it, so an output
 * by up to 2^-11 of sum p |v|, besides its own rounding.
 * 0, -1 for bad arguments, -2 for too small a ws, SH_EHIP. Deterministic; how keys are shared out depends on the whole
 * batch, so a request's low bits may differ with its neighbours. */
int sh_attention_kv(uint64_t q, uint64_t o, const sh_kv_cache *c, uint64_t table, uint32_t ld_table, uint64_t kv_len, uint64_t row_start,
                    uint32_t B, uint32_t rows, uint32_t max_q, uint32_t H, uint32_t ldq, uint32_t ldo, float scale, uint32_t window,
                    uint64_t ws, uint64_t ws_bytes);
uint64_t sh_attention_kv_ws_bytes(const sh_kv_cache *c, uint32_t B, uint32_t rows, uint32_t max_q, uint32_t H, uint32_t ld_table);

/* ---- rotary positions (no counterpart in the reference but sh_rope's formula) ---------------------------------------
 * The first `rot` columns of a head are turned in pairs by an angle that grows with the row's position: pair i by a =
 * 2 pi position step[i] / 2^64 (whole turns fall off), (x1, x2) -> (x1 c - x2 s, x2 c + x1 s) with c, s = mscale (cos a, sin a); the other
 * columns stay. Cosine and sine are rounded to fp32 from 64 bits, products and sums to fp32, the result to fp16: by given steps the farthest position is turned
 * as exactly as the first. What a step is off counts once for each position (sh_rope_steps: 1.5e-16 turns, below). */
enum { SH_ROPE_HALF = 0,      /* pair i: columns i and i + rot / 2 */
       SH_ROPE_PAIRS = 1 };   /* pair i: columns 2 i and 2 i + 1 */
enum { SH_ROPE_NONE = 0, SH_ROPE_LINEAR = 1, SH_ROPE_BANDS = 2, SH_ROPE_RAMP = 3 };
typedef struct {
    uint64_t step;        /* uint64 [rot / 2] in GPU memory, 8-byte aligned: turns per position x 2^64, of sh_rope_steps or the caller's */
    uint32_t rot;         /* turned columns of a head: even, 2 .. the head's width */
    uint32_t layout;      /* SH_ROPE_HALF | SH_ROPE_PAIRS */
    float mscale;         /* 1: cosine and sine as they are */
    uint32_t reserved;    /* 0 */
} sh_rope_plan;

/* The steps of a model, once: w_i = base^(-2 i / rot) radians a position (base > 1), for contexts `factor` times longer than the
 * first one of `ctx` positions brought to w_i (keep + (1 - keep) / factor), where keep is
 *   SH_ROPE_NONE    1 (factor, lo, hi, ctx are not read)
 *   SH_ROPE_LINEAR  0: every position counts 1 / factor
 *   SH_ROPE_BANDS   by the pair's turns n = ctx w_i / (2 pi) in the first context: 0 for n <= lo, 1 for n >= hi, linear in n between
 *   SH_ROPE_RAMP    by its index: 1 up to the index (rounded down, at least 0) whose pair turns hi times in it, 0 from that (rounded up, at most
 *                   rot - 1) of lo turns, linear in the index between
 * Frequencies are computed in fp64: of w_i up to 1 a step is within 1.5e-16 turns of the formula's (for bands while hi^2 / (hi - lo) is far below ctx), a position's
 * angle within that many times the position: 1e-9 rad at 2^20, 2e-6 at 2^31 - 1. A caller with exacter frequencies writes the steps.
 * 0, -1 for bad arguments (0 < lo < hi), SH_EHIP. */
int sh_rope_steps(uint64_t step, uint32_t rot, double base, uint32_t scaling, double factor, double lo, double hi, uint32_t ctx);

/* `heads` heads of dh columns (dh even) of each row, turned by pos[row] (int32): y = the turned x (fp16, leading dims ldy / ldx). A row with a
 * negative position is left as it is in y. y is x (with the same leading dim: in place) or does not overlap it. Query and key heads that lie
 * side by side in a projection's rows are one call. 0, -1, SH_EHIP. */
int sh_rope_pos(uint64_t y, uint64_t x, uint64_t pos, const sh_rope_plan *p, uint32_t rows, uint32_t heads, uint32_t dh, uint32_t ldy, uint32_t ldx);

/* sh_kv_append of keys turned on the way, the values as they are, and the step's queries turned into yq (H heads; 0: none; yq as y of
 * sh_rope_pos), in one launch: the bits of sh_rope_pos on q and k, then sh_kv_append. rot a multiple of 8. A row with a negative position
 * counts as one with a slot outside the cache, and its queries are left as they are in yq; the queries of other rows with such a slot are turned. yq does not
 * overlap k or v. 0, -1, SH_EHIP. */
int sh_kv_append_rope(const sh_kv_cache *c, const sh_rope_plan *p, uint64_t yq, uint64_t q, uint64_t k, uint64_t v, uint64_t pos, uint64_t slots, uint32_t rows,
                      uint32_t H, uint32_t ldyq, uint32_t ldq, uint32_t ldk, uint32_t ldv);

/* Few rows times a weight of 4-bit codes (no counterpart in the reference): z = act(x . W + bias) rounded to fp16, then
 * [+ residual, rounded again], W[k][n] = (code[k][n] - zero[k / group][n]) scale[k / group][n]. w: words [K / 8][N]
 * (uint32, leading dim ldw), bits 4 j .. 4 j + 3 of word (i, n) the code of k = 8 i + j. scale: fp16 [ceil(K / group)][N],
 * zero: one byte (0 .. 15) each, same shape and leading dim lds; zero = 0: 8 throughout. K a multiple of 8, group a multiple of 32
 * (the last group may be short). epi: bias, act, residual as sh_gemm_ex (splits 0 or 1, no LayerNorm fold, no row
 * partials). fp32 sums, scales applied in fp32: z = sum over groups of scale (x . code - zero sum x), so a row with an infinity
 * gives NaN. Written for M up to 64: the weight is read again (from cache) for every 16 or 32 rows. A row's bits do not depend on M
 * or on the other rows. M <= 2^19, N <= 2^26. 0, -1 for bad arguments, SH_EHIP. softhier_mlir_amd/w4.py makes words, scales and zeros of
 * an fp16 weight. */
int sh_gemm_w4(uint64_t x, uint64_t w, uint64_t scale, uint64_t zero, uint64_t z, uint32_t M, uint32_t N, uint32_t K, uint32_t group,
               uint32_t ldx, uint32_t ldw, uint32_t lds, uint32_t ldz, const sh_gemm_epi *epi);

/* ---- microscaled 4-bit floating point (no counterpart in the reference) -----------------------------------------------
 * A row of K numbers as codes and scales, both operands of a product alike (a weight W [K, N] as the N rows of W^T): codes of e2m1 (sign,
 * 2 bits of exponent, 1 of fraction: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte, the lower k in the low four bits, 16 bytes for each
 * block of 32 k; a scale byte e for each block, 2^(e - 127), 255: NaN. Codes: 16-byte aligned, leading dim in bytes a multiple of 16, at least 16
 * ceil(K / 32) (multiples of 64 are read fastest). Scales: 4-byte aligned, leading dim in bytes a multiple of 4, at least ceil(K / 32) (of 16: fastest).
 * All rows have their leading dim in memory, the last one too. */

/* Rows x (fp16 [rows][cols], leading dim ldx) as codes and scales. The scale of a block is the smallest power of two s >= 2^-32 with |x| <= 6 s; codes
 * are nearest, ties to even. (The OCP conversion takes half this scale where a block's largest |x| is then between 6 and 8 times the scale, and cuts it to 6: codes
 * of such blocks differ from other programs', and the products take either.) A block with a NaN or an infinity has scale 255 and codes of 0. Codes behind `cols` in the last block are 0; bytes
 * behind the last block and the last scale are left as they are. 0, -1, SH_EHIP. */
int sh_mx4_quant(uint64_t codes, uint64_t scales, uint64_t x, uint32_t rows, uint32_t cols, uint32_t ldc, uint32_t lds, uint32_t ldx);

/* z = act(x . W + bias) rounded to fp16, then [+ residual, rounded again], of rows in 4 bits: xc, xs [M], wc, ws [N] (the rows of W^T). fp32
 * sums of exact products. Codes behind K in the last block count where both operands' are not 0 (sh_mx4_quant's are 0); scale bytes behind the last block are
 * not used. A row of x or W with a scale of 255 gives NaN. epi: bias, act, residual as sh_gemm_ex (splits 0 or 1, no LayerNorm
 * fold, no row partials). M, N <= 2^26. 0, -1 for bad arguments, SH_EHIP. Deterministic; which kernel runs depends on M, N and
 * the leading dims, so a row's low bits may. A workgroup sums all of K: few columns of a long K take longest for their size (128 x 1024 x 16384: 24 us). Leading dims
 * of codes or scales above 2^24 are for few rows or columns (700 x 1024 x 2880 with the weight's rows so far apart: 12.4 us, else 7.1). */
int sh_gemm_mx4(uint64_t xc, uint64_t xs, uint64_t wc, uint64_t ws, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                uint32_t ldxc, uint32_t ldxs, uint32_t ldwc, uint32_t ldws, uint32_t ldz, const sh_gemm_epi *epi);

/* The same for up to 16 rows x of fp16 [M][K] (leading dim ldx), brought into 4 bits on the way as sh_mx4_quant does: one launch for single tokens,
 * and the bits of the two calls. */
int sh_gemm_mx4_f16(uint64_t x, uint64_t wc, uint64_t ws, uint64_t z, uint32_t M, uint32_t N, uint32_t K,
                    uint32_t ldx, uint32_t ldwc, uint32_t ldws, uint32_t ldz, const sh_gemm_epi *epi);

/* LayerNorm with separate input / output leading dims (fused residual stream layouts). */
void sh_layernorm_ld(uint64_t y, uint64_t x, uint64_t gamma, uint64_t beta, uint32_t rows, uint32_t cols,
                     uint32_t ldy, uint32_t ldx, float eps);

#ifdef __cplusplus
}
#endif
#endif /* SH_OPS_H */

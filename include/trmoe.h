/*
 * trmoe — MI355X (gfx950) HIP implementation of tr-infer's MoE block behind a C ABI.
 *
 * Drop-in for the CPU MoE path of tokenring-ai/tr-infer: the router, top-k / cumulative-mass
 * routing, the token-to-expert dispatch, the Q4_K/Q6_K SwiGLU experts against int8-quantised
 * activations, the shared expert with its sigmoid gate, and the combine.  Results follow the
 * reference's CPU arithmetic (per-block f32 epilogue, FMA chains, accumulation order).
 *
 * Conventions (mirroring the kernel contracts of crates/tr-kernels/src in the reference):
 *   - every pointer argument is a DEVICE pointer unless stated otherwise; the caller owns all
 *     buffers (the reference preallocates workspaces at load, exec.rs:733-779);
 *   - `stream` is a hipStream_t (0 = the null stream); all work is stream-ordered and
 *     asynchronous unless a function says it synchronises;
 *   - functions return a trk_status; the reference's asserts/panics (gemv.rs:35, quant.rs:68-71,
 *     router.rs:75) become TRK_E_INVALID and MoePolicy::validate errors (router.rs:32-44) become
 *     TRK_E_POLICY, with the message in trk_last_error();
 *   - nothing here allocates device memory except trk_create.
 */
#ifndef TRMOE_H
#define TRMOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TRK_ABI_VERSION 4
#define TRK_MOE_K_MAX 32 /* router.rs:6 MOE_K_MAX */

typedef enum {
    TRK_OK = 0,
    TRK_E_INVALID = -1,  /* bad shape / pointer / codec: the reference asserts */
    TRK_E_POLICY = -2,   /* MoePolicy::validate (router.rs:32-44) */
    TRK_E_CAPACITY = -3, /* more rows than the context was created for */
    TRK_E_HIP = -4,      /* a HIP runtime call failed */
    TRK_E_NOMEM = -5,
    TRK_E_TIMEOUT = -6   /* a device-side wait of the one-launch decode layer gave up (bounded spin):
                            the outputs of the calls since the last trk_get_stats are invalid */
} trk_status;

enum { TRK_FMT_Q5_1 = 7, TRK_FMT_Q8_0 = 8, TRK_FMT_Q4_K = 12, TRK_FMT_Q6_K = 14 }; /* GGML type ids (python/trpack/blocks.py:11) */
/* The reference's packed TQ codecs (crates/tr-format/src/codec.rs:1-46, Codec {bits, kb}):
 * fmt = bits << 8 | kb.  A TQ matrix is ceil(rows / 16) strips of k / kb blocks, each block
 * d[16] f16 | m[16] f16 | q | (5-bit) high-bit plane, exactly as trpack writes it. */
enum {
    TRK_FMT_TQ4_16 = 0x410, TRK_FMT_TQ4_32 = 0x420, TRK_FMT_TQ5_16 = 0x510,
    TRK_FMT_TQ5_32 = 0x520, TRK_FMT_TQ8_16 = 0x810, TRK_FMT_TQ8_32 = 0x820
};
enum { TRK_BASIS_ALL = 0, TRK_BASIS_TOP = 1 }; /* MassBasis (router.rs:9-16) */

/* A stack of `count` weight matrices [rows][k], `stride` bytes apart.  Replaces
 * tr_model::weights::TqMat {ptr, rows, k, codec, count, stride} (crates/tr-model/src/weights.rs:
 * 14-35); `fmt` says how the bytes are laid out:
 *   - a TQ codec (TRK_FMT_TQ*): the reference's packed strips exactly as trpack writes them, a
 *     pack's TensorKind::Tq entry uploaded unchanged.  register() (weights.rs:207-210) fills
 *     rows, k, codec, count and stride from the manifest entry (manifest.rs:65-94): pass the same
 *     values, with fmt = bits << 8 | kb.  Gate/up take a kb-32 codec, downs a kb-16 codec (the
 *     activations' block sizes).  16-byte aligned (every TQ block is a multiple of 16 bytes).
 *   - a GGUF block format read in place on the GPU (the CPU path reads its TQ re-layout):
 *     gate/up Q4_K; down (routed and shared alike) Q4_K, Q6_K, Q8_0 or Q5_1 (blocks.py:57-78);
 *     row-major rows of superblocks.  Q4_K, Q8_0 and Q5_1 stacks are 16-byte aligned, Q6_K 2-byte.
 * tile_stride: bytes from one tile's tensor to the next in a layer packed for n_tiles > 1 tiles
 * (trk_cfg): tile t's tensor (the pack's entry for tile t) starts at ptr + t * tile_stride, and
 * rows / k give ONE tile's shape (gate/up [n_ff / T][H], down [H][n_ff / T], python/trpack/
 * plan.py:106-118).  Ignored with one tile. */
typedef struct {
    const void *ptr;
    uint32_t rows, k;
    uint32_t fmt;
    uint32_t count;
    uint64_t stride;
    uint64_t tile_stride;
} trk_mat;

/* One layer's MoE weights. Replaces tr_model::exec::MoeW (crates/tr-model/src/exec.rs:86-96). */
typedef struct {
    const float *router;      /* [E][H] f32 (ffn_gate_inp); packed for T > 1 tiles: the tiles'
                                 K-split slices back to back, [T][E][H / T] (plan.py:174-181) */
    const float *router_bias; /* [E] f32 or NULL: additive logit bias for synthetic load skew;
                                 the reference has no bias (pass NULL for its semantics) */
    const float *shexp_gate;  /* [H] f32 (ffn_gate_inp_shexp) */
    trk_mat gate, up, down;   /* routed experts: gate/up [F][H] (Q4_K), down [H][F] (Q4_K|Q6_K) */
    trk_mat sh_gate, sh_up, sh_down; /* shared expert, count 1 */
} trk_moe_w;

/* Cumulative-mass routing. Replaces tr_kernels::router::MoePolicy (router.rs:18-30). */
typedef struct {
    uint32_t min, max;
    float mass;
    uint32_t basis;
} trk_moe_policy;

/* Layer shape and workspace sizing (ModelConfig, crates/tr-model/src/config.rs:5-99). */
typedef struct {
    uint32_t hidden;           /* H (multiple of 256) */
    uint32_t n_expert;         /* E (<= 1024) */
    uint32_t n_ff;             /* F, per routed and shared expert (a multiple of 256 for GGUF
                                  experts, of 16 per tile for TQ experts) */
    uint32_t n_expert_used;    /* k of the fixed top-k routing (<= 32) */
    uint32_t m_max;            /* most rows one call may carry (the reference's batch_max) */
    uint32_t k_cap;            /* most experts one token may select, sizes the entry buffers
                                  (0 = n_expert_used; a policy's max must not exceed it) */
    uint32_t router_dot_max_m; /* batch logits use the per-row dot order when M < this, else the
                                  gemm_f32_nt order (exec_batch.rs:989-1019: the reference
                                  switches at its tile's core count); 0 = 16 */
    int32_t hiprec;            /* M == 1: two-level activations (TR_HIPREC, exec.rs:782) */
    uint32_t n_tiles;          /* T, the tiles the pack was written for (ModelConfig::n_tiles,
                                  plan.py:88): 0 or 1 = one.  With T > 1 (TQ experts only) the
                                  router is K-split and every expert is split by n_ff into T
                                  tiles, as trpack shards them; the layer then sums the tiles'
                                  router partials and down partials in tile order (exchange.rs:
                                  122-136), as the reference's tiles do */
    uint32_t n_expert_packed;  /* experts in the pack (ModelConfig::n_expert_packed, a subset
                                  pack of the first experts, exec.rs:1545-1549): routed ids are
                                  folded onto them (fold_ids, exec_batch.rs:214-225); 0 = n_expert */
} trk_cfg;

/* Replaces tr_model::exec::MoeStats counters rows/experts (exec.rs:558-605). */
typedef struct {
    uint64_t rows, experts;
} trk_moe_stats;

typedef struct trk_ctx trk_ctx;

/* ---- layer-level entry points ---------------------------------------------------------- */

/* Allocate the device workspaces for cfg (Model::load_with sizing, exec.rs:733-779) on the
 * current HIP device. */
int trk_create(const trk_cfg *cfg, trk_ctx **out);
int trk_destroy(trk_ctx *ctx);

/* Switch the routing policy; NULL = the fixed top-n_expert_used.
 * Replaces Model::set_moe (exec.rs:619-625). */
int trk_set_moe(trk_ctx *ctx, const trk_moe_policy *policy);

/* out[M][H] = MoE(x[M][H]).  M == 1 follows Model::moe_block (exec.rs:1540-1623, with the S5
 * router dot of exec.rs:1003-1011); M >= 2 follows Model::moe_batch (exec_batch.rs:1404-1580,
 * with the router of exec_batch.rs:989-1019).  rlog: [M][E] precomputed logits or NULL to
 * compute them from w->router.  Replaces both call sites' worker-side bodies (one call per layer
 * from one host thread instead of an SPMD pool run). */
int trk_moe_forward(trk_ctx *ctx, const trk_moe_w *w, const float *x, const float *rlog, uint32_t m,
                    float *out, void *stream);

/* The device workspace, in bytes, that the layer needs for m rows of this configuration: what
 * trk_create allocates for m_max = m, and what trk_moe_forward_noalloc needs of its static scratch.
 * Host-only (no GPU call); errors as for trk_create.  Sizing helper for callers that preallocate,
 * as Model::load_with sizes its arenas (exec.rs:733-779, exec_batch.rs:127-211). */
int trk_workspace_bytes(const trk_cfg *cfg, uint32_t m, size_t *bytes);

/* Config-5 layer: h[M][H] += MoE(rmsnorm(h; rms_w, eps)).  Composes elem::rmsnorm
 * (elem.rs:255-262), the MoE block and elem::add_inplace (elem.rs:104-118).  Below the router
 * GEMM threshold (and with the one-launch decode layer off) the logits launch normalises h as it
 * reads it, with the same bits as a separate rmsnorm; otherwise rmsnorm runs as its own launch. */
int trk_moe_residual(trk_ctx *ctx, const trk_moe_w *w, const float *rms_w, float eps, float *h,
                     uint32_t m, void *stream);

/* trk_moe_forward without a context and without allocating anything: no counterpart in the
 * reference.  For callers that cannot allocate (code under HIP graph capture, serving loops or
 * harnesses that forbid hipMalloc).  cfg gives the layer shape as for trk_create (m_max is
 * ignored: the workspace is laid out for this call's m), policy the routing (NULL = top
 * n_expert_used).  The workspace lives in a static device array of TRK_NOALLOC_SCRATCH_BYTES per
 * GPU, held until the process ends; a call whose workspace does not fit returns TRK_E_CAPACITY (at
 * H = 2048, E = 512, F = 512, k = 10 that is M above 100; trk_workspace_bytes gives the need of any
 * shape).  Every call on one GPU shares that array:
 * calls that overlap on one GPU (several host threads or streams) race.  MoeStats are not counted
 * and the one-launch decode layer is not used.  Results are those of trk_moe_forward. */
#define TRK_NOALLOC_SCRATCH_BYTES (16u << 20)
int trk_moe_forward_noalloc(const trk_cfg *cfg, const trk_moe_policy *policy, const trk_moe_w *w, const float *x,
                            const float *rlog, uint32_t m, float *out, void *stream);

/* Read (and optionally reset) the routing counters, ordered after the work queued on `stream`
 * (synchronises that stream only).  Returns TRK_E_TIMEOUT, with the counters filled, when a
 * device-side wait of the one-launch decode layer timed out since the last call (and clears that
 * flag): the outputs of those calls are invalid.  Replaces MoeStats::snapshot (exec.rs:593-595). */
int trk_get_stats(trk_ctx *ctx, trk_moe_stats *out, int reset, void *stream);

/* Router-mass profiling: MoeStats::profile_start (exec.rs:567-573) zeroes the profile and turns it
 * on; every later forward then adds each row's router::mass_profile (router.rs:152-166: the
 * cumulative softmax mass of its best 1..32 experts, fixed point 1e-6) to it, as
 * MoeStats::profile_row (exec.rs:582-592) does.  trk_profile_report (exec.rs:575-581) writes the
 * mean cumulative mass of the best k experts, k = 1..32, to cum[32] (host memory) and the number of
 * profiled rows to *rows, ordered after `stream` (synchronises it); on = 0 in trk_profile_start
 * turns profiling off. */
int trk_profile_start(trk_ctx *ctx, int on, void *stream);
int trk_profile_report(trk_ctx *ctx, double *cum, uint64_t *rows, void *stream);

/* Message of the last error on this thread (static storage). */
const char *trk_last_error(void);

/* ---- kernel-level entry points (mirrors of tr-kernels, on caller buffers) --------------- */

/* Router logits rlog[m][E] = router . x[m] (+ bias): gemm_order 0 = attn::dot per row
 * (attn.rs:329-357), 1 = smallgemm::gemm_f32_nt (smallgemm.rs:8-59).  Also the shared-gate
 * logit sh[m] = dot(shexp_gate, x[m]) when shexp_gate is not NULL. */
int trk_router_logits(const float *router, const float *bias, const float *shexp_gate, const float *x,
                      uint32_t m, uint32_t n_expert, uint32_t hidden, int gemm_order, float *rlog,
                      float *sh, void *stream);

/* The hyper-connection mix of the FFN input, part B (tr_model::exec::HcW {up}, exec.rs:49-55):
 * up = the low-rank up projection [hc * hidden][lr] in a kb-32 TQ codec, hc streams (1..8), low
 * rank lr (a multiple of 32, at most 1024).  A batch call keeps the quantised lo rows (1.375 lr
 * bytes per row, rows rounded up to 16) in the context's per-entry output rows, which hold at least
 * 4 (k + 1) m_max hidden bytes; a call beyond them returns TRK_E_CAPACITY. */
typedef struct {
    trk_mat up;
    uint32_t hc, lr;
} trk_hc_w;

/* out[M][H] = MoE(mixed) where mixed is the MoE input the hyper-connection mix produces from the
 * normed streams xn[M][hc][H] (hc_mix_a's output) and the low-rank projection lo[M][lr] summed
 * over tiles: Model::hc_mix_b (exec.rs:1196-1234) + the S5 router + moe_block at M = 1 (two-level
 * lo with hiprec), hc_b_batch (exec_batch.rs:929-1019) + moe_batch at M >= 2, on one tile.  The
 * mix runs as the layer's input stage (one launch at M = 1; at M >= 2 a quantisation of lo, then
 * the mix); the router then reads the mixed rows. */
int trk_moe_forward_hc(trk_ctx *ctx, const trk_moe_w *w, const trk_hc_w *hc, const float *xn, const float *lo,
                       uint32_t m, float *out, void *stream);

/* Per-row routing: route_topk (router.rs:106-113) or, with a policy, route_mass
 * (router.rs:118-148).  ids/w: [m][32], n_sel: [m]. */
int trk_route(const float *logits, uint32_t m, uint32_t n_expert, uint32_t k, const trk_moe_policy *policy,
              uint32_t *ids, float *w, uint32_t *n_sel, void *stream);

/* int8 activation quantisation per kb-block (kb 16 or 32): QActRef::quantize_into
 * (quant.rs:36-48); pair != 0 quantises ONE row into (coarse, residual) rows, quantize_pair_into
 * (quant.rs:50-53).  q [m or 2][k], scale/sum [m or 2][k/kb]. */
int trk_quantize(const float *x, uint32_t m, uint32_t k, uint32_t kb, int pair, int8_t *q, float *scale,
                 int32_t *sum, void *stream);

/* y[rows[i] * ldy + r] (+)= W_item[r] . x_i for the rows r of 16-row strips [s0, s1) and int8
 * activation rows x: gemv_tq_rows / gemm_tq_rows (gemv.rs:16-78) with w = the strip-s0 pointer of
 * matrix `item`.  Any number of activation rows (gemm_tq_rows' chunking is internal); logical
 * rows are written in order, so a row map with repeats accumulates as the reference's does.
 *   w->fmt  a TQ codec (kb must equal the codec's, gemv.rs:27; k a multiple of kb), or a GGUF
 *           block format (k a multiple of 256) read as its TQ conversion: Q4_K with kb 32 or 16,
 *           Q6_K with kb 16, Q8_0 / Q5_1 with kb 32 or 16 (blocks.py:57-113);
 *   s1      at most ceil(rows / 16).  TQ writes every row of each strip (zero padding rows
 *           included, as the reference's 16-wide stores do); GGUF writes rows < w->rows;
 *   pair    rows come in (coarse, residual) pairs, m counts physical rows;
 *   rows    NULL = identity (logical row i to y row i).
 * q: 16-byte aligned, [m][k]; scale / sum: [m][k / kb]. */
int trk_gemv(const trk_mat *w, uint32_t item, uint32_t s0, uint32_t s1, uint32_t kb, const int8_t *q,
             const float *scale, const int32_t *sum, uint32_t m, int pair, float *y, uint32_t ldy,
             const uint32_t *rows, int accumulate, void *stream);

/* ---- routing by scores, and 8-bit products with a scale per token and per channel -------- */
/* No counterpart in the reference, whose router knows trk_route's rules and whose weights and
 * activations carry a scale per 16 or 32 values.  These serve layers whose experts or dense
 * projections are int8 matrices with one scale per output channel, multiplied with activation rows
 * quantised as a whole, and routers that choose by sigmoid scores, a balance bias or groups:
 *
 *   trk_route_scores -> trk_experts_plan -> trk_quantize_rows (x) -> trk_experts_up_i8
 *                    -> trk_quantize_rows (h) -> trk_experts_down_i8
 *
 * Element types of the floating arrays: */
enum { TRK_DT_F32 = 0, TRK_DT_BF16 = 1, TRK_DT_F16 = 2 };

enum { TRK_SCORE_SOFTMAX = 0, TRK_SCORE_SIGMOID = 1 };

/* How trk_route_scores chooses.  k experts per token (1..32, at most n_expert); score: softmax over
 * the row's experts, or the sigmoid of each logit.  n_group (1..32) equal groups of neighbouring
 * experts, of which the topk_group best may be chosen from (n_group = topk_group = 1: no groups);
 * a group is worth the sum of its group_top (1 or 2) best experts' keys.  renorm: the chosen
 * experts' scores are divided by their sum; factor: what every weight is multiplied with. */
typedef struct {
    uint32_t k, score;
    uint32_t n_group, topk_group, group_top;
    int32_t renorm;
    float factor;
} trk_score_policy;

/* Per-row routing by scores.  Expert e's key is its score plus bias[e] (bias NULL: the order of the
 * logits); the k largest keys of the kept groups are chosen, in descending order, the lower index
 * first among equal ones, and weighted by their scores, without the bias.  Keys, group sums and
 * weights are computed as if in 64 bits, the weights then rounded once.  An expert whose logit or
 * key is NaN or -inf is never chosen: a row chooses fewer than k, or none, where the others run out.
 * By its logit it adds nothing to the softmax's sum either; by its bias alone it does.
 * ids / w: [m][32], n_sel: [m]; slots n_sel .. k - 1 get id 0xffffffff and weight 0, later ones stay
 * as they were.  A softmax row with a logit of +inf has NaN scores: nothing is chosen where they enter
 * the choice (a bias, or groups by the sum of two), else by the logits, with NaN weights.
 * n_expert at most 1024. */
int trk_route_scores(const float *logits, const float *bias, uint32_t m, uint32_t n_expert,
                     const trk_score_policy *policy, uint32_t *ids, float *w, uint32_t *n_sel, void *stream);

/* A stack of `count` int8 matrices [rows][k]: matrix i's row r is the k bytes at
 * ptr + i * stride + r * ld, and stands for scale[i * rows + r] times them.  ptr, ld and (count > 1)
 * stride are multiples of 16; rows are read in 16-byte pieces, so the bytes behind a row's k-th up
 * to the next multiple of 16 have to be there (any value).  k at most 131071: every product
 * of two rows then fits its 32-bit sum.  rows, and the tokens of trk_gemm_i8, at most 2^32 - 256. */
typedef struct {
    const int8_t *ptr;
    const float *scale;
    uint32_t rows, k, count;
    uint64_t ld, stride; /* bytes */
} trk_i8_mat;

/* Rows quantised as a whole: scale[i] = max |x[i]| / 127, q[i][j] = 127 x[i][j] / max |x[i]| rounded
 * to the nearest integer, ties to even, as if computed exactly.  x: [m][k] of type `dtype`, rows ldx
 * elements apart; q: rows ldq bytes apart, only the k bytes of each written.  A row whose largest
 * magnitude is under 127 * 2^-126 (its scale would be no normal number) gets scale 0 and zeros; one
 * with a NaN or an infinity gets scale NaN and zeros, which makes every product of it NaN. */
int trk_quantize_rows(const void *x, uint32_t dtype, uint64_t ldx, uint32_t m, uint32_t k, int8_t *q, uint64_t ldq,
                      float *scale, void *stream);

/* y[i][r] = scale[i] * w.scale[r] * sum_j q[i][j] w[r][j] (+ bias[r]) (+ y[i][r] with accumulate),
 * for every row r of matrix `item`: the sum is an exact integer, the scaling in 32 bits, rounded to
 * y's type once.  q: rows ldq bytes apart, laid out as a trk_i8_mat's; y: rows ldy elements apart;
 * bias: [rows] or NULL. */
int trk_gemm_i8(const trk_i8_mat *w, uint32_t item, const int8_t *q, uint64_t ldq, const float *scale, uint32_t m,
                const float *bias, void *y, uint32_t dtype, uint64_t ldy, int accumulate, void *stream);

/* The products of each token with the experts it was routed to.  ids / w [m][32] and n_sel [m] as
 * trk_route, trk_route_scores or the caller leaves them; `slots` (1..32) of each row are looked at.
 * Slot j of token t is an entry where j < n_sel[t] and ids[t][j] is below the stack's count (an
 * expert that lives elsewhere is passed over); its row of h is t * slots + j.
 *
 * plan: the entries sorted by expert, of trk_experts_plan_words words, made by trk_experts_plan for
 * the same ids, n_sel, m, slots and n_expert (= the stacks' count).  Up to TRK_EXPERTS_DIRECT_M tokens it has
 * 0 words: the products take their entries one by one, and no plan (NULL).  A plan made for another m, slots
 * or n_expert is not followed: every entry's row of h, and of y every token's that has one, are NaN.  (One made for
 * more experts is where m * slots does not exceed the stacks' count; the experts beyond are passed over.) */
#define TRK_EXPERTS_DIRECT_M 8
int trk_experts_plan_words(uint32_t m, uint32_t slots, uint32_t n_expert, uint64_t *words);
int trk_experts_plan(const uint32_t *ids, const uint32_t *n_sel, uint32_t m, uint32_t slots, uint32_t n_expert,
                     uint32_t *plan, void *stream);

/* h[t * slots + j][F] = silu(g) * u of every entry, g and u the products of row t of q with its expert's gate and
 * up rows (as trk_gemm_i8, in 32 bits), rounded once to `dtype`; rows of h that are no entry's stay as they were. */
int trk_experts_up_i8(const trk_i8_mat *gate, const trk_i8_mat *up, const int8_t *q, uint64_t ldq, const float *scale,
                      uint32_t m, const uint32_t *ids, const uint32_t *n_sel, uint32_t slots, const uint32_t *plan,
                      void *h, uint32_t dtype, uint64_t ldh, void *stream);

/* y[t] (+)= sum_j w[t][j] * (product of h row t * slots + j, quantised to q / scale, with its
 * expert's down rows) over the token's entries, in slot order, in 32 bits; a token without entries
 * gets zeros.  work: trk_experts_down_work_bytes of device memory, 16-byte aligned (NULL where that is 0). */
int trk_experts_down_work_bytes(uint32_t m, uint32_t slots, uint32_t n_expert, uint32_t rows, uint64_t *bytes);
int trk_experts_down_i8(const trk_i8_mat *down, const int8_t *q, uint64_t ldq, const float *scale, uint32_t m,
                        const uint32_t *ids, const float *w, const uint32_t *n_sel, uint32_t slots,
                        const uint32_t *plan, void *work, void *y, uint32_t dtype, uint64_t ldy, int accumulate,
                        void *stream);

/* ---- microscaled 4-bit rows: their products, dense and for experts, and a whole layer ---- */
/* No counterpart in the reference.  For layers whose experts or dense projections are 4-bit floating point with a
 * power of two for each 32 neighbours of a row, multiplied with activation rows in the same form:
 *
 *   trk_route_scores -> trk_experts_plan -> trk_quantize_mx4 (x) -> trk_experts_up_mx4
 *                    -> trk_quantize_mx4 (h) -> trk_experts_down_mx4
 *
 * or, for up to TRK_EXPERTS_DIRECT_M tokens and with activations that stay as they are, trk_moe_mx4.  The two differ by the
 * rounding of x and h to 4 bits: a program that goes from one to the other with the size of its batch gets other results.
 * Experts are SwiGLU without biases or clamps.  Shared experts go through the calls above as further entries of every token:
 * their ids and weights behind the chosen ones, n_sel and slots by as many more.
 *
 * A row of k values is ceil(k / 32) blocks of 16 bytes, two values a byte, the first in the low four bits; the last block's
 * values behind the k-th are zeros.  A value's four bits are a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A block's scale is
 * a byte s that stands for 2^(s - 127); with s = 255 (NaN) the block's values, and every product of the row, are NaN.
 * Rows of values begin at multiples of 16 bytes, rows of scales at multiples of 4; scales are read in 4-byte pieces, so the bytes
 * behind a row's last up to the next multiple of 4 have to be there (any value). */

/* A stack of `count` 4-bit matrices [rows][k]: matrix i's row r has its values at ptr + i * stride + r * ld, its scales at
 * scale + i * scale_stride + r * scale_ld (all in bytes; the strides count where count > 1).  k at most 2^30, rows, and the
 * tokens of trk_gemm_mx4, at most 2^32 - 256. */
typedef struct {
    const uint8_t *ptr, *scale;
    uint32_t rows, k, count;
    uint64_t ld, stride;
    uint64_t scale_ld, scale_stride;
} trk_mx4_mat;

/* Rows to 4-bit values: a block's scale is 2^e, e = floor(log2 max |x|) - 2, held to -127 from below; its values x / 2^e are
 * rounded to the nearest of the sixteen, ties to the even one of two neighbours (0.25 to 0, 0.75 to 1, 1.25 to 1, 1.75 and
 * 2.5 to 2, 3.5 and 5 to 4), magnitudes above 6 to 6, with x's sign.  A block of zeros gets scale byte 0; one with a NaN or an
 * infinity gets 255, and zeros.  x: [m][k] of type `dtype`, rows ldx elements apart; whole blocks of q are written,
 * and ceil(k / 32) scale bytes a row. */
int trk_quantize_mx4(const void *x, uint32_t dtype, uint64_t ldx, uint32_t m, uint32_t k, uint8_t *q, uint64_t ldq,
                     uint8_t *scale, uint64_t scale_ld, void *stream);

/* What 4-bit rows stand for: y [m][k] of type `dtype`, rows ldy elements apart, rounded once. */
int trk_dequantize_mx4(const uint8_t *q, uint64_t ldq, const uint8_t *scale, uint64_t scale_ld, uint32_t m, uint32_t k,
                       void *y, uint32_t dtype, uint64_t ldy, void *stream);

/* y[i][r] = sum_j q[i][j] w[r][j] (+ bias[r]) (+ y[i][r] with accumulate), for every row r of matrix `item`: products
 * and a block's sum of them are exact, blocks are added in 32 bits, y's type is rounded to once.  y: rows ldy elements
 * apart; bias: [rows] or NULL. */
int trk_gemm_mx4(const trk_mx4_mat *w, uint32_t item, const uint8_t *q, uint64_t ldq, const uint8_t *scale,
                 uint64_t scale_ld, uint32_t m, const float *bias, void *y, uint32_t dtype, uint64_t ldy, int accumulate,
                 void *stream);

/* trk_experts_up_i8 and trk_experts_down_i8 for 4-bit stacks and rows: entries, plan, h, y and work (of
 * trk_experts_down_work_bytes) are theirs.  Up takes rows and slots of which (rows / 16 rounded up) * slots is at most 2^32. */
int trk_experts_up_mx4(const trk_mx4_mat *gate, const trk_mx4_mat *up, const uint8_t *q, uint64_t ldq,
                       const uint8_t *scale, uint64_t scale_ld, uint32_t m, const uint32_t *ids, const uint32_t *n_sel,
                       uint32_t slots, const uint32_t *plan, void *h, uint32_t dtype, uint64_t ldh, void *stream);
int trk_experts_down_mx4(const trk_mx4_mat *down, const uint8_t *q, uint64_t ldq, const uint8_t *scale,
                         uint64_t scale_ld, uint32_t m, const uint32_t *ids, const float *w, const uint32_t *n_sel,
                         uint32_t slots, const uint32_t *plan, void *work, void *y, uint32_t dtype, uint64_t ldy,
                         int accumulate, void *stream);

/* A MoE layer on 4-bit experts.  The stacks hold n_expert routed experts, then n_shared (0..32) that every token takes:
 * gate / up [n_expert + n_shared][F][H], down [n_expert + n_shared][H][F].  router: [n_expert][H], or NULL where each call
 * brings its logits; bias: trk_route_scores', or NULL; shared_gate: [H], the shared experts are weighted with
 * sigmoid(shared_gate . x), or NULL, with 1. */
typedef struct {
    const float *router, *bias, *shared_gate;
    trk_mx4_mat gate, up, down;
    uint32_t n_shared;
} trk_moe_mx4_w;

/* y[t] = sum_j w_j down_j (silu(gate_j x[t]) * up_j x[t]) over the experts that trk_route_scores chooses by the router's
 * logits (rlog [m][n_expert] where it is given, else router . x in 32 bits), in that order, then the shared ones.  Up to
 * TRK_EXPERTS_DIRECT_M tokens (more: TRK_E_CAPACITY), hidden size and width up to 2^24.  Activations are not quantised: x, h
 * and every sum are as 32 bits hold them (a value to 2^-26 of the largest of its 32, and to 2^-129; a sum whose terms'
 * magnitudes add up to half of 2^128 or more may overflow), y is rounded to once.  A token with a NaN or an infinity in x
 * gets a row of NaN, also where no expert is chosen; an expert whose h has either gives NaN.
 * x: rows ldx elements apart, of type xdtype; y: rows ldy apart, of type ydtype.  work: trk_moe_mx4_work_bytes of device memory,
 * 16-byte aligned, of any content; calls that may overlap need one each.  k: the policy's. */
int trk_moe_mx4_work_bytes(const trk_moe_mx4_w *w, uint32_t k, uint32_t m, uint64_t *bytes);
int trk_moe_mx4(const trk_moe_mx4_w *w, const trk_score_policy *policy, const void *x, uint32_t xdtype, uint64_t ldx,
                const float *rlog, uint32_t m, void *work, void *y, uint32_t ydtype, uint64_t ldy, void *stream);

/* y = silu(g) * u (elem::swiglu_vec, elem.rs:173-175) over n floats. */
int trk_swiglu(const float *g, const float *u, float *y, size_t n, void *stream);

/* y[m][n] = rmsnorm(x[m][n]; w, eps) (elem.rs:255-262). */
int trk_rmsnorm(const float *x, const float *w, float eps, uint32_t m, uint32_t n, float *y, void *stream);

/* y[i] += a[i] (elem.rs:104-118). */
int trk_add_inplace(float *y, const float *a, size_t n, void *stream);

/* ---- synthetic data (bit-identical to the test oracle's generator) ---------------------- */
/* GGUF superblocks of a [rows][k] matrix: d (and dmin) ~ U(dlo, dhi) as f16, all other bytes
 * uniform; fmt Q4_K, Q6_K, Q8_0 or Q5_1 (Q8_0 / Q5_1: every block's d, Q5_1 m = -16 U). */
int trk_gen_gguf(uint32_t fmt, uint64_t seed, uint64_t stream_id, uint32_t rows, uint32_t k, float dlo,
                 float dhi, void *out, void *stream);
/* The same for a stack of `count` matrices `stride` bytes apart, matrix e drawing from stream
 * stream0 + e * stream_step (one launch; what trk_gen_gguf gives per matrix). */
int trk_gen_gguf_stack(uint32_t fmt, uint64_t seed, uint64_t stream0, uint64_t stream_step, uint32_t count,
                       uint32_t rows, uint32_t k, float dlo, float dhi, void *out, uint64_t stride, void *stream);
/* n normals N(0, sigma) (Box-Muller in double, rounded to f32). */
int trk_gen_normal(uint64_t seed, uint64_t stream_id, size_t n, double sigma, float *out, void *stream);

/* ---- measurement and introspection ------------------------------------------------------ */
/* M == 1: run the whole layer as one launch when the layer's shape has a fused kernel and the GPU
 * can hold its grid at once (on), or as the three launches router / gate-up / down (off, the
 * default).  Both follow exec.rs:1540-1623 with identical results; no counterpart in the
 * reference, whose decode layer is one pool run. */
int trk_set_fusion(trk_ctx *ctx, int on);

/* M >= 2: grouped work items (one expert's entry rows, at most 16) of at most `rows` rows run on
 * the streaming GEMV kernels, larger ones on the int8 MFMA tiles.  rows = -1 (the default) picks
 * 16 for M <= 16 (every item streams), 4 while M * k_cap <= 2 * n_expert, else 0 (every item on
 * the tiles).  Every choice gives the same bits (moe_batch, exec_batch.rs:1404-1580); no
 * counterpart in the reference, which runs one grouped kernel per expert matrix. */
int trk_set_stream_rows(trk_ctx *ctx, int rows);

/* 2 <= M <= rows (default 8, 0..16): every token runs as a decode (its routing inside its gate/up
 * workgroups, its rows added by the down launch in the batch combine's order: shared expert
 * first, then ascending expert), three launches with no dispatch, grouped items or combine.  GGUF
 * layers with one tile; TQ layers where the decode kernels take the shape (the real one: kb-32
 * gate/up, kb-16 down, one tile, k_cap <= 15).  The same bits as the grouped path
 * (exec_batch.rs:1404-1580); the dispatch arrays (TRK_WS_ENT_*, items) are then not written.
 * No counterpart in the reference. */
int trk_set_decode_rows(trk_ctx *ctx, int rows);

/* Layers on TQ experts: the int8 MFMA kernels (on, the default, where H / 32 units of staged
 * activations fit a workgroup's LDS) or the generic grouped TQ GEMV (off).  Both give the same
 * bits; no counterpart in the reference. */
int trk_set_tq_mfma(trk_ctx *ctx, int on);

/* Per-kernel timing (the HIP counterpart of the reference's TR_PROFILE laps, exec.rs:344-430):
 * when on, every kernel a forward launches is bracketed by HIP events on the call's stream. */
int trk_set_timing(trk_ctx *ctx, int on);
/* Sum of the recorded durations per kernel since the last call, then forget them (synchronises).
 * Fills up to cap entries (kernel name, total ms, launches); returns the number of kernels. */
int trk_get_timing(trk_ctx *ctx, const char **names, double *ms, uint64_t *launches, int cap);

/* Launch only the kernel `name` (a name trk_get_timing reports) of the forward sequence for
 * (w, x, rlog, m, out), on the workspace as the previous calls left it.  For timing one kernel in
 * isolation (bench.py; the reference's kbench, crates/tr-kernels/benches): the results are only
 * meaningful when the calls before it prepared the workspace for the same inputs. */
int trk_launch_kernel(trk_ctx *ctx, const trk_moe_w *w, const float *x, const float *rlog, uint32_t m,
                      float *out, const char *name, void *stream);

/* Copy an internal workspace buffer of the last forward to host memory. */
enum {
    TRK_WS_RLOG = 1,     /* [M][E] f32 */
    TRK_WS_IDS = 2,      /* [M][32] u32 */
    TRK_WS_W = 3,        /* [M][32] f32 */
    TRK_WS_NSEL = 4,     /* [M] u32 */
    TRK_WS_ENT_TOK = 5,  /* [n_ent] u32 */
    TRK_WS_ENT_W = 6,    /* [n_ent] f32 */
    TRK_WS_ENT_EXP = 7,  /* [n_ent] u32 */
    TRK_WS_GRP_START = 8,/* [n_groups+1] u32 */
    TRK_WS_GRP_EXP = 9,  /* [n_groups] u32 */
    TRK_WS_NGROUPS = 10, /* [2] u32: n_groups, n_ent */
    TRK_WS_XQ = 11,      /* [rows][H] i8 (pair: 2 rows) */
    TRK_WS_XS = 12,      /* [rows][H/32] f32 */
    TRK_WS_ACTQ = 13,    /* activation rows of the down input, i8 */
    TRK_WS_ACTS = 14,    /* their folded scales, f32 */
    TRK_WS_SHLOGIT = 15, /* [M] f32: dot(shexp_gate, x) */
    TRK_WS_BARRIER_ERR = 16, /* u32: nonzero if a one-launch decode layer ever timed out at a grid barrier */
    TRK_WS_MIXED = 17    /* [M][H] f32: the MoE input trk_moe_forward_hc mixed */
};
/* Ordered after the work queued on `stream` (synchronises that stream only). */
int trk_debug_read(trk_ctx *ctx, int which, void *host_dst, size_t bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif

/* strixite_amd: MI355X (gfx950, CDNA4, wave64) kernels for strixite's MTP verify path, behind a C ABI.
 *
 * Every entry point is asynchronous on the caller's HIP stream (passed as `sx_stream`, a hipStream_t) unless it says
 * otherwise, takes plain device pointers and sizes, and returns SX_OK (0) or an error code; sx_last_error() returns the
 * calling thread's message for the last failure. Preconditions are checked on the host before any launch (the
 * reference's STRIX_CHECK set); data-dependent failures go to 3-word device error slots (first writer wins) and NaN
 * outputs, as in the reference. Nothing here allocates device memory: callers pass workspaces sized by the
 * *_workspace_bytes functions.
 *
 * Each declaration names the reference interface it replaces (file:line in TheBeaninator/strixite). The C++ shim that
 * gives the reference's own kernels/ *.hpp signatures on top of these is strixite_amd/integration/strix_kernels_shim.cpp.
 */
#ifndef STRIXITE_AMD_H
#define STRIXITE_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void *sx_stream; /* hipStream_t */

enum sx_status { SX_OK = 0, SX_EINVAL = 1, SX_EHIP = 2, SX_EUNSUPPORTED = 3 };

/* Activation dtype: strix::kernels::Act (kernels/norm.hpp:20), F32 or BF16 raw bits. */
enum sx_act { SX_ACT_F32 = 0, SX_ACT_BF16 = 1 };

/* strix::kernels::MoeMath (kernels/moe_grouped.hpp:35). On gfx950 all three run the MFMA path on exact codes with
 * FP32 accumulation (F32 semantics: the tightest of the three); the value is accepted for API compatibility. */
enum sx_moe_math { SX_MOE_F32 = 0, SX_MOE_WMMA_BF16 = 1, SX_MOE_WMMA_F16 = 2 };

/* Q4DeviceView (runtime/q4_device.hpp:13-18) / Q8DeviceView (runtime/q8_device.hpp:12-17): non-owning device views of
 * a [N, K] weight in the formats/q4.hpp:3-6 / q8.hpp:3-11 layout. q: N*K/2 (q4, low nibble = even k) or N*K (q8) bytes,
 * 16-byte aligned; scale, minv: [N, K/G] BF16 bits; G in {32, 64, 128}; w = code * scale + min. */
typedef struct sx_qview {
    const uint8_t *q;
    const uint16_t *scale;
    const uint16_t *minv;
    int64_t N, K, G;
} sx_qview;

const char *sx_last_error(void);
const char *sx_version(void);

/* ---- dense dequantizing GEMV/GEMM: y[M, N] = x[M, K] * deq(W)^T, FP32 accumulation, one rounding at the store ----
 * kernels/linear_q4.hpp:26-30 and kernels/linear_q8.hpp:13-14. out_act == act, or BF16 x -> F32 y. */
int sx_linear_q4(const void *x, const sx_qview *w, void *y, int64_t M, int act, int out_act, sx_stream stream);
int sx_linear_q8(const void *x, const sx_qview *w, void *y, int64_t M, int act, int out_act, sx_stream stream);
/* The kernel such a call runs on a device of `cus` compute units (<= 0: the current device), without running it: "k_split",
 * "register_tiles", "wide_tiles_k_split", "wide_tiles" or "qmm"; NULL for a view or width no call takes (sx_last_error).
 * For tests and profiles; no reference counterpart. */
const char *sx_linear_kernel(const sx_qview *w, int bits, int64_t M, int act, int out_act, int cus);
/* The same for the grouped expert calls (gather, its SwiGLU form, combine): "register_tiles", "wide_tiles" or "qmm". */
const char *sx_experts_grouped_kernel(const sx_qview *w, int64_t E, int64_t M, int64_t A, int act, int cus);

/* ---- per-slot MoE experts (decode / short verify), kernels/linear_q4.hpp:32-58 ----
 * w: E experts stacked [E*N, K]; ids [M, A] int32 device. err: >= 3 zeroed uint32 (device).
 *   gather:         y[m, a, :] = x[m, :] * W[ids[m, a]]^T                          (linear_q4.hpp:42-43)
 *   gather_swiglu:  h[m, a, j] = silu(g) * u over rows [gate (I) | up (I)]          (linear_q4.hpp:55-56)
 *   combine:        y[m, :] = sum_a coef[m, a] * (h[m, a, :] * W[ids[m, a]]^T)      (linear_q4.hpp:44-46) */
int sx_linear_q4_experts_gather(const void *x, const sx_qview *w, int64_t E, const int32_t *ids, int64_t M, int64_t A,
                                void *y, int act, uint32_t *err, sx_stream stream);
int sx_linear_q4_experts_gather_swiglu(const void *x, const sx_qview *w, int64_t E, const int32_t *ids, int64_t M,
                                       int64_t A, void *h, int act, uint32_t *err, sx_stream stream);
int sx_linear_q4_experts_combine(const void *h, const sx_qview *w, int64_t E, const int32_t *ids, const float *coef,
                                 int64_t M, int64_t A, void *y, int act, uint32_t *err, sx_stream stream);
/* report_expert_error (kernels/linear_q4.hpp:61): the 3 words already on the host; SX_EINVAL + message if set. */
int sx_report_expert_error(const uint32_t e[3], const char *what);

/* ---- MoE router, kernels/moe_router.hpp:33-43 ----
 * Top k of E logits per token (value desc, lower index on a tie), coef = softmax over the k (FP32); optional shared
 * slot k with id shared_id and coef sigmoid(shared logit). Non-finite logit: ids -1, coef NaN, err {1, token, expert}.
 * k in 1..min(E, 32); E in 1..1024. */
int sx_moe_router(const void *logits, int64_t ld, int64_t M, int64_t E, int64_t k, const void *shared_logit,
                  int64_t shared_ld, int32_t shared_id, int32_t *ids, float *coef, int act, uint32_t *err,
                  sx_stream stream);
/* report_router_error (kernels/moe_router.hpp:43). */
int sx_report_router_error(const uint32_t e[3], const char *what);
/* moe_shared_add / moe_shared_add_inject (kernels/moe_router.hpp:53-63). */
int sx_moe_shared_add(void *y, const void *s, const float *gate_logit, int64_t gate_ld, int64_t M, int64_t N,
                      uint32_t gate_index, int act, uint32_t *err, sx_stream stream);
int sx_moe_shared_add_inject(void *y, const void *s, const float *gate_logit, int64_t gate_ld, int64_t M, int64_t N,
                             uint32_t gate_index, void *x, const float *w_in, int64_t H, int act, uint32_t *err,
                             sx_stream stream);

/* ---- grouped MoE experts (verify width and prefill), kernels/moe_grouped.hpp:42-62 ----
 * moe_group_routes buckets the M*A slots by expert into ws (int32 layout of moe_grouped.hip:63-81: header [n_tiles,
 * S, E, n_wtiles], offsets [E+2], slots [S], 16-slot tiles, 64-slot tiles); slot order within a bucket is unspecified
 * and no output depends on it. Bad ids go to bucket E and set err {1, id, slot}. */
int sx_moe_route_workspace_bytes(int64_t M, int64_t A, int64_t E, size_t *bytes);
int sx_moe_group_routes(const int32_t *ids, int64_t M, int64_t A, int64_t E, void *ws, size_t ws_bytes, uint32_t *err,
                        sx_stream stream);
/* moe_router (no shared slot) then moe_group_routes in one launch, for M*k <= 2048: the same ids, coef, error words
 * and workspace as those two calls (kernels/moe_router.hpp:38-40 + kernels/moe_grouped.hpp:47-49, the sequence
 * runtime/qwen4exp.cpp:1139-1147 runs at verify width). No reference counterpart as one call. */
int sx_moe_router_group(const void *logits, int64_t ld, int64_t M, int64_t E, int64_t k, int act, int32_t *ids,
                        float *coef, uint32_t *router_err, void *ws, size_t ws_bytes, uint32_t *expert_err,
                        sx_stream stream);
/* ---- verify-width MoE FFN in two launches (after the router projection) ----
 * The sequence runtime/qwen4exp.cpp:1139-1163 runs below kGroupedMinTokens - moe_router (moe_router.hpp:38-40),
 * linear_q4_experts_gather_swiglu (linear_q4.hpp:55-56), linear_q4_experts_combine (linear_q4.hpp:44-46) - with the
 * same ids, coef, h, y and error words; no reference counterpart as two calls. q4 G = 128, BF16 activations;
 * M <= 16, M * A <= 64 (A = k + 1 with a shared slot), gate_up K in {512 .. 4096}, down K in {1024, 2048};
 * sx_moe_verify_supported says whether a shape qualifies (SX_OK) or why not. Ew: experts stacked in the weights
 * (E, or E + 1 with the shared expert stacked). A repeated id within a token counts as an invalid slot. */
int sx_moe_verify_supported(int64_t M, int64_t A, int64_t E, int64_t k, int64_t Ew, const sx_qview *gate_up,
                            const sx_qview *down, int act);
/* route (ids, coef [M, A]; router_err) + h [M, A, I] = silu(x W_gate^T) * (x W_up^T) per slot (expert_err, NaN rows
 * for invalid slots). shared_logit nullable. h_sums (nullable, 16-byte aligned): FP32 [M * A, ceil(I / 16)], the sum
 * of each 16-feature run of the valid slots' h rows as stored, for sx_moe_verify_down. sync (nullable): a buffer of
 * sx_moe_verify_layer_sync_bytes bytes as sx_moe_verify_layer takes it (zeroed once, one per stream, may be the same
 * buffer): with K = 4096 each compute unit then streams a fixed run of about 4/5 of an equal share of the weight
 * tiles and takes the rest from a shared pool, so faster ones take more (without it each takes a fixed equal
 * share); the outputs are the same either way. plan (nullable): a device buffer of SX_VERIFY_PLAN_BYTES bytes,
 * 16-byte aligned, that receives the launch's routing in the form sx_moe_verify_down takes it. */
#define SX_VERIFY_PLAN_BYTES 4096
int sx_moe_verify_gate_up(const void *x, int64_t M, const float *logits, int64_t ld, int64_t E, int64_t k,
                          const float *shared_logit, int64_t shared_ld, int32_t shared_id, const sx_qview *gate_up,
                          int64_t Ew, int32_t *ids, float *coef, void *h, float *h_sums, int act,
                          uint32_t *router_err, uint32_t *expert_err, void *sync, void *plan, sx_stream stream);
/* y [M, N] = sum_a coef[m, a] * (h[m, a] W_down[ids[m, a]]^T); NaN rows for tokens with an invalid slot. h_sums
 * (nullable): the h_sums sx_moe_verify_gate_up wrote with this h (saves the kernel summing h itself). plan
 * (nullable): the plan sx_moe_verify_gate_up wrote with these ids and coef; the launch then takes the routing from
 * it (ids and coef are not read) instead of rebuilding the expert list, so its first weight loads go out sooner. */
int sx_moe_verify_down(const void *h, const float *h_sums, int64_t M, int64_t A, const int32_t *ids,
                       const float *coef, const sx_qview *down, int64_t Ew, void *y, int act, uint32_t *expert_err,
                       const void *plan, sx_stream stream);
/* ---- the whole verify-width MoE sublayer in one launch ----
 * runtime/qwen4exp.cpp:1132-1163 below kGroupedMinTokens - the router projection (linear_bf16w, kernels/linear.hpp:19-24,
 * or an FP32 weight), moe_router (moe_router.hpp:38-40), linear_q4_experts_gather_swiglu (linear_q4.hpp:55-56) and
 * linear_q4_experts_combine (linear_q4.hpp:44-46) - as one kernel whose phases hand over through counters in `sync`
 * instead of kernel boundaries; no reference counterpart as one call. wr: router weight [rows, d], FP32 (wr_act F32)
 * or BF16 bits; logits [M, rows] FP32 are written; shared != 0: slot k is expert shared_id with coefficient
 * sigmoid(logits[m, E]) (rows >= E + 1). ids, coef, h, h_sums, y, router_err, expert_err as sx_moe_verify_gate_up /
 * sx_moe_verify_down. Shapes: those sx_moe_verify_supported takes, with d = 4096 and E <= 1024. sync: a device buffer
 * of sx_moe_verify_layer_sync_bytes bytes, 16-byte aligned, zeroed once by the caller; one per stream: launches that
 * overlap in time must not share it. The launch runs one block per compute unit and needs them resident together; a
 * phase that waits more than 20 ms for another (another kernel holding compute units that long) gives up and sets
 * expert_err {1, 0xFFFFFFFE, phase} instead of hanging. */
int sx_moe_verify_layer_sync_bytes(size_t *bytes);
/* Diagnostic: a device buffer of (compute units x 16) uint64 that later sx_moe_verify_layer launches (any thread) fill
 * with each block's phase timestamps (s_memrealtime, 100 MHz): [0] start, [1] projection items done, [2] logits
 * fresh (wave 0), [8] tokens routed, [9] expert list built, [3] first gate_up weight loads issued, [4] gate_up done,
 * [5] h complete, [6] h staged, [7] end; and two counts: [10] polls of the logits, [11] gate_up rounds taken. NULL
 * turns it off (the default). No reference counterpart: the
 * reference's tracing (common/trace.hpp) marks host-side launch ranges, which cannot show phases inside a launch. */
int sx_moe_verify_layer_trace(uint64_t *buf);
int sx_moe_verify_layer(const void *x, int64_t M, const void *wr, int wr_act, int64_t rows, int64_t E, int64_t k,
                        int shared, int32_t shared_id, const sx_qview *gate_up, const sx_qview *down, int64_t Ew,
                        float *logits, int32_t *ids, float *coef, void *h, float *h_sums, void *y, int act,
                        uint32_t *router_err, uint32_t *expert_err, void *sync, sx_stream stream);
/* y [M, A, N] (linear_q4_experts_gather_grouped, moe_grouped.hpp:53-55). */
int sx_linear_q4_experts_gather_grouped(const void *x, const sx_qview *w, int64_t E, const void *ws, size_t ws_bytes,
                                        int64_t M, int64_t A, void *y, int act, int math, sx_stream stream);
/* y [M, N]; partial: M*A*N FP32 scratch (linear_q4_experts_combine_grouped, moe_grouped.hpp:60-62). */
int sx_linear_q4_experts_combine_grouped(const void *h, const sx_qview *w, int64_t E, const int32_t *ids,
                                         const float *coef, const void *ws, size_t ws_bytes, float *partial, int64_t M,
                                         int64_t A, void *y, int act, int math, sx_stream stream);
/* Grouped gather with the SwiGLU epilogue: h [M, A, N/2] = swiglu(gather_grouped(x)), bit-identical to
 * sx_linear_q4_experts_gather_grouped followed by sx_swiglu. No single reference counterpart: it fuses the two calls
 * runtime/qwen4exp.cpp:1154-1156 makes. */
int sx_linear_q4_experts_gather_swiglu_grouped(const void *x, const sx_qview *w, int64_t E, const void *ws,
                                               size_t ws_bytes, int64_t M, int64_t A, void *h, int act,
                                               sx_stream stream);

/* ---- SwiGLU, kernels/swiglu.hpp:21: gu [rows, 2I] -> h [rows, I]; BF16: h = bf16(bf16(silu(g)) * u). ---- */
int sx_swiglu(const void *gu, void *h, int64_t rows, int64_t I, int act, sx_stream stream);

/* ---- dense FP32-weight projection: y[M, N] (F32) = x[M, K] (act) * W[N, K]^T. The router logits of the
 * benchmark's MoE layers (fp32 Wr); plays the role kernels/linear.hpp linear_bf16w plays at runtime/qwen4exp.cpp:1132-1137. ---- */
int sx_linear_f32w(const void *x, const float *W, int64_t N, int64_t K, float *y, int64_t M, int act,
                   sx_stream stream);

/* ---- BF16-weight linear, kernels/linear.hpp:14-24 (linear_bf16w) and kernels/linear_wmma.hpp:25-28
 * (linear_bf16w_wmma): y[M, N] = x[M, K] * W^T, W [N, K] raw BF16 bits row-major, FP32 accumulation, one rounding at
 * the store; out_act == act, or BF16 x -> F32 y (the router logits of the served model: W [E + 1, d], the shared
 * expert's gate in the last row, runtime/qwen4exp.cpp:1132-1137). y must not overlap x. _wmma: x rounded to BF16
 * before the products, K % 64 == 0 and 16-byte aligned x and W (its prefill contract). ---- */
int sx_linear_bf16w(const void *x, const uint16_t *w, void *y, int64_t M, int64_t N, int64_t K, int act, int out_act,
                    sx_stream stream);
int sx_linear_bf16w_wmma(const void *x, const uint16_t *w, void *y, int64_t M, int64_t N, int64_t K, int act,
                         int out_act, sx_stream stream);

/* ---- logits top-k, kernels/logits_topk.hpp:26-46 ----
 * Per row the best k (value desc, lower id on a tie; -0 ties +0) of ids [0, n_valid); NaN left out and flagged in
 * nan[row]; optional allow mask [rows, mask_words]; padding (-inf, INT32_MAX). k in 1..64 (the reference: 20). */
typedef struct sx_logit_cand {
    float v;
    int32_t id;
} sx_logit_cand; /* LogitCand, kernels/logits_topk.hpp:29-33 */
int sx_logits_topk_workspace_bytes(int64_t rows, int64_t n_valid, int64_t k, size_t *bytes);
int sx_logits_topk(const float *logits, int64_t rows, int64_t ld, int64_t n_valid, int64_t k, sx_logit_cand *out,
                   uint32_t *nan, void *workspace, size_t workspace_bytes, const uint32_t *mask, int64_t mask_words,
                   sx_stream stream);
/* sx_logits_topk without a workspace argument and without allocating: the level candidates live in a fixed scratch
 * array of SX_TOPK_SCRATCH_BYTES the library holds on each device it runs on (until the process ends). No counterpart
 * in the reference: it is for callers that cannot allocate (HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc). The same outputs as sx_logits_topk; SX_EINVAL when sx_logits_topk_workspace_bytes for the shape
 * exceeds the scratch (e.g. 64 rows of 248,320 logits at k = 64 still fit). Calls on one device share the scratch:
 * two that overlap in time (different streams) race. */
#define SX_TOPK_SCRATCH_BYTES (4u << 20)
int sx_logits_topk_noalloc(const float *logits, int64_t rows, int64_t ld, int64_t n_valid, int64_t k,
                           sx_logit_cand *out, uint32_t *nan, const uint32_t *mask, int64_t mask_words,
                           sx_stream stream);

/* ---- the MTP draft head's Q4 copy of the Q8 LM head: formats/q4_from_q8.hpp:17-27 (quantize_q4_from_q8), which
 * runtime/qwen4exp.cpp:192-238 runs on the host at load; here on the device, from the resident Q8 rows ----
 * src: a Q8 view [N, K] (its first N rows: a row prefix of the head); G: the Q4 group (32, 64, 128; the served draft
 * head uses 64); q [N, K/2], scale / minv [N, K/G] BF16: the Q4 weight, byte-identical to the reference's. A
 * non-finite dequantized value (the reference throws) sets err {1, row, first k of its group} and that group's scale,
 * min and codes to zero. */
int sx_quantize_q4_from_q8(const sx_qview *src, int64_t G, uint8_t *q, uint16_t *scale, uint16_t *minv,
                           uint32_t *err, sx_stream stream);

/* ---- MTP draft pick, kernels/mtp_pick.hpp:20-33: top-2 + NaN flag + the forward's error words, one 64-byte block.
 * emb_err points at the 8-byte EmbeddingError slot (kernels/embedding.hpp:26-28). ---- */
typedef struct sx_mtp_pick_s {
    int32_t best;
    float best_v, second_v;
    uint32_t nan;
    uint32_t err[9];
    uint32_t pad;
    unsigned long long emb;
} sx_mtp_pick_t;
int sx_mtp_pick(const float *logits, int64_t n, const uint32_t *router_err, const uint32_t *expert_err,
                const uint32_t *attn_err, const unsigned long long *emb_err, sx_mtp_pick_t *out, sx_stream stream);
/* The same pick (kernels/mtp_pick.hpp:20-33, the same output bit for bit) read by many blocks at once, one launch:
 * each block reduces its run of the logits to a top-2 in `workspace` and the last block to finish merges them.
 * workspace: device, 16-byte aligned, sx_mtp_pick_ws_bytes long, ZEROED before its first use (it holds a counter that
 * every call leaves ready for the next). Calls that share a workspace must be ordered on one stream. */
int sx_mtp_pick_ws_bytes(int64_t n, size_t *bytes);
/* The MTP draft head's LM head and pick in one launch (runtime/qwen4exp.cpp:1408-1413: the head's logits, then
 * kernels::mtp_pick over them): logits[N] = x[1, K] (BF16) . deq(w)^T in FP32 as sx_linear_q4 / q8 write them, and
 * `out` the pick of those logits, bit-identical to sx_mtp_pick's. bits 4 or 8; workspace as sx_mtp_pick_ws's (zeroed
 * before its first use). Shapes the fused GEMV does not take run sx_linear_q4 / q8 and then sx_mtp_pick_ws. */
int sx_mtp_head_pick(const void *x, const sx_qview *w, int bits, float *logits, const uint32_t *router_err,
                     const uint32_t *expert_err, const uint32_t *attn_err, const unsigned long long *emb_err,
                     sx_mtp_pick_t *out, void *workspace, size_t workspace_bytes, sx_stream stream);
int sx_mtp_pick_ws(const float *logits, int64_t n, const uint32_t *router_err, const uint32_t *expert_err,
                   const uint32_t *attn_err, const unsigned long long *emb_err, sx_mtp_pick_t *out, void *workspace,
                   size_t workspace_bytes, sx_stream stream);

/* ---- logits top-k and acceptance in one launch (the verify tail after the LM head) ----
 * sx_logits_topk (kernels/logits_topk.hpp:35-46) followed by sx_mtp_accept (serve/engine.cpp:592-653 with
 * serve/sampler.cpp:183-248), as one kernel whose blocks hand over through counters in `workspace`; no reference
 * counterpart as one call. cands / nan: as sx_logits_topk's out / nan (k = kc), for every row. out (nullable: top-k
 * only): as sx_mtp_accept's, for drafts [k] (rows >= k + 1). workspace: sx_verify_tail_workspace_bytes bytes, 8-byte
 * aligned, ZEROED before its first use (it holds counters each launch leaves at zero); one per stream. Rows of more
 * than 262,144 logits are refused (sx_logits_topk takes them). */
int sx_verify_tail_workspace_bytes(int64_t rows, int64_t n_valid, int64_t kc, size_t *bytes);
int sx_verify_tail(const float *logits, int64_t rows, int64_t ld, int64_t n_valid, int64_t kc, sx_logit_cand *cands,
                   uint32_t *nan, const uint32_t *mask, int64_t mask_words, const int32_t *drafts, int64_t k,
                   const double *u, double temperature, int64_t top_k, double top_p, int32_t *out, void *workspace,
                   size_t workspace_bytes, sx_stream stream);
/* ---- draft acceptance on the device: serve/engine.cpp:592-610 with Sampler semantics (serve/sampler.cpp:183-248) ----
 * cands [k+1, kc] (from sx_logits_topk, value desc), nan [k+1], drafts [k] (device). Row j is sampled (greedy:
 * candidate 0; else temperature -> top_k (<= kc) -> top_p -> draw r = u[j] * kept, u[j] a host draw of
 * std::generate_canonical<double, 53> from the engine's mt19937_64, in order), accepting while the sample equals
 * drafts[j]. Writes out[0] = j (0..k), out[1] = status (0, or 1 + the row whose sampling failed: NaN or non-finite top
 * logit), out[2 .. 2+j] = the j+1 tokens committed (the accepted drafts, then row j's sample: the correction, or row
 * k's when all were accepted). Draws consumed on the host side: 0 (greedy) or j+1 (j on failure). */
int sx_mtp_accept(const sx_logit_cand *cands, const uint32_t *nan, int64_t kc, const int32_t *drafts, int64_t k,
                  const double *u, double temperature, int64_t top_k, double top_p, int64_t n_valid, int32_t *out,
                  sx_stream stream);

/* ---- a verify layer's attention half: norm with FP8 output, FP8 linear, attention of drafted tokens over a paged
 * cache, append to that cache. No reference counterparts (its attention, kernels/attention.hpp, reads a contiguous
 * BF16 cache and one chain of tokens; its norm, kernels/norm.hpp, has no 8-bit output). ---- */
/* r = x + residual (rounded to act, stored to residual_out), y = r / sqrt(mean(r^2) + eps) * (weight + w_add).
 * x [M, K] with row stride ldx; residual (nullable: r = x), residual_out, y (nullable) [M, K] and weight [K] in act; q
 * (nullable) [M, K] e4m3 codes of y with scale [M, K / 128] FP32 = amax(|y|) / 448 of each run of 128 features: the
 * activations sx_linear_fp8 takes. A run of zeros has scale 0 and codes 0; a run that holds NaN comes out NaN.
 * K a multiple of 128, up to 32768. y may be x or the residual, residual_out the residual or x, row for row. */
int sx_add_rms_norm_fp8(const void *x, int64_t ldx, const void *residual, const void *weight, int64_t M, int64_t K,
                        float eps, float w_add, void *residual_out, void *y, uint8_t *q, float *scale, int act,
                        sx_stream stream);

/* An FP8 weight: q [N, K] e4m3 (OCP) row-major, 16-byte aligned; scale [ceil(N / 128), K / 128] FP32, one for each
 * 128 x 128 tile; w = code * scale. K a multiple of 128. */
typedef struct sx_fp8_view {
    const uint8_t *q;
    const float *scale;
    int64_t N, K;
} sx_fp8_view;
/* y[M, N] (out_act) = x * w^T with x [M, K] e4m3 codes (16-byte aligned) and x_scale [M, K / 128] FP32; blocks of 128
 * are summed in FP32, one rounding at the store. FP32 outputs: products exact, sums FP32 inside a block too. BF16 outputs:
 * inside a block the FP8 matrix instruction, which cuts the products of eight neighbouring codes at 2^-13 of the largest
 * one's power of two (codes under 2^-6 counting as 2^-6): an error of 2^-10 sum |x w| at most for normal codes, 1.4e-5 of
 * the result (rms) for random ones; where large products cancel, small ones beside them are lost. */
int sx_linear_fp8(const uint8_t *x, const float *x_scale, const sx_fp8_view *w, void *y, int64_t M, int out_act,
                  sx_stream stream);

/* BF16 rows of heads: element [t, h, d] at p[t * token + h * head + d] (with layers: + l * layer). Strides in
 * elements, multiples of 8; p 16-byte aligned. A slice of a packed query / key / value projection is one. */
typedef struct sx_head_rows {
    void *p;
    int64_t token, head, layer;
} sx_head_rows;
enum sx_kv_dtype { SX_KV_BF16 = 0, SX_KV_E4M3 = 1 };
/* A paged cache of keys and values: position p of sequence b is row p % page_size of page table[b, p / page_size],
 * at k[layer * k_layer + page * k_page + row * k_token + head * k_head + d] (strides in elements, multiples of 16
 * bytes, any order; v alike). page_size a power of two, 16 to 65536. table [batch, pages_per_seq] with row stride
 * table_ld and lens [batch] (cached tokens) are device int32. E4M3: value = code * k_scale (v_scale), both 2^-100 to
 * 2^100. */
typedef struct sx_kv_cache {
    void *k, *v;
    int32_t dtype;
    float k_scale, v_scale;
    int64_t pages, page_size, heads, dim, layers;
    int64_t k_page, k_token, k_head, k_layer;
    int64_t v_page, v_token, v_head, v_layer;
    const int32_t *table;
    int64_t table_ld, pages_per_seq;
    const int32_t *lens;
    int64_t batch;
} sx_kv_cache;
/* Attention of drafted tokens: sequence b's are rows starts[b] .. starts[b + 1] - 1 (device int32 [batch + 1]) of q
 * [T, Hq, dim], k_new and v_new [T, heads, dim]; none to max_new (1..256) of them, T (under 2^24) bounds them all. Token t sees
 * every cached token of its sequence and, of the drafted ones, number j of the sequence where bit j % 64 of
 * mask[t * mask_ld + j / 64] is set (its ancestors and itself for a tree; a chain: all up to itself). out = softmax(
 * scale * q k^T) v per query head h over key head h / (Hq / heads); a row that sees nothing is zero. A drafted token
 * that a row does not see does not touch it, NaN and infinities included (an infinite value that it sees may come out as
 * NaN). Scores, maxima and sums are FP32; softmax terms meet BF16 values to 2^-17 where max_new * Hq / heads <= 64 and
 * rounded to BF16 above, E4M3 values in FP16 (2^-12; 2^-32 of a row's maximum and less may be lost). lse (nullable) [T,
 * Hq] FP32: the natural logarithm of each row's sum of exp(score). Rows behind starts[batch] are left as they are. dim 64, 128 or 256; Hq a
 * multiple of heads; batch up to 1024. ws: sx_tree_attention_workspace_bytes bytes, 16-byte aligned, its contents
 * never read before they are written; one per stream. out, lse and ws lie apart from each other and from all that is read
 * (out may be a slice of the buffer that holds q). A sequence with impossible words (a length its table does not
 * hold, a run of tokens that is negative, over max_new or outside T) or a page outside the cache is not read: its
 * rows come out NaN (none, where the run itself is impossible) and err (nullable) is {1, the length or page, the
 * sequence}. */
int sx_tree_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, size_t *bytes);
int sx_tree_attention(const sx_head_rows *q, const sx_head_rows *k_new, const sx_head_rows *v_new, int64_t T, int64_t Hq,
                      const sx_kv_cache *cache, const int32_t *starts, int64_t max_new, const uint64_t *mask,
                      int64_t mask_ld, float scale, const sx_head_rows *out, float *lse, void *ws, size_t ws_bytes,
                      uint32_t *err, sx_stream stream);
/* The accepted tokens into every layer of the cache: for i < count[b] (device int32 [batch], up to max_count), drafted
 * row starts[b] + path[b * path_ld + i] (path null: starts[b] + i) goes to position lens[b] + i. BF16 rows are copied,
 * E4M3 takes the nearest code of x / scale (one FP32 division), saturating at 448. lens is only read; lens_out (nullable, apart from all
 * that is read) gets lens + count. Keys, values (in one
 * buffer, interleaved too) and k_new, v_new lie apart. The pages for
 * the new positions are the caller's to provide, each to one sequence. A sequence
 * with an impossible word (a run of tokens as above, a count over max_count or the table, a path entry outside the
 * sequence's drafted tokens, a page outside the cache) keeps its length and gets nothing; err (nullable) is then {1,
 * the count, path entry or page, the sequence}. */
int sx_kv_append(const sx_head_rows *k_new, const sx_head_rows *v_new, int64_t T, const sx_kv_cache *cache,
                 const int32_t *starts, const int32_t *count, int64_t max_count, const int32_t *path, int64_t path_ld,
                 int32_t *lens_out, uint32_t *err, sx_stream stream);

/* ---- routing by scores (no reference counterpart; sx_moe_router is the reference's) ----
 * s = sigmoid(logit) or the softmax over the E experts, c = s + bias[e] (bias nullable, FP32). With groups > 1 (equal
 * runs of E / groups experts) only the top_groups groups with the largest sum of their group_best (1 or 2) best c stay
 * in the choice. ids: the k largest c, larger first; every tie, of groups too, goes to the lower index. coef = s of
 * the chosen ones (without the bias), divided by their sum if renorm (a sum of zero leaves them zero), times factor.
 * Scores and choices are FP64, coef rounded once. ids and coef lie apart from each other and from all that is read.
 * Shared slot, errors (a non-finite logit or bias; err nullable) and layouts as sx_moe_router's; factor does not touch
 * the shared slot. groups <= 64, k in 1..min(E, 32), E in 1..1024. */
enum sx_score { SX_SCORE_SIGMOID = 0, SX_SCORE_SOFTMAX = 1 };
int sx_moe_router_scored(const void *logits, int64_t ld, int64_t M, int64_t E, int64_t k, int score, const float *bias,
                         int64_t groups, int64_t top_groups, int64_t group_best, int renorm, float factor,
                         const void *shared_logit, int64_t shared_ld, int32_t shared_id, int32_t *ids, float *coef,
                         int act, uint32_t *err, sx_stream stream);

/* Acceptance of drafted tokens against the target's probabilities (rejection sampling; sx_mtp_accept compares a sample with the
 * draft, this keeps what the draft's probabilities allow). Sequence b's rows are starts[b] .. starts[b + 1] - 1 (device int32
 * [batch + 1], none to max_rows, 1..256) of logits [T, >= n_valid] (act, rows ld apart); drafts[t] is the token proposed behind row t
 * (a sequence's last row has none), draft_logits [T, >= n_draft] (nullable: the draft was certain) what it was drawn from,
 * n_draft <= n_valid (the rest of the vocabulary: probability 0). With p, q the softmax of a row of each over temperature[b] and u
 * [T, 2] FP64 in [0, 1): draft d of row t stays if u[t, 0] q(d) < p(d). At the first that does not, a token from max(p - q, 0), behind the
 * last draft one from p: the first place at which the running sum passes u[t, 1] times the total. temperature 0 or less: a draft
 * stays if it is the row's largest logit (ties: the lowest place), which is the token otherwise. Probabilities and sums are FP64,
 * exponentials good to 1e-14 of themselves.
 * tokens [batch, max_rows]: the drafts that stay, the token, then -1; count: how many; status 0. A row that counts and holds NaN or
 * no finite largest logit, a draft outside the vocabulary or a temperature that is not finite: status 1 + the row, count and tokens
 * the drafts before it. Impossible starts (negative, over max_rows, outside T, or behind a start that is below the one before it):
 * status -1, count 0. ws: sx_mtp_accept_sampled_workspace_bytes, 16-byte aligned, never read before it is written; one per
 * stream. T up to 32767, batch up to 1024. */
int sx_mtp_accept_sampled_workspace_bytes(int64_t T, int64_t batch, int64_t n_valid, int64_t n_draft, size_t *bytes);
int sx_mtp_accept_sampled(const void *logits, int64_t ld, int64_t T, int64_t n_valid, const void *draft_logits, int64_t draft_ld,
                          int64_t n_draft, int act, const int32_t *drafts, const int32_t *starts, int64_t batch, int64_t max_rows,
                          const double *u, const float *temperature, int32_t *tokens, int32_t *count, int32_t *status, void *ws,
                          size_t ws_bytes, sx_stream stream);

/* The norms around a block, its gate, the residual and an 8-bit output in one launch; rows of K features in act:
 *   h = x / sqrt(mean(x^2) + eps) * (post + w_add)   over the row, or each run of `group` features (0: the row; else a power of
 *                                                    two, 8..512, that divides K); post null: h = x
 *   h = h * gate, h * silu(gate) or h * sigmoid(gate)   gate rows ld_gate apart (0: one row for all); null: left out
 *   r = residual_scale * residual + branch_scale * h    rounded to act and stored to residual_out; residual null: branch_scale * h
 *   y = r / sqrt(mean(r^2) + eps) * (pre + w_add)       pre null: y = r
 * Outputs: residual_out (with a residual), y (nullable) [M, K] in act, q (nullable) [M, K] int8 codes of y with scale [M] FP32 =
 * amax(|y|) / 127, the activations sx_linear_int8 takes. A code is the nearest whole number, ties to even, to 127 t / amax(|t|) with
 * t = r (pre + w_add) (the second root is in both and cancels; pre null: t = r), where r is as the formulas give it in FP64, in their
 * order: a mean is the sum times the rounded 1 / K, root and quotient are the nearest, and only the order in which squares are
 * added is open. silu and sigmoid are good to 1e-14. A row of zeros has scale 0 and codes 0, one that holds NaN or an infinity scale
 * NaN and codes 0. post has post_len values: K (0 says so too) or the group's. K a multiple of 8, up to 16384. residual_out and y may be x,
 * the residual or the gate, row for row. No reference counterpart. */
enum sx_gate_act { SX_GATE_NONE = 0, SX_GATE_SILU = 1, SX_GATE_SIGMOID = 2 };
typedef struct sx_block_norm {
    const void *x, *post, *gate, *residual, *pre;
    void *residual_out, *y;
    int8_t *q;
    float *scale;
    int64_t ldx, ld_gate, group, post_len;
    int32_t gate_act;
    double eps, w_add, residual_scale, branch_scale;
} sx_block_norm;
int sx_block_norm_int8(const sx_block_norm *p, int64_t M, int64_t K, int act, sx_stream stream);

/* An 8-bit integer weight: q [N, K] int8 row-major, 16-byte aligned, scale [N] FP32, one for each channel; w = code * scale. K a
 * multiple of 16, up to 131056. */
typedef struct sx_int8_view {
    const int8_t *q;
    const float *scale;
    int64_t N, K;
} sx_int8_view;
/* y[M, N] (out_act) = x * w^T with x [M, K] int8 codes (16-byte aligned) and x_scale [M] FP32, one for each token: the codes' sum
 * is exact (32-bit integers), then rounded to FP32, times x_scale, times scale, one more rounding at a BF16 store. No reference
 * counterpart. */
int sx_linear_int8(const int8_t *x, const float *x_scale, const sx_int8_view *w, void *y, int64_t M, int out_act,
                   sx_stream stream);

/* ---- the gated delta rule: layers whose memory is a state and not a cache (no reference counterparts here; its
 * kernels/gdn.hpp runs chains of tokens). A state S [key_dim, dim] FP32 for each of `heads` value heads; for each token
 *   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q.
 * q, k [T, key_heads, key_dim], v [T, heads, dim] BF16; value head h goes with key head h / (heads / key_heads). normalize: k
 * and q are divided by sqrt(sum of squares + 1e-6) first; q is then multiplied by scale. A key whose FP32 sum of squares is not
 * finite is no number, normalized or not, and so is such a query where it is normalized. Gates a, b [T, heads] in gate_act, rows
 * a_token and b_token elements apart: with A_log and dt_bias (FP32 [heads]) g = -exp(A_log) softplus(a + dt_bias) and beta =
 * sigmoid(b); without (both null) g = a (0 or less) and beta = b. A g of -1e4 or less, -inf too, says: forget everything.
 * Sequence b's tokens are rows starts[b] .. starts[b + 1] - 1 (device int32 [batch + 1]); its state is number slot[b] (null: b)
 * of `slots` states, state_slot floats apart, each [heads, key_dim, dim] dense. key_dim 64 or 128, dim a multiple of 16 up to
 * 1024, batch up to 1024. States, sums and norms are FP32. A state enters all its products whole, as three BF16 terms; of a
 * product of two FP32 values (corrections, products of tokens) the six largest of nine products of such terms are taken. A sequence
 * whose run of tokens is impossible (negative, over the call's limit, outside T, or behind a start that is below the one before it) is
 * left alone; one with tokens whose slot is none of the states, or (where states are written) is another such sequence's too, keeps
 * its state and its rows come out NaN. err (nullable) is then {1, the first row or the slot, the sequence}. Sequences of no tokens
 * need no slot. Rows behind starts[batch] are left as they are. */
typedef struct sx_delta {
    sx_head_rows q, k, v;
    const void *a, *b;
    int64_t a_token, b_token;
    const float *A_log, *dt_bias;
    float *state;
    const int32_t *slot, *starts;
    int64_t T, key_heads, heads, key_dim, dim, slots, state_slot, batch;
    int32_t gate_act, normalize;
    float scale;
} sx_delta;
/* Tokens through the states, which are updated in place; out [T, heads, dim] BF16. max_len bounds a sequence's tokens: up to 16
 * they go one by one, in one launch without a workspace (sx_gated_delta_workspace_bytes says 0; ws may be null); above in chunks
 * of 64, two launches, ws 16-byte aligned, its contents never read before they are written, one per stream. A token that is no
 * number makes the rows from it on NaN (a value, or a correction too large for FP32: its column of them), and the state. */
int sx_gated_delta_workspace_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t Dk, int64_t max_len, size_t *bytes);
int sx_gated_delta(const sx_delta *d, int64_t max_len, const sx_head_rows *out, void *ws, size_t ws_bytes, uint32_t *err,
                   sx_stream stream);
/* The same for drafted tokens, whose states must not be kept before it is known which are accepted: the states are only read. A
 * sequence's tokens (none to max_new, 1..64) are a tree, parents first: bit j of mask[t * mask_ld] says that token t goes on from
 * token j of its sequence (bits at and above its own number are not looked at). out as above; u [T, heads, dim] and decay [T, heads]
 * FP32 are what sx_gated_delta_commit takes: u / |k| and g. A token touches only those that see it, NaN included. */
int sx_gated_delta_verify(const sx_delta *d, int64_t max_new, const uint64_t *mask, int64_t mask_ld, const sx_head_rows *out,
                          float *u, float *decay, uint32_t *err, sx_stream stream);
/* The accepted path into the states of all layers: for tokens i < count[b] (device int32 [batch], up to max_count), number
 * path[b * path_ld + i] of the sequence (path null: i), a path from a root down, S <- e^g S + k u^T. k as the verify had it (layer
 * stride: `layer`), u [layers, T, Hv, Dv], decay [layers, T, Hv]; states state_layer floats apart. A sequence with an impossible
 * word (as above; a count below 0 or over max_count or its tokens, a path entry outside them) keeps its states; err (nullable) is
 * then {1, the word, the sequence}. */
int sx_gated_delta_commit(const sx_head_rows *k, const float *u, const float *decay, int64_t layers, int64_t T, int64_t Hk,
                          int64_t Hv, int64_t Dk, int64_t Dv, float *state, int64_t state_layer, int64_t state_slot,
                          int64_t slots, const int32_t *slot, const int32_t *starts, int64_t batch, const int32_t *count,
                          int64_t max_count, const int32_t *path, int64_t path_ld, uint32_t *err, sx_stream stream);

/* ---- strixw weight files: formats/strixw.hpp (the reader, StrixwFile :86-112) and runtime/strixw_loader.hpp (the
 * upload, StrixwDevice :22-52) ----
 * A file is a 128-byte header (magic "STRIXWT\0", format version 1..4, index and data-region offsets, file size, the
 * index's and the header's own strix_hash64), an index (metadata key/value pairs; one record per tensor: name,
 * encoding, shape, group size, experts, source parts, and each component's role, absolute offset, size and hash) and
 * a data region on a 4096-byte boundary: tensors start on 4096-byte boundaries, components on 256-byte ones.
 * Encodings and component roles carry the file's own numbering (formats/strixw.hpp:17-19). */
enum sx_strixw_encoding {
    SX_STRIXW_Q4 = 1, SX_STRIXW_Q4_CHUNK_MAJOR = 2, SX_STRIXW_BF16 = 3, SX_STRIXW_F32 = 4, SX_STRIXW_I64 = 5,
    SX_STRIXW_Q8 = 6, SX_STRIXW_Q8_CHUNK_MAJOR = 7, SX_STRIXW_Q6 = 8, SX_STRIXW_Q5 = 9
};
enum sx_strixw_role { SX_STRIXW_DATA = 0, SX_STRIXW_Q = 1, SX_STRIXW_SCALE = 2, SX_STRIXW_MIN = 3 };

typedef struct sx_strixw sx_strixw; /* an open, validated file (read-only mapping) */

/* StrixwComponent (formats/strixw.hpp:30-33): offset absolute in the file. */
typedef struct sx_strixw_component {
    uint8_t role;
    uint64_t offset, bytes, hash;
} sx_strixw_component;

/* StrixwTensor (formats/strixw.hpp:35-44); name points into the open file and lives as long as it. */
typedef struct sx_strixw_tensor {
    const char *name;
    int32_t encoding, ndim;
    int64_t shape[8];
    int64_t group_size, experts;
    int32_t nparts, ncomp;
    sx_strixw_component comp[4];
} sx_strixw_tensor;

/* strix_hash64 (formats/strixw.hpp:50): the file's 64-bit checksum of n bytes (host memory). */
uint64_t sx_strix_hash64(const void *data, uint64_t n);
/* StrixwFile::StrixwFile (formats/strixw.hpp:88): maps path and validates the header, the index and every record
 * (the same checks, in the same order, as formats/strixw.cpp:398-500); on failure SX_EINVAL with a message naming the
 * file and the problem ("bad magic", "header hash mismatch", "truncated", "components overlap", ...), *out NULL.
 * Host only: no HIP call. */
int sx_strixw_open(const char *path, sx_strixw **out);
void sx_strixw_close(sx_strixw *f);
/* version, file_bytes, data_offset, tensor and metadata counts (any pointer may be NULL). */
int sx_strixw_summary(const sx_strixw *f, uint32_t *version, uint64_t *file_bytes, uint64_t *data_offset,
                      int64_t *tensors, int64_t *meta);
/* StrixwFile::meta() (formats/strixw.hpp:95-96): the i-th pair in the file's key order, or the value of `key`
 * (SX_EINVAL naming the file when absent). Strings live as long as the file. */
int sx_strixw_meta_at(const sx_strixw *f, int64_t i, const char **key, const char **value);
int sx_strixw_meta(const sx_strixw *f, const char *key, const char **value);
/* StrixwFile::find / tensors() (formats/strixw.hpp:97-98): *index = the record's position, or -1 when absent. */
int sx_strixw_find(const sx_strixw *f, const char *name, int64_t *index);
int sx_strixw_tensor_at(const sx_strixw *f, int64_t i, sx_strixw_tensor *out);
/* StrixwPart (formats/strixw.hpp:25-28) of a record: the checkpoint tensor and the rows it fills. */
int sx_strixw_part_at(const sx_strixw *f, int64_t tensor, int64_t part, const char **source, int64_t *row_offset,
                      int64_t *rows);
/* StrixwFile::verify_hashes (formats/strixw.hpp:102): rehashes every component on `threads` host threads; SX_EINVAL
 * naming the first corrupt component in file order. */
int sx_strixw_verify_hashes(const sx_strixw *f, int threads);
/* StrixwDevice::StrixwDevice (runtime/strixw_loader.hpp:27): copies the data region (file_bytes - data_offset bytes)
 * to dst (device memory of at least that size, 256-byte aligned, owned by the caller) through pinned staging slots
 * filled by read_threads (1..64) concurrent pread()s, the copies queued on `stream`. Synchronous: returns once the
 * region is on the device; *seconds (may be NULL) = wall time. Component hashes are not rechecked (the header and
 * index hashes were, at open). */
int sx_strixw_load(const sx_strixw *f, void *dst, uint64_t dst_bytes, int read_threads, double *seconds,
                   sx_stream stream);
/* StrixwDevice::q4 / q8 / qw (runtime/strixw_loader.hpp:36-41): the view of a row-major q4 (bits 4), q8 (8) or either
 * (0) tensor of shape [N, K], checked, with pointers into the region loaded at `base` (base + offset - data_offset),
 * or into the file's mapping when base is NULL. */
int sx_strixw_qview(const sx_strixw *f, const void *base, const char *name, int bits, int64_t N, int64_t K,
                    sx_qview *out);
/* StrixwDevice::bf16 / f32 (runtime/strixw_loader.hpp:46-47), and i64: a dense tensor's data, encoding and shape
 * checked; base as for sx_strixw_qview. */
int sx_strixw_data(const sx_strixw *f, const void *base, const char *name, int encoding, const int64_t *shape,
                   int ndim, const void **out);

/* ---------------- measurement probes (no counterpart in the reference: the ceilings the roofline fractions are
 * judged against, measured on the part) ---------------- */
/* A streaming read of `bytes` (16-byte aligned) by `blocks` blocks of 512 threads, 16-byte loads, nothing stored
 * (sink: 4 bytes, written only in a case the data practically never gives). */
int sx_probe_stream_read(const void *buf, uint64_t bytes, int blocks, uint32_t *sink, sx_stream stream);
/* `blocks` blocks of 4 waves, each wave `iters` x 4 independent v_mfma_f32_32x32x16_bf16; *flops (may be NULL) = the
 * launch's dense BF16 flops. */
int sx_probe_mfma(int blocks, int iters, float *sink, double *flops, sx_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* STRIXITE_AMD_H */

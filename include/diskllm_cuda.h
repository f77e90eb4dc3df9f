/*
 * diskllm_cuda.h -- C ABI of libdiskllm_cuda.so, the B200 (sm_100a) sampler for DiskLLM.
 *
 * Two layers:
 *   1. Drop-in replacements for DiskLLM's sampler.h (include/sampler.h:7-34 in DiskLLM),
 *      declared in this repo's include/sampler.h with identical names and signatures.
 *      Linking libdiskllm_cuda.so instead of compiling src/sampler.c keeps
 *      src/core/sampler_api.c and every caller unchanged.
 *   2. A batched, device-resident entry point (dllm_cuda_sample_batch) that runs the whole
 *      per-row chain of src/core/sampler_api.c:48-63 -- grammar mask, presence,
 *      frequency, repetition, sampler_sample -- for many rows in one launch.
 *
 * Every pointer in dllm_batch_desc is a device pointer unless stated otherwise.  The
 * caller owns all buffers.  Streams are passed as void* (a cudaStream_t).
 */
#ifndef DISKLLM_CUDA_H
#define DISKLLM_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifndef DLLM_API
#if defined(__GNUC__)
#define DLLM_API __attribute__((visibility("default")))
#else
#define DLLM_API
#endif
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    DLLM_OK = 0,
    DLLM_ERR_INVALID_ARG = 1,
    DLLM_ERR_OOM = 2,
    DLLM_ERR_CUDA = 3,
    DLLM_ERR_NCCL = 4,
    DLLM_ERR_TIMEOUT = 5,
    DLLM_ERR_UNSUPPORTED = 6,
} dllm_status;

enum {
    DLLM_DTYPE_F32 = 0,
    DLLM_DTYPE_BF16 = 1,
    DLLM_DTYPE_F16 = 2,   /* dllm_cuda_lmhead_logits's output weights, the int8 and beam calls */
};

/* mode flags */
#define DLLM_MODE_TOPP_SORTED   0x1u  /* sorted-nucleus mode for rows with top-k off and
                                         temperature > 0: entries ordered by (t desc, id asc),
                                         masses rint(expf(t) * 2^42) summed exactly, min-p the
                                         sorted prefix above the threshold, top-p the shortest
                                         prefix reaching top_p of the kept mass, the draw the
                                         first entry whose prefix mass exceeds r * (nucleus
                                         mass).  Not the reference's behaviour (its top-p keeps
                                         an index-order prefix when top-k is off); vocab <= 2^21 */
#define DLLM_MODE_PEN_TRUE_DIV  0x2u  /* positive logits divided by the repetition penalty
                                         (IEEE) instead of multiplied by 1/penalty, which is
                                         what the reference's -ffast-math build computes */
#define DLLM_MODE_MINP_RELATIVE 0x4u  /* min-p keeps p >= min_p * (largest p) instead of the
                                         reference's absolute p >= min_p */

/* Sampling parameters of one row.  Fields mirror DiskLLM's sampler_config
 * (include/sampler.h:10-16) plus the penalties of diskllm_sampler_params
 * (include/diskllm.h:48-56) and the frequency extension. */
typedef struct {
    float temperature;   /* 0 -> greedy (src/sampler.c:140-142) */
    float top_p;         /* >= 1 -> off */
    float min_p;         /* <= 0 -> off; absolute threshold as in src/sampler.c:188-202 */
    int   top_k;         /* <= 0 or >= vocab -> off */
    float repetition;    /* <= 1 -> off (src/sampler.c:21-33, src/core/sampler_api.c:59) */
    float presence;      /* 0 -> off (src/sampler.c:35-52, src/core/sampler_api.c:55) */
    float frequency;     /* 0 -> off; not in the reference: x -= (float)count * frequency,
                            applied after presence, before repetition */
} dllm_sampler_params;

typedef struct {
    int rows;                 /* batch rows */
    int vocab;                /* columns of logits (= vocabulary) */
    int64_t row_stride;       /* elements between consecutive rows (>= vocab) */
    int dtype;                /* DLLM_DTYPE_F32 or DLLM_DTYPE_BF16 (upcast exactly) */
    const void *logits;       /* [rows][row_stride] */

    const uint32_t *mask;     /* grammar allow-mask or NULL: bit (i & 31) of word (i >> 5)
                                 set = token i allowed; cleared -> -INFINITY, the effect of
                                 diskllm_grammar_apply_mask (src/core/grammar.c:275-308) */
    int64_t mask_stride;      /* words between rows (>= (vocab + 31) / 32) */

    const int32_t *hist_ids;  /* token history, CSR; NULL = none */
    const int64_t *hist_off;  /* [rows + 1] offsets into hist_ids */
    int hist_max;             /* upper bound on any row's history length (host value) */

    const float *uniforms;    /* [rows] draws in [0, 1), one per row */

    dllm_sampler_params params;            /* host value, used for every row ... */
    const dllm_sampler_params *row_params; /* ... unless this device array is given */
    int topk_max;             /* upper bound on top_k over rows when row_params is given.
                                 Any top_k works (as in the reference, src/sampler.c:165-170);
                                 rows with top_k above 1024 take a slower sort-based pass */

    unsigned flags;           /* DLLM_MODE_* */

    int32_t *token;           /* [rows] out: sampled token id */
    float *probs;             /* optional [rows][probs_stride] out: final draw probability
                                 of every token (0 outside the draw list) */
    int64_t probs_stride;
    float *pen_logits;        /* optional [rows][pen_stride] out: logits after mask and
                                 penalties (what the reference leaves in its logits array) */
    int64_t pen_stride;
    int32_t *status;          /* optional [rows] out: 0 or DLLM_ROW_ERR_* bits */
    int32_t *topk_ids;        /* optional [rows][topk_stride] out: the top-k ids, best first
                                 (rows where top-k is active) */
    int64_t topk_stride;

    void *workspace;          /* optional device scratch of >= dllm_cuda_workspace_bytes()
                                 bytes (256-byte aligned); NULL: the library keeps one
                                 buffer per (device, stream) and grows it with cudaMalloc.
                                 Several host threads may call with NULL at once, on one
                                 stream too, and with cudaStreamPerThread each has its own
                                 buffer.  A buffer given here serves one call at a time */
    size_t workspace_bytes;
} dllm_batch_desc;

/* per-row status bits */
#define DLLM_ROW_ERR_HIST_TABLE 1   /* more distinct history ids than the table holds */
#define DLLM_ROW_ERR_NONFINITE  2   /* a NaN among a top-k row's candidates: the reference's
                                       -ffast-math build leaves its order undefined.  (Rows with
                                       +inf, all-NaN rows and NaN rows with top-k off get the
                                       reference's id: its list's last entry) */
#define DLLM_ROW_ERR_TOPK_LARGE 4   /* a top_k dllm_cuda_merge_sample cannot serve (above its
                                       gathered k); whole-row calls serve every top_k */
#define DLLM_ROW_ERR_WALK       8   /* internal consistency check of the draw failed */
#define DLLM_ROW_ERR_TIMEOUT   16   /* a bounded wait on a bulk copy expired */
#define DLLM_ROW_TOPP_EDGE     32   /* information, not an error: the index-order top-p prefix
                                       at the cut, or just before it, lies within
                                       top_p * (one ulp of (float)(1/sum) + 6e-8) of the
                                       threshold.  The reference's exponentials (glibc's scalar
                                       and vector expf) differ from this library's by a few ulp,
                                       so its (float)(1/sum) can be one ulp away and, on such a
                                       row only, its cut one entry earlier or later
                                       (src/sampler.c:204-222); its probabilities and id follow
                                       that cut */

/* Samples every row of the batch on `stream` (stream-ordered; returns after the launch).
 * Replaces, per row, the sequence of src/core/sampler_api.c:48-63:
 *   diskllm_grammar_apply_mask -> sampler_apply_presence_penalty ->
 *   sampler_apply_repetition_penalty -> sampler_sample.
 * Row i draws with uniforms[i] where the reference draws rand_f32 (src/sampler.c:225). */
DLLM_API dllm_status dllm_cuda_sample_batch(const dllm_batch_desc *desc, void *stream);

/* Scratch the sampler needs for this descriptor: per-row headers, warp-level draw records and
 * stashed probabilities (the size depends on the vocabulary's launch configuration: about 30 KB
 * per row at vocab 256000), plus the sorted-nucleus passes' and the large-top-k pass's buffers
 * when the descriptor uses them.  0 on invalid descriptors. */
DLLM_API size_t dllm_cuda_workspace_bytes(const dllm_batch_desc *desc);

/* Allocation-free variant of dllm_cuda_sample_batch; it has no counterpart in the reference.
 * For callers that cannot call cudaMalloc -- an embedder whose device memory is all owned by
 * its own allocator, or a decode loop that must not stall on the device-wide synchronisation
 * of cudaMalloc/cudaFree.  Instead of a caller buffer or a library-grown one, it uses a
 * 16 MiB scratch array compiled into the library (held on every GPU that loads the library
 * until the process exits); desc->workspace is ignored.  Batches whose
 * dllm_cuda_workspace_bytes() exceeds 16 MiB (about 550 rows of vocab 256000) are rejected
 * with DLLM_ERR_UNSUPPORTED and a message in dllm_cuda_last_error().  The first call on a
 * device looks up the array's device address and picks the launch configuration, so make it
 * before any stream capture.  The address is kept for the life of the process: after a
 * cudaDeviceReset of a device this entry point must not be called on it again.  Every call shares the one array: calls whose work overlaps on the
 * GPU (other streams, other host threads) race and must be serialised by the caller.  The
 * kernels write every scratch field before reading it, so leftover contents from an earlier
 * call need no clearing. */
DLLM_API dllm_status dllm_cuda_sample_batch_static(const dllm_batch_desc *desc, void *stream);

/* Diagnostics: when given a device array of 32 zeroed unsigned 64-bit counters, the sampler
 * kernels accumulate per-phase cycle counts of each cluster's first CTA and draw-walk
 * statistics into it; NULL switches it off.  No effect on results. */
DLLM_API dllm_status dllm_cuda_set_debug_counters(unsigned long long *device_counters);

/* Test hooks for failure detection (no counterpart in the reference).  Both are off by default
 * and change nothing while off.
 *   dllm_cuda_debug_inject_wait_timeout(site, polls): from the next sampling launch on, the
 *     cluster kernel adds, on each cluster's first row, one bounded wait that nothing completes
 *     (site 1: CTA 0 waits for its slice barrier's next phase after the bulk copy landed; site 2:
 *     the last CTA waits for exchange #1's next phase after the exchange completed), giving up
 *     after `polls` polls instead of about a second.  No copy or store is in flight to the waited
 *     barrier, so the kernel goes on and the row's status gets DLLM_ROW_ERR_TIMEOUT.  Site 8: in the
 *     int8 product kernels, each CTA's issuing thread waits, before its first product, for a barrier
 *     that nothing completes; the CTA gives up, waits for its copies and returns, the outputs are not
 *     written or not meaningful, and the call's status word gets DLLM_ROW_ERR_TIMEOUT.  Site 0
 *     switches it off.
 *   dllm_cuda_debug_fail_allocations(count): the next `count` device allocations the library
 *     makes for its own buffers fail as if cudaMalloc had run out of memory, so the calls that
 *     needed them return DLLM_ERR_OOM. */
DLLM_API dllm_status dllm_cuda_debug_inject_wait_timeout(int site, long long polls);
DLLM_API dllm_status dllm_cuda_debug_fail_allocations(int count);

/* Vocabulary-sharded sampling (a row's logits split over N GPUs, as a tensor-parallel LM head
 * leaves them).  No counterpart in the reference, whose sampler sees whole rows; together the
 * two calls and one all-gather give the tokens sampler_sample would (src/sampler.c:136-234)
 * for rows with 0 < top_k <= k.
 *
 * Step 1, on each GPU: `desc` describes this GPU's columns [vocab_offset, vocab_offset +
 * desc->vocab) of vocab_total-wide rows (logits, mask words of those columns, history as global
 * ids, params; uniforms and token are not used).  Writes the k best entries of each row after
 * mask and penalties, by (value desc, id asc): cand_val / cand_id [rows][k] (device), values are
 * the penalised logits (fp32), ids global.  k <= 256.
 * Step 2, the caller: all-gather the two arrays over the N GPUs into [N][rows][k].
 * Step 3, on any GPU: one token per row from the gathered candidates (per-row or broadcast
 * params; uniforms, token and the optional status are device arrays [rows]).  A sampling row
 * (temperature > 0) needs 1 <= top_k <= k: broadcast params outside that range are rejected
 * with DLLM_ERR_UNSUPPORTED; a per-row top_k outside it gets the greedy token and status bit
 * DLLM_ROW_ERR_TOPK_LARGE. */
DLLM_API dllm_status dllm_cuda_shard_candidates(const dllm_batch_desc *desc, int64_t vocab_offset,
                                                int64_t vocab_total, int k, float *cand_val,
                                                int32_t *cand_id, void *stream);
DLLM_API dllm_status dllm_cuda_merge_sample(int rows, int nshards, int k, const float *cand_val,
                                            const int32_t *cand_id, const dllm_sampler_params *params,
                                            const dllm_sampler_params *row_params,
                                            const float *uniforms, int32_t *token, int32_t *status,
                                            void *stream);

/* Peer exchange for vocabulary-sharded sampling (no counterpart in the reference): the candidate
 * kernel stores each row's k candidates straight into every rank's exchange buffer over NVLink
 * (plain peer stores, no multicast) and counts the row in that rank's arrival counter, so the
 * exchange overlaps the candidate computation row by row instead of following it as a collective.
 *   dllm_cuda_peer_exchange_create: on each rank, a zeroed device buffer for `rows` x `k`
 *     candidates of `world` ranks (arrival counters, then two slots used by alternate steps) and
 *     its cudaIpcMemHandle (64 bytes, written to ipc_handle) for the other ranks.
 *   dllm_cuda_peer_exchange_open / _close: map / unmap another rank's buffer on this GPU.
 *   dllm_cuda_peer_exchange_free: release this rank's buffer.
 *   dllm_cuda_shard_candidates_peer: step `epoch` (1, 2, ...; the same on every rank) of
 *     dllm_cuda_shard_candidates, writing into every rank's buffer; peer_bufs is a DEVICE array
 *     [world] of the buffers as mapped on this GPU (this rank's own buffer at index rank).
 *     Needs k + the history bound <= 256.
 *   dllm_cuda_merge_sample_peer: dllm_cuda_merge_sample over this rank's buffer for step `epoch`;
 *     each row's block waits until every rank's rows have arrived.  The wait is bounded: a rank
 *     missing after 2 s makes the rows time out (token 0, status DLLM_ROW_ERR_TIMEOUT) and the
 *     kernel returns.
 * Every rank must run every step, in the same order, on one stream per rank: a rank's next step's
 * stores reuse the slot of the step before last, which every rank has finished merging by then. */
DLLM_API dllm_status dllm_cuda_peer_exchange_create(int rows, int k, int world, void **buf, void *ipc_handle);
DLLM_API dllm_status dllm_cuda_peer_exchange_open(const void *ipc_handle, void **peer_buf);
DLLM_API dllm_status dllm_cuda_peer_exchange_close(void *peer_buf);
DLLM_API dllm_status dllm_cuda_peer_exchange_free(void *buf);
DLLM_API dllm_status dllm_cuda_shard_candidates_peer(const dllm_batch_desc *desc, int64_t vocab_offset,
                                                     int64_t vocab_total, int k, void *const *peer_bufs, int rank,
                                                     int world, uint64_t epoch, void *stream);
DLLM_API dllm_status dllm_cuda_merge_sample_peer(int rows, int world, int k, const void *local_buf, uint64_t epoch,
                                                 const dllm_sampler_params *params,
                                                 const dllm_sampler_params *row_params, const float *uniforms,
                                                 int32_t *token, int32_t *status, void *stream);

/* The step before the sampler (src/core/context.c:854-876): the final RMSNorm of `rows` hidden
 * states h [rows][hidden] (fp32; src/rmsnorm.c:4-27, norm_w may be NULL, add_one for Gemma's
 * (w + 1)), the logits matvec against unquantised output weights w [vocab][hidden]
 * (DLLM_DTYPE_F32 / BF16 / F16, 16-byte aligned; src/matvec.c:251-366, a double-precision dot
 * product per row rounded once), and, when softcap > 0, logit = softcap * tanhf(logit / softcap).
 * Writes logits [rows][vocab] (fp32) ready for dllm_cuda_sample_batch.  hidden must be a multiple
 * of 8.  All pointers are device memory. */
DLLM_API dllm_status dllm_cuda_lmhead_logits(int rows, int hidden, int vocab, const float *h, const float *norm_w,
                                             float eps, int add_one, const void *w, int w_dtype, float softcap,
                                             float *logits, void *stream);

/* The LM-head tail with 8-bit integer weights (no counterpart in the reference).  Codes are
 * symmetric, from -127 to 127, with one fp32 scale for each row; rows of codes start on multiples
 * of 16 bytes (base and stride), so a row may be followed by padding, which is not read as data.
 *
 * dllm_cuda_quantize_rows_i8: `rows` rows of `cols` values (fp32 / bf16 / fp16, x_stride elements
 *   apart) to codes q [rows][q_stride] and scales [rows].  Without norm y = x; with norm
 *   y = x * g / sqrt(mean(x^2) + eps), g = norm_w, norm_w + 1 (add_one) or 1 (norm_w NULL).
 *   scale = (float)(max|y| / 127) and q = y / scale rounded to the nearest integer, ties to even,
 *   both decided in 64 bits.  A row whose scale would lie below the smallest normal float has
 *   scale 0 and codes 0; a row with an infinity or a NaN has scale NaN and codes 0.  Quantises
 *   output weights (rows = vocabulary) once, and activations (rows = tokens) each step.
 *   Padding behind a row is left as it was.
 * dllm_cuda_matmul_i8: out[i][j] = (sum over k of a[i][k] * b[j][k]) * a_scale[i] * b_scale[j], for m
 *   rows of a (tokens) and n rows of b (channels): the sum exact in 32-bit integers (k <= 131071) and
 *   rounded to fp32, the two products in fp32 in this order (the first may overflow where scales are
 *   near the ends of fp32's range), the softcap cap * tanh(out / cap) when softcap > 0, and one rounding
 *   to out_dtype (fp32 / bf16 / fp16).  Before that rounding a normal result is within 10 x 2^-24 of the
 *   exact one, relative to it.  Codes may be -128 too.
 *   softcap is 0 or a normal float.  A channel whose b_scale / softcap is below the smallest normal float
 *   counts as 0.
 *   status (optional, one device word): DLLM_ROW_ERR_TIMEOUT is ORed in if a bounded wait expired.
 * dllm_cuda_lmhead_logits_i8: dllm_cuda_lmhead_logits with int8 output weights w [vocab][w_stride]
 *   and their scales: the final RMSNorm and the codes of h [rows][hidden] in one kernel, then the
 *   product and the softcap, writing fp32 logits [rows][vocab].  `workspace` holds the codes
 *   (dllm_cuda_lmhead_i8_workspace_bytes, 256-byte aligned); NULL: the library's buffer of the
 *   (device, stream), as in dllm_batch_desc, which is refused while the stream is being captured. */
DLLM_API dllm_status dllm_cuda_quantize_rows_i8(int rows, int cols, const void *x, int64_t x_stride, int x_dtype,
                                                int norm, const float *norm_w, float eps, int add_one, int8_t *q,
                                                int64_t q_stride, float *scale, void *stream);
DLLM_API dllm_status dllm_cuda_matmul_i8(int m, int n, int k, const int8_t *a, int64_t a_stride, const float *a_scale,
                                         const int8_t *b, int64_t b_stride, const float *b_scale, float softcap,
                                         void *out, int64_t out_stride, int out_dtype, int32_t *status, void *stream);
DLLM_API size_t dllm_cuda_lmhead_i8_workspace_bytes(int rows, int hidden);
DLLM_API dllm_status dllm_cuda_lmhead_logits_i8(int rows, int hidden, int vocab, const float *h, const float *norm_w,
                                                float eps, int add_one, const int8_t *w, int64_t w_stride,
                                                const float *w_scale, float softcap, float *logits, int32_t *status,
                                                void *workspace, size_t workspace_bytes, void *stream);

/* One step of beam search (no counterpart in the reference, which draws one token per row).
 *
 * dllm_cuda_beam_select: for each of `batch` sequences, the k best continuations of its `beams`
 * beams.  With lp(b, i) = x_bi - log(sum over allowed j of exp(x_bj)) over beam b's logits row,
 * a continuation (b, i) has the score cum = scores[b] + lp(b, i) and the rank cum / L^alpha, where
 * L = lengths[b] + 1 is its length in tokens (alpha = length_penalty; without lengths or with
 * alpha = 0 the rank is the score).  Order: rank descending, then beam, then logit descending,
 * then id ascending; sums and ranks are held in 64 bits, L^alpha within 1e-200 and 1e200.
 *   - A cleared mask bit leaves id i out, whatever its logit.  Continuations of probability 0
 *     (logit -inf, score -inf) are never chosen: slots that nothing fills get score -inf,
 *     parent -1, token -1.  A score below fp32's range is written as -inf too, with its parent and token.
 *   - An ended beam (finished[b] != 0) has one continuation, the token `eos` with its own score
 *     and L = max(lengths[b], 1); its logits are not read.
 *   - A row with an unmasked NaN or +inf, or a score of NaN or +inf, offers nothing; its status
 *     word gets DLLM_ROW_ERR_NONFINITE.
 * beams <= DLLM_BEAM_MAX, k <= DLLM_BEAM_K_MAX, vocab <= 2^30.  Outputs may be the arrays of the inputs of the
 * same shape (k = beams).
 *
 * dllm_cuda_beam_reorder: state[s][b] = state[s][parent[s][b]] for each of `ntensors` tensors, in
 * place (parent: device [batch][beams], values outside 0 .. beams - 1 leave the beam as it is).
 * `tensors` is a HOST array of device pointers to tensors that share no byte with one another or with
 * `parent` (others are refused); each holds batch x beams rows row_stride bytes apart, a row being `segs`
 * runs of run_bytes bytes, seg_stride bytes apart.
 * Bytes between runs are not touched.  Beams that keep their own state are neither read nor
 * written. */
#define DLLM_BEAM_MAX   128
#define DLLM_BEAM_K_MAX 256

typedef struct {
    int batch, beams, vocab, k;
    int64_t row_stride;       /* elements between consecutive rows (>= vocab) */
    int dtype;                /* DLLM_DTYPE_F32 / BF16 / F16 */
    const void *logits;       /* [batch * beams][row_stride] */
    const uint32_t *mask;     /* allow-mask of each row or NULL, as in dllm_batch_desc */
    int64_t mask_stride;      /* words between rows */
    const float *scores;      /* [batch][beams] sums of log-probabilities so far */
    const uint8_t *finished;  /* [batch][beams] ended beams, or NULL */
    int eos;                  /* end token (>= 0 when finished or out_finished is given) */
    const int32_t *lengths;   /* [batch][beams] tokens so far, or NULL */
    float length_penalty;     /* alpha; finite, needs lengths when it is not 0 */

    float *out_score;         /* [batch][k] scores (not ranks), best rank first */
    int32_t *out_parent;      /* [batch][k] beam that each continues */
    int32_t *out_token;       /* [batch][k] id that it adds */
    uint8_t *out_finished;    /* optional [batch][k]: ended before, or by this token */
    int32_t *out_lengths;     /* optional [batch][k]: tokens including this one; needs lengths */
    int32_t *status;          /* optional [batch][beams] out: 0 or DLLM_ROW_ERR_NONFINITE */

    void *workspace;          /* device scratch of dllm_cuda_beam_workspace_bytes() bytes, 256-byte
                                 aligned; NULL: the library's buffer of the (device, stream), as in
                                 dllm_batch_desc, refused while the stream is being captured */
    size_t workspace_bytes;
} dllm_beam_desc;

DLLM_API size_t dllm_cuda_beam_workspace_bytes(const dllm_beam_desc *desc);
DLLM_API dllm_status dllm_cuda_beam_select(const dllm_beam_desc *desc, void *stream);
DLLM_API dllm_status dllm_cuda_beam_reorder(int batch, int beams, const int32_t *parent, int ntensors,
                                            void *const *tensors, int64_t row_stride, int segs, int64_t seg_stride,
                                            int64_t run_bytes, void *stream);

/* Decode-loop glue (no counterpart in the reference, whose caller appends to its seen-token
 * array on the host): appends token[0] (device) to one sequence's device history
 * hist_ids[hist_off[0], hist_off[1]), which has room for `cap` ids from hist_off[0]; when full,
 * the oldest id is dropped.  Stream-ordered, so "sample, append" steps can run back to back and
 * be captured in a CUDA graph (sample with a caller-provided workspace, or make one call before
 * the capture, so that nothing is allocated during it). */
DLLM_API dllm_status dllm_cuda_append_history(const int32_t *token, int32_t *hist_ids, int64_t *hist_off,
                                              int64_t cap, void *stream);

/* Diagnostics: when given two CUDA events (cudaEvent_t, created by the caller), every later
 * sampling call records `before` on its stream right before the cluster kernel and `after` right
 * after it, so the caller can time that kernel alone; NULLs switch it off.  No counterpart in
 * the reference. */
DLLM_API dllm_status dllm_cuda_set_timing_events(void *before, void *after);

/* Version and build information ("diskllm_cuda <ver> sm_100a"). */
DLLM_API const char *dllm_cuda_version(void);

/* Last CUDA error string recorded by the library on this thread (or ""). */
DLLM_API const char *dllm_cuda_last_error(void);

/* Draw state of a drop-in sampler (the xorshift64 state of src/sampler.c:63), so that a
 * resumed stream reproduces its ids. */
struct sampler;
DLLM_API uint64_t dllm_sampler_get_rng_state(const struct sampler *s);
DLLM_API void     dllm_sampler_set_rng_state(struct sampler *s, uint64_t state);

#ifdef __cplusplus
}
#endif
#endif /* DISKLLM_CUDA_H */

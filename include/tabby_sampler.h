/*
 * tabby_sampler -- C ABI of the MI355X (gfx950) token sampler.
 *
 * For each row of logits it computes, in one stream-ordered launch sequence:
 *   maxLogit, sumExp = sum exp(x - maxLogit) over the whole row, the exact top-k
 *   (value descending, ties to the lower index), and then sampleFromTopK's temperature /
 *   top-p / categorical draw from a caller-supplied uniform.
 *
 * It replaces, in the reference (xOAviOx/tabby):
 *   - ForwardPass.encodeSampling            src/engine/forward.ts:522-601   (GPU head)
 *   - the sample-block readback + decode    src/engine/forward.ts:142-157, 442-451
 *   - sampleFromTopK                        src/engine/sampler.ts:147-212   (CPU tail)
 * composed as the worker does (src/worker/inference.worker.ts:162-168), for many rows at once.
 *
 * Conventions: plain C types only; every function returns a tabby_status; device pointers
 * are owned by the caller, scratch is owned by the handle; one handle per host thread and
 * stream (calls on one handle must not overlap). tabby_last_error() gives the message of
 * the calling thread's most recent failure.
 */
#ifndef TABBY_SAMPLER_H
#define TABBY_SAMPLER_H

#include <stdint.h>

#if defined(__GNUC__)
#define TABBY_API __attribute__((visibility("default")))
#else
#define TABBY_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  TABBY_OK = 0,
  TABBY_EINVAL = 1,    /* bad argument; e.g. topK outside [0, k_max] (forward.ts:348-351) */
  TABBY_EHIP = 2,      /* HIP runtime / launch failure */
  TABBY_EEMPTY = 3,    /* empty candidate pool (sampler.ts:153) */
  TABBY_EDOMAIN = 4,   /* row outside the contract: NaN, +inf, or every entry -inf */
  TABBY_ECAPACITY = 5  /* request exceeds what the handle was created for */
} tabby_status;

typedef enum { TABBY_F32 = 0, TABBY_F16 = 1, TABBY_BF16 = 2 } tabby_dtype;

/* Per-row sampling parameters: SamplingParams (sampler.ts:83-98) plus the uniform that
 * SeededRandom.next() (sampler.ts:112-118) would return for this row. All f64, as JS
 * numbers are: 0.9 as f32 is not 0.9, and a mulberry32 draw has 32 significant bits. */
typedef struct {
  double temperature; /* <= 0 (-0, -inf included): greedy, the uniform is not used
                         (sampler.ts:159-167); NaN and +inf are refused (TABBY_EINVAL) */
  double top_p;       /* any value, as sampler.ts:177-186 takes it: >= 1 or NaN, no nucleus
                         cut; <= 0 keeps the first candidate */
  double uniform;     /* in [0, 1) */
  int32_t top_k;      /* 1..k_max candidates; 0 = the whole vocabulary */
  int32_t reserved;   /* must be 0 */
} tabby_row_params;

/* Per-row result: SampleOutcome (sampler.ts:121-135) plus the TopKResult header
 * (forward.ts:93-103). */
typedef struct {
  int32_t id;            /* chosen token id */
  uint32_t considered;   /* consideredCount: candidates that survived top-p */
  double probability;    /* exp(l - maxLogit) / sumExp of the chosen id */
  double pool_mass;      /* full-vocabulary mass of the k candidates */
  float max_logit;       /* largest logit of the row */
  int32_t pool_exhausted;/* 1 when poolMass < topP (top-p clipped by k) */
  double sum_exp;        /* sum over the row of exp(x - maxLogit) */
  int32_t status;        /* tabby_status of this row */
  int32_t topk_count;    /* entries written to the row's top-k output, if requested */
} tabby_row_result;

typedef struct tabby_sampler tabby_sampler;

/* Allocates the scratch a ForwardPass allocates for sampling (forward.ts:243-248), sized
 * for up to rows_max rows of up to vocab_max entries and top_k up to k_max (<= 1024).
 * `device` is a HIP device ordinal. */
TABBY_API int tabby_sampler_create(int device, int32_t vocab_max, int32_t rows_max, int32_t k_max,
                         tabby_sampler **out);

/* Frees the handle's scratch (ForwardPass.destroy, forward.ts:309-315). NULL is a no-op. */
TABBY_API int tabby_sampler_destroy(tabby_sampler *sampler);

/*
 * Device-resident form: logits_dev is [rows, vocab] row-major of `dtype`; params_dev and
 * results_dev have `rows` entries in device memory. If topk_cap > 0, topk_ids_dev and
 * topk_logits_dev ([rows, topk_cap]) receive each row's candidates, highest first (the
 * TopKResult ids/logits, forward.ts:93-103). Asynchronous on `stream` (a hipStream_t, NULL
 * for the default stream). Parameters are validated on the device: a bad row gets a
 * nonzero status and the other rows are still sampled.
 * `flags`: TABBY_FLAG_FULL_VOCAB must be set if any row may have top_k = 0 (or >= vocab)
 * with vocab above the pool capacity; such a row's pool is the whole vocabulary, and its
 * top-k output holds the first min(topk_cap, vocab) entries of it (topk_cap <= k_max).
 */
#define TABBY_FLAG_FULL_VOCAB 1u
TABBY_API int tabby_sampler_sample_device(tabby_sampler *sampler, const void *logits_dev, int32_t dtype,
                                int32_t rows, int32_t vocab, const tabby_row_params *params_dev,
                                tabby_row_result *results_dev, int32_t *topk_ids_dev,
                                float *topk_logits_dev, int32_t topk_cap, uint32_t flags,
                                void *stream);

/*
 * Host-parameter form, the decode-loop entry (forward.ts:430-451 + inference.worker.ts:162-168):
 * params_host are validated before any GPU work (TABBY_EINVAL with the reference's
 * "topK must be between 0 and <k_max>, got <k>" message), uploaded, sampled, and
 * results_host (and the optional top-k arrays, host memory) are filled when it returns.
 * Returns the first nonzero row status, if any.
 */
TABBY_API int tabby_sampler_sample(tabby_sampler *sampler, const void *logits_dev, int32_t dtype,
                         int32_t rows, int32_t vocab, const tabby_row_params *params_host,
                         tabby_row_result *results_host, int32_t *topk_ids_host,
                         float *topk_logits_host, int32_t topk_cap, void *stream);

/*
 * Allocation-free form of tabby_sampler_sample_device. It has no counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). It takes no handle and
 * calls no hipMalloc, hipFree or allocating routine; its scratch is a fixed 16 MiB array in
 * the library's device image, one per GPU, kept until the process ends (the first call on a
 * device looks up its address). The 16 MiB are taken on every device the library's code is
 * loaded on, whether or not this entry is ever called. The caller passes inputs and outputs as for
 * tabby_sampler_sample_device, with flags = 0, on the current device. Limits: k_max <= 256,
 * and rows whose pool is the whole vocabulary (top_k = 0 or >= vocab, vocab > 256) get
 * status TABBY_EINVAL; a batch whose scratch would exceed 16 MiB returns TABBY_ECAPACITY
 * (batches of the sizes of the reference's configurations need at most ~10 MiB). Calls that
 * overlap on one GPU share that scratch and race: serialise them (one stream).
 */
TABBY_API int tabby_sampler_sample_device_noalloc(const void *logits_dev, int32_t dtype, int32_t rows,
                                                  int32_t vocab, int32_t k_max,
                                                  const tabby_row_params *params_dev,
                                                  tabby_row_result *results_dev, int32_t *topk_ids_dev,
                                                  float *topk_logits_dev, int32_t topk_cap, void *stream);

/*
 * Greedy fast path: ids_dev[r] = argmax of row r (src/engine/sampler.ts:13-23: the lowest
 * index among equal maxima, +0 equal to -0, NaN never chosen; 0 when the row's first entry
 * is NaN or nothing lies above -inf), for logits_dev [rows, vocab] of `dtype` in device
 * memory. max_logits_dev (may be NULL) receives the chosen entry's value. It replaces the
 * one-candidate sampling pass the reference's greedy and profile paths make
 * (forward.runSegment with {topK: 1}, src/worker/inference.worker.ts:216-229, read back by
 * argmaxOf) and generateGreedy's host argmax (sampler.ts:54-76): one read of the logits, no
 * pool, no uniform. Uses the handle's scratch; asynchronous on `stream`.
 */
TABBY_API int tabby_argmax_device(tabby_sampler *sampler, const void *logits_dev, int32_t dtype,
                                  int32_t rows, int32_t vocab, int32_t *ids_dev,
                                  float *max_logits_dev, void *stream);
/*
 * Row softmax of attention scores, replacing the softmax_rows kernel
 * (src/shaders/softmax_rows.wgsl:1-55, dispatched at src/engine/forward.ts:912-926) with the
 * results of its CPU reference softmaxRows (src/reference/cpu.ts:238-264) bit for bit.
 * x_dev and out_dev are [n_rows, row_len] f32 in device memory; out_dev may be x_dev (in
 * place, as the reference runs it) or a buffer that does not overlap it. With
 * causal_period > 0, row r covers its first causal_offset + (r % causal_period) + 1 entries
 * and the rest of the row is written 0; causal_period = 0 softmaxes whole rows.
 * causal_offset + causal_period must not exceed row_len. Asynchronous on `stream`; no
 * scratch.
 */
TABBY_API int tabby_softmax_rows_device(const float *x_dev, float *out_dev, int32_t n_rows,
                                        int32_t row_len, int32_t causal_period,
                                        int32_t causal_offset, void *stream);
/*
 * The lm_head's int4 weights (src/engine/forward.ts:408-428, encodeQuantMatmul :732-770;
 * src/shaders/matvec_q4.wgsl), repacked once into this library's layout. Input: the
 * reference's layout (tools/convert.py): words_dev u32 [vocab][hidden / 8] (eight 4-bit
 * values per word, value j at bits 4j, dequant(q) = (q - 8) * scale) and scales_dev f16 bits
 * [vocab][hidden / block_size]. Output: packed_dev u32 [hidden / 32][vocab][4] and
 * packed_scales_dev f16 bits [hidden / block_size][vocab] (a wave's 64 output rows read
 * contiguous bytes). hidden and block_size are multiples of 32, block_size divides hidden;
 * word arrays 16-byte aligned. Asynchronous on `stream`.
 */
TABBY_API int tabby_lmhead_q4_pack_device(const uint32_t *words_dev, const uint16_t *scales_dev,
                                          int32_t vocab, int32_t hidden, int32_t block_size,
                                          uint32_t *packed_dev, uint16_t *packed_scales_dev,
                                          void *stream);
/*
 * The lm_head matmul on its own (matvec_q4.wgsl's contract): logits_dev [rows][vocab] f32 =
 * hidden_dev [rows][hidden] f32 times the packed weights (+ bias_dev [vocab], may be NULL),
 * bit for bit the CPU reference matmulQuantized (src/reference/cpu.ts:352-393). Any number of
 * rows (weights re-read per eight rows). Asynchronous on `stream`.
 */
TABBY_API int tabby_lmhead_q4_device(const uint32_t *packed_dev, const uint16_t *packed_scales_dev,
                                     const float *bias_dev, const float *hidden_dev, int32_t rows,
                                     int32_t vocab, int32_t hidden, int32_t block_size,
                                     float *logits_dev, void *stream);
/*
 * The lm_head fused with sampling: for each of `rows` (1..8) hidden states, the logits of
 * tabby_lmhead_q4_device are computed and sampled without being written to memory -- the
 * composition of the reference's lm_head (forward.ts:408-428), encodeSampling
 * (forward.ts:522-601) and sampleFromTopK (sampler.ts:147-212) in one pass over the weights.
 * params_dev / results_dev as for tabby_sampler_sample_device. Pools of at most 64 (the
 * reference's topK bound, forward.ts:348-351; top_k 0 or above 64 gives the row TABBY_EINVAL);
 * no top-k lists. Uses the handle's scratch (vocab <= vocab_max, rows <= rows_max).
 * Asynchronous on `stream`.
 */
TABBY_API int tabby_sampler_sample_lmhead_q4_device(tabby_sampler *sampler, const uint32_t *packed_dev,
                                                    const uint16_t *packed_scales_dev,
                                                    const float *bias_dev, const float *hidden_dev,
                                                    int32_t rows, int32_t vocab, int32_t hidden,
                                                    int32_t block_size,
                                                    const tabby_row_params *params_dev,
                                                    tabby_row_result *results_dev, void *stream);
/*
 * Microscaled 4-bit floating point (MXFP4) beside the int4 weights of the reference's
 * encodeQuantMatmul (src/engine/forward.ts:732-770): values of 4 bits (e2m1: 0, 1/2, 1, 3/2,
 * 2, 3, 4, 6 and a sign) in blocks of 32 along a row, each block with a power of two as a
 * biased 8-bit exponent. A matrix [rows, cols] is held as two device arrays in this
 * library's panel layout; this call gives their sizes (both multiples of 256). What the calls
 * below write must not overlap what they read (TABBY_EINVAL), but for the product's result on x.
 */
TABBY_API int tabby_mx4_bytes(int32_t rows, int32_t cols, int64_t *code_bytes, int64_t *scale_bytes);
/*
 * x_dev [rows, cols] of `dtype` (TABBY_F32, TABBY_F16 or TABBY_BF16; rows row_stride elements
 * apart) to MXFP4, as a loader would convert weights for encodeQuantMatmul
 * (src/engine/forward.ts:732-770). A block's power is floor(log2(max |x|)) - 2, held to
 * [-127, 127]; a value is divided by it, rounded to the nearest of the sixteen codes (ties to
 * the even one) and held to 6. A block that holds a NaN or an infinity is NaN as a whole.
 * codes_dev is 16-byte aligned, scales_dev 4-byte. Asynchronous on `stream`.
 */
TABBY_API int tabby_mx4_quantize_device(const void *x_dev, int32_t dtype, int32_t rows, int32_t cols,
                                        int64_t row_stride, void *codes_dev, void *scales_dev, void *stream);
/*
 * The way back: out_dev [rows, cols] of `dtype` receives the values that the codes stand for,
 * as encodeQuantMatmul's shader expands its codes (src/engine/forward.ts:732-770): exact in
 * f32 and bf16 (above their range: infinity), rounded to nearest even in f16. Asynchronous on
 * `stream`.
 */
TABBY_API int tabby_mx4_dequantize_device(const void *codes_dev, const void *scales_dev, int32_t rows,
                                          int32_t cols, void *out_dev, int32_t dtype, int64_t row_stride,
                                          void *stream);
/*
 * A checkpoint's MXFP4 weights, repacked once as the int4 ones are for encodeQuantMatmul
 * (src/engine/forward.ts:732-770). Input: row_codes_dev [rows][ceil(cols / 32)][16], two codes
 * to a byte with the lower column in the low half, and row_scales_dev
 * [rows][ceil(cols / 32)], the biased exponents (255: a block of NaN). Codes past the last
 * column are taken as 0. Asynchronous on `stream`.
 */
TABBY_API int tabby_mx4_pack_device(const void *row_codes_dev, const void *row_scales_dev, int32_t rows,
                                    int32_t cols, void *codes_dev, void *scales_dev, void *stream);
/*
 * The product that stands in encodeQuantMatmul's place (src/engine/forward.ts:732-770) where
 * both sides are MXFP4: out_dev [rows, n] of `out_dtype` (rows out_stride elements apart) =
 * x [rows, k] times the transpose of w [n, k], plus bias_dev [n] (f32, may be NULL). Products
 * are exact, their sums f32, rounded once to out_dtype. Asynchronous on `stream`; no scratch.
 */
TABBY_API int tabby_mx4_matmul_device(const void *x_codes_dev, const void *x_scales_dev, int32_t rows,
                                      const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                      int32_t n, int32_t k, void *out_dev, int32_t out_dtype,
                                      int64_t out_stride, void *stream);
/*
 * The same from activations as the lm_head finds them (src/engine/forward.ts:408-428): x_dev
 * [rows, k] of `x_dtype`, rows x_stride elements apart, is quantised to MXFP4 in the call. The
 * caller's workspace_dev (16-byte aligned) holds at least code_bytes + scale_bytes of
 * [rows, k]; calls that may overlap need a workspace each. out_dev may lie on x_dev, in whole or
 * in part: x is read before any of it is written. Asynchronous on `stream`.
 */
TABBY_API int tabby_mx4_linear_device(const void *x_dev, int32_t x_dtype, int64_t x_stride, int32_t rows,
                                      const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                      int32_t n, int32_t k, void *out_dev, int32_t out_dtype,
                                      int64_t out_stride, void *workspace_dev, int64_t workspace_bytes,
                                      void *stream);
/*
 * Bytes of the workspace of the beam selection declared next, which stands where a search has
 * more than sampleFromTopK's one continuation (src/engine/sampler.ts:147-212).
 */
TABBY_API int tabby_beam_workspace(int32_t groups, int32_t beams, int32_t vocab, int32_t count, int64_t *bytes);
/*
 * Beam search's selection, in the place of encodeSampling and sampleFromTopK
 * (src/engine/forward.ts:522-601, src/engine/sampler.ts:147-212). Row g * beams + b of
 * logits_dev [groups * beams, vocab] (`dtype` TABBY_F32, TABBY_F16 or TABBY_BF16, rows
 * row_stride elements apart) holds the logits of beam b of group g, whose score so far is
 * scores_dev [groups, beams] (f32). A continuation by token t scores
 *   scores[g, b] + (x_t - log sum over the row's allowed entries of exp(x)),
 * in 64 bits, the logarithm within 1e-10. allowed_dev (may be NULL: everything) has ceil(vocab / 32) words to a row, entry t
 * at bit t % 32 of word t / 32; what is not allowed is never looked at, NaN included.
 * done_dev [groups, beams] (may be NULL): a beam with a nonzero entry has ended, and its one
 * continuation is pad_id at its own score, whatever its logits hold. A beam whose score is
 * -inf has no continuations, nor has an entry of -inf or a row in which nothing is allowed.
 * The `count` (1..128) best of each group's beams (1..64), equal scores in the order of (beam,
 * token) -- of each beam only its first `count` entries by (logit, token) are looked at, which
 * matters where 64 bits do not tell their scores apart -- go to tokens_dev, parents_dev (the beam within its group) and out_scores_dev, each
 * [groups, count]; where there are fewer the rest is -1, -1 and -inf. status_dev [groups] (may
 * be NULL) receives TABBY_OK, TABBY_EEMPTY (no continuation at all) or TABBY_EDOMAIN (an
 * allowed entry of a row that is read is NaN or +inf, or a score is NaN or +inf; the group's
 * outputs are as if it had none). The outputs lie apart from the inputs and from each other, but
 * out_scores_dev may be scores_dev where count is beams. workspace_dev: 16-byte aligned, of the
 * size given above; calls that may overlap need one each. Asynchronous on `stream`.
 */
TABBY_API int tabby_beam_select_device(const void *logits_dev, int32_t dtype, int64_t row_stride, int32_t groups,
                                       int32_t beams, int32_t vocab, const float *scores_dev,
                                       const uint32_t *allowed_dev, const int32_t *done_dev, int32_t pad_id,
                                       int32_t count, int32_t *tokens_dev, int32_t *parents_dev,
                                       float *out_scores_dev, int32_t *status_dev, void *workspace_dev,
                                       int64_t workspace_bytes, void *stream);
/*
 * The cached states (the reference's KV cache, src/engine/kvcache.ts:14-104, or anything else
 * kept by row) follow the beams that survived a selection. src_dev and dst_dev are host arrays
 * of `states` device addresses, all of one shape: groups * beams rows, row_stride bytes apart,
 * each of `segments` segments, segment_stride bytes apart, of `capacity` positions of unit_bytes
 * each. In every segment the first lengths_dev[g] positions (NULL: all; held to
 * [0, capacity]) of row (g, b) of dst become those of row (g, parents_dev[g, b]) of src; the rest
 * of dst stays. parents_dev [groups, beams]; a row whose parent is not within [0, beams) stays
 * as it is. Every state's dst is its src (in place, any parents), or none is; nothing that is
 * written may overlap another state (TABBY_EINVAL), while states may lie side by side in one
 * buffer. beams 1..64. Asynchronous on `stream`; no scratch.
 */
TABBY_API int tabby_beam_reorder_device(const void *const *src_dev, void *const *dst_dev, int32_t states,
                                        int32_t groups, int32_t beams, int32_t segments, int64_t capacity,
                                        int64_t unit_bytes, int64_t row_stride, int64_t segment_stride,
                                        const int32_t *parents_dev, const int32_t *lengths_dev, void *stream);
/*
 * 8-bit floating point (FP8: e4m3, largest value 448, no infinities) beside the int4 weights of the
 * reference's encodeQuantMatmul (src/engine/forward.ts:732-770): a matrix [rows, cols] in blocks of
 * `block_rows` x 128, each with an f32 that its codes are multiplied by. block_rows is 128 for weights
 * and 1 for activations. A matrix is held as two device arrays in this library's panel layout;
 * this call gives their sizes (both multiples of 256). What the calls below write must not overlap what they
 * read (TABBY_EINVAL), but for the product's result on x.
 */
TABBY_API int tabby_fp8_bytes(int32_t rows, int32_t cols, int32_t block_rows, int64_t *code_bytes, int64_t *scale_bytes);
/*
 * x_dev [rows, cols] of `dtype` (TABBY_F32, TABBY_F16 or TABBY_BF16; rows row_stride elements
 * apart) to FP8, as a loader would convert weights for encodeQuantMatmul
 * (src/engine/forward.ts:732-770). A block's scale is the smallest power of two, 2^-126 or more, with
 * max |x| <= 448 times it (1 for zeros); a value is divided by it and rounded to the nearest code (ties to the
 * even one). A block that holds a NaN or an infinity is NaN as a whole. codes_dev is 16-byte
 * aligned, scales_dev 4-byte. Asynchronous on `stream`.
 */
TABBY_API int tabby_fp8_quantize_device(const void *x_dev, int32_t dtype, int32_t rows, int32_t cols,
                                        int64_t row_stride, int32_t block_rows, void *codes_dev, void *scales_dev,
                                        void *stream);
/*
 * The way back: out_dev [rows, cols] of `dtype` receives code times scale, as encodeQuantMatmul's
 * shader expands its codes (src/engine/forward.ts:732-770): the f32 product (above f32's range: infinity), rounded
 * to nearest even in f16 and bf16. Asynchronous on `stream`.
 */
TABBY_API int tabby_fp8_dequantize_device(const void *codes_dev, const void *scales_dev, int32_t rows, int32_t cols,
                                          int32_t block_rows, void *out_dev, int32_t dtype, int64_t row_stride,
                                          void *stream);
/*
 * A checkpoint's FP8 weights, repacked once as the int4 ones are for encodeQuantMatmul
 * (src/engine/forward.ts:732-770). Input: row_codes_dev [rows][cols] and block_scales_dev
 * [ceil(rows / 128)][ceil(cols / 128)] f32, of any value. Output: a matrix with block_rows 128.
 * Asynchronous on `stream`.
 */
TABBY_API int tabby_fp8_pack_device(const void *row_codes_dev, const float *block_scales_dev, int32_t rows, int32_t cols,
                                    void *codes_dev, void *scales_dev, void *stream);
#define TABBY_FP8_FAST_SUMS 0x100
/*
 * The product that stands in encodeQuantMatmul's place (src/engine/forward.ts:732-770) where
 * both sides are FP8: out_dev [rows, n] of `out_dtype` (rows out_stride elements apart) =
 * x [rows, k] (block_rows 1) times the transpose of w [n, k] (block_rows 128), plus bias_dev [n] (f32, may be
 * NULL). Products of codes are exact, their sums and the scales' application f32, rounded once to
 * out_dtype. TABBY_FP8_FAST_SUMS, added to an out_dtype of TABBY_F16 or TABBY_BF16, lets more than 64 rows go through the
 * matrix cores as codes, at twice the rate: eight products at a time are added, each to 2^-13 of the
 * largest of them or better. Asynchronous on `stream`; no scratch.
 */
TABBY_API int tabby_fp8_matmul_device(const void *x_codes_dev, const void *x_scales_dev, int32_t rows,
                                      const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                      int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                      void *stream);
/*
 * The same from activations as the lm_head finds them (src/engine/forward.ts:408-428): x_dev
 * [rows, k] of `x_dtype`, rows x_stride elements apart, is quantised (block_rows 1) in the call. The
 * caller's workspace_dev (16-byte aligned) holds at least code_bytes + scale_bytes of
 * [rows, k]; calls that may overlap need a workspace each. out_dev may lie on x_dev, in whole or
 * in part: x is read before any of it is written. Asynchronous on `stream`.
 */
TABBY_API int tabby_fp8_linear_device(const void *x_dev, int32_t x_dtype, int64_t x_stride, int32_t rows,
                                      const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                      int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                      void *workspace_dev, int64_t workspace_bytes, void *stream);
/*
 * Bytes of the workspace of the verification declared next, which stands where a decode step has
 * drafted tokens to check in the place of sampleFromTopK's one token (src/engine/sampler.ts:147-212).
 */
TABBY_API int tabby_draft_workspace(int32_t requests, int32_t drafts_max, int32_t vocab, int64_t *bytes);
/*
 * Verification of drafted tokens, in the place of encodeSampling and sampleFromTopK
 * (src/engine/forward.ts:522-601, src/engine/sampler.ts:147-212) where a smaller model, or a lookup,
 * has proposed a request's next tokens. Request r's rows of logits_dev [rows, vocab] (`dtype`
 * TABBY_F32, TABBY_F16 or TABBY_BF16, rows row_stride elements apart) are offsets_dev[r] to
 * offsets_dev[r + 1] - 1 (NULL: drafts_max + 1 rows to each): row j after j of its drafted tokens. It has one
 * drafted token less than rows, at most drafts_max (0..63); they, their uniforms (uniforms_dev, in [0, 1))
 * and, with draft_logits_dev, the rows they were drawn from lie one request after another, [rows - requests]. Without
 * draft_logits_dev (NULL) the tokens were certain. params_dev [requests] holds each request's
 * settings, those of the target and of the draft, and the uniform of its last draw.
 * P and Q are what sampleFromTopK draws from for a row of the target and of the draft: the first top_k
 * entries by (logit, lower index), weights exp((x - max) / temperature), those up to and with the first at
 * which their running sum reaches top_p of the total (of more than 128 entries: to within 1e-11 of it, 2.5e-10
 * where the call has more than 4,096 rows, and 2^-52 of the largest weight to an entry), divided by their sum; temperature <= 0: the first
 * entry. A drafted token d is accepted while uniform * Q(d) < P(d), Q(d) being 1 where the tokens were certain and where
 * temperature <= 0. The next token is drawn from max(P - Q, 0) at the first refusal (from P without d where d was
 * certain), from the last row's P if there is none: the first token in the vocabulary's order at which the
 * running sum exceeds params' uniform times the total.
 * tokens_dev [requests, drafts_max + 1] receives the accepted tokens, the drawn one and -1s, accepted_dev
 * [requests] how many were accepted, status_dev [requests] (may be NULL) TABBY_OK, TABBY_EINVAL
 * (settings as tabby_sampler_sample_device refuses them, offsets that do not ascend within the rows, a
 * drafted token outside the vocabulary) or TABBY_EDOMAIN (a row with a NaN, +inf or nothing above -inf);
 * such a request's tokens are -1, none accepted. Rows after the first refusal do not matter.
 * `flags`: TABBY_FLAG_FULL_VOCAB must be set if a request may have temperature > 0 and top_k 0, or above 128, with a
 * vocabulary of more than 128 (such a request is refused without it). vocab is at most 2^24. What is written lies apart from
 * what is read. workspace_dev: 16-byte aligned, of the size given above; calls that may overlap need one
 * each. Asynchronous on `stream`.
 */
TABBY_API int tabby_draft_verify_device(const void *logits_dev, int32_t dtype, int64_t row_stride, int32_t rows,
                                        const void *draft_logits_dev, int64_t draft_row_stride,
                                        const int32_t *drafts_dev, const double *uniforms_dev,
                                        const int32_t *offsets_dev, int32_t requests, int32_t drafts_max, int32_t vocab,
                                        const tabby_row_params *params_dev, int32_t *tokens_dev, int32_t *accepted_dev,
                                        int32_t *status_dev, void *workspace_dev, int64_t workspace_bytes,
                                        uint32_t flags, void *stream);
/* Message of the calling thread's last failure ("" if none). */
TABBY_API const char *tabby_last_error(void);

/* Library version string. */
TABBY_API const char *tabby_version(void);

/*
 * Diagnostic: y[i] = exp(x[i]) over device arrays with the device's f64 exp, the fdlibm
 * method that V8's Math.exp uses (the exp of sampler.ts:156,170). For parity tests.
 */
TABBY_API int tabby_debug_exp(const double *x_dev, double *y_dev, int64_t n, void *stream);

/*
 * Diagnostic: y[i] = fround(Math.exp(x[i])) for x[i] <= 0 (or NaN), the f32 exps of the row
 * softmax (src/reference/cpu.ts:253), as tabby_softmax_rows_device computes them. For
 * parity tests.
 */
TABBY_API int tabby_debug_exp_f32(const float *x_dev, float *y_dev, int64_t n, void *stream);
/*
 * Diagnostic: the device's bit-exact sequential f64 sum (the left-to-right sums of
 * sampler.ts:156-203: poolMass, the scaled total, the running sums), computed in parallel by
 * one wave. terms_dev[0..n) must be >= 0 with terms_dev[0] > 0; prefix_dev[j] receives the
 * j-th partial sum up to the first that is >= stop_at (INFINITY: none), and *count_dev the
 * number of partial sums written. wide = 1 selects the form used for long sums (16 terms per
 * lane per step), wide = 2 the same taken by a four-wave workgroup, wide = 3 by an eight-wave
 * workgroup (the form that finishes whole-vocabulary heads), wide = 4 the register form for
 * n <= 64 (term i in lane i: the form that finishes pools of at most 64). prefix_dev may be terms_dev
 * itself (the sums are then written over their terms, as whole-vocabulary heads run them).
 * For parity tests.
 */
TABBY_API int tabby_debug_seq_sum(const double *terms_dev, int32_t n, double stop_at,
                                  double *prefix_dev, int32_t *count_dev, int32_t wide,
                                  void *stream);

/*
 * Diagnostic: the draw of sampleFromTopK (sampler.ts:195-203) as whole-vocabulary rows run
 * it, a 64-ary search by one wave: for each of the m targets, out_dev[j] = the first i in
 * [0, n) with targets_dev[j] < c_dev[i] (c non-decreasing), or n - 1 when there is none.
 * For parity tests.
 */
TABBY_API int tabby_debug_first_above(const double *c_dev, int32_t n, const double *targets_dev,
                                      int32_t m, int32_t *out_dev, void *stream);
/*
 * Diagnostic with no counterpart in the reference, for measurements (bench.py
 * --read-ceiling and the FETCH_SIZE calibration): reads src_dev ([rows, row_floats] f32,
 * 16-byte aligned, row_floats a multiple of 4) once with the sampling kernels' 16-byte
 * nontemporal loads in their launch shape (one 1,024-lane workgroup per row) and does nothing
 * else with it -- the read ceiling of those bytes on this GPU, and a kernel whose FETCH_SIZE
 * per dispatch must equal a known byte count. sink_dev ([rows] u32) is almost never written.
 */
TABBY_API int tabby_debug_stream_read(const float *src_dev, int32_t rows, int64_t row_floats,
                                      uint32_t *sink_dev, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TABBY_SAMPLER_H */

/*
 * ytm.h -- C-ABI of libytm.so, the MI355X (gfx950) Tsetlin Machine hot path.
 *
 * This boundary replaces the reference's PyCUDA layer (src/cutm/base.py:128-206 compiles
 * src/cutm/cuda/kernel.cu and drives its 9 kernels with prepared_call).  Every entry point
 * below names the reference interface it stands in for.  Plain pointers and sizes only:
 * host arrays are caller-owned and borrowed for the duration of a call; device memory is
 * owned by the model / dataset handles.  Calls are synchronous on return, one HIP stream
 * per model, not re-entrant per handle.  Every function returns 0 on success and a
 * nonzero status otherwise; ytm_last_error() then describes the failure (thread-local).
 */
#ifndef YTM_H
#define YTM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
enum {
    YTM_OK = 0,
    YTM_EINVAL = 1,   /* bad argument / unsupported configuration */
    YTM_EHIP = 2,     /* HIP runtime error */
    YTM_ETIMEOUT = 3, /* a persistent kernel's bounded wait expired (2 s of real time, which
                         also runs while the GPU is preempted); the model's state is then a mix
                         of samples, and ytm_fit*, ytm_score* and ytm_transform refuse it
                         (YTM_EINVAL) until ytm_set_ta_state, ytm_set_weights and
                         ytm_set_patch_weights have all loaded a state again */
    YTM_ERANGE = 4    /* state value outside what the model can represent */
};

/* Element types of the binarizer inputs (ytm_binarize). */
enum {
    YTM_DTYPE_U8 = 0,
    YTM_DTYPE_I8 = 1,
    YTM_DTYPE_U16 = 2,
    YTM_DTYPE_I16 = 3,
    YTM_DTYPE_U32 = 4,
    YTM_DTYPE_I32 = 5,
    YTM_DTYPE_I64 = 6,
    YTM_DTYPE_F32 = 7,
    YTM_DTYPE_F64 = 8,
    /* of the answering operators alone: */
    YTM_DTYPE_F16 = 9,
    YTM_DTYPE_BF16 = 10,
    YTM_DTYPE_BITS = 11 /* uint32 words, bit b of word j = clause 32 j + b */
};

/* Model hyperparameters, resolved on the host exactly as src/cutm/base.py:60-121,129-152
 * resolves them into #defines.  s_inv and q_prob are S_INV and Q_PROB as the reference's
 * C preprocessor types them (float or double, kernel.cu:31-32), widened to double. */
typedef struct ytm_params {
    int32_t clauses;               /* CLAUSES = banks * number_of_clauses_per_class */
    int32_t classes;               /* CLASSES */
    int32_t dim0, dim1, dim2;      /* DIM0 (width), DIM1 (height), DIM2 (channels) */
    int32_t patch_dim0, patch_dim1;/* PATCH_DIM0, PATCH_DIM1 */
    int32_t number_of_ta_states;   /* MAX_TA_STATE */
    int32_t max_included_literals; /* MAX_INCLUDED_LITERALS (resolved: LITERALS if None) */
    int32_t append_negated;        /* APPEND_NEGATED */
    int32_t encode_loc;            /* ENCODE_LOC */
    int32_t coalesced;             /* COALESCED (CLAUSE_BANKS = coalesced ? 1 : CLASSES) */
    int32_t negative_polarity;     /* NEGATIVE_CLAUSES */
    int32_t init_neg_weights;      /* INIT_NEG_WEIGHTS */
    int32_t thresh;                /* THRESH (T) */
    double s_inv;                  /* S_INV */
    double q_prob;                 /* Q_PROB */
    uint64_t seed;                 /* key of the counter-based random stream */
} ytm_params;

typedef struct ytm_model ytm_model;
typedef struct ytm_dataset ytm_dataset;

/* Per-model counters and timings of the most recent calls (HIP events on the model's
 * stream around the kernels named). */
typedef struct ytm_stats {
    uint64_t step;               /* samples trained so far (the random stream's step) */
    uint64_t last_fit_samples;
    uint64_t last_fit_updates;   /* (sample, clause) pairs that ran a Type Ia/Ib/II branch */
    uint64_t total_updates;
    double last_fit_kernel_ms;   /* sum over the training kernel launches of the last fit */
    int32_t last_fit_launches;
    int32_t train_workgroups;    /* persistent grid size used by the training kernel (clause
                                    banks: workgroups of each per-sample launch) */
    double last_score_kernel_ms; /* class-sum kernel of the last score */
    double last_encode_kernel_ms;
    double last_fit_wait_frac;   /* share of the training kernel's time workgroups spent
                                    waiting for the per-sample class sums */
    int32_t train_kind;          /* 0 = clause state resident in LDS, 1 = global (one
                                    patch), 2 = global (several patches), 3 = resident and
                                    streaming (one patch), 4 = one ordinary launch per
                                    sample: clause banks (coalesced=0), more than 64
                                    classes, or a persistent grid that does not fit */
    int32_t train_specialised;   /* 1 when the last fit ran a training kernel compiled at run
                                    time for this model's geometry (hipRTC), 0 when it ran the
                                    built-in kernel (YTM_JIT=0, or the compile was unavailable) */
    double last_fit_phase_us[8]; /* with YTM_TRAIN_PROFILE=1: average microseconds per sample
                                    that wave 0 of each workgroup spends in each phase of the
                                    training kernel (resident: exchange, barrier, D1, barrier,
                                    D2, D3, barrier, and the slowest other wave's time in the
                                    exchange step; global: staging, publish and exchange,
                                    wait for the next sample's evaluation, decisions, literal
                                    updates, re-evaluation of the updated clauses).  YTM_TRAIN_PROFILE=2 / =3 restrict that last
                                    resident slot to the next sample's evaluation / its
                                    evaluation and the staging of the sample after it */
    uint64_t last_fit_feedback_samples; /* samples of the last fit at which some class had an
                                    update probability above zero (the streaming kernel stops
                                    there to apply feedback); the sample count for the others */
    uint64_t last_fit_evaluations; /* clause evaluations of a sample per workgroup, averaged:
                                    the sample count plus the speculative ones discarded at
                                    stops (streaming kernel); the sample count for the others */
    int32_t last_fit_stream;     /* 1 when the last fit ran the streaming kernel (train_kind
                                    is then 3) */
    int16_t train_product;       /* 1 when the last fit evaluated its clauses on the matrix cores
                                    (train_kind 2) */
    int16_t score_path;          /* scorer of the last score: 0 none yet, 1 a class sum per sample and
                                    clause, 2 register tiles (one patch), 3 literal lists (one
                                    patch), 4 literal lists (several patches), 5 matrix cores */
    uint64_t last_fit_draws[3];  /* with YTM_TRAIN_PROFILE=4: counter-stream words computed
                                    by the last fit's training kernel, one per lane and draw
                                    site (a Philox4x32-10 call): reservoir draws, Q-skip /
                                    update draws, literal draws.  Zero otherwise */
} ytm_stats;

/* Thread-local description of the last failure. */
const char *ytm_last_error(void);

/* Unloads the training-kernel modules compiled at run time (each on its device, after a
 * device synchronize), so that nothing of the library is left on a GPU when the process
 * exits; call it after destroying every model and dataset.  A later fit loads what it needs
 * again.  Replaces the context teardown that `import pycuda.autoinit` registers for process
 * exit (src/cutm/base.py:5), which releases the modules SourceModule loaded
 * (src/cutm/base.py:155-159).  Also frees every device block kept between calls (ytm_create) and
 * the pinned buffers of large copies.  YTM_EHIP when a module fails to unload. */
int ytm_shutdown(void);

/* Model lifetime.  Replaces BaseTM._gpu_init / _reset_clauses / _reset_weights
 * (src/cutm/base.py:128-222; kernel.cu:46-73 init_weights): TA states start at
 * number_of_ta_states/2, weights from the INIT random site, patch weights and bias 0.
 * Geometry bounds: at most 4096 classes (the reference's kernels take any CLASSES; more
 * than 64 train one sample per launch), any number of patches, any int32
 * number_of_ta_states (up to 32 bit-planes), classes * literal words * 6 below 2^32 (the
 * 32-bit literal-draw site index of the counter stream).  YTM_EINVAL otherwise.
 *
 * Device memory that a call is done with (buffers of its host arrays, a destroyed data set's or
 * model's) is kept for later calls, the longest unused freed first: at most 1 GiB of it idle
 * while a model lives on that device, and 256 MiB once ytm_destroy ended the last one, until
 * ytm_shutdown.  Another allocator of the process cannot have it before.  Pinned host memory is
 * kept alike, at most 64 and 16 MiB, and 16 MiB a device for large copies.  A model holds the room of its scorers' operands from the
 * start where it is no larger than its TA states and than 256 MiB and memory allows. */
int ytm_create(const ytm_params *params, ytm_model **out);
void ytm_destroy(ytm_model *m);
/* L, W (=number_of_literal_chunks), P (=number_of_patches), number of TA bit-planes. */
int ytm_geometry(const ytm_model *m, int64_t out[4]);
int ytm_get_stats(const ytm_model *m, ytm_stats *out);
/* Reseed the random stream and reset its step to 0 (what re-running __init__ does). */
int ytm_set_seed(ytm_model *m, uint64_t seed);
/* Compile (and cache for this process) the training kernel specialised for the geometry
 * of *params and the launch shape used on a device with compute_units CUs (0: 256, an
 * MI355X), without touching a GPU.  train_kind as in ytm_stats (0 resident: one patch, or
 * several with ceil(P/32) <= 64; 1 global one patch; 2 global several patches; 3 streaming:
 * one patch, coalesced, counter stream only); injected != 0 for the injected-draw variant.
 * Clause-bank models (coalesced = 0) and models of more than 64 classes train with built-in
 * kernels only (train_kind 4): YTM_EINVAL.
 * The counterpart of the per-model kernel compile in BaseTM.__init__
 * (src/cutm/base.py:129-159); ytm_fit compiles on first use anyway, so calling this is
 * optional (warm-up, or checking that the compiler is available).  YTM_EHIP with the
 * compiler log in ytm_last_error() on failure. */
int ytm_compile_train_kernel(const ytm_params *params, int train_kind, int injected,
                             int compute_units);
/* Compile (when not cached) and load onto the model's device every counter-stream training
 * kernel that ytm_fit may choose for this model (the streaming kernel of a one-patch model and
 * the resident or global one), so that no fit pays for it later; the kinds loaded (train_kind
 * values) go to kinds[0 .. *n_kinds).  The counterpart of the per-model kernel compile in
 * BaseTM.__init__ (src/cutm/base.py:129-159).  Nothing is loaded for clause banks or with
 * YTM_JIT=0 (*n_kinds = 0).  Optional: ytm_fit loads a kernel on first use anyway. */
int ytm_load_train_kernels(ytm_model *m, int32_t kinds[4], int32_t *n_kinds);

/* encode: BaseTM.encode (src/cutm/base.py:224-263; kernel.cu:76-152 encode_batch).
 * X: uint32 (N, dim0*dim1*dim2), any value > 0 is a set pixel.  out: uint32 (N, P, W). */
int ytm_encode(ytm_model *m, const uint32_t *X, int64_t N, uint32_t *out);

/* encode of binned raw values in one pass, without the binned array: the transform of
 * Binarizer / ThermometerBinarizer (src/tm_utils/binarizer.py:9-22,63-86) followed by
 * BaseTM.encode (src/cutm/base.py:224-263; kernel.cu:76-152).  X holds N samples of
 * dim0*dim1*dim2 / width raw values of type x_dtype (YTM_DTYPE_*); value i of a sample
 * becomes the width levels (kind 0 thermometer: width = nthr; kind 1 one-hot: width =
 * nthr - 1 + 2 * edge_bins) at positions [i * width, (i + 1) * width) of the binned row,
 * as ytm_binarize lays them out, with the same thresholds and comparison types.  out: uint32
 * (N, P, W), equal to ytm_encode of the binned rows. */
int ytm_encode_binarized(ytm_model *m, const void *X, int x_dtype, int64_t N, const void *thresholds,
                         int int_thresholds, int nthr, int kind, int edge_bins, uint32_t *out);

/* Device-resident training / scoring data, so repeated epochs do not re-copy it.
 * encX: uint32 (N, P, W); encY: int32 (N, classes) or NULL for score-only data. */
int ytm_dataset_create(ytm_model *m, const uint32_t *encX, const int32_t *encY, int64_t N,
                       ytm_dataset **out);
void ytm_dataset_destroy(ytm_dataset *ds);

/* fit: BaseTM._fit's per-sample loop (src/cutm/base.py:266-359; kernel.cu pack_clauses
 * :155-204, fast_eval :255-282, select_active :285-316, clause_update :531-613).
 * Samples [first, first+count) of ds, in order.  drop: uint32 (clauses) clause drop mask
 * (base.py:288-293) or NULL for none.  inject: NULL for the counter-based stream, or a
 * float buffer of count sample blocks [sel C*P | q C*K | upd C*K | lit C*K*L] replacing
 * every draw (test mode).  Advances the model's step by count. */
int ytm_fit_dataset(ytm_model *m, const ytm_dataset *ds, int64_t first, int64_t count,
                    const uint32_t *drop, const float *inject);
/* Host-array convenience form of the same (copies encX/encY in, like base.py:275-279). */
int ytm_fit(ytm_model *m, const uint32_t *encX, const int32_t *encY, int64_t N,
            const uint32_t *drop, const float *inject);

/* score: BaseTM._score_batch (src/cutm/base.py:375-420; kernel.cu:319-343).
 * class_sums: float (N, classes) = bias + sum of weights of non-empty firing clauses. */
int ytm_score_dataset(ytm_model *m, const ytm_dataset *ds, float *class_sums);
/* ytm_score_dataset without any device allocation.  No counterpart in the reference: it is
 * for callers that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc).  d_class_sums is a DEVICE pointer to
 * float (N, classes), written with the same values ytm_score_dataset returns.  The
 * model's operands or literal lists and the samples' firing words or int64 class-sum
 * accumulators live in a static per-GPU scratch array of YTM_NOALLOC_SCRATCH_BYTES (32 MiB; it is part of libytm's code object, so every
 * GPU on which the library's kernels are loaded holds it until the process ends, whether or
 * not this entry point is called there); samples go through in passes that fit it.  Models
 * whose matrix operands do not fit are scored on literal lists; YTM_EINVAL when these and one
 * sample's accumulators do not fit either (e.g. one-patch models of more than about 65000 wide
 * clauses).  Calls on one GPU share the array, so overlapping calls
 * would race: the library serialises them per GPU with a lock.  Synchronous on return. */
#define YTM_NOALLOC_SCRATCH_BYTES (32u << 20)
int ytm_score_dataset_noalloc(ytm_model *m, const ytm_dataset *ds, float *d_class_sums);
int ytm_score(ytm_model *m, const uint32_t *encX, int64_t N, float *class_sums);

/* transform / transform_patchwise (src/cutm/base.py:465-542; kernel.cu:346-394).
 * mode 0: out uint32 (N, clauses), 1 where some patch fires;
 * mode 1: out uint32 (N, clauses, P), one value per patch;
 * mode 2: out uint32 (N, clauses, ceil(P/32)), the mode-1 values bit-packed: bit b of word j
 *         is patch 32j + b, bits beyond P are 0 (an option the reference does not have, for
 *         outputs of C*P*N values that would not fit as one uint32 each).
 * Empty clauses output 1.  Samples are processed in chunks, so device memory stays bounded
 * whatever N is. */
int ytm_transform(ytm_model *m, const uint32_t *encX, int64_t N, int mode, uint32_t *out);

/* State accessors (src/cutm/base.py:423-461, 561-593), flat C-order.
 * ta_state: uint32 (clauses, L); weights: float (clauses, classes);
 * patch_weights: int32 (clauses, P); bias: float (classes). */
int ytm_get_ta_state(ytm_model *m, uint32_t *out);
int ytm_set_ta_state(ytm_model *m, const uint32_t *in);
int ytm_get_weights(ytm_model *m, float *out);
int ytm_set_weights(ytm_model *m, const float *in);
int ytm_get_patch_weights(ytm_model *m, int32_t *out);
int ytm_set_patch_weights(ytm_model *m, const int32_t *in);
int ytm_get_bias(ytm_model *m, float *out);

/* ---- Host preprocessing: the binarizers of src/tm_utils/binarizer.py (no model needed).
 *
 * ytm_binarize replaces the transform of Binarizer (binarizer.py:63-86, 107-113) and the
 * binarize_gray / binarize_rgb of ThermometerBinarizer (binarizer.py:9-22): X holds n values
 * of type x_dtype (YTM_DTYPE_*), thresholds nthr values, int64 when int_thresholds else
 * double.  Comparisons are made in int64 when X and the thresholds are integers, else in
 * double (numpy's promotion for these operands).
 *   kind 0, thermometer: out uint32 (n, nthr), out[i][j] = X[i] >= t[j];
 *   kind 1, one-hot: out uint32 (n, nthr - 1 + 2 * edge_bins); the nthr - 1 intervals
 *           t[j] <= X[i] < t[j + 1], preceded by X[i] < t[0] and followed by
 *           X[i] >= t[nthr - 1] when edge_bins.
 * ytm_collapse_bins replaces Binarizer.collapse_bins (binarizer.py:88-129): B uint32
 * (rows, width) -> out int64 (rows): kind 0, the index of the last non-zero value + 1 (0 if
 * none); kind 1, the index of the first maximum; minus 1 when edge_bins. */
int ytm_binarize(const void *X, int x_dtype, int64_t n, const void *thresholds, int int_thresholds, int nthr,
                 int kind, int edge_bins, uint32_t *out);
int ytm_collapse_bins(const uint32_t *B, int64_t rows, int64_t width, int kind, int edge_bins, int64_t *out);

/* ---- From clause outputs to an answer (not in the reference): class sums through weights
 * held in 4 bits, scores shaped by history, bias and grammar, and the choice of an answer.
 *
 * Unlike the calls above these take DEVICE pointers and put their work on `stream` (a
 * hipStream_t of the current device, NULL the default one) without waiting for it: what they
 * read must stay until the stream has passed, and results are there once it has.  They allocate
 * nothing and may be captured into a graph.  Rows may be any distance apart (strides in
 * elements, of codes in bytes; 0 in what is read: one row, or one output's codes or scales, for
 * all); a row's elements follow one another.  Their errors are those of their arguments and of the
 * launch.  What they write must not overlap what they read (adjust_scores in place apart).  Sums are
 * made in f32 and rounded once; results do not depend on the order in which blocks run.
 *
 * ytm_readout: out[n][o] = sum over clauses c of x[n][c] * value(code[o][c]) * scale[o][c / group]
 * for N rows (at most 65535), C clauses (2097120) and K outputs (8388608).  x: YTM_DTYPE_BITS
 * (clause outputs, (N, ceil(C/32)) words; bits past C are ignored), F32 (whose parts below 2^-133
 * are ignored), F16 or BF16 (N, C).  codes: E2M1 floats (codes 0..7 are 0, 0.5, 1, 1.5, 2, 3, 4, 6;
 * 8..15 their negatives), two a byte, the even clause in the low half, 16 ceil(C/32) bytes an
 * output, each output's at a multiple of 16 bytes (codes past C are ignored).  scales:
 * (K, ceil(C/group)), group a multiple of 32.  scales and out: F32, F16 or BF16.  Rows of x, codes
 * and scales are at most 8 MiB apart.  workspace: device memory of ytm_readout_workspace's bytes at
 * a multiple of 16 bytes, for the time of the call's work (NULL where that is 0). */
int ytm_readout_workspace(int x_dtype, int64_t N, int64_t C, int64_t K, int64_t *bytes);
int ytm_readout(const void *x, int x_dtype, int64_t x_stride, int64_t N, int64_t C, const uint8_t *codes,
                int64_t code_stride, const void *scales, int scale_dtype, int64_t scale_stride, int64_t group,
                int64_t K, void *out, int out_dtype, int64_t out_stride, void *workspace, int64_t workspace_bytes,
                void *stream);

/* ytm_adjust_scores: for row n (at most 65535 rows) and answer v of V (at most 8388608), with h
 * the first lengths[n] (NULL: T) entries of tokens[n] (N, T; T at most 2147483647), c the number of
 * h's entries from prompt[n] on (NULL: 0) that are v:
 *   s = score; if v is in h: s = s > 0 ? s / repetition[n] : s * repetition[n];
 *   s = s - frequency[n] * c - presence[n] * (c > 0); s = s + bias[v];
 *   s = -inf if bit v % 32 of allowed word v / 32 is 0.
 * Entries outside 0..V-1 stand for no answer.  Anything NULL is left out; bias_stride or
 * allowed_stride 0: one row for all.  A lengths[n] above T counts as T.  scores and out: F32,
 * F16 or BF16, each its own; out may be scores or bias itself, with elements of the same size and rows
 * of the same distance. */
int ytm_adjust_scores(const void *scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t *tokens,
                      int64_t token_stride, int64_t T, const int32_t *lengths, const int32_t *prompt,
                      const float *repetition, const float *frequency, const float *presence, const float *bias,
                      int64_t bias_stride, const uint32_t *allowed, int64_t allowed_stride, void *out, int out_dtype,
                      int64_t out_stride, void *stream);

/* ytm_choose: one of V (at most 8388608) answers for each of N (2147483647) rows.  With z = score / temperature[n]
 * (NULL: 1; 0 or less: temperature 1 and top_k 1; less than the smallest normal float, or NaN:
 * that; a z that is NaN counts as -inf, one of +inf as the largest float) and the answers in the
 * order of z descending, then index ascending, the filters keep a first part of that order, the
 * first answer always among it:
 *   min_p: z >= max z + log(min_p[n]) (0 or less, or NaN: all; above 1: the first answer alone);
 *   top_k: the first top_k[n] of these (0 or less: all);
 *   top_p: of these, with masses exp(z - max z), those before which less than top_p[n] of the mass
 *   stands (1 or more, or NaN: all).
 * tokens[n] = the index of the largest z + noise[n][v] (NULL: of z) of the kept answers, the
 * lowest of equal ones, and logprobs[n] = z of it - log of the kept answers' sum of exp(z).
 * With standard Gumbel noise -log(-log(u)) that is a draw from softmax(z) over the kept
 * answers.  Noise is finite.  -1 and -inf where no z is above -inf.  workspace: device memory
 * of ytm_choose_workspace's bytes at a multiple of 16 bytes, for the time of the call's work (NULL
 * where that is 0: rows that are short or many). */
int ytm_choose_workspace(int dtype, int64_t N, int64_t V, int64_t *bytes);
int ytm_choose(const void *scores, int dtype, int64_t stride, int64_t N, int64_t V, const float *temperature,
               const int32_t *top_k, const float *top_p, const float *min_p, const float *noise, int64_t noise_stride,
               int32_t *tokens, float *logprobs, void *workspace, int64_t workspace_bytes, void *stream);

/* ---- Adapting a model's answers and learning from them (not in the reference): low-rank
 * adapters beside ytm_readout, losses of answers with the gradient of the scores, and a step of the
 * adapters.  Device pointers, streams, strides, errors and graphs as above.  Sums and states are made in
 * f32 and rounded once; results do not depend on the order in which blocks run.
 *
 * ytm_adapt: with a = which[n] one of M (at most 65535) adapters of rank r (1 to 256),
 *   hidden[n][j] = sum over clauses c of x[n][c] * down[a][j][c]
 *   out[n][o] = scores[n][o] + scale * sum over j of up[a][o][j] * hidden[n][j]
 * for N rows (at most 65535), C clauses (2097120) and K outputs (8388608); where which[n] is outside
 * 0..M-1 the row has no adapter, out is its scores and hidden 0.  x as for ytm_readout (bits past C are
 * ignored).  down: (M, r, C), up: (M, K, r), both of w_dtype, a distance from an adapter to the next and
 * from a row to the next; scores, out and adapters: F32, F16 or BF16.  hidden: f32 (N, r), or NULL.  out
 * may be scores itself, with elements of the same size and rows of the same distance.  workspace: device
 * memory of ytm_adapt_workspace's bytes at a multiple of 16 bytes, for the time of the call's work. */
int ytm_adapt_workspace(int64_t N, int64_t C, int64_t M, int64_t r, int64_t *bytes);
int ytm_adapt(const void *scores, int dtype, int64_t stride, int64_t N, int64_t K, const void *x, int x_dtype,
              int64_t x_stride, int64_t C, const void *down, int64_t down_adapter, int64_t down_rank, const void *up,
              int64_t up_adapter, int64_t up_output, int w_dtype, int64_t M, int64_t r, const int32_t *which,
              float scale, float *hidden, int64_t hidden_stride, void *out, int out_dtype, int64_t out_stride,
              void *workspace, int64_t workspace_bytes, void *stream);

/* ytm_adapt_gradient: of a loss whose gradient by out is grad (N, K), with hidden as ytm_adapt gave it:
 *   d_up[a][o][j] = scale * sum over rows n of a of grad[n][o] * hidden[n][j]
 *   d_down[a][j][c] = sum over rows n of a of x[n][c] * scale * sum over o of grad[n][o] * up[a][o][j]
 * 0 for adapters that no row names.  (The gradient by scores is grad itself.)  Sums with a value that is not
 * finite are infinite or NaN.  d_down (M, r, C) and d_up (M, K, r) are of w_dtype; grad F32, F16 or BF16.
 * Bounds and workspace as for ytm_adapt.
 * ytm_adapt_gradient_as: the same with d_down and d_up of d_dtype, which is w_dtype or F32: means over a batch
 * of unlikely answers are less than the 2^-24 that float16 holds. */
int ytm_adapt_gradient_workspace(int64_t N, int64_t C, int64_t K, int64_t M, int64_t r, int64_t *bytes);
int ytm_adapt_gradient(const void *grad, int dtype, int64_t stride, int64_t N, int64_t K, const void *x, int x_dtype,
                       int64_t x_stride, int64_t C, const void *up, int64_t up_adapter, int64_t up_output, int w_dtype,
                       int64_t M, int64_t r, const int32_t *which, float scale, const float *hidden,
                       int64_t hidden_stride, void *d_down, int64_t d_down_adapter, int64_t d_down_rank, void *d_up,
                       int64_t d_up_adapter, int64_t d_up_output, void *workspace, int64_t workspace_bytes,
                       void *stream);
int ytm_adapt_gradient_as(const void *grad, int dtype, int64_t stride, int64_t N, int64_t K, const void *x, int x_dtype,
                          int64_t x_stride, int64_t C, const void *up, int64_t up_adapter, int64_t up_output,
                          int w_dtype, int64_t M, int64_t r, const int32_t *which, float scale, const float *hidden,
                          int64_t hidden_stride, int d_dtype, void *d_down, int64_t d_down_adapter, int64_t d_down_rank,
                          void *d_up, int64_t d_up_adapter, int64_t d_up_output, void *workspace,
                          int64_t workspace_bytes, void *stream);

/* Both losses take N rows (at most 65535) of V scores (8388608), F32, F16 or BF16, the answer tokens[n]
 * of each, and a temperature (NULL: 1; 0 or less counts as 1, less than the smallest normal float or NaN
 * as that, an infinite one as the largest float).  A score that is NaN counts as -inf, one of +inf as the
 * largest float.  With p = softmax(score / temperature) and lp = log p[tokens[n]], grad (F32, F16 or BF16;
 * scores itself too, with elements of the same size and rows of the same distance) becomes the gradient of the
 * losses' sum by the scores.  A row whose answer is outside 0..V-1 or has a score of -inf is left out: its lp
 * and loss are 0, and so is its gradient.
 *
 * ytm_policy_loss: with ratio = exp(lp - old[n]), d = reference[n] - lp,
 *   losses[n] = weights[n] * (kl * (exp(d) - d - 1)
 *               - min(ratio * advantages[n], clamp(ratio, 1 - low, 1 + high) * advantages[n]))
 * (where the two are equal, the first counts); weights NULL: 1 / N; 0: the row has a loss and gradient of 0,
 * whatever its other numbers; reference NULL: kl must be 0.  Of other rows a number that is NaN makes loss and
 * gradient NaN.
 * logprobs[n] = lp.
 *
 * ytm_preference_loss: rows starts[s] .. starts[s + 1] - 1 are sequence s of 2 pairs (at most 65535),
 * starts (2 pairs + 1) not falling, between 0 and N (elsewhere cut to that; where they fall,
 * results are unspecified).  With l[s] the sum of its rows' lp, of pair p
 *   m = beta * ((l[2p] - reference[2p]) - (l[2p+1] - reference[2p+1]))
 *   losses[p] = ((1 - smoothing) * log(1 + exp(-m)) + smoothing * log(1 + exp(m))) / pairs
 * in which 0 times an infinity (from a reference of -inf) is 0.  logprobs[s] = l[s].  Rows of no sequence are left out.
 *
 * workspace: device memory of the _workspace's bytes at a multiple of 16 bytes, for the time of the
 * call's work (NULL where that is 0). */
int ytm_policy_loss_workspace(int64_t N, int64_t V, int64_t *bytes);
int ytm_policy_loss(const void *scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t *tokens,
                    const float *old, const float *advantages, const float *reference, float kl, float low, float high,
                    const float *weights, const float *temperature, float *losses, float *logprobs, void *grad,
                    int grad_dtype, int64_t grad_stride, void *workspace, int64_t workspace_bytes, void *stream);
int ytm_preference_loss_workspace(int64_t N, int64_t V, int64_t *bytes);
int ytm_preference_loss(const void *scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t *tokens,
                        const int32_t *starts, int64_t pairs, const float *reference, float beta, float smoothing,
                        const float *temperature, float *losses, float *logprobs, void *grad, int grad_dtype,
                        int64_t grad_stride, void *workspace, int64_t workspace_bytes, void *stream);

/* ytm_adamw: a step of AdamW on n (at most 16777216) tensors at once.  Of tensor i it is the step k =
 * ++steps[i], for each element with gradient g
 *   m = beta1 m + (1 - beta1) g; v = beta2 v + (1 - beta2) g^2
 *   p = (1 - rate decay) p - rate / (1 - beta1^k) * m / (sqrt(v / (1 - beta2^k)) + eps)
 * and none where active[i] (NULL: all are) is 0.  rate_at (or NULL) has the rate instead of `rate`.
 * steps (0 or more before the step), active, rate_at: device.  The tensors are in a table
 * that ytm_adamw_table writes to host memory (NULL: says only its bytes and its chunks, which ytm_adamw
 * takes) and that the caller copies to device memory at a multiple of 16 bytes; ytm_adamw writes to it,
 * so two steps of one table follow each other.  parameter: F32, F16 or BF16; gradient: of the same type or
 * F32.  With bits 32 first (m) and second (v) are f32.  With bits 8 they are E4M3 floats (sign, four bits
 * of exponent with bias 7, three of fraction, 127 a NaN) times a power of two for each 256 elements in a
 * row (2^-98 or more; of roots 2^-54 or more but for zeros alone), m itself and v as its root.  What is stored
 * in fewer bits than f32 is rounded up or down at random, with the chances that keep the mean of parameters, of
 * m and of v, from `seed`, the step and the element's place (each tensor before it counts as a multiple of 256
 * long); a v above 0 stays above 0, what is not finite becomes NaN in 8 bits.  Operations are f32, each rounded
 * (of the rate and of k in f64, rounded once), but with bits 8 the quotient, which is within two units in its
 * last place.  The operands of different tensors must not overlap. */
typedef struct {
  void *parameter;
  const void *gradient;
  void *first, *second;
  float *first_scales, *second_scales; /* bits 8: (ceil(count / 256)) each */
  int64_t count;
  int32_t parameter_dtype, gradient_dtype;
} ytm_adamw_tensor;
int ytm_adamw_table(const ytm_adamw_tensor *tensors, int64_t n, int bits, void *table, int64_t *bytes,
                    int64_t *chunks);
int ytm_adamw(void *table, int64_t n, int64_t chunks, int bits, int64_t *steps, const uint8_t *active, double rate,
              const float *rate_at, double beta1, double beta2, double eps, double decay, uint32_t seed, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* YTM_H */

/**
 * vitna_serve.h - Operators for serving several continuations at once, on
 * device memory: attention for a batch whose rows share a long prefix, with
 * or without a sliding window and sinks; the same window over a prompt's
 * chunk; beam search's selection; and the reordering of its sequences'
 * key-value caches. Then the model calls that use them: a cache forked for
 * several sequences, a model's window, and a step of beam search.
 *
 * No counterpart in the reference's interface. The error convention is
 * vitna_hip.h's: false, with a sentence in err[err_len]. The operators take
 * no model: every pointer marked DEVICE is memory of one GPU, the call's work
 * is enqueued on stream (a hipStream_t of that GPU, or NULL for its default
 * stream) and nothing waits or allocates, so that a call can be captured into
 * a HIP graph. What lies in device memory (rows, parents, spans) is read by
 * the kernels when they run and checked there; what the host passes is
 * checked by the call. work is scratch memory for one call at a time: two
 * calls that may run at once, or two graphs, need one each. Its contents mean
 * nothing before or after a call. A call may come from any thread; the GPU it
 * runs on is that of its device pointers, whatever GPU is current.
 */

#ifndef VITNA_SERVE_H
#define VITNA_SERVE_H

#include "vitna_model.h"
#include "vitna_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/** A layer's key-value cache of several sequences, and how it is read.
    Element (sequence, position, head, d) of the keys and of the values lies
    seq * seq_stride + pos * pos_stride + head * head_stride + d elements
    behind k and v. k, v and every stride are whole multiples of 16 bytes,
    pos_stride at most 2^23 elements. */
typedef struct {
    const void* k;             /* DEVICE */
    const void* v;             /* DEVICE */
    vitna_dtype_t dtype;       /* F32, F16 or BF16 */
    size_t n_heads;            /* query heads: a multiple of n_kv_heads, at most 16 of each; head h reads key-value head h / (n_heads / n_kv_heads) */
    size_t n_kv_heads;
    size_t head_dim;           /* 64 or 128 */
    size_t ctx;                /* positions a sequence, at most 2^30 */
    size_t seqs;
    size_t seq_stride, pos_stride, head_stride;
    size_t window;             /* 0: a row at position p sees positions 0 .. p; else the last window of those ... */
    size_t sinks;              /* ... and the first sinks of them, which stay visible */
    float scale;               /* scores are scale q . k; 0: 1 / sqrt(head_dim) */
} vitna_hip_kv_view_t;

/** A row of vitna_hip_attention_rows: the token at position pos of sequence
    seq, whose positions 0 .. shared - 1 are read from sequence base (their
    positions there are the same; shared 0: none). Rows next to each other with the same base and
    shared read those positions once. A row outside the cache (seq or base not a
    sequence, shared below 0, pos not a position: pos -1 is a batch's padding) sees
    nothing. */
typedef struct {
    int32_t seq, pos, base, shared;
} vitna_hip_attention_row_t;

/** Bytes of work that vitna_hip_attention_rows needs for these arguments; 0
    if it refuses them. */
size_t vitna_hip_attention_rows_work(const vitna_hip_kv_view_t* c, size_t n, size_t own_max, size_t shared_max);

/** Attention of n rows (1 <= n <= 65535, n x n_kv_heads at most 2^22), each a token of its own: out[i] =
    softmax(scale q[i] k) v over the positions that row i sees, head by head,
    with float32 sums. q and out are n rows of n_heads x head_dim float32,
    q_stride and out_stride floats apart (0: back to back; multiples of 4).
    out may be q. A row that sees nothing gets zeros. own_max is about how
    many positions a row has of its own (pos + 1 - shared) at most, and shared_max
    the most that rows share (0: read them with the row's own); they size the
    launch, and rows beyond them get the same values, later. The keys and
    values of the positions that a row sees have to be in the cache; what lies
    at the others, infinities and NaN among it, has no effect on the row, but
    for this: where many rows see positions together, their keys and their
    values are taken to within 2^-20 of themselves and 2^-28 of the largest
    finite one of the positions before and around them that any of the rows
    sees. */
bool vitna_hip_attention_rows(const vitna_hip_kv_view_t* c, const float* q, size_t q_stride, const vitna_hip_attention_row_t* rows, size_t n,
                              size_t own_max, size_t shared_max, float* out, size_t out_stride, void* work, size_t work_bytes, void* stream,
                              char* err, size_t err_len);

/** Bytes of work that vitna_hip_attention_run needs; 0 if it refuses. */
size_t vitna_hip_attention_run_work(const vitna_hip_kv_view_t* c, size_t pos0, size_t n);

/** The same for n tokens of one sequence (n <= 2^20, n x n_kv_heads at
    most 2^22), at positions pos0 ..
    pos0 + n - 1: a prompt's chunk, whose keys and values are in the cache. */
bool vitna_hip_attention_run(const vitna_hip_kv_view_t* c, size_t seq, size_t pos0, const float* q, size_t q_stride, size_t n, float* out,
                             size_t out_stride, void* work, size_t work_bytes, void* stream, char* err, size_t err_len);

#define VITNA_HIP_BEAMS_MAX 64

/** Bytes of work that vitna_hip_beam_select needs; 0 if it refuses. */
size_t vitna_hip_beam_select_work(size_t groups, size_t width, size_t vocab, size_t keep);

/** Beam search's selection: for each of groups prompts with width beams (1 ..
    VITNA_HIP_BEAMS_MAX, at most 2^20 beams in all), the keep (1 .. VITNA_HIP_BEAMS_MAX) best of its width
    x vocab continuations. logits is groups x width rows of vocab float32,
    stride floats apart (0: back to back); scores each beam's sum of log
    probabilities so far. Continuation (b, v) is worth
    scores[b] + logits[b][v] - log(sum over u of exp(logits[b][u])). A beam
    with ended[b] not 0 (ended NULL: none) continues by end_token alone, at its score. Largest
    first; of equal values the one of lower b, then of lower v. best (its
    value), parents (its beam, 0 .. width - 1) and tokens are groups x keep.
    A logit of -inf or NaN is no continuation, nor is any of a beam whose
    score is -inf or NaN; where fewer than keep remain the rest is -inf, -1, -1.
    Logits of +inf share a probability of 1. Values of different beams that
    differ by less than about 1e-7 may change places. */
bool vitna_hip_beam_select(const float* logits, size_t stride, size_t vocab, size_t groups, size_t width, size_t keep, const float* scores,
                           const uint8_t* ended, int32_t end_token, float* best, int32_t* parents, int32_t* tokens, void* work,
                           size_t work_bytes, void* stream, char* err, size_t err_len);

/** The caches of groups x width beams after a selection, in place: beam b of
    group g, sequence seqs[g width + b], gets positions spans[g][0] ..
    spans[g][1] - 1 of every layer from the sequence of beam parents[g width +
    b] of its group, as that was before the call. c describes the first of
    layers layers, the next layer_stride elements behind it (c's n_heads,
    window, sinks and scale are not read); its elements do not overlap.
    seqs, parents and spans (groups x 2) are DEVICE; the sequences are
    distinct. A beam whose sequence is outside the cache, whose parent is not
    a beam of its group or whose parent's sequence is outside the cache stays
    as it is; a span is cut to the cache. longest is about the positions of
    the longest span (0: ctx); it sizes the launch, and longer spans are copied too. */
bool vitna_hip_kv_reorder(const vitna_hip_kv_view_t* c, size_t layers, size_t layer_stride, const int32_t* seqs, const int32_t* parents,
                          const int32_t* spans, size_t groups, size_t width, size_t longest, void* stream, char* err, size_t err_len);

/* ---- the same on a model (vitna_cuda_create) ---- */

/** A sliding window for every later step and pass of g: a row at position p
    attends to positions p - window + 1 .. p and to the first sinks of its
    sequence. window 0, or as long as the cache: none (as after
    vitna_cuda_create). Every path honours it except the persistent step
    kernel, whose steps then run the per-layer kernels. Passes of up to
    vitna_hip_set_exact_rows rows still give each row the bits of its own
    step. Keys and values behind the window stay in the cache. */
bool vitna_hip_set_window(struct vitna_cuda_model* g, size_t window, size_t sinks, char* err, size_t err_len);

/** The first n_pos positions of sequence src, every layer, copied into the n
    sequences dst (distinct, none of them src), enqueued on the model's stream.
    Until one of them changes such a position (a row or vitna_hip_kv at it),
    rows steps (vitna_hip_moe_rows_step) whose rows of these sequences stand
    next to each other read the positions once for all of them: the same
    logits to the multi-row kernels' accuracy (two such passes lie within 4e-5
    of max |logit| of each other), not the same bits. */
bool vitna_hip_kv_fork(struct vitna_cuda_model* g, size_t src, size_t n_pos, const int32_t* dst, size_t n, char* err, size_t err_len);

/** One step of beam search for groups prompts with width beams each
    (groups x width rows, at most a pass's): the rows step of rows, the width
    best continuations of each group (as vitna_hip_beam_select chooses them,
    largest first), and the caches for the next step. rows[i] is beam i %
    width of group i / width, each in a sequence of its own. On return rows
    holds the continuations (token, position and the sequence that holds their
    cache), scores their sums of log probabilities, ended whether their last
    token was end_token (-1: there is none), parents (or NULL) the beam each
    came from. The first continuation of a beam stays in its sequence; others
    take the sequences of beams without one, whose positions behind the prefix
    that the group shares (vitna_hip_kv_fork) are copied over. A beam that has
    ended stays as it is, with its score. For a prompt's first step give its
    last token to width sequences that hold the rest, and the scores 0, -inf,
    -inf, ...: all continuations then come from the first. Where fewer than
    width continuations remain, the rest have score -inf and parent -1. */
bool vitna_hip_beam_step(struct vitna_cuda_model* g, vitna_cuda_row_t* rows, size_t groups, size_t width, float* scores, uint8_t* ended,
                         int32_t end_token, int32_t* parents, char* err, size_t err_len);

#ifdef __cplusplus
}
#endif

#endif

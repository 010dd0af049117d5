/**
 * serving.hip - The C entry points of the serving operators
 * (include/vitna_serve.h): their checks, the GPU they run on, and the launch.
 */

#include "serve_kernels.h"
#include "../../include/vitna_serve.h"

#include <algorithm>
#include <stdarg.h>
#include <stdio.h>

static_assert(sizeof(attend_row) == sizeof(vitna_hip_attention_row_t), "the rows are read as they are given");

static bool fail(char* err, size_t len, const char* fmt, ...) {
    if (err && len) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err, len, fmt, ap);
        va_end(ap);
    }
    return false;
}

/* The GPU of a call's pointers, current while the call launches and the caller's again after. */
class on_device {
    int before = -1, mine = -1;

public:
    ~on_device() {
        if (before >= 0 && before != mine) (void)hipSetDevice(before);
    }
    /* p is device memory of the call's GPU (the first one names it) */
    bool holds(const void* p, const char* what, char* err, size_t err_len) {
        if (!p) return fail(err, err_len, "%s is missing", what);
        hipPointerAttribute_t at;
        const hipError_t e = hipPointerGetAttributes(&at, p);
        if (e != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
            (void)hipGetLastError(); /* an address that HIP does not know leaves an error behind */
            return fail(err, err_len, "%s is not device memory", what);
        }
        if (mine < 0) mine = at.device;
        if (at.device != mine) return fail(err, err_len, "%s is on device %d, the call's other memory on device %d", what, at.device, mine);
        return true;
    }
    bool enter(hipStream_t s, char* err, size_t err_len) {
        if (s) {
            hipDevice_t d = -1;
            if (hipStreamGetDevice(s, &d) != hipSuccess) {
                (void)hipGetLastError();
                return fail(err, err_len, "the stream is not usable");
            }
            if (d != mine) return fail(err, err_len, "the stream is on device %d, the call's memory on device %d", (int)d, mine);
        }
        int now = -1;
        hipError_t e = hipGetDevice(&now);
        if (e == hipSuccess && now != mine) e = hipSetDevice(mine);
        if (e != hipSuccess) return fail(err, err_len, "selecting device %d: %s", mine, hipGetErrorString(e));
        before = now;
        return true;
    }
};

static bool launched(hipError_t e, const char* what, char* err, size_t err_len) {
    if (e == hipSuccess) return true;
    if (e == hipErrorInvalidValue) return fail(err, err_len, "%s: a kernel was asked for a shape it does not take", what);
    return fail(err, err_len, "%s: %s (%s)", what, hipGetErrorString(e), hipGetErrorName(e));
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static size_t elem_bytes(int dtype) { return dtype == VITNA_DTYPE_F32 ? 4 : dtype == VITNA_DTYPE_F16 || dtype == VITNA_DTYPE_BF16 ? 2 : 0; }

#define POSITIONS_MAX ((size_t)1 << 30)
/* 64 positions lie within 2^31 bytes, so that kernels reach them with 32-bit offsets */
#define POS_STRIDE_MAX ((size_t)1 << 23)
/* no element of a view lies this far behind its start, so that offsets in bytes stay within 63 bits */
#define EXTENT_MAX ((size_t)1 << 58)

/* Whether the furthest element of n steps of stride stays below EXTENT_MAX, added to *sum. */
static bool extend(size_t n, size_t stride, size_t* sum) {
    if (n > 1 && stride > EXTENT_MAX / (n - 1)) return false;
    *sum += n > 1 ? (n - 1) * stride : 0;
    return *sum <= EXTENT_MAX;
}

static bool check_view(const vitna_hip_kv_view_t* c, char* err, size_t err_len) {
    if (!c) return fail(err, err_len, "no cache");
    const size_t eb = elem_bytes(c->dtype);
    if (!eb) return fail(err, err_len, "a cache of dtype %d; F32, F16 and BF16 are read", (int)c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128) return fail(err, err_len, "heads of %zu dimensions; 64 and 128 are served", c->head_dim);
    if (c->n_kv_heads < 1 || c->n_kv_heads > 4096) return fail(err, err_len, "%zu key-value heads; 1 to 4096 are served", c->n_kv_heads);
    if (c->ctx < 1 || c->ctx > POSITIONS_MAX) return fail(err, err_len, "a cache of %zu positions; 1 to %zu are served", c->ctx, POSITIONS_MAX);
    if (c->seqs < 1 || c->seqs > (size_t)INT32_MAX) return fail(err, err_len, "a cache of %zu sequences", c->seqs);
    const size_t lane = 16 / eb;
    if (c->seq_stride % lane || c->pos_stride % lane || c->head_stride % lane)
        return fail(err, err_len, "strides of %zu, %zu and %zu elements; whole multiples of %zu (16 bytes) are read", c->seq_stride, c->pos_stride,
                    c->head_stride, lane);
    if (c->pos_stride > POS_STRIDE_MAX) return fail(err, err_len, "positions %zu elements apart; at most %zu are read", c->pos_stride, POS_STRIDE_MAX);
    if (!aligned16(c->k) || !aligned16(c->v)) return fail(err, err_len, "the keys and values have to be 16-byte aligned");
    size_t far = c->head_dim;
    if (!extend(c->seqs, c->seq_stride, &far) || !extend(c->ctx, c->pos_stride, &far) || !extend(c->n_kv_heads, c->head_stride, &far))
        return fail(err, err_len, "a cache of %zu x %zu x %zu with strides of %zu, %zu and %zu elements is too large", c->seqs, c->ctx, c->n_kv_heads,
                    c->seq_stride, c->pos_stride, c->head_stride);
    return true;
}

static bool attend_shape(const vitna_hip_kv_view_t* c, size_t n, attend_args* a, char* err, size_t err_len) {
    if (!check_view(c, err, err_len)) return false;
    if (c->n_heads < 1 || c->n_heads % c->n_kv_heads || c->n_heads / c->n_kv_heads > ATTEND_G_MAX)
        return fail(err, err_len, "%zu query heads of %zu key-value heads; 1 to %d of each are served", c->n_heads, c->n_kv_heads, ATTEND_G_MAX);
    /* the launches' threads stay within 32 bits */
    if (n * c->n_kv_heads > ((size_t)1 << 22)) return fail(err, err_len, "%zu rows of %zu key-value heads; %d of both are served", n, c->n_kv_heads, 1 << 22);
    if (!(c->scale >= 0.0f) || c->scale > 3e38f) return fail(err, err_len, "a scale of %g; 0 or a positive number is needed", (double)c->scale);
    *a = attend_args();
    a->k = c->k; a->v = c->v;
    a->seq_stride = c->seq_stride; a->pos_stride = c->pos_stride; a->head_stride = c->head_stride;
    a->dtype = c->dtype; a->n_heads = (int)c->n_heads; a->n_kv = (int)c->n_kv_heads; a->hd = (int)c->head_dim;
    a->ctx = (int)c->ctx; a->seqs = (int)c->seqs;
    a->window = (int)std::min(c->window, POSITIONS_MAX);
    a->sinks = (int)std::min(c->sinks, c->ctx);
    a->scale = c->scale > 0.0f ? c->scale : (float)(c->head_dim == 128 ? 0.08838834764831844 : 0.125);
    a->n = (int)n;
    return true;
}

static bool rows_shape(const vitna_hip_kv_view_t* c, size_t n, size_t own_max, size_t shared_max, attend_args* a, char* err, size_t err_len) {
    if (n < 1 || n > 65535) return fail(err, err_len, "%zu rows; 1 to 65535 are served", n);
    if (!attend_shape(c, n, a, err, err_len)) return false;
    a->own_max = own_max && own_max < c->ctx ? (int)own_max : (int)c->ctx;
    a->shared_max = (int)std::min(shared_max, c->ctx);
    return true;
}

static bool run_shape(const vitna_hip_kv_view_t* c, size_t pos0, size_t n, attend_args* a, char* err, size_t err_len) {
    if (n < 1 || n > ((size_t)1 << 20)) return fail(err, err_len, "%zu rows; 1 to %d are served", n, 1 << 20);
    if (!attend_shape(c, n, a, err, err_len)) return false;
    if (pos0 > c->ctx || n > c->ctx - pos0) return fail(err, err_len, "positions %zu .. %zu: the cache holds %zu", pos0, pos0 + n - 1, c->ctx);
    a->run = 1;
    a->run_pos = (int)pos0;
    a->own_max = (int)(pos0 + n);
    return true;
}

/* Queries, outputs and scratch of an attention call, and the launch. */
static bool attend(attend_args& a, const float* q, size_t q_stride, float* out, size_t out_stride, void* work, size_t work_bytes, void* stream,
                   char* err, size_t err_len) {
    const size_t width = (size_t)a.n_heads * a.hd;
    a.q = q; a.out = out; a.work = work; a.work_bytes = work_bytes;
    a.q_stride = q_stride ? q_stride : width;
    a.out_stride = out_stride ? out_stride : width;
    if (a.q_stride % 4 || a.out_stride % 4 || (a.out_stride < width && a.n > 1) || a.q_stride > EXTENT_MAX / (1 << 20) || a.out_stride > EXTENT_MAX / (1 << 20))
        return fail(err, err_len, "rows %zu and %zu floats apart; a multiple of 4 is needed, the output's at least %zu", a.q_stride, a.out_stride, width);
    if (q == out && a.q_stride != a.out_stride && a.n > 1) return fail(err, err_len, "out is q, with rows %zu floats apart for %zu", a.out_stride, a.q_stride);
    if (!aligned16(q) || !aligned16(out) || !aligned16(work) || !aligned16(a.rows)) return fail(err, err_len, "q, out, rows and work have to be 16-byte aligned");
    const size_t need = attend_work(a);
    if (work_bytes < need) return fail(err, err_len, "%zu bytes of work; the call needs %zu", work_bytes, need);
    on_device at;
    if (!at.holds(a.k, "k", err, err_len) || !at.holds(a.v, "v", err, err_len) || !at.holds(q, "q", err, err_len) || !at.holds(out, "out", err, err_len) ||
        !at.holds(work, "work", err, err_len) || (a.rows && !at.holds(a.rows, "rows", err, err_len)) || !at.enter((hipStream_t)stream, err, err_len))
        return false;
    return launched(launch_attend(a, (hipStream_t)stream), "the attention", err, err_len);
}

extern "C" size_t vitna_hip_attention_rows_work(const vitna_hip_kv_view_t* c, size_t n, size_t own_max, size_t shared_max) {
    attend_args a;
    return rows_shape(c, n, own_max, shared_max, &a, nullptr, 0) ? attend_work(a) : 0;
}

extern "C" bool vitna_hip_attention_rows(const vitna_hip_kv_view_t* c, const float* q, size_t q_stride, const vitna_hip_attention_row_t* rows,
                                         size_t n, size_t own_max, size_t shared_max, float* out, size_t out_stride, void* work,
                                         size_t work_bytes, void* stream, char* err, size_t err_len) {
    attend_args a;
    if (!rows_shape(c, n, own_max, shared_max, &a, err, err_len)) return false;
    if (!rows) return fail(err, err_len, "rows is missing");
    a.rows = reinterpret_cast<const attend_row*>(rows);
    return attend(a, q, q_stride, out, out_stride, work, work_bytes, stream, err, err_len);
}

extern "C" size_t vitna_hip_attention_run_work(const vitna_hip_kv_view_t* c, size_t pos0, size_t n) {
    attend_args a;
    return run_shape(c, pos0, n, &a, nullptr, 0) ? attend_work(a) : 0;
}

extern "C" bool vitna_hip_attention_run(const vitna_hip_kv_view_t* c, size_t seq, size_t pos0, const float* q, size_t q_stride, size_t n, float* out,
                                        size_t out_stride, void* work, size_t work_bytes, void* stream, char* err, size_t err_len) {
    attend_args a;
    if (!run_shape(c, pos0, n, &a, err, err_len)) return false;
    if (seq >= c->seqs) return fail(err, err_len, "sequence %zu: the cache holds %zu", seq, c->seqs);
    a.run_seq = (int)seq;
    return attend(a, q, q_stride, out, out_stride, work, work_bytes, stream, err, err_len);
}

static bool select_shape(size_t groups, size_t width, size_t vocab, size_t keep, char* err, size_t err_len) {
    if (groups < 1 || groups > 65535) return fail(err, err_len, "%zu groups; 1 to 65535 are served", groups);
    if (width < 1 || width > VITNA_HIP_BEAMS_MAX) return fail(err, err_len, "%zu beams; 1 to %d are served", width, VITNA_HIP_BEAMS_MAX);
    if (keep < 1 || keep > VITNA_HIP_BEAMS_MAX) return fail(err, err_len, "%zu results; 1 to %d are served", keep, VITNA_HIP_BEAMS_MAX);
    if (groups * width > ((size_t)1 << 20)) return fail(err, err_len, "%zu groups of %zu beams; %d beams in all are served", groups, width, 1 << 20);
    if (vocab < 1 || vocab > ((size_t)1 << 24)) return fail(err, err_len, "a vocabulary of %zu; 1 to %d are served", vocab, 1 << 24);
    return true;
}

extern "C" size_t vitna_hip_beam_select_work(size_t groups, size_t width, size_t vocab, size_t keep) {
    return select_shape(groups, width, vocab, keep, nullptr, 0) ? beam_select_work((int)groups, (int)width, vocab, (int)keep) : 0;
}

extern "C" bool vitna_hip_beam_select(const float* logits, size_t stride, size_t vocab, size_t groups, size_t width, size_t keep,
                                      const float* scores, const uint8_t* ended, int32_t end_token, float* best, int32_t* parents,
                                      int32_t* tokens, void* work, size_t work_bytes, void* stream, char* err, size_t err_len) {
    if (!select_shape(groups, width, vocab, keep, err, err_len)) return false;
    if (!stride) stride = vocab;
    if (stride < vocab || stride > EXTENT_MAX / (65535 * VITNA_HIP_BEAMS_MAX)) return fail(err, err_len, "rows %zu floats apart for a vocabulary of %zu", stride, vocab);
    if (ended && (end_token < 0 || (size_t)end_token >= vocab)) return fail(err, err_len, "token %d is outside the vocabulary of %zu", end_token, vocab);
    if (((uintptr_t)logits | (uintptr_t)scores | (uintptr_t)best | (uintptr_t)parents | (uintptr_t)tokens) & 3 || !aligned16(work))
        return fail(err, err_len, "the arrays have to be 4-byte aligned, work 16-byte");
    const size_t need = beam_select_work((int)groups, (int)width, vocab, (int)keep);
    if (work_bytes < need) return fail(err, err_len, "%zu bytes of work; the call needs %zu", work_bytes, need);
    on_device at;
    if (!at.holds(logits, "logits", err, err_len) || !at.holds(scores, "scores", err, err_len) || (ended && !at.holds(ended, "ended", err, err_len)) ||
        !at.holds(best, "best", err, err_len) || !at.holds(parents, "parents", err, err_len) || !at.holds(tokens, "tokens", err, err_len) ||
        !at.holds(work, "work", err, err_len) || !at.enter((hipStream_t)stream, err, err_len))
        return false;
    beam_select_args a = {};
    a.logits = logits; a.stride = stride; a.vocab = vocab;
    a.groups = (int)groups; a.width = (int)width; a.keep = (int)keep;
    a.scores = scores; a.ended = ended; a.end_token = end_token;
    a.best = best; a.parents = parents; a.tokens = tokens; a.work = work;
    return launched(launch_beam_select(a, (hipStream_t)stream), "the selection", err, err_len);
}

extern "C" bool vitna_hip_kv_reorder(const vitna_hip_kv_view_t* c, size_t layers, size_t layer_stride, const int32_t* seqs, const int32_t* parents,
                                     const int32_t* spans, size_t groups, size_t width, size_t longest, void* stream, char* err,
                                     size_t err_len) {
    if (!check_view(c, err, err_len)) return false;
    if (groups < 1 || groups > 65535) return fail(err, err_len, "%zu groups; 1 to 65535 are served", groups);
    if (width < 1 || width > VITNA_HIP_BEAMS_MAX) return fail(err, err_len, "%zu beams; 1 to %d are served", width, VITNA_HIP_BEAMS_MAX);
    if (layers < 1 || layers > 32767) return fail(err, err_len, "%zu layers; 1 to 32767 are served", layers);
    const size_t eb = elem_bytes(c->dtype);
    size_t far = 0;
    if (layer_stride % (16 / eb) || !extend(layers, layer_stride, &far)) return fail(err, err_len, "layers %zu elements apart", layer_stride);
    /* a thread writes what no other reads: the elements may not overlap */
    struct { size_t n, stride; } dims[4] = {{c->n_kv_heads, c->head_stride}, {c->ctx, c->pos_stride}, {layers, layer_stride}, {c->seqs, c->seq_stride}};
    std::sort(dims, dims + 4, [](const auto& x, const auto& y) { return x.stride < y.stride; });
    size_t block = c->head_dim;
    for (const auto& d : dims) {
        if (d.n < 2) continue;
        if (d.stride < block) return fail(err, err_len, "a cache whose elements overlap cannot be reordered in place");
        if (!extend(d.n, d.stride, &block)) return fail(err, err_len, "the cache is too large");
    }
    if (((uintptr_t)seqs | (uintptr_t)parents | (uintptr_t)spans) & 3) return fail(err, err_len, "seqs, parents and spans have to be 4-byte aligned");
    on_device at;
    if (!at.holds(c->k, "k", err, err_len) || !at.holds(c->v, "v", err, err_len) || !at.holds(seqs, "seqs", err, err_len) ||
        !at.holds(parents, "parents", err, err_len) || !at.holds(spans, "spans", err, err_len) || !at.enter((hipStream_t)stream, err, err_len))
        return false;
    kv_reorder_args a = {};
    a.k = (char*)const_cast<void*>(c->k); a.v = (char*)const_cast<void*>(c->v);
    a.seq_bytes = c->seq_stride * eb; a.layer_bytes = layer_stride * eb; a.pos_bytes = c->pos_stride * eb; a.head_bytes = c->head_stride * eb;
    a.dim_bytes = c->head_dim * eb;
    a.n_kv = (int)c->n_kv_heads; a.ctx = (int)c->ctx; a.seqs = (int)c->seqs; a.layers = (int)layers;
    a.list = seqs; a.parents = parents; a.spans = spans;
    a.groups = (int)groups; a.width = (int)width;
    a.longest = (int)(longest && longest < c->ctx ? longest : c->ctx);
    return launched(launch_kv_reorder(a, (hipStream_t)stream), "the reordering", err, err_len);
}

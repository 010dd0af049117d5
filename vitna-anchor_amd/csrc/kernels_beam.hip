/**
 * kernels_beam.hip - Beam search's selection over beams and vocabulary, and
 * the reordering of the beams' key-value caches (include/vitna_serve.h).
 */

#include "serve_kernels.h"

#include <algorithm>
#include <type_traits>

/* ---- selection ----
   Two kernels. beam_scan_kernel reads each beam's logits once: a block takes a slice, and leaves the slice's maximum,
   its sum of exponentials and its `keep` largest logits in order. beam_pick_kernel, a block a group, adds the sums
   up, gives those logits their values in 64 bits (two beams' values can lie as near as they like, and which is larger
   decides) and ranks the ones that can be among the group's `keep` best.

   The slice's largest: every lane's values are four sets, and the keep largest values of a wave's 4096 (or 1024) are
   at least as large as the keep-th largest of its 256 sets' maxima. That bound is found by halving over the values'
   order (20 steps of four compares and four counts), the largest of the four waves' bounds holds for the block, and
   one and a half to four times keep values pass it: each counts those before it. Where more than BEAM_CAP pass (many
   equal values) the block picks its keep one by one. */

#define BEAM_WAVES 4
#define BEAM_CAP 128 /* a wave's */

/* float order as unsigned order, no NaN */
__device__ __forceinline__ uint32_t beam_order(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ unsigned long long beam_order64(double x) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return u ^ (u >> 63 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double beam_value64(unsigned long long o) { return __longlong_as_double((long long)(o >> 63 ? o ^ (1ull << 63) : ~o)); }

/* A continuation's place in the order of equal values: its beam, then its token (below 2^24). */
__device__ __forceinline__ int beam_index(int b, int v) { return b << 24 | v; }

struct beam_cand {
    float x; /* a logit, -inf: none */
    int v;   /* its token */
};

/* A candidate as one number: the earlier, the larger. */
__device__ __forceinline__ uint64_t beam_key(float x, int v) { return (uint64_t)beam_order(x == 0.0f ? 0.0f : x) << 32 | (uint32_t)~v; }
__device__ __forceinline__ beam_cand beam_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return beam_cand{__uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o), (int)~(uint32_t)key};
}

/* What beam_scan_kernel leaves: (maximum, sum) of [rows][splits], then beam_cand of [rows][splits][keep]. */
static __host__ __device__ size_t beam_sums_bytes(size_t slices) { return (slices * sizeof(float2) + 255) & ~(size_t)255; }

/* x at i comes before y at j: larger, or equal and of lower index */
__device__ __forceinline__ bool beam_before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

/* Bound by the logits' bytes where they are many: 64 rows of 151936, 39 MB in 14-16 us, 2.4-2.8 TB/s; by the chain of its
   steps where they are few (4 rows: 9 us, with slices of 16 a lane 7). */
template <int E, bool VEC>
__global__ __launch_bounds__(64 * BEAM_WAVES) void beam_scan_kernel(beam_select_args a, int splits) {
    __shared__ float sm[BEAM_WAVES], ss[BEAM_WAVES];
    __shared__ uint32_t st[BEAM_WAVES];
    __shared__ int sn[BEAM_WAVES];
    __shared__ uint64_t sc[BEAM_WAVES][BEAM_CAP]; /* beam_key */
    const int split = blockIdx.x % splits, row = blockIdx.x / splits, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    if (a.ended && a.ended[row]) return; /* its one continuation needs no logits */
    beam_cand* out = reinterpret_cast<beam_cand*>(static_cast<char*>(a.work) + beam_sums_bytes((size_t)a.groups * a.width * splits)) +
                     (size_t)blockIdx.x * a.keep;
    const float* x = a.logits + (size_t)row * a.stride;
    const int V = (int)a.vocab, first = (split * BEAM_WAVES + wave) * 64 * E;
    /* value 4 e + j of a lane: VEC token first + 256 e + 4 lane + j, else first + 64 (4 e + j) + lane */
    auto token = [&](int e, int j) { return VEC ? first + 256 * e + 4 * lane + j : first + 64 * (4 * e + j) + lane; };
    float v[E / 4][4];
    if (first + 64 * E <= V) {
#pragma unroll
        for (int e = 0; e < E / 4; e++) {
            if constexpr (VEC) {
                const float4 q = *reinterpret_cast<const float4*>(x + token(e, 0));
                v[e][0] = q.x; v[e][1] = q.y; v[e][2] = q.z; v[e][3] = q.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[e][j] = x[token(e, j)];
            }
        }
    } else { /* the row's end */
#pragma unroll
        for (int e = 0; e < E / 4; e++)
#pragma unroll
            for (int j = 0; j < 4; j++) v[e][j] = token(e, j) < V ? x[token(e, j)] : -INFINITY;
    }
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < E / 4; e++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[e][j] = fmaxf(v[e][j], -INFINITY); /* a NaN is no continuation */
            top[j] = fmaxf(top[j], v[e][j]);
        }
    const float m = wave_max_dpp(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    /* sum of exp(x - m): log2(e) in two parts, so that the argument is off by its own rounding alone */
    float s = 0.0f;
    if (m > -INFINITY && m < INFINITY) {
#pragma unroll
        for (int e = 0; e < E / 4; e++) {
            float t[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float d = v[e][j] - m;
                t[j] = __builtin_amdgcn_exp2f(fmaf(d, 1.44269502162933349609f, d * 1.92596299112661746887e-8f));
            }
            s += (t[0] + t[1]) + (t[2] + t[3]);
        }
    } else if (m == INFINITY) { /* those alone count */
#pragma unroll 1
        for (int e = 0; e < E / 4; e++)
            for (int j = 0; j < 4; j++) {
                const int i = token(e, j);
                if (i < V && x[i] == INFINITY) s += 1.0f;
            }
    }
    s = wave_sum_dpp(s);
    /* the bound: the largest with at least keep of the wave's 256 maxima at or above it, nearly */
    uint32_t o[4], lo, hi = beam_order(m);
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = beam_order(top[j]);
    auto above = [&](uint32_t t) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) n += __builtin_popcountll(__ballot(o[j] >= t));
        return n;
    };
    {
        /* from the smallest of the lanes' maxima, which 64 of them reach */
        lo = ~wave_umax(~max(max(o[0], o[1]), max(o[2], o[3])));
        for (int step = 0; step < 20 && lo < hi; step++) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            const int n = above(mid);
            if (n >= a.keep) {
                lo = mid;
                if (n == a.keep) break;
            } else {
                hi = mid - 1;
            }
        }
    }
    if (lane == 0) {
        sm[wave] = m;
        ss[wave] = s;
        st[wave] = lo;
    }
    __syncthreads();
    lo = max(max(st[0], st[1]), max(st[2], st[3]));
    const float bound = fmaxf(__uint_as_float(lo >> 31 ? lo ^ 0x80000000u : ~lo), -3.402823466e38f);
    if (tid == 0) {
        float M = -INFINITY, S = 0.0f;
        for (int w = 0; w < BEAM_WAVES; w++) M = fmaxf(M, sm[w]);
        for (int w = 0; w < BEAM_WAVES; w++)
            if (ss[w] > 0.0f) S += ss[w] * (sm[w] == M ? 1.0f : expf(sm[w] - M));
        static_cast<float2*>(a.work)[blockIdx.x] = make_float2(M, S);
    }
    /* the wave's that reach it */
    int mine = 0;
#pragma unroll
    for (int e = 0; e < E / 4; e++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint64_t mask = __ballot(v[e][j] >= bound);
            if (mask) {
                const int at = mine + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
                if (v[e][j] >= bound && at < BEAM_CAP) sc[wave][at] = beam_key(v[e][j], token(e, j));
                mine += __builtin_popcountll(mask);
            }
        }
    if (lane == 0) sn[wave] = mine;
    __syncthreads();
    int n = 0, most = 0;
#pragma unroll
    for (int w = 0; w < BEAM_WAVES; w++) {
        n += sn[w];
        most = max(most, sn[w]);
    }
    for (int i = n + tid; i < a.keep; i += 64 * BEAM_WAVES) out[i] = beam_cand{-INFINITY, INT32_MAX};
    if (most <= BEAM_CAP) {
        /* each wave its own in order, then a candidate's place among the others' by halving */
        uint64_t key[BEAM_CAP / 64];
        int rank[BEAM_CAP / 64];
#pragma unroll
        for (int u = 0; u < BEAM_CAP / 64; u++) {
            key[u] = lane + 64 * u < mine ? sc[wave][lane + 64 * u] : 0;
            rank[u] = 0;
        }
        int j = 0;
        for (; j + 4 <= mine; j += 4) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint64_t other = sc[wave][j + q];
#pragma unroll
                for (int u = 0; u < BEAM_CAP / 64; u++) rank[u] += other > key[u] ? 1 : 0;
            }
        }
        for (; j < mine; j++) {
            const uint64_t other = sc[wave][j];
#pragma unroll
            for (int u = 0; u < BEAM_CAP / 64; u++) rank[u] += other > key[u] ? 1 : 0;
        }
        /* LDS operations of one wave complete in order */
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int u = 0; u < BEAM_CAP / 64; u++)
            if (lane + 64 * u < mine) sc[wave][rank[u]] = key[u];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < BEAM_CAP / 64; u++) {
            if (lane + 64 * u >= mine || rank[u] >= a.keep) continue;
            int place = rank[u];
            for (int o = 1; o < BEAM_WAVES; o++) {
                const int w = (wave + o) & (BEAM_WAVES - 1);
                int lo_ = 0, hi_ = sn[w];
                while (lo_ < hi_) {
                    const int mid = (lo_ + hi_) >> 1;
                    if (sc[w][mid] > key[u]) lo_ = mid + 1;
                    else hi_ = mid;
                }
                place += lo_;
            }
            if (place < a.keep) out[place] = beam_of(key[u]);
        }
        return;
    }
    /* many alike: the keep first of them, one a round */
    __shared__ float rx[BEAM_WAVES];
    __shared__ int ri[BEAM_WAVES];
    float lx = INFINITY;
    int li = -1;
    for (int round = 0; round < a.keep; round++) {
        float bx = -INFINITY;
        int bi = INT32_MAX;
#pragma unroll
        for (int e = 0; e < E / 4; e++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float y = v[e][j];
                const int i = token(e, j);
                if (y > -INFINITY && beam_before(lx, li, y, i) && beam_before(y, i, bx, bi)) { bx = y; bi = i; }
            }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const float y = __shfl_xor(bx, d, WAVE);
            const int i = __shfl_xor(bi, d, WAVE);
            if (beam_before(y, i, bx, bi)) { bx = y; bi = i; }
        }
        if (lane == 0) { rx[wave] = bx; ri[wave] = bi; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < BEAM_WAVES; w++)
            if (beam_before(rx[w], ri[w], bx, bi)) { bx = rx[w]; bi = ri[w]; }
        __syncthreads();
        if (tid == 0) out[round] = beam_cand{bx, bi};
        lx = bx;
        li = bi;
    }
}

#define PICK_THREADS 1024
#define PICK_WAVES (PICK_THREADS / 64)
#define PICK_HELD 7168 /* candidates that are kept in LDS */
#define PICK_BINS 2048
#define PICK_CAP 512   /* continuations that are ranked by counting, at most */
#define PICK_FEW 96    /* and without cutting them first (with 512: 8 beams of 16 kept 24 us for 21, 8 groups of those 26 for 23; with 32: 15 for 13 where 8 are kept) */

/* Latency: a block a group, its slices' sums and candidates (one load each), the bound, the candidates that reach it, their
   ranks. 5 us for 4 beams of 151936, 9 for 8, 15 for 32 beams of 40000 with 64 kept. */
__global__ __launch_bounds__(PICK_THREADS) void beam_pick_kernel(beam_select_args a, int splits) {
    __shared__ beam_cand s_cand[PICK_HELD];
    __shared__ double s_score[64], s_log[64]; /* of a beam: its score (-inf: it has no continuations), log of its sum of exponentials */
    __shared__ unsigned long long s_bound, s_top; /* keep of some beam's continuations are worth this or more; the best is worth (in order) */
    __shared__ float s_most[64];              /* its largest logit */
    __shared__ int s_hist[PICK_BINS], s_wave[PICK_WAVES], s_found[2], s_n;
    __shared__ double r_v[PICK_WAVES];
    __shared__ int r_i[PICK_WAVES];
    __shared__ double c_v[PICK_CAP];
    __shared__ int c_i[PICK_CAP];
    const int group = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, W = a.width, K = a.keep;
    const size_t slices = (size_t)a.groups * W * splits;
    const float2* sums = static_cast<const float2*>(a.work) + (size_t)group * W * splits;
    const beam_cand* cands = reinterpret_cast<const beam_cand*>(static_cast<const char*>(a.work) + beam_sums_bytes(slices)) + (size_t)group * W * splits * K;
    const int row_cands = splits * K, total = W * row_cands;
    if (tid == 0) {
        s_bound = s_top = 0;
        s_n = 0;
    }
    __syncthreads();
    const bool held = total <= PICK_HELD;
    if (held) {
        constexpr int N = PICK_HELD / PICK_THREADS;
        beam_cand c[N]; /* all asked for at once */
#pragma unroll
        for (int u = 0; u < N; u++)
            if (tid + PICK_THREADS * u < total) c[u] = cands[tid + PICK_THREADS * u];
#pragma unroll
        for (int u = 0; u < N; u++)
            if (tid + PICK_THREADS * u < total) s_cand[tid + PICK_THREADS * u] = c[u];
    }
    /* sixteen lanes a beam */
    {
        const int b = tid >> 4, l = tid & 15, row = group * W + b;
        const bool there = b < W;
        const float score = there ? a.scores[row] : -INFINITY;
        const bool ended = there && a.ended && a.ended[row]; /* its slices hold nothing */
        float2 t[4];
        float least = -INFINITY, m = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            t[u] = make_float2(-INFINITY, 0.0f);
            if (there && l + 16 * u < splits) {
                t[u] = sums[b * splits + l + 16 * u];
                least = fmaxf(least, cands[(b * splits + l + 16 * u) * K + K - 1].x);
            }
            m = fmaxf(m, t[u].x);
        }
        if (there)
            for (int i = l + 64; i < splits; i += 16) {
                m = fmaxf(m, sums[b * splits + i].x);
                least = fmaxf(least, cands[(b * splits + i) * K + K - 1].x);
            }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            m = fmaxf(m, __shfl_xor(m, d, WAVE));
            least = fmaxf(least, __shfl_xor(least, d, WAVE));
        }
        double s = 0.0;
        auto add = [&](float2 u) {
            if (u.y > 0.0f) s += (double)(u.y * (u.x == m ? 1.0f : expf(u.x - m)));
        };
#pragma unroll
        for (int u = 0; u < 4; u++) add(t[u]);
        if (there)
            for (int i = l + 64; i < splits; i += 16) add(sums[b * splits + i]);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) s += __shfl_xor(s, d, WAVE);
        if (there && l == 0) {
            const double log_s = log(s);
            const bool on = score > -INFINITY && !ended;
            s_score[b] = on ? (double)score : -INFINITY;
            s_most[b] = m;
            s_log[b] = log_s;
            const double worth = (double)score + ((least == m ? 0.0 : (double)least - (double)m) - log_s);
            if (on && least > -INFINITY && worth == worth) atomicMax(&s_bound, beam_order64(worth));
            const double best = ended ? (double)score : (double)score - log_s; /* of the largest logit */
            if (score > -INFINITY && best == best) atomicMax(&s_top, beam_order64(best));
        }
    }
    __syncthreads();
    const double bound = s_bound ? beam_value64(s_bound) : -INFINITY;
    /* every continuation that reaches the bound, to f(value, index) */
    auto one = [&](int at, beam_cand t, auto f) {
        const int b = at / row_cands;
        const double score = s_score[b];
        if (!(score > -INFINITY) || !(t.x > -INFINITY)) return;
        const double v = score + ((t.x == s_most[b] ? 0.0 : (double)t.x - (double)s_most[b]) - s_log[b]);
        if (v > -INFINITY && v >= bound) f(v, beam_index(b, t.v));
    };
    auto each = [&](auto f) {
        for (int at = tid; at < total; at += PICK_THREADS) one(at, held ? s_cand[at] : cands[at], f);
        if (a.ended && tid < W && a.ended[group * W + tid]) {
            const double v = (double)a.scores[group * W + tid];
            if (v > -INFINITY && v >= bound) f(v, beam_index(tid, a.end_token));
        }
    };
    float* best = a.best + (size_t)group * K;
    int *parents = a.parents + (size_t)group * K, *tokens = a.tokens + (size_t)group * K;
    auto put = [&](int at, double v, int i) {
        best[at] = (float)v;
        parents[at] = i >> 24;
        tokens[at] = i & 0xffffff;
    };
    auto none_from = [&](int n) {
        for (int j = n + tid; j < K; j += PICK_THREADS) {
            best[j] = -INFINITY;
            parents[j] = -1;
            tokens[j] = -1;
        }
    };
    /* the n continuations of c_v and c_i to their places: several threads count those before one */
    auto rank_all = [&](int n) {
        int parts = 1;
        while (parts < 16 && n * parts * 2 <= PICK_THREADS) parts *= 2;
        for (int i = tid; i < n; i += PICK_THREADS) s_hist[i] = 0;
        __syncthreads();
        const int i = tid / parts;
        if (i < n) {
            const double v = c_v[i];
            const int at = c_i[i];
            int before = 0;
            int j = tid % parts;
            for (; j + 3 * parts < n; j += 4 * parts) {
                double w[4];
                int k[4];
#pragma unroll
                for (int u = 0; u < 4; u++) { w[u] = c_v[j + u * parts]; k[u] = c_i[j + u * parts]; }
#pragma unroll
                for (int u = 0; u < 4; u++) before += (int)(w[u] > v) | ((int)(w[u] == v) & (int)(k[u] < at));
            }
            for (; j < n; j += parts) before += (int)(c_v[j] > v) | ((int)(c_v[j] == v) & (int)(c_i[j] < at));
            if (before) atomicAdd(&s_hist[i], before);
        }
        __syncthreads();
        if (tid < n && s_hist[tid] < K) put(s_hist[tid], c_v[tid], c_i[tid]);
        none_from(n);
    };
    /* Collected once whole; if they are many (beams as good as each other, equal values), they are cut by their distance t
       to the largest, in bins: those with t < from + width are kept, the bin that holds the keep-th is cut again while
       they are many, and the kept are collected. All of them lie above some value, so the keep best are among them if
       they are enough (a value on a bin's edge may fall to either side). */
    const double most = beam_value64(s_top), least = fmax(bound, most - 100.0);
    const double scale = most > least && most < INFINITY ? PICK_BINS / (most - least) : 0.0;
    auto below = [&](double v) { return v == most ? 0.0 : fmin(fmax((most - v) * scale, 0.0), (double)PICK_BINS); };
    double limit = INFINITY;
    int keep = K;
    for (bool whole = true;; whole = false) {
        each([&](double v, int i) {
            if (below(v) < limit) {
                const int at = atomicAdd(&s_n, 1); /* in any order: they are ranked */
                if (at < PICK_CAP) { c_v[at] = v; c_i[at] = i; }
            }
        });
        __syncthreads();
        const int many = s_n;
        if (whole) keep = min(K, many);
        if (many <= (whole ? PICK_FEW : PICK_CAP) && many >= keep) {
            rank_all(many);
            return;
        }
        if (!whole) break;
        double from = 0.0, width = PICK_BINS + 1.0;
        int before = 0, kept = many;
        for (int level = 0; level < 5 && kept > PICK_FEW; level++) {
            const double bins = PICK_BINS / width;
            for (int i = tid; i < PICK_BINS; i += PICK_THREADS) s_hist[i] = 0;
            if (tid == 0) { s_found[0] = 0; s_found[1] = before; s_n = kept; }
            __syncthreads();
            each([&](double v, int) {
                const double t = (below(v) - from) * bins;
                if (t >= 0.0 && t < PICK_BINS) atomicAdd(&s_hist[(int)t], 1);
            });
            __syncthreads();
            /* two bins a thread: the bin where before + the counts so far reaches keep */
            const int h0 = s_hist[2 * tid], h1 = s_hist[2 * tid + 1];
            int run = h0 + h1;
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(run, d, WAVE);
                if (lane >= d) run += o;
            }
            if (lane == 63) s_wave[wave] = run;
            __syncthreads();
            int at = before;
            for (int w = 0; w < wave; w++) at += s_wave[w];
            const int b0 = at + run - h0 - h1, b1 = b0 + h0, b2 = b1 + h1; /* before bin 2 tid, before 2 tid + 1, behind it */
            if (b0 < keep && b1 >= keep) { s_found[0] = 2 * tid; s_found[1] = b0; s_n = b1; }
            if (b1 < keep && b2 >= keep) { s_found[0] = 2 * tid + 1; s_found[1] = b1; s_n = b2; }
            __syncthreads();
            from += s_found[0] / bins;
            width /= PICK_BINS;
            before = s_found[1];
            kept = s_n;
            __syncthreads();
        }
        limit = from + width;
        if (tid == 0) s_n = 0;
        __syncthreads();
    }
    /* more alike than can be ranked so: one a round */
    double last = INFINITY;
    int last_i = -1;
    for (int round = 0; round < keep; round++) {
        double bv = -INFINITY;
        int bi = INT32_MAX;
        each([&](double v, int i) {
            if ((v < last || (v == last && i > last_i)) && (v > bv || (v == bv && i < bi))) { bv = v; bi = i; }
        });
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double v = __shfl_xor(bv, d, WAVE);
            const int i = __shfl_xor(bi, d, WAVE);
            if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; }
        }
        __syncthreads();
        if (lane == 0) { r_v[wave] = bv; r_i[wave] = bi; }
        __syncthreads();
        for (int w = 0; w < PICK_WAVES; w++)
            if (r_v[w] > bv || (r_v[w] == bv && r_i[w] < bi)) { bv = r_v[w]; bi = r_i[w]; }
        if (tid == 0) put(round, bv, bi);
        last = bv;
        last_i = bi;
    }
    none_from(keep);
}

/* Values a lane of the scan: 64 where that leaves most compute units a block, or where slices of 16 would be so many a group
   that the pick of their candidates costs more than the scan gains (112 of 64 are what it holds in LDS); else 16. In us of a
   call, 16 and 64 (groups x width, vocabulary, keep): 1 x 2, 151936, 4: 11.6, 13.8; 1 x 4, 151936, 8 (152 slices): 15.9, 14.9;
   1 x 8, 151936, 16: 20.6, 18.5; 1 x 8, 32000, 16 (64 slices): 15.8, 16.3; 16 x 4, 32000, 8: 13.6, 15.4; 32 x 4, 32000, 8:
   16.0, 15.5; 8 x 8, 151936, 16: 36, 23. */
static int beam_lane_values(int rows, int width, size_t vocab) {
    const size_t small = (vocab + BEAM_WAVES * 64 * 16 - 1) / (BEAM_WAVES * 64 * 16);
    return (size_t)rows * vocab >= (size_t)224 * BEAM_WAVES * 64 * 64 || (size_t)width * small * 64 > PICK_HELD ? 64 : 16;
}
static int beam_splits(int rows, int width, size_t vocab) {
    const size_t slice = (size_t)BEAM_WAVES * 64 * beam_lane_values(rows, width, vocab);
    return (int)((vocab + slice - 1) / slice);
}

size_t beam_select_work(int groups, int width, size_t vocab, int keep) {
    const size_t slices = (size_t)groups * width * beam_splits(groups * width, width, vocab);
    return beam_sums_bytes(slices) + slices * keep * sizeof(beam_cand);
}

hipError_t launch_beam_select(const beam_select_args& a, hipStream_t s) {
    if (a.groups < 1 || a.width < 1 || a.width > 64 || a.keep < 1 || a.keep > 64) return hipErrorInvalidValue;
    const int rows = a.groups * a.width, splits = beam_splits(rows, a.width, a.vocab), E = beam_lane_values(rows, a.width, a.vocab);
    if ((size_t)rows * splits > ((size_t)1 << 23)) return hipErrorInvalidValue; /* threads of a launch stay within 32 bits */
    const int grid = rows * splits;
    const bool vec = ((uintptr_t)a.logits & 15) == 0 && a.stride % 4 == 0;
    if (E == 64) {
        if (vec) beam_scan_kernel<64, true><<<grid, 64 * BEAM_WAVES, 0, s>>>(a, splits);
        else beam_scan_kernel<64, false><<<grid, 64 * BEAM_WAVES, 0, s>>>(a, splits);
    } else {
        if (vec) beam_scan_kernel<16, true><<<grid, 64 * BEAM_WAVES, 0, s>>>(a, splits);
        else beam_scan_kernel<16, false><<<grid, 64 * BEAM_WAVES, 0, s>>>(a, splits);
    }
    beam_pick_kernel<<<a.groups, PICK_THREADS, 0, s>>>(a, splits);
    return hipGetLastError();
}

/* ---- reordering ----
   A thread takes the same few bytes of every beam of a group: all that moves is read before any is written, so a beam
   may take another's place while that takes a third's, and no thread waits for another. What it takes lies at the same
   place in every layer, so a block walks over layers with its beams and offsets at hand. Bound by memory: half a beam's
   worth is read and half written for each that changes (8 groups of 8 beams over 24 layers, 830 MB in 160-180 us, 4.6-5.2
   TB/s). */

typedef u32x4 piece_t; /* what a thread takes of a beam, of 64 beams too (400 registers; pieces of 8 bytes: 33 beams 28 us for 17, 64 beams 36 for 29) */

template <int W>
__global__ __launch_bounds__(256) void kv_reorder_kernel(kv_reorder_args a) {
    __shared__ int s_from[W], s_to[W];
    const int group = blockIdx.z, tid = threadIdx.x;
    if (tid < W) {
        int from = -1, to = -1;
        if (tid < a.width) {
            const int p = a.parents[group * a.width + tid];
            to = a.list[group * a.width + tid];
            if (p >= 0 && p < a.width && p != tid) from = a.list[group * a.width + p];
            if (from < 0 || from >= a.seqs || to < 0 || to >= a.seqs) from = -1;
        }
        s_from[tid] = from;
        s_to[tid] = to;
    }
    const int first = max(a.spans[2 * group], 0), last = min(a.spans[2 * group + 1], a.ctx);
    const int head_pieces = (int)(a.dim_bytes / sizeof(piece_t)), pieces = a.n_kv * head_pieces;
    const int64_t many = last > first ? (int64_t)(last - first) * pieces : 0;
    __syncthreads();
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < many; i += (int64_t)gridDim.x * 256) {
        const int64_t pos = many <= INT32_MAX ? first + (int)i / pieces : first + i / pieces;
        const int piece = (int)(i - (pos - first) * pieces);
        const size_t at = (size_t)pos * a.pos_bytes + (size_t)(piece / head_pieces) * a.head_bytes + (size_t)(piece % head_pieces) * sizeof(piece_t);
        for (int y = blockIdx.y; y < 2 * a.layers; y += gridDim.y) {
            char* cache = (y & 1 ? a.v : a.k) + (size_t)(y >> 1) * a.layer_bytes + at;
            piece_t v[W];
#pragma unroll
            for (int b = 0; b < W; b++) {
                const int from = __builtin_amdgcn_readfirstlane(s_from[b]);
                if (from >= 0) v[b] = *reinterpret_cast<const piece_t*>(cache + (size_t)from * a.seq_bytes);
            }
#pragma unroll
            for (int b = 0; b < W; b++)
                if (__builtin_amdgcn_readfirstlane(s_from[b]) >= 0)
                    *reinterpret_cast<piece_t*>(cache + (size_t)__builtin_amdgcn_readfirstlane(s_to[b]) * a.seq_bytes) = v[b];
        }
    }
}

template <int W>
static void reorder(const kv_reorder_args& a, hipStream_t s) {
    /* blocks over the positions, then over the layers until there are eight a compute unit */
    const int64_t pieces = (int64_t)a.longest * a.n_kv * (int64_t)(a.dim_bytes / sizeof(piece_t));
    const unsigned x = (unsigned)std::min<int64_t>(std::max<int64_t>((pieces + 255) / 256, 1), 4096);
    const int64_t want = 2048 / ((int64_t)x * a.groups) + 1;
    kv_reorder_kernel<W><<<dim3(x, (unsigned)std::min<int64_t>(2 * a.layers, want), a.groups), 256, 0, s>>>(a);
}

hipError_t launch_kv_reorder(const kv_reorder_args& a, hipStream_t s) {
    if (a.groups < 1 || a.width < 1 || a.width > 64 || a.layers < 1 || a.dim_bytes % 16) return hipErrorInvalidValue;
    if (a.width <= 4) reorder<4>(a, s);
    else if (a.width <= 8) reorder<8>(a, s);
    else if (a.width <= 16) reorder<16>(a, s);
    else if (a.width <= 32) reorder<32>(a, s);
    else reorder<64>(a, s);
    return hipGetLastError();
}

/**
 * kernels_beam.hip - Beam search's selection over beams and vocabulary, and
 * the reordering of the beams' key-value caches (include/vitna_serve.h).
 */

#include "serve_kernels.h"

#include <algorithm>

/* ---- selection ---- */

/* a row's log of the sum of exponentials, as its maximum and sum */
__global__ __launch_bounds__(256) void beam_sums_kernel(beam_select_args a) {
    __shared__ double red[4];
    __shared__ float redm[4];
    const int row = blockIdx.x, tid = threadIdx.x;
    const float* x = a.logits + (size_t)row * a.stride;
    float m = -INFINITY;
    for (size_t i = tid; i < a.vocab; i += 256) m = fmaxf(m, x[i]); /* fmaxf passes over NaN */
    m = wave_max(m);
    if ((tid & 63) == 0) redm[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3]));
    double s = 0.0;
    for (size_t i = tid; i < a.vocab; i += 256) {
        const float v = x[i];
        if (v == v && v != -INFINITY) s += v == m ? 1.0 : (double)expf(v - m);
    }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, WAVE);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
        double* out = (double*)a.work + 2 * (size_t)row;
        out[0] = (double)m;
        out[1] = log((red[0] + red[1]) + (red[2] + red[3]));
    }
}

__device__ __forceinline__ bool beam_better(double v, int64_t i, double w, int64_t j) { return v > w || (v == w && i < j); }

/* one round a result: the best continuation behind the last one in the order */
__global__ __launch_bounds__(256) void beam_rounds_kernel(beam_select_args a) {
    __shared__ double rv[4];
    __shared__ int64_t ri[4];
    const int group = blockIdx.x, tid = threadIdx.x;
    const int64_t V = (int64_t)a.vocab;
    double last = INFINITY;
    int64_t last_at = -1;
    for (int round = 0; round < a.keep; round++) {
        double bv = -INFINITY;
        int64_t bi = INT64_MAX;
        for (int b = 0; b < a.width; b++) {
            const int row = group * a.width + b;
            const double score = (double)a.scores[row], m = ((double*)a.work)[2 * (size_t)row], l = ((double*)a.work)[2 * (size_t)row + 1];
            if (!(score > -INFINITY)) continue;
            const bool ended = a.ended && a.ended[row];
            for (int64_t i = tid; i < V; i += 256) {
                double v;
                if (ended) {
                    if (i != a.end_token) continue;
                    v = score;
                } else {
                    const double x = (double)a.logits[(size_t)row * a.stride + i];
                    if (!(x > -INFINITY)) continue;
                    v = score + ((x == m ? 0.0 : x - m) - l);
                    if (!(v > -INFINITY)) continue;
                }
                const int64_t at = b * V + i;
                if (beam_better(v, at, bv, bi) && beam_better(last, last_at, v, at)) { bv = v; bi = at; }
            }
        }
        for (int o = 32; o > 0; o >>= 1) {
            const double ov = __shfl_xor(bv, o, WAVE);
            const int64_t oi = __shfl_xor(bi, o, WAVE);
            if (beam_better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
        }
        __syncthreads();
        if ((tid & 63) == 0) { rv[tid >> 6] = bv; ri[tid >> 6] = bi; }
        __syncthreads();
        for (int w = 0; w < 4; w++)
            if (beam_better(rv[w], ri[w], bv, bi)) { bv = rv[w]; bi = ri[w]; }
        const bool none = bi == INT64_MAX;
        if (tid == 0) {
            const int at = group * a.keep + round;
            a.best[at] = none ? -INFINITY : (float)bv;
            a.parents[at] = none ? -1 : (int)(bi / V);
            a.tokens[at] = none ? -1 : (int)(bi % V);
        }
        last = bv;
        last_at = bi;
    }
}

size_t beam_select_work(int groups, int width, size_t vocab, int keep) {
    (void)vocab;
    (void)keep;
    return (size_t)groups * width * 16;
}

hipError_t launch_beam_select(const beam_select_args& a, hipStream_t s) {
    if (a.groups < 1 || a.width < 1 || a.keep < 1) return hipErrorInvalidValue;
    beam_sums_kernel<<<a.groups * a.width, 256, 0, s>>>(a);
    beam_rounds_kernel<<<a.groups, 256, 0, s>>>(a);
    return hipGetLastError();
}

/* ---- reordering ---- */

/* A thread takes the same 16 bytes of every beam of a group: all it needs are read before any is written, so a beam
   may take another's place while that takes a third's, and no thread waits for another. */
template <int W>
__global__ __launch_bounds__(256) void kv_reorder_kernel(kv_reorder_args a) {
    const int group = blockIdx.z, layer = blockIdx.y >> 1;
    char* cache = (blockIdx.y & 1 ? a.v : a.k) + (size_t)layer * a.layer_bytes;
    const int from = max(a.spans[2 * group], 0), to = min(a.spans[2 * group + 1], a.ctx);
    const int head_pieces = (int)(a.dim_bytes / 16), pieces = a.n_kv * head_pieces;
    const int64_t many = to > from ? (int64_t)(to - from) * pieces : 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < many; i += (int64_t)gridDim.x * 256) {
        const int64_t pos = from + i / pieces;
        const int piece = (int)(i % pieces);
        const size_t at = (size_t)pos * a.pos_bytes + (size_t)(piece / head_pieces) * a.head_bytes + (size_t)(piece % head_pieces) * 16;
        u32x4 v[W];
        bool on[W];
#pragma unroll
        for (int b = 0; b < W; b++) {
            on[b] = false;
            if (b < a.width) {
                const int p = a.parents[group * a.width + b], to_seq = a.list[group * a.width + b];
                if (p >= 0 && p < a.width && p != b && to_seq >= 0 && to_seq < a.seqs) {
                    const int seq = a.list[group * a.width + p];
                    if (seq >= 0 && seq < a.seqs) {
                        on[b] = true;
                        v[b] = *reinterpret_cast<const u32x4*>(cache + (size_t)seq * a.seq_bytes + at);
                    }
                }
            }
        }
#pragma unroll
        for (int b = 0; b < W; b++)
            if (on[b]) *reinterpret_cast<u32x4*>(cache + (size_t)a.list[group * a.width + b] * a.seq_bytes + at) = v[b];
    }
}

hipError_t launch_kv_reorder(const kv_reorder_args& a, hipStream_t s) {
    if (a.groups < 1 || a.width < 1 || a.width > 64 || a.layers < 1 || a.dim_bytes % 16) return hipErrorInvalidValue;
    const int64_t pieces = (int64_t)a.longest * a.n_kv * (int64_t)(a.dim_bytes / 16);
    const dim3 grid((unsigned)std::min<int64_t>(std::max<int64_t>((pieces + 255) / 256, 1), 4096), 2 * a.layers, a.groups);
    if (a.width <= 4) kv_reorder_kernel<4><<<grid, 256, 0, s>>>(a);
    else if (a.width <= 16) kv_reorder_kernel<16><<<grid, 256, 0, s>>>(a);
    else kv_reorder_kernel<64><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

/**
 * kernels_attend.hip - Attention for serving: rows that share a prefix, a
 * sliding window with sinks, and a prompt's chunk (include/vitna_serve.h).
 *
 * Row r with visible positions T, head h of key-value head c:
 *   s_t = scale q_h . K_c[t],   m = max s_t,   out_h = sum exp(s_t - m) V_c[t] / sum exp(s_t - m),
 * T = { t <= pos : no window, or t > pos - window, or t < sinks }; t < shared reads sequence base. One pass over T
 * with a running maximum and sum; both and the weighted values in float32.
 */

#include "serve_kernels.h"

template <typename T>
__device__ __forceinline__ float at_load(const T* p) { return (float)*p; }

/* A block a (key-value head, row): 256 positions at a time, a thread a position in the scores and a few (head,
   dimension)s in the values. */
template <int HD, typename T>
__global__ __launch_bounds__(256) void attend_simple_kernel(attend_args a) {
    __shared__ float sq[ATTEND_G_MAX * HD], sp[ATTEND_G_MAX][256], red[4];
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, G = a.n_heads / a.n_kv;
    attend_row r = a.rows ? a.rows[row] : attend_row{a.run_seq, a.run_pos + row, 0, 0};
    if (a.run) r.shared = 0;
    const bool ok = r.seq >= 0 && r.seq < a.seqs && r.pos >= 0 && r.pos < a.ctx && r.shared >= 0 && (!r.shared || (r.base >= 0 && r.base < a.seqs));
    const int end = ok ? r.pos + 1 : 0;
    const int sinks = a.window ? min(a.sinks, end) : 0, first = a.window ? max(end - a.window, sinks) : 0;
    const int count = sinks + (end - first);
    for (int i = tid; i < G * HD; i += 256) sq[i] = a.q[(size_t)row * a.q_stride + (size_t)h * G * HD + i] * a.scale;
    const T* kc = (const T*)a.k + (size_t)h * a.head_stride;
    const T* vc = (const T*)a.v + (size_t)h * a.head_stride;
    auto place = [&](int i) {
        const int t = i < sinks ? i : first + (i - sinks);
        return (size_t)(t < r.shared ? r.base : r.seq) * a.seq_stride + (size_t)t * a.pos_stride;
    };
    constexpr int NA = ATTEND_G_MAX * HD / 256;
    float acc[NA], m_run[ATTEND_G_MAX], l_run[ATTEND_G_MAX];
    for (int i = 0; i < NA; i++) acc[i] = 0.0f;
    for (int g = 0; g < G; g++) { m_run[g] = -INFINITY; l_run[g] = 0.0f; }
    for (int i0 = 0; i0 < count; i0 += 256) {
        const int i = i0 + tid;
        const bool on = i < count;
        __syncthreads();
        float f[ATTEND_G_MAX];
        for (int g = 0; g < G; g++) {
            float s = 0.0f;
            if (on) {
                const T* kp = kc + place(i);
                for (int d = 0; d < HD; d++) s = fmaf(sq[g * HD + d], at_load(kp + d), s);
            }
            const float wm = wave_max(on ? s : -INFINITY);
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = wm;
            __syncthreads();
            const float m = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m_run[g]);
            const float base = m == -INFINITY ? 0.0f : m;
            const float p = on ? expf(s - base) : 0.0f;
            const float ws = wave_sum(p);
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = ws;
            __syncthreads();
            f[g] = expf(m_run[g] - base);
            l_run[g] = l_run[g] * f[g] + ((red[0] + red[1]) + (red[2] + red[3]));
            m_run[g] = m;
            sp[g][tid] = p;
        }
        __syncthreads();
        const int many = min(256, count - i0);
        for (int j = 0; j < NA; j++) {
            const int at = tid + 256 * j, g = at / HD, d = at % HD;
            if (g >= G) break;
            float s = acc[j] * f[g];
            for (int p = 0; p < many; p++) s = fmaf(sp[g][p], at_load(vc + place(i0 + p) + d), s);
            acc[j] = s;
        }
    }
    for (int j = 0; j < NA; j++) {
        const int at = tid + 256 * j, g = at / HD;
        if (g >= G) break;
        a.out[(size_t)row * a.out_stride + (size_t)h * G * HD + at] = count ? acc[j] / l_run[g] : 0.0f;
    }
}

size_t attend_work(const attend_args& a) {
    (void)a;
    return 256;
}

hipError_t launch_attend(const attend_args& a, hipStream_t s) {
    if (a.n < 1 || a.n_kv < 1 || a.n_heads % a.n_kv || a.n_heads / a.n_kv > ATTEND_G_MAX) return hipErrorInvalidValue;
    const dim3 grid(a.n, a.n_kv);
#define SIMPLE(HD, T) attend_simple_kernel<HD, T><<<grid, 256, 0, s>>>(a)
    if (a.hd == 128) {
        if (a.dtype == VITNA_DTYPE_F32) SIMPLE(128, float);
        else if (a.dtype == VITNA_DTYPE_F16) SIMPLE(128, _Float16);
        else SIMPLE(128, __bf16);
    } else if (a.hd == 64) {
        if (a.dtype == VITNA_DTYPE_F32) SIMPLE(64, float);
        else if (a.dtype == VITNA_DTYPE_F16) SIMPLE(64, _Float16);
        else SIMPLE(64, __bf16);
    } else {
        return hipErrorInvalidValue;
    }
#undef SIMPLE
    return hipGetLastError();
}

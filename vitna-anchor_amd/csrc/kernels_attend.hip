/**
 * kernels_attend.hip - Attention for serving: rows that share a prefix, a
 * sliding window with sinks, and a prompt's chunk (include/vitna_serve.h).
 *
 * Row r with visible positions T, head h of key-value head c:
 *   s_t = scale q_h . K_c[t],   m = max s_t,   out_h = sum exp(s_t - m) V_c[t] / sum exp(s_t - m),
 * T = { t <= pos : no window, or t > pos - window, or t < sinks }; t < shared reads sequence base. One pass over T
 * with a running maximum and sum, both and the weighted values in float32 (the scores in units of log 2, so that
 * exp is exp2). Two kinds of block take parts of it:
 *
 *   own_part   a row's own positions (or all of them), for the G query heads of one key-value head: every position it
 *              loads is seen by all its columns. Bound by the cache's bytes; products on v_mfma_f32_16x16x4_f32.
 *   tile_part  positions that many rows see (a shared prefix, a prompt's chunk): 32 columns (row, query head) a wave,
 *              64 positions at a time through LDS, read once for all the block's columns. Products on
 *              v_mfma_f32_32x32x16_f16.
 *
 * Where a row's positions are split over several blocks, each leaves its maximum, sum and weighted values, and
 * attend_merge_kernel joins them.
 *
 * The f16 products. A float32 operand x goes in as two f16 parts, hi = f16(x 2^k) and lo = f16(x 2^k - hi), and a
 * product as hi hi + hi lo + lo hi, summed in float32: hi leaves up to 2^-10 of x (it is cut, not rounded) and lo 2^-10
 * of that, so 2^-20 of each product is lost at most and about 2^-23 at random, beside float32's own 2^-24. (bfloat16
 * parts lose 2^-16; an outputs' 2-norm then is 4 to 8e-6 off, where float32 sums are 1e-6.) 2^k brings the largest value
 * of the column's query, of the 64 positions' keys or of their values to 2^14 .. 2^15, so any float32 cache fits f16's
 * range, and what lies 2^28 below the largest of its 64 positions is cut off. f16 and bfloat16 caches need no lo part
 * (bfloat16's 8 bits fit f16's 11 once scaled).
 */

#include "serve_kernels.h"

#include <algorithm>
#include <type_traits>

typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __fp16 h2v __attribute__((ext_vector_type(2)));

template <typename T, int N>
struct vec_of {
    typedef T type __attribute__((ext_vector_type(N), aligned(N * sizeof(T) < 16 ? N * sizeof(T) : 16)));
};
template <typename T, int N>
using vec = typename vec_of<T, N>::type;

struct attend_parts {
    float2* ml;  /* [n][n_kv][splits][G]: maximum (log 2 units) and sum of a part */
    float* acc;  /* [n][n_kv][splits][G][hd]: its weighted values; unset where the sum is 0 */
    int own, tile; /* splits of the own parts and of the tiles' */
    int tiles;     /* tiles of rows */
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ attend_row row_of(const attend_args& a, int r) {
    attend_row x = a.rows ? a.rows[r] : attend_row{a.run_seq, a.run_pos + r, 0, 0};
    if (a.run) x.shared = 0;
    const bool ok = x.seq >= 0 && x.seq < a.seqs && x.pos >= 0 && x.pos < a.ctx && x.shared >= 0 && (!x.shared || (x.base >= 0 && x.base < a.seqs));
    if (!ok) x = attend_row{0, -1, 0, 0};
    return x;
}

/* LDS written before is read after, by the whole block. Global loads in flight stay so. */
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

/* ---- a row's own positions ---- */

/* Dimension of element j of lane column c: pieces of 16 bytes (f16 heads of 64: 8), a wave's load whole rows. */
template <int HD, typename T>
struct own_dims {
    static constexpr int DPL = HD / 16;                                   /* dimensions a lane */
    static constexpr int PE = sizeof(T) == 4 ? 4 : DPL;                   /* of one piece */
    static constexpr int NP = DPL / PE;
};

/* The loads of one step: a lane's key (position c16 of the wave's 16, dimensions 32 t + 8 kq ..) and its values (positions
   4 kq + r). */
template <int HD, typename T>
struct own_step {
    vec<T, 8> k[HD / 32];
    vec<T, own_dims<HD, T>::PE> v[4][own_dims<HD, T>::NP];
};

template <int HD, typename T, int NW>
__device__ __forceinline__ void own_part(const attend_args& a, const attend_parts& p, int split, int h, int row, char* lds) {
    constexpr int DPL = own_dims<HD, T>::DPL, PE = own_dims<HD, T>::PE, NP = own_dims<HD, T>::NP, STEP = 16 * NW;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c16 = lane & 15, kq = lane >> 4, G = a.n_heads / a.n_kv;
    const attend_row r = row_of(a, row);
    const int end = r.pos + 1, begin = p.tile ? min(r.shared, end) : 0;
    /* seen: [begin, sink) and [from, end) */
    const int sink = a.window ? max(begin, min(a.sinks, end)) : begin, from = a.window ? max(sink, end - a.window) : begin;
    const int n_sink = sink - begin, count = n_sink + (end - from);
    const int per = ((count + p.own - 1) / p.own + STEP - 1) / STEP * STEP;
    const int i0 = (int)min((long)split * per, (long)count), i1 = min(i0 + per, count);
    const int S = p.own + p.tile;
    const size_t part = ((size_t)row * a.n_kv + h) * S + split;
    const bool direct = S == 1;
    if (i0 >= i1) {
        if (!direct) {
            if (tid < G) p.ml[part * G + tid] = make_float2(-INFINITY, 0.0f);
        } else {
            for (int i = tid; i < G * HD / 4; i += 64 * NW)
                reinterpret_cast<float4*>(a.out + (size_t)row * a.out_stride + (size_t)h * G * HD)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        return;
    }
    const T* kc = (const T*)a.k + (size_t)h * a.head_stride;
    const T* vc = (const T*)a.v + (size_t)h * a.head_stride;
    const size_t mine = (size_t)r.seq * a.seq_stride, other = (size_t)r.base * a.seq_stride;
    auto place = [&](int i) {
        const int t = i < n_sink ? begin + i : from + (i - n_sink);
        return (t < r.shared ? other : mine) + (size_t)t * a.pos_stride;
    };
    auto load = [&](int ib, own_step<HD, T>& s) {
        const int ik = ib + 16 * wave + c16;
        if (ik < i1) {
            const T* at = kc + place(ik) + 8 * kq;
#pragma unroll
            for (int t = 0; t < HD / 32; t++) s.k[t] = *reinterpret_cast<const vec<T, 8>*>(at + 32 * t);
        } else {
#pragma unroll
            for (int t = 0; t < HD / 32; t++) s.k[t] = vec<T, 8>{};
        }
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int iv = ib + 16 * wave + 4 * kq + x;
            if (iv < i1) {
                const T* at = vc + place(iv) + PE * c16;
#pragma unroll
                for (int n = 0; n < NP; n++) s.v[x][n] = *reinterpret_cast<const vec<T, PE>*>(at + 64 * n);
            } else {
#pragma unroll
                for (int n = 0; n < NP; n++) s.v[x][n] = vec<T, PE>{};
            }
        }
    };
    own_step<HD, T> cur, nxt;
    load(i0, cur);
    /* head c16's query in units of log 2: B operand of step (t, m), dimension 32 t + 8 kq + m */
    float q[HD / 32][8];
    const float qs = a.scale * 1.44269504088896340736f;
#pragma unroll
    for (int t = 0; t < HD / 32; t++) {
        const float4* at = reinterpret_cast<const float4*>(a.q + (size_t)row * a.q_stride + (size_t)(h * G + min(c16, G - 1)) * HD + 32 * t + 8 * kq);
        const float4 x = at[0], y = at[1];
        const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int m = 0; m < 8; m++) q[t][m] = c16 < G ? w[m] * qs : 0.0f;
    }
    float m_run = -INFINITY, l_run = 0.0f;
    f4v O[DPL];
#pragma unroll
    for (int j = 0; j < DPL; j++) O[j] = f4v{0.f, 0.f, 0.f, 0.f};
    for (int ib = i0; ib < i1; ib += STEP) {
        if (ib + STEP < i1) load(ib + STEP, nxt);
        /* S: positions 4 kq + x of head c16 */
        f4v s[HD / 32];
#pragma unroll
        for (int t = 0; t < HD / 32; t++) {
            s[t] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 8; m++) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)cur.k[t][m], q[t][m], s[t], 0, 0, 0);
        }
        f4v S4 = s[0] + s[1];
        if constexpr (HD == 128) S4 = S4 + (s[2] + s[3]);
        const int left = i1 - (ib + 16 * wave + 4 * kq); /* the lane's positions x < left are there */
        float m = m_run;
#pragma unroll
        for (int x = 0; x < 4; x++) m = fmaxf(m, x < left ? S4[x] : -INFINITY);
        m = fmaxf(m, __shfl_xor(m, 16, WAVE));
        m = fmaxf(m, __shfl_xor(m, 32, WAVE));
        const float base = m == -INFINITY ? 0.0f : m, f = exp2_hw(m_run - base);
        float w[4], l = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            w[x] = x < left ? exp2_hw(S4[x] - base) : 0.0f;
            l += w[x];
        }
        l_run = fmaf(l_run, f, l);
        m_run = m;
        if (__any(f != 1.0f)) {
#pragma unroll
            for (int j = 0; j < DPL; j++) O[j] = O[j] * f;
        }
        /* O^T: element 4 kq + i of piece dimensions, head c16 */
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int j = 0; j < DPL; j++) O[j] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)cur.v[x][j / PE][j % PE], w[x], O[j], 0, 0, 0);
        cur = nxt;
    }
    l_run += __shfl_xor(l_run, 16, WAVE);
    l_run += __shfl_xor(l_run, 32, WAVE);
    /* the waves joined: m and l [NW][16], then the values [NW][G][HD] */
    float* wm = reinterpret_cast<float*>(lds);
    float* wl = wm + NW * 16;
    float* wacc = wl + NW * 16;
    if (kq == 0) {
        wm[wave * 16 + c16] = m_run;
        wl[wave * 16 + c16] = l_run;
    }
    if (c16 < G) {
#pragma unroll
        for (int j = 0; j < DPL; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) wacc[(wave * G + c16) * HD + 64 * (j / PE) + PE * (4 * kq + i) + j % PE] = O[j][i];
    }
    __syncthreads();
    for (int i = tid; i < G * HD / 4; i += 64 * NW) {
        const int g = i / (HD / 4), d = i % (HD / 4);
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w * 16 + g]);
        const float base = M == -INFINITY ? 0.0f : M;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = exp2_hw(wm[w * 16 + g] - base);
            const float4 x = reinterpret_cast<const float4*>(wacc + (w * G + g) * HD)[d];
            L = fmaf(wl[w * 16 + g], f, L);
            o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
        }
        if (direct) {
            const float inv = 1.0f / L;
            reinterpret_cast<float4*>(a.out + (size_t)row * a.out_stride + (size_t)h * G * HD)[i] = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
            reinterpret_cast<float4*>(p.acc + (part * G + g) * HD)[d] = o;
            if (d == 0) p.ml[part * G + g] = make_float2(M, L);
        }
    }
}

/* ---- positions that many rows see ---- */

/* f16 parts, cut: two at once */
__device__ __forceinline__ uint32_t pack_cut(float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y)); }
__device__ __forceinline__ float half_lo(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }
__device__ __forceinline__ float half_hi(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16)); }
/* hi and lo of four values times a power of two */
__device__ __forceinline__ void cut4(float x0, float x1, float x2, float x3, float s, uint2& hi, uint2& lo) {
    hi = make_uint2(pack_cut(x0 * s, x1 * s), pack_cut(x2 * s, x3 * s));
    lo = make_uint2(pack_cut(fmaf(x0, s, -half_lo(hi.x)), fmaf(x1, s, -half_hi(hi.x))), pack_cut(fmaf(x2, s, -half_lo(hi.y)), fmaf(x3, s, -half_hi(hi.y))));
}

__device__ __forceinline__ void cut4(float x0, float x1, float x2, float x3, uint2& hi, uint2& lo) {
    hi = make_uint2(pack_cut(x0, x1), pack_cut(x2, x3));
    lo = make_uint2(pack_cut(fmaf(half_lo(hi.x), -1.0f, x0), fmaf(half_hi(hi.x), -1.0f, x1)),
                    pack_cut(fmaf(half_lo(hi.y), -1.0f, x2), fmaf(half_hi(hi.y), -1.0f, x3)));
}

/* Values as keys for a maximum of magnitudes: the sign shifted out, so a NaN is the largest, then an infinity. */
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) << 1; }
#define MAG_INF 0xff000000u
/* The k of 2^k that brings a magnitude to 2^14 .. 2^15 (0 and numbers near it: as far as 2^k reaches). */
__device__ __forceinline__ int to_half_range(uint32_t mag) { return min(141 - (int)(mag >> 24), 126); }
__device__ __forceinline__ float two_to(int k) { return __int_as_float((k + 127) << 23); } /* -126 .. 127 */

template <int HD, typename T, int NW>
struct tile_shape {
    static constexpr bool PARTS = sizeof(T) == 4;                        /* operands in hi and lo */
    static constexpr bool SCALED = !std::is_same<T, _Float16>::value;
    static constexpr int NT = 64 * NW, CC = HD / 4, U = 16 * CC / NT;    /* a thread's groups of 4 positions x 4 dimensions */
    static constexpr int HALF = 64 * HD;                                 /* values of one part of 64 positions' keys */
    static constexpr int ROWS = 32 * NW;                                 /* the most rows of a tile */
    static constexpr size_t LDS = (PARTS ? 4 : 2) * HALF * 2 + ROWS * sizeof(attend_row) + 2 * NW * 4 + 8;
    static_assert(U >= 1 && U * NT == 16 * CC, "whole groups a thread");
};

/* RUN: the rows are tokens of one sequence, each seeing up to itself; otherwise each sees its shared prefix. */
template <int HD, typename T, int NW, bool RUN>
__device__ __forceinline__ void tile_part(const attend_args& a, const attend_parts& p, int split, int h, int tile, char* lds) {
    typedef tile_shape<HD, T, NW> sh;
    constexpr bool PARTS = sh::PARTS, SCALED = sh::SCALED;
    constexpr int KS = HD / 16, DT = HD / 32, U = sh::U, CC = sh::CC, HALF = sh::HALF;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c32 = lane & 31, hh = lane >> 5;
    const int G = a.n_heads / a.n_kv, TR = 32 * NW / G, r0 = tile * TR, nr = min(TR, a.n - r0);
    /* Keys [part][64 positions][HD] in pieces of 8 dimensions, piece x of position t at x ^ t mod (HD / 8). Values
       [part][HD][64 positions] in units of two pieces of 4 positions, those of one MFMA operand (positions 16 s + 4 hh ..
       and 16 s + 8 + 4 hh ..: unit 2 s + hh), unit x of dimension d at x ^ (d / 2 ^ d / 16) mod 8. Sixteen lanes'
       16-byte reads then take every bank once, and all places are one lane's ^ and + a constant. */
    char* sk = lds;
    char* sv = sk + (PARTS ? 2 : 1) * HALF * 2;
    attend_row* srow = reinterpret_cast<attend_row*>(sv + (PARTS ? 2 : 1) * HALF * 2);
    auto key_to = [&](int pg, int cc) { return (uint32_t)(4 * pg * HD * 2 + (((cc >> 1) ^ ((4 * pg) & (HD / 8 - 1))) << 4) + 8 * (cc & 1)); };
    auto value_to = [&](int pg, int cc) {
        const int unit = 2 * (pg >> 2) + (pg & 1), half = (pg >> 1) & 1;
        return (uint32_t)(4 * cc * 128 + ((unit ^ (((2 * cc) ^ (cc >> 2)) & 7)) << 4) + 8 * half);
    };
    uint32_t* smax = reinterpret_cast<uint32_t*>(srow + sh::ROWS); /* [2][NW]: magnitudes of keys, of values */
    uint32_t* sbad = smax + 2 * NW;                        /* positions whose values are not finite */

    for (int i = tid; i < nr; i += sh::NT) srow[i] = row_of(a, r0 + i);
    if (tid < 2) sbad[tid] = 0;
    lds_barrier();

    /* the lane's column */
    const int col = 32 * wave + c32, lr = col / G, g = col - lr * G;
    const bool there = lr < nr;
    const attend_row me = srow[there ? lr : 0];
    const int last = !there ? -1 : RUN ? me.pos : min(me.shared, me.pos + 1) - 1; /* the last position it may see here */
    const int low = a.window ? me.pos - a.window + 1 : INT32_MIN;
    h8v qh[KS], ql[KS];
    float to_score; /* from the products' sums to scores in units of log 2, with the keys' power of two */
    {
        const float* at = a.q + (size_t)(r0 + (there ? lr : 0)) * a.q_stride + (size_t)(h * G + g) * HD + 8 * hh;
        /* read twice: kept between, the values would take the registers that the loop needs */
        uint32_t mag = 0;
#pragma unroll
        for (int s = 0; s < 2 * KS; s++) {
            const float4 x = *reinterpret_cast<const float4*>(at + 16 * (s >> 1) + 4 * (s & 1));
            mag = max(max(mag, max(magnitude(x.x), magnitude(x.y))), max(magnitude(x.z), magnitude(x.w)));
        }
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32, WAVE));
        const int k = to_half_range(mag);
        const float f = two_to(k);
        to_score = a.scale * 1.44269504088896340736f * two_to(-k);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const float4 x = *reinterpret_cast<const float4*>(at + 16 * s), y = *reinterpret_cast<const float4*>(at + 16 * s + 4);
            uint2 h0, l0, h1, l1;
            cut4(x.x, x.y, x.z, x.w, f, h0, l0);
            cut4(y.x, y.y, y.z, y.w, f, h1, l1);
            qh[s] = __builtin_bit_cast(h8v, u32x4{h0.x, h0.y, h1.x, h1.y});
            ql[s] = __builtin_bit_cast(h8v, u32x4{l0.x, l0.y, l1.x, l1.y});
        }
    }
    const char* key_at = sk + c32 * HD * 2;
    const uint32_t key_x = (hh ^ (c32 & (HD / 8 - 1))) << 4; /* piece 2 s + hh: ^ s << 5 */
    const char* value_at = sv + c32 * 128;
    const uint32_t value_x = (hh ^ ((c32 >> 1) & 7) ^ (c32 >> 4)) << 4; /* unit 2 s + hh of dimension 32 d + c32: ^ (s ^ d) << 5 */
    float m_run = -INFINITY, l_run = 0.0f;
    int e_run = 126, e_out = 126; /* the values' power of two, of the block and in this wave's O */
    f16v O[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) O[d][i] = 0.0f;

    const T* kh = (const T*)a.k + (size_t)h * a.head_stride;
    const T* vh = (const T*)a.v + (size_t)h * a.head_stride;
    const uint32_t pos_bytes = (uint32_t)(a.pos_stride * sizeof(T)); /* 64 of them stay within 31 bits */
    int first = 0;
    while (first < nr) {
        /* rows first .. next - 1 read the same positions of the same sequence */
        int next = nr;
        if constexpr (!RUN) {
            for (int w = first >> 6; w <= (nr - 1) >> 6; w++) {
                const int i = 64 * w + lane;
                bool starts = false;
                if (i > first && i < nr) starts = srow[i].base != srow[i - 1].base || srow[i].shared != srow[i - 1].shared;
                const uint64_t mask = __ballot(starts);
                if (mask) {
                    next = 64 * w + __builtin_ctzll(mask);
                    break;
                }
            }
        }
        const int mine0 = first;
        first = next;
        const int seq = __builtin_amdgcn_readfirstlane(RUN ? (a.rows ? srow[mine0].seq : a.run_seq) : srow[mine0].base);
        int end = __builtin_amdgcn_readfirstlane(srow[mine0].shared), least = 0;
        if (RUN || a.window) {
            /* the rows' furthest and nearest positions */
            uint32_t far = 0, near = 0; /* pos + 1, and 2^31 - pos: both maxima */
            for (int i = mine0 + lane; i < next; i += 64) {
                const int pos = srow[i].pos;
                if (pos >= 0) {
                    far = max(far, (uint32_t)pos + 1);
                    near = max(near, 0x80000000u - (uint32_t)pos);
                }
            }
            far = wave_umax(far);
            near = wave_umax(near);
            end = RUN ? (int)far : min(end, (int)far);
            least = near ? (int)(0x80000000u - near) : 0;
        }
        end = min(end, a.ctx);
        /* seen by some row: [0, sink) and [from, end), in chunks of 64 */
        const int sink = a.window ? min(a.sinks, end) : 0, from = a.window ? min(max(sink, least - a.window + 1), end) : 0;
        const int n_sink = (sink + 63) >> 6, n_chunks = n_sink + ((end - from + 63) >> 6);
        const int per = (n_chunks + p.tile - 1) / p.tile, c0 = split * per, c1 = min(c0 + per, n_chunks);
        if (c0 >= c1) continue;
        const bool on = there && lr >= mine0 && lr < next && last >= 0;
        const bool wave_on = __any(on);
        const T* ks = kh + (size_t)seq * a.seq_stride;
        const T* vs = vh + (size_t)seq * a.seq_stride;
        auto start = [&](int c) { return c < n_sink ? 64 * c : from + 64 * (c - n_sink); };
        auto stop = [&](int c) { return c < n_sink ? sink : end; };
        vec<T, 4> rk[U][4], rv[U][4];
        /* (positions behind the chunk's end read its last again: their scores are masked) */
        auto fetch = [&](const T* src, int c, vec<T, 4> (&x)[U][4]) {
            const int t0 = start(c);
            const uint32_t most = (uint32_t)(min(stop(c) - t0, 64) - 1);
            const char* from_ = reinterpret_cast<const char*>(src + (size_t)t0 * a.pos_stride);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int at = tid + sh::NT * u, pg = at / CC, cc = at % CC;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    x[u][i] = *reinterpret_cast<const vec<T, 4>*>(from_ + (min((uint32_t)(4 * pg + i), most) * pos_bytes + (uint32_t)(4 * sizeof(T)) * cc));
            }
        };
        auto publish = [&](const vec<T, 4> (&x)[U][4], uint32_t* to) {
            uint32_t mag = 0;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int d = 0; d < 4; d++) mag = max(mag, magnitude((float)x[u][i][d]));
            mag = wave_umax(mag);
            if (lane == 0) to[wave] = mag;
        };
        auto largest = [&](const uint32_t* from_) {
            uint32_t mag = from_[0];
#pragma unroll
            for (int w = 1; w < NW; w++) mag = max(mag, from_[w]);
            return (uint32_t)__builtin_amdgcn_readfirstlane((int)mag);
        };
        /* the finite values' largest magnitude, where some are not: a rare way round, of the whole block */
        auto finite_largest = [&](const vec<T, 4> (&x)[U][4], uint32_t* slots) {
            uint32_t mag = 0;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        const uint32_t v = magnitude((float)x[u][i][d]);
                        mag = max(mag, v >= MAG_INF ? 0u : v);
                    }
            mag = wave_umax(mag);
            lds_barrier(); /* every wave has read the slots */
            if (lane == 0) slots[wave] = mag;
            lds_barrier();
            return largest(slots);
        };
        fetch(ks, c0, rk);
        fetch(vs, c0, rv);
        publish(rk, smax);
        lds_barrier();
        for (int c = c0; c < c1; c++) {
            const int t0 = start(c), t1 = stop(c);
            /* keys to LDS; every wave is past the last chunk's scores */
            float from_keys = to_score;
            {
                float f = 1.0f;
                if constexpr (SCALED) {
                    uint32_t mag = largest(smax);
                    if (__builtin_expect(mag >= MAG_INF, 0)) mag = finite_largest(rk, smax);
                    const int k = to_half_range(mag);
                    f = two_to(k);
                    from_keys = fmaxf(to_score * two_to(-k), 1e-37f); /* (a masked score's -inf times 0 would be NaN) */
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int at = tid + sh::NT * u, pg = at / CC, cc = at % CC;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t to = (key_to(pg, cc) ^ (i << 4)) + i * HD * 2;
                        uint2 hi, lo;
                        if constexpr (SCALED) {
                            cut4((float)rk[u][i][0], (float)rk[u][i][1], (float)rk[u][i][2], (float)rk[u][i][3], f, hi, lo);
                        } else {
                            hi = __builtin_bit_cast(uint2, rk[u][i]);
                        }
                        *reinterpret_cast<uint2*>(sk + to) = hi;
                        if constexpr (PARTS) *reinterpret_cast<uint2*>(sk + HALF * 2 + to) = lo;
                    }
                }
            }
            publish(rv, smax + NW);
            if (c + 1 < c1) fetch(ks, c + 1, rk);
            lds_barrier();
            f16v S[2];
            if (wave_on) {
#pragma unroll
                for (int pt = 0; pt < 2; pt++) {
                    f16v acc;
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[i] = 0.0f;
#pragma unroll
                    for (int s = 0; s < KS; s++) {
                        const char* at = key_at + (key_x ^ (s << 5)) + 32 * pt * HD * 2;
                        const h8v k8 = *reinterpret_cast<const h8v*>(at);
                        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, qh[s], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, ql[s], acc, 0, 0, 0);
                        if constexpr (PARTS) {
                            const h8v kl = *reinterpret_cast<const h8v*>(at + HALF * 2);
                            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[s], acc, 0, 0, 0);
                        }
                    }
                    S[pt] = acc;
                }
            }
            /* the values' power of two */
            float to_half = 1.0f;
            uint32_t mag = largest(smax + NW);
            const bool bad = mag >= MAG_INF;
            if (__builtin_expect(bad, 0)) {
                mag = finite_largest(rv, smax + NW);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int pg = (tid + sh::NT * u) / CC;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        bool b = false;
#pragma unroll
                        for (int d = 0; d < 4; d++)
                            if (magnitude((float)rv[u][i][d]) >= MAG_INF) {
                                rv[u][i][d] = (T)0.0f;
                                b = true;
                            }
                        if (b) atomicOr(&sbad[(4 * pg + i) >> 5], 1u << ((4 * pg + i) & 31));
                    }
                }
                lds_barrier();
            }
            if constexpr (SCALED) {
                e_run = min(e_run, to_half_range(mag));
                to_half = two_to(e_run);
            }
            if (wave_on) {
                /* lane: positions t0 + 32 pt + 8 (i / 4) + 4 hh + i % 4 of its column */
                const bool whole = !__any(on && !(t0 + 64 <= t1 && t0 + 63 <= last && (t0 >= low || t0 + 64 <= a.sinks))) && __all(on);
                if (!whole) {
                    /* of the lane's positions, t0 + 4 hh + 32 pt + 8 (i / 4) + i % 4 */
                    const int to_last = on ? min(last, t1 - 1) - t0 - 4 * hh : -1, to_low = max(low, -1) - t0 - 4 * hh, to_sink = a.sinks - t0 - 4 * hh;
#pragma unroll
                    for (int pt = 0; pt < 2; pt++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int t = 32 * pt + 8 * (i >> 2) + (i & 3);
                            const bool sees = t <= to_last && (t >= to_low || t < to_sink);
                            S[pt][i] = sees ? S[pt][i] : -INFINITY;
                        }
                }
                float m = -INFINITY;
#pragma unroll
                for (int pt = 0; pt < 2; pt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) m = fmaxf(m, S[pt][i]);
                m = fmaxf(m, __shfl_xor(m, 32, WAVE));
                m = fmaxf(m_run, m * from_keys);
                const float base = m == -INFINITY ? 0.0f : m;
                float f = exp2_hw(m_run - base);
                const float up = 14.0f - base; /* weights up to 2^14 */
                float l = 0.0f;
                if (__builtin_expect(bad, 0)) {
                    for (int pt = 0; pt < 2; pt++) {
                        const uint32_t poison = sbad[pt];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float x = pt ? S[1][i] : S[0][i];
                            if (((poison >> (8 * (i >> 2) + 4 * hh + (i & 3))) & 1) && !(x == -INFINITY)) l = NAN;
                        }
                    }
                }
#pragma unroll
                for (int pt = 0; pt < 2; pt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        S[pt][i] = exp2_hw(fmaf(S[pt][i], from_keys, up));
                        l += S[pt][i];
                    }
                l_run = fmaf(l_run, f, l);
                m_run = m;
                if constexpr (SCALED) {
                    f *= two_to(max(e_run - e_out, -126));
                    e_out = e_run;
                }
                if (__any(f != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int i = 0; i < 16; i++) O[d][i] *= f;
                }
            }
            /* values to LDS, four positions of a dimension together; every wave is past the last chunk's values */
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int at = tid + sh::NT * u, pg = at / CC, cc = at % CC;
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const uint32_t to = (value_to(pg, cc) ^ ((d >> 1) << 4)) + d * 128;
                    uint2 hi, lo;
                    if constexpr (SCALED) {
                        cut4((float)rv[u][0][d], (float)rv[u][1][d], (float)rv[u][2][d], (float)rv[u][3][d], to_half, hi, lo);
                    } else {
                        hi = __builtin_bit_cast(uint2, vec<T, 4>{rv[u][0][d], rv[u][1][d], rv[u][2][d], rv[u][3][d]});
                    }
                    *reinterpret_cast<uint2*>(sv + to) = hi;
                    if constexpr (PARTS) *reinterpret_cast<uint2*>(sv + HALF * 2 + to) = lo;
                }
            }
            if constexpr (SCALED) {
                if (c + 1 < c1) publish(rk, smax);
            }
            if (c + 1 < c1) fetch(vs, c + 1, rv);
            lds_barrier();
            if (bad && tid < 2) sbad[tid] = 0; /* read before this barrier, next written behind another */
            if (wave_on) {
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    /* positions 16 s + 8 (j / 4) + 4 hh + j % 4 as the MFMA's eight, on both operands */
                    const f16v& P = S[s >> 1];
                    const int o = 8 * (s & 1);
                    uint2 h0, l0, h1, l1;
                    cut4(P[o], P[o + 1], P[o + 2], P[o + 3], h0, l0);
                    cut4(P[o + 4], P[o + 5], P[o + 6], P[o + 7], h1, l1);
                    const h8v ph = __builtin_bit_cast(h8v, u32x4{h0.x, h0.y, h1.x, h1.y}), pl = __builtin_bit_cast(h8v, u32x4{l0.x, l0.y, l1.x, l1.y});
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        const char* at = value_at + (value_x ^ ((s ^ d) << 5)) + 32 * d * 128;
                        const h8v v8 = *reinterpret_cast<const h8v*>(at);
                        O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, ph, O[d], 0, 0, 0);
                        O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, pl, O[d], 0, 0, 0);
                        if constexpr (PARTS) {
                            const h8v vl = *reinterpret_cast<const h8v*>(at + HALF * 2);
                            O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph, O[d], 0, 0, 0);
                        }
                    }
                }
            }
        }
        lds_barrier(); /* every wave is past the last chunk before another group's first */
    }

    l_run += __shfl_xor(l_run, 32, WAVE);
    if (!there) return;
    const int S = p.own + p.tile;
    const float back = SCALED ? two_to(-e_out) : 1.0f;
    float* to;
    float f;
    if (S == 1) {
        to = a.out + (size_t)(r0 + lr) * a.out_stride + (size_t)(h * G + g) * HD;
        f = l_run == 0.0f ? 0.0f : back / l_run;
    } else {
        const size_t part = (((size_t)(r0 + lr) * a.n_kv + h) * S + p.own + split) * G + g;
        if (hh == 0) p.ml[part] = make_float2(m_run, l_run * 0x1p-14f);
        if (l_run == 0.0f) return;
        to = p.acc + part * HD;
        f = back * 0x1p-14f;
    }
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<float4*>(to + 32 * d + 8 * i + 4 * hh) = make_float4(O[d][4 * i] * f, O[d][4 * i + 1] * f, O[d][4 * i + 2] * f, O[d][4 * i + 3] * f);
}

/* ---- the kernels ---- */

template <int HD>
constexpr int tile_waves = HD == 128 ? 8 : 4;
#define OWN_WAVES 4

template <int HD, typename T>
__global__ __launch_bounds__(64 * OWN_WAVES, 2) void attend_own_kernel(attend_args a, attend_parts p) {
    __shared__ __attribute__((aligned(16))) char lds[OWN_WAVES * (32 + ATTEND_G_MAX * HD) * 4];
    own_part<HD, T, OWN_WAVES>(a, p, blockIdx.y, blockIdx.x % a.n_kv, blockIdx.x / a.n_kv, lds);
}

template <int HD, typename T>
__global__ __launch_bounds__(64 * tile_waves<HD>, 2) void attend_run_kernel(attend_args a, attend_parts p) {
    __shared__ __attribute__((aligned(16))) char lds[tile_shape<HD, T, tile_waves<HD>>::LDS];
    tile_part<HD, T, tile_waves<HD>, true>(a, p, blockIdx.y, blockIdx.x % a.n_kv, blockIdx.x / a.n_kv, lds);
}

/* shared prefixes and the rows' own parts in one launch: the tiles' blocks first */
template <int HD, typename T>
__global__ __launch_bounds__(64 * tile_waves<HD>, 2) void attend_shared_kernel(attend_args a, attend_parts p) {
    constexpr int NW = tile_waves<HD>;
    constexpr size_t A = tile_shape<HD, T, NW>::LDS, B = NW * (32 + ATTEND_G_MAX * HD) * 4;
    __shared__ __attribute__((aligned(16))) char lds[A > B ? A : B];
    const int tiles = p.tiles * a.n_kv * p.tile;
    int b = blockIdx.x;
    if (b < tiles) {
        const int h = b % a.n_kv;
        b /= a.n_kv;
        tile_part<HD, T, NW, false>(a, p, b % p.tile, h, b / p.tile, lds);
    } else {
        b -= tiles;
        const int h = b % a.n_kv;
        b /= a.n_kv;
        own_part<HD, T, NW>(a, p, b % p.own, h, b / p.own, lds);
    }
}

/* HB heads of a row a block, SG threads for each four dimensions of one: the parts' factors once in LDS, then each
   thread adds up every SG-th part, all its loads asked for before the first is used. */
#define MERGE_SPLITS 512 /* parts of a row at most */
#define MERGE_AHEAD 8
template <int HD, int SG>
__global__ __launch_bounds__(256) void attend_merge_kernel(attend_args a, attend_parts p) {
    constexpr int D = HD / 4, HB = 256 / D / SG;
    __shared__ float sf[HB][MERGE_SPLITS];
    __shared__ float4 so[SG > 1 ? 256 : 1];
    const int G = a.n_heads / a.n_kv, S = p.own + p.tile, tid = threadIdx.x, blocks = (a.n_heads + HB - 1) / HB;
    const int row = blockIdx.x / blocks, head0 = blockIdx.x % blocks * HB;
    /* a head's parts: of key-value head head / G, split s, at ((row n_kv + head / G) S + s) G + head % G */
    auto part = [&](int head, int s) { return (((size_t)row * a.n_kv + head / G) * S + s) * G + head % G; };
    constexpr int LF = 256 / HB < 64 ? 256 / HB : 64; /* lanes for a head's factors */
    {
        const int at = tid / LF, l = tid % LF, head = head0 + at;
        if (at < HB && head < a.n_heads) {
            float2 x[2];
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                x[u] = l + LF * u < S ? p.ml[part(head, l + LF * u)] : make_float2(-INFINITY, 0.0f);
                if (x[u].y != 0.0f) m = fmaxf(m, x[u].x);
            }
            for (int s = l + 2 * LF; s < S; s += LF) {
                const float2 y = p.ml[part(head, s)];
                if (y.y != 0.0f) m = fmaxf(m, y.x);
            }
#pragma unroll
            for (int d = 1; d < LF; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, WAVE));
            const float base = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (x[u].y != 0.0f) sum = fmaf(x[u].y, exp2_hw(x[u].x - base), sum);
            for (int s = l + 2 * LF; s < S; s += LF) {
                const float2 y = p.ml[part(head, s)];
                if (y.y != 0.0f) sum = fmaf(y.y, exp2_hw(y.x - base), sum);
            }
#pragma unroll
            for (int d = 1; d < LF; d <<= 1) sum += __shfl_xor(sum, d, WAVE);
            const float inv = 1.0f / sum;
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (l + LF * u < S) sf[at][l + LF * u] = x[u].y != 0.0f ? exp2_hw(x[u].x - base) * inv : 0.0f;
            for (int s = l + 2 * LF; s < S; s += LF) {
                const float2 y = p.ml[part(head, s)];
                sf[at][s] = y.y != 0.0f ? exp2_hw(y.x - base) * inv : 0.0f;
            }
        }
    }
    __syncthreads();
    const int d = tid % D, sg = tid / D % SG, at = tid / D / SG, head = head0 + at;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (head < a.n_heads) {
        for (int s0 = sg; s0 < S; s0 += SG * MERGE_AHEAD) {
            float4 x[MERGE_AHEAD];
#pragma unroll
            for (int u = 0; u < MERGE_AHEAD; u++)
                if (s0 + SG * u < S) x[u] = reinterpret_cast<const float4*>(p.acc + part(head, s0 + SG * u) * HD)[d];
#pragma unroll
            for (int u = 0; u < MERGE_AHEAD; u++) {
                if (s0 + SG * u >= S) continue;
                const float f = sf[at][s0 + SG * u];
                if (f == 0.0f) continue; /* a part without a sum has no values */
                o.x = fmaf(x[u].x, f, o.x); o.y = fmaf(x[u].y, f, o.y); o.z = fmaf(x[u].z, f, o.z); o.w = fmaf(x[u].w, f, o.w);
            }
        }
    }
    if constexpr (SG > 1) {
        so[tid] = o;
        __syncthreads();
        if (sg) return;
#pragma unroll
        for (int g = 1; g < SG; g++) {
            const float4 x = so[tid + D * g];
            o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        }
    }
    if (head < a.n_heads) reinterpret_cast<float4*>(a.out + (size_t)row * a.out_stride + (size_t)head * HD)[d] = o;
}

/* How a call is cut into blocks. */
static attend_parts plan(const attend_args& a) {
    attend_parts p = {};
    const int G = a.n_heads / a.n_kv, nw = a.hd == 128 ? 8 : 4, rows = 32 * nw / G;
    p.tiles = (a.n + rows - 1) / rows;
    const long seen = a.window ? std::min<long>(a.own_max, (long)a.window + a.sinks) : a.own_max;
    const long blocks = 256; /* a block a compute unit */
    if (a.run) {
        const long chunks = (a.window ? std::min<long>(a.own_max, (long)a.window + a.sinks + rows) : a.own_max) / 64 + 1;
        p.tile = (int)std::min<long>(std::min<long>(chunks, 64), std::max<long>(1, blocks / ((long)p.tiles * a.n_kv)));
        return p;
    }
    if (a.shared_max) {
        const long chunks = (a.window ? std::min<long>(a.shared_max, (long)a.window + a.sinks) : a.shared_max) / 64 + 1;
        p.tile = (int)std::min<long>(std::min<long>(chunks, 64), std::max<long>(1, blocks / ((long)p.tiles * a.n_kv)));
    }
    const long step = 16 * (a.shared_max ? nw : OWN_WAVES);
    p.own = (int)std::min<long>(std::min<long>((seen + step - 1) / step, 256), std::max<long>(1, 1024 / ((long)a.n * a.n_kv)));
    return p;
}

static size_t parts_bytes(const attend_args& a, const attend_parts& p, size_t* acc) {
    const size_t S = (size_t)p.own + p.tile, heads = (size_t)a.n * a.n_heads * S;
    *acc = align256(heads * sizeof(float2));
    return S > 1 ? *acc + heads * a.hd * sizeof(float) : 16;
}

size_t attend_work(const attend_args& a) {
    size_t acc;
    return parts_bytes(a, plan(a), &acc);
}

template <int HD, typename T>
static hipError_t launch(const attend_args& a, const attend_parts& p, hipStream_t s) {
    constexpr int NW = tile_waves<HD>;
    const unsigned heads = (unsigned)a.n_kv;
    if (a.run) {
        attend_run_kernel<HD, T><<<dim3(p.tiles * heads, p.tile), 64 * NW, 0, s>>>(a, p);
    } else if (p.tile) {
        attend_shared_kernel<HD, T><<<heads * ((unsigned)p.tiles * p.tile + (unsigned)a.n * p.own), 64 * NW, 0, s>>>(a, p);
    } else {
        attend_own_kernel<HD, T><<<dim3(a.n * heads, p.own), 64 * OWN_WAVES, 0, s>>>(a, p);
    }
    const int S = p.own + p.tile;
    if (S > 1) {
        constexpr int at_once = 1024 / HD; /* heads a block of one thread for each four dimensions */
        const auto blocks = [&](int sg) { return (unsigned)a.n * ((a.n_heads + at_once / sg - 1) / (at_once / sg)); };
        if (S <= MERGE_AHEAD) attend_merge_kernel<HD, 1><<<blocks(1), 256, 0, s>>>(a, p);
        else attend_merge_kernel<HD, 8><<<blocks(8), 256, 0, s>>>(a, p);
    }
    return hipGetLastError();
}

hipError_t launch_attend(const attend_args& a, hipStream_t s) {
    if (a.n < 1 || a.n_kv < 1 || a.n_heads % a.n_kv || a.n_heads / a.n_kv > ATTEND_G_MAX) return hipErrorInvalidValue;
    attend_parts p = plan(a);
    size_t acc;
    if (parts_bytes(a, p, &acc) > a.work_bytes || p.own + p.tile > MERGE_SPLITS) return hipErrorInvalidValue;
    if ((long)a.n * a.n_kv > INT32_MAX || (long)a.n_kv * ((long)p.tiles * p.tile + (long)a.n * p.own) > INT32_MAX) return hipErrorInvalidValue;
    p.ml = static_cast<float2*>(a.work);
    p.acc = reinterpret_cast<float*>(static_cast<char*>(a.work) + acc);
    if (a.hd == 128) {
        if (a.dtype == VITNA_DTYPE_F32) return launch<128, float>(a, p, s);
        if (a.dtype == VITNA_DTYPE_F16) return launch<128, _Float16>(a, p, s);
        if (a.dtype == VITNA_DTYPE_BF16) return launch<128, __bf16>(a, p, s);
    } else if (a.hd == 64) {
        if (a.dtype == VITNA_DTYPE_F32) return launch<64, float>(a, p, s);
        if (a.dtype == VITNA_DTYPE_F16) return launch<64, _Float16>(a, p, s);
        if (a.dtype == VITNA_DTYPE_BF16) return launch<64, __bf16>(a, p, s);
    }
    return hipErrorInvalidValue;
}

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
 *   columns_part  16 columns (row, query head) of one key-value head: a row's own positions, or a prefix that few columns
 *                 share. Each wave takes other positions, straight to registers. Bound by the cache's bytes; products on
 *                 v_mfma_f32_16x16x4_f32.
 *   group_part    positions that many columns see (a shared prefix, a prompt's chunk): 32 columns a wave, 128 a block, 64
 *                 positions at a time through LDS, read once for all the block's columns. Products on
 *                 v_mfma_f32_32x32x16_f16. A long chunk of a prompt takes the same steps from images of the cache
 *                 (attend_image_kernel, attend_imaged_kernel).
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
typedef int int4_ __attribute__((ext_vector_type(4)));

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
    int few;       /* a group's columns for few_part at most */
    int few_blocks, tile_blocks, busy; /* a tile's blocks, of a key-value head: of few_part, of tile_part, and of each those that get work */
    /* a run's chunks ready for LDS (attend_image_kernel): slots of them for each key-value head; 0: none */
    int slots;
    char* images;  /* [n_kv][slots] */
    int4* meta;    /* [0]: where the slots lie; [1 + n_kv slots]: of each, its keys' and values' powers of two, and the positions whose values are no numbers */
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ attend_row row_of(const attend_args& a, int r) {
    attend_row x = {a.run_seq, a.run_pos + r, 0, 0};
    if (a.rows) {
        x = a.rows[r];
    } else if (a.recs) {
        x.seq = a.recs[r].seq;
        x.pos = a.recs[r].pos;
        if (a.share && x.seq >= 0 && x.seq < a.seqs) {
            const int2 s = a.share[x.seq];
            x.base = s.x;
            x.shared = s.y;
        }
    }
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

/* ---- few columns: each wave other positions ---- */

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

/* What columns_part reads: positions begin .. begin + n_sink - 1, then from .. , numbered 0, 1, ...; of them i0 .. i1 - 1.
   Positions before shared lie `other` elements behind the cache's start, the rest `mine`. */
struct positions {
    int begin, n_sink, from, i0, i1, shared;
    size_t other, mine;
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) << 1; }
#define MAG_INF 0xff000000u /* a magnitude that is no number's: the sign shifted out, a NaN is the largest, then an infinity */

/* n_cols columns (16 at most) of key-value head h from col0 on (column x: row row0 + x / G, query head h G + x mod G), each
   wave 16 positions a step, then the waves joined in LDS ([NW][16] maxima and sums, [NW][16][HD] values). MASK: a column
   sees what its row (rows[x / G]) shares and its window leaves; otherwise all. Whole block; ends with LDS read. */
template <int HD, typename T, int NW, bool MASK>
__device__ __forceinline__ void columns_part(const attend_args& a, const attend_parts& p, const positions& at, int split, int h, int row0,
                                             const attend_row* rows, int col0, int n_cols, char* lds) {
    constexpr int DPL = own_dims<HD, T>::DPL, PE = own_dims<HD, T>::PE, NP = own_dims<HD, T>::NP, STEP = 16 * NW;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c16 = lane & 15, kq = lane >> 4, G = a.n_heads / a.n_kv;
    const int S = p.own + p.tile, i0 = at.i0, i1 = at.i1;
    const bool direct = S == 1;
    auto part_of = [&](int c) { const int col = col0 + c; return (((size_t)(row0 + col / G) * a.n_kv + h) * S + split) * G + col % G; };
    auto out_of = [&](int c) { const int col = col0 + c; return a.out + (size_t)(row0 + col / G) * a.out_stride + (size_t)(h * G + col % G) * HD; };
    if (i0 >= i1) {
        if (!direct) {
            if (tid < n_cols) p.ml[part_of(tid)] = make_float2(-INFINITY, 0.0f);
        } else {
            for (int i = tid; i < n_cols * HD / 4; i += 64 * NW) reinterpret_cast<float4*>(out_of(i / (HD / 4)))[i % (HD / 4)] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        return;
    }
    const T* kc = (const T*)a.k + (size_t)h * a.head_stride;
    const T* vc = (const T*)a.v + (size_t)h * a.head_stride;
    auto position = [&](int i) { return i < at.n_sink ? at.begin + i : at.from + (i - at.n_sink); };
    auto place = [&](int i) {
        const int t = position(i);
        return (t < at.shared ? at.other : at.mine) + (size_t)t * a.pos_stride;
    };
    auto load = [&](int ib, own_step<HD, T>& s) {
        const int ik = ib + 16 * wave + c16;
        if (ik < i1) {
            const T* k = kc + place(ik) + 8 * kq;
#pragma unroll
            for (int t = 0; t < HD / 32; t++) s.k[t] = *reinterpret_cast<const vec<T, 8>*>(k + 32 * t);
        } else {
#pragma unroll
            for (int t = 0; t < HD / 32; t++) s.k[t] = vec<T, 8>{};
        }
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int iv = ib + 16 * wave + 4 * kq + x;
            if (iv < i1) {
                const T* v = vc + place(iv) + PE * c16;
#pragma unroll
                for (int n = 0; n < NP; n++) s.v[x][n] = *reinterpret_cast<const vec<T, PE>*>(v + 64 * n);
            } else {
#pragma unroll
                for (int n = 0; n < NP; n++) s.v[x][n] = vec<T, PE>{};
            }
        }
    };
    own_step<HD, T> cur, nxt;
    load(i0, cur);
    /* the queries in units of log 2: B operand of step (t, m), dimension 32 t + 8 kq + m of column 16 ct + c16 */
    float q[HD / 32][8];
    int last = INT32_MAX, low = INT32_MIN;
    const float qs = a.scale * 1.44269504088896340736f;
    {
        const int col = col0 + min(c16, n_cols - 1), lr = col / G;
#pragma unroll
        for (int t = 0; t < HD / 32; t++) {
            const float4* src = reinterpret_cast<const float4*>(a.q + (size_t)(row0 + lr) * a.q_stride + (size_t)(h * G + col - lr * G) * HD + 32 * t + 8 * kq);
            const float4 x = src[0], y = src[1];
            const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int m = 0; m < 8; m++) q[t][m] = c16 < n_cols ? w[m] * qs : 0.0f;
        }
        if constexpr (MASK) {
            const attend_row r = rows[lr];
            last = min(r.shared, r.pos + 1) - 1;
            if (a.window) low = r.pos - a.window + 1;
        }
    }
    float m_run = -INFINITY, l_run = 0.0f;
    f4v O[DPL];
#pragma unroll
    for (int j = 0; j < DPL; j++) O[j] = f4v{0.f, 0.f, 0.f, 0.f};
    for (int ib = i0; ib < i1; ib += STEP) {
        if (ib + STEP < i1) load(ib + STEP, nxt);
        const int mine = ib + 16 * wave + 4 * kq, left = i1 - mine; /* the lane's positions x < left are there */
        uint32_t bad = 0; /* bit x: position 4 kq + x has values that are not finite */
        if constexpr (MASK) {
            uint32_t mag = 0;
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int j = 0; j < DPL; j++) mag = max(mag, magnitude((float)cur.v[x][j / PE][j % PE]));
            if (__builtin_expect(__any(mag >= MAG_INF), 0)) {
                /* a weight of 0 would make NaN of them: taken out, and the columns that see one marked */
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    bool b = false;
#pragma unroll
                    for (int j = 0; j < DPL; j++)
                        if (magnitude((float)cur.v[x][j / PE][j % PE]) >= MAG_INF) {
                            cur.v[x][j / PE][j % PE] = (T)0.0f;
                            b = true;
                        }
                    const uint64_t any = __ballot(b);
                    if ((any >> (16 * kq)) & 0xffff) bad |= 1u << x;
                }
            }
        }
        {
            /* S: positions 4 kq + x of the column */
            f4v s[HD / 32];
#pragma unroll
            for (int t = 0; t < HD / 32; t++) {
                s[t] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int m = 0; m < 8; m++) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)cur.k[t][m], q[t][m], s[t], 0, 0, 0);
            }
            f4v S4 = s[0] + s[1];
            if constexpr (HD == 128) S4 = S4 + (s[2] + s[3]);
            bool sees[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                sees[x] = x < left;
                if constexpr (MASK) {
                    const int t = position(mine + x);
                    sees[x] = sees[x] && t <= last && (t >= low || t < a.sinks);
                }
            }
            float m = m_run;
#pragma unroll
            for (int x = 0; x < 4; x++) m = fmaxf(m, sees[x] ? S4[x] : -INFINITY);
            m = fmaxf(m, __shfl_xor(m, 16, WAVE));
            m = fmaxf(m, __shfl_xor(m, 32, WAVE));
            const float base = m == -INFINITY ? 0.0f : m, f = exp2_hw(m_run - base);
            float w[4], l = 0.0f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                w[x] = sees[x] ? exp2_hw(S4[x] - base) : 0.0f;
                l += w[x];
                if constexpr (MASK)
                    if (__builtin_expect(bad >> x & 1, 0) && sees[x]) l = NAN;
            }
            l_run = fmaf(l_run, f, l);
            m_run = m;
            if (__any(f != 1.0f)) {
#pragma unroll
                for (int j = 0; j < DPL; j++) O[j] = O[j] * f;
            }
            /* O^T: element 4 kq + i of piece dimensions, column c16 */
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int j = 0; j < DPL; j++)
                    O[j] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)cur.v[x][j / PE][j % PE], w[x], O[j], 0, 0, 0);
        }
        cur = nxt;
    }
    float* wm = reinterpret_cast<float*>(lds);
    float* wl = wm + NW * 16;
    float* wacc = wl + NW * 16;
    l_run += __shfl_xor(l_run, 16, WAVE);
    l_run += __shfl_xor(l_run, 32, WAVE);
    if (kq == 0) {
        wm[wave * 16 + c16] = m_run;
        wl[wave * 16 + c16] = l_run;
    }
    if (c16 < n_cols) {
#pragma unroll
        for (int j = 0; j < DPL; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) wacc[(wave * n_cols + c16) * HD + 64 * (j / PE) + PE * (4 * kq + i) + j % PE] = O[j][i];
    }
    __syncthreads();
    for (int i = tid; i < n_cols * HD / 4; i += 64 * NW) {
        const int c = i / (HD / 4), d = i % (HD / 4);
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w * 16 + c]);
        const float base = M == -INFINITY ? 0.0f : M;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = exp2_hw(wm[w * 16 + c] - base);
            const float4 x = reinterpret_cast<const float4*>(wacc + (w * n_cols + c) * HD)[d];
            L = fmaf(wl[w * 16 + c], f, L);
            o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
        }
        if (direct) {
            const float inv = 1.0f / L;
            reinterpret_cast<float4*>(out_of(c))[d] = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
            const size_t part = part_of(c);
            reinterpret_cast<float4*>(p.acc + part * HD)[d] = o;
            if (d == 0) p.ml[part] = make_float2(M, L);
        }
    }
}
template <int HD, int NW>
constexpr size_t columns_lds = NW * (32 + 16 * HD) * 4;

/* A row's own positions, those that its window leaves. */
template <int HD, typename T, int NW>
__device__ __forceinline__ void own_part(const attend_args& a, const attend_parts& p, int split, int h, int row, char* lds) {
    const attend_row r = row_of(a, row);
    const int end = r.pos + 1, begin = p.tile ? min(r.shared, end) : 0;
    /* seen: [begin, sink) and [from, end) */
    const int sink = a.window ? max(begin, min(a.sinks, end)) : begin, from = a.window ? max(sink, end - a.window) : begin;
    const int count = sink - begin + (end - from), per = ((count + p.own - 1) / p.own + 16 * NW - 1) / (16 * NW) * (16 * NW);
    positions at;
    at.begin = begin; at.n_sink = sink - begin; at.from = from;
    at.i0 = (int)min((long)split * per, (long)count);
    at.i1 = min(at.i0 + per, count);
    at.shared = r.shared;
    at.other = (size_t)r.base * a.seq_stride;
    at.mine = (size_t)r.seq * a.seq_stride;
    columns_part<HD, T, NW, false>(a, p, at, split, h, row, nullptr, 0, a.n_heads / a.n_kv, lds);
}

/* ---- rows that share ---- */

/* A group with so many columns at most goes to few_part, any other to tile_part; a call of FEW_CALL columns or fewer, or of
   FEW_WORK columns times shared positions, has no other groups. 8 rows of 8 heads a key-value head behind 777 positions (float32): 18 us in few_part, 25 in tile_part;
   behind 4096, 24 and 31. Four such groups, 32 rows: behind 777 25 and 30, behind 4096 49 and 43 (bfloat16 54 and 34). Eight
   groups of 32 columns behind 4096: 51 and 55 (bfloat16 55 and 43). Two of 64 behind 160: 14 and 23. */
#define FEW_COLUMNS 32
#define FEW_CALL 64
#define FEW_WORK (1L << 18)

/* A tile: 32 columns each of TILE_COLUMNS waves; for tile_part of heads of 128 two waves take the same columns, each half of
   a chunk's positions. */
#define TILE_COLUMNS 4
template <int HD>
constexpr int tile_waves = HD == 128 ? 2 * TILE_COLUMNS : TILE_COLUMNS;
/* Rows of a tile. Rows next to each other in a tile that read the same positions of the same sequence are a group. */
template <int HD>
__host__ __device__ constexpr int tile_rows(int G) { return 32 * TILE_COLUMNS / G; }

/* A tile's rows to LDS (the caller waits). */
template <int NT>
__device__ __forceinline__ void load_rows(const attend_args& a, int r0, int nr, attend_row* srow) {
    for (int i = threadIdx.x; i < nr; i += NT) srow[i] = row_of(a, r0 + i);
}
/* The row behind the group that begins at row first of the tile's nr. */
__device__ __forceinline__ int group_end(const attend_row* srow, int first, int nr) {
    const int lane = threadIdx.x & 63;
    for (int w = first >> 6; w <= (nr - 1) >> 6; w++) {
        const int i = 64 * w + lane;
        bool starts = false;
        if (i > first && i < nr) starts = srow[i].base != srow[i - 1].base || srow[i].shared != srow[i - 1].shared;
        const uint64_t mask = __ballot(starts);
        if (mask) return 64 * w + (int)__builtin_ctzll(mask);
    }
    return nr;
}
/* What some rows first .. next - 1 of a group see: [0, sink) and [from, end) of sequence seq. */
struct group_span {
    int seq, sink, from, end;
};
template <bool RUN>
__device__ __forceinline__ group_span group_seen(const attend_args& a, const attend_row* srow, int first, int next) {
    group_span s;
    s.seq = __builtin_amdgcn_readfirstlane(RUN ? (a.recs ? srow[first].seq : a.run_seq) : srow[first].base);
    int end = __builtin_amdgcn_readfirstlane(srow[first].shared), least = 0;
    if (RUN || a.window) {
        /* the rows' furthest and nearest positions */
        uint32_t far = 0, near = 0; /* pos + 1, and 2^31 - pos: both maxima */
        for (int i = first + (threadIdx.x & 63); i < next; i += 64) {
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
    s.end = min(end, a.ctx);
    s.sink = a.window ? min(a.sinks, s.end) : 0;
    s.from = a.window ? min(max(s.sink, least - a.window + 1), s.end) : 0;
    return s;
}

/* How a tile's blocks take its units: block y takes unit y mod units, part y / units of its positions (there are blocks for
   every unit). A unit's parts are the first of the tile's p.tile splits, the others get an empty part of its columns.
   (Blocks that each took their part of unit after unit had 36 rows in groups of two behind 426 positions in 68 us; so 21.) */
struct unit_share {
    int units, y, parts;
    __device__ __forceinline__ unit_share(int units_, int busy, int y_, int splits) : units(units_), y(y_), parts(min(max(busy / units_, 1), splits)) {}
    __device__ __forceinline__ bool mine(int unit) const { return y % units == unit && y / units < parts; }
    __device__ __forceinline__ int part() const { return y / units; }
};
/* The splits that a unit of n_cols columns from column col on leaves empty, of the part's share. */
__device__ __forceinline__ void empty_parts(const attend_args& a, const attend_parts& p, const unit_share& u, int h, int row, int col, int n_cols) {
    const int G = a.n_heads / a.n_kv, S = p.own + p.tile, c = col + (int)threadIdx.x;
    if ((int)threadIdx.x >= n_cols) return;
    for (int x = u.part() + u.parts; x < p.tile; x += u.parts)
        p.ml[(((size_t)(row + c / G) * a.n_kv + h) * S + p.own + x) * G + c % G] = make_float2(-INFINITY, 0.0f);
}

/* Block y's of the prefixes of a tile's groups of few columns. A unit is 16 columns of such a group. */
template <int HD, typename T, int NW>
__device__ __forceinline__ void few_part(const attend_args& a, const attend_parts& p, int y, int h, int tile, char* lds) {
    const int G = a.n_heads / a.n_kv, TR = tile_rows<HD>(G), r0 = tile * TR, nr = min(TR, a.n - r0);
    attend_row* srow = reinterpret_cast<attend_row*>(lds);
    char* rest = lds + tile_rows<HD>(1) * sizeof(attend_row);
    load_rows<64 * NW>(a, r0, nr, srow);
    lds_barrier();
    int units = 0;
    for (int first = 0, next; first < nr; first = next) {
        next = group_end(srow, first, nr);
        const int n_cols = (next - first) * G;
        if (n_cols <= p.few) units += (n_cols + 15) >> 4;
    }
    if (!units) return;
    const unit_share u(units, p.busy, y, p.tile);
    int unit = 0;
    for (int first = 0, next; first < nr; first = next) {
        next = group_end(srow, first, nr);
        const int n_cols = (next - first) * G;
        if (n_cols > p.few) continue;
        for (int col = 0; col < n_cols; col += 16, unit++) {
            if (!u.mine(unit)) continue;
            const int many = min(16, n_cols - col);
            empty_parts(a, p, u, h, r0 + first, col, many);
            const group_span s = group_seen<false>(a, srow, first, next);
            const int count = s.sink + (s.end - s.from), per = ((count + u.parts - 1) / u.parts + 15) & ~15;
            positions at;
            at.begin = 0; at.n_sink = s.sink; at.from = s.from;
            at.i0 = (int)min((long)u.part() * per, (long)count);
            at.i1 = min(at.i0 + per, count);
            at.shared = INT32_MAX;
            at.other = at.mine = (size_t)s.seq * a.seq_stride;
            columns_part<HD, T, NW, true>(a, p, at, p.own + u.part(), h, r0 + first, srow + first, col, many, rest);
            lds_barrier();
        }
    }
}

/* ---- positions that many rows see ---- */

/* f16 parts, cut: two at once */
__device__ __forceinline__ uint32_t pack_cut(float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y)); }
/* x less a half of h: one instruction (the compiler widens the half first) */
__device__ __forceinline__ float less_lo(float x, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float less_hi(float x, uint32_t h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
/* hi and lo of four values, and of four times a power of two */
__device__ __forceinline__ void cut4(float x0, float x1, float x2, float x3, uint2& hi, uint2& lo) {
    hi = make_uint2(pack_cut(x0, x1), pack_cut(x2, x3));
    lo = make_uint2(pack_cut(less_lo(x0, hi.x), less_hi(x1, hi.x)), pack_cut(less_lo(x2, hi.y), less_hi(x3, hi.y)));
}

__device__ __forceinline__ void cut4(float x0, float x1, float x2, float x3, float s, uint2& hi, uint2& lo) { cut4(x0 * s, x1 * s, x2 * s, x3 * s, hi, lo); }

/* The k of 2^k that brings a magnitude to 2^14 .. 2^15 (0 and numbers near it: as far as 2^k reaches). */
__device__ __forceinline__ int to_half_range(uint32_t mag) { return min(141 - (int)(mag >> 24), 126); }
__device__ __forceinline__ float two_to(int k) { return __int_as_float((k + 127) << 23); } /* -126 .. 127 */

template <int HD, typename T, int NW>
struct tile_shape {
    static constexpr bool PARTS = sizeof(T) == 4;                        /* operands in hi and lo */
    static constexpr bool SCALED = !std::is_same<T, _Float16>::value;
    static constexpr int NT = 64 * NW, CC = HD / 4, U = 16 * CC / NT;    /* a thread's groups of 4 positions x 4 dimensions */
    static constexpr int HALF = 64 * HD;                                 /* values of one part of 64 positions' keys */
    static constexpr int ROWS = 32 * TILE_COLUMNS;                       /* the most rows of a tile */
    static constexpr int SIDES = NW / TILE_COLUMNS, POS = 64 / SIDES;    /* waves of the same columns, each one's positions of a chunk */
    static constexpr int KEYS = (PARTS ? 2 : 1) * HALF * 2;              /* bytes of a chunk's keys, and of its values */
    static constexpr int SIDE = KEYS / SIDES;
    static constexpr int MEET = SIDES > 1 ? TILE_COLUMNS * 64 * (HD / 2 + 8) * 4 : 0; /* what the sides exchange at the end */
    static constexpr int ROOM = 2 * KEYS > MEET ? 2 * KEYS : MEET;
    static constexpr size_t HEAD = (2 * NW * 4 + 8 + 15) / 16 * 16, LDS = ROWS * sizeof(attend_row) + HEAD + ROOM;
    static_assert(NW * 4096 <= ROOM, "the queries pass through the keys' and values' room");
    static_assert(SIDES * TILE_COLUMNS == NW && U >= 1 && U * NT == 16 * CC, "whole groups a thread");
};

/* Places in LDS (and in an image) of POS = 64 or 32 positions. Keys [part][POS][HD] in pieces of 8 dimensions, piece x of
   position t at x ^ t mod (HD / 8). Values [part][HD][POS] in units of two pieces of 4 positions, those of one MFMA operand
   (positions 16 s + 4 hh .. and 16 s + 8 + 4 hh ..: unit 2 s + hh), unit x of dimension d at x ^ (d / 2 ^ d / 16) mod 8
   (POS 32: x ^ d / 4 mod 4). Sixteen lanes' 16-byte reads then take every bank once, and all places are one lane's ^ and +
   a constant. Thread group (pg, cc) holds positions 4 pg + i and dimensions 4 cc + d: key i at (key_to ^ i << 4) + i rows,
   values d at (value_to ^ value_swap(d)) + d rows. */
template <int HD>
__device__ __forceinline__ uint32_t key_to(int pg, int cc) {
    return (uint32_t)(4 * pg * HD * 2 + (((cc >> 1) ^ ((4 * pg) & (HD / 8 - 1))) << 4) + 8 * (cc & 1));
}
template <int POS>
__device__ __forceinline__ uint32_t value_to(int pg, int cc) {
    const int unit = 2 * (pg >> 2) + (pg & 1), half = (pg >> 1) & 1, x = POS == 64 ? ((2 * cc) ^ (cc >> 2)) & 7 : cc & 3;
    return (uint32_t)(4 * cc * POS * 2 + ((unit ^ x) << 4) + 8 * half);
}
template <int POS>
__device__ __forceinline__ constexpr uint32_t value_swap(int d) { return POS == 64 ? (d >> 1) << 4 : 0; }

/* A thread's share of 64 positions' keys or values: U groups of 4 positions x 4 dimensions. */
template <int HD, typename T, int NT>
struct chunk_share {
    static constexpr int CC = HD / 4, U = 16 * CC / NT;
    vec<T, 4> x[U][4];
    /* positions t0 .. t1 - 1 (64 at most) of src (a head's positions). Those that no row sees, behind t1 and gap0 .. gap1 - 1, take
       a place that one does (their scores are masked, and their values would set the others' powers of two). */
    __device__ __forceinline__ void fetch(const T* src, size_t pos_stride, int t0, int t1, int gap0 = 0, int gap1 = 0) {
        const int most = min(t1 - t0, 64) - 1, skip = gap0 - t0, to = gap1 - t0;
        const uint32_t pos_bytes = (uint32_t)(pos_stride * sizeof(T)); /* 64 of them stay within 31 bits */
        const char* from = reinterpret_cast<const char*>(src + (size_t)t0 * pos_stride);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = threadIdx.x + NT * u, pg = at / CC, cc = at % CC;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                int t = min(4 * pg + i, most);
                if (t >= skip && t < to) t = to <= most ? to : max(skip - 1, 0);
                x[u][i] = *reinterpret_cast<const vec<T, 4>*>(from + ((uint32_t)t * pos_bytes + (uint32_t)(4 * sizeof(T)) * cc));
            }
        }
    }
    /* the wave's largest magnitude to its slot; finite: of the numbers among them */
    __device__ __forceinline__ void publish(uint32_t* slots, bool finite = false) const {
        uint32_t mag = 0;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    uint32_t v = magnitude((float)x[u][i][d]);
                    if (finite && v >= MAG_INF) v = 0;
                    mag = max(mag, v);
                }
        mag = wave_umax(mag);
        if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = mag;
    }
    static __device__ __forceinline__ uint32_t largest(const uint32_t* slots) {
        uint32_t mag = slots[0];
#pragma unroll
        for (int w = 1; w < NT / 64; w++) mag = max(mag, slots[w]);
        return (uint32_t)__builtin_amdgcn_readfirstlane((int)mag);
    }
    /* the finite ones' largest, where some are not: a rare way round, of the whole block */
    __device__ __forceinline__ uint32_t finite_largest(uint32_t* slots) const {
        lds_barrier(); /* every wave has read the slots */
        publish(slots, true);
        lds_barrier();
        return largest(slots);
    }
    /* values that are no numbers taken out (a weight of 0 would make NaN of them), their positions' bits set in bad */
    __device__ __forceinline__ void take_out(uint32_t* bad) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int pg = (threadIdx.x + NT * u) / CC;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                bool b = false;
#pragma unroll
                for (int d = 0; d < 4; d++)
                    if (magnitude((float)x[u][i][d]) >= MAG_INF) {
                        x[u][i][d] = (T)0.0f;
                        b = true;
                    }
                if (b) atomicOr(&bad[(4 * pg + i) >> 5], 1u << ((4 * pg + i) & 31));
            }
        }
    }
    /* times f, in parts; POS 32: the second half of the positions next bytes behind the first */
    template <int POS = 64>
    __device__ __forceinline__ void store_keys(char* sk, float f, size_t next = 0) const {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = threadIdx.x + NT * u, pg = at / CC, cc = at % CC;
            char* to = sk + (POS == 32 && pg >= 8 ? next : 0);
#pragma unroll
            for (int i = 0; i < 4; i++) put<POS>(to + (key_to<HD>(pg & (POS / 4 - 1), cc) ^ (i << 4)) + i * HD * 2, x[u][i][0], x[u][i][1], x[u][i][2], x[u][i][3], f);
        }
    }
    template <int POS = 64>
    __device__ __forceinline__ void store_values(char* sv, float f, size_t next = 0) const {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = threadIdx.x + NT * u, pg = at / CC, cc = at % CC;
            char* to = sv + (POS == 32 && pg >= 8 ? next : 0);
#pragma unroll
            for (int d = 0; d < 4; d++) put<POS>(to + (value_to<POS>(pg & (POS / 4 - 1), cc) ^ value_swap<POS>(d)) + d * POS * 2, x[u][0][d], x[u][1][d], x[u][2][d], x[u][3][d], f);
        }
    }
    template <int POS>
    static __device__ __forceinline__ void put(char* to, T a, T b, T c, T d, float f) {
        uint2 hi, lo;
        if constexpr (std::is_same<T, _Float16>::value) hi = __builtin_bit_cast(uint2, vec<T, 4>{a, b, c, d});
        else cut4((float)a, (float)b, (float)c, (float)d, f, hi, lo);
        *reinterpret_cast<uint2*>(to) = hi;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint2*>(to + POS * HD * 2) = lo;
    }
};

#define WEIGHT_EXP 6
#define WEIGHT_SLACK 8.0f

/* A wave's 32 columns: queries, running maximum, sum and weighted values. Column 32 wave + c32 is row row0 + x / G, query
   head h G + x mod G; lanes c32 and c32 + 32 hold its halves. */
template <int HD, typename T, int POS>
struct wave_columns {
    static constexpr bool PARTS = sizeof(T) == 4, SCALED = !std::is_same<T, _Float16>::value;
    static constexpr int KS = HD / 16, DT = HD / 32, PT = POS / 32, LO = POS * HD * 2; /* bytes from a hi part to its lo part */
    h8v qh[KS], ql[KS];
    f16v S[PT], O[DT];
    float to_score; /* from the products' sums to scores in units of log 2, but for the keys' power of two */
    float m_run, l_run;
    int e_out;      /* the values' power of two in O */
    int lr, g, last, low, hh;
    bool there, on, wave_on;
    const char *key_at, *value_at;
    uint32_t key_x, value_x;

    /* the keys and values to work on */
    __device__ __forceinline__ void at(const char* sk, const char* sv) {
        const int c32 = threadIdx.x & 31;
        key_at = sk + c32 * HD * 2;
        value_at = sv + c32 * POS * 2;
    }
    template <bool RUN>
    __device__ __forceinline__ void init(const attend_args& a, const attend_row* srow, int n_rows, const char* sk, const char* sv) {
        const int lane = threadIdx.x & 63, c32 = lane & 31, G = a.n_heads / a.n_kv, col = 32 * (int)(threadIdx.x / WAVE % TILE_COLUMNS) + c32;
        hh = lane >> 5;
        lr = col / G;
        g = col - lr * G;
        there = lr < n_rows;
        const attend_row me = srow[there ? lr : 0];
        last = !there ? -1 : RUN ? me.pos : min(me.shared, me.pos + 1) - 1; /* the last position it may see here */
        low = a.window ? me.pos - a.window + 1 : INT32_MIN;
        on = there && last >= 0;
        wave_on = __any(on);
        at(sk, sv);
        key_x = (hh ^ (c32 & (HD / 8 - 1))) << 4; /* piece 2 s + hh: ^ s << 5 */
        /* unit 2 s + hh of dimension 32 d + c32: ^ (s ^ d) << 5 (POS 32: ^ s << 5) */
        value_x = (POS == 64 ? hh ^ ((c32 >> 1) & 7) ^ (c32 >> 4) : hh ^ ((c32 >> 2) & 3)) << 4;
        m_run = -INFINITY;
        l_run = 0.0f;
        e_out = 126;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) O[d][i] = 0.0f;
    }
    /* The queries, through 4 KB of LDS of the wave's own, 32 dimensions at a time: loaded 128 bytes a column (a lane a
       column would ask for 64 lines an instruction, 18000 cycles a block), taken as operand 16 s + 8 hh ..; meanwhile asks
       for more behind them */
    template <typename F>
    __device__ __forceinline__ void load_queries(const attend_args& a, int h, int row0, int n_rows, char* mine, F&& meanwhile) {
        const int wave = threadIdx.x / WAVE % TILE_COLUMNS, lane = threadIdx.x & 63, c32 = lane & 31, G = a.n_heads / a.n_kv;
        float4 in[KS / 2][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = 32 * wave + 8 * i + (lane >> 3), r = min(c / G, n_rows - 1);
            const float* from = a.q + (size_t)(row0 + r) * a.q_stride + (size_t)(h * G + c % G) * HD + 4 * (lane & 7);
#pragma unroll
            for (int t = 0; t < KS / 2; t++) in[t][i] = *reinterpret_cast<const float4*>(from + 32 * t);
        }
        __builtin_amdgcn_sched_barrier(0);
        meanwhile();
        __builtin_amdgcn_sched_barrier(0);
        /* a column's largest magnitude, from its eight lanes to its two */
        uint32_t mag = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t most = 0;
#pragma unroll
            for (int t = 0; t < KS / 2; t++) most = max(max(most, max(magnitude(in[t][i].x), magnitude(in[t][i].y))), max(magnitude(in[t][i].z), magnitude(in[t][i].w)));
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d, WAVE));
            most = (uint32_t)__shfl((int)most, 8 * (c32 & 7), WAVE);
            if ((c32 >> 3) == i) mag = most;
        }
        const int k = to_half_range(mag);
        const float f = two_to(k);
        to_score = a.scale * 1.44269504088896340736f * two_to(-k);
#pragma unroll
        for (int t = 0; t < KS / 2; t++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = 8 * i + (lane >> 3);
                *reinterpret_cast<float4*>(mine + c * 128 + (((lane & 7) ^ (c & 7)) << 4)) = in[t][i];
            }
            __builtin_amdgcn_wave_barrier(); /* LDS operations of one wave complete in order */
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const float4 x = *reinterpret_cast<const float4*>(mine + c32 * 128 + (((4 * s + 2 * hh) ^ (c32 & 7)) << 4));
                const float4 y = *reinterpret_cast<const float4*>(mine + c32 * 128 + (((4 * s + 2 * hh + 1) ^ (c32 & 7)) << 4));
                uint2 h0, l0, h1, l1;
                cut4(x.x, x.y, x.z, x.w, f, h0, l0);
                cut4(y.x, y.y, y.z, y.w, f, h1, l1);
                qh[2 * t + s] = __builtin_bit_cast(h8v, u32x4{h0.x, h0.y, h1.x, h1.y});
                ql[2 * t + s] = __builtin_bit_cast(h8v, u32x4{l0.x, l0.y, l1.x, l1.y});
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
    /* S: sums of products of the keys in LDS; lane: positions 32 pt + 8 (i / 4) + 4 hh + i % 4 of its column */
    __device__ __forceinline__ void scores() {
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
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
                    const h8v kl = *reinterpret_cast<const h8v*>(at + LO);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[s], acc, 0, 0, 0);
                }
            }
            S[pt] = acc;
        }
    }
    /* S from sums to weights of positions t0 .. t1 - 1, 2^(WEIGHT_EXP + down) exp2(score - m_run) (down <= 0). m_run, and
       with it O and the sum, follows the maximum only where that is WEIGHT_SLACK above it: a weight then is 2^14 at most, as
       f16 holds, and after a few chunks hardly any rescale O (a wave's 32 columns would at every other). keys: to_score with
       the keys' power of two; e: the values' power of two in LDS, less down; bad0, bad1: the positions whose values are no
       numbers. */
    __device__ __forceinline__ void weights(const attend_args& a, int t0, int t1, float keys, int e, int down, uint32_t bad0, uint32_t bad1) {
        keys = fmaxf(keys, 1e-37f); /* (a masked score's -inf times 0 would be NaN) */
        const bool whole = !__any(on && !(t0 + POS <= t1 && t0 + POS - 1 <= last && (t0 >= low || t0 + POS <= a.sinks))) && __all(on);
        if (!whole) {
            /* of the lane's positions, t0 + 4 hh + 32 pt + 8 (i / 4) + i % 4 */
            const int to_last = on ? min(last, t1 - 1) - t0 - 4 * hh : -1, to_low = max(low, -1) - t0 - 4 * hh, to_sink = a.sinks - t0 - 4 * hh;
#pragma unroll
            for (int pt = 0; pt < PT; pt++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = 32 * pt + 8 * (i >> 2) + (i & 3);
                    const bool sees = t <= to_last && (t >= to_low || t < to_sink);
                    S[pt][i] = sees ? S[pt][i] : -INFINITY;
                }
        }
        float m = -INFINITY;
#pragma unroll
        for (int pt = 0; pt < PT; pt++)
#pragma unroll
            for (int i = 0; i < 16; i++) m = fmaxf(m, S[pt][i]);
        m = fmaxf(m, __shfl_xor(m, 32, WAVE)) * keys;
        m = m > m_run + WEIGHT_SLACK ? m : m_run;
        const float base = m == -INFINITY ? 0.0f : m;
        float f = exp2_hw(m_run - base), l = 0.0f;
        const float up = (float)(WEIGHT_EXP + down) - base;
        if (__builtin_expect((bad0 | bad1) != 0, 0)) {
#pragma unroll
            for (int pt = 0; pt < PT; pt++) {
                const uint32_t poison = pt ? bad1 : bad0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float x = S[pt][i];
                    if (((poison >> (8 * (i >> 2) + 4 * hh + (i & 3))) & 1) && !(x == -INFINITY)) l = NAN;
                }
            }
        }
#pragma unroll
        for (int pt = 0; pt < PT; pt++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                S[pt][i] = exp2_hw(fmaf(S[pt][i], keys, up));
                l += S[pt][i];
            }
        l *= two_to(min(-down, 126));
        l_run = fmaf(l_run, f, l);
        m_run = m;
        if constexpr (SCALED) {
            f *= two_to(max(e - e_out, -126));
            e_out = e;
        }
        if (__any(f != 1.0f)) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) O[d][i] *= f;
        }
    }
    /* O += weights of the values in LDS */
    __device__ __forceinline__ void values() {
#pragma unroll
        for (int s = 0; s < POS / 16; s++) {
            /* positions 16 s + 8 (j / 4) + 4 hh + j % 4 as the MFMA's eight, on both operands */
            const f16v& P = S[s >> 1];
            const int o = 8 * (s & 1);
            uint2 h0, l0, h1, l1;
            cut4(P[o], P[o + 1], P[o + 2], P[o + 3], h0, l0);
            cut4(P[o + 4], P[o + 5], P[o + 6], P[o + 7], h1, l1);
            const h8v ph = __builtin_bit_cast(h8v, u32x4{h0.x, h0.y, h1.x, h1.y}), pl = __builtin_bit_cast(h8v, u32x4{l0.x, l0.y, l1.x, l1.y});
            h8v v[DT], vl[DT];
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const char* at = value_at + (value_x ^ ((POS == 64 ? s ^ d : s) << 5)) + 32 * d * POS * 2;
                v[d] = *reinterpret_cast<const h8v*>(at);
                if constexpr (PARTS) vl[d] = *reinterpret_cast<const h8v*>(at + LO);
            }
            /* one accumulator's products apart */
#pragma unroll
            for (int d = 0; d < DT; d++) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph, O[d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < DT; d++) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl, O[d], 0, 0, 0);
            if constexpr (PARTS) {
#pragma unroll
                for (int d = 0; d < DT; d++) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl[d], ph, O[d], 0, 0, 0);
            }
        }
    }
    /* Two waves of the same columns: half HALF of the dimensions of this one's O, m and l to room; the other's to this one's
       O. m_run and e_out are the same in a column's two lanes. */
    template <int HALF>
    __device__ __forceinline__ void give(float4* room) const {
        const int at = threadIdx.x % (WAVE * TILE_COLUMNS);
#pragma unroll
        for (int x = 0; x < DT * 2; x++) {
            const f16v& o = O[HALF * DT / 2 + x / 4];
            const int i = 4 * (x % 4);
            room[x * WAVE * TILE_COLUMNS + at] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
        room[DT * 2 * WAVE * TILE_COLUMNS + at] = make_float4(m_run, l_run, 0.0f, 0.0f);
    }
    template <int HALF>
    __device__ __forceinline__ void take(const float4* room) {
        const int at = threadIdx.x % (WAVE * TILE_COLUMNS);
        const float4 ml = room[DT * 2 * WAVE * TILE_COLUMNS + at];
        const float m = fmaxf(m_run, ml.x), base = m == -INFINITY ? 0.0f : m, f = exp2_hw(m_run - base), g_ = exp2_hw(ml.x - base);
        l_run = fmaf(l_run, f, ml.y * g_);
        m_run = m;
#pragma unroll
        for (int x = 0; x < DT * 2; x++) {
            const float4 y = room[x * WAVE * TILE_COLUMNS + at];
            f16v& o = O[HALF * DT / 2 + x / 4];
            const int i = 4 * (x % 4);
            o[i] = fmaf(o[i], f, y.x * g_); o[i + 1] = fmaf(o[i + 1], f, y.y * g_); o[i + 2] = fmaf(o[i + 2], f, y.z * g_); o[i + 3] = fmaf(o[i + 3], f, y.w * g_);
        }
    }
    /* dimensions 32 D0 .. 32 D1 - 1 */
    template <int D0, int D1>
    __device__ __forceinline__ void flush(const attend_args& a, const attend_parts& p, int split, int h, int row0) {
        l_run += __shfl_xor(l_run, 32, WAVE);
        if (!there) return;
        const int S_ = p.own + p.tile, G = a.n_heads / a.n_kv;
        const size_t row = (size_t)(row0 + lr), part = ((row * a.n_kv + h) * S_ + p.own + split) * G + g;
        const float back = SCALED ? two_to(-e_out) : 1.0f;
        float* to;
        float f;
        if (S_ == 1) {
            to = a.out + row * a.out_stride + (size_t)(h * G + g) * HD;
            f = l_run == 0.0f ? 0.0f : back / l_run;
        } else {
            if (hh == 0 && D0 == 0) p.ml[part] = make_float2(m_run, l_run * two_to(-WEIGHT_EXP));
            if (l_run == 0.0f) return;
            to = p.acc + part * HD;
            f = back * two_to(-WEIGHT_EXP);
        }
#pragma unroll
        for (int d = D0; d < D1; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<float4*>(to + 32 * d + 8 * i + 4 * hh) = make_float4(O[d][4 * i] * f, O[d][4 * i + 1] * f, O[d][4 * i + 2] * f, O[d][4 * i + 3] * f);
    }
};

/* Split split of splits of what the columns of rows row0 + 0 .. n_rows - 1 see together: RUN, rows of one sequence, each up to itself;
   otherwise a group's shared prefix. srow are the rows. */
template <int HD, typename T, int NW, bool RUN>
__device__ __forceinline__ void group_part(const attend_args& a, const attend_parts& p, int split, int splits, int h, int row0, int n_rows,
                                           const attend_row* srow, const group_span& s, char* lds) {
    typedef tile_shape<HD, T, NW> sh;
    typedef chunk_share<HD, T, 64 * NW> share;
    typedef wave_columns<HD, T, sh::POS> columns;
    const int tid = threadIdx.x, side = __builtin_amdgcn_readfirstlane(tid / (WAVE * TILE_COLUMNS));
    uint32_t* smax = reinterpret_cast<uint32_t*>(lds); /* [2][NW]: magnitudes of keys, of values */
    uint32_t* sbad = smax + 2 * NW;                    /* positions whose values are not finite */
    char* sk = lds + sh::HEAD;
    char* sv = sk + sh::KEYS;
    /* seen, in chunks of 64 */
    const int n_sink = (s.sink + 63) >> 6, n_chunks = n_sink + ((s.end - s.from + 63) >> 6);
    const int per = (n_chunks + splits - 1) / splits, c0 = split * per, c1 = min(c0 + per, n_chunks);
    columns w;
    w.template init<RUN>(a, srow, n_rows, sk + side * sh::SIDE, sv + side * sh::SIDE);
    if (c0 < c1) {
        if (tid < 2) sbad[tid] = 0;
        const T* ks = (const T*)a.k + (size_t)h * a.head_stride + (size_t)s.seq * a.seq_stride;
        const T* vs = (const T*)a.v + (size_t)h * a.head_stride + (size_t)s.seq * a.seq_stride;
        auto start = [&](int c) { return c < n_sink ? 64 * c : s.from + 64 * (c - n_sink); };
        auto stop = [&](int c) { return c < n_sink ? s.sink : s.end; };
        int e_run = 126; /* the values' power of two, the least so far */
        share rk, rv;
        w.load_queries(a, h, row0, n_rows, sk + (tid >> 6) * 4096, [&] {
            rk.fetch(ks, a.pos_stride, start(c0), stop(c0));
            rv.fetch(vs, a.pos_stride, start(c0), stop(c0));
        });
        rk.publish(smax);
        lds_barrier();
        for (int c = c0; c < c1; c++) {
            const int t0 = start(c), t1 = stop(c);
            /* keys to LDS; every wave is past the last chunk's scores */
            float from_keys = w.to_score, f = 1.0f;
            if constexpr (sh::SCALED) {
                uint32_t mag = share::largest(smax);
                if (__builtin_expect(mag >= MAG_INF, 0)) mag = rk.finite_largest(smax);
                const int k = to_half_range(mag);
                f = two_to(k);
                from_keys *= two_to(-k);
            }
            rk.template store_keys<sh::POS>(sk, f, sh::SIDE);
            rv.publish(smax + NW);
            if (c + 1 < c1) rk.fetch(ks, a.pos_stride, start(c + 1), stop(c + 1));
            lds_barrier();
            if (w.wave_on) w.scores();
            uint32_t mag = share::largest(smax + NW);
            const bool bad = mag >= MAG_INF;
            if (__builtin_expect(bad, 0)) {
                mag = rv.finite_largest(smax + NW);
                rv.take_out(sbad);
                lds_barrier();
            }
            if constexpr (sh::SCALED) e_run = min(e_run, to_half_range(mag));
            if (w.wave_on) w.weights(a, t0 + side * sh::POS, t1, from_keys, e_run, 0, bad ? sbad[side] : 0, bad && sh::SIDES == 1 ? sbad[1] : 0);
            /* values to LDS; every wave is past the last chunk's values */
            rv.template store_values<sh::POS>(sv, sh::SCALED ? two_to(e_run) : 1.0f, sh::SIDE);
            if constexpr (sh::SCALED) {
                if (c + 1 < c1) rk.publish(smax);
            }
            if (c + 1 < c1) rv.fetch(vs, a.pos_stride, start(c + 1), stop(c + 1));
            lds_barrier();
            if (bad && tid < 2) sbad[tid] = 0; /* read before this barrier, next written behind another */
            if (w.wave_on) w.values();
        }
    }
    if constexpr (sh::SIDES == 1) {
        w.template flush<0, columns::DT>(a, p, split, h, row0);
    } else {
        /* each side the other's half of what it has, through LDS, then to memory its own */
        float4* room = reinterpret_cast<float4*>(sk);
        float4* other = room + sh::MEET / 32;
        lds_barrier(); /* every wave is past the last values */
        if (side) w.template give<0>(other);
        else w.template give<1>(room);
        lds_barrier();
        if (side) {
            w.template take<1>(room);
            w.template flush<columns::DT / 2, columns::DT>(a, p, split, h, row0);
        } else {
            w.template take<0>(other);
            w.template flush<0, columns::DT / 2>(a, p, split, h, row0);
        }
    }
}

/* ---- a prompt's chunk over images of the cache ----
   Cutting 64 positions into parts is as much vector work as one wave's products with them is matrix work, and every tile of
   rows repeats it, in step with its barriers. Where many tiles read the same positions they are cut once, into images of what
   the LDS then holds, 32 positions each. A tile's block only copies: the next 32 positions while it works on these, so that
   a copy has the time of 96 products to arrive, and the two blocks of a compute unit (four waves, 64 KB each) fill each
   other's gaps. */
#define IMAGE_WAVES 4
template <int HD, typename T>
constexpr int image_part = (sizeof(T) == 4 ? 2 : 1) * 32 * HD * 2; /* bytes of 32 positions' keys, and of their values behind them */

/* Chunk c (positions 64 c ..) lies in slot c (c < x) or c - y; no row sees positions z .. w - 1. */
__device__ __forceinline__ int4 image_slots(const attend_args& a, uint32_t far, uint32_t near) {
    const int end = min((int)far, a.ctx), least = near ? (int)(0x80000000u - near) : 0;
    const int sink = a.window ? min(a.sinks, end) : 0, from = a.window ? min(max(sink, least - a.window + 1), end) : 0;
    const int n_sink = (sink + 63) >> 6;
    return make_int4(n_sink, max(n_sink, from >> 6) - n_sink, sink, max(sink, from));
}

/* Block (key-value head, slot): 64 positions. Bound by bytes: the 5120 positions behind 1024 rows of a 4096 window, 21 MB in
   and as many out in 10-11 us. */
template <int HD, typename T>
__global__ __launch_bounds__(256) void attend_image_kernel(attend_args a, attend_parts p) {
    typedef chunk_share<HD, T, 256> share;
    constexpr int PART = image_part<HD, T>;
    __shared__ __attribute__((aligned(16))) char image[4 * PART];
    __shared__ uint32_t smax[2][4], sbad[2];
    const int tid = threadIdx.x, wave = tid >> 6, h = blockIdx.x % a.n_kv, slot = blockIdx.x / a.n_kv;
    /* the run's furthest and nearest positions */
    uint32_t far = 0, near = 0;
    int seq = a.run_seq;
    if (a.recs) {
        for (int i = tid; i < a.n; i += 256) {
            const attend_row r = row_of(a, i);
            if (r.pos >= 0) {
                far = max(far, (uint32_t)r.pos + 1);
                near = max(near, 0x80000000u - (uint32_t)r.pos);
            }
        }
        far = wave_umax(far);
        near = wave_umax(near);
        if ((tid & 63) == 0) { smax[0][wave] = far; smax[1][wave] = near; }
        __syncthreads();
        far = share::largest(smax[0]);
        near = share::largest(smax[1]);
        seq = row_of(a, 0).seq;
        __syncthreads();
    } else {
        far = a.run_pos + a.n;
        near = 0x80000000u - (uint32_t)a.run_pos;
    }
    if (tid < 2) sbad[tid] = 0;
    const int4 at = image_slots(a, far, near);
    if (blockIdx.x == 0 && tid == 0) p.meta[0] = make_int4(at.x, at.y, 0, 0);
    const int end = min((int)far, a.ctx), c = slot < at.x ? slot : slot + at.y;
    if (64 * c >= end) return;
    const T* ks = (const T*)a.k + (size_t)h * a.head_stride + (size_t)seq * a.seq_stride;
    const T* vs = (const T*)a.v + (size_t)h * a.head_stride + (size_t)seq * a.seq_stride;
    share rk, rv;
    rk.fetch(ks, a.pos_stride, 64 * c, end, at.z, at.w);
    rv.fetch(vs, a.pos_stride, 64 * c, end, at.z, at.w);
    rk.publish(smax[0]);
    rv.publish(smax[1]);
    __syncthreads();
    uint32_t mk = share::largest(smax[0]), mv = share::largest(smax[1]);
    if (__builtin_expect(mk >= MAG_INF, 0)) mk = rk.finite_largest(smax[0]);
    if (__builtin_expect(mv >= MAG_INF, 0)) {
        mv = rv.finite_largest(smax[1]);
        rv.take_out(sbad);
    }
    const int kk = to_half_range(mk), kv = to_half_range(mv);
    rk.template store_keys<32>(image, two_to(kk), 2 * PART);
    rv.template store_values<32>(image + PART, two_to(kv), 2 * PART);
    __syncthreads();
    const size_t to = (size_t)h * p.slots + slot;
    u32x4* out = reinterpret_cast<u32x4*>(p.images + to * 4 * PART);
    for (int i = tid; i < 4 * PART / 16; i += 256) out[i] = reinterpret_cast<const u32x4*>(image)[i];
    if (tid == 0) p.meta[1 + to] = make_int4(kk, kv, (int)sbad[0], (int)sbad[1]);
}

/* A wave's share of BYTES to LDS, asked for; image_wait waits for all waves'. */
template <int BYTES>
__device__ __forceinline__ void image_load(const char* from, char* to) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < BYTES / 1024 / IMAGE_WAVES; j++) {
        const int at = (j * IMAGE_WAVES + wave) * 1024;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + at + 16 * lane),
                                         (__attribute__((address_space(3))) void*)(to + at), 16, 0, 0);
    }
}
__device__ __forceinline__ void image_wait() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
}

/* Block (tile, key-value head), split. Bound by the matrix cores and what the waves do beside them: 1024 rows of 32 heads with
   a 4096 window and four sinks (4 heads of 128, float32), 206 GFLOP as three products each, in 185-205 us: 1.0-1.1 PFLOP/s
   of the 2.07 that products alone reach; 57 % of a SIMD's cycles are products, 25 % of a wave's waits for the others of its
   block. (The next step's scores formed beside this one's weights, 256 registers: 229 us for the call, 214 so.) */
template <int HD, typename T>
__global__ __launch_bounds__(64 * IMAGE_WAVES, HD == 128 ? 2 : 3) void attend_imaged_kernel(attend_args a, attend_parts p) {
    constexpr int PART = image_part<HD, T>, ROOM = 2 * PART > IMAGE_WAVES * 4096 ? 2 * PART : IMAGE_WAVES * 4096; /* (the queries pass through the first) */
    typedef wave_columns<HD, T, 32> columns;
    /* arrays of their own: a copy into one is not waited for before the other is read */
    __shared__ __attribute__((aligned(1024))) char even[ROOM];
    __shared__ __attribute__((aligned(1024))) char odd[2 * PART];
    __shared__ attend_row srow[32 * IMAGE_WAVES];
    const int tid = threadIdx.x, split = blockIdx.y, h = blockIdx.x % a.n_kv, G = a.n_heads / a.n_kv, TR = 32 * IMAGE_WAVES / G;
    const int r0 = blockIdx.x / a.n_kv * TR, nr = min(TR, a.n - r0);
    load_rows<64 * IMAGE_WAVES>(a, r0, nr, srow);
    lds_barrier();
    const group_span s = group_seen<true>(a, srow, 0, nr);
    const int4 at = p.meta[0];
    /* seen, in steps of 32 positions: u < n_sink, and from first on */
    const int n_sink = (s.sink + 31) >> 5, first = max(n_sink, s.from >> 5), steps = n_sink + max(((s.end + 31) >> 5) - first, 0);
    const int per = (steps + p.tile - 1) / p.tile, i0 = split * per, i1 = min(i0 + per, steps);
    columns w;
    w.template init<true>(a, srow, nr, even, even + PART);
    if (i0 < i1) {
        w.load_queries(a, h, r0, nr, even + (tid >> 6) * 4096, [] {});
        const char* images = p.images + (size_t)h * p.slots * 4 * PART;
        const int4* meta = p.meta + 1 + (size_t)h * p.slots;
        auto step = [&](int i) { return i < n_sink ? i : first + (i - n_sink); };
        auto slot = [&](int i) { const int c = step(i) >> 1; return c < at.x ? c : c - at.y; };
        auto image = [&](int i) { return images + ((size_t)slot(i) * 2 + (step(i) & 1)) * 2 * PART; };
        int e_run = 126;
        /* a step's powers and bad positions, by scalar loads (vector ones would wait for the copies asked for before them) */
        auto meta_of = [&](int i) { return *(const __attribute__((address_space(4))) int4_*)(const int4_*)(meta + slot(i)); };
        auto work = [&](int i, int4_ m, const char* room) {
            const int u = step(i);
            w.at(room, room + PART);
            w.scores();
            /* operands two steps ahead of their products */
            constexpr int R = columns::PARTS ? 2 : 1, M = columns::PARTS ? 3 : 2;
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * R, 0);
#pragma unroll
            for (int g = 0; g < columns::KS - 2; g++) {
                __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * M, 0);
            if constexpr (columns::SCALED) e_run = min(e_run, m.y);
            w.weights(a, 32 * u, s.end, columns::SCALED ? w.to_score * two_to(-m.x) : w.to_score, e_run, columns::SCALED ? e_run - m.y : 0,
                      u & 1 ? m.w : m.z, 0);
            w.values();
        };
        lds_barrier(); /* every wave has its queries */
        image_load<2 * PART>(image(i0), even);
        for (int i = i0; i < i1; i += 2) {
            const int4_ m0 = meta_of(i);
            image_wait(); /* this step's images are there; every wave is past the last one's */
            if (i + 1 < i1) image_load<2 * PART>(image(i + 1), odd);
            if (w.wave_on) work(i, m0, even);
            if (i + 1 >= i1) break;
            const int4_ m1 = meta_of(i + 1);
            image_wait();
            if (i + 2 < i1) image_load<2 * PART>(image(i + 2), even);
            if (w.wave_on) work(i + 1, m1, odd);
        }
    }
    w.template flush<0, columns::DT>(a, p, split, h, r0);
}

/* Block y's of a tile's rows: RUN its split of all together, otherwise of the groups of many columns, each a unit. */
template <int HD, typename T, int NW, bool RUN>
__device__ __forceinline__ void tile_part(const attend_args& a, const attend_parts& p, int y, int h, int tile, char* lds) {
    const int G = a.n_heads / a.n_kv, TR = tile_rows<HD>(G), r0 = tile * TR, nr = min(TR, a.n - r0);
    attend_row* srow = reinterpret_cast<attend_row*>(lds);
    char* rest = lds + tile_rows<HD>(1) * sizeof(attend_row);
    load_rows<64 * NW>(a, r0, nr, srow);
    lds_barrier();
    if constexpr (RUN) {
        group_part<HD, T, NW, true>(a, p, y, p.tile, h, r0, nr, srow, group_seen<true>(a, srow, 0, nr), rest);
    } else {
        int units = 0;
        for (int first = 0, next; first < nr; first = next) {
            next = group_end(srow, first, nr);
            units += (next - first) * G > p.few;
        }
        if (!units) return;
        const unit_share u(units, p.busy, y, p.tile);
        int unit = 0;
        for (int first = 0, next; first < nr; first = next) {
            next = group_end(srow, first, nr);
            if ((next - first) * G <= p.few || !u.mine(unit++)) continue;
            empty_parts(a, p, u, h, r0 + first, 0, (next - first) * G);
            group_part<HD, T, NW, false>(a, p, u.part(), u.parts, h, r0 + first, next - first, srow + first, group_seen<false>(a, srow, first, next), rest);
            lds_barrier();
        }
    }
}

/* ---- the kernels ---- */

#define OWN_WAVES 4

/* Rows' own parts alone: block (row, key-value head), split. Bound by the cache's bytes: 32 rows of a 4096 window and four
   sinks (f16, 4 heads of 128), 270 MB in 69-71 us, 3.8-3.9 TB/s, where a large copy reaches 4.8. One row's 1028 float32
   positions: 7 us, five of them a launch, the rows and two dependent steps. */
template <int HD, typename T>
__global__ __launch_bounds__(64 * OWN_WAVES, 2) void attend_own_kernel(attend_args a, attend_parts p) {
    __shared__ __attribute__((aligned(16))) char lds[columns_lds<HD, OWN_WAVES>];
    own_part<HD, T, OWN_WAVES>(a, p, blockIdx.y, blockIdx.x % a.n_kv, blockIdx.x / a.n_kv, lds);
}

/* The prefixes of groups of few columns and the rows' own parts. 40 rows of 16 heads of 128 in groups of eight behind 2048
   positions (bfloat16): 139 MB in 46-49 us, 3 TB/s; the blocks of a group's prefix are long ones, and its products (16
   columns, half of them used) run beside the loads of the next step. 32 rows' own 256 positions (float32): 11 us. */
template <int HD, typename T>
__global__ __launch_bounds__(64 * OWN_WAVES, 2) void attend_columns_kernel(attend_args a, attend_parts p) {
    __shared__ __attribute__((aligned(16))) char lds[columns_lds<HD, OWN_WAVES> + tile_rows<HD>(1) * sizeof(attend_row)];
    /* first the blocks of few_part that get work if any do, behind the own parts those that only many groups need (idle ones
       before the own parts: 40 rows in groups of eight behind 2048 positions 61.5 us; so 53.9) */
    const int heads = a.n_kv, h = blockIdx.x % heads, busy = min(p.busy, p.few_blocks) * p.tiles, own = a.n * p.own, b = blockIdx.x / heads;
    if (b >= busy && b < busy + own) {
        own_part<HD, T, OWN_WAVES>(a, p, (b - busy) % p.own, h, (b - busy) / p.own, lds);
    } else {
        const int x = b < busy ? b : b - own; /* block x / tiles of tile x mod tiles */
        few_part<HD, T, OWN_WAVES>(a, p, x / p.tiles, h, x % p.tiles, lds);
    }
}

/* 32 rows of 32 heads behind 8192 positions (4 heads of 128, float32): 32 us, of which a block works 27: 2 for its rows, 6
   until its queries and first chunk are there, 15 for four chunks (7700 cycles each, 3100 of them products) and 4 to
   exchange and write. Blocks of 256 columns and half as many chunks wrote and read back twice as many parts (the call 54
   us for 45). */
#define XCDS 8
template <int HD, typename T, bool RUN>
__global__ __launch_bounds__(64 * tile_waves<HD>, 2) void attend_tile_kernel(attend_args a, attend_parts p) {
    __shared__ __attribute__((aligned(16))) char lds[tile_shape<HD, T, tile_waves<HD>>::LDS];
    /* the tiles of a head's split next to each other on one die, whose cache then serves all but the first */
    const int tile = blockIdx.x / XCDS % p.tiles, pair = blockIdx.x / (XCDS * p.tiles) * XCDS + blockIdx.x % XCDS;
    if (pair < a.n_kv * p.tile_blocks) tile_part<HD, T, tile_waves<HD>, RUN>(a, p, pair / a.n_kv, pair % a.n_kv, tile, lds);
}

/* HB heads of a row a block, SG threads for each four dimensions of one: the parts' factors once in LDS, then each
   thread adds up every SG-th part, all its loads asked for before the first is used. Bound by the parts'
   bytes: 1024 rows of 32 heads in two parts, 50 MB in 12 us, 4.3 TB/s; 32 rows in 40 parts, 21 MB in 5.5. */
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

/* A run of so many tiles or more goes over images, if they take no more bytes than this. Behind 3000 positions, 32 heads of
   128 on 4, float32: 8 tiles 46 us over images and 41 without, 12 tiles 56 and 81, 21 tiles 79 and 135; 8 heads of 64 on 2,
   bfloat16: 6 tiles 25 and 18, 11 tiles 28 and 29. */
#define IMAGE_TILES 9
#define IMAGE_BYTES_MAX ((size_t)256 << 20)

/* How a call is cut into blocks. */
static attend_parts plan(const attend_args& a) {
    attend_parts p = {};
    const int G = a.n_heads / a.n_kv, rows = (a.hd == 128 ? tile_rows<128>(G) : tile_rows<64>(G));
    p.tiles = (a.n + rows - 1) / rows;
    const long seen = a.window ? std::min<long>(a.own_max, (long)a.window + a.sinks) : a.own_max;
    const long blocks = 256; /* a block a compute unit */
    if (a.run) {
        const int few_rows = 32 * IMAGE_WAVES / G, few_tiles = (a.n + few_rows - 1) / few_rows;
        /* the images' slots: consecutive rows see window + n positions and the sinks */
        const long reach = (a.own_max + 63) / 64 + 1, near = a.window ? (std::min(a.sinks, a.own_max) + 63) / 64 + ((long)a.window + a.n + 63) / 64 + 2 : reach;
        const long slots = a.recs ? reach : std::min(reach, near);
        const size_t bytes = (size_t)slots * a.n_kv * 2 * 64 * a.hd * 2 * (a.dtype == VITNA_DTYPE_F32 ? 2 : 1);
        if (few_tiles >= IMAGE_TILES && bytes <= IMAGE_BYTES_MAX) {
            const long per_tile = (a.window ? std::min<long>(a.own_max, (long)a.window + a.sinks + few_rows) : a.own_max) / 64 + 2;
            p.tiles = few_tiles;
            p.slots = (int)slots;
            p.tile = (int)std::min<long>(std::min<long>(per_tile, 64), std::max<long>(1, 2 * blocks / ((long)few_tiles * a.n_kv)));
            return p;
        }
        const long chunks = (a.window ? std::min<long>(a.own_max, (long)a.window + a.sinks + rows) : a.own_max) / 64 + 1;
        p.tile = p.tile_blocks = (int)std::min<long>(std::min<long>(chunks, 64), std::max<long>(1, blocks / ((long)p.tiles * a.n_kv)));
        return p;
    }
    if (a.shared_max) {
        /* a block a compute unit; a tile's groups may need a block each */
        const long chunks = (a.window ? std::min<long>(a.shared_max, (long)a.window + a.sinks) : a.shared_max) / 64 + 1;
        const long columns = (long)a.n * G;
        const bool few = columns <= FEW_CALL || columns * std::min(chunks * 64, (long)a.shared_max) <= FEW_WORK;
        p.few = few ? 32 * TILE_COLUMNS : FEW_COLUMNS;
        /* Twice as many splits: 40 rows of 16 key-value heads in groups of eight behind 2048 positions (float32) 52 us for 44,
           behind 8000 134 for 128 (bfloat16 94 for 112), 32 rows of 4 behind 8192 60 for 45. */
        const long at_once = std::max<long>(1, blocks / ((long)p.tiles * a.n_kv));
        const long groups = std::min(a.n, rows), big = std::min<long>(32 * TILE_COLUMNS / (FEW_COLUMNS + 1), groups); /* a tile's units at most: a row is one at most */
        p.tile = (int)std::min<long>(std::min<long>(chunks, 64), at_once);
        p.busy = (int)at_once;
        p.few_blocks = (int)std::min<long>(std::max<long>(p.busy, groups), groups * p.tile);
        p.tile_blocks = few ? 0 : (int)std::min<long>(std::max<long>(p.busy, big), big * p.tile);
    }
    p.own = (int)std::min<long>(std::min<long>((seen + 16 * OWN_WAVES - 1) / (16 * OWN_WAVES), ATTEND_SPLITS_MAX), std::max<long>(1, 1024 / ((long)a.n * a.n_kv)));
    if (a.splits) p.own = std::min(a.splits, ATTEND_SPLITS_MAX);
    return p;
}

/* Bytes of work: maxima and sums, values, images and their meta; where they lie in it, into p (base may be null). */
static size_t place_parts(const attend_args& a, attend_parts& p, char* base) {
    const size_t S = (size_t)p.own + p.tile, heads = S > 1 ? (size_t)a.n * a.n_heads * S : 0, slots = (size_t)p.slots * a.n_kv;
    const size_t ml = align256(heads * sizeof(float2)), acc = align256(heads * a.hd * sizeof(float));
    const size_t meta = p.slots ? align256((1 + slots) * sizeof(int4)) : 0, images = slots * 2 * 64 * a.hd * 2 * (a.dtype == VITNA_DTYPE_F32 ? 2 : 1);
    p.ml = reinterpret_cast<float2*>(base);
    p.acc = reinterpret_cast<float*>(base + ml);
    p.meta = reinterpret_cast<int4*>(base + ml + acc);
    p.images = base + ml + acc + meta;
    return std::max<size_t>(ml + acc + meta + images, 16);
}

size_t attend_work(const attend_args& a) {
    attend_parts p = plan(a);
    return place_parts(a, p, nullptr);
}

template <int HD, typename T>
static hipError_t launch(const attend_args& a, const attend_parts& p, hipStream_t s) {
    constexpr int NW = tile_waves<HD>;
    const unsigned heads = (unsigned)a.n_kv, tile_blocks = (heads * p.tile_blocks + XCDS - 1) / XCDS * XCDS * p.tiles;
    if (p.slots) {
        attend_image_kernel<HD, T><<<p.slots * heads, 256, 0, s>>>(a, p);
        attend_imaged_kernel<HD, T><<<dim3(p.tiles * heads, p.tile), 64 * IMAGE_WAVES, 0, s>>>(a, p);
    } else if (a.run) {
        attend_tile_kernel<HD, T, true><<<tile_blocks, 64 * NW, 0, s>>>(a, p);
    } else if (p.tile) {
        attend_columns_kernel<HD, T><<<heads * ((unsigned)p.tiles * p.few_blocks + (unsigned)a.n * p.own), 64 * OWN_WAVES, 0, s>>>(a, p);
        if (p.tile_blocks) attend_tile_kernel<HD, T, false><<<tile_blocks, 64 * NW, 0, s>>>(a, p);
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
    if (place_parts(a, p, static_cast<char*>(a.work)) > a.work_bytes || p.own + p.tile > MERGE_SPLITS) return hipErrorInvalidValue;
    if ((long)a.n * a.n_kv > (1L << 22)) return hipErrorInvalidValue; /* threads of a launch stay within 32 bits */
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

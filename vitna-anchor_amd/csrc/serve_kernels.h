/**
 * serve_kernels.h - Host-side launchers of the serving operators' kernels
 * (kernels_attend.hip, kernels_beam.hip), shared by their C entry points
 * (serving.hip) and the engine. Each checks on the host that the shapes it is
 * given are those its kernels assume, and returns hipErrorInvalidValue
 * otherwise, before anything is launched.
 */

#ifndef SERVE_KERNELS_H
#define SERVE_KERNELS_H

#include "vitna_kernels.h"

/* Maximum over the wave of unsigned numbers, in every lane. */
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#define STEP_(C, RM) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, C, RM, 0xf, false))
    STEP_(DPP_ROW_SHR(1), 0xf); STEP_(DPP_ROW_SHR(2), 0xf); STEP_(DPP_ROW_SHR(4), 0xf); STEP_(DPP_ROW_SHR(8), 0xf);
    STEP_(DPP_ROW_BCAST15, 0xa); STEP_(DPP_ROW_BCAST31, 0xc);
#undef STEP_
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

#define ATTEND_G_MAX 16 /* query heads a key-value head */

/* A row of the attention, as the caller's vitna_hip_attention_row_t. */
struct attend_row {
    int32_t seq, pos, base, shared;
};

struct attend_args {
    const void *k, *v; /* element (seq, pos, head, d) at seq * seq_stride + pos * pos_stride + head * head_stride + d */
    size_t seq_stride, pos_stride, head_stride;
    int dtype, n_heads, n_kv, hd, ctx, seqs;
    int window, sinks; /* window 0: none */
    float scale;       /* of the scores */
    const float* q;
    size_t q_stride;
    float* out;
    size_t out_stride;
    int n;
    /* the rows: n of them in rows; or a model's in recs, which share what share (of each sequence: base and number of
       positions; null: nothing) says; or, both null, positions run_pos .. run_pos + n - 1 of sequence run_seq */
    const attend_row* rows;
    const row_rec* recs;
    const int2* share;
    int run_seq, run_pos;
    /* 1: the rows are tokens of one sequence (a prompt's chunk) and share nothing */
    int run;
    int own_max, shared_max; /* the longest own part and the longest shared prefix, about: they size the launch */
    int splits;              /* 0, or the blocks that a row's own part is split over whatever n is (then its bits are, too) */
    void* work;
    size_t work_bytes;
};
/* Bytes of work that launch_attend needs for a's shapes (its pointers are not read). */
size_t attend_work(const attend_args& a);
#define ATTEND_SPLITS_MAX 256 /* of a row's own part */
hipError_t launch_attend(const attend_args& a, hipStream_t s);

struct beam_select_args {
    const float* logits;
    size_t stride, vocab;
    int groups, width, keep;
    const float* scores;
    const uint8_t* ended; /* or null */
    int end_token;
    float* best;
    int *parents, *tokens;
    void* work;
};
size_t beam_select_work(int groups, int width, size_t vocab, int keep);
hipError_t launch_beam_select(const beam_select_args& a, hipStream_t s);

struct kv_reorder_args {
    char *k, *v;
    size_t seq_bytes, layer_bytes, pos_bytes, head_bytes, dim_bytes; /* strides, and a head's bytes */
    int n_kv, ctx, seqs, layers;
    const int *list, *parents, *spans;
    int groups, width, longest;
};
hipError_t launch_kv_reorder(const kv_reorder_args& a, hipStream_t s);

#endif

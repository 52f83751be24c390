// attn_internal.hpp -- argument block and launchers of the attention kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_ffn.h"

namespace moe {

// A decode unit and its pieces: sequence b, head block hb, n pieces of workgroups w0 and on (n < 2: nothing
// to join).
struct Piece {
    int b, hb, w0, n;
};

// One call's sequences, cache and rows (see moe_seq_batch and moe_kv_cache for the layout).
struct AttnArgs {
    const void *q;
    void *o;
    float *lse;               // or null
    int64_t q_stride, o_stride; // elements between rows
    uint8_t *k, *v;
    int64_t page_stride, head_stride, token_stride; // elements
    const int32_t *pages;
    int64_t pages_stride;
    const int32_t *kv_len, *row_start;
    uint32_t *flags;
    int n_pages, max_pages, page_shift;
    int n_seqs, n_rows;
    int hq, hkv, group;       // group = hq / hkv
    float scale_log2;         // scale * log2(e): exponentials are taken in base 2
    float *part;              // workspace: partial rows of pieces (see k_attn_decode.hip)
    float *part_ml;           // ... and each partial row's running maximum and sum
    Piece *piece;             // ... and the units to join
    int n_wg;                 // workgroups of a decode launch
    int n_cu;
    int splits;               // prompt: most pieces of a row (1: not cut)
    unsigned splits_below;    // ... and the most tiles of rows that are cut
    int64_t part_rows;        // rows that part and part_ml hold
};

// Decode: heads of one matrix tile, waves of a workgroup, tokens of a wave's step.
constexpr int DEC_HEADS = 16;
constexpr int DEC_WAVES = 4;
constexpr int DEC_WAVE_TOK = 32;
constexpr int DEC_MAX_WG = 1024;
// Prompt: (token, head) rows of a workgroup.
constexpr int PR_ROWS = 128;
// Workgroups of a prompt's rows however these are divided: each sequence's last tile may be short.
inline int64_t prompt_places(const AttnArgs &a) {
    return ((int64_t)a.n_rows * a.group / PR_ROWS + a.n_seqs) * a.hkv;
}

struct AppendArgs {
    const uint8_t *src[2];    // new keys, new values
    uint8_t *dst[2];
    int64_t src_stride[2];    // bytes between rows
    AttnArgs c;
};

hipError_t launch_kv_append(const AppendArgs &a, int type, int in_type, int d, hipStream_t st);
hipError_t launch_attn_decode(const AttnArgs &a, int type, int d, hipStream_t st);
hipError_t launch_attn_prompt(const AttnArgs &a, int type, int d, hipStream_t st);
hipError_t launch_attn_flags(uint32_t *flags, uint32_t *dst, hipStream_t st);

} // namespace moe

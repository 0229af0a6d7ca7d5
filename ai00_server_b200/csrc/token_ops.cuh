// Tokens from rows of logits as the C entry and the engine ask for them (token_ops.cu; the kernel is in sample_tokens.cuh).
#pragma once
#include "common.cuh"
#include "host.cuh"

namespace b200 {

constexpr int DRAW_MOST_CTAS = 16;
constexpr int DRAW_MAX_VOCAB = 1 << 19;
constexpr int DRAW_MAX_SLICE = DRAW_MAX_VOCAB / DRAW_MOST_CTAS;      // tokens of a CTA

struct DrawParams {
    const void* in;
    long long in_stride;             // elements
    const int* in_row;               // row of `in` of each output row (null: the same)
    const float* uniform;            // [rows], as all of these; null: no limit (temperature: 1)
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* tokens;
    float* probs;                    // null: not wanted
    int V, type;                     // B200RWKV_TYPE_*
    int vec;                         // fours of a CTA's run lie on boundaries
    int ctas_log, slice;             // CTAs of a row, tokens of each (a multiple of four)
};

// ctas_log, slice and vec of p are filled in here; V is at most DRAW_MAX_VOCAB
B200_HIDDEN void draw_rows(cudaStream_t s, DrawParams p, int rows);

}  // namespace b200

// Tokens from rows of logits as the C entry and the engine ask for them (token_ops.cu; the kernel is in sample_tokens.cuh).
#pragma once
#include "common.cuh"
#include "host.cuh"

namespace b200 {

constexpr int DRAW_MOST_CTAS = 16;
constexpr int DRAW_MAX_VOCAB = 1 << 19;
constexpr int DRAW_THREADS = 512;
constexpr int DRAW_SHARED_SLICE = 40960;         // tokens of a CTA that stay in its shared memory
constexpr int DRAW_CLUSTER_SLICE = 65535;        // tokens of a cluster's CTA: its bins hold 16 bits
constexpr int DRAW_ALONE_SLICE = 1 << 18;          // of a CTA that has a row: its bins hold sums of 14 bits each in 32
static_assert(DRAW_MAX_VOCAB / DRAW_MOST_CTAS <= DRAW_CLUSTER_SLICE, "the widest rows fit");

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
    int ctas_log, slice;             // CTAs of a row, tokens of each (a multiple of four)
};

// ctas_log and slice of p are filled in here; V is at most DRAW_MAX_VOCAB
B200_HIDDEN void draw_rows(cudaStream_t s, DrawParams p, int rows);

}  // namespace b200

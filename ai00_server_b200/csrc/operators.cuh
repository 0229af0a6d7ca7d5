// Operators on device memory: their parameters, and their launches as the C entries and the engine make them (operators.cu; the kernels are in
// adapters.cuh and logits.cuh).
#pragma once
#include "common.cuh"
#include "host.cuh"

namespace b200 {

// ---- low-rank adapters ----
constexpr int ADP_CTAS = 8, ADP_THREADS = 256, ADP_WARPS = ADP_THREADS / 32;
constexpr int ADP_TOK = 8;                       // tokens of a group: the N of the products
constexpr int ADP_MAX_PARTS = 8, ADP_MAX_RANK = 256, ADP_MAX_ADAPTERS = 1024;
constexpr int ADP_INLINE = ADP_THREADS;          // tokens of a call whose groups every CTA finds by itself; more take adapter_plan_kernel
constexpr int ADP_PLAN_THREADS = 1024;
constexpr int ADP_TILE = 128;                    // tokens of a tile (adapter_tiles.cuh)

// one adapter of one projection, where adapters lie apart
struct AdapterEntry {
    const void* a;
    const void* b;
    int rank;                    // 0: the adapter leaves this projection alone
    float scale;
};

struct AdapterPart {
    const void* x;               // rows of K, or (x_a16) the A16 layout of common.cuh with x_th as its height
    long long x_stride;          // elements
    int x_a16, x_th;
    int x_lo;                    // rows to the low half of split operands (0: none)
    const void* a;               // [adapters][R][K]
    const void* b;               // [adapters][N][R]
    const AdapterEntry* table;   // instead of a and b
    const void* base;
    long long base_stride;
    void* out;
    long long out_stride;
    int K, N, R;                 // R: the largest rank
    int vec;                     // rows of base and out take accesses of four elements
    int fin;                     // (AdapterParams::finish) `out` has the activation `act` of the sums: AdapterFin
    int act, out_th;             // out_th: height of an A16 output
};
enum AdapterFin : int { ADP_SUMS = 0, ADP_F32 = 1, ADP_A16 = 2, ADP_A16_SPLIT = 3 };

// a call of more tokens than ADP_INLINE: counts of groups (adapters.cuh) and of tiles (adapter_tiles.cuh), {adapter, first place, tokens} of each, tokens by place
struct AdapterPlan {
    int* base;
    int groups, tiles;           // room: as many as there can be
    __host__ __device__ int* count() const { return base; }
    __host__ __device__ int4* group() const { return reinterpret_cast<int4*>(base) + 1; }
    __host__ __device__ int4* tile() const { return group() + groups; }
    __host__ __device__ int* place() const { return reinterpret_cast<int*>(tile() + tiles); }
    __host__ __device__ static size_t ints(int tokens, int groups, int tiles) { return 4 * (1 + (size_t)groups + tiles) + tokens; }
};

struct AdapterParams {
    int tokens, adapters;
    int copy;                    // tokens without an adapter have their base copied (base and out differ)
    int finish;                  // some parts end in their activation (up to ADP_INLINE tokens, f16 to f32); index -2 is then a row behind the last token
    const int* index;
    const float* scale;
    AdapterPlan plan;
    int rank;                    // the largest of the parts
    int nparts;
    int tile_least;              // adapters with fewer tokens than this go by groups
    int out_tokens;              // tokens of a unit of the second tile kernel
    uint8_t* low;                // S between the tile kernels (adapter_tiles.cuh)
    AdapterPart part[ADP_MAX_PARTS];
};

// groups of up to ADP_TOK tokens that `tokens` tokens can need: all with their own adapter, or full groups and a broken one for each adapter (and for none)
__host__ __device__ inline int adapter_groups(int tokens, int adapters) {
    const long long full = (long long)adapters + 1 + tokens / ADP_TOK;
    return (int)(full < tokens ? full : tokens);
}

// bytes that a call of this many tokens needs (0: none), for parts of up to this rank
B200_HIDDEN size_t adapters_workspace(int tokens, int adapters, int nparts, int rank);
// p.plan, p.low and the forms its tokens take, from p.tokens, p.adapters, p.rank and the types
B200_HIDDEN void adapters_shape(AdapterParams& p, void* workspace, int type, int out_type);
// sets up the kernels of a type; a captured call needs it beforehand
B200_HIDDEN void adapters_prepare(int type, int out_type);
// orders the tokens of a longer call by adapter; its groups serve any number of adapters_apply calls with the same tokens
B200_HIDDEN void adapters_plan(cudaStream_t s, const AdapterParams& p);
// the p.nparts parts of p; type: B200RWKV_TYPE_F16 / _BF16, out_type: that or _F32.  Kernels launched
B200_HIDDEN int adapters_apply(cudaStream_t s, const AdapterParams& p, int type, int out_type);

// ---- rows of logits ----
constexpr int LOGITS_STRIPE = 64;                // neighbouring tokens of a CTA; the next ones are the next CTA's
constexpr int LOGITS_MOST_CTAS = 16;             // CTAs of a row
constexpr int LOGITS_LIST_TOKENS = 16384;        // tokens of a CTA whose sums lie in shared memory at once
constexpr int LOGITS_MAX_HISTORY = (1 << 17) - 1;
constexpr int LOGITS_MAX_VOCAB = 1 << 19;
enum LogitsKind : int { LOGITS_ROWS = 0, LOGITS_PROBS = 1, LOGITS_LOGPROBS = 2 };

struct LogitsParams {
    const void* in;
    long long in_stride;         // elements
    float* out;
    long long out_stride;
    int V;
    int kind;
    int vec;                     // fours of a row of `out` on a boundary lie on one in `in`
    int ctas_log;                // log2 of the CTAs of a row
    int list_tokens;             // tokens of a CTA whose sums lie in shared memory at once (0: no lists)
    const int* in_row;           // row of `in` of each output row (null: the same)
    const float* controls;       // [rows][5]: repetition, presence, frequency, decay, temperature
    const int* hist_off;
    const int* hist;
    const int* hist_from;
    const unsigned* allow;
    int words, allow_rows;
    const int* allow_row;
    const int* bias_off;
    const int* bias_tok;
    const float* bias_val;
};

// ctas_log, list_tokens and vec of p are filled in here; V is at most LOGITS_MAX_VOCAB
B200_HIDDEN void logits_rows(cudaStream_t s, LogitsParams p, int rows, int type);

}  // namespace b200

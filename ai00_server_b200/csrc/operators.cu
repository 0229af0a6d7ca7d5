// Operators on device memory: adapters of many requests (adapters.cuh) and adjusted logits (logits.cuh), their C entries and the launches
// the engine makes of them.
#include "operators.cuh"
#include "op_host.cuh"
#include "adapters.cuh"
#include "adapter_tiles.cuh"
#include "logits.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>

namespace b200 {

// tiles that `tokens` tokens can need
static int adapter_tiles(int tokens, int adapters) { return (int)std::min<long long>((long long)adapters + 1 + tokens / ADP_TILE, tokens); }
static size_t adapter_plan_bytes(int tokens, int adapters) {
    return (AdapterPlan::ints(tokens, adapter_groups(tokens, adapters), adapter_tiles(tokens, adapters)) * 4 + 255) & ~(size_t)255;
}

size_t adapters_workspace(int tokens, int adapters, int nparts, int rank) {
    if (tokens <= ADP_INLINE) return 0;
    return adapter_plan_bytes(tokens, adapters) + (size_t)nparts * adt_low_bytes(tokens, rank, 3);
}

// f(element, output) of the types of a call
template <typename F>
static void with_types(int type, int out_type, F&& f) {
    const bool wide = out_type == B200RWKV_TYPE_F32;
    if (type == B200RWKV_TYPE_F16) wide ? f(__half{}, float{}) : f(__half{}, __half{});
    else wide ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

void adapters_shape(AdapterParams& p, void* workspace, int type, int out_type) {
    p.plan.base = nullptr;
    if (p.tokens <= ADP_INLINE) return;
    with_types(type, out_type, [&](auto e, auto o) { p.out_tokens = adt_out_tokens(p.rank, AdpParts<decltype(e), decltype(o)>::N); });
    // tiles for adapters with ADT_LEAST tokens and more; for all of them where there are that many an adapter on average
    p.tile_least = p.tokens >= (long long)ADT_LEAST * p.adapters ? 1 : ADT_LEAST;
    p.plan.base = (int*)workspace;
    p.plan.groups = adapter_groups(p.tokens, p.adapters);
    p.plan.tiles = adapter_tiles(p.tokens, p.adapters);
    p.low = (uint8_t*)workspace + adapter_plan_bytes(p.tokens, p.adapters);
}

void adapters_plan(cudaStream_t s, const AdapterParams& p) { launch(adapter_plan_kernel, dim3(1), ADP_PLAN_THREADS, 0, s, p); }

// types of the engine's own calls
template <typename E, typename O> constexpr bool adapter_finishes = std::is_same_v<E, __half> && std::is_same_v<O, float>;

template <typename E, typename O>
static void ready() {
    constexpr int NP = AdpParts<E, O>::N;
    struct Most { size_t low = 0, out = 0; };
    static const Most most = [] {
        Most m;
        for (int r = 8; r <= ADP_MAX_RANK; r += 8) {
            m.low = std::max<size_t>(m.low, adt_low_smem(r));
            m.out = std::max<size_t>(m.out, adt_out_smem(r, NP));
        }
        return m;
    }();
    prepare<adapter_few_kernel<E, O, false, false>>(adapter_few_smem(ADP_MAX_RANK, NP));
    prepare<adapter_few_kernel<E, O, true, false>>(adapter_few_smem(ADP_MAX_RANK, NP));
    if constexpr (adapter_finishes<E, O>) {
        prepare<adapter_few_kernel<E, O, false, true>>(adapter_few_smem(ADP_MAX_RANK, NP));
    }
    prepare<adapter_low_kernel<E, NP>>(most.low);
    prepare<adapter_out_kernel<E, O>>(most.out);
}

template <typename E, typename O>
static int apply(cudaStream_t s, const AdapterParams& p) {
    constexpr int NP = AdpParts<E, O>::N;
    ready<E, O>();
    int launched = 0;
    int groups = adapter_groups(p.tokens, p.adapters);
    if (p.plan.base) {
        const int tiles = std::min(p.plan.tiles, p.tile_least > 1 ? p.tokens / p.tile_least + p.tokens / ADP_TILE : p.plan.tiles);
        if (tiles > 0) {
            launch(adapter_low_kernel<E, NP>, dim3(ADP_CTAS * tiles, p.nparts), ADT_LOW_THREADS, adt_low_smem(p.rank), s, p);
            // as many CTAs as run at once, or a unit each
            long long units = 0;
            for (int i = 0; i < p.nparts; ++i) units += (long long)tiles * (ADP_TILE / p.out_tokens) * ((p.part[i].N + 127) / 128);
            const size_t smem = adt_out_smem(p.rank, NP);
            const int most = sm_count() * (smem <= ADT_HALF_SM ? 2 : 1);
            launch(adapter_out_kernel<E, O>, dim3((unsigned)std::min<long long>(units, most)), ADT_THREADS, smem, s, p);
            launched += 2;
        }
        groups = p.tile_least > 1 ? std::min(groups, (p.adapters + (p.copy ? 1 : 0)) * ((p.tile_least - 1 + ADP_TOK - 1) / ADP_TOK)) : 0;
    }
    if (groups > 0) {
        const bool many = (long long)ADP_CTAS * groups * p.nparts > 3 * sm_count();
        auto kern = many ? adapter_few_kernel<E, O, true, false> : adapter_few_kernel<E, O, false, false>;
        if constexpr (adapter_finishes<E, O>) {
            if (p.finish) kern = adapter_few_kernel<E, O, false, true>;
        }
        launch(kern, dim3(ADP_CTAS * groups, p.nparts), ADP_THREADS, adapter_few_smem(p.rank, NP), s, p);
        ++launched;
    }
    return launched;
}

void adapters_prepare(int type, int out_type) {
    with_types(type, out_type, [](auto e, auto o) { ready<decltype(e), decltype(o)>(); });
}

int adapters_apply(cudaStream_t s, const AdapterParams& p, int type, int out_type) {
    int launched = 0;
    with_types(type, out_type, [&](auto e, auto o) { launched = apply<decltype(e), decltype(o)>(s, p); });
    return launched;
}

template <typename E, int TH, int NV, bool VEC>
static void logits_launch(cudaStream_t s, const LogitsParams& p, int rows) {
    constexpr size_t most = (size_t)std::min(LOGITS_LIST_TOKENS, TH * NV * 4) * sizeof(uint2);
    prepare<logits_kernel<E, TH, NV, VEC>>(most, true);
    launch(logits_kernel<E, TH, NV, VEC>, dim3(rows << p.ctas_log), TH, (size_t)p.list_tokens * sizeof(uint2), s, p, 1 << p.ctas_log);
}

void logits_rows(cudaStream_t s, LogitsParams p, int rows, int type) {
    const int size = type == B200RWKV_TYPE_F32 ? 4 : 2;
    // fours that lie on boundaries in both buffers: rows start alike, modulo four (rows that are picked: on boundaries)
    const bool whole = p.in_stride % 4 == 0 && p.out_stride % 4 == 0;
    p.vec = (uintptr_t)p.in % (4 * size) == 0 && (uintptr_t)p.out % 16 == 0 && (whole || (!p.in_row && p.in_stride % 4 == p.out_stride % 4));
    // places of a row's tokens: up to three more in front of rows that start off a boundary
    int stripes = (p.V + (whole ? 0 : 3) + LOGITS_STRIPE - 1) / LOGITS_STRIPE;
    auto tokens_of = [&](int lg) { return ((stripes - 1) >> lg) * LOGITS_STRIPE + LOGITS_STRIPE; };
    constexpr int MOST = 512 * 64;               // places that a CTA of the widest form has
    static_assert(LOGITS_MAX_VOCAB == MOST * LOGITS_MOST_CTAS && LOGITS_MAX_VOCAB % LOGITS_STRIPE == 0, "the widest rows fit");
    if (tokens_of(4) > MOST) {                   // not with those in front: one token at a time
        p.vec = 0;
        stripes = (p.V + LOGITS_STRIPE - 1) / LOGITS_STRIPE;
    }
    // up to 16 tokens a thread and CTAs of 512 while all rows find room at once; 32 tokens a thread beyond, sixteen CTAs and 64 tokens for the widest rows
    const int sms = sm_count();
    int threads = 512, nv = 4;
    p.ctas_log = rows * 16 <= sms ? 4 : 3;
    if (rows * 8 > sms && tokens_of(3) <= 256 * 32) threads = 256, nv = tokens_of(3) <= 256 * 16 ? 4 : 8;
    else if (tokens_of(p.ctas_log) > 512 * 16) {
        nv = 8;
        if (tokens_of(3) > 512 * 32) p.ctas_log = 4;
        if (tokens_of(4) > 512 * 32) nv = 16;
    }
    p.list_tokens = p.hist_off || p.bias_off ? std::min(tokens_of(p.ctas_log), LOGITS_LIST_TOKENS) : 0;
    auto typed = [&](auto e) {
        using E = decltype(e);
        auto form = [&](auto th, auto n) {
            constexpr int TH = decltype(th)::value, NV = decltype(n)::value;
            p.vec ? logits_launch<E, TH, NV, true>(s, p, rows) : logits_launch<E, TH, NV, false>(s, p, rows);
        };
        using std::integral_constant;
        if (threads == 256 && nv == 4) form(integral_constant<int, 256>{}, integral_constant<int, 4>{});
        else if (threads == 256) form(integral_constant<int, 256>{}, integral_constant<int, 8>{});
        else if (nv == 4) form(integral_constant<int, 512>{}, integral_constant<int, 4>{});
        else if (nv == 8) form(integral_constant<int, 512>{}, integral_constant<int, 8>{});
        else form(integral_constant<int, 512>{}, integral_constant<int, 16>{});
    };
    if (type == B200RWKV_TYPE_F32) typed(float{});
    else if (type == B200RWKV_TYPE_F16) typed(__half{});
    else typed(__nv_bfloat16{});
}

unsigned adapters_lost_waits() {
    unsigned n = 0;
    CK(cudaMemcpyFromSymbol(&n, lost_waits, sizeof(n)));
    return n;
}

}  // namespace b200

using namespace b200;

extern "C" {

int64_t b200rwkv_op_adapters_workspace(int32_t tokens, int32_t adapters, int32_t num_parts, int32_t rank) {
    if (tokens < 0 || tokens > (1 << 20) || adapters < 1 || adapters > B200RWKV_MAX_ADAPTERS || num_parts < 1 || num_parts > B200RWKV_MAX_PARTS || rank < 1 || rank > B200RWKV_MAX_RANK) {
        last_error_text() = "op_adapters_workspace: bad argument";
        return B200RWKV_ERR_INVALID;
    }
    return (int64_t)adapters_workspace(tokens, adapters, num_parts, rank);
}

int32_t b200rwkv_op_adapters(int32_t device, void* stream, const b200rwkv_adapters* q, const b200rwkv_adapter_part* parts) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    static_assert(B200RWKV_MAX_PARTS == ADP_MAX_PARTS && B200RWKV_MAX_RANK == ADP_MAX_RANK && B200RWKV_MAX_ADAPTERS == ADP_MAX_ADAPTERS &&
                      B200RWKV_ADAPTERS_WITHOUT_WORKSPACE == ADP_INLINE, "limits");
    REQUIRE(q && q->struct_bytes == sizeof(*q), B200RWKV_ERR_INVALID, "op_adapters: struct_bytes must be sizeof(b200rwkv_adapters)");
    REQUIRE(q->type == B200RWKV_TYPE_F16 || q->type == B200RWKV_TYPE_BF16, B200RWKV_ERR_UNSUPPORTED, "op_adapters: x, a and b are f16 or bf16");
    REQUIRE(q->out_type == q->type || q->out_type == B200RWKV_TYPE_F32, B200RWKV_ERR_UNSUPPORTED, "op_adapters: out is f32 or of the type of x");
    REQUIRE(q->tokens >= 0 && q->tokens <= (1 << 20), B200RWKV_ERR_INVALID, "op_adapters: tokens must be in [0, 2^20]");
    REQUIRE(q->adapters >= 1 && q->adapters <= B200RWKV_MAX_ADAPTERS, B200RWKV_ERR_INVALID, "op_adapters: adapters must be in [1, 1024]");
    REQUIRE(q->num_parts >= 1 && q->num_parts <= B200RWKV_MAX_PARTS && parts, B200RWKV_ERR_INVALID, "op_adapters: num_parts must be in [1, 8]");
    REQUIRE(q->tokens == 0 || (q->index && q->scale), B200RWKV_ERR_INVALID, "op_adapters: null index or scale");
    AdapterParams p;
    memset(&p, 0, sizeof(p));
    p.tokens = q->tokens;
    p.adapters = q->adapters;
    p.index = q->index;
    p.scale = q->scale;
    const int osize = q->out_type == B200RWKV_TYPE_F32 ? 4 : 2;
    for (int i = 0; i < q->num_parts; ++i) {
        const b200rwkv_adapter_part& s = parts[i];
        AdapterPart& d = p.part[i];
        REQUIRE(s.in_features >= 8 && s.in_features % 8 == 0 && s.in_features <= (1 << 24), B200RWKV_ERR_UNSUPPORTED, "op_adapters: in_features must be a multiple of 8");
        REQUIRE(s.out_features >= 1 && s.out_features <= (1 << 24), B200RWKV_ERR_INVALID, "op_adapters: out_features must be positive");
        REQUIRE(s.rank >= 8 && s.rank % 8 == 0 && s.rank <= B200RWKV_MAX_RANK, B200RWKV_ERR_UNSUPPORTED, "op_adapters: rank must be a multiple of 8, at most 256");
        if (q->tokens == 0) continue;
        REQUIRE(s.x && s.a && s.b && s.out, B200RWKV_ERR_INVALID, "op_adapters: null x, a, b or out");
        REQUIRE(s.x_stride >= s.in_features && s.out_stride >= s.out_features && (!s.base || s.base_stride >= s.out_features), B200RWKV_ERR_INVALID,
                "op_adapters: rows overlap (a stride is smaller than a row)");
        REQUIRE(s.x_stride % 8 == 0 && ((uintptr_t)s.x | (uintptr_t)s.a | (uintptr_t)s.b) % 16 == 0, B200RWKV_ERR_INVALID,
                "op_adapters: rows of x, a and b must start on 16-byte boundaries");
        REQUIRE(((uintptr_t)s.out | (uintptr_t)s.base) % osize == 0, B200RWKV_ERR_INVALID, "op_adapters: misaligned base or out");
        d.x = s.x; d.x_stride = s.x_stride;
        d.a = s.a; d.b = s.b;
        d.base = s.base; d.base_stride = s.base_stride;
        d.out = s.out; d.out_stride = s.out_stride;
        d.K = s.in_features; d.N = s.out_features; d.R = s.rank;
        d.vec = ((uintptr_t)s.out | (uintptr_t)s.base) % (4 * osize) == 0 && s.out_stride % 4 == 0 && (!s.base || s.base_stride % 4 == 0);
        p.rank = std::max(p.rank, s.rank);
        REQUIRE(s.base != s.out || s.base_stride == s.out_stride || q->tokens == 1, B200RWKV_ERR_INVALID, "op_adapters: base is out, but with another stride");
        if (s.base != s.out) p.copy = 1;
    }
    if (q->tokens == 0) return B200RWKV_OK;
    const size_t need = adapters_workspace(q->tokens, q->adapters, q->num_parts, p.rank);
    p.nparts = q->num_parts;
    REQUIRE(need == 0 || (q->workspace && (uintptr_t)q->workspace % 16 == 0 && q->workspace_bytes >= need), B200RWKV_ERR_INVALID,
            "op_adapters: workspace is missing, misaligned or smaller than b200rwkv_op_adapters_workspace");
    // the projections of a call run side by side, and the tokens of each
    for (int i = 0; i < p.nparts; ++i) {
        const AdapterPart& s = p.part[i];
        const RowSpan out(s.out, p.tokens, s.out_stride, s.N, osize);
        for (int j = 0; j < p.nparts; ++j) {
            const AdapterPart& t = p.part[j];
            REQUIRE(!overlap(out, RowSpan(t.x, p.tokens, t.x_stride, t.K, 2)), B200RWKV_ERR_INVALID, i == j ? "op_adapters: the out of a part overlaps its own x" :
                    "op_adapters: the out of a part overlaps the x of another");
            REQUIRE(j == i || (!overlap(out, RowSpan(t.out, p.tokens, t.out_stride, t.N, osize)) && !(t.base && overlap(out, RowSpan(t.base, p.tokens, t.base_stride, t.N, osize)))),
                    B200RWKV_ERR_INVALID, "op_adapters: the out of a part overlaps the base or out of another");
        }
        REQUIRE(!s.base || s.base == s.out || !overlap(out, RowSpan(s.base, p.tokens, s.base_stride, s.N, osize)), B200RWKV_ERR_INVALID,
                "op_adapters: the out of a part overlaps its own base without being it");
    }
    OnDevice on(device);
    adapters_shape(p, q->workspace, q->type, q->out_type);
    if (p.plan.base) adapters_plan((cudaStream_t)stream, p);
    adapters_apply((cudaStream_t)stream, p, q->type, q->out_type);
    API_END
}

int32_t b200rwkv_op_logits(int32_t device, void* stream, const b200rwkv_logits* q) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    REQUIRE(q && q->struct_bytes == sizeof(*q), B200RWKV_ERR_INVALID, "op_logits: struct_bytes must be sizeof(b200rwkv_logits)");
    REQUIRE(q->type >= B200RWKV_TYPE_F32 && q->type <= B200RWKV_TYPE_BF16, B200RWKV_ERR_UNSUPPORTED, "op_logits: logits are f32, f16 or bf16");
    REQUIRE(q->kind >= B200RWKV_LOGITS && q->kind <= B200RWKV_LOG_PROBS, B200RWKV_ERR_INVALID, "op_logits: kind must be logits, probabilities or log-probabilities");
    REQUIRE(q->rows >= 0 && q->rows <= (1 << 24) && q->vocab >= 1, B200RWKV_ERR_INVALID, "op_logits: rows or vocab out of range");
    REQUIRE(q->vocab <= LOGITS_MAX_VOCAB, B200RWKV_ERR_UNSUPPORTED, "op_logits: vocabularies above 524288 are not supported");
    if (q->rows == 0) return B200RWKV_OK;
    const int size = q->type == B200RWKV_TYPE_F32 ? 4 : 2;
    REQUIRE(q->logits && q->out, B200RWKV_ERR_INVALID, "op_logits: null logits or out");
    REQUIRE(q->logits_stride >= q->vocab && q->out_stride >= q->vocab, B200RWKV_ERR_INVALID, "op_logits: rows overlap (a stride is smaller than the vocabulary)");
    REQUIRE((uintptr_t)q->logits % size == 0 && (uintptr_t)q->out % 4 == 0, B200RWKV_ERR_INVALID, "op_logits: misaligned logits or out");
    REQUIRE((const void*)q->out != q->logits || (q->type == B200RWKV_TYPE_F32 && (q->rows == 1 || q->logits_stride == q->out_stride)), B200RWKV_ERR_INVALID,
            "op_logits: out is logits, but their rows do not lie alike");
    REQUIRE((const void*)q->out == q->logits || !overlap(RowSpan(q->out, q->rows, q->out_stride, q->vocab, 4), RowSpan(q->logits, q->rows, q->logits_stride, q->vocab, size)),
            B200RWKV_ERR_INVALID, "op_logits: out overlaps logits without being it");
    REQUIRE(!q->history_offset || q->history, B200RWKV_ERR_INVALID, "op_logits: history offsets without tokens");
    REQUIRE(!q->bias_offset || (q->bias_token && q->bias_value), B200RWKV_ERR_INVALID, "op_logits: bias offsets without tokens or values");
    REQUIRE(!q->allow || q->allow_rows >= (q->allow_row ? 0 : q->rows), B200RWKV_ERR_INVALID, "op_logits: fewer masks than rows");
    LogitsParams p;
    memset(&p, 0, sizeof(p));
    p.in = q->logits; p.in_stride = q->logits_stride;
    p.out = q->out; p.out_stride = q->out_stride;
    p.V = q->vocab; p.kind = q->kind;
    p.controls = q->controls;
    p.hist_off = q->history_offset; p.hist = q->history; p.hist_from = q->history_from;
    p.allow = q->allow; p.words = (q->vocab + 31) / 32; p.allow_rows = q->allow_rows; p.allow_row = q->allow_row;
    p.bias_off = q->bias_offset; p.bias_tok = q->bias_token; p.bias_val = q->bias_value;
    OnDevice on(device);
    logits_rows((cudaStream_t)stream, p, q->rows, q->type);
    API_END
}

}  // extern "C"

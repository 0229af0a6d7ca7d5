// Operators on device memory from the residual rows of a step to its tokens: norms and rows in 8-bit floating point (e4m3.cuh), their products (e4m3_linear.cuh),
// tokens from rows of logits (sample_tokens.cuh); their C entries, and the launches the engine makes of the last.
#include "op_host.cuh"
#include "token_ops.cuh"
#include "e4m3.cuh"
#include "e4m3_linear.cuh"
#include "sample_tokens.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {

static int size_of(int type) { return type == B200RWKV_TYPE_E4M3 ? 1 : (type == B200RWKV_TYPE_F32 ? 4 : 2); }
static bool is_float(int type) { return type >= B200RWKV_TYPE_F32 && type <= B200RWKV_TYPE_BF16; }
// f(a value of the type)
template <typename F>
static void of_type(int type, F&& f) {
    if (type == B200RWKV_TYPE_F32) f(float{});
    else if (type == B200RWKV_TYPE_F16) f(__half{});
    else f(__nv_bfloat16{});
}
static bool on(const void* p, long long stride, int size, int boundary) { return (uintptr_t)p % boundary == 0 && (stride * size) % boundary == 0; }

// ---- norms ----
// EIGHTS: all rows on 16-byte boundaries, of whole eights
template <bool EIGHTS, typename E, typename R>
static void norm_form(cudaStream_t s, const NormParams& p, int rows) {
    // threads of so many times eight values (of which a warp has two groups of 128 columns where rows start anywhere)
    const int eights = EIGHTS ? p.width / 8 : (p.width + 255) / 256 * 32;
    auto threads = [&](int nv) { return ((eights + nv - 1) / nv + 31) / 32 * 32; };
    // more rows than CTAs that stay (2048 rows of 4096 bf16 12.3 us; a CTA a row 15.7, with 256 threads or 512)
    if (threads(2) <= NORM_MANY_THREADS) {
        const int ctas = sm_count() * (norm_many_per_sm<E, R, EIGHTS>() * NORM_MANY_THREADS / threads(2));
        if (rows > ctas) return launch(rms_norm_kernel<E, R, 2, EIGHTS, true>, dim3(ctas), threads(2), 0, s, p);
    }
    // few rows: a thread for every eight columns; many: sixteen, so that an SM has several rows in flight (1024 rows of 8192 16.6 us and 19.8); wider ones what the largest CTA needs
    int nv = 1;
    if (eights > 1024 || (rows > 2 * sm_count() && eights > 256)) nv = eights <= 1024 ? 2 : (eights <= 2048 ? 4 : 8);
    auto form = [&](auto n) { launch(rms_norm_kernel<E, R, decltype(n)::value, EIGHTS, false>, dim3(rows), threads(nv), 0, s, p); };
    if (nv == 1) form(std::integral_constant<int, 1>{});
    else if (nv == 2) form(std::integral_constant<int, 2>{});
    else if (nv == 4) form(std::integral_constant<int, 4>{});
    else form(std::integral_constant<int, 8>{});
}

// ---- products ----
static PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        CK(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q));
        REQUIRE(f && q == cudaDriverEntryPointSuccess, B200RWKV_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
        return (PFN_cuTensorMapEncodeTiled_v12000)f;
    }();
    return enc;
}
// rows of bytes, boxes of 128 bytes of `box_rows` rows in the 128-byte swizzle
static void rows_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t width, uint64_t stride, uint32_t box_rows) {
    const cuuint64_t dim[2] = {width, rows}, step[1] = {stride};
    const cuuint32_t box[2] = {E4L_KB, box_rows}, es[2] = {1, 1};
    const CUresult r = map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dim, step, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    REQUIRE(r == CUDA_SUCCESS, B200RWKV_ERR_CUDA, "cuTensorMapEncodeTiled failed");
}

struct LinearCall {
    const b200rwkv_linear_e4m3* q;
    cudaStream_t s;
    E4LinearParams p;
    void maps(int x_rows, int w_rows) {
        rows_map(&p.tx, q->x, q->tokens, q->in_features, q->x_stride, x_rows);
        rows_map(&p.tw, q->w, q->out_features, q->in_features, q->in_features, w_rows);
    }
    // CTAs of a cluster, among which e4_few_kernel deals the blocks of inputs: as many as run at once, with four blocks each at least
    template <int TT>
    int splits() const {
        const long long tiles = (long long)((q->out_features + 127) / 128) * ((q->tokens + TT - 1) / TT);
        int split = 1;
        while (split < 8 && tiles * split * 2 <= E4Few<TT>::PER_SM * sm_count() && p.kblocks >= split * 8) split *= 2;
        return split;
    }
    template <int TT>
    void few() {
        using C = E4Few<TT>;
        p.split = splits<TT>();
        maps(TT, 128);
        of_type(q->out_type, [&](auto o) {
            prepare<e4_few_kernel<TT, decltype(o)>>(C::SMEM);
            launch(e4_few_kernel<TT, decltype(o)>, dim3((q->out_features + 127) / 128 * p.split, (q->tokens + TT - 1) / TT), C::THREADS, C::SMEM, s, p, p.split);
        });
    }
    long long pairs() const { return (long long)((q->tokens + 255) / 256) * ((q->out_features + E4Pair::BN - 1) / E4Pair::BN); }
    void pair() {
        using C = E4Pair;
        maps(128, C::BN / 2);
        of_type(q->out_type, [&](auto o) {
            prepare<e4_pair_kernel<decltype(o)>>(C::SMEM);
            launch(e4_pair_kernel<decltype(o)>, dim3((unsigned)(2 * std::min<long long>(pairs(), sm_count() / 2))), C::THREADS, C::SMEM, s, p);
        });
    }
    void run() {
        if (q->tokens <= 16) return few<16>();
        if (q->tokens <= 32) return few<32>();
        if (q->tokens <= 64) return few<64>();
        // Beyond, the form that is through earlier, in rounds of all SMs: of a pair's tile a block of inputs takes 0.45 us, its ends 2.7, and a launch 4.6; of 128 tokens and outputs 0.47 and, with
        // CTAs that come and go, 7.  Both, us: 333 tokens 8960 -> 2560 44 and 23, 2560 -> 8960 18 and 32; 512 tokens 4096 -> 4096 24 and 22; 1024 tokens 24 and 43; 200 tokens
        // 4096 -> 14336 25 and 41; 128 tokens 25 and 23, 192 -> 75776 21 and 39
        const int split = splits<128>(), sms = sm_count();
        const long long ctas = (long long)((q->out_features + 127) / 128) * ((q->tokens + 127) / 128) * split;
        const long long in_few = (ctas + sms - 1) / sms * ((p.kblocks + split - 1) / split * 47 + 700), in_pairs = (pairs() + sms / 2 - 1) / (sms / 2) * (p.kblocks * 45 + 270) + 460;
        if (in_pairs < in_few) pair();
        else few<128>();
    }
};

// ---- tokens ----
void draw_rows(cudaStream_t s, DrawParams p, int rows) {
    // a CTA for every SM that there is for a row, of a thousand tokens at least
    const int size = size_of(p.type), sms = sm_count();
    int log = 0;
    while (log < 4 && (long long)rows << (log + 1) <= sms && p.V >> (log + 1) >= 1024) ++log;
    if (p.V > DRAW_ALONE_SLICE) log = max(log, 1);
    while (log > 0 && log < 4 && ((p.V + (1 << log) - 1) >> log) + 3 > DRAW_CLUSTER_SLICE) ++log;
    p.ctas_log = log;
    p.slice = (((p.V + (1 << log) - 1) >> log) + 3) & ~3;
    const bool vec = on(p.in, p.in_stride, size, 4 * size);
    auto form = [&](auto e, auto resident, auto aligned, auto per_sm) {
        constexpr bool RESIDENT = decltype(resident)::value;
        constexpr auto KERN = draw_kernel<decltype(e), DRAW_THREADS, RESIDENT, decltype(aligned)::value, decltype(per_sm)::value>;
        prepare<KERN>(draw_smem<DRAW_THREADS, RESIDENT>(RESIDENT ? DRAW_SHARED_SLICE : DRAW_MAX_VOCAB), true);
        launch(KERN, dim3(rows << log), DRAW_THREADS, draw_smem<DRAW_THREADS, RESIDENT>(p.slice), s, p, 1 << log);
    };
    using std::integral_constant;
    auto shape = [&](auto e, auto aligned) {
        // (registers for two CTAs an SM spill, which many rows take for the second: 512 rows of 65536, top-p 0.9, 235 us and 273 with one; 96 rows of 100003 164 and 131)
        if (((long long)rows << log) > sms) form(e, std::false_type{}, aligned, integral_constant<int, 2>{});
        else if (p.slice > DRAW_SHARED_SLICE) form(e, std::false_type{}, aligned, integral_constant<int, 1>{});
        else form(e, std::true_type{}, aligned, integral_constant<int, 1>{});
    };
    of_type(p.type, [&](auto e) { vec ? shape(e, std::true_type{}) : shape(e, std::false_type{}); });
}

}  // namespace b200

using namespace b200;

extern "C" {

int32_t b200rwkv_op_norm(int32_t device, void* stream, const b200rwkv_norm* q) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    REQUIRE(q && q->struct_bytes == sizeof(*q), B200RWKV_ERR_INVALID, "op_norm: struct_bytes must be sizeof(b200rwkv_norm)");
    REQUIRE(is_float(q->type), B200RWKV_ERR_UNSUPPORTED, "op_norm: x is f32, f16 or bf16");
    REQUIRE(q->residual_type == q->type || q->residual_type == B200RWKV_TYPE_F32, B200RWKV_ERR_UNSUPPORTED, "op_norm: the residual is f32 or of the type of x");
    REQUIRE(is_float(q->weight_type), B200RWKV_ERR_UNSUPPORTED, "op_norm: the weight is f32, f16 or bf16");
    REQUIRE(q->out_type == B200RWKV_TYPE_E4M3 || q->out_type == q->type, B200RWKV_ERR_UNSUPPORTED, "op_norm: out is e4m3 or of the type of x");
    REQUIRE(q->rows >= 0 && q->rows <= (1 << 24), B200RWKV_ERR_INVALID, "op_norm: rows must be in [0, 2^24]");
    REQUIRE(q->width >= 1, B200RWKV_ERR_INVALID, "op_norm: width must be positive");
    REQUIRE(q->width <= NORM_MAX_WIDTH, B200RWKV_ERR_UNSUPPORTED, "op_norm: widths above 32768 are not supported");
    REQUIRE(q->eps >= 0.f, B200RWKV_ERR_INVALID, "op_norm: eps must not be negative");
    if (q->rows == 0) return B200RWKV_OK;
    const bool eight = q->out_type == B200RWKV_TYPE_E4M3;
    const int size = size_of(q->type), rsize = size_of(q->residual_type), wsize = size_of(q->weight_type), osize = size_of(q->out_type);
    REQUIRE(q->x && q->out && (!eight || q->scale), B200RWKV_ERR_INVALID, "op_norm: null x, out or scale");
    REQUIRE(!q->residual == !q->residual_out, B200RWKV_ERR_INVALID, "op_norm: residual and residual_out come together");
    REQUIRE(q->x_stride >= q->width && q->out_stride >= q->width && (!q->residual || (q->residual_stride >= q->width && q->residual_out_stride >= q->width)),
            B200RWKV_ERR_INVALID, "op_norm: rows overlap (a stride is smaller than the width)");
    REQUIRE((uintptr_t)q->x % size == 0 && ((uintptr_t)q->residual | (uintptr_t)q->residual_out) % rsize == 0 && (uintptr_t)q->weight % wsize == 0 &&
                (uintptr_t)q->out % osize == 0 && (uintptr_t)q->scale % 4 == 0, B200RWKV_ERR_INVALID, "op_norm: misaligned buffer");
    const int groups = (q->width + E4_GROUP - 1) / E4_GROUP;
    const RowSpan x(q->x, q->rows, q->x_stride, q->width, size), out(q->out, q->rows, q->out_stride, q->width, osize), weight(q->weight, 1, q->width, q->width, wsize),
        scale(q->scale, 1, (long long)q->rows * groups, (long long)q->rows * groups, 4);
    REQUIRE(!overlap(out, x) && !(q->weight && overlap(out, weight)), B200RWKV_ERR_INVALID, "op_norm: out overlaps x or weight");
    REQUIRE(!eight || (!overlap(scale, x) && !overlap(scale, out) && !(q->weight && overlap(scale, weight))), B200RWKV_ERR_INVALID, "op_norm: scale overlaps x, out or weight");
    if (q->residual) {
        const RowSpan res(q->residual, q->rows, q->residual_stride, q->width, rsize), sum(q->residual_out, q->rows, q->residual_out_stride, q->width, rsize);
        const bool is_res = q->residual_out == q->residual && (q->residual_out_stride == q->residual_stride || q->rows == 1);
        const bool is_x = q->residual_out == q->x && q->residual_type == q->type && (q->residual_out_stride == q->x_stride || q->rows == 1);
        REQUIRE((is_res || !overlap(sum, res)) && (is_x || !overlap(sum, x)), B200RWKV_ERR_INVALID, "op_norm: residual_out overlaps residual or x without being it");
        REQUIRE(!overlap(out, res) && !overlap(out, sum) && !(q->weight && overlap(sum, weight)) && !(eight && (overlap(scale, res) || overlap(scale, sum))), B200RWKV_ERR_INVALID,
                "op_norm: outputs overlap one another, residual or weight");
    }
    NormParams p;
    memset(&p, 0, sizeof(p));
    p.x = q->x; p.x_stride = q->x_stride;
    p.residual = q->residual; p.residual_stride = q->residual_stride;
    p.residual_out = q->residual_out; p.residual_out_stride = q->residual_out_stride;
    p.weight = q->weight; p.weight_type = q->weight_type;
    p.out = q->out; p.out_stride = q->out_stride;
    p.scale = eight ? q->scale : nullptr;
    p.rows = q->rows; p.width = q->width; p.groups = groups;
    p.eps = q->eps; p.offset = q->offset;
    const bool eights = q->width % 8 == 0 && on(q->x, q->x_stride, size, 16) && (uintptr_t)q->weight % 16 == 0 && on(q->out, q->out_stride, osize, eight ? 8 : 16) &&
                        (!q->residual || (on(q->residual, q->residual_stride, rsize, 16) && on(q->residual_out, q->residual_out_stride, rsize, 16)));
    OnDevice here(device);
    of_type(q->type, [&](auto e) {
        using E = decltype(e);
        auto form = [&](auto r) {
            if (eights) norm_form<true, E, decltype(r)>((cudaStream_t)stream, p, q->rows);
            else norm_form<false, E, decltype(r)>((cudaStream_t)stream, p, q->rows);
        };
        if (q->residual_type == q->type) form(e);
        else if constexpr (!std::is_same_v<E, float>) form(0.f);
    });
    API_END
}

int32_t b200rwkv_op_e4m3(int32_t device, void* stream, const b200rwkv_e4m3* q) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    REQUIRE(q && q->struct_bytes == sizeof(*q), B200RWKV_ERR_INVALID, "op_e4m3: struct_bytes must be sizeof(b200rwkv_e4m3)");
    REQUIRE(is_float(q->type), B200RWKV_ERR_UNSUPPORTED, "op_e4m3: x is f32, f16 or bf16");
    REQUIRE(q->block_rows == 1 || q->block_rows == E4_GROUP, B200RWKV_ERR_UNSUPPORTED, "op_e4m3: a scale is for 1 or 128 rows");
    REQUIRE(q->rows >= 0 && q->rows <= (1 << 24) && q->width >= 1 && q->width <= (1 << 24), B200RWKV_ERR_INVALID, "op_e4m3: rows must be in [0, 2^24], width in [1, 2^24]");
    if (q->rows == 0) return B200RWKV_OK;
    const int size = size_of(q->type), groups = (q->width + E4_GROUP - 1) / E4_GROUP;
    const long long blocks = (q->rows + q->block_rows - 1) / q->block_rows;
    REQUIRE(q->x && q->out && q->scale, B200RWKV_ERR_INVALID, "op_e4m3: null x, out or scale");
    REQUIRE(q->x_stride >= q->width && q->out_stride >= q->width, B200RWKV_ERR_INVALID, "op_e4m3: rows overlap (a stride is smaller than the width)");
    REQUIRE((uintptr_t)q->x % size == 0 && (uintptr_t)q->scale % 4 == 0, B200RWKV_ERR_INVALID, "op_e4m3: misaligned x or scale");
    const long long units = blocks * groups;
    const RowSpan x(q->x, q->rows, q->x_stride, q->width, size), out(q->out, q->rows, q->out_stride, q->width, 1), scale(q->scale, 1, units, units, 4);
    REQUIRE(!overlap(out, x) && !overlap(scale, x) && !overlap(scale, out), B200RWKV_ERR_INVALID, "op_e4m3: x, out and scale overlap");
    const bool eights = q->width % 8 == 0 && on(q->x, q->x_stride, size, 16) && on(q->out, q->out_stride, 1, 8);
    const long long threads = eights ? units * E4_PER_ROW : q->rows * (long long)((groups + 1) / 2) * 32, ctas = q->block_rows == 1 ? (threads + E4_THREADS - 1) / E4_THREADS : units;
    REQUIRE(ctas <= 0x7FFFFFFFll, B200RWKV_ERR_UNSUPPORTED, "op_e4m3: too many values for one call");
    const E4Params p{q->x, q->x_stride, (uint8_t*)q->out, q->out_stride, q->scale, q->rows, q->width, groups, on(q->out, q->out_stride, 1, 16)};
    OnDevice here(device);
    of_type(q->type, [&](auto e) {
        using E = decltype(e);
        auto form = [&](auto whole) {
            constexpr bool EIGHTS = decltype(whole)::value;
            launch(q->block_rows == 1 ? e4_rows_kernel<EIGHTS, E> : e4_blocks_kernel<EIGHTS, E>, dim3((unsigned)ctas), E4_THREADS, 0, (cudaStream_t)stream, p);
        };
        if (eights) form(std::true_type{});
        else form(std::false_type{});
    });
    API_END
}

int32_t b200rwkv_op_linear_e4m3(int32_t device, void* stream, const b200rwkv_linear_e4m3* q) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    REQUIRE(q && q->struct_bytes == sizeof(*q), B200RWKV_ERR_INVALID, "op_linear_e4m3: struct_bytes must be sizeof(b200rwkv_linear_e4m3)");
    REQUIRE(is_float(q->out_type), B200RWKV_ERR_UNSUPPORTED, "op_linear_e4m3: out is f32, f16 or bf16");
    REQUIRE(q->tokens >= 0 && q->tokens <= (1 << 20), B200RWKV_ERR_INVALID, "op_linear_e4m3: tokens must be in [0, 2^20]");
    REQUIRE(q->in_features >= 16 && q->in_features % 16 == 0 && q->in_features <= (1 << 24), B200RWKV_ERR_UNSUPPORTED, "op_linear_e4m3: in_features must be a multiple of 16");
    REQUIRE(q->out_features >= 1 && q->out_features <= (1 << 24), B200RWKV_ERR_INVALID, "op_linear_e4m3: out_features must be in [1, 2^24]");
    if (q->tokens == 0) return B200RWKV_OK;
    const int osize = size_of(q->out_type), kblocks = (q->in_features + E4L_KB - 1) / E4L_KB, nblocks = (q->out_features + 127) / 128;
    REQUIRE(q->x && q->x_scale && q->w && q->w_scale && q->out, B200RWKV_ERR_INVALID, "op_linear_e4m3: null x, x_scale, w, w_scale or out");
    REQUIRE(q->x_stride >= q->in_features && q->out_stride >= q->out_features && (!q->base || q->base_stride >= q->out_features), B200RWKV_ERR_INVALID,
            "op_linear_e4m3: rows overlap (a stride is smaller than a row)");
    REQUIRE(on(q->x, q->x_stride, 1, 16) && (uintptr_t)q->w % 16 == 0, B200RWKV_ERR_INVALID, "op_linear_e4m3: rows of x and w must start on 16-byte boundaries");
    REQUIRE(((uintptr_t)q->x_scale | (uintptr_t)q->w_scale) % 4 == 0 && ((uintptr_t)q->out | (uintptr_t)q->base) % osize == 0, B200RWKV_ERR_INVALID,
            "op_linear_e4m3: misaligned scales, base or out");
    REQUIRE(q->base != q->out || q->base_stride == q->out_stride || q->tokens == 1, B200RWKV_ERR_INVALID, "op_linear_e4m3: base is out, but with another stride");
    const RowSpan out(q->out, q->tokens, q->out_stride, q->out_features, osize), x(q->x, q->tokens, q->x_stride, q->in_features, 1),
        w(q->w, q->out_features, q->in_features, q->in_features, 1), xs(q->x_scale, q->tokens, kblocks, kblocks, 4), ws(q->w_scale, nblocks, kblocks, kblocks, 4);
    REQUIRE(!overlap(out, x) && !overlap(out, w) && !overlap(out, xs) && !overlap(out, ws), B200RWKV_ERR_INVALID, "op_linear_e4m3: out overlaps x, w or their scales");
    REQUIRE(!q->base || q->base == q->out || !overlap(out, RowSpan(q->base, q->tokens, q->base_stride, q->out_features, osize)), B200RWKV_ERR_INVALID,
            "op_linear_e4m3: out overlaps base without being it");
    LinearCall c;
    memset(&c.p, 0, sizeof(c.p));
    c.q = q;
    c.s = (cudaStream_t)stream;
    c.p.xs = q->x_scale; c.p.ws = q->w_scale;
    c.p.base = q->base; c.p.base_stride = q->base_stride;
    c.p.out = q->out; c.p.out_stride = q->out_stride;
    c.p.tokens = q->tokens; c.p.N = q->out_features; c.p.kblocks = kblocks;
    c.p.vec = on(q->out, q->out_stride, osize, 16) && (!q->base || on(q->base, q->base_stride, osize, 16));
    OnDevice here(device);
    c.run();
    API_END
}

int32_t b200rwkv_op_sample(int32_t device, void* stream, const b200rwkv_sample* q) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    REQUIRE(q && q->struct_bytes == sizeof(*q), B200RWKV_ERR_INVALID, "op_sample: struct_bytes must be sizeof(b200rwkv_sample)");
    REQUIRE(is_float(q->type), B200RWKV_ERR_UNSUPPORTED, "op_sample: logits are f32, f16 or bf16");
    REQUIRE(q->rows >= 0 && q->rows <= (1 << 24) && q->vocab >= 1, B200RWKV_ERR_INVALID, "op_sample: rows or vocab out of range");
    REQUIRE(q->vocab <= DRAW_MAX_VOCAB, B200RWKV_ERR_UNSUPPORTED, "op_sample: vocabularies above 524288 are not supported");
    if (q->rows == 0) return B200RWKV_OK;
    const int size = size_of(q->type);
    REQUIRE(q->logits && q->uniform && q->tokens, B200RWKV_ERR_INVALID, "op_sample: null logits, uniform or tokens");
    REQUIRE(q->logits_stride >= q->vocab, B200RWKV_ERR_INVALID, "op_sample: rows overlap (a stride is smaller than the vocabulary)");
    REQUIRE((uintptr_t)q->logits % size == 0 && ((uintptr_t)q->uniform | (uintptr_t)q->temperature | (uintptr_t)q->top_k | (uintptr_t)q->top_p | (uintptr_t)q->min_p |
             (uintptr_t)q->tokens | (uintptr_t)q->probs) % 4 == 0, B200RWKV_ERR_INVALID, "op_sample: misaligned buffer");
    const RowSpan logits(q->logits, q->rows, q->logits_stride, q->vocab, size), tokens(q->tokens, 1, q->rows, q->rows, 4), probs(q->probs, 1, q->rows, q->rows, 4);
    const void* const in[] = {q->uniform, q->temperature, q->top_k, q->top_p, q->min_p};
    for (const void* x : in)
        REQUIRE(!x || (!overlap(tokens, RowSpan(x, 1, q->rows, q->rows, 4)) && !(q->probs && overlap(probs, RowSpan(x, 1, q->rows, q->rows, 4)))), B200RWKV_ERR_INVALID,
                "op_sample: tokens or probs overlap what the call reads");
    REQUIRE(!overlap(tokens, logits) && !(q->probs && (overlap(probs, logits) || overlap(probs, tokens))), B200RWKV_ERR_INVALID, "op_sample: tokens, probs and logits overlap");
    DrawParams p;
    memset(&p, 0, sizeof(p));
    p.in = q->logits; p.in_stride = q->logits_stride;
    p.uniform = q->uniform; p.temperature = q->temperature; p.top_k = q->top_k; p.top_p = q->top_p; p.min_p = q->min_p;
    p.tokens = q->tokens; p.probs = q->probs;
    p.V = q->vocab; p.type = q->type;
    OnDevice here(device);
    draw_rows((cudaStream_t)stream, p, q->rows);
    API_END
}

int32_t b200rwkv_op_lost_waits(int32_t device, int64_t* total) {
    API_BEGIN((b200rwkv_engine*)nullptr)
    REQUIRE(total, B200RWKV_ERR_INVALID, "op_lost_waits: null total");
    OnDevice here(device);
    unsigned n = 0;
    CK(cudaMemcpyFromSymbol(&n, lost_waits, sizeof(n)));
    *total = (int64_t)n + adapters_lost_waits();
    API_END
}

}  // extern "C"

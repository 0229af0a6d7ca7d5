// A token for each row of logits from a given random number, under a temperature, top-k, top-p and min-p.  For a row l, its largest logit m, temperature T:
//     w_t = exp((l_t - m) / T);  tokens in order: larger logit first, of equal ones the lower id
//     kept are the first k of them; of these the shortest beginning that holds top_p of their weights; of these the ones with w_t >= min_p (the first always)
//     the token is the lowest id at which the sum of kept weights, ids ascending, exceeds u times all of it
// Reference: what its samplers do behind the softmax (sampler/nucleus.rs:69-123, sampler/typical.rs:70-131), whose own orders the host classes keep.
//
// A sum that ends beside a border decides about a token, so that 32 bits would draw other tokens than the definition: weights are whole numbers of 2^-40 of the
// row's largest, from exponentials in 64 bits, and their sums are exact in any order.  Tokens below half a unit weigh nothing and are never drawn.
//
// Bound: a row is read once from memory (512 rows of 65536 f32: 20 us); then instructions (some 25 a token for its 64-bit exponential and its bin), and latency.  Nothing is sorted: a beginning of
// the order is found from its end, the token with which a sum over the order (of ones, or of weights) reaches a target.
//   * 2048 bins of tokens over the distance from the largest logit tell between which two the end lies (weights differ by a hundredth within a bin, so that counts are enough for both sums);
//   * where no more tokens than a list are that near (top-k, peaked rows), one CTA ranks them one against another and has the row's token.  A top-k of a CTA's whole row takes its bins from the
//     threads' best tokens alone;
//   * else the sum in front of the two bins is worked out exactly, and their tokens are ranked; where they are too many, 512 bins between the two, now with their weights, narrow them down
//     first (and, as with thousands of equal logits, bins over nine bits at a time of (logit, id));
//   * sums over 128 neighbouring tokens of what is kept, written on the way, lead to the token.
// Shape: as many CTAs a row as SMs there are for it, a cluster of sixteen at most; what they tell one another costs a microsecond each time.  Runs that fit stay in shared memory, others are read again
// from L2 for every step.  More rows than SMs: a CTA a row, two to an SM.  Steps that only a few tokens take part in gather those of 128 first, so that a warp's exponentials are not one lane's.
// Measured, us: a row of 65536 with top-k 50 and top-p 0.95 12, 16 rows of top-p 0.9 26; 96 rows of 100003 in bf16, top-k 1000 and top-p 0.98 (every fourth top-p alone), 130; 512
// rows of 65536: the best token 39, top-k 50 59, no limit 109, top-p 0.9 222 to 233.
// Tried: bins' sums from the front alone (half a hundredth of all weights are a tail of thousands of tokens: 410 for the 96 rows, 310 for the 512); rows in the registers or the shared memory of eight CTAs with exact weights in all bins (620 us for the last), steps unrolled four times (fetching their code took longer than
// running it), a closure that was not inlined (its variables in memory: two to three times as long).
#pragma once
#include "float_types.cuh"
#include "sm_pair.cuh"
#include "token_ops.cuh"

#include <cfloat>
#include <type_traits>

namespace b200 {

constexpr int DRAW_FINE = 2048;                  // bins of tokens alone
constexpr int DRAW_BINS = 512, DRAW_BIN_BITS = 9;
constexpr int DRAW_LIST = 512;                   // tokens that are ranked one against another
constexpr int DRAW_UNIT = 40;                    // weights are multiples of 2^-40
constexpr int DRAW_LIMB = 14;                    // bits of a weight in each of three words of a bin: sums of 2^18 of them fit 32 bits
static_assert(3 * DRAW_LIMB > DRAW_UNIT, "the largest weight fits");

typedef unsigned long long u64;
#define DRAW_INLINE __attribute__((always_inline))         // a lambda that is not inlined keeps all variables that it refers to in memory

__device__ __forceinline__ float draw_max(float a, float b) {      // NaN where one of them is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
// four neighbouring logits as they lie in memory
template <typename E> struct DrawRaw;
template <> struct DrawRaw<float> {
    using Four = float4;
    static __device__ __forceinline__ float4 widen4(float4 v) { return v; }
};
template <> struct DrawRaw<__half> {
    using Four = uint2;
    static __device__ __forceinline__ float4 widen4(uint2 u) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
};
template <> struct DrawRaw<__nv_bfloat16> {
    using Four = uint2;
    static __device__ __forceinline__ float4 widen4(uint2 u) {
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
    }
};
// larger logit, larger number (-0 and +0 are one value)
__device__ __forceinline__ unsigned draw_order(float x) {
    const unsigned b = __float_as_uint(x == 0.f ? 0.f : x);
    return b ^ (0x80000000u | (unsigned)((int)b >> 31));
}
// place in the order as one number of 51 bits: larger logit first, then lower id
constexpr int DRAW_ID_BITS = 19;
__device__ __forceinline__ u64 draw_key(unsigned order, int id) { return ((u64)order << DRAW_ID_BITS) | (unsigned)((1 << DRAW_ID_BITS) - 1 - id); }
__device__ __forceinline__ float draw_logit(u64 key) {
    const unsigned o = (unsigned)(key >> DRAW_ID_BITS);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// round(2^40 2^y), y = d `over` no less than -43 (0 where `there` does not hold): 2^y = 2^n 2^(j/64) 2^g with whole n, j and |g| <= 1/128.  2^(j/64) is a table's (times 2^40), 2^g its
// power series (|g ln 2| < 0.0055: the terms from the fifth on are below 2^-44).  Whole numbers in a double: sums of up to 2^13 are exact there
constexpr int DRAW_TABLE = 64;
__device__ __forceinline__ double draw_exp2(double d, double over, const double* table, bool there) {
    const double magic = 6755399441055744.0 / DRAW_TABLE;    // 1.5 2^52 / 64: the sum's last bits are the number of 64ths
    const double t = fma(d, over, magic), g = fma(d, over, magic - t);
    const int m = __double2loint(t);
    constexpr double L = 0.6931471805599453094;
    double s = L * L * L * L / 24;
    s = fma(s, g, L * L * L / 6); s = fma(s, g, L * L / 2); s = fma(s, g, L); s = fma(s, g, 1.0);
    const double unit = table[m & (DRAW_TABLE - 1)];
    const int hi = __double2hiint(unit) + ((m >> 6) << 20);              // (times 2^n)
    return fma(s, __hiloint2double(there ? hi : 0, __double2loint(unit)), 4503599627370496.0) - 4503599627370496.0;       // (2^52 + x: to the nearest whole number)
}
__device__ __forceinline__ u64 draw_whole(double v) { return (u64)(__double_as_longlong(v + 4503599627370496.0) - 0x4330000000000000ll); }       // of one below 2^52

// sums over a warp: in whole numbers, a few bits at a time by the unit's own additions
__device__ __forceinline__ u64 draw_warp_sum(u64 v) {      // v < 2^46
    const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x7FFFFFu), b = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 23));
    return (u64)a + ((u64)b << 23);
}
__device__ __forceinline__ u64 draw_warp_sum_wide(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 draw_warp_scan(u64 v) {     // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
__device__ __forceinline__ unsigned draw_remote(uint32_t addr, int cta) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(addr, (uint32_t)cta)) : "memory");
    return v;
}
__device__ __forceinline__ u64 draw_remote64(uint32_t addr, int cta) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_u32(addr, (uint32_t)cta)) : "memory");
    return v;
}
__device__ __forceinline__ void draw_tell(u64* slot, u64 v, int cta) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_u32(smem_u32(slot), (uint32_t)cta)), "l"(v) : "memory");
}

// a cluster's CTA in shared memory; the row behind it (fours), then sums over 128 neighbouring tokens
template <int TH>
struct DrawShared {
    static constexpr int WARPS = TH / 32;
    double table[DRAW_TABLE];                    // 2^(40 + j / 64)
    union {
        unsigned fine[DRAW_FINE];                // tokens
        unsigned bins[4][DRAW_BINS];             // tokens, and their weights in three parts
    };
    u64 packed[2][DRAW_BINS];                    // the same, four or one to a word, for the other CTAs; two, so that one may be read while the next is filled
    u64 list[DRAW_LIST];
    union {
        float queue[WARPS][128];
        struct { u64 all[DRAW_LIST], sorted[DRAW_LIST], weight[DRAW_LIST]; };
    };
    u64 warp[2][WARPS];
    float warp_f[WARPS];
    u64 slot[4][DRAW_MOST_CTAS];                 // what the CTAs tell one another
    u64 found, found_before;
    int found_bin, found_count, found_upto, found_hi, list_n;
};
__host__ __device__ constexpr int draw_segments(int slice) { return (slice + 127) / 128; }
template <int TH, bool RESIDENT>
__host__ __device__ constexpr size_t draw_smem(int slice) {
    return ((sizeof(DrawShared<TH>) + 15) & ~(size_t)15) + (RESIDENT ? (size_t)draw_segments(slice) * 512 : 0) + (size_t)draw_segments(slice) * 8;
}

template <typename E, int TH, bool RESIDENT, bool VEC, int PER_SM>
__global__ void __launch_bounds__(TH, PER_SM) draw_kernel(const __grid_constant__ DrawParams p) {
    extern __shared__ __align__(16) unsigned char draw_bytes[];
    using Shared = DrawShared<TH>;
    Shared& s = *reinterpret_cast<Shared*>(draw_bytes);
    constexpr int WARPS = Shared::WARPS;
    static_assert(TH >= DRAW_BINS && TH >= DRAW_LIST, "a thread for every bin and every entry");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = 1 << p.ctas_log, cta = blockIdx.x & (ctas - 1), row = blockIdx.x >> p.ctas_log;
    const int lo = min(cta * p.slice, p.V), cnt = min(lo + p.slice, p.V) - lo, segments = draw_segments(p.slice);
    float4* const fours = reinterpret_cast<float4*>(draw_bytes + ((sizeof(Shared) + 15) & ~(size_t)15));
    u64* const segment = reinterpret_cast<u64*>(fours + (RESIDENT ? segments * 32 : 0));
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");        // no CTA writes to another's memory before all have started
    if (tid < DRAW_TABLE) s.table[tid] = ldexp(exp2(tid / (double)DRAW_TABLE), DRAW_UNIT);
    for (int i = tid; i < DRAW_FINE; i += TH) s.fine[i] = 0u;
    if (tid == 0) s.list_n = 0;
    pdl_wait();
    pdl_launch_dependents();

    // ---- the CTA's tokens, 128 to a warp, four to a lane: f(their logits, id of the first, which 128) with all lanes, -inf behind the run ----
    using Raw = typename DrawRaw<E>::Four;
    const E* const in = reinterpret_cast<const E*>(p.in) + (long long)(p.in_row ? p.in_row[row] : row) * p.in_stride + lo;
    const int full = cnt / 128;                  // where all lanes have four
    // (without a branch, so that several can be on their way)
    auto ask = [&](int g) DRAW_INLINE {
        const E* const q = in + (g * 32 + lane) * 4;
        Raw r;
        if (VEC) {
            r = *reinterpret_cast<const Raw*>(q);
        } else {
            E* const e = reinterpret_cast<E*>(&r);
#pragma unroll
            for (int c = 0; c < 4; ++c) e[c] = q[c];
        }
        return r;
    };
    auto ragged = [&](int g) DRAW_INLINE {
        const int i = (g * 32 + lane) * 4;
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = i + c < cnt ? widened<E>(in[i + c]) : -INFINITY;
        return make_float4(x[0], x[1], x[2], x[3]);
    };
    // Short steps take four turns' tokens at a time.  Long ones run a few times a CTA only, and fetching their code would take longer than running it were they unrolled: they have
    // two turns' on their way while they work on two
    auto four_turns = [&](bool from_memory, auto&& f) DRAW_INLINE {
        constexpr int U = 4;
#pragma unroll 1
        for (int g0 = warp; g0 < segments; g0 += WARPS * U) {
            Raw r[U];
            if (from_memory) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (g0 + u * WARPS < full) r[u] = ask(g0 + u * WARPS);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int g = g0 + u * WARPS;
                if (g >= segments) break;
                float4 b;
                if (from_memory) {
                    b = g < full ? DrawRaw<E>::widen4(r[u]) : ragged(g);
                    if (RESIDENT) fours[g * 32 + lane] = b;
                } else {
                    b = fours[g * 32 + lane];
                }
                const float x[4] = {b.x, b.y, b.z, b.w};
                f(x, lo + (g * 32 + lane) * 4, g);
            }
        }
    };
    auto tokens = [&](auto&& f) DRAW_INLINE {
        constexpr int U = 2;
        Raw next[U];
        if (!RESIDENT) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (warp + u * WARPS < full) next[u] = ask(warp + u * WARPS);
        }
#pragma unroll 1
        for (int g0 = warp; g0 < segments; g0 += WARPS * U) {
            Raw now[U];
            if (!RESIDENT) {
#pragma unroll
                for (int u = 0; u < U; ++u) now[u] = next[u];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (g0 + (U + u) * WARPS < full) next[u] = ask(g0 + (U + u) * WARPS);
            }
#pragma unroll 1
            for (int u = 0; u < U; ++u) {
                const int g = g0 + u * WARPS;
                if (g >= segments) break;
                const float4 b = RESIDENT ? fours[g * 32 + lane] : (g < full ? DrawRaw<E>::widen4(u == 0 ? now[0] : now[1]) : ragged(g));
                const float x[4] = {b.x, b.y, b.z, b.w};
                f(x, lo + (g * 32 + lane) * 4, g);
            }
        }
    };
    float top = 0.f;                             // the largest logit
    // f(logit, whether there is one) with 32 lanes at a time for those of a warp's 128 that `want` tells
    auto gather = [&](const float (&x)[4], const bool (&want)[4], auto&& f) DRAW_INLINE {
        unsigned who[4];
        int n = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            who[c] = __ballot_sync(0xffffffffu, want[c]);
            n += __popc(who[c]);
        }
        if (n == 0) return;
        if (n > 64) {                            // most of them: where they are (four chains of operations side by side)
#pragma unroll
            for (int c = 0; c < 4; ++c) f(x[c], want[c]);
            return;
        }
        float* const q = s.queue[warp];
        int at = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (want[c]) q[at + __popc(who[c] & ((1u << lane) - 1))] = x[c];
            at += __popc(who[c]);
        }
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < n; i += 32) f(i + lane < n ? q[i + lane] : top, i + lane < n);
        __syncwarp();
    };

    float mine = -INFINITY;                      // (NaN where one is)
    four_turns(true, [&](const float (&x)[4], int, int) { mine = draw_max(draw_max(draw_max(mine, x[0]), draw_max(x[1], x[2])), x[3]); });
    const float u = p.uniform[row], given = p.temperature ? p.temperature[row] : 1.f, top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
    const int top_k = p.top_k ? p.top_k[row] : 0;
    // a value of each warp over the block and the cluster's CTAs, by `combine` of two: every CTA has all CTAs' values afterwards
    auto exchange = [&](int which, u64 x, auto&& combine) DRAW_INLINE {
        if (lane == 0) s.warp[0][warp] = x;
        __syncthreads();
        if (tid < ctas) {
            u64 a = s.warp[0][0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) a = combine(a, s.warp[0][w]);
            draw_tell(&s.slot[which][cta], a, tid);
        }
        cluster_sync_all();
        u64 a = s.slot[which][0];
        for (int c = 1; c < ctas; ++c) a = combine(a, s.slot[which][c]);
        return a;
    };
    const unsigned order = __reduce_max_sync(0xffffffffu, draw_order(mine)), any_nan = __any_sync(0xffffffffu, isnan(mine));
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const u64 best = exchange(0, ((u64)any_nan << 32) | order, [](u64 a, u64 b) { return ((a | b) >> 32 << 32) | max((unsigned)a, (unsigned)b); });
    top = draw_logit((u64)(unsigned)best << DRAW_ID_BITS);
    if (best >> 32 || isnan(u) || isnan(top_p) || isnan(min_p) || !(given >= 0.f && given < INFINITY) || top == -INFINITY) {
        if (cta == 0 && tid == 0) {
            p.tokens[row] = -1;
            if (p.probs) p.probs[row] = top == -INFINITY && !(best >> 32) ? 0.f : __int_as_float(0x7fc00000);
        }
        return;
    }

    // ---- the best token alone ----
    if (given == 0.f || top_k == 1) {
        unsigned id = ~0u;
        four_turns(!RESIDENT, [&](const float (&x)[4], int i, int) {
#pragma unroll
            for (int c = 3; c >= 0; --c)
                if (x[c] == top) id = min(id, (unsigned)(i + c));
        });
        const u64 a = exchange(1, __reduce_min_sync(0xffffffffu, id), [](u64 x, u64 y) { return x < y ? x : y; });
        if (cta == 0 && tid == 0) {
            p.tokens[row] = (int)a;
            if (p.probs) p.probs[row] = 1.f;
        }
        return;
    }

    // ---- weights ----
    const float temperature = fmaxf(given, 0x1p-100f);
    const double over = 1.4426950408889634074 / (double)temperature, top_d = fminf(top, FLT_MAX);
    // Tokens below `nearest` are not kept: at first, those that weigh less than half a unit (-inf is not within any reach).  Bins are over half of the distance from the largest logit, which does
    // not overflow: to the nearest of DRAW_FINE, by an addition that leaves it in the last bits (where both are infinite: the first)
    const float half_top = 0.5f * top, reach = fminf(21.f * 0.6931472f * 1.00001f * temperature, FLT_MAX), bins_over = (DRAW_FINE - 1) / reach;
    auto from_top = [&](float x) DRAW_INLINE { return fmaf(-0.5f, x, half_top); };
    // (of a token within reach, or 0: one that is not there may be infinitely far away, and nothing may be computed from that)
    auto weight_if = [&](float x, bool there) DRAW_INLINE { return draw_exp2((double)fminf(there ? x : top, FLT_MAX) - top_d, over, s.table, there); };
    auto weight = [&](float x) DRAW_INLINE { return draw_whole(weight_if(x, true)); };
    auto bin_of = [&](float x) DRAW_INLINE { return min(DRAW_FINE - 1, __float_as_int(fmaf(fmaxf(from_top(x), 0.f), bins_over, 0x1p23f)) - 0x4B000000); };
    auto nearest_of = [&](float far) DRAW_INLINE { return fmaxf(2.f * (half_top - far), -FLT_MAX); };
    // a token further away than half of this weighs less than so many units
    auto distance = [&](double units) DRAW_INLINE { return fminf(reach, (float)(DRAW_UNIT - log2(units)) * 0.6931472f * 0.5f * temperature * 1.0001f); };
    const u64 floor_weight = (u64)ceil(fmin(fmax((double)min_p, 0.0), 1.0) * (double)(1ull << DRAW_UNIT));
    float nearest = nearest_of(reach);
    float last = __int_as_float(0x7fc00000);     // and of those with this logit, the ones behind this id
    int last_id = 0;
    bool tied = false;                           // (there are such)
    auto among_kept = [&](float x, int id) DRAW_INLINE -> bool { return (x >= nearest) & !((x == last) & (id > last_id)); };
    auto which_kept = [&](const float (&x)[4], int id, bool (&want)[4]) DRAW_INLINE {
#pragma unroll
        for (int c = 0; c < 4; ++c) want[c] = x[c] >= nearest;
        if (tied) {
#pragma unroll
            for (int c = 0; c < 4; ++c) want[c] = want[c] & !((x[c] == last) & (id + c > last_id));
        }
    };

    // weights of what is kept: over the row and over 128 neighbouring tokens of what weighs at least `lower` (`apart`), or else of all over the row, beside bins of the tokens
    auto add_up = [&](double lower, bool apart) DRAW_INLINE {
        double run = 0.0;
        u64 sum = 0;
        tokens([&](const float (&x)[4], int id, int g) {
            bool want[4];
            which_kept(x, id, want);
            double a = 0.0;
            auto add = [&](float y, bool there) DRAW_INLINE {
                const double w = weight_if(y, there);
                a += w >= lower ? w : 0.0;
            };
            if (apart) {
                gather(x, want, add);
                const u64 whole = draw_warp_sum(draw_whole(a));
                if (lane == 0) segment[g] = whole;
                sum += whole;
            } else {                             // (nearly all)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    a += weight_if(x[c], want[c]);
                    if (want[c]) atomicAdd(&s.fine[bin_of(x[c])], 1u);
                }
                run += a;
            }
        });
        if (!apart) sum = draw_warp_sum_wide((u64)run);
        return exchange(3, sum, [](u64 a, u64 b) { return a + b; });
    };

    // The list: tokens are put to it in each CTA's memory; behind a barrier of the cluster, n of them are sorted in s.sorted
    unsigned use = 0;
    int n = 0;
    auto append = [&](const float (&x)[4], int id, unsigned mine) DRAW_INLINE {
        while (mine) {                           // (few)
            const int c = __ffs(mine) - 1, at = atomicAdd(&s.list_n, 1);
            mine &= mine - 1;
            if (at < DRAW_LIST) s.list[at] = draw_key(draw_order(c < 2 ? (c == 0 ? x[0] : x[1]) : (c == 2 ? x[2] : x[3])), id + c);
        }
    };
    // f(logit, which) for a lane's tokens of `mine` (few)
    auto each_of = [&](const float (&x)[4], unsigned mine, auto&& f) DRAW_INLINE {
        while (mine) {
            const int c = __ffs(mine) - 1;
            mine &= mine - 1;
            f(c < 2 ? (c == 0 ? x[0] : x[1]) : (c == 2 ? x[2] : x[3]), c);
        }
    };
    auto fetch_list = [&]() DRAW_INLINE {
        const int m = lane < ctas ? (int)draw_remote(smem_u32(&s.list_n), lane) : 0;
        int from = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, from, o);
            if (lane >= o) from += v;
        }
        n = __shfl_sync(0xffffffffu, from, 31);
        from -= m;
        if (n > DRAW_LIST) return;               // (where it was not counted before)
        const int c = warp % ctas, mc = __shfl_sync(0xffffffffu, m, c), fc = __shfl_sync(0xffffffffu, from, c);      // warps c, c + ctas, ...: those of CTA c
        for (int i = warp / ctas * 32 + lane; i < mc; i += WARPS / ctas * 32) s.all[fc + i] = draw_remote64(smem_u32(&s.list[i]), c);
        __syncthreads();
        {                                        // four, two or one thread an entry
            const int lg = n <= TH / 4 ? 2 : (n <= TH / 2 ? 1 : 0);
            const u64 key = s.all[min(tid >> lg, DRAW_LIST - 1)];
            int rank = 0;
#pragma unroll 4
            for (int j = tid & ((1 << lg) - 1); j < n; j += 1 << lg) rank += s.all[j] > key;
            for (int o = 1; o < 1 << lg; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
            if ((tid & ((1 << lg) - 1)) == 0 && tid >> lg < n) s.sorted[rank] = key;
        }
        __syncthreads();
    };
    auto make_list = [&](auto&& want) DRAW_INLINE {
        four_turns(!RESIDENT, [&](const float (&x)[4], int id, int) {
            unsigned mine = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) mine |= (unsigned)want(x[c], id + c) << c;
            append(x, id, mine);
        });
        cluster_sync_all();
    };

    // The token with which the order's sum of ones (weights: of weights) over what is kept reaches `target`; nothing behind it is kept afterwards, and `segment` has the sums of what is and weighs
    // at least `lower`, over 128 neighbouring tokens; `sum_kept` is the sum of all that is.  Where the sum stays below the target, neither changes.  True where instead the list, of the row's
    // first CTA, has all that can be kept
    enum { LISTED, ENDED, UNENDED };
    u64 sum_kept = 0, total = 0;
    auto search = [&](const bool weights, const u64 target, const double lower, const bool binned) DRAW_INLINE -> int {
        // ---- bins of tokens, over all that matters ----
        if (!binned) four_turns(!RESIDENT, [&](const float (&x)[4], int id, int) {
            bool want[4];
            which_kept(x, id, want);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (want[c]) atomicAdd(&s.fine[bin_of(x[c])], 1u);
        });
        __syncthreads();
        constexpr int PER = DRAW_FINE / DRAW_BINS;           // neighbouring bins of a thread
        unsigned ones[PER] = {0, 0, 0, 0};
        if (tid < DRAW_BINS) {
            const uint4 x = *reinterpret_cast<const uint4*>(s.fine + tid * PER);
            ones[0] = x.x; ones[1] = x.y; ones[2] = x.z; ones[3] = x.w;
            if (ctas > 1) s.packed[use & 1u][tid] = (u64)x.x | (u64)x.y << 16 | (u64)x.z << 32 | (u64)x.w << 48;       // (runs of a cluster are below 2^16 tokens)
            *reinterpret_cast<uint4*>(s.fine + tid * PER) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (tid == 0) {
            s.found_bin = -1;
            s.found_hi = DRAW_FINE - 1;
            s.found_upto = 1 << 30;
        }
        if (ctas > 1) {
            cluster_sync_all();
            if (tid < DRAW_BINS) {
                const uint32_t at = smem_u32(&s.packed[use & 1u][tid]);
                ones[0] = ones[1] = ones[2] = ones[3] = 0u;
#pragma unroll 8
                for (int c = 0; c < ctas; ++c) {
                    const u64 x = draw_remote64(at, c);
                    ones[0] += (unsigned)x & 0xFFFFu; ones[1] += (unsigned)x >> 16; ones[2] += (unsigned)(x >> 32) & 0xFFFFu; ones[3] += (unsigned)(x >> 48);
                }
            }
        }
        ++use;
        // Sums up to each bin.  Of weights, a token's is between that of its bin's nearer and its further edge (a hundredth apart; a ten-thousandth more covers all rounding here), so that
        // the token is between the first bin whose larger sum reaches the target and the first whose smaller one does.  A target beyond the half is counted from the other end, as what is
        // behind it: a hundredth of that is less (there, whole numbers may be half a unit off for every token)
        constexpr float SLACK = 1e-4f;
        const float step = 2.f / (bins_over * temperature);
        unsigned count = ones[0] + ones[1] + ones[2] + ones[3];
        float share = 0.f;
        const float edge = expf(-step * (float)(tid * PER)), ratio = expf(-step);
        if (weights && tid < DRAW_BINS) share = edge * ((float)ones[0] + ratio * ((float)ones[1] + ratio * ((float)ones[2] + ratio * (float)ones[3])));
        unsigned count_at = (unsigned)draw_warp_scan(count);
        const bool behind = weights && 2 * target > total;           // (total: of what is in the bins)
        float share_at = share;                  // of this thread and all before it, or all behind
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float v = __shfl_sync(0xffffffffu, share_at, behind ? lane + o : lane - o);
            if (behind ? lane + o < 32 : lane >= o) share_at += v;
        }
        if (lane == 31) s.warp[0][warp] = count_at;
        if (lane == (behind ? 0 : 31)) s.warp_f[warp] = share_at;
        const float next = __shfl_sync(0xffffffffu, share_at, behind ? lane + 1 : lane - 1);
        float share_without = lane == (behind ? 31 : 0) ? 0.f : next;
        __syncthreads();
        for (int w = 0; w < min(warp, DRAW_BINS / 32); ++w) count_at += (unsigned)s.warp[0][w];
        for (int w = behind ? warp + 1 : 0; w < (behind ? DRAW_BINS / 32 : min(warp, DRAW_BINS / 32)); ++w) share_without += s.warp_f[w];
        if (weights && tid < DRAW_BINS) {
            // (a bin of none moves no sum: borders are found at one thread each but for rounding, the lowest and the highest count)
            const float half_step = sqrtf(ratio), goal = (float)((double)(behind ? total - target : target) * 0x1p-40), off = behind ? (float)p.V * 0x1p-41f : 0.f;
            float w[PER] = {edge, edge * ratio, edge * ratio * ratio, edge * ratio * ratio * ratio}, sh = share_without;
            if (behind) {
                const float near_goal = (goal + off) * (1.f + SLACK) / half_step, far_goal = (goal - off) * (1.f - SLACK) * half_step;
#pragma unroll
                for (int i = PER - 1; i >= 0; --i) {
                    const float sh1 = sh + w[i] * (float)ones[i];
                    if (ones[i] && sh <= near_goal && sh1 * (1.f + SLACK) > near_goal) atomicMax(&s.found_bin, (DRAW_FINE - 1) - (tid * PER + i));
                    if (ones[i] && sh <= far_goal && sh1 * (1.f + SLACK) > far_goal) atomicMin(&s.found_hi, tid * PER + i);
                    sh = sh1;
                }
            } else {
                const float near_goal = goal * (1.f - SLACK) * half_step, far_goal = goal * (1.f + SLACK) / half_step;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const float sh1 = sh + w[i] * (float)ones[i];
                    if (ones[i] && sh1 >= near_goal && sh * (1.f - SLACK) < near_goal) atomicMax(&s.found_bin, (DRAW_FINE - 1) - (tid * PER + i));
                    if (ones[i] && sh1 >= far_goal && sh * (1.f - SLACK) < far_goal) atomicMin(&s.found_hi, tid * PER + i);
                    sh = sh1;
                }
            }
        } else if (!weights && tid < DRAW_BINS) {
            unsigned c = count_at - count;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const unsigned c1 = c + ones[i];
                if (c < target && c1 >= target) {
                    s.found_bin = (DRAW_FINE - 1) - (tid * PER + i);
                    s.found_hi = tid * PER + i;
                }
                c = c1;
            }
        }
        __syncthreads();
        if (s.found_bin < 0) return UNENDED;
        const int lo_bin = (DRAW_FINE - 1) - s.found_bin, hi_bin = s.found_hi;
        {                                        // tokens up to hi_bin, and in front of lo_bin
            unsigned c = count_at - count;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (tid * PER + i == lo_bin && tid < DRAW_BINS) s.found_count = (int)c;
                c += ones[i];
                if (tid * PER + i == hi_bin && tid < DRAW_BINS) s.found_upto = (int)c;
            }
        }
        __syncthreads();
        const int ahead = s.found_count, upto = s.found_upto;
        if (upto <= DRAW_LIST) {
            make_list([&](float x, int id) { return among_kept(x, id) & (bin_of(x) <= hi_bin); });
            if (cta == 0) fetch_list();
            return LISTED;
        }
        // ---- between two bins: the sum in front of them, exactly, and their tokens to the list; where it has no room for them all, narrower ones ----
        int sub = -1, shift = 64, left = upto - ahead;
        u64 begin = 0;
        constexpr unsigned LOW = (1u << DRAW_LIMB) - 1;
        auto put = [&](int at, float y) DRAW_INLINE {
            atomicAdd(&s.bins[0][at], 1u);
            if (weights) {
                const u64 w = weight(y);
                atomicAdd(&s.bins[1][at], (unsigned)w & LOW);
                atomicAdd(&s.bins[2][at], (unsigned)(w >> DRAW_LIMB) & LOW);
                atomicAdd(&s.bins[3][at], (unsigned)(w >> 2 * DRAW_LIMB));
            }
        };
        const float sub_over = (float)DRAW_BINS / (float)(hi_bin - lo_bin + 1);
        auto sub_of = [&](float x) { return max(0, min(DRAW_BINS - 1, (int)((from_top(x) * bins_over - (float)lo_bin) * sub_over))); };
        auto among = [&](float x, int id) -> bool {
            const int b = bin_of(x);
            bool in = among_kept(x, id) & (b >= lo_bin) & (b <= hi_bin);
            if (sub >= 0) in = in & (sub_of(x) == sub);
            if (shift < 64) in = in & (draw_key(draw_order(x), id) >> shift == begin);
            return in;
        };
        double run = 0.0;
        tokens([&](const float (&x)[4], int id, int g) {
            bool want[4];
            which_kept(x, id, want);
            unsigned mine = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int b = bin_of(x[c]);
                mine |= (unsigned)(want[c] & (b >= lo_bin) & (b <= hi_bin)) << c;
                want[c] = want[c] & (b < lo_bin);
            }
            double counted = 0.0;
            gather(x, want, [&](float y, bool there) DRAW_INLINE {
                const double w = weight_if(y, there);
                run += w;
                counted += w >= lower ? w : 0.0;
            });
            const u64 whole = draw_warp_sum(draw_whole(counted));
            if (lane == 0) segment[g] = whole;
            if (left <= DRAW_LIST) append(x, id, mine);
            else each_of(x, mine, [&](float y, int) DRAW_INLINE { put(sub_of(y), y); });
        });
        const u64 sum_ahead = exchange(1, draw_warp_sum_wide((u64)run), [](u64 a, u64 b) { return a + b; });
        u64 before = weights ? sum_ahead : ahead;
        const bool narrower = left > DRAW_LIST;
        while (left > DRAW_LIST) {
            const int next = sub < 0 ? 64 : (shift >= 64 ? 45 : shift - DRAW_BIN_BITS);
            if (sub >= 0) tokens([&](const float (&x)[4], int id, int) {
                unsigned mine = 0;
#pragma unroll
                for (int c = 0; c < 4; ++c) mine |= (unsigned)among(x[c], id + c) << c;
                each_of(x, mine, [&](float y, int c) DRAW_INLINE { put(DRAW_BINS - 1 - (int)((draw_key(draw_order(y), id + c) >> next) & (DRAW_BINS - 1)), y); });
            });
            __syncthreads();
            constexpr int MANY = 255;                        // a CTA's tokens of a bin, eight bits of a cluster's word (its runs are below 2^16 tokens, their weights below 2^56)
            u64 sum = 0;
            unsigned tokens_here = 0;
            if (tid < DRAW_BINS) {
                tokens_here = s.bins[0][tid];
                sum = weights ? s.bins[1][tid] + ((u64)s.bins[2][tid] << DRAW_LIMB) + ((u64)s.bins[3][tid] << 2 * DRAW_LIMB) : tokens_here;
                s.packed[use & 1u][tid] = weights ? sum + ((u64)min(tokens_here, (unsigned)MANY) << 56) : sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) s.bins[i][tid] = 0u;
            }
            if (tid == 0) s.found_bin = -1;
            cluster_sync_all();
            if (ctas > 1 && tid < DRAW_BINS) {
                const uint32_t at = smem_u32(&s.packed[use & 1u][tid]);
                sum = 0;
                tokens_here = 0;
#pragma unroll 1
                for (int c = 0; c < ctas; ++c) {
                    const u64 x = draw_remote64(at, c);
                    sum += weights ? x & ((1ull << 56) - 1) : x;
                    tokens_here += weights ? (x >> 56 == MANY ? 1u << 20 : (unsigned)(x >> 56)) : (unsigned)x;
                }
            }
            ++use;
            u64 at = draw_warp_scan(sum);
            if (lane == 31) s.warp[0][warp] = at;
            __syncthreads();
            at += before;
            for (int w = 0; w < min(warp, DRAW_BINS / 32); ++w) at += s.warp[0][w];
            if (tid < DRAW_BINS && at - sum < target && at >= target) {
                s.found_bin = tid;
                s.found_before = at - sum;
                s.found_count = (int)tokens_here;
            }
            __syncthreads();
            if (s.found_bin < 0) return UNENDED;
            before = s.found_before;
            left = s.found_count;
            if (sub < 0) {
                sub = s.found_bin;
            } else {
                begin = (begin << DRAW_BIN_BITS) | (unsigned)(DRAW_BINS - 1 - s.found_bin);
                shift = next;
            }
            __syncthreads();                     // (what was found is read before it is written again)
        }
        u64 sum_between = 0;                     // of what lies between the bins in front and the list
        if (narrower) {
            double more = 0.0;
            four_turns(!RESIDENT, [&](const float (&x)[4], int id, int g) {
                unsigned mine = 0, front = 0;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int b = bin_of(x[c]);
                    if ((b >= lo_bin) & (b <= hi_bin)) {
                        mine |= (unsigned)among(x[c], id + c) << c;
                        front |= (unsigned)(among_kept(x[c], id + c) & (sub_of(x[c]) < sub)) << c;
                    }
                }
                append(x, id, mine);
                each_of(x, front, [&](float y, int) DRAW_INLINE {
                    const double w = weight_if(y, true);
                    more += w;
                    if (w >= lower) atomicAdd(segment + g, draw_whole(w));
                });
            });
            sum_between = exchange(0, draw_warp_sum_wide((u64)more), [](u64 a, u64 b) { return a + b; });
        }
        fetch_list();
        const u64 w = tid < n ? weight(draw_logit(s.sorted[tid])) : 0ull, one = weights ? w : (u64)(tid < n);
        u64 at = draw_warp_scan(one);
        if (lane == 31) s.warp[0][warp] = at;
        if (tid == 0) s.found_hi = -1;
        __syncthreads();
        at += before;
        for (int v = 0; v < warp; ++v) at += s.warp[0][v];
        if (tid < n && at - one < target && at >= target) s.found_hi = tid;
        __syncthreads();
        const int end = s.found_hi;
        if (end < 0) return UNENDED;
        const u64 key = s.sorted[end];
        last = nearest = draw_logit(key);
        tied = true;
        last_id = (1 << DRAW_ID_BITS) - 1 - (int)(key & ((1u << DRAW_ID_BITS) - 1));
        if (shift < 64) {                        // (equal logits: what lies between the list and narrower bins is not in the sums)
            __syncthreads();                     // (all have read their entry: the warps' queues lie over the list)
            return UNENDED;
        }
        // the list's part of the sums
        const bool kept = tid <= end;
        const u64 listed = draw_warp_sum(kept ? w : 0);
        if (lane == 0) s.warp[1][warp] = listed;
        if (kept && (double)w >= lower) {
            const int i = (1 << DRAW_ID_BITS) - 1 - (int)(s.sorted[tid] & ((1u << DRAW_ID_BITS) - 1)) - lo;
            if (i >= 0 && i < cnt) atomicAdd(segment + i / 128, w);
        }
        __syncthreads();
        sum_kept = sum_ahead + sum_between;
        for (int v = 0; v < WARPS; ++v) sum_kept += s.warp[1][v];
        return ENDED;
    };
    // the number of 2^-40 with which a sum of them reaches top_p
    auto share_of = [&](u64 total) DRAW_INLINE { return max((u64)ceil(fmax((double)top_p, 0.0) * (double)total), 1ull); };

    // the rest, from the sorted list of n tokens that have all that can be kept: first `k` of them, then those that reach top_p of `total` (0: of the weights of these)
    auto finish = [&](int k, u64 total) DRAW_INLINE {
        const bool real = tid < n && tid < k;
        const u64 key = tid < n ? s.sorted[tid] : 0, w = real ? weight(draw_logit(key)) : 0;
        u64 upto = draw_warp_scan(w);
        if (lane == 31) s.warp[0][warp] = upto;
        __syncthreads();
        u64 all = 0;
        for (int v = 0; v < WARPS; ++v) {
            if (v < warp) upto += s.warp[0][v];
            all += s.warp[0][v];
        }
        bool keep = real && (w >= floor_weight || tid == 0);
        if (top_p < 1.f) keep = keep && (upto - w < share_of(total ? total : all));
        const u64 kept = draw_warp_sum(keep ? w : 0);
        if (lane == 0) s.warp[1][warp] = kept;
        if (tid < n) s.weight[tid] = keep ? w : 0;
        __syncthreads();
        u64 whole_kept = 0;
        for (int v = 0; v < WARPS; ++v) whole_kept += s.warp[1][v];
        u64 target = (u64)fmax(floor((double)u * (double)whole_kept), 0.0);
        target = target < whole_kept ? target : whole_kept - 1;
        {                                        // four, two or one thread an entry
            constexpr unsigned IDS = (1u << DRAW_ID_BITS) - 1;
            const int lg = n <= TH / 4 ? 2 : (n <= TH / 2 ? 1 : 0), e = min(tid >> lg, DRAW_LIST - 1);
            const unsigned rest = (unsigned)(s.sorted[e] & IDS);             // (larger for lower ids)
            const u64 mine_w = e < n ? s.weight[e] : 0;
            u64 at = 0;
#pragma unroll 4
            for (int j = tid & ((1 << lg) - 1); j < n; j += 1 << lg) at += (unsigned)(s.sorted[j] & IDS) > rest ? s.weight[j] : 0;
            for (int o = 1; o < 1 << lg; o <<= 1) at += __shfl_xor_sync(0xffffffffu, at, o);
            if (tid >> lg < n && (tid & ((1 << lg) - 1)) == 0 && at <= target && target < at + mine_w) {
                p.tokens[row] = (int)(IDS - rest);
                if (p.probs) p.probs[row] = (float)((double)mine_w / (double)whole_kept);
            }
        }
    };

    bool narrow = false;                         // the list has everything
    int state = UNENDED;
    int k = 1 << 30;
    if (top_k > 0 && top_k < p.V) {
        if (ctas == 1 && top_k <= TH) {
            // At least top_k tokens are as near as the top_k-th of the threads' best: bins of these alone tell a distance beyond which none of the first is.  (Tokens up to there, about as many,
            // go to the list uncounted; where they are more than it holds, everything is as if this had not been tried)
            if (mine >= nearest) atomicAdd(&s.fine[bin_of(mine)], 1u);
            __syncthreads();
            constexpr int PER = DRAW_FINE / DRAW_BINS;
            unsigned ones[PER] = {0, 0, 0, 0};
            if (tid < DRAW_BINS) {
                const uint4 x = *reinterpret_cast<const uint4*>(s.fine + tid * PER);
                ones[0] = x.x; ones[1] = x.y; ones[2] = x.z; ones[3] = x.w;
                *reinterpret_cast<uint4*>(s.fine + tid * PER) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (tid == 0) s.found_hi = -1;
            unsigned at = (unsigned)draw_warp_scan(ones[0] + ones[1] + ones[2] + ones[3]);
            if (lane == 31) s.warp[0][warp] = at;
            __syncthreads();
            for (int w = 0; w < min(warp, DRAW_BINS / 32); ++w) at += (unsigned)s.warp[0][w];
            at -= ones[0] + ones[1] + ones[2] + ones[3];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (at < (unsigned)top_k && at + ones[i] >= (unsigned)top_k) s.found_hi = tid * PER + i;
                at += ones[i];
            }
            __syncthreads();
            const int edge = s.found_hi;
            if (edge >= 0) {
                make_list([&](float x, int id) { return (x >= nearest) & (bin_of(x) <= edge); });
                fetch_list();
                narrow = n <= DRAW_LIST;
                __syncthreads();
                if (!narrow && tid == 0) s.list_n = 0;
                __syncthreads();
            }
        }
        if (narrow) k = top_k;
    }
    // the first top_k; those that reach top_p; the sum of what is left (one place for each step: a lambda that is called from two keeps its variables in memory)
#pragma unroll 1
    for (int by = top_k > 0 && top_k < p.V ? 0 : 1; by < 3 && !narrow; ++by) {
        if (by == 1 && top_p >= 1.f) continue;
        u64 target = (u64)max(top_k, 1);
        bool binned = false;
        if (by > 0) {
            const bool lastly = by == 2;
            if (state == ENDED) {
                cluster_sync_all();              // (all CTAs have read the lists and one another's sums; and the CTA's own)
                total = sum_kept;
                if (lastly) {
                    u64 sum = 0;
                    for (int g = tid; g < segments; g += TH) sum += segment[g];
                    total = exchange(2, draw_warp_sum_wide(sum), [](u64 a, u64 b) { return a + b; });
                }
            } else {
                if (lastly && floor_weight > 1) nearest = fmaxf(nearest, nearest_of(distance((double)floor_weight)));
                total = add_up(lastly ? (double)floor_weight : 0.0, lastly);
                binned = true;
            }
            if (lastly) break;
            if (tid == 0) s.list_n = 0;
            target = share_of(total);
        }
        state = search(by == 1, target, by == 0 && top_p < 1.f ? 0.0 : (double)floor_weight, binned);
        narrow = state == LISTED;
        if (narrow && by == 0) k = top_k;
    }
    if (narrow) {
        if (cta == 0) finish(k, total);
        if (ctas > 1) cluster_sync_all();        // no CTA leaves while its list is read
        return;
    }

    // ---- the token: its CTA, its 128 tokens, itself ----
    u64 target = (u64)fmax(floor((double)u * (double)total), 0.0), before = 0;
    target = target < total ? target : total - 1;
    for (int c = 0; c < cta; ++c) before += s.slot[state == ENDED ? 2 : 3][c];
    if (warp != 0 || target < before || target - before >= s.slot[state == ENDED ? 2 : 3][cta]) return;
    int where = -1;
    for (int g0 = 0; g0 < segments; g0 += 32) {
        const u64 x = g0 + lane < segments ? segment[g0 + lane] : 0, upto = draw_warp_scan(x);
        const unsigned hit = __ballot_sync(0xffffffffu, target - before < upto);
        if (hit) {
            const int from = __ffs(hit) - 1;
            where = g0 + from;
            before += __shfl_sync(0xffffffffu, upto - x, from);
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const float4 x4 = RESIDENT ? fours[where * 32 + lane] : (where < full ? DrawRaw<E>::widen4(ask(where)) : ragged(where));
    const float x[4] = {x4.x, x4.y, x4.z, x4.w};
    const int id = lo + (where * 32 + lane) * 4;
    u64 w[4], run = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        w[c] = among_kept(x[c], id + c) ? weight(x[c]) : 0ull;
        if (w[c] < floor_weight) w[c] = 0;
        run += w[c];
    }
    u64 at = before + draw_warp_scan(run) - run;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (at <= target && target < at + w[c]) {
            p.tokens[row] = id + c;
            if (p.probs) p.probs[row] = (float)((double)w[c] / (double)total);
        }
        at += w[c];
    }
}

}  // namespace b200

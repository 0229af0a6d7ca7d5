// A token for each row of logits from a given random number, under a temperature, top-k, top-p and min-p.  For a row l, its largest logit m, temperature T:
//     w_t = exp((l_t - m) / T);  tokens in order: larger logit first, of equal ones the lower id
//     kept are the first k of them; of these the shortest beginning that holds top_p of their weights; of these the ones with w_t >= min_p (the first always)
//     the token is the lowest id at which the sum of kept weights, ids ascending, exceeds u times all of it
// Reference: what its samplers do behind the softmax (sampler/nucleus.rs:69-123, sampler/typical.rs:70-131), whose own orders the host classes keep.
//
// A sum that ends beside a border decides about a token, so that 32 bits would draw other tokens than the definition: weights are whole numbers of 2^-40 of the
// row's largest, from exponentials in 64 bits, and their sums are exact in any order.  Tokens below half a unit weigh nothing and are never drawn.
//
// Bound: a row is read once (512 rows of 65536 f32: 20 us), and then held in the shared memory of a cluster of eight or sixteen CTAs, a run of it each; one row is latency: exchanges in the
// cluster, about a microsecond each.  Nothing is sorted: a beginning of the order is found from its end, the token with which a sum over the order (of ones, or of weights) reaches a
// target.  512 bins over the distance from the largest logit tell between which two distances it lies, each CTA adds up all CTAs' bins; the tokens of that bin
// (a few dozen) are then ranked one against another.  Where a bin holds more than a list, as with thousands of equal logits, bins over nine bits at a time
// of (logit, id) narrow it down first.
#pragma once
#include <cuda_bf16.h>

#include "sm_pair.cuh"
#include "token_ops.cuh"

#include <type_traits>

namespace b200 {

constexpr int DRAW_BINS = 512, DRAW_BIN_BITS = 9;
constexpr int DRAW_LIST = 512;                   // tokens that are ranked one against another
constexpr int DRAW_UNIT = 40;                    // weights are multiples of 2^-40
constexpr int DRAW_LIMB = 14;                    // bits of a weight in each of three words of a bin: sums of 2^15 of them fit 32 bits
static_assert(3 * DRAW_LIMB > DRAW_UNIT, "the largest weight fits");

typedef unsigned long long u64;

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
// round(2^40 2^y) for y <= 0: 2^y = 2^n 2^f with n the nearest whole number, 2^f by its power series (|f ln 2| < 0.347: the terms from the twelfth on are
// below 2^-47)
__device__ __forceinline__ u64 draw_exp2(double y) {
    if (!(y > -(DRAW_UNIT + 1.5))) return 0;
    const double magic = 6755399441055744.0;             // 1.5 2^52: the sum's last bits are the whole number
    const double t = y + magic, f = y - (t - magic);
    const int n = (int)(unsigned)__double_as_longlong(t);
    constexpr double L = 0.6931471805599453094;
    constexpr double C2 = L * L / 2, C3 = C2 * L / 3, C4 = C3 * L / 4, C5 = C4 * L / 5, C6 = C5 * L / 6, C7 = C6 * L / 7, C8 = C7 * L / 8, C9 = C8 * L / 9, C10 = C9 * L / 10,
                     C11 = C10 * L / 11;
    double s = C11;
    s = fma(s, f, C10); s = fma(s, f, C9); s = fma(s, f, C8); s = fma(s, f, C7); s = fma(s, f, C6); s = fma(s, f, C5);
    s = fma(s, f, C4); s = fma(s, f, C3); s = fma(s, f, C2); s = fma(s, f, L); s = fma(s, f, 1.0);
    const double unit = __longlong_as_double((long long)(n + DRAW_UNIT + 1023) << 52);
    return (u64)(__double_as_longlong(fma(s, unit, 4503599627370496.0)) - 0x4330000000000000ll);       // (2^52 + x: x in the last bits, to nearest)
}

// sums over a warp: in whole numbers, a few bits at a time by the unit's own additions
__device__ __forceinline__ u64 draw_warp_sum(u64 v) {      // v < 2^46
    const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x7FFFFFu), b = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 23));
    return (u64)a + ((u64)b << 23);
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

template <int TH>
struct DrawShared {
    unsigned bins[2][4][DRAW_BINS];          // tokens, and their weights in three parts; two, so that one may be read by other CTAs while the next is filled
    u64 list[DRAW_LIST], all[DRAW_LIST], sorted[DRAW_LIST];
    u64 segment[DRAW_MAX_SLICE / 128];       // sums over 128 neighbouring tokens
    u64 warp[TH / 32];
    u64 slot[3][DRAW_MOST_CTAS];             // what the CTAs tell one another
    u64 found, found_before;
    int found_count, found_bin, list_n;
};

template <int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) draw_kernel(const __grid_constant__ DrawParams p) {
    extern __shared__ __align__(16) float4 fours[];          // the CTA's run, -inf behind it
    __shared__ __align__(16) DrawShared<TH> s;
    constexpr int WARPS = TH / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = 1 << p.ctas_log, cta = blockIdx.x & (ctas - 1), row = blockIdx.x >> p.ctas_log;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");        // no CTA writes to another's memory before all have started
    pdl_wait();
    pdl_launch_dependents();
    const int lo = min(cta * p.slice, p.V), cnt = min(lo + p.slice, p.V) - lo, nf = p.slice / 4;

    // ---- the row, its largest logit ----
    float mine = -INFINITY;
    bool nan = false;
    {
        const long long first = (long long)(p.in_row ? p.in_row[row] : row) * p.in_stride + lo;
        auto read = [&](auto from, auto four, auto one) {
#pragma unroll 4
            for (int f = tid; f < nf; f += TH) {
                const int i = f * 4;
                float x[4];
                if (p.vec && i + 3 < cnt) {
                    four(from + i, x);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[c] = i + c < cnt ? one(from[i + c]) : -INFINITY;
                }
                fours[f] = make_float4(x[0], x[1], x[2], x[3]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    mine = fmaxf(mine, x[c]);
                    nan |= isnan(x[c]);
                }
            }
        };
        if (p.type == 0) {
            read((const float*)p.in + first, [](const float* q, float (&o)[4]) { const float4 x = *(const float4*)q; o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w; },
                 [](float x) { return x; });
        } else if (p.type == 1) {
            read((const __half*)p.in + first,
                 [](const __half* q, float (&o)[4]) {
                     const uint2 u = *(const uint2*)q;
                     const float2 a = __half22float2(*(const __half2*)&u.x), b = __half22float2(*(const __half2*)&u.y);
                     o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
                 },
                 [](__half x) { return __half2float(x); });
        } else {
            read((const __nv_bfloat16*)p.in + first,
                 [](const __nv_bfloat16* q, float (&o)[4]) {
                     const uint2 u = *(const uint2*)q;
                     o[0] = __uint_as_float(u.x << 16); o[1] = __uint_as_float(u.x & 0xFFFF0000u); o[2] = __uint_as_float(u.y << 16); o[3] = __uint_as_float(u.y & 0xFFFF0000u);
                 },
                 [](__nv_bfloat16 x) { return __bfloat162float(x); });
        }
    }
    // f(logit, id) for the thread's tokens (its own: no barrier is needed between the loop above and these)
    auto each = [&](auto&& f) {
        for (int q = tid; q < nf; q += TH) {
            const float4 x = fours[q];
            const int id = lo + q * 4;
            f(x.x, id); f(x.y, id + 1); f(x.z, id + 2); f(x.w, id + 3);
        }
    };
    const float u = p.uniform[row], temperature = p.temperature ? p.temperature[row] : 1.f, top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
    const int top_k = p.top_k ? p.top_k[row] : 0;
    // a value of each warp over the block and the cluster's CTAs, by `combine` of two: every CTA has all CTAs' values afterwards
    auto exchange = [&](int which, u64 x, auto&& combine) {
        if (lane == 0) s.warp[warp] = x;
        __syncthreads();
        if (tid < ctas) {
            u64 a = s.warp[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) a = combine(a, s.warp[w]);
            draw_tell(&s.slot[which][cta], a, tid);
        }
        cluster_sync_all();
        u64 a = s.slot[which][0];
        for (int c = 1; c < ctas; ++c) a = combine(a, s.slot[which][c]);
        return a;
    };
    // (the bins of the first search)
    for (int i = tid; i < 4 * DRAW_BINS; i += TH) (&s.bins[0][0][0])[i] = 0u;
    if (tid == 0) s.list_n = 0;
    const unsigned order = __reduce_max_sync(0xffffffffu, draw_order(mine)), any_nan = __any_sync(0xffffffffu, nan);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const u64 best = exchange(0, ((u64)any_nan << 32) | order, [](u64 a, u64 b) { return ((a | b) >> 32 << 32) | max((unsigned)a, (unsigned)b); });
    const float top = draw_logit((u64)(unsigned)best << DRAW_ID_BITS);
    if (best >> 32 || isnan(u) || isnan(top_p) || isnan(min_p) || !(temperature >= 0.f && temperature < INFINITY) || top == -INFINITY) {
        if (cta == 0 && tid == 0) {
            p.tokens[row] = -1;
            if (p.probs) p.probs[row] = top == -INFINITY && !(best >> 32) ? 0.f : __int_as_float(0x7fc00000);
        }
        return;
    }

    // ---- the best token alone ----
    if (temperature == 0.f || top_k == 1) {
        unsigned id = ~0u;
        each([&](float x, int i) {
            if (x == top) id = min(id, (unsigned)i);
        });
        const u64 a = exchange(1, __reduce_min_sync(0xffffffffu, id), [](u64 x, u64 y) { return x < y ? x : y; });
        if (cta == 0 && tid == 0) {
            p.tokens[row] = (int)a;
            if (p.probs) p.probs[row] = 1.f;
        }
        return;
    }

    // ---- weights ----
    const double over = 1.4426950408889634074 / (double)temperature;
    const float reach = 42.f * 0.6931472f * 1.00001f * temperature;          // further from the largest logit, a weight is less than half a unit
    const float bins_over = (DRAW_BINS - 1) / reach;
    auto near = [&](float x, float far) { return x == top || top - x <= far; };
    auto weight = [&](float x) { return x == top ? 1ull << DRAW_UNIT : draw_exp2(((double)x - (double)top) * over); };
    auto bin_of = [&](float x) { return x == top ? 0 : min(DRAW_BINS - 1, (int)((top - x) * bins_over)); };
    u64 least = 0;                               // keys below it are not kept
    auto kept = [&](float x, int id) { return draw_key(draw_order(x), id) >= least; };

    // weights of what is kept and weighs at least `floor_weight`: over 128 neighbouring tokens, and over the row
    auto add_up = [&](int which, u64 floor_weight) {
        u64 sum = 0;
        for (int q0 = warp * 32; q0 < nf; q0 += TH) {
            const int q = q0 + lane;
            u64 a = 0;
            if (q < nf) {
                const float4 x4 = fours[q];
                const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (!near(x[c], reach) || (least && !kept(x[c], lo + q * 4 + c))) continue;
                    const u64 w = weight(x[c]);
                    if (w >= floor_weight) a += w;
                }
            }
            a = draw_warp_sum(a);
            if (lane == 0) s.segment[q0 / 32] = a;
            sum += a;
        }
        return exchange(which, sum, [](u64 a, u64 b) { return a + b; });
    };

    // least = the key at which the order's sum of ones (WEIGHTS: of weights) over what is kept reaches `target`.  far: tokens further from the largest cannot be it
    unsigned use = 0;
    auto search = [&](auto by_weight, u64 target, float far) {
        constexpr bool WEIGHTS = decltype(by_weight)::value;
        int shift = 64, bin = -1;                // tokens looked at: of one bin, then of keys that begin alike
        u64 begin = 0, before = 0;
        auto among = [&](float x, int id) {
            if (!near(x, far) || (least && !kept(x, id))) return false;
            if (bin < 0) return true;
            if (bin_of(x) != bin) return false;
            return shift >= 64 || draw_key(draw_order(x), id) >> shift == begin;
        };
        // neighbouring values to a thread: the place at which the running sum from `before` on reaches the target is told
        auto reaches = [&](auto& sums, auto&& tell) {
            constexpr int PER = sizeof(sums) / sizeof(sums[0]);
            u64 run = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) run += sums[i];
            const u64 upto = draw_warp_scan(run);
            if (lane == 31) s.warp[warp] = upto;
            __syncthreads();
            u64 at = before + upto - run;
            for (int w = 0; w < warp; ++w) at += s.warp[w];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (at < target && at + sums[i] >= target) tell(i, at);
                at += sums[i];
            }
        };
        for (;;) {
            unsigned (*const b)[DRAW_BINS] = s.bins[use & 1u];
            const int next = shift >= 64 ? 45 : shift - DRAW_BIN_BITS;
            each([&](float x, int id) {
                if (!among(x, id)) return;
                const int at = bin < 0 ? bin_of(x) : DRAW_BINS - 1 - (int)((draw_key(draw_order(x), id) >> next) & (DRAW_BINS - 1));
                atomicAdd(&b[0][at], 1u);
                if (WEIGHTS) {
                    const u64 w = weight(x);
                    constexpr unsigned LOW = (1u << DRAW_LIMB) - 1;
                    const unsigned w0 = (unsigned)w & LOW, w1 = (unsigned)(w >> DRAW_LIMB) & LOW, w2 = (unsigned)(w >> 2 * DRAW_LIMB);
                    if (w0) atomicAdd(&b[1][at], w0);
                    if (w1) atomicAdd(&b[2][at], w1);
                    if (w2) atomicAdd(&b[3][at], w2);
                }
            });
            cluster_sync_all();
            if (tid == 0) s.found_bin = -1;      // (all threads have read what the last round found)
            // all CTAs' bins
            constexpr int PER = DRAW_BINS / TH;
            u64 ones[PER], sums[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = tid * PER + i;
                ones[i] = 0;
                u64 w0 = 0, w1 = 0, w2 = 0;
#pragma unroll 8
                for (int c = 0; c < ctas; ++c) {
                    ones[i] += draw_remote(smem_u32(&b[0][at]), c);
                    if (WEIGHTS) {
                        w0 += draw_remote(smem_u32(&b[1][at]), c);
                        w1 += draw_remote(smem_u32(&b[2][at]), c);
                        w2 += draw_remote(smem_u32(&b[3][at]), c);
                    }
                }
                sums[i] = WEIGHTS ? w0 + (w1 << DRAW_LIMB) + (w2 << 2 * DRAW_LIMB) : ones[i];
            }
            reaches(sums, [&](int i, u64 at) {
                s.found_bin = tid * PER + i;
                s.found_before = at;
                s.found_count = (int)ones[i];
            });
            // (the other bins are read no more: all CTAs have come through the barrier above)
            ++use;
            for (int i = tid; i < 4 * DRAW_BINS; i += TH) (&s.bins[use & 1u][0][0])[i] = 0u;
            __syncthreads();
            const int found = s.found_bin, count = s.found_count;
            if (found < 0) return;               // the sum stays below the target: nothing ends
            before = s.found_before;
            if (bin < 0) {
                bin = found;
            } else {
                begin = (begin << DRAW_BIN_BITS) | (unsigned)(DRAW_BINS - 1 - found);
                shift = next;
            }
            if (count <= DRAW_LIST) break;
        }
        // ---- what is left, one against another ----
        each([&](float x, int id) {
            if (among(x, id)) s.list[atomicAdd(&s.list_n, 1)] = draw_key(draw_order(x), id);
        });
        cluster_sync_all();
        int n = 0;
        for (int c = 0; c < ctas; ++c) {
            const int m = (int)draw_remote(smem_u32(&s.list_n), c);
            for (int i = tid; i < m; i += TH) s.all[n + i] = draw_remote64(smem_u32(&s.list[i]), c);
            n += m;
        }
        __syncthreads();
        for (int i = tid; i < n; i += TH) {
            const u64 key = s.all[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += s.all[j] > key;
            s.sorted[rank] = key;
        }
        __syncthreads();
        constexpr int PER = DRAW_LIST / TH;
        u64 sums[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) sums[i] = tid * PER + i < n ? (WEIGHTS ? weight(draw_logit(s.sorted[tid * PER + i])) : 1ull) : 0ull;
        reaches(sums, [&](int i, u64) { s.found = s.sorted[tid * PER + i]; });
        __syncthreads();
        least = s.found;
    };

    if (top_k > 0 && top_k < p.V) search(std::false_type{}, (u64)top_k, reach);
    if (top_p < 1.f) {
        const u64 total = add_up(1, 0);
        if (tid == 0) s.list_n = 0;              // (the search in front has read the lists: all CTAs have come through the barrier of the sum)
        // the shortest beginning that holds top_p of the sum.  Tokens of less than (1 - top_p) / V of it lie behind, all of them together
        const double share = fmax((double)top_p, 0.0) * (double)total, tail = ((double)total - share) / (double)p.V * 0.999;
        const float far = tail > 1.0 ? fminf(reach, (float)(DRAW_UNIT - log2(tail)) * 0.6931472f * temperature * 1.0001f) : reach;
        search(std::true_type{}, max((u64)ceil(share), 1ull), far);
    }
    const u64 floor_weight = (u64)ceil(fmin(fmax((double)min_p, 0.0), 1.0) * (double)(1ull << DRAW_UNIT));
    const u64 total = add_up(2, floor_weight);

    // ---- the token: its CTA, its 128 tokens, itself ----
    u64 target = (u64)fmax(floor((double)u * (double)total), 0.0), before = 0;
    target = target < total ? target : total - 1;
    for (int c = 0; c < cta; ++c) before += s.slot[2][c];
    if (warp != 0 || target < before || target - before >= s.slot[2][cta]) return;
    constexpr int SEGMENTS = DRAW_MAX_SLICE / 128, EACH = SEGMENTS / 32;
    const int segments = (nf + 31) / 32;
    u64 run = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) run += lane * EACH + i < segments ? s.segment[lane * EACH + i] : 0;
    u64 at = before + draw_warp_scan(run) - run;
    int where = -1;
    u64 where_before = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const u64 x = lane * EACH + i < segments ? s.segment[lane * EACH + i] : 0;
        if (at <= target && target < at + x) {
            where = lane * EACH + i;
            where_before = at;
        }
        at += x;
    }
    const int from = __ffs(__ballot_sync(0xffffffffu, where >= 0)) - 1;
    where = __shfl_sync(0xffffffffu, where, from);
    where_before = __shfl_sync(0xffffffffu, where_before, from);
    const int q = where * 32 + lane;
    const float4 x4 = q < nf ? fours[q] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    const float x[4] = {x4.x, x4.y, x4.z, x4.w};
    u64 w[4];
    run = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        w[c] = near(x[c], reach) && (!least || kept(x[c], lo + q * 4 + c)) ? weight(x[c]) : 0;
        if (w[c] < floor_weight) w[c] = 0;
        run += w[c];
    }
    at = where_before + draw_warp_scan(run) - run;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (at <= target && target < at + w[c]) {
            p.tokens[row] = lo + q * 4 + c;
            if (p.probs) p.probs[row] = (float)((double)w[c] / (double)total);
        }
        at += w[c];
    }
}

}  // namespace b200

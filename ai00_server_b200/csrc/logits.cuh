// Rows of logits adjusted for the requests they belong to, and what a sampler reads of them: for row i and token t
//     l = seen(t) ? (l > 0 ? l / repetition : l * repetition) : l            seen: t is in the row's token history
//     l = l - said(t) * presence - weight(t) * frequency                     said: it is there at or behind `history_from`,
//                                                                            weight: sum of decay^age over those places, the newest token has age 0
//     l = l + bias(t);  l = -inf where the row's mask forbids t;  l = l / temperature
// (as the reference's sampler has them for a prompt; after generated tokens it decays presence too, which biases can state)
// written as they are, as softmax or as its logarithm.  Reference: penalties sampler/nucleus.rs:49-67, mask sampler/bnf.rs:37-40, bias run.rs:679-681,
// softmax run.rs:1179; the samplers that need whole rows are sampler/mirostat.rs:44-90 and sampler/typical.rs:70-131.
//
// Bound: a row is read and written once, 8 bytes a token for f32 rows (row of 65536: 0.5 MB; 512 rows 41 us at the copy rate); one row is latency.
// Shape: a cluster of eight or sixteen CTAs a row, the row in their registers (16 to 64 tokens a thread) between the only read and the only write; 32 tokens a
// thread and CTAs of 256 where there are many rows (512 rows of 65536: 56 us, with 16 tokens and CTAs of 512 70, with 32 and sixteen CTAs of 128 63), which settle their sums more quickly.
// Tokens go to the CTAs in stripes of 64, so that frequent tokens that are neighbours in a vocabulary spread over all of them.
//   * a history is added up in shared memory, a pair of words for each token of the CTA: decay^age in units of 2^-28, its lower 14 bits to one word
//     and the others to the other, so that neither overflows 31 bits (2^17 - 1 entries; of a longer history the newest count), no atomic has to answer,
//     and their order changes nothing.  An entry is off by half a unit at most, and one of less than that adds nothing: bit 31 of the first word then says
//     that its token counts, as that of the second does for a token that is in the history alone;
//   * one pass over the registers for the thread's maximum and its sum of exponentials, which are what the probabilities are made of; pairs are
//     combined over the CTA, and over the cluster in one exchange.
#pragma once
#include <cuda_bf16.h>

#include "operators.cuh"

namespace b200 {

template <typename E> __device__ __forceinline__ float logit_of(E v);
template <> __device__ __forceinline__ float logit_of<float>(float v) { return v; }
template <> __device__ __forceinline__ float logit_of<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float logit_of<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// four neighbouring logits on a boundary of their size
__device__ __forceinline__ float4 logits4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 logits4(const __half* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 logits4(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
}

constexpr unsigned LOGITS_SEEN = 1u << 31;        // flag in the upper word of a token that is in the history and does not count there
constexpr unsigned LOGITS_SAID = 1u << 31;        // flag in the lower word of one that counts with less than half a unit

// 2^x by the unit's instruction, good to 2^-22; what is below 2^-126 is zero.  (expf is eight instructions)
__device__ __forceinline__ float logits_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float logits_exp(float x) { return logits_exp2(x * 1.4426950408889634f); }

// sum of exponentials relative to a maximum.  NaN never becomes the maximum: it stays in the sum, and through it reaches the whole row
struct LogitsSum {
    float m, s;
    __device__ __forceinline__ void raise(float to) {
        if (to > m) {
            s *= expf(m - to);
            m = to;
        }
    }
};
template <int TH>
__device__ __forceinline__ LogitsSum logits_block(LogitsSum a, LogitsSum* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto whole = [](LogitsSum x) {
        x.raise(warp_max(x.m));
        x.s = warp_sum(x.s);
        return x;
    };
    a = whole(a);
    if (lane == 0) red[warp] = a;
    __syncthreads();
    return whole(lane < TH / 32 ? red[lane] : LogitsSum{-INFINITY, 0.f});
}

// TH: threads of a CTA, each with NV fours of tokens.  VEC: fours are neighbours, moved in one access; a row may start anywhere if it does so in both buffers
// alike: its fours then start up to three tokens in front of it.  Else a thread's tokens are TH apart
template <typename E, int TH, int NV, bool VEC>
__global__ void __launch_bounds__(TH, (NV <= 4 ? 1536 : (NV <= 8 ? 1024 : 512)) / TH) logits_kernel(const __grid_constant__ LogitsParams p) {
    extern __shared__ __align__(16) uint2 sums[];
    __shared__ LogitsSum red[TH / 32];
    __shared__ float2 stats[LOGITS_MOST_CTAS];
    const int tid = threadIdx.x, lg_ctas = p.ctas_log, ctas = 1 << lg_ctas, cta = blockIdx.x & (ctas - 1), row = blockIdx.x >> lg_ctas;
    const bool softmax = p.kind != LOGITS_ROWS;
    // no CTA writes to another's memory before all have started
    if (softmax) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_wait();
    const E* const in = reinterpret_cast<const E*>(p.in) + (size_t)(p.in_row ? p.in_row[row] : row) * p.in_stride;
    float* const out = p.out + (size_t)row * p.out_stride;
    // The CTA's tokens by place: stripes cta, cta + ctas, ... of the row with `ahead` places in front, so that fours lie on boundaries
    const int V = p.V, ahead = VEC ? (int)((uintptr_t)out / 4 & 3) : 0;
    const int stripes = (V + ahead + LOGITS_STRIPE - 1) / LOGITS_STRIPE, places = max((stripes - cta + ctas - 1) >> lg_ctas, 0) * LOGITS_STRIPE;
    // of the thread's c-th token in its k-th four: place, and the token itself (places are a whole number of stripes apart, so tokens are an even step apart)
    auto place = [&](int k, int c) { return VEC ? (k * TH + tid) * 4 + c : (k * 4 + c) * TH + tid; };
    constexpr int PER = VEC ? 4 : 1;
    int t_first = (((tid * PER / LOGITS_STRIPE) << lg_ctas) | cta) * LOGITS_STRIPE + tid * PER % LOGITS_STRIPE - ahead;
    const int t_step = ((TH * PER / LOGITS_STRIPE) << lg_ctas) * LOGITS_STRIPE;
    auto token = [&](int k, int c) { return VEC ? t_first + k * t_step + c : t_first + (k * 4 + c) * t_step; };
    // (worked out again in every part below: kept over all of them, tokens and what is known of them take more registers than the row)
    auto again = [&] { asm volatile("" : "+r"(t_first)); };
    auto there = [&](int t) { return t >= 0 && t < V; };
    auto whole = [&](int t) { return VEC && t >= 0 && t + 3 < V; };
    const float* const ctl = p.controls ? p.controls + (size_t)row * 5 : nullptr;
    const int h0 = p.hist_off ? p.hist_off[row] : 0, hn = p.hist_off ? p.hist_off[row + 1] - h0 : 0;
    const int b0 = p.bias_off ? p.bias_off[row] : 0, bn = p.bias_off ? p.bias_off[row + 1] - b0 : 0;
    float v[NV][4];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int t = token(k, 0);
        if (whole(t)) {
            const float4 x = logits4(in + t);
            v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int u = token(k, c);
                v[k][c] = there(u) ? logit_of<E>(in[u]) : -INFINITY;
            }
        }
    }
    again();

    // ---- lists, for as many of the CTA's tokens at a time as have their sums in shared memory ----
    if (hn > 0 || bn > 0) {
        // f(j, place of its token) for the entries of a list from `first` on that are among them
        auto each = [&](const int* tok, int first, int count, int s0, auto&& f) {
            constexpr int U = 4;                     // entries in flight (96 rows of 100003 with histories of 8000: 67 us, with one 75; with eight single rows take 15 % longer)
            for (int j0 = first + tid; j0 < count; j0 += TH * U) {
                unsigned t[U];
#pragma unroll
                for (int u = 0; u < U; ++u) t[u] = j0 + u * TH < count ? (unsigned)tok[j0 + u * TH] : 0xFFFFFFFFu;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const unsigned at = t[u] + (unsigned)ahead, st = at / LOGITS_STRIPE;
                    const int i = (int)((st >> lg_ctas) * LOGITS_STRIPE + at % LOGITS_STRIPE) - s0;
                    if (t[u] < (unsigned)V && (int)(st & (ctas - 1)) == cta && i >= 0 && i < p.list_tokens) f(j0 + u * TH, i);
                }
            }
        };
        // f(logit, sums) for those of the thread's tokens
        auto apply = [&](int s0, auto&& f) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int i = place(k, 0) - s0;
                if (VEC) {
                    if (i < 0 || i >= p.list_tokens) continue;
                    const uint4 a = *reinterpret_cast<const uint4*>(sums + i), b = *reinterpret_cast<const uint4*>(sums + i + 2);
                    if ((a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) == 0u) continue;
                    f(v[k][0], make_uint2(a.x, a.y)); f(v[k][1], make_uint2(a.z, a.w)); f(v[k][2], make_uint2(b.x, b.y)); f(v[k][3], make_uint2(b.z, b.w));
                    *reinterpret_cast<uint4*>(sums + i) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(sums + i + 2) = make_uint4(0, 0, 0, 0);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int e = place(k, c) - s0;
                        if (e < 0 || e >= p.list_tokens) continue;
                        const uint2 a = sums[e];
                        if ((a.x | a.y) == 0u) continue;
                        f(v[k][c], a);
                        sums[e] = make_uint2(0, 0);
                    }
                }
            }
        };
        // (what is not zero after `apply` is zeroed there: the sums start at zero every time)
        for (int i = tid * 2; i < p.list_tokens; i += TH * 2) *reinterpret_cast<uint4*>(sums + i) = make_uint4(0, 0, 0, 0);
        for (int s0 = 0; s0 < places; s0 += p.list_tokens) {
            if (hn > 0) {
                const float rep = ctl ? ctl[0] : 1.f, presence = ctl ? ctl[1] : 0.f, frequency = ctl ? ctl[2] : 0.f;
                const float lg = log2f(fminf(fmaxf(ctl ? ctl[3] : 1.f, 0.f), 1.f));
                const int from = p.hist_from ? p.hist_from[row] : 0;
                __syncthreads();
                auto flag = [](unsigned* word, unsigned bit) {
                    if (!(*reinterpret_cast<volatile unsigned*>(word) & bit)) atomicOr(word, bit);
                };
                each(p.hist + h0, max(0, hn - LOGITS_MAX_HISTORY), hn, s0, [&](int j, int i) {
                    if (j < from) return flag(&sums[i].y, LOGITS_SEEN);
                    const int age = hn - 1 - j;
                    const unsigned c = age == 0 ? 1u << 28 : (unsigned)(logits_exp2(lg * (float)age) * 268435456.f + 0.5f);      // (zero decay: nothing from the second newest on)
                    if (c == 0u) return flag(&sums[i].x, LOGITS_SAID);
                    if (c & 0x3FFFu) atomicAdd(&sums[i].x, c & 0x3FFFu);
                    if (c >> 14) atomicAdd(&sums[i].y, c >> 14);
                });
                __syncthreads();
                apply(s0, [&](float& l, uint2 a) {
                    if ((a.x | a.y) == 0u) return;
                    l = l > 0.f ? l / rep : l * rep;
                    const unsigned up = a.y & ~LOGITS_SEEN, low = a.x & ~LOGITS_SAID;
                    if (a.x | up) l -= presence + frequency * ((float)up * 0x1p-14f + (float)low * 0x1p-28f);
                });
            }
            if (bn > 0) {
                // a token listed twice has its last value: the highest place wins
                __syncthreads();
                each(p.bias_tok + b0, 0, bn, s0, [&](int j, int i) { atomicMax(&sums[i].x, (unsigned)j + 1u); });
                __syncthreads();
                apply(s0, [&](float& l, uint2 a) {
                    if (a.x) l += p.bias_val[b0 + a.x - 1u];
                });
            }
        }
    }

    // ---- mask and temperature ----
    again();
    const float temperature = ctl ? ctl[4] : 1.f;
    // a temperature that is not a positive number, or has no reciprocal, makes the row NaN
    const float over = 1.f / temperature, scale = temperature > 0.f && temperature < INFINITY && over < INFINITY ? over : __int_as_float(0x7fc00000);
    const int allow_row = p.allow ? (p.allow_row ? p.allow_row[row] : row) : -1;
    if (allow_row >= 0 && allow_row < p.allow_rows) {
        const unsigned* const allow = p.allow + (size_t)allow_row * p.words;
        if (VEC) {
            unsigned w[NV];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int t = token(k, 0);
                w[k] = 0u;
                if (t <= -4 || t >= V) continue;
                // four tokens from t on: of one word, or of two
                const int q = t >> 5;
                const unsigned lo = q >= 0 ? allow[q] : 0u, hi = (t & 31) > 28 && q + 1 < p.words ? allow[q + 1] : 0u;
                w[k] = __funnelshift_r(lo, hi, t & 31);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (!((w[k] >> c) & 1u)) v[k][c] = -INFINITY;
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                unsigned w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int t = token(k, c);
                    w[c] = there(t) ? allow[t / 32] >> (t % 32) : 0u;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (!(w[c] & 1u)) v[k][c] = -INFINITY;
            }
        }
    }
    auto put = [&](auto&& last) {
        again();
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int t = token(k, 0);
            if (whole(t)) {
                *reinterpret_cast<float4*>(out + t) = make_float4(last(v[k][0]), last(v[k][1]), last(v[k][2]), last(v[k][3]));
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int u = token(k, c);
                    if (there(u)) out[u] = last(v[k][c]);
                }
            }
        }
    };
    if (!softmax) {
        put([&](float l) { return l * scale; });
        return;
    }

    // ---- the thread's maximum and sum; from here on a probability is its exponential ----
    again();
    const bool probs = p.kind == LOGITS_PROBS;
    LogitsSum sum{-INFINITY, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (there(token(k, c))) v[k][c] *= scale;       // (what is not of the row stays -inf under every scale)
            sum.m = fmaxf(sum.m, v[k][c]);
        }
    const float mine = sum.m, shift = mine == -INFINITY ? 0.f : mine;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float e = logits_exp(v[k][c] - shift);
            sum.s += e;
            if (probs) v[k][c] = e;
        }

    // ---- the CTAs' statistics, in their order ----
    sum = logits_block<TH>(sum, red);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < ctas) {
        uint32_t remote;
        const uint32_t local = smem_u32(&stats[cta]);
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(tid));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(sum.m), "f"(sum.s) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    float top = -INFINITY, z = 0.f;
    for (int c = 0; c < ctas; ++c) top = fmaxf(top, stats[c].x);
    for (int c = 0; c < ctas; ++c) z += stats[c].y * (stats[c].x == -INFINITY ? 1.f : expf(stats[c].x - top));
    // nothing left of the row (its sums are zero, not NaN): probabilities 0, logarithms -inf
    const bool none = top == -INFINITY && z == 0.f;
    if (probs) {
        const float mul = none ? 0.f : (mine == -INFINITY ? 1.f : expf(mine - top)) / z;
        put([&](float e) { return e * mul; });
    } else {
        const float base = top == -INFINITY ? 0.f : top, sub = none ? 0.f : logf(z);
        put([&](float l) { return (l - base) - sub; });
    }
}

}  // namespace b200

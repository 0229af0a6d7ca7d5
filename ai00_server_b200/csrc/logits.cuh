// Rows of logits adjusted for the requests they belong to, and what a sampler reads of them: for row i and token t
//     l = seen(t) ? (l > 0 ? l / repetition : l * repetition) : l            seen: t is in the row's token history
//     l = l - said(t) * presence - weight(t) * frequency                     said: it is there at or behind `history_from`,
//                                                                            weight: sum of decay^age over those places, the newest token has age 0
//     l = l + bias(t);  l = -inf where the row's mask forbids t;  l = l / temperature
// written as they are, as softmax or as its logarithm.  Reference: penalties sampler/nucleus.rs:49-67, mask sampler/bnf.rs:37-40, bias run.rs:679-681,
// softmax run.rs:1179; the samplers that need whole rows are sampler/mirostat.rs:44-90 and sampler/typical.rs:70-131.
//
// Bound: a row is read and written once, 8 bytes a token for f32 rows (row of 65536: 0.5 MB; 512 rows 41 us at the copy rate); one row is latency.
// Shape: a cluster of eight CTAs a row, an eighth of the row each, which stays in shared memory between the only read and the only write.
//   * lists touch few tokens: they are applied to the slice in shared memory, not looked up by every element.  A history entry adds decay^age to its
//     token's sum in 32.32 fixed point (a word of fraction, whose carries go to a word of whole counts with the two flags), so that the order
//     of the atomics changes nothing; whoever then takes a token's counts first (exchange with zero) applies them;
//   * a CTA's maximum and its sum of exponentials go to the other seven in one exchange; a softmax entry is computed once, relative to the CTA's
//     maximum, and scaled by the row's factor on its way out.
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

// NaN is kept: it reaches the sum, and through it the whole row
__device__ __forceinline__ float logits_block(float v, float* red, const bool is_max) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = is_max ? warp_max(v) : warp_sum(v);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    float t = lane < LOGITS_THREADS / 32 ? red[lane] : (is_max ? -INFINITY : 0.f);
    return is_max ? warp_max(t) : warp_sum(t);
}

constexpr unsigned LOGITS_SEEN = 1u << 31, LOGITS_SAID = 1u << 30, LOGITS_COUNT = LOGITS_SAID - 1;

template <typename E>
__global__ void __cluster_dims__(LOGITS_CTAS, 1, 1) __launch_bounds__(LOGITS_THREADS) logits_kernel(const __grid_constant__ LogitsParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float red[32];
    __shared__ float2 stats[LOGITS_CTAS];
    const int tid = threadIdx.x, cta = blockIdx.x % LOGITS_CTAS, row = blockIdx.x / LOGITS_CTAS;
    const bool softmax = p.kind != LOGITS_ROWS;
    // no CTA writes to another's memory before all have started
    if (softmax) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_wait();
    const int t0 = min(cta * p.slice, p.V), n = min(p.slice, p.V - t0);
    const E* const in = reinterpret_cast<const E*>(p.in) + (size_t)(p.in_row ? p.in_row[row] : row) * p.in_stride + t0;
    float* const out = p.out + (size_t)row * p.out_stride + t0;
    float* const buf = p.buffered ? reinterpret_cast<float*>(smem_raw) : out;
    unsigned* const acc_lo = reinterpret_cast<unsigned*>(smem_raw + (p.buffered ? (size_t)p.slice * 4 : 0));
    unsigned* const acc_hi = acc_lo + p.sub;

    float rep = 1.f, presence = 0.f, frequency = 0.f, decay = 1.f, temperature = 1.f;
    if (p.controls) {
        const float* c = p.controls + (size_t)row * 5;
        rep = c[0]; presence = c[1]; frequency = c[2]; decay = c[3]; temperature = c[4];
    }
    const int h0 = p.hist_off ? p.hist_off[row] : 0, hn = p.hist_off ? p.hist_off[row + 1] - h0 : 0;
    const int b0 = p.bias_off ? p.bias_off[row] : 0, bn = p.bias_off ? p.bias_off[row + 1] - b0 : 0;
    const int allow_row = p.allow ? (p.allow_row ? p.allow_row[row] : row) : -1;
    const unsigned* const allow = allow_row >= 0 && allow_row < p.allow_rows ? p.allow + (size_t)allow_row * p.words : nullptr;
    // a temperature that is not a positive number makes the row NaN
    const float scale = temperature > 0.f && temperature < INFINITY ? 1.f / temperature : __int_as_float(0x7fc00000);

    const bool lists = hn > 0 || bn > 0;
    // one element of the row after its lists: mask and temperature
    auto finish = [&](float l, int i) {
        const int t = t0 + i;
        if (allow && !((allow[t >> 5] >> (t & 31)) & 1u)) l = -INFINITY;
        return l * scale;
    };
    float mx = -INFINITY;
    if (p.vec) {
        constexpr int U = 8;
        for (int i0 = tid * 4; i0 < n; i0 += LOGITS_THREADS * 4 * U) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * LOGITS_THREADS * 4;
                if (i + 3 < n) v[u] = logits4(in + i);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * LOGITS_THREADS * 4;
                if (i >= n) break;
                if (i + 3 < n) {
                    if (!lists) {
                        if (allow) {
                            const unsigned w = allow[(t0 + i) >> 5] >> ((t0 + i) & 31);       // four tokens of a word: i and t0 are multiples of 4
                            if (!(w & 1u)) v[u].x = -INFINITY;
                            if (!(w & 2u)) v[u].y = -INFINITY;
                            if (!(w & 4u)) v[u].z = -INFINITY;
                            if (!(w & 8u)) v[u].w = -INFINITY;
                        }
                        v[u].x *= scale; v[u].y *= scale; v[u].z *= scale; v[u].w *= scale;
                        mx = fmaxf(fmaxf(fmaxf(mx, v[u].x), fmaxf(v[u].y, v[u].z)), v[u].w);
                    }
                    *reinterpret_cast<float4*>(buf + i) = v[u];
                } else {
                    for (int k = i; k < n; ++k) {
                        float l = logit_of<E>(in[k]);
                        if (!lists) { l = finish(l, k); mx = fmaxf(mx, l); }
                        buf[k] = l;
                    }
                }
            }
        }
    } else {
        for (int i = tid; i < n; i += LOGITS_THREADS) {
            float l = logit_of<E>(in[i]);
            if (!lists) { l = finish(l, i); mx = fmaxf(mx, l); }
            buf[i] = l;
        }
    }
    if (lists) {
        const int from = p.hist_from ? p.hist_from[row] : 0;
        const float lg = log2f(fminf(fmaxf(decay, 0.f), 1.f));
        for (int s0 = 0; s0 < n; s0 += p.sub) {
            const int sn = min(p.sub, n - s0);
            const unsigned first = (unsigned)(t0 + s0);
            if (hn > 0) {
                __syncthreads();
                for (int j = tid; j < hn; j += LOGITS_THREADS) {
                    const unsigned e = (unsigned)p.hist[h0 + j] - first;
                    if (e < (unsigned)sn) acc_lo[e] = acc_hi[e] = 0u;
                }
                __syncthreads();
                for (int j = tid; j < hn; j += LOGITS_THREADS) {
                    const unsigned e = (unsigned)p.hist[h0 + j] - first;
                    if (e >= (unsigned)sn) continue;
                    unsigned hi = LOGITS_SEEN;
                    if (j >= from) {
                        hi |= LOGITS_SAID;
                        const int age = hn - 1 - j;
                        const float w = age == 0 ? 1.f : exp2f(lg * (float)age);        // (zero decay: 0 from the second newest on)
                        if (w >= 1.f) {
                            atomicAdd(&acc_hi[e], 1u);
                        } else {
                            const unsigned c = (unsigned)(w * 4294967296.f);
                            if (atomicAdd(&acc_lo[e], c) + c < c) atomicAdd(&acc_hi[e], 1u);
                        }
                    }
                    atomicOr(&acc_hi[e], hi);
                }
                __syncthreads();
                for (int j = tid; j < hn; j += LOGITS_THREADS) {
                    const unsigned e = (unsigned)p.hist[h0 + j] - first;
                    if (e >= (unsigned)sn || acc_hi[e] == 0u) continue;
                    const unsigned hi = atomicExch(&acc_hi[e], 0u);
                    if (hi == 0u) continue;
                    float l = buf[s0 + e];
                    l = l > 0.f ? l / rep : l * rep;
                    if (hi & LOGITS_SAID) l -= presence + frequency * ((float)(hi & LOGITS_COUNT) + (float)acc_lo[e] * 0x1p-32f);
                    buf[s0 + e] = l;
                }
            }
            if (bn > 0) {
                // a token listed twice has its last value: the highest place wins
                __syncthreads();
                for (int j = tid; j < bn; j += LOGITS_THREADS) {
                    const unsigned e = (unsigned)p.bias_tok[b0 + j] - first;
                    if (e < (unsigned)sn) acc_lo[e] = 0u;
                }
                __syncthreads();
                for (int j = tid; j < bn; j += LOGITS_THREADS) {
                    const unsigned e = (unsigned)p.bias_tok[b0 + j] - first;
                    if (e < (unsigned)sn) atomicMax(&acc_lo[e], (unsigned)j + 1u);
                }
                __syncthreads();
                for (int j = tid; j < bn; j += LOGITS_THREADS) {
                    const unsigned e = (unsigned)p.bias_tok[b0 + j] - first;
                    if (e < (unsigned)sn && acc_lo[e] == (unsigned)j + 1u) buf[s0 + e] += p.bias_val[b0 + j];
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < n; i += LOGITS_THREADS) {
            const float l = finish(buf[i], i);
            buf[i] = l;
            mx = fmaxf(mx, l);
        }
    }
    if (!softmax) {
        if (!p.buffered) return;
        __syncthreads();
        if (p.vec) {
            for (int i = tid * 4; i < n; i += LOGITS_THREADS * 4) {
                if (i + 3 < n) *reinterpret_cast<float4*>(out + i) = *reinterpret_cast<const float4*>(buf + i);
                else for (int k = i; k < n; ++k) out[k] = buf[k];
            }
        } else {
            for (int i = tid; i < n; i += LOGITS_THREADS) out[i] = buf[i];
        }
        return;
    }
    mx = logits_block(mx, red, true);          // (its barriers also stand between the writes to the slice and its readers)
    const float shift = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    const bool probs = p.kind == LOGITS_PROBS;
    for (int i = tid; i < n; i += LOGITS_THREADS) {
        const float e = expf(buf[i] - shift);
        sum += e;
        if (probs) buf[i] = e;
    }
    sum = logits_block(sum, red, false);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < LOGITS_CTAS) {
        uint32_t remote;
        const uint32_t local = smem_u32(&stats[cta]);
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(tid));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(mx), "f"(sum) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < LOGITS_CTAS; ++c) top = fmaxf(top, stats[c].x);
    float z = 0.f;
#pragma unroll
    for (int c = 0; c < LOGITS_CTAS; ++c) z += stats[c].y * (stats[c].x == -INFINITY ? 1.f : expf(stats[c].x - top));
    // nothing left of the row (its sums are zero, not NaN): probabilities 0, logarithms -inf
    const bool none = top == -INFINITY && z == 0.f;
    const float mul = probs ? (none ? 0.f : (mx == -INFINITY ? 1.f : expf(mx - top)) / z) : 1.f;
    const float sub = probs || none ? 0.f : logf(z), base = probs || none ? 0.f : top;
    auto last = [&](float v) { return probs ? v * mul : (v - base) - sub; };
    if (p.vec) {
        for (int i = tid * 4; i < n; i += LOGITS_THREADS * 4) {
            if (i + 3 < n) {
                float4 v = *reinterpret_cast<const float4*>(buf + i);
                v.x = last(v.x); v.y = last(v.y); v.z = last(v.z); v.w = last(v.w);
                *reinterpret_cast<float4*>(out + i) = v;
            } else {
                for (int k = i; k < n; ++k) out[k] = last(buf[k]);
            }
        }
    } else {
        for (int i = tid; i < n; i += LOGITS_THREADS) out[i] = last(buf[i]);
    }
}

}  // namespace b200

// Low-rank adapters of many requests beside their shared projection: token t of a request with adapter a adds to the projection's output
//     out[t, n] = base[t, n] + scale[a] * sum_r S[t, r] B[a][n, r],      S[t, r] = sum_k x[t, k] A[a][r, k]
// and a token without one (an index that names no adapter) keeps its base.  The reference blends such pairs into the weights when a model is loaded
// (lib.rs:466-485); here they stay apart, so that the requests of a batch can have different ones.
//
// Tokens are taken in groups that share an adapter (tokens of a batch lie in any order).  Bound: a decode batch reads every adapter of its requests
// once, 2 R (K + N) bytes each, beside rows of a few KB, so what counts is how soon the two dependent products are through.
//
// adapter_few_kernel: a cluster of eight CTAs takes eight tokens of one adapter.  Each CTA has an eighth of k for the first product and an eighth of n for
// the second; between them the eight partial S (R x 8 floats) go to every CTA of the cluster in one exchange, so that nothing but x, A, B, base and out
// touches memory.  Both products are m16n8k16 with the adapter's rows as M and the eight tokens as N: a lane reads 16 bytes of a row at a time, which
// is two steps of k for it (the order of k within 32 is the same permutation on both sides of a product, so it is never undone).
// A group of a single token (every request with its own adapter) goes without the tensor cores, of which it would use one column in eight: 448 units of 32
// outputs at rank 32 for each of 64 tokens are 12400 cycles of m16n8k16 and 4100 of f32 multiply-adds.
// S is f32; the second product takes it as two or three 16-bit parts, enough for the output's type, scaled per token by a power of two.
#pragma once
#include <cuda_bf16.h>

#include "operators.cuh"

namespace b200 {

template <typename E> struct AdpType;
template <> struct AdpType<__half> {
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        mma_16816(c, a0, a1, a2, a3, b0, b1);
    }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
};
template <> struct AdpType<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
};

// 16-bit parts of S in the second product: what they leave out is far below half a step of the output's type (two parts of f16 leave 2^-22, of bf16 2^-17,
// three of bf16 2^-25)
template <typename E, typename O> struct AdpParts { static constexpr int N = 2; };
template <> struct AdpParts<__nv_bfloat16, float> { static constexpr int N = 3; };

__device__ __forceinline__ uint4 adp_ld16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

// four neighbours of a row as they lie in memory: widened where they are used, or a load would be waited for where it is made
template <typename O> struct AdpRaw {
    using Four = uint2;
    static __device__ __forceinline__ void widen(const uint2& r, float (&v)[4]) {
        const O* const e = reinterpret_cast<const O*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = AdpType<O>::widen(e[i]);
    }
};
template <> struct AdpRaw<float> {
    using Four = float4;
    static __device__ __forceinline__ void widen(const float4& r, float (&v)[4]) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
};
__device__ __forceinline__ void adp_store4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <typename O>
__device__ __forceinline__ void adp_store4(O* p, const float (&v)[4]) {
    uint2 u;
    O* e = reinterpret_cast<O*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = AdpType<O>::round(v[i]);
    *reinterpret_cast<uint2*>(p) = u;
}
__device__ __forceinline__ float adp_widen(float v) { return v; }
__device__ __forceinline__ float adp_widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float adp_widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void adp_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void adp_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void adp_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// eight 16-bit numbers, widened
__device__ __forceinline__ void adp_widen8(const uint4& u, float (&f)[8], __half) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = v.x; f[2 * i + 1] = v.y;
    }
}
__device__ __forceinline__ void adp_widen8(const uint4& u, float (&f)[8], __nv_bfloat16) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <typename E>
__device__ __forceinline__ float adp_dot8(const uint4& a, const float (&x)[8], float s) {
    float f[8];
    adp_widen8(a, f, E{});
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(f[i], x[i], s);
    return s;
}

// the activations that projections with adapters end in (gate, channel-mix key and receptance), as the projection's own epilogue computes them: tokens without
// an adapter have the same bits beside those with one
__device__ __forceinline__ float adp_act(float v, int act) {
    if (act == ACT_RELU2) {
        const float r = fmaxf(v, 0.f);
        return r * r;
    }
    const float s = sigmoidf_(v);
    return act == ACT_SILU ? v * s : s;
}

struct AdpGroup {
    int tok[ADP_TOK];            // tokens, -1 behind the last
    int adapter;                 // -1: none
    int found;
    int alone;                   // a single token
};

// group `want` of a call of up to ADP_INLINE tokens, found by every CTA for itself: a group starts at a token whose number of earlier tokens with
// the same adapter is a multiple of ADP_TOK, groups count in the order of their first tokens.  Up to 32 tokens are one warp's work and one barrier
__device__ __forceinline__ void adapter_find_group(const AdapterParams& p, const int want, AdpGroup& g, int* s_idx, int* s_cnt) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool one = p.tokens <= 32;
    const unsigned before = (1u << lane) - 1u;
    int id = -2;
    if (tid < p.tokens) {
        id = p.index[tid];
        if (id < 0 || id >= p.adapters) id = p.copy && !(p.finish && id == -2) ? -1 : -2;
    }
    if (one) {
        if (warp == 0) {
            const int rank = __popc(__match_any_sync(0xffffffffu, id) & before);
            const bool start = id >= -1 && rank % ADP_TOK == 0;
            const unsigned starts = __ballot_sync(0xffffffffu, start), mine = __ballot_sync(0xffffffffu, start && __popc(starts & before) == want);
            const int from = mine ? __ffs(mine) - 1 : 0;
            const int adapter = __shfl_sync(0xffffffffu, id, from), first = __shfl_sync(0xffffffffu, rank, from);
            if (lane < ADP_TOK) g.tok[lane] = -1;
            __syncwarp();
            if (mine && id == adapter && rank >= first && rank < first + ADP_TOK) g.tok[rank - first] = lane;
            if (lane == 0) {
                g.adapter = adapter;
                g.found = mine != 0;
            }
        }
        __syncthreads();
        return;
    }
    s_idx[tid] = id;
    if (tid < ADP_TOK) g.tok[tid] = -1;
    if (tid == 0) g.found = 0;
    __syncthreads();
    int rank = __popc(__match_any_sync(0xffffffffu, id) & before);
    if (warp * 32 < p.tokens)
        for (int w = 0; w < warp * 32; w += 4) {
            const int4 v = *reinterpret_cast<const int4*>(s_idx + w);
            rank += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
        }
    const bool start = id >= -1 && rank % ADP_TOK == 0;
    const unsigned starts = __ballot_sync(0xffffffffu, start);
    if (lane == 0) s_cnt[warp] = __popc(starts);
    __syncthreads();
    int number = __popc(starts & before);
    for (int w = 0; w < warp; ++w) number += s_cnt[w];
    if (start && number == want) {
        g.adapter = id;
        g.found = rank + 1;
    }
    __syncthreads();
    if (g.found && id >= -1 && id == g.adapter && rank >= g.found - 1 && rank < g.found - 1 + ADP_TOK) g.tok[rank - (g.found - 1)] = tid;
    __syncthreads();
}

// MANY: registers for four CTAs on an SM instead of three, where a call has more than three for each (64 tokens with adapters of rank 32 to 14336 outputs, 512
// CTAs: 20 us, with three 30; 16 tokens of four projections, 320 CTAs, stay at three: 7.7 us, with four 8.5)
// FIN: parts may end in an activation, as f32 rows or as the operand of the next projection
template <typename E, typename O, bool MANY, bool FIN>
__global__ void __cluster_dims__(ADP_CTAS, 1, 1) __launch_bounds__(ADP_THREADS, MANY ? 4 : 3) adapter_few_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ AdpGroup g;
    __shared__ __align__(16) int s_idx[ADP_THREADS];
    __shared__ int s_cnt[ADP_WARPS];
    __shared__ float s_back[ADP_TOK];
    constexpr int NP = AdpParts<E, O>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = lane >> 2, quad = lane & 3;
    const int cta = blockIdx.x % ADP_CTAS, want = blockIdx.x / ADP_CTAS;
    const AdapterPart& q = p.part[blockIdx.y];
    pdl_wait();
    pdl_launch_dependents();                     // (a projection behind this one then has its first weights when its turn comes)
    if (p.plan.base) {
        if (want >= p.plan.count()[0]) return;
        const int4 gr = p.plan.group()[want];
        if (tid < ADP_TOK) g.tok[tid] = tid < gr.z ? p.plan.place()[gr.y + tid] : -1;
        if (tid == 0) {
            g.adapter = gr.x;
            g.alone = gr.w;
        }
        __syncthreads();
    } else {
        adapter_find_group(p, want, g, s_idx, s_cnt);
        if (!g.found) return;
        if (tid == 0) g.alone = g.tok[1] < 0;
        __syncthreads();
    }
    const int adapter = g.adapter, K = q.K, N = q.N;
    O* const out = reinterpret_cast<O*>(q.out);
    const O* const base = reinterpret_cast<const O*>(q.base);
    // outputs n (.. n + 3) of token t
    auto put = [&](int t, int n, float v) {
        if constexpr (FIN) {
            if (q.fin) v = adp_act(v, q.act);
            if (q.fin >= ADP_A16) {
                __half hi = __float2half_rn(v), lo;
                if (q.fin == ADP_A16_SPLIT) {
                    split_h(v, hi, lo);
                    reinterpret_cast<__half*>(q.out)[a16_index(t + 16, n, q.out_th)] = lo;
                } else {
                    hi = f2h_sat(v);
                }
                reinterpret_cast<__half*>(q.out)[a16_index(t, n, q.out_th)] = hi;
                return;
            }
        }
        adp_put(out + (size_t)t * q.out_stride + n, v);
    };
    auto put4 = [&](int t, int n, float (&v)[4]) {
        if constexpr (FIN) {
            if (q.fin) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = adp_act(v[i], q.act);
            }
            if (q.fin >= ADP_A16) {
                uint2 hi, lo;
                if (q.fin == ADP_A16_SPLIT) {
                    split_pack_h2(v[0], v[1], hi.x, lo.x);
                    split_pack_h2(v[2], v[3], hi.y, lo.y);
                    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(q.out) + a16_index(t + 16, n, q.out_th)) = lo;
                } else {
                    hi = make_uint2(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]));
                }
                *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(q.out) + a16_index(t, n, q.out_th)) = hi;
                return;
            }
        }
        adp_store4(out + (size_t)t * q.out_stride + n, v);
    };
    const E *A = nullptr, *B = nullptr;
    int R = 0;
    float scale = 0.f;
    if (adapter >= 0) {
        if (q.table) {
            const AdapterEntry e = q.table[adapter];
            A = reinterpret_cast<const E*>(e.a); B = reinterpret_cast<const E*>(e.b); R = e.rank; scale = e.scale;
        } else {
            R = q.R;
            A = reinterpret_cast<const E*>(q.a) + (size_t)adapter * R * K;
            B = reinterpret_cast<const E*>(q.b) + (size_t)adapter * N * R;
            scale = p.scale[adapter];
        }
    }
    const int units = (N + 31) / 32, u0 = (int)((long long)units * cta / ADP_CTAS), u1 = (int)((long long)units * (cta + 1) / ADP_CTAS);
    if (R == 0) {
        if (!p.copy || (q.base == q.out && q.base_stride == q.out_stride)) return;
        for (int j = warp; j < ADP_TOK; j += ADP_WARPS) {
            const int t = g.tok[j];
            if (t < 0) continue;
            for (int n = u0 * 32 + lane; n < min(u1 * 32, N); n += 32)
                put(t, n, base ? adp_widen(base[(size_t)t * q.base_stride + n]) : 0.f);
        }
        return;
    }
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    if (g.alone) {
        // ---- one token ----
        const int tok = g.tok[0];
        float* const part = reinterpret_cast<float*>(smem_raw);                  // [warp][R]
        float* const all = part + ADP_WARPS * p.rank;                            // [CTA][R]
        float* const sum = all + ADP_CTAS * p.rank;                              // [R rounded to 32]
        const E* const x = reinterpret_cast<const E*>(q.x);
        auto xat = [&](int k, int lo) { return q.x_a16 ? x + a16_index(tok + lo, k, q.x_th) : x + (size_t)(tok + lo) * q.x_stride + k; };
        const int nk = (K + 31) / 32, c0 = (int)((long long)nk * cta / ADP_CTAS), c1 = (int)((long long)nk * (cta + 1) / ADP_CTAS);
        for (int m0 = 0; m0 < R; m0 += 64) {
            float acc[8] = {};                       // ranks m0 + row + 8 i
            for (int c = c0 + warp; c < c1; c += ADP_WARPS) {
                const int k = c * 32 + quad * 8;
                if (k >= K) continue;
                uint4 a[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[i] = make_uint4(0, 0, 0, 0);
                    if (m0 + i * 8 < R) a[i] = adp_ld16(A + (size_t)(m0 + i * 8 + row) * K + k);
                }
                float xf[8];
                adp_widen8(adp_ld16(xat(k, 0)), xf, E{});
                if (q.x_lo) {                        // (hi + lo is exact in f32)
                    float xl[8];
                    adp_widen8(adp_ld16(xat(k, q.x_lo)), xl, E{});
#pragma unroll
                    for (int i = 0; i < 8; ++i) xf[i] += xl[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = adp_dot8<E>(a[i], xf, acc[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 1);
                acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 2);
                if (quad == 0 && m0 + i * 8 < R) part[warp * R + m0 + i * 8 + row] = acc[i];
            }
        }
        __syncthreads();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // every CTA of the cluster has started
        for (int r = tid; r < R; r += ADP_THREADS) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < ADP_WARPS; ++w) v += part[w * R + r];
            const uint32_t local = smem_u32(all + cta * R + r);
#pragma unroll
            for (int c = 0; c < ADP_CTAS; ++c) {
                uint32_t remote;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(c));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
            }
        }
        uint4 w[4];
        auto load_b = [&](int u, int r0) {           // four rows of B for a lane, 32 ranks at a time
            const int n = u * 32 + row * 4, r = r0 + quad * 8;
            const E* const from = B + (size_t)n * R + r;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = make_uint4(0, 0, 0, 0);
                if (u < u1 && n + i < N && r < R) w[i] = adp_ld16(from + (size_t)i * R);
            }
        };
        load_b(u0 + warp, 0);
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int r = tid; r < ((R + 31) & ~31); r += ADP_THREADS) {
            float v = 0.f;
            if (r < R)
#pragma unroll
                for (int c = 0; c < ADP_CTAS; ++c) v += all[c * R + r];
            sum[r] = v * scale;
        }
        __syncthreads();
        for (int u = u0 + warp; u < u1; u += ADP_WARPS) {
            const int n = u * 32 + lane;             // the column that this lane ends up with
            const bool ok = n < N;
            const O y = ok && base ? base[(size_t)tok * q.base_stride + n] : O(0.f);
            float acc[4] = {};
            for (int r0 = 0; r0 < R; r0 += 32) {
                float s[8];
                *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sum + r0 + quad * 8);
                *reinterpret_cast<float4*>(s + 4) = *reinterpret_cast<const float4*>(sum + r0 + quad * 8 + 4);
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = w[i];
                if (r0 + 32 < R) load_b(u, r0 + 32);
                else load_b(u + ADP_WARPS, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = adp_dot8<E>(v[i], s, acc[i]);
            }
            // four columns over four lanes: each lane keeps its own
            const bool up = quad & 2, odd = quad & 1;
            const float k0 = (up ? acc[2] : acc[0]) + __shfl_xor_sync(0xffffffffu, up ? acc[0] : acc[2], 2);
            const float k1 = (up ? acc[3] : acc[1]) + __shfl_xor_sync(0xffffffffu, up ? acc[1] : acc[3], 2);
            const float d = (odd ? k1 : k0) + __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 1);
            if (ok) put(tok, n, adp_widen(y) + d);
        }
        return;
    }

    const int R8 = R * ADP_TOK, Rp = (R + 31) & ~31, pitch = Rp + 8;
    float* const part = reinterpret_cast<float*>(smem_raw);                      // [warp][R][8]: partial sums of the CTA's warps
    float* const all = part + (size_t)ADP_WARPS * p.rank * ADP_TOK;                 // [CTA][R][8]
    E* const frag = reinterpret_cast<E*>(all + (size_t)ADP_CTAS * p.rank * ADP_TOK);        // [part][token][pitch]

    // four rows of B for a lane, 32 ranks at a time
    auto load_b = [&](int u, int r0, uint4 (&w)[4]) {
        const int n = u * 32 + row * 4, r = r0 + quad * 8;
        const E* const from = B + (size_t)n * R + r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = make_uint4(0, 0, 0, 0);
            if (u < u1 && n + i < N && r < R) w[i] = adp_ld16(from + (size_t)i * R);
        }
    };

    // ---- S: this CTA's k, a run of 32 of them to a warp at a time ----
    {
        const int tok = g.tok[row];
        const E* const x = reinterpret_cast<const E*>(q.x);
        auto xat = [&](int k, int lo) {
            return q.x_a16 ? x + a16_index(tok + lo, k, q.x_th) : x + (size_t)(tok + lo) * q.x_stride + k;
        };
        const int nk = (K + 31) / 32, c0 = (int)((long long)nk * cta / ADP_CTAS), c1 = (int)((long long)nk * (cta + 1) / ADP_CTAS);
        for (int m0 = 0; m0 < R; m0 += 64) {
            float acc[4][4] = {};
            for (int c = c0 + warp; c < c1; c += ADP_WARPS) {
                const int k = c * 32 + quad * 8;
                const bool in = k < K;
                uint4 xv = make_uint4(0, 0, 0, 0), xl = xv, lo[4], hi[4];
                if (in && tok >= 0) {
                    xv = adp_ld16(xat(k, 0));
                    if (q.x_lo) xl = adp_ld16(xat(k, q.x_lo));
                }
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int r = m0 + m * 16 + row;
                    lo[m] = hi[m] = make_uint4(0, 0, 0, 0);
                    if (in && r < R) lo[m] = adp_ld16(A + (size_t)r * K + k);
                    if (in && r + 8 < R) hi[m] = adp_ld16(A + (size_t)(r + 8) * K + k);
                }
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    AdpType<E>::mma(acc[m], lo[m].x, hi[m].x, lo[m].y, hi[m].y, xv.x, xv.y);
                    AdpType<E>::mma(acc[m], lo[m].z, hi[m].z, lo[m].w, hi[m].w, xv.z, xv.w);
                    if (q.x_lo) {
                        AdpType<E>::mma(acc[m], lo[m].x, hi[m].x, lo[m].y, hi[m].y, xl.x, xl.y);
                        AdpType<E>::mma(acc[m], lo[m].z, hi[m].z, lo[m].w, hi[m].w, xl.z, xl.w);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int r = m0 + m * 16 + row;
                float* const d = part + (size_t)warp * R8 + r * ADP_TOK + quad * 2;
                if (r < R) *reinterpret_cast<float2*>(d) = make_float2(acc[m][0], acc[m][1]);
                if (r + 8 < R) *reinterpret_cast<float2*>(d + 8 * ADP_TOK) = make_float2(acc[m][2], acc[m][3]);
            }
        }
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");          // every CTA of the cluster has started
    for (int i = tid * 4; i < R8; i += ADP_THREADS * 4) {
        float4 s = *reinterpret_cast<const float4*>(part + i);
#pragma unroll
        for (int w = 1; w < ADP_WARPS; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(part + (size_t)w * R8 + i);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const uint32_t local = smem_u32(all + (size_t)cta * R8 + i);
#pragma unroll
        for (int c = 0; c < ADP_CTAS; ++c) {
            uint32_t remote;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(c));
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(s.x), "f"(s.y), "f"(s.z), "f"(s.w) : "memory");
        }
    }
    uint4 w[4];
    load_b(u0 + warp, 0, w);
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

    // ---- S of a token (one to a warp): sum over the CTAs in their order, scale, 16-bit parts relative to the token's largest ----
    {
        float v[ADP_MAX_RANK / 32], top = 0.f;
#pragma unroll
        for (int i = 0; i < ADP_MAX_RANK / 32; ++i) {
            const int r = i * 32 + lane;
            v[i] = 0.f;
            if (r < R) {
#pragma unroll
                for (int c = 0; c < ADP_CTAS; ++c) v[i] += all[(size_t)c * R8 + r * ADP_TOK + warp];
                v[i] *= scale;
            }
            top = fmaxf(top, fabsf(v[i]));
        }
        top = warp_max(top);
        // a power of two near the largest (its exponent field alone; the smallest and the largest few stay within normal numbers)
        const unsigned ex = min(max((__float_as_uint(top) >> 23) & 255u, 2u), 252u);
        const float down = __uint_as_float((254u - ex) << 23), back = __uint_as_float(ex << 23);
        if (lane == 0) s_back[warp] = back;
#pragma unroll
        for (int i = 0; i < ADP_MAX_RANK / 32; ++i) {
            const int r = i * 32 + lane;
            if (r < Rp) {
                float left = v[i] * down;
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const E h = AdpType<E>::round(left);
                    const float w = AdpType<E>::widen(h);
                    frag[((size_t)k * ADP_TOK + warp) * pitch + r] = h;
                    left = fabsf(w) < INFINITY ? left - w : 0.f;
                }
            }
        }
    }
    __syncthreads();

    // ---- out: 32 columns to a warp at a time, four neighbours of them to a lane ----
    const int ta = g.tok[quad * 2], tb = g.tok[quad * 2 + 1];
    const float backa = s_back[quad * 2], backb = s_back[quad * 2 + 1];
    for (int u = u0 + warp; u < u1; u += ADP_WARPS) {
        const int n = u * 32 + row * 4;
        const bool four = q.vec && n + 3 < N;
        typename AdpRaw<O>::Four ya{}, yb{};             // base of the lane's two tokens
        if (base && four) {
            if (ta >= 0) ya = *reinterpret_cast<const typename AdpRaw<O>::Four*>(base + (size_t)ta * q.base_stride + n);
            if (tb >= 0) yb = *reinterpret_cast<const typename AdpRaw<O>::Four*>(base + (size_t)tb * q.base_stride + n);
        }
        float acc[2][4] = {};
        for (int r0 = 0; r0 < R; r0 += 32) {
            uint4 v[4];
            if (r0 + 32 < R) load_b(u, r0 + 32, v);
            else load_b(u + ADP_WARPS, 0, v);
            const int r = r0 + quad * 8;
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                const uint4 s = adp_ld16(frag + ((size_t)k * ADP_TOK + row) * pitch + r);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    AdpType<E>::mma(acc[i], w[2 * i].x, w[2 * i + 1].x, w[2 * i].y, w[2 * i + 1].y, s.x, s.y);
                    AdpType<E>::mma(acc[i], w[2 * i].z, w[2 * i + 1].z, w[2 * i].w, w[2 * i + 1].w, s.z, s.w);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = v[i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int t = h ? tb : ta;
            if (t < 0) continue;
            const float back = h ? backb : backa;
            const float d[4] = {acc[0][h] * back, acc[0][2 + h] * back, acc[1][h] * back, acc[1][2 + h] * back};
            const O* const y = base ? base + (size_t)t * q.base_stride + n : nullptr;
            if (four) {
                float v[4];
                AdpRaw<O>::widen(h ? yb : ya, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += d[i];
                put4(t, n, v);
            } else {
                for (int i = 0; i < 4 && n + i < N; ++i) put(t, n + i, (y ? adp_widen(y[i]) : 0.f) + d[i]);
            }
        }
    }
}

inline size_t adapter_few_smem(int R, int elem_parts) {
    return (size_t)(ADP_WARPS + ADP_CTAS) * R * ADP_TOK * 4 + (size_t)elem_parts * ADP_TOK * (((R + 31) & ~31) + 8) * 2;
}

// Tokens of a longer call ordered by adapter, its groups and its tiles: one CTA, a counting sort.  Where a token lands within its adapter depends on the order of
// the atomics, its result does not: columns and rows of a product do not see each other, and a token goes alone only where its adapter has no other
// (the one left over from groups of eight could be any).
__global__ void __launch_bounds__(ADP_PLAN_THREADS) adapter_plan_kernel(const __grid_constant__ AdapterParams p) {
    constexpr int KEPT = 8192;                   // tokens whose bins are kept between the two passes
    __shared__ int s_count[ADP_MAX_ADAPTERS + 1], s_first[ADP_MAX_ADAPTERS + 1], s_warp[3][ADP_PLAN_THREADS / 32], s_total[3];
    __shared__ short s_bin[KEPT];
    pdl_launch_dependents();                     // (they wait for this kernel's end before they read anything)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = p.adapters + (p.copy ? 1 : 0);
    for (int i = tid; i < bins; i += ADP_PLAN_THREADS) s_count[i] = 0;
    if (tid < 3) s_total[tid] = 0;
    pdl_wait();
    __syncthreads();
    auto bin_of = [&](int t) {
        const int id = p.index[t];
        return id >= 0 && id < p.adapters ? id : (p.copy ? p.adapters : -1);
    };
    for (int t0 = 0; t0 < p.tokens; t0 += ADP_PLAN_THREADS) {
        const int b = t0 + tid < p.tokens ? bin_of(t0 + tid) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, b);
        if (b >= 0 && lane == __ffs(same) - 1) atomicAdd(&s_count[b], __popc(same));
        if (t0 + tid < KEPT) s_bin[t0 + tid] = (short)b;
    }
    __syncthreads();
    // exclusive sums over the bins of tokens, groups and tiles, ADP_PLAN_THREADS bins at a time
    for (int b0 = 0; b0 < bins; b0 += ADP_PLAN_THREADS) {
        const int b = b0 + tid, c = b < bins ? s_count[b] : 0;
        const bool tiled = c >= p.tile_least;
        const int own[3] = {c, tiled ? 0 : (c + ADP_TOK - 1) / ADP_TOK, tiled ? (c + ADP_TILE - 1) / ADP_TILE : 0};
        int at[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            at[i] = own[i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, at[i], o);
                if (lane >= o) at[i] += v;
            }
            if (lane == 31) s_warp[i][warp] = at[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            // (a warp's sum over the warps in front: one lane each)
            int v = lane < warp ? s_warp[i][lane] : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            at[i] += s_total[i] + v - own[i];
        }
        if (b < bins) {
            const int id = b == p.adapters ? -1 : b, step = tiled ? ADP_TILE : ADP_TOK;
            s_first[b] = at[0];
            int4* const to = tiled ? p.plan.tile() + at[2] : p.plan.group() + at[1];
            for (int i = 0; i * step < c; ++i) to[i] = make_int4(id, at[0] + i * step, min(step, c - i * step), c == 1);
        }
        __syncthreads();
        if (tid == ADP_PLAN_THREADS - 1)
            for (int i = 0; i < 3; ++i) s_total[i] = at[i] + own[i];
        __syncthreads();
    }
    if (tid == 0) {
        p.plan.count()[0] = s_total[1];
        p.plan.count()[1] = s_total[2];
    }
    for (int t0 = 0; t0 < p.tokens; t0 += ADP_PLAN_THREADS) {
        const int b = t0 + tid >= p.tokens ? -1 : (t0 + tid < KEPT ? s_bin[t0 + tid] : bin_of(t0 + tid));
        const unsigned same = __match_any_sync(0xffffffffu, b);
        int at = 0;
        const int leader = __ffs(same) - 1;
        if (b >= 0 && lane == leader) at = atomicAdd(&s_first[b], __popc(same));
        at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1u));
        if (b >= 0) p.plan.place()[at] = t0 + tid;
    }
}

}  // namespace b200

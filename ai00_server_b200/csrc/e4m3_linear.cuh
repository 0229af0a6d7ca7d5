// Products of e4m3 rows with a scale for every 128 of their inputs and e4m3 weights with a scale for every block of 128 x 128:
//     out[t, n] = base[t, n] + sum_b xs[t, b] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]
// The products of a block of 128 inputs are summed by the tensor core (tcgen05, kind::f8f6f4: products of e4m3 numbers are exact in its f32), scaled and
// added up in f32 registers: one multiply-add for every output and block.  Accumulators alternate between buffers in tensor memory, so that the products of the next blocks run
// meanwhile.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "f32x2.cuh"
#include "sm_pair.cuh"

namespace b200 {

constexpr int E4L_KB = 128;                      // inputs of a scale, and bytes of a row of an operand tile: the 128-byte swizzle

struct alignas(64) E4LinearParams {
    CUtensorMap tx, tw;              // rows of x and w, boxes of 128 inputs
    const float* xs;                 // [tokens][kblocks]
    const float* ws;                 // [N / 128][kblocks]
    const void* base;                // null: zeros
    long long base_stride;
    void* out;
    long long out_stride;
    int tokens, N, kblocks;
    int split;                       // e4_few_kernel: CTAs of a cluster, among which the blocks of inputs are dealt
    int vec;                         // e4_pair_kernel: sixteen-byte accesses to base and out
};

// K-major operand in the 128-byte swizzle: 8-row atoms of 1024 bytes; 32 inputs further are 32 bytes further
__device__ __forceinline__ uint64_t e4l_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// instruction descriptor, kind::f8f6f4: e4m3 x e4m3 -> f32, both K-major
__host__ __device__ constexpr uint32_t e4l_idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
__device__ __forceinline__ void e4l_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void e4l_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                 "r"(bar)
                 : "memory");
}
// waits of these kernels end: a thread whose barrier does not come within about a second goes on without it, and what hangs on it becomes NaN.  A role that
// lost a wait arrives nowhere any more, so that those behind it lose theirs
__device__ __forceinline__ bool e4l_wait(uint32_t bar, uint32_t parity) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try(bar, parity))
        if (globaltimer_ns() - t0 > 1000000000ull) return false;
    return true;
}
template <int N>
__device__ __forceinline__ void e4l_tmem(uint32_t at, float (&v)[N]) {
    static_assert(N == 16 || N == 32, "columns");
    uint32_t r[N];
    if constexpr (N == 16) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                       "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                     : "r"(at)
                     : "memory");
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
              "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
              "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(at)
            : "memory");
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}
template <typename O> __device__ __forceinline__ float e4l_widen(O v);
template <> __device__ __forceinline__ float e4l_widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float e4l_widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float e4l_widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename O> __device__ __forceinline__ O e4l_round(float v);
template <> __device__ __forceinline__ float e4l_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half e4l_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 e4l_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- few tokens: the weights' bytes are what a call costs ----
// 128 weight rows are the rows of the accumulator (a lane an output), up to TT tokens its columns; a cluster of `split` CTAs deals the blocks of inputs among
// itself, so that all SMs stream weights, and adds its sums in the order of its CTAs: CTA r finishes tokens r, r + split, ...
template <int TT>
struct E4Few {
    static constexpr int THREADS = 6 * 32;                       // four warps of outputs, one that loads, one that multiplies
    static constexpr int W_BYTES = 128 * E4L_KB, STAGE = W_BYTES + TT * E4L_KB;
    static constexpr int STAGES = 98304 / STAGE;                 // two CTAs to an SM
    static constexpr int BUFS = TT == 128 ? 2 : 4, COLUMNS = BUFS * TT;      // 64 .. 256
    static constexpr int CHUNK = TT == 128 ? 16 : 32;                          // blocks of inputs whose scales lie in shared memory at a time
    static constexpr int SCALES = STAGES * STAGE, BARS = SCALES + CHUNK * TT * 4, SMEM = BARS + (2 * STAGES + 2 * BUFS) * 8 + 16 + 1024;
    static_assert(TT * 128 * 4 <= STAGES * STAGE, "the sums of a CTA fit where the operands were");
    static_assert(SMEM <= 113 * 1024, "two CTAs to an SM");
};

template <int TT, typename O>
__global__ void __launch_bounds__(E4Few<TT>::THREADS, 2) e4_few_kernel(const __grid_constant__ E4LinearParams p) {
    using C = E4Few<TT>;
    extern __shared__ uint8_t e4_smem[];
    const uint32_t ring = (smem_u32(e4_smem) + 1023u) & ~1023u;
    uint8_t* const ring_p = e4_smem + (ring - smem_u32(e4_smem));
    const uint32_t full = ring + C::BARS, empty = full + C::STAGES * 8, tfull = empty + C::STAGES * 8, tempty = tfull + C::BUFS * 8, slot = tempty + C::BUFS * 8;
    unsigned* const lost = reinterpret_cast<unsigned*>(ring_p + (slot - ring)) + 1;      // some thread of this CTA lost a wait
    float* const scales = reinterpret_cast<float*>(ring_p + C::SCALES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = p.split, rank = blockIdx.x % split, tile = blockIdx.x / split, t0 = blockIdx.y * TT, nt = min(TT, p.tokens - t0);
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(full + i * 8, 1); mbar_init(empty + i * 8, 1); }
        for (int i = 0; i < C::BUFS; ++i) { mbar_init(tfull + i * 8, 1); mbar_init(tempty + i * 8, 4); }
        *lost = 0u;
        mbar_fence_init();
    }
    if (warp == 5) tc_alloc(slot, C::COLUMNS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(ring_p + (slot - ring));
    pdl_launch_dependents();
    pdl_wait();
    // this CTA's blocks of inputs: a run of them
    const int per = (p.kblocks + split - 1) / split, b0 = min(rank * per, p.kblocks), nb = min(per, p.kblocks - b0);
    float acc[TT];
    if (warp == 4) {
        if (lane == 0) {
            bool fine = true;
            for (int i = 0; i < nb && fine; ++i) {
                const int s = i % C::STAGES;
                if (i >= C::STAGES) fine = e4l_wait(empty + s * 8, (unsigned)(i / C::STAGES - 1) & 1u);
                if (!fine) break;
                mbar_expect_tx(full + s * 8, C::STAGE);
                e4l_load(ring + s * C::STAGE, &p.tw, (b0 + i) * E4L_KB, tile * 128, full + s * 8);
                e4l_load(ring + s * C::STAGE + C::W_BYTES, &p.tx, (b0 + i) * E4L_KB, t0, full + s * 8);
            }
        }
    } else if (warp == 5) {
        if (lane == 0) {
            constexpr uint32_t IDESC = e4l_idesc(128, TT);
            for (int i = 0; i < nb; ++i) {
                const int s = i % C::STAGES, b = i % C::BUFS;
                if (!e4l_wait(full + s * 8, (unsigned)(i / C::STAGES) & 1u)) break;
                if (i >= C::BUFS && !e4l_wait(tempty + b * 8, (unsigned)(i / C::BUFS - 1) & 1u)) break;
                tc_fence_after();
                const uint32_t st = ring + s * C::STAGE;
#pragma unroll
                for (int k = 0; k < E4L_KB / 32; ++k) e4l_mma(tmem + b * TT, e4l_desc(st + k * 32), e4l_desc(st + C::W_BYTES + k * 32), IDESC, k > 0);
                tc_commit(empty + s * 8);
                tc_commit(tfull + b * 8);
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[t] = 0.f;
        bool fine = true;
        const float* const ws = p.ws + (size_t)tile * p.kblocks + b0;
        for (int i = 0; i < nb; ++i) {
            if (i % C::CHUNK == 0) {                     // scales of the next blocks: both factors' product
                if (i) named_bar_sync(1, 128);
                const int n = min(C::CHUNK, nb - i);
                for (int e = tid; e < nt * n; e += 128) {
                    const int t = e / n, j = e - t * n;
                    scales[j * TT + t] = p.xs[(size_t)(t0 + t) * p.kblocks + b0 + i + j] * ws[i + j];
                }
                for (int e = tid; e < (TT - nt) * n; e += 128) scales[(e % n) * TT + nt + e / n] = 0.f;
                named_bar_sync(1, 128);
            }
            const int b = i % C::BUFS;
            fine = fine && e4l_wait(tfull + b * 8, (unsigned)(i / C::BUFS) & 1u);
            __syncwarp();
            tc_fence_after();
            const float* const sc = scales + (i % C::CHUNK) * TT;
            constexpr int STEP = TT < 32 ? 16 : 32;
#pragma unroll
            for (int c = 0; c < TT; c += STEP) {
                float v[STEP];
                e4l_tmem<STEP>(tmem + ((uint32_t)(warp * 32) << 16) + b * TT + c, v);
#pragma unroll
                for (int t = 0; t < STEP; t += 4) {
                    const float4 s = *reinterpret_cast<const float4*>(sc + c + t);
                    acc[c + t] = fmaf(v[t], s.x, acc[c + t]);
                    acc[c + t + 1] = fmaf(v[t + 1], s.y, acc[c + t + 1]);
                    acc[c + t + 2] = fmaf(v[t + 2], s.z, acc[c + t + 2]);
                    acc[c + t + 3] = fmaf(v[t + 3], s.w, acc[c + t + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && fine) mbar_arrive(tempty + b * 8);
        }
        if (!fine) {
            *lost = 1u;
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[t] = __int_as_float(0x7fc00000);
        }
    }
    // (a thread whose waits came has seen every copy and product of its CTA end; sums beside a lost wait may be written over by a late copy, and are not used)
    float* const sums = reinterpret_cast<float*>(ring_p);                // [token][128 outputs]
    if (warp < 4) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
            if (t < nt) sums[t * 128 + tid] = acc[t];
    }
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (warp < 4) {
        const int n = tile * 128 + tid;
        O* const out = reinterpret_cast<O*>(p.out) + n;
        const O* const base = p.base ? reinterpret_cast<const O*>(p.base) + n : nullptr;
        unsigned bad = 0;
        for (int c = 0; c < split; ++c) {
            unsigned x;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(mapa_u32(smem_u32(lost), c)) : "memory");
            bad |= x;
        }
#pragma unroll 2
        for (int t = rank; t < nt; t += split) {
            const O old = base && n < p.N ? base[(size_t)(t0 + t) * p.base_stride] : e4l_round<O>(0.f);
            const uint32_t at = smem_u32(sums + t * 128 + tid);
            float v = bad ? __int_as_float(0x7fc00000) : 0.f;
#pragma unroll 8
            for (int c = 0; c < split; ++c) {
                float x;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(mapa_u32(at, c)) : "memory");
                v += x;
            }
            if (n < p.N) out[(size_t)(t0 + t) * p.out_stride] = e4l_round<O>(v + e4l_widen<O>(old));
        }
    }
    if (split > 1) cluster_sync_all();      // no CTA leaves while another reads its sums
    tc_fence_before();
    __syncthreads();
    if (warp == 5) tc_dealloc(tmem, C::COLUMNS);
}

// ---- many tokens: the tensor cores' rate ----
// Pairs of SMs share tiles of 256 tokens x BN outputs (cta_group::2): each CTA holds 128 tokens, half of the weight rows, and the accumulators of its tokens: 32 KB an
// SM for 128 inputs, where one SM alone would take in 48 KB for the same products.  A lane is a token, so that a thread has one factor for all of its columns in a block
// of inputs.  Persistent clusters walk the tiles, tokens first, so that those that run together share weights in L2.
template <int BN>
struct E4Pair {
    static constexpr int EPI_WARPS = 8, THREADS = EPI_WARPS * 32 + 64;       // eight warps of outputs, one that multiplies, one that loads
    static constexpr int X_BYTES = 128 * E4L_KB, W_BYTES = BN / 2 * E4L_KB, STAGE = X_BYTES + W_BYTES;
    static constexpr int STAGES = BN == 256 ? 6 : 8;
    static constexpr int BARS = STAGES * STAGE, SMEM = BARS + (2 * STAGES + 4) * 8 + 16 + 1024;
    static constexpr int COLUMNS = 2 * BN, MINE = BN / 2;        // columns of a thread
};
__device__ __forceinline__ void e4l_mma2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// counted on the leader's barrier
__device__ __forceinline__ void e4l_load2(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x),
                 "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool e4l_wait_cluster(uint32_t bar, uint32_t parity) {
    if (mbar_try_cluster(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_cluster(bar, parity))
        if (globaltimer_ns() - t0 > 1000000000ull) return false;
    return true;
}

template <int BN, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(E4Pair<BN>::THREADS, 1) e4_pair_kernel(const __grid_constant__ E4LinearParams p) {
    using C = E4Pair<BN>;
    extern __shared__ uint8_t e4_smem[];
    const uint32_t ring = (smem_u32(e4_smem) + 1023u) & ~1023u;
    uint8_t* const ring_p = e4_smem + (ring - smem_u32(e4_smem));
    const uint32_t full = ring + C::BARS, empty = full + C::STAGES * 8, tfull = empty + C::STAGES * 8, tempty = tfull + 16, slot = tempty + 16;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank();
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(full + i * 8, 1); mbar_init(empty + i * 8, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(tfull + i * 8, 1); mbar_init(tempty + i * 8, 2 * C::EPI_WARPS); }
        mbar_fence_init();
    }
    if (warp == C::EPI_WARPS) tc_alloc2(slot, C::COLUMNS);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                      // the peer's barriers exist before anything arrives there
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(ring_p + (slot - ring));
    pdl_launch_dependents();
    pdl_wait();
    const int ttiles = (p.tokens + 255) / 256, ntiles = (p.N + BN - 1) / BN, nb = p.kblocks;
    const long long units = (long long)ttiles * ntiles;
    const long long u0 = cluster_id_x(), step = ncluster_x();

    if (warp == C::EPI_WARPS + 1) {
        if (lane == 0) {
            const uint32_t lead = mapa_u32(full, 0);
            unsigned i = 0;                                  // blocks of inputs so far
            bool fine = true;
            for (long long u = u0; u < units && fine; u += step) {
                const int xrow = (int)(u % ttiles) * 256 + rank * 128, wrow = (int)(u / ttiles) * BN + rank * (BN / 2);
                for (int b = 0; b < nb; ++b, ++i) {
                    const unsigned s = i % C::STAGES;
                    if (i >= C::STAGES && !(fine = e4l_wait_cluster(empty + s * 8, (i / C::STAGES - 1) & 1u))) break;
                    const uint32_t st = ring + s * C::STAGE;
                    if (rank == 0) mbar_expect_tx(full + s * 8, 2 * C::STAGE);
                    e4l_load2(st, &p.tx, b * E4L_KB, xrow, lead + s * 8);
                    e4l_load2(st + C::X_BYTES, &p.tw, b * E4L_KB, wrow, lead + s * 8);
                }
            }
            // every stage in use is released before this CTA may end: the leader's last commits arrive here
            for (unsigned k = 1; fine && k <= min(i, (unsigned)C::STAGES); ++k) fine = e4l_wait_cluster(empty + ((i - k) % C::STAGES) * 8, ((i - k) / C::STAGES) & 1u);
        }
    } else if (warp == C::EPI_WARPS) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t IDESC = e4l_idesc(256, BN);
            unsigned i = 0;
            bool fine = true;
            for (long long u = u0; u < units && fine; u += step)
                for (int b = 0; b < nb; ++b, ++i) {
                    const unsigned s = i % C::STAGES, acc = i & 1u;
                    if (!(fine = e4l_wait_cluster(full + s * 8, (i / C::STAGES) & 1u))) break;
                    if (i >= 2 && !(fine = e4l_wait_cluster(tempty + acc * 8, (i / 2 - 1) & 1u))) break;
                    tc_fence_after();
                    const uint32_t st = ring + s * C::STAGE;
#pragma unroll
                    for (int k = 0; k < E4L_KB / 32; ++k) e4l_mma2(tmem + acc * BN, e4l_desc(st + k * 32), e4l_desc(st + C::X_BYTES + k * 32), IDESC, k > 0);
                    tc_commit2(empty + s * 8);
                    tc_commit2(tfull + acc * 8);
                }
        }
    } else {
        // warps w and w + 4: the same 32 tokens, one half of the columns each
        const int half = warp >> 2;
        const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * C::MINE, lead = mapa_u32(tempty, 0);
        unsigned i = 0;
        bool fine = true;
        for (long long u = u0; u < units; u += step) {
            const int t = (int)(u % ttiles) * 256 + rank * 128 + (warp & 3) * 32 + lane, n0 = (int)(u / ttiles) * BN + half * C::MINE;
            const bool real = t < p.tokens && n0 < p.N;
            const float* const xs = p.xs + (size_t)min(t, p.tokens - 1) * nb;
            const float* const ws = p.ws + (size_t)min(n0 / 128, (p.N - 1) / 128) * nb;
            f32x2 acc[C::MINE / 2];
#pragma unroll
            for (int c = 0; c < C::MINE / 2; ++c) acc[c] = 0ull;
            // factors come a few blocks ahead: a block is a few hundred cycles
            constexpr int AHEAD = 4;
            float sx[AHEAD], sw[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                sx[a] = a < nb ? xs[a] : 0.f;
                sw[a] = a < nb ? ws[a] : 0.f;
            }
            for (int b = 0; b < nb; b += AHEAD) {
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    if (b + a >= nb) break;
                    const float f = sx[a] * sw[a];
                    if (b + a + AHEAD < nb) {
                        sx[a] = xs[b + a + AHEAD];
                        sw[a] = ws[b + a + AHEAD];
                    }
                    const f32x2 ff = pack2(f, f);
                    const unsigned buf = i & 1u;
                    fine = fine && e4l_wait_cluster(tfull + buf * 8, (i >> 1) & 1u);
                    __syncwarp();
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < C::MINE; c += 16) {
                        float v[16];
                        e4l_tmem<16>(tm + buf * BN + c, v);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) fma2(acc[(c + j) / 2], pack2(v[j], v[j + 1]), ff);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && fine) mbar_arrive_cluster(lead + buf * 8);
                    ++i;
                }
            }
            if (!real) continue;
            O* const out = reinterpret_cast<O*>(p.out) + (size_t)t * p.out_stride + n0;
            const O* const base = p.base ? reinterpret_cast<const O*>(p.base) + (size_t)t * p.base_stride + n0 : nullptr;
            const int left = p.N - n0;
            constexpr int PER = 16 / (int)sizeof(O);         // values of an access
#pragma unroll
            for (int c = 0; c < C::MINE; c += PER) {
                float v[PER];
#pragma unroll
                for (int j = 0; j < PER; j += 2) {
                    const float2 q = unpack2(acc[(c + j) / 2]);
                    v[j] = fine ? q.x : __int_as_float(0x7fc00000);
                    v[j + 1] = fine ? q.y : __int_as_float(0x7fc00000);
                }
                if (p.vec && c + PER <= left) {
                    O e[PER];
                    if (base) {
                        const uint4 w = *reinterpret_cast<const uint4*>(base + c);
                        memcpy(e, &w, 16);
#pragma unroll
                        for (int j = 0; j < PER; ++j) v[j] += e4l_widen<O>(e[j]);
                    }
#pragma unroll
                    for (int j = 0; j < PER; ++j) e[j] = e4l_round<O>(v[j]);
                    uint4 w;
                    memcpy(&w, e, 16);
                    *reinterpret_cast<uint4*>(out + c) = w;
                } else {
#pragma unroll
                    for (int j = 0; j < PER; ++j)
                        if (c + j < left) out[c + j] = e4l_round<O>(v[j] + (base ? e4l_widen<O>(base[c + j]) : 0.f));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                      // no CTA leaves while its peer's products read its shared memory or arrive on its barriers
    tc_fence_after();
    if (warp == C::EPI_WARPS) tc_dealloc2(tmem, C::COLUMNS);
}

}  // namespace b200

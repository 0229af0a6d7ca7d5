// Products of e4m3 rows with a scale for every 128 of their inputs and e4m3 weights with a scale for every block of 128 x 128:
//     out[t, n] = base[t, n] + sum_b xs[t, b] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]
// The products of a block of 128 inputs are summed by the tensor core (tcgen05, kind::f8f6f4: products of e4m3 numbers are exact in its f32), scaled and
// added up in f32 registers: one multiply-add for every output and block.  Accumulators alternate between buffers in tensor memory, so that the products of the next blocks run
// meanwhile.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "common.cuh"
#include "f32x2.cuh"
#include "float_types.cuh"
#include "lost_waits.cuh"
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
// one lane of the warp, the same every time: code behind it keeps its addresses in uniform registers, which the tensor core's instructions want (behind `lane == 0`
// four products and two commits took 480 cycles to issue, and their loop 1 060 a block of inputs)
__device__ __forceinline__ bool e4l_elect() {
    uint32_t is;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(is));
    return is != 0;
}
// waits of these kernels end: a thread whose barrier does not come within about a second goes on without it, and what hangs on it becomes NaN, and is counted (once for each thread of outputs, at its end: in the wait itself, 3 in 100 of a call).  A role that
// lost a wait arrives nowhere any more, so that those behind it lose theirs; before its CTA ends it waits once more, as long again at most, for the copies and products that it
// asked for: nothing is written to shared memory that is another's by then
// (the clock is asked every 256 tries: reading it takes longer than most waits).  WARP: all of a warp have the same answer, or, where one had lost its wait, the others would
// elect a lane without it
template <bool WARP>
__device__ __forceinline__ bool e4l_wait_as(uint32_t bar, uint32_t parity) {
    unsigned long long t0 = 0;
    for (;;) {
        for (int i = 0; i < 256; ++i) {
            const bool there = mbar_try(bar, parity);
            if (WARP ? __all_sync(0xffffffffu, there) : there) return true;
        }
        unsigned long long t = globaltimer_ns();
        if (WARP) t = __shfl_sync(0xffffffffu, t, 0);
        if (t0 == 0) t0 = t;
        else if (t - t0 > 1000000000ull) return false;
    }
}
__device__ __forceinline__ bool e4l_wait(uint32_t bar, uint32_t parity) { return e4l_wait_as<false>(bar, parity); }
__device__ __forceinline__ bool e4l_wait_warp(uint32_t bar, uint32_t parity) { return e4l_wait_as<true>(bar, parity); }
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
template <typename O> __device__ __forceinline__ O e4l_round(float v);
template <> __device__ __forceinline__ float e4l_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half e4l_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 e4l_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- few tokens: the weights' bytes are what a call costs ----
// 128 weight rows are the rows of the accumulator (a lane an output), up to TT tokens its columns; a cluster of `split` CTAs deals the blocks of inputs among
// itself, so that all SMs stream weights, and adds its sums in the order of its CTAs: CTA r finishes tokens r, r + split, ...
// Measured: 16 tokens 4096 -> 14336 14.2 us (58.7 MB of weights: 4.1 TB/s; the start and the end of a launch are 4 of them), 4096 -> 65536 47 us (6.0 TB/s), one token 2560 -> 2560 5.0, or 6.4 with weights from memory;
// 32 tokens 4096 -> 14336 16, 64 tokens 18, 333 tokens 8960 -> 2560 24.  Of those 24, loads alone take 15.5 and loads with products 21: 32 KB a block of inputs come in and are read by the
// products at 128 bytes a cycle.  Clusters of five to seven CTAs leave SMs idle (22 us for 14.5); a request for the weights in L2 ahead of the wait for the kernel in
// front lost (16 to 17 us).
template <int TT>
struct E4Few {
    static constexpr int EPI = TT >= 64 ? 8 : 4, THREADS = (EPI + 2) * 32;       // warps of outputs (eight: half of the tokens each), one that loads, one that multiplies
    static constexpr int MINE = TT * 4 / EPI;                    // tokens of a thread
    static constexpr int PER_SM = TT <= 32 ? 4 : (TT == 64 ? 2 : 1);              // CTAs
    static constexpr int W_BYTES = 128 * E4L_KB, STAGE = W_BYTES + TT * E4L_KB, STAGES = TT <= 32 ? 2 : (TT == 64 ? 4 : 6);
    static constexpr int BUFS = 4, COLUMNS = BUFS * TT < 32 ? 32 : BUFS * TT;      // 64 .. 256
    static constexpr int CHUNK = TT <= 16 ? 32 : 16;             // blocks of inputs whose scales lie in shared memory at a time
    static constexpr int SCALES = STAGES * STAGE, BARS = SCALES + CHUNK * TT * 4, SMEM = BARS + (2 * STAGES + 2 * BUFS) * 8 + 16 + 1024;
    static_assert(TT * 128 * 4 <= STAGES * STAGE, "the sums of a CTA fit where the operands were");
    static_assert(PER_SM * (SMEM + 1024) <= 228 * 1024 && PER_SM * COLUMNS <= 512, "CTAs of an SM");
};

template <int TT, typename O>
__global__ void __launch_bounds__(E4Few<TT>::THREADS, E4Few<TT>::PER_SM) e4_few_kernel(const __grid_constant__ E4LinearParams p) {
    using C = E4Few<TT>;
    extern __shared__ uint8_t e4_smem[];
    const uint32_t ring = (smem_u32(e4_smem) + 1023u) & ~1023u;
    uint8_t* const ring_p = e4_smem + (ring - smem_u32(e4_smem));
    const uint32_t full = ring + C::BARS, empty = full + C::STAGES * 8, tfull = empty + C::STAGES * 8, tempty = tfull + C::BUFS * 8, slot = tempty + C::BUFS * 8;
    unsigned* const lost = reinterpret_cast<unsigned*>(ring_p + (slot - ring)) + 1;      // some thread of this CTA lost a wait
    float* const scales = reinterpret_cast<float*>(ring_p + C::SCALES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = p.split, rank = blockIdx.x % split, tile = blockIdx.x / split, t0 = blockIdx.y * TT, nt = min(TT, p.tokens - t0);
    // this CTA's blocks of inputs: a run of them
    const int b0 = p.kblocks * rank / split, nb = p.kblocks * (rank + 1) / split - b0;
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(full + i * 8, 1); mbar_init(empty + i * 8, 1); }
        for (int i = 0; i < C::BUFS; ++i) { mbar_init(tfull + i * 8, 1); mbar_init(tempty + i * 8, C::EPI); }
        *lost = 0u;
        mbar_fence_init();
    }
    if (warp == C::EPI + 1) tc_alloc(slot, C::COLUMNS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(ring_p + (slot - ring));
    pdl_launch_dependents();
    pdl_wait();
    f32x2 acc[C::MINE / 2];                                  // of two tokens each
    if (warp == C::EPI) {
        unsigned s = 0, phase = 1;
        int i = 0;
        for (; i < nb; ++i) {
            if (i >= C::STAGES && !e4l_wait_warp(empty + s * 8, phase)) break;
            if (e4l_elect()) {
                mbar_expect_tx(full + s * 8, C::STAGE);
                e4l_load(ring + s * C::STAGE, &p.tw, (b0 + i) * E4L_KB, tile * 128, full + s * 8);
                e4l_load(ring + s * C::STAGE + C::W_BYTES, &p.tx, (b0 + i) * E4L_KB, t0, full + s * 8);
            }
            __syncwarp();
            if (++s == C::STAGES) { s = 0; phase ^= 1u; }
        }
        bool fine = true;
        for (int k = 1; fine && k <= min(i, C::STAGES); ++k) fine = e4l_wait(full + (i - k) % C::STAGES * 8, (unsigned)((i - k) / C::STAGES) & 1u);      // the copies of this CTA have landed
    } else if (warp == C::EPI + 1) {
        constexpr uint32_t IDESC = e4l_idesc(128, TT);
        unsigned s = 0, phase = 0, b = 0, bphase = 1;
        int i = 0;
        for (; i < nb; ++i) {
            if (!e4l_wait_warp(full + s * 8, phase)) break;
            if (i >= C::BUFS && !e4l_wait_warp(tempty + b * 8, bphase)) break;
            tc_fence_after();
            if (e4l_elect()) {
                const uint64_t w = e4l_desc(ring + s * C::STAGE), x = e4l_desc(ring + s * C::STAGE + C::W_BYTES);
#pragma unroll
                for (int k = 0; k < E4L_KB / 32; ++k) e4l_mma(tmem + b * TT, w + k * 2, x + k * 2, IDESC, k > 0);        // (32 bytes further: two units of the descriptor)
                tc_commit(empty + s * 8);
                tc_commit(tfull + b * 8);
            }
            __syncwarp();
            if (++s == C::STAGES) { s = 0; phase ^= 1u; }
            if (++b == C::BUFS) { b = 0; bphase ^= 1u; }
        }
        if (i > 0) e4l_wait(empty + (i - 1) % C::STAGES * 8, (unsigned)((i - 1) / C::STAGES) & 1u);      // and its products, too
    } else {
#pragma unroll
        for (int t = 0; t < C::MINE / 2; ++t) acc[t] = 0ull;
        bool fine = true;
        const int first = (warp >> 2) * C::MINE;             // token of acc[0]
        const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + first;
        // Scales of the next blocks: a thread has one block and some of the tokens, and asks for them a chunk ahead (from the loop itself, one at a time, a chunk of 128 tokens
        // took 8 000 cycles)
        constexpr int THREADS = C::EPI * 32, NS = TT * C::CHUNK / THREADS;
        const int sj = tid % C::CHUNK, st = tid / C::CHUNK;
        const float* const xs = p.xs + (size_t)t0 * p.kblocks + b0;
        const float* const ws = p.ws + (size_t)tile * p.kblocks + b0;
        float sx[NS], sw = 0.f;
        auto ask = [&](int i) {                              // (blocks and tokens that are not there read the last ones': loads under conditions of their own take as long as one after the other)
            const int at = min(i + sj, nb - 1);
            sw = ws[at];
#pragma unroll
            for (int k = 0; k < NS; ++k) sx[k] = xs[(size_t)min(st + k * (THREADS / C::CHUNK), nt - 1) * p.kblocks + at];
        };
        ask(0);
        unsigned b = 0, bphase = 0;
        for (int i = 0; i < nb; ++i) {
            if (i % C::CHUNK == 0) {
                if (i) named_bar_sync(1, THREADS);
#pragma unroll
                for (int k = 0; k < NS; ++k) scales[sj * TT + st + k * (THREADS / C::CHUNK)] = sx[k] * sw;       // both factors' product
                named_bar_sync(1, THREADS);
                ask(i + C::CHUNK);
            }
            fine = fine && e4l_wait(tfull + b * 8, bphase);
            __syncwarp();
            tc_fence_after();
            const float* const sc = scales + (i % C::CHUNK) * TT + first;
            constexpr int STEP = C::MINE < 32 ? 16 : 32;
#pragma unroll
            for (int c = 0; c < C::MINE; c += STEP) {
                float v[STEP];
                e4l_tmem<STEP>(tm + b * TT + c, v);
                if (c + STEP == C::MINE) {                   // the accumulator is free again
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && fine) mbar_arrive(tempty + b * 8);
                }
#pragma unroll
                for (int t = 0; t < STEP; t += 4) {
                    const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(sc + c + t);
                    fma2(acc[(c + t) / 2], pack2(v[t], v[t + 1]), s.x);
                    fma2(acc[(c + t) / 2 + 1], pack2(v[t + 2], v[t + 3]), s.y);
                }
            }
            if (++b == C::BUFS) { b = 0; bphase ^= 1u; }
        }
        // a thread whose waits came has seen every copy and product of its CTA end; sums beside a lost wait may be written over by a late copy, and are not used
        if (!fine) {
            *lost = 1u;
            lost_wait();
        }
    }
    // (nothing is in flight any more, or lost: the operands' place is free)
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(ring_p);                // [token][128 outputs]
    if (warp < C::EPI) {
        const int first = (warp >> 2) * C::MINE;
#pragma unroll
        for (int t = 0; t < C::MINE; t += 2) {
            const float2 x = unpack2(acc[t / 2]);
            if (first + t < nt) sums[(first + t) * 128 + (tid & 127)] = x.x;
            if (first + t + 1 < nt) sums[(first + t + 1) * 128 + (tid & 127)] = x.y;
        }
    }
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (warp < C::EPI) {
        const int n = tile * 128 + (tid & 127);
        O* const out = reinterpret_cast<O*>(p.out) + n;
        const O* const base = p.base ? reinterpret_cast<const O*>(p.base) + min(n, p.N - 1) : nullptr;
        unsigned bad = 0;
        for (int c = 0; c < split; ++c) {
            unsigned x;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(mapa_u32(smem_u32(lost), c)) : "memory");
            bad |= x;
        }
        // several tokens at a time: their parts are on their way from the other CTAs together (one after the other, 32 tokens of two CTAs took 10 us)
        constexpr int EVERY = C::EPI / 4, BATCH = TT <= 32 ? 4 : 16;
        const int step = split * EVERY;
        for (int tb = rank * EVERY + (warp >> 2); tb < nt; tb += step * BATCH) {
            float v[BATCH];
            O old[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                v[j] = bad ? __int_as_float(0x7fc00000) : 0.f;
                old[j] = e4l_round<O>(0.f);
            }
            if (base) {
#pragma unroll
                for (int j = 0; j < BATCH; ++j) old[j] = base[(size_t)(t0 + min(tb + j * step, nt - 1)) * p.base_stride];
            }
            const uint32_t at = smem_u32(sums + tb * 128 + (tid & 127));
#pragma unroll 2
            for (int c = 0; c < split; ++c) {
                float x[BATCH];
                const uint32_t there = mapa_u32(at, c);
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[j]) : "r"(there + (uint32_t)min(j * step, nt - 1 - tb) * 512u) : "memory");
#pragma unroll
                for (int j = 0; j < BATCH; ++j) v[j] += x[j];
            }
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (n < p.N && tb + j * step < nt) out[(size_t)(t0 + tb + j * step) * p.out_stride] = e4l_round<O>(v[j] + widened<O>(old[j]));
        }
    }
    if (split > 1) cluster_sync_all();      // no CTA leaves while another reads its sums
    tc_fence_before();
    __syncthreads();
    if (warp == C::EPI + 1) tc_dealloc(tmem, C::COLUMNS);
}

// ---- many tokens: the tensor cores' rate ----
// Pairs of SMs share tiles of 256 tokens x 256 outputs (cta_group::2): each CTA holds 128 tokens, half of the weight rows, and the accumulators of its tokens: 32 KB an
// SM for 128 inputs, where one SM alone would take in 48 KB for the same products.  A lane is a token, so that a thread has one factor for all of its columns in a block
// of inputs.  Persistent clusters walk the tiles, tokens first, so that those that run together share weights in L2.
// What bounds it: a block of inputs is 512 cycles of the tensor cores and 1 000 of the eight warps that scale its sums, a chain of a wait, four reads of tensor memory and their
// multiply-adds (without scales, a whole k range summed in tensor memory, 2048 tokens 4096 -> 14336 took 108 us where these took 133).  Those warps have 224 registers, so that a read is in flight
// beside each quarter's multiply-adds; scales come through shared memory by warps of their own; sums leave through shared memory.
// Measured: 2048 tokens 4096 -> 14336 119 to 141 us, 1.7 to 2.0 PFLOP/s (119 in short runs, 141 for seconds, at the power limit and 1605 MHz), with a base 133, to 14337 outputs with a base 166;
// 4096 tokens 8192 -> 8192 238 us, 2.3 PFLOP/s; 256 tokens 192 -> 75776 19 us, with a base 26.
// Tried: sixteen warps for the sums (146 us), a read ahead over the ends of blocks (140: registers spill, and spilled ones are waited for at every arrival), tiles of 128 outputs (160), the
// last tiles of a launch in halves and quarters (133).
struct E4Pair {
    static constexpr int BN = 256;                               // outputs of a tile
    static constexpr int EPI_WARPS = 8, THREADS = 12 * 32;       // eight warps of outputs, one that multiplies, one that loads operands, two that load scales
    static constexpr int EPI_REGS = 224, REST_REGS = 56;         // registers of a thread: three groups of four warps have the 168 of the launch among them
    static_assert(2 * EPI_REGS + REST_REGS <= 3 * 168, "the registers of the launch");
    static constexpr int X_BYTES = 128 * E4L_KB, W_BYTES = BN / 2 * E4L_KB, STAGE = X_BYTES + W_BYTES;
    static constexpr int STAGES = 5;
    static constexpr int CHUNK = 16;                             // blocks of inputs whose scales lie in shared memory at a time; two of them
    static constexpr int SCALES = STAGES * STAGE, CHUNK_FLOATS = CHUNK * (128 + 2);
    static constexpr int PITCH = 128 + 16;                       // of a token's 128 bytes on their way out (readers and writers are off one another's banks)
    static constexpr int OUT = SCALES + 2 * CHUNK_FLOATS * 4, BARS = OUT + EPI_WARPS * 32 * PITCH, SMEM = BARS + (2 * STAGES + 8) * 8 + 16 + 1024;
    static constexpr int COLUMNS = 2 * BN, MINE = BN / 2;        // columns of a thread
    static_assert(SMEM <= 227 * 1024, "an SM's shared memory");
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
// an arrival at another CTA's barrier.  (What it stands for, reads of tensor memory, is ordered by the tcgen05 fence in front; with .release.cluster a warp waited
// 1 000 to 1 500 cycles for its loads from global memory here)
__device__ __forceinline__ void e4l_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// 32 lanes x 32 columns on their way to registers, and the wait for them
__device__ __forceinline__ void e4l_fetch(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void e4l_fetched(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                   "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

template <typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(E4Pair::THREADS, 1) e4_pair_kernel(const __grid_constant__ E4LinearParams p) {
    using C = E4Pair;
    constexpr int BN = C::BN;
    extern __shared__ uint8_t e4_smem[];
    const uint32_t ring = (smem_u32(e4_smem) + 1023u) & ~1023u;
    uint8_t* const ring_p = e4_smem + (ring - smem_u32(e4_smem));
    const uint32_t full = ring + C::BARS, empty = full + C::STAGES * 8, tfull = empty + C::STAGES * 8, tempty = tfull + 16, sfull = tempty + 16, sempty = sfull + 16, slot = sempty + 16;
    float* const scales = reinterpret_cast<float*>(ring_p + C::SCALES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_rank();
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) { mbar_init(full + i * 8, 1); mbar_init(empty + i * 8, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(tfull + i * 8, 1); mbar_init(tempty + i * 8, 2 * C::EPI_WARPS); mbar_init(sfull + i * 8, 64); mbar_init(sempty + i * 8, C::EPI_WARPS); }
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
    const int units = ttiles * ntiles, u0 = (int)cluster_id_x(), step = (int)ncluster_x();

    if (warp >= C::EPI_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REST_REGS));
        if (warp == C::EPI_WARPS + 1 && lane == 0) {
            const uint32_t lead = mapa_u32(full, 0);
            unsigned i = 0;                                  // blocks of inputs so far
            bool fine = true;
            for (int u = u0; u < units && fine; u += step) {
                const int xrow = u % ttiles * 256 + rank * 128, wrow = u / ttiles * BN + rank * (BN / 2);
                for (int b = 0; b < nb; ++b, ++i) {
                    const unsigned s = i % C::STAGES;
                    if (i >= C::STAGES && !(fine = e4l_wait(empty + s * 8, (i / C::STAGES - 1) & 1u))) break;
                    const uint32_t st = ring + s * C::STAGE;
                    if (rank == 0) mbar_expect_tx(full + s * 8, 2 * C::STAGE);
                    e4l_load2(st, &p.tx, b * E4L_KB, xrow, lead + s * 8);
                    e4l_load2(st + C::X_BYTES, &p.tw, b * E4L_KB, wrow, lead + s * 8);
                }
            }
            // every stage in use is released before this CTA may end: the leader's last commits arrive here.  Where a wait was lost, the leader waits for the pair's copies at least
            for (unsigned k = 1; fine && k <= min(i, (unsigned)C::STAGES); ++k) fine = e4l_wait(empty + ((i - k) % C::STAGES) * 8, ((i - k) / C::STAGES) & 1u);
            bool landed = !fine && rank == 0;
            for (unsigned k = 1; landed && k <= min(i, (unsigned)C::STAGES); ++k) landed = e4l_wait(full + ((i - k) % C::STAGES) * 8, ((i - k) / C::STAGES) & 1u);
        } else if (warp == C::EPI_WARPS && rank == 0) {
            constexpr uint32_t IDESC = e4l_idesc(256, BN);
            unsigned i = 0, s = 0, phase = 0;
            bool fine = true;
            for (int u = u0; u < units && fine; u += step)
                for (int b = 0; b < nb; ++b, ++i) {
                    const unsigned acc = i & 1u;
                    if (!(fine = e4l_wait_warp(full + s * 8, phase))) break;
                    if (i >= 2 && !(fine = e4l_wait_warp(tempty + acc * 8, (i / 2 - 1) & 1u))) break;
                    tc_fence_after();
                    if (e4l_elect()) {
                        const uint64_t x = e4l_desc(ring + s * C::STAGE), w = e4l_desc(ring + s * C::STAGE + C::X_BYTES);
#pragma unroll
                        for (int k = 0; k < E4L_KB / 32; ++k) e4l_mma2(tmem + acc * BN, x + k * 2, w + k * 2, IDESC, k > 0);       // (32 bytes further: two units of the descriptor)
                        tc_commit2(empty + s * 8);
                        tc_commit2(tfull + acc * 8);
                    }
                    __syncwarp();
                    if (++s == C::STAGES) { s = 0; phase ^= 1u; }
                }
            if (!fine && i > 0) e4l_wait(empty + ((i - 1) % C::STAGES) * 8, ((i - 1) / C::STAGES) & 1u);       // the products that were asked for have ended
        } else if (warp >= C::EPI_WARPS + 2) {
            // scales of the tile's tokens and outputs, a token of a block beside the next
            const int me = tid - (C::EPI_WARPS + 2) * 32;
            unsigned c = 0;                                  // chunks so far
            bool fine = true;
            for (int u = u0; u < units && fine; u += step) {
                const int t0 = u % ttiles * 256 + rank * 128, n0 = u / ttiles * BN;
                for (int b0 = 0; b0 < nb; b0 += C::CHUNK, ++c) {
                    float* const to = scales + (c & 1u) * C::CHUNK_FLOATS;
                    if (c >= 2 && !(fine = e4l_wait(sempty + (c & 1u) * 8, (c / 2 - 1) & 1u))) break;
                    const int n = min(C::CHUNK, nb - b0);
#pragma unroll 1
                    for (int r = me; r < 128; r += 64) {
                        const float* const from = p.xs + (size_t)min(t0 + r, p.tokens - 1) * nb + b0;
                        float v[C::CHUNK];
#pragma unroll
                        for (int j = 0; j < C::CHUNK; ++j) v[j] = j < n ? from[j] : 0.f;
#pragma unroll
                        for (int j = 0; j < C::CHUNK; ++j) to[j * 128 + r] = v[j];
                    }
                    if (me < 2 * C::CHUNK) {
                        const int half = me / C::CHUNK, j = me % C::CHUNK;
                        to[C::CHUNK * 128 + me] = j < n ? p.ws[(size_t)min((n0 + half * C::MINE) / 128, (p.N - 1) / 128) * nb + b0 + j] : 0.f;
                    }
                    mbar_arrive(sfull + (c & 1u) * 8);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::EPI_REGS));
        // warps w and w + 4: the same 32 tokens, one half of the columns each
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * C::MINE, lead = mapa_u32(tempty, 0);
        unsigned i = 0, chunk = 0;
        bool fine = true;
        for (int u = u0; u < units; u += step) {
            const int n0 = u / ttiles * BN + half * C::MINE;
            const int tw = u % ttiles * 256 + rank * 128 + (warp & 3) * 32, rows = min(32, p.tokens - tw);
            // base of the tile to L2, a token's columns a lane, while its products are summed
            if (p.base && lane < rows) {
                const char* const at = reinterpret_cast<const char*>(reinterpret_cast<const O*>(p.base) + (size_t)(tw + lane) * p.base_stride + n0);
                const int bytes = min(C::MINE, p.N - n0) * (int)sizeof(O);
                for (int i = 0; i < bytes; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + i));
            }
            f32x2 acc[C::MINE / 2];
#pragma unroll
            for (int c = 0; c < C::MINE / 2; ++c) acc[c] = 0ull;
            for (int b0 = 0; b0 < nb; b0 += C::CHUNK, ++chunk) {
                const float* const sc = scales + (chunk & 1u) * C::CHUNK_FLOATS;
                fine = fine && e4l_wait(sfull + (chunk & 1u) * 8, (chunk >> 1) & 1u);
                const int n = min(C::CHUNK, nb - b0);
                for (int b = 0; b < n; ++b, ++i) {
                    const float f = sc[b * 128 + row] * sc[C::CHUNK * 128 + half * C::CHUNK + b];
                    const f32x2 ff = pack2(f, f);
                    const unsigned buf = i & 1u;
                    fine = fine && e4l_wait(tfull + buf * 8, (i >> 1) & 1u);
                    __syncwarp();
                    tc_fence_after();
                    uint32_t v[2][32];
                    e4l_fetch(tm + buf * BN, v[0]);
#pragma unroll
                    for (int c = 0; c < C::MINE / 32; ++c) {
                        e4l_fetched(v[c & 1]);
                        if (c + 1 < C::MINE / 32) {
                            e4l_fetch(tm + buf * BN + (c + 1) * 32, v[(c + 1) & 1]);
                        } else {                             // the accumulator is free again
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0 && fine) e4l_arrive(lead + buf * 8);
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            fma2(acc[c * 16 + j / 2], pack2(__uint_as_float(v[c & 1][j]), __uint_as_float(v[c & 1][j + 1])), ff);
                    }
                }
                __syncwarp();
                if (lane == 0 && fine) mbar_arrive(sempty + (chunk & 1u) * 8);
            }
            // out through the warp's piece of shared memory, 128 bytes of its 32 tokens at a time, so that accesses to base and out are runs of 128 bytes
            constexpr int PER = 16 / (int)sizeof(O), COLS = PER * 8;
            uint8_t* const mine = ring_p + C::OUT + warp * (32 * C::PITCH);
#pragma unroll
            for (int c0 = 0; c0 < C::MINE; c0 += COLS) {
                const int cols = min(COLS, p.N - n0 - c0);
                if (rows <= 0 || cols <= 0) break;
                O* const out = reinterpret_cast<O*>(p.out) + (size_t)tw * p.out_stride + n0 + c0;
                const O* const base = p.base ? reinterpret_cast<const O*>(p.base) + (size_t)tw * p.base_stride + n0 + c0 : nullptr;
                const int r4 = lane >> 3, c8 = (lane & 7) * PER;
                // (rows and columns that are not there read the last ones': loads under a condition of their own each take as long as one after the other)
                if (base) {
                    const int whole = p.vec ? cols / PER * PER : 0;
                    if (whole) {
                        uint4 w[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] = *reinterpret_cast<const uint4*>(base + (size_t)min(k * 4 + r4, rows - 1) * p.base_stride + min(c8, whole - PER));
#pragma unroll
                        for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(mine + (k * 4 + r4) * C::PITCH + (lane & 7) * 16) = w[k];
                        __syncwarp();
                    }
                    // where rows start off boundaries, and what is left of a row: a lane a column
                    for (int e0 = whole; e0 < cols; e0 += 32) {
                        const int e = min(e0 + lane, cols - 1);
                        O w[32];
#pragma unroll
                        for (int r = 0; r < 32; ++r) w[r] = base[(size_t)min(r, rows - 1) * p.base_stride + e];
#pragma unroll
                        for (int r = 0; r < 32; ++r) reinterpret_cast<O*>(mine + r * C::PITCH)[e] = w[r];
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int c = 0; c < COLS; c += PER) {
                    uint4* const at = reinterpret_cast<uint4*>(mine + lane * C::PITCH + c * (int)sizeof(O));
                    float v[PER];
                    O e[PER];
#pragma unroll
                    for (int j = 0; j < PER; j += 2) {
                        const float2 q = unpack2(acc[(c0 + c + j) / 2]);
                        v[j] = fine ? q.x : __int_as_float(0x7fc00000);
                        v[j + 1] = fine ? q.y : __int_as_float(0x7fc00000);
                    }
                    if (base) {
                        const uint4 w = *at;
                        memcpy(e, &w, 16);
#pragma unroll
                        for (int j = 0; j < PER; ++j) v[j] += widened<O>(e[j]);
                    }
#pragma unroll
                    for (int j = 0; j < PER; ++j) e[j] = e4l_round<O>(v[j]);
                    uint4 w;
                    memcpy(&w, e, 16);
                    *at = w;
                }
                __syncwarp();
                if (p.vec) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k * 4 + r4 < rows && c8 + PER <= cols)
                            *reinterpret_cast<uint4*>(out + (size_t)(k * 4 + r4) * p.out_stride + c8) = *reinterpret_cast<const uint4*>(mine + (k * 4 + r4) * C::PITCH + (lane & 7) * 16);
                }
                for (int e = (p.vec ? cols / PER * PER : 0) + lane; e < cols; e += 32) {
#pragma unroll
                    for (int r = 0; r < 32; ++r)
                        if (r < rows) out[(size_t)r * p.out_stride + e] = reinterpret_cast<const O*>(mine + r * C::PITCH)[e];
                }
                __syncwarp();
            }
        }
        if (!fine) lost_wait();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                      // no CTA leaves while its peer's products read its shared memory or arrive on its barriers
    tc_fence_after();
    if (warp == C::EPI_WARPS) tc_dealloc2(tmem, C::COLUMNS);
}

}  // namespace b200

// Low-rank adapters of prompt steps: many tokens of one adapter.  The formulas and the tokens' order by adapter are those of adapters.cuh.
//
// Bound: base and out are most of the bytes (2048 tokens, 4096 inputs, 14336 f32 outputs: 235 of 261 MB, 40 us at the copy rate); the products are 5 GFLOP
// there, 3 us of the tensor cores' bf16 rate, 35 us of what mma.sync reaches.  So: tcgen05 for both products, and a second kernel that does nothing but
// stream base and out through all SMs.
//   adapter_low_kernel: S = x A^T for up to 128 tokens of one adapter, a cluster of eight CTAs with an eighth of k each.  Tokens are the 128 rows of the
//     accumulator, ranks its columns; x rows (gathered: a tile's tokens lie anywhere) and A rows go to shared memory in the 128-byte swizzle by
//     cp.async, 64 k at a time, a slab to a pair of warps.  (The fence between a thread's copies and the tensor core waits for all of its copies, later
//     slabs' too: with slabs loaded by all warps one was in flight, however many there was room for, and took 1350 to 1900 cycles.)  The eight partial S are added through distributed shared memory, an eighth of the tokens
//     to a CTA, in the order of the CTAs; S leaves as 16-bit parts (adapters.cuh) in the rows the second kernel's operand has.
//   adapter_out_kernel: out^T = B S^T.  Units of (tile of tokens, 128 outputs) go to the CTAs in turn, outputs first, so that at any time the CTAs write whole
//     neighbouring rows (a run of outputs for each CTA, 38000 rows open at once, copied base to out in 50 us where this order takes 42 and a
//     linear copy 36).  128 outputs are the rows of the accumulator, the tile's tokens its columns; 32 tokens at a time pass through shared memory, so
//     that a warp adds and stores 128 neighbours of one token's row with 16-byte accesses.  (Straight from the accumulator, 32 neighbours a warp access, it
//     took 14 instructions an element, and the eight warps of a CTA 130 us for the case above, whatever was in flight.)  The operands of the
//     next unit arrive while one is written, its product runs during the last rows.
#pragma once
#include "adapters.cuh"

namespace b200 {

constexpr int ADT_THREADS = 256;
constexpr int ADT_LEAST = 24;                    // tokens of an adapter from which a tile is quicker than groups of eight
constexpr int ADT_TOK = ADP_TILE;                // tokens of a tile
constexpr int ADT_ROWS = 32;                     // tokens that pass through shared memory at a time
constexpr int ADT_TABLE = 256;                   // tiles whose places the second kernel keeps in shared memory
constexpr int ADT_PITCH = 128 + 4;               // floats between their rows

__host__ __device__ constexpr int adt_r16(int R) { return (R + 15) & ~15; }
__host__ __device__ constexpr int adt_chunks(int R) { return (R + 63) / 64; }                        // operand tiles of 64 ranks
// first kernel: slabs of x and A, where later the partial sums lie; two CTAs to an SM up to 64 ranks
__host__ __device__ constexpr int adt_stage(int R) { return ADT_TOK * 128 + adt_r16(R) * 128; }
constexpr int ADT_STAGES = 4;                    // slabs in flight, each the work of two warps; the partial sums fit in their place
constexpr int ADT_LOW_THREADS = (2 * ADT_STAGES + 1) * 32;       // and a warp for the products
__host__ __device__ constexpr int adt_low_smem(int R) { return ADT_STAGES * adt_stage(R) + 1024; }
__host__ __device__ constexpr int adt_low_columns(int R) { return R <= 32 ? 32 : (R <= 64 ? 64 : (R <= 128 ? 128 : 256)); }
// second kernel: S of up to 128 tokens, a tile of weights, two of rows; as many tokens as leave room for two CTAs on an SM
__host__ __device__ constexpr int adt_weights(int R) { return adt_chunks(R) * 128 * 128; }
__host__ __device__ constexpr int adt_out_bytes(int R, int parts, int tok) { return parts * adt_chunks(R) * tok * 128 + adt_weights(R) + 2 * ADT_ROWS * ADT_PITCH * 4 + 1024; }
constexpr int ADT_HALF_SM = 104 * 1024;
__host__ __device__ constexpr int adt_out_tokens(int R, int parts) {
    return adt_out_bytes(R, parts, 128) <= ADT_HALF_SM ? 128 : (adt_out_bytes(R, parts, 64) <= ADT_HALF_SM ? 64 : 32);
}
__host__ __device__ constexpr int adt_operand(int R, int parts) { return parts * adt_chunks(R) * adt_out_tokens(R, parts) * 128; }
__host__ __device__ constexpr int adt_out_smem(int R, int parts) { return adt_out_bytes(R, parts, adt_out_tokens(R, parts)); }

// S of a projection between the two kernels: [part][64 ranks][place] rows of 128 bytes, then the powers of two by place.  Whole rows, or the next projection's
// would not start where 16-byte accesses may (the powers of two alone take 4 bytes a token)
__host__ __device__ constexpr size_t adt_low_bytes(int tokens, int R, int parts) { return ((size_t)tokens * ((size_t)parts * adt_chunks(R) * 128 + 4) + 127) & ~(size_t)127; }
static_assert(adt_low_bytes(257, 8, 2) % 128 == 0 && adt_low_bytes(1021, 256, 2) % 128 == 0 && adt_low_bytes(1022, 64, 3) % 128 == 0, "rows of S on boundaries");

__device__ __forceinline__ uint64_t adt_desc(uint32_t saddr) {        // K-major operand in the 128-byte swizzle: 8-row atoms of 1024 bytes
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
template <typename E> __device__ __forceinline__ constexpr uint32_t adt_idesc(int M, int N) { return umma_idesc_f16(M, N); }
template <> __device__ __forceinline__ constexpr uint32_t adt_idesc<__nv_bfloat16>(int M, int N) { return umma_idesc_f16(M, N) | (1u << 7) | (1u << 10); }
// 16 bytes of a row's 128, or zeros
__device__ __forceinline__ void adt_cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// shared memory alone: the general form waits for the loads and stores to global memory in flight as well (a slab of 64 k took 2100 cycles with it, 1350 without)
__device__ __forceinline__ void adt_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void adt_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void adt_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t adt_swizzled(int row, int chunk) { return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4)); }
// waits of these kernels end: a thread whose barrier does not come within about a second goes on without it, and makes NaN of what hangs on it
__device__ __forceinline__ bool adt_bar_wait(uint32_t bar, uint32_t parity) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try(bar, parity))
        if (globaltimer_ns() - t0 > 1000000000ull) return false;
    return true;
}

// the adapter of a tile in one projection
template <typename E>
struct AdtWeights {
    const E *A = nullptr, *B = nullptr;
    int R = 0;
    float scale = 0.f;
    __device__ __forceinline__ AdtWeights(const AdapterParams& p, const AdapterPart& q, int adapter) {
        if (adapter < 0) return;
        if (q.table) {
            const AdapterEntry e = q.table[adapter];
            A = reinterpret_cast<const E*>(e.a); B = reinterpret_cast<const E*>(e.b); R = e.rank; scale = e.scale;
        } else {
            R = q.R;
            A = reinterpret_cast<const E*>(q.a) + (size_t)adapter * R * q.K;
            B = reinterpret_cast<const E*>(q.b) + (size_t)adapter * q.N * R;
            scale = p.scale[adapter];
        }
    }
};

template <typename E, int NP>
__global__ void __cluster_dims__(ADP_CTAS, 1, 1) __launch_bounds__(ADT_LOW_THREADS) adapter_low_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ unsigned char smem_any[];
    __shared__ int s_tok[ADT_TOK];
    __shared__ __align__(8) uint64_t s_bar[2 * ADT_STAGES + 1];      // slabs there, slabs read, S complete
    __shared__ uint32_t s_tmem;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cta = blockIdx.x % ADP_CTAS, want = blockIdx.x / ADP_CTAS;
    const AdapterPart& q = p.part[blockIdx.y];
    pdl_wait();
    if (want >= p.plan.count()[1]) return;
    const int4 gr = p.plan.tile()[want];
    const int cnt = gr.z, K = q.K;
    const AdtWeights<E> ad(p, q, gr.x);
    const int R = ad.R;
    if (R == 0) return;
    if (tid < ADT_TOK) s_tok[tid] = tid < cnt ? p.plan.place()[gr.y + tid] : 0;
    // layout by the call's largest rank: all CTAs of a launch agree on it
    const int L = p.rank, stage_bytes = adt_stage(L);
    const uint32_t ring = (smem_u32(smem_any) + 1023u) & ~1023u;
    const int Rn = adt_r16(R);
    const uint32_t full = smem_u32(s_bar), free_bar = full + ADT_STAGES * 8, bar_s = free_bar + ADT_STAGES * 8;
    if (tid == 0) {
        for (int i = 0; i < ADT_STAGES; ++i) {
            mbar_init(full + i * 8, 64);
            mbar_init(free_bar + i * 8, 1);
        }
        mbar_init(bar_s, 1);
        mbar_fence_init();
    }
    if (warp == 0) tc_alloc(smem_u32(&s_tmem), adt_low_columns(L));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    bool fine = true;

    // slabs go to the CTAs in turn: what the cluster reads of a row at a time is one run of it
    const int nk = (K + 63) / 64, slabs = (nk - cta + ADP_CTAS - 1) / ADP_CTAS;
    if (warp < 2 * ADT_STAGES) {
        const E* const x = reinterpret_cast<const E*>(q.x);
        const int slot = warp >> 1, me = tid & 63;
        const uint32_t st = ring + (uint32_t)slot * stage_bytes;
        unsigned pass = 0;
        for (int i = slot; i < slabs; i += ADT_STAGES, ++pass) {
            // (a slab that is still read is not loaded over: its barrier then does not come either, nor S)
            if (pass > 0 && !(fine = adt_bar_wait(free_bar + slot * 8, (pass - 1) & 1u))) break;
            const int k = (i * ADP_CTAS + cta) * 64 + (me & 7) * 8;
            const bool in = k < K;
            const int kk = in ? k : 0;
#pragma unroll 4
            for (int r = me >> 3; r < cnt; r += 8) {
                const int t = s_tok[r];
                adt_cp16(st + adt_swizzled(r, me & 7), q.x_a16 ? x + a16_index(t, kk, q.x_th) : x + (size_t)t * q.x_stride + kk, in);
            }
#pragma unroll 4
            for (int r = me >> 3; r < R; r += 8) adt_cp16(st + ADT_TOK * 128 + adt_swizzled(r, me & 7), ad.A + (size_t)r * K + kk, in);
            asm volatile("cp.async.wait_all;" ::: "memory");
            adt_fence();
            mbar_arrive(full + slot * 8);
        }
    } else if (lane == 0) {
        const uint32_t idesc = adt_idesc<E>(128, Rn);
        for (int i = 0; i < slabs; ++i) {
            const int slot = i % ADT_STAGES;
            if (!(fine = adt_bar_wait(full + slot * 8, (uint32_t)(i / ADT_STAGES) & 1u))) break;
            tc_fence_after();
            const uint32_t st = ring + (uint32_t)slot * stage_bytes;
#pragma unroll
            for (int k = 0; k < 4; ++k) tc_mma_f16(tmem, adt_desc(st + k * 32), adt_desc(st + ADT_TOK * 128 + k * 32), idesc, i > 0 || k > 0);
            tc_commit(free_bar + slot * 8);
        }
        if (fine) tc_commit(bar_s);
    }
    fine = fine && adt_bar_wait(bar_s, 0);
    if (!fine) adt_bar_wait(bar_s, 0);               // (the slabs are not written over while another thread may still see the products end)
    __syncwarp();
    tc_fence_after();

    // ---- the partial sums, a token's ranks in a row: the pitch keeps both its writers (a lane a token) and its readers (a lane four ranks) off one another's banks ----
    const int pitch = Rn + 4;
    float* const exch = reinterpret_cast<float*>(smem_any + (ring - smem_u32(smem_any)));
    {
        const int row = (warp & 3) * 32 + lane;
        for (int c = (warp >> 2) * 16; warp < 8 && c < Rn; c += 32) {
            float v[16];
            if (slabs > 0) {
                __syncwarp();
                tc_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c, v);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0.f;
            }
            if (!fine) v[0] = __int_as_float(0x7fc00000);        // (one rank of the thread's token is enough)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<float4*>(exch + row * pitch + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
        tc_fence_before();
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // (of the arrival at the start)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

    // ---- sixteen tokens, sixteen threads each: sum, scale, parts ----
    {
        constexpr int V4 = ADP_MAX_RANK / 4 / 16, MINE = ADT_TOK / ADP_CTAS;
        const int sub = tid % 16, tok = cta * MINE + tid / 16;
        const bool work = tid < 16 * MINE && tok < cnt;
        float4 s[V4];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < V4; ++i) {
            const int r4 = sub + i * 16;
            s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (work && r4 * 4 < R) {
                const uint32_t at = smem_u32(exch + tok * pitch + r4 * 4);
                float4 v[ADP_CTAS];
#pragma unroll
                for (int c = 0; c < ADP_CTAS; ++c) {
                    uint32_t remote;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(c));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[c].x), "=f"(v[c].y), "=f"(v[c].z), "=f"(v[c].w) : "r"(remote) : "memory");
                }
#pragma unroll
                for (int c = 0; c < ADP_CTAS; ++c) { s[i].x += v[c].x; s[i].y += v[c].y; s[i].z += v[c].z; s[i].w += v[c].w; }
                s[i].x *= ad.scale; s[i].y *= ad.scale; s[i].z *= ad.scale; s[i].w *= ad.scale;
            }
            top = fmaxf(fmaxf(fmaxf(top, fabsf(s[i].x)), fmaxf(fabsf(s[i].y), fabsf(s[i].z))), fabsf(s[i].w));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const unsigned ex = min(max((__float_as_uint(top) >> 23) & 255u, 2u), 252u);
        const float down = __uint_as_float((254u - ex) << 23), back = __uint_as_float(ex << 23);
        if (work) {
            uint8_t* const low = p.low + (size_t)blockIdx.y * adt_low_bytes(p.tokens, L, NP);
            const int at = gr.y + tok;
#pragma unroll
            for (int i = 0; i < V4; ++i) {
                const int r = (sub + i * 16) * 4;
                if (r >= Rn) continue;               // (zeros from the rank to the next multiple of 16)
                float left[4] = {s[i].x * down, s[i].y * down, s[i].z * down, s[i].w * down};
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    uint2 h;
                    E* const e = reinterpret_cast<E*>(&h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        e[j] = AdpType<E>::round(left[j]);
                        const float w = AdpType<E>::widen(e[j]);
                        left[j] = fabsf(w) < INFINITY ? left[j] - w : 0.f;
                    }
                    *reinterpret_cast<uint2*>(low + ((size_t)(k * adt_chunks(L) + r / 64) * p.tokens + at) * 128 + (r % 64) * 2) = h;
                }
            }
            if (sub == 0) *reinterpret_cast<float*>(low + (size_t)NP * adt_chunks(L) * p.tokens * 128 + (size_t)at * 4) = back;
        }
    }
    // no CTA leaves while another may read its sums
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) tc_dealloc(tmem, adt_low_columns(L));
}

template <typename E, typename O>
__global__ void __launch_bounds__(ADT_THREADS, 2) adapter_out_kernel(const __grid_constant__ AdapterParams p) {
    constexpr int NP = AdpParts<E, O>::N;
    extern __shared__ unsigned char smem_any[];
    __shared__ longlong2 s_at[3][ADT_TOK];           // elements to the tokens' rows of base and out: of this unit, the next, and the last, which a warp may still write
    __shared__ float s_back[3][ADT_TOK];
    __shared__ int4 s_tiles[ADT_TABLE];
    __shared__ __align__(8) uint64_t s_bar[2];
    __shared__ uint32_t s_tmem;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int L = p.rank, TT = p.out_tokens;
    const uint32_t oper = (smem_u32(smem_any) + 1023u) & ~1023u, wts = oper + adt_operand(L, NP);
    float* const rows = reinterpret_cast<float*>(smem_any + (wts + adt_weights(L) - smem_u32(smem_any)));
    const uint32_t bar = smem_u32(s_bar);
    if (tid == 0) {
        mbar_init(bar, 1);
        mbar_init(bar + 8, 1);
        mbar_fence_init();
    }
    pdl_wait();
    if (warp == 0) tc_alloc(smem_u32(&s_tmem), 2 * TT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    const int tiles = p.plan.count()[1];
    const size_t low_bytes = adt_low_bytes(p.tokens, L, NP);
    for (int i = tid; i < min(tiles, ADT_TABLE); i += ADT_THREADS) s_tiles[i] = p.plan.tile()[i];
    __syncthreads();

    struct Unit {
        const E* w;                                  // the unit's rows of B
        const O* base;                               // its first output of token 0
        O* out;
        const uint8_t* low;                          // S of its first token
        long long base_stride, out_stride;
        int cnt, first, left, R;                     // left: outputs from its first on
        bool vec;
    };
    // where the CTA is: projection, tile (in pieces of TT tokens), block of outputs
    const int sub_log = TT == 128 ? 0 : (TT == 64 ? 1 : 2);
    int part = 0, ts = 0, block = blockIdx.x, nb = (p.part[0].N + 127) / 128;
    // the unit there, or the next one of the CTA that has something to do; and on to the one behind it
    auto fetch = [&](Unit& x) {
        while (part < p.nparts) {
            while (block >= nb) {
                block -= nb;
                ++ts;
            }
            const int tile = ts >> sub_log;
            if (tile >= tiles) {
                // the rest of the way in blocks of the next projection
                const long long over = (long long)(ts - (tiles << sub_log)) * nb + block;
                if (++part == p.nparts) break;
                nb = (p.part[part].N + 127) / 128;
                ts = (int)(over / nb);
                block = (int)(over % nb);
                continue;
            }
            const AdapterPart& q = p.part[part];
            const int n0 = block * 128, skip = (ts - (tile << sub_log)) * TT;
            block += gridDim.x;
            const int4 gr = tile < ADT_TABLE ? s_tiles[tile] : p.plan.tile()[tile];
            x.cnt = min(TT, gr.z - skip);
            if (x.cnt <= 0) continue;
            const AdtWeights<E> ad(p, q, gr.x);
            if (ad.R == 0 && (!p.copy || (q.base == q.out && q.base_stride == q.out_stride))) continue;
            x.R = ad.R;
            x.w = ad.B + (size_t)n0 * ad.R;
            x.base = q.base ? reinterpret_cast<const O*>(q.base) + n0 : nullptr;
            x.out = reinterpret_cast<O*>(q.out) + n0;
            x.base_stride = q.base_stride; x.out_stride = q.out_stride;
            x.first = gr.y + skip;
            x.low = p.low + (size_t)part * low_bytes + (size_t)x.first * 128;
            x.left = q.N - n0;
            x.vec = q.vec && x.left >= 128;
            return true;
        }
        return false;
    };
    const size_t tile_bytes = (size_t)p.tokens * 128;        // of 64 ranks of S
    // a thread: 16 bytes at one place of every 32nd row
    const int c16 = tid & 7, r8 = tid >> 3;
    const uint32_t swz = adt_swizzled(r8, c16);              // (rows 32 apart: 4096 bytes further)
    auto load_operands = [&](const Unit& x) {
        const int have = min(128, x.left), r16 = adt_r16(x.R);
        for (int r0 = 0; r0 < r16; r0 += 64) {
            const int rank = r0 + c16 * 8;
            if (rank >= r16) continue;
            const bool real = rank < x.R;
            const E* w = x.w + r8 * x.R + (real ? rank : 0);
            const uint32_t to = wts + (r0 >> 6) * (128 * 128) + swz;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (r8 + i * 32 < have) adt_cp16(to + i * 4096, w, real);
                w += 32 * x.R;
            }
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                const int tile = k * adt_chunks(L) + (r0 >> 6);
                const uint8_t* const s = x.low + tile * tile_bytes + r8 * 128 + c16 * 16;
                const uint32_t at = oper + (uint32_t)tile * (TT * 128) + swz;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r8 + i * 32 < x.cnt) adt_cp16(at + i * 4096, s + i * 4096, true);
            }
        }
    };
    auto multiply = [&](const Unit& x, unsigned use) {       // one thread
        tc_fence_after();
        const uint32_t idesc = adt_idesc<E>(128, (x.cnt + 15) & ~15), d = tmem + (use & 1u) * TT;
        uint32_t accumulate = 0;
        for (int k = 0; k < NP; ++k)
            for (int r = 0; r < x.R; r += 16) {
                tc_mma_f16(d, adt_desc(wts + (r / 64) * (128 * 128) + (r % 64) * 2), adt_desc(oper + (uint32_t)(k * adt_chunks(L) + r / 64) * (TT * 128) + (r % 64) * 2), idesc,
                           accumulate);
                accumulate = 1;
            }
        tc_commit(bar + (use & 1u) * 8);
    };
    auto token_of = [&](const Unit& x) { return tid < x.cnt ? p.plan.place()[x.first + tid] : 0; };
    auto back_of = [&](const Unit& x) {
        return x.R && tid < x.cnt ? *reinterpret_cast<const float*>(x.low + NP * adt_chunks(L) * tile_bytes - (size_t)x.first * 124 + tid * 4) : 0.f;
    };
    // a thread's token: where its rows are; its base is asked of L2
    auto place_token = [&](const Unit& x, int buf, int t, float back) {
        if (tid >= x.cnt) return;
        s_at[buf][tid] = make_longlong2((long long)t * x.base_stride, (long long)t * x.out_stride);
        s_back[buf][tid] = back;
        if (x.base) {
            const O* const row = x.base + (long long)t * x.base_stride;
#pragma unroll
            for (int i = 0; i < (int)sizeof(O); ++i)
                if (i * (128 / (int)sizeof(O)) < x.left) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + i * (128 / (int)sizeof(O))));
        }
    };
    // base of four tokens of the 32, four outputs a lane, as they lie in memory: widened where they are used, or the loads would be waited for here
    constexpr int OWN = ADT_ROWS / (ADT_THREADS / 32);
    using Raw = typename AdpRaw<O>::Four;
    Raw y[OWN];
    auto load_base = [&](const Unit& x, int buf, int c) {
        const int t0 = c + warp * OWN;
        const O* const from = x.base + lane * 4;
        if (!x.base) {
#pragma unroll
            for (int i = 0; i < OWN; ++i) y[i] = Raw{};
        } else if (x.vec) {
#pragma unroll
            for (int i = 0; i < OWN; ++i)
                if (t0 + i < x.cnt) y[i] = *reinterpret_cast<const Raw*>(from + s_at[buf][t0 + i].x);
        } else {
            // (loops, not predicated code beside the accesses above)
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                Raw r{};
                O* const e = reinterpret_cast<O*>(&r);
                if (t0 + i < x.cnt) {
                    const O* const at = from + s_at[buf][t0 + i].x;
                    const int n = min(4, x.left - lane * 4);
#pragma unroll 1
                    for (int k = 0; k < n; ++k) {
                        const O o = at[k];
                        if (k == 0) e[0] = o;
                        else if (k == 1) e[1] = o;
                        else if (k == 2) e[2] = o;
                        else e[3] = o;
                    }
                }
                y[i] = r;
            }
        }
    };
#pragma unroll
    for (int i = 0; i < OWN; ++i) y[i] = Raw{};

    bool fine = true;
    unsigned uses = 0, pass = 0;                     // accumulators and buffers of rows so far
    int buf = 0;
    Unit cur;
    bool have = fetch(cur);
    if (have) {
        if (cur.R) load_operands(cur);
        place_token(cur, 0, token_of(cur), back_of(cur));
        asm volatile("cp.async.wait_all;" ::: "memory");
        adt_fence();
    }
    __syncthreads();
    if (have) {
        if (cur.R && tid == 0) multiply(cur, 0);
        load_base(cur, 0, 0);
    }
    while (have) {
        Unit next;
        const bool more = fetch(next);
        const int buf_next = buf == 2 ? 0 : buf + 1;
        int t_next = 0;
        float back_next = 0.f;
        if (cur.R) {
            fine = fine && adt_bar_wait(bar + (uses & 1u) * 8, (uses >> 1) & 1u);
            if (!fine)                               // (no one reads them before all have come through the barrier below)
                for (int i = 0; i < cur.cnt; ++i) s_back[buf][i] = __int_as_float(0x7fc00000);
            __syncwarp();
            tc_fence_after();
        }
        if (more) {
            t_next = token_of(next);
            back_next = back_of(next);
            if (next.R && cur.cnt <= ADT_ROWS) load_operands(next);         // (this unit's product has read its own)
        }
        for (int c = 0; c < cur.cnt; c += ADT_ROWS) {
            const bool last = c + ADT_ROWS >= cur.cnt;
            float* const st = rows + (pass & 1u) * ADT_ROWS * ADT_PITCH;
            if (cur.R) {
                const int half = (warp >> 2) * 16;
                if (c + half < cur.cnt) {
                    float v[16];
                    tc_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uses & 1u) * TT + c + half, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[(half + i) * ADT_PITCH + (warp & 3) * 32 + lane] = v[i];
                }
                ++pass;
            }
            if (last && more) {
                place_token(next, buf_next, t_next, back_next);
                asm volatile("cp.async.wait_all;" ::: "memory");
                adt_fence();
                tc_fence_before();
            }
            if (cur.R || last) __syncthreads();
            if (last && more && next.R && tid == 0) multiply(next, uses + (cur.R ? 1u : 0u));
            const int t0 = warp * OWN;
            float w[OWN][4];
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                AdpRaw<O>::widen(y[i], w[i]);
                if (!cur.R) continue;
                const float back = s_back[buf][(c + t0 + i) & (ADT_TOK - 1)];
                const float4 x = *reinterpret_cast<const float4*>(st + (t0 + i) * ADT_PITCH + lane * 4);
                w[i][0] = fmaf(x.x, back, w[i][0]);
                w[i][1] = fmaf(x.y, back, w[i][1]);
                w[i][2] = fmaf(x.z, back, w[i][2]);
                w[i][3] = fmaf(x.w, back, w[i][3]);
            }
            if (!last) load_base(cur, buf, c + ADT_ROWS);
            else if (more) load_base(next, buf_next, 0);
            O* const to = cur.out + lane * 4;
            if (cur.vec) {
#pragma unroll
                for (int i = 0; i < OWN; ++i)
                    if (c + t0 + i < cur.cnt) adp_store4(to + s_at[buf][c + t0 + i].y, w[i]);
            } else {
#pragma unroll
                for (int i = 0; i < OWN; ++i) {
                    const int n = c + t0 + i < cur.cnt ? min(4, cur.left - lane * 4) : 0;
#pragma unroll 1
                    for (int e = 0; e < n; ++e) adp_put(to + s_at[buf][c + t0 + i].y + e, e == 0 ? w[i][0] : (e == 1 ? w[i][1] : (e == 2 ? w[i][2] : w[i][3])));
                }
            }
            if (c == 0 && !last && more && next.R) load_operands(next);
        }
        if (cur.R) ++uses;
        cur = next;
        have = more;
        buf = buf_next;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tc_dealloc(tmem, 2 * TT);
}

}  // namespace b200

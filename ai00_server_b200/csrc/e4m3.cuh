// Rows in 8-bit floating point (e4m3) with a scale for every 128 columns of a row, or for every block of 128 x 128: as they are, or behind a root-mean-square
// norm that first adds the residual:
//     h = x + residual (f32; handed on rounded to the residual's type),  y = h rsqrt(mean(h^2) + eps) (offset + weight)
//     s = max(max |y| over the group, 2^-100) / 448,  q = y / s rounded once, to nearest
// (the floor keeps 1 / s a number; a group of zeros is zeros.)
//
// Bound: memory, each value read once and written once, as far as the instructions let it: two divisions for every scale in all of its lanes, conversions two values at a time, sixteen columns
// of a scale to a lane where no row has to stay.  Measured, with inputs larger than L2: rows of 4096 bf16 (14336 of them) 29 us, 6.0 TB/s, as a plain copy of these bytes (sixteen lanes of eight
// columns, two to a thread: 35); blocks 28 us, 6.4 TB/s (with a test at every load and widened values kept instead of made again: 65).
// A row of the norm stays in the registers of its CTA between the statistics and the outputs.  Few rows take a thread for every eight columns (latency).  Many rows: CTAs that stay, sixteen
// columns a thread, with the next row on its way while one is worked on and the weights kept: 2048 rows of 4096, residual and all in bf16, 12.7 us, 4.6 TB/s (a CTA a row 15.7;
// a copy of these bytes 12.2).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace b200 {

constexpr int E4_GROUP = 128;                    // columns of a scale
constexpr float E4_TOP = 448.f;                  // the largest number
constexpr int NORM_MAX_WIDTH = 32768;            // 512 threads of 64 columns

template <typename E> __device__ __forceinline__ float e4_widen(E v);
template <> __device__ __forceinline__ float e4_widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float e4_widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float e4_widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename E> __device__ __forceinline__ E e4_round(float v);
template <> __device__ __forceinline__ float e4_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half e4_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 e4_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// eight neighbouring values as they lie in memory
template <typename E> struct E4Raw { uint4 u[sizeof(E) * 8 / 16]; };
// eight values from p on, of which n are there (the others read as zeros); whole: all are there, on a boundary of 16 bytes
template <typename E>
__device__ __forceinline__ E4Raw<E> e4_load(const E* p, int n, bool whole) {
    E4Raw<E> r;
    if (whole) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
        E e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : e4_round<E>(0.f);
        memcpy(&r, e, sizeof(r));
    }
    return r;
}
template <typename E>
__device__ __forceinline__ void e4_values(const E4Raw<E>& r, float (&v)[8]) {
    if constexpr (std::is_same_v<E, __nv_bfloat16>) {
        const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
        E e[8];
        memcpy(e, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e4_widen<E>(e[i]);
    }
}
// eight values rounded, two at a time
template <typename E>
__device__ __forceinline__ E4Raw<E> e4_rounded(const float (&v)[8]) {
    E4Raw<E> r;
    if constexpr (std::is_same_v<E, float>) {
        memcpy(&r, v, sizeof(r));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<E, __half>) {
                const __half2 two = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                memcpy(&w[i], &two, 4);
            } else {
                const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                memcpy(&w[i], &two, 4);
            }
        }
        r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}
template <typename E>
__device__ __forceinline__ void e4_store(E* p, const float (&v)[8], int n, bool whole) {
    const E4Raw<E> r = e4_rounded<E>(v);
    if (whole) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.u[i];
    } else {
        E e[8];
        memcpy(e, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = e[i];
    }
}
// eight values times inv as e4m3.  (satfinite: the group's largest times the rounded reciprocal may come out a hair above 448; NaN stays NaN)
__device__ __forceinline__ uint2 e4_pack(const float (&v)[8], float inv) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}
__device__ __forceinline__ void e4_put(uint8_t* p, uint2 q, int n, bool whole) {
    if (whole) {
        *reinterpret_cast<uint2*>(p) = q;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}
__device__ __forceinline__ float e4_most(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    return m;
}
__device__ __forceinline__ float e4_scale(float most) { return fmaxf(most, 0x1p-100f) / E4_TOP; }

struct NormParams {
    const void* x;
    long long x_stride;              // elements, as all strides here
    const void* residual;            // null: none
    long long residual_stride;
    void* residual_out;
    long long residual_out_stride;
    const void* weight;              // null: ones
    int weight_type;                 // B200RWKV_TYPE_*
    void* out;
    long long out_stride;
    float* scale;                    // [rows][groups]; null: `out` has the type of x
    int rows, width, groups;
    float eps, offset;
    int vec;                         // eights of a row lie on 16-byte boundaries in x, residual, residual_out and weight
    int vec_out;                     // and, as they have to, in out
};

// E: x; R: residual and the sum that is handed on.  NV: eights of a thread; MANY: a CTA takes row after row, all of whole eights
constexpr int NORM_MANY_THREADS = 256;
template <typename E, typename R> constexpr int norm_many_per_sm() { return sizeof(E) == 4 || sizeof(R) == 4 ? 2 : 3; }         // CTAs of so many threads
template <typename E, typename R, int NV, bool MANY>
__global__ void __launch_bounds__(MANY ? NORM_MANY_THREADS : (NV == 1 ? 1024 : 512), MANY ? norm_many_per_sm<E, R>() : 1) rms_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float red[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const bool add = p.residual != nullptr;
    auto column = [&](int k) { return (k * (int)blockDim.x + tid) * 8; };
    auto whole_in = [&](int n) { return MANY || (p.vec && n >= 8); };
    E4Raw<E> a[NV];
    E4Raw<R> b[NV];
    auto fetch = [&](int row) {
        const E* const x = reinterpret_cast<const E*>(p.x) + row * p.x_stride;
        const R* const res = reinterpret_cast<const R*>(p.residual) + row * p.residual_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = column(k), n = p.width - c;
            if (n <= 0) continue;
            a[k] = e4_load<E>(x + c, n, whole_in(n));
            if (add) b[k] = e4_load<R>(res + c, n, whole_in(n));
        }
    };
    auto weights = [&](int k, float (&g)[8]) {   // offset + weight
        const int c = column(k), n = p.width - c;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = 1.f;
        if (n > 0 && p.weight) {
            if (p.weight_type == B200RWKV_TYPE_F32) e4_values<float>(e4_load<float>(reinterpret_cast<const float*>(p.weight) + c, n, whole_in(n)), g);
            else if (p.weight_type == B200RWKV_TYPE_F16) e4_values<__half>(e4_load<__half>(reinterpret_cast<const __half*>(p.weight) + c, n, whole_in(n)), g);
            else e4_values<__nv_bfloat16>(e4_load<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(p.weight) + c, n, whole_in(n)), g);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] += p.offset;
    };
    pdl_wait();
    int row = blockIdx.x;
    fetch(row);
    constexpr bool EARLY = NV <= 4;              // (wider rows have no registers left for these while they are summed up)
    float g[EARLY ? NV : 1][8];
    if (EARLY) {
#pragma unroll
        for (int k = 0; k < NV; ++k) weights(k, g[k]);
    }
    for (int turn = 0;; ++turn) {
        float h[NV][8];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (p.width - column(k) <= 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[k][i] = 0.f;
                continue;
            }
            e4_values<E>(a[k], h[k]);
            if (add) {
                float r[8];
                e4_values<R>(b[k], r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[k][i] += r[i];
            }
        }
        const int next = row + (int)gridDim.x;
        if (MANY && next < p.rows) fetch(next);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(h[k][i], h[k][i], sum);
        sum = warp_sum(sum);
        if (lane == 0) red[turn & 1][warp] = sum;          // (two, so that one barrier a row is enough)
        __syncthreads();
        sum = warp_sum(lane < warps ? red[turn & 1][lane] : 0.f);
        const float over = rsqrtf(sum / (float)p.width + p.eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = column(k), n = p.width - c;
            // (all sixteen lanes of a scale take part in its maximum, those behind the row with zeros)
            const bool whole = whole_in(n), whole_out = MANY || (p.vec_out && n >= 8);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = 0.f;
            if (n > 0) {
                if (add) e4_store<R>(reinterpret_cast<R*>(p.residual_out) + row * p.residual_out_stride + c, h[k], n, whole);
                if (!EARLY) weights(k, g[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (whole || i < n) y[i] = h[k][i] * over * g[EARLY ? k : 0][i];
            }
            if (p.scale) {
                float most = e4_most(y);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float s = e4_scale(most);
                if (n > 0) {
                    e4_put(reinterpret_cast<uint8_t*>(p.out) + row * p.out_stride + c, e4_pack(y, __frcp_rn(s)), n, whole_out);
                    if ((lane & 15) == 0) p.scale[(long long)row * p.groups + c / E4_GROUP] = s;
                }
            } else if (n > 0) {
                e4_store<E>(reinterpret_cast<E*>(p.out) + row * p.out_stride + c, y, n, whole_out);
            }
        }
        row = next;
        if (!MANY || row >= p.rows) break;
    }
}

struct E4Params {
    const void* x;
    long long x_stride;
    uint8_t* out;
    long long out_stride;
    float* scale;                    // [rows, or blocks of 128 rows][groups]
    int rows, width, groups;
    int vec;                         // eights of a row lie on 16-byte boundaries in x, on 8-byte ones in out; 2: sixteens of out on 16-byte ones
};

constexpr int E4_THREADS = 256, E4_PER_ROW = E4_GROUP / 16;         // lanes of a scale in a row
// a scale for 128 columns of a row: eight lanes of sixteen columns.  They lie one behind another over the rows
template <typename E>
__global__ void __launch_bounds__(E4_THREADS) e4_rows_kernel(const __grid_constant__ E4Params p) {
    pdl_wait();
    const unsigned per_row = (unsigned)p.groups * E4_PER_ROW;
    const unsigned long long at = (unsigned long long)blockIdx.x * E4_THREADS + threadIdx.x;
    const unsigned row = at >> 32 ? (unsigned)(at / per_row) : (unsigned)at / per_row;
    const int col = (int)(unsigned)(at - (unsigned long long)row * per_row) * 16, n = row < (unsigned)p.rows ? p.width - col : 0;
    const E* const x = reinterpret_cast<const E*>(p.x) + (long long)row * p.x_stride + col;
    auto whole = [&](int left) { return p.vec && left >= 8; };
    E4Raw<E> a[2];
    float v[2][8], most = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (n > 8 * j) a[j] = e4_load<E>(x + 8 * j, n - 8 * j, whole(n - 8 * j));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
        if (n > 8 * j) e4_values<E>(a[j], v[j]);
        most = fmaxf(most, e4_most(v[j]));
    }
#pragma unroll
    for (int o = E4_PER_ROW / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float s = e4_scale(most), inv = __frcp_rn(s);
    if (n <= 0) return;
    uint8_t* const out = p.out + (long long)row * p.out_stride + col;
    const uint2 q[2] = {e4_pack(v[0], inv), e4_pack(v[1], inv)};
    if (p.vec > 1 && n >= 16) {
        *reinterpret_cast<uint4*>(out) = make_uint4(q[0].x, q[0].y, q[1].x, q[1].y);
    } else {
        e4_put(out, q[0], n, whole(n));
        e4_put(out + 8, q[1], n - 8, whole(n - 8));
    }
    if (threadIdx.x % E4_PER_ROW == 0) p.scale[(long long)row * p.groups + col / E4_GROUP] = s;
}

// the same bits, of which the compiler knows nothing: what was made of them is made again instead of kept
template <typename E>
__device__ __forceinline__ void e4_anew(E4Raw<E>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) asm volatile("" : "+r"(r.u[i].x), "+r"(r.u[i].y), "+r"(r.u[i].z), "+r"(r.u[i].w));
}

// a scale for a block of 128 x 128: a CTA, in its registers; sixteen lanes along a row, sixteen rows at a time
template <typename E>
__global__ void __launch_bounds__(E4_THREADS, sizeof(E) == 4 ? 2 : 4) e4_blocks_kernel(const __grid_constant__ E4Params p) {
    __shared__ float red[E4_THREADS / 32];
    constexpr int ROWS = E4_THREADS / 16, N = E4_GROUP / ROWS;
    pdl_wait();
    const int g = blockIdx.x % p.groups, b = blockIdx.x / p.groups, c = g * E4_GROUP + (threadIdx.x & 15) * 8, n = p.width - c;
    const long long first = (long long)b * E4_GROUP + (threadIdx.x >> 4);
    const E* const x = reinterpret_cast<const E*>(p.x) + first * p.x_stride + c;
    uint8_t* const out = p.out + first * p.out_stride + c;
    auto work = [&](auto inside) {               // whether all rows and columns are
        constexpr bool INSIDE = decltype(inside)::value;
        const bool whole = INSIDE || (p.vec && n >= 8);
        auto there = [&](int i) { return INSIDE || (first + i * ROWS < p.rows && n > 0); };
        E4Raw<E> a[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (there(i)) a[i] = e4_load<E>(x + i * ROWS * p.x_stride, n, whole);
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!there(i)) continue;
            float v[8];
            e4_values<E>(a[i], v);
            most = fmaxf(most, e4_most(v));
            e4_anew(a[i]);
        }
        most = warp_max(most);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
        __syncthreads();
        most = 0.f;
#pragma unroll
        for (int i = 0; i < E4_THREADS / 32; ++i) most = fmaxf(most, red[i]);
        const float s = e4_scale(most), inv = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!there(i)) continue;
            float v[8];
            e4_values<E>(a[i], v);
            e4_put(out + i * ROWS * p.out_stride, e4_pack(v, inv), n, whole);
        }
        if (threadIdx.x == 0) p.scale[(long long)b * p.groups + g] = s;
    };
    if (p.vec && (g + 1) * E4_GROUP <= p.width && (b + 1) * E4_GROUP <= p.rows) work(std::true_type{});
    else work(std::false_type{});
}

}  // namespace b200

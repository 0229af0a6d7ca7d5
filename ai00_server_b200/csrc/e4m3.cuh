// Rows in 8-bit floating point (e4m3) with a scale for every 128 columns of a row, or for every block of 128 x 128: as they are, or behind a root-mean-square
// norm that first adds the residual:
//     h = x + residual (f32; handed on rounded to the residual's type),  y = h rsqrt(mean(h^2) + eps) (offset + weight)
//     s = max(max |y| over the group, 2^-100) / 448,  q = y / s rounded once, to nearest
// (the floor keeps 1 / s a number; a group of zeros is zeros.)
//
// Bound: memory, each value read once and written once.  A row of the norm stays in the registers of its CTA between the statistics and the outputs; sixteen lanes
// hold the 128 columns of a scale, so that its maximum is four exchanges.  Few rows take a thread for every eight columns (latency), many rows 16 or 32 columns a
// thread, so that several rows are in flight on an SM.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

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
    E e[8];
    memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e4_widen<E>(e[i]);
}
template <typename E>
__device__ __forceinline__ void e4_store(E* p, const float (&v)[8], int n, bool whole) {
    E e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = e4_round<E>(v[i]);
    if (whole) {
        E4Raw<E> r;
        memcpy(&r, e, sizeof(r));
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.u[i];
    } else {
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
    int width, groups;
    float eps, offset;
    int vec;                         // eights of a row lie on 16-byte boundaries in x, residual, residual_out and weight
    int vec_out;                     // and, as they have to, in out
};

// E: x; R: residual and the sum that is handed on (void where there is none).  NV: eights of a thread
template <typename E, typename R, int NV>
__global__ void __launch_bounds__(NV == 1 ? 1024 : 512) rms_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float red[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const long long row = blockIdx.x;
    pdl_wait();
    const E* const x = reinterpret_cast<const E*>(p.x) + row * p.x_stride;
    const R* const res = p.residual ? reinterpret_cast<const R*>(p.residual) + row * p.residual_stride : nullptr;
    auto column = [&](int k) { return (k * (int)blockDim.x + tid) * 8; };
    float h[NV][8];
    {
        E4Raw<E> a[NV];
        E4Raw<R> b[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = column(k), n = p.width - c;
            const bool whole = p.vec && n >= 8;
            if (n > 0) {
                a[k] = e4_load<E>(x + c, n, whole);
                if (res) b[k] = e4_load<R>(res + c, n, whole);
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (p.width - column(k) <= 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[k][i] = 0.f;
                continue;
            }
            e4_values<E>(a[k], h[k]);
            if (res) {
                float r[8];
                e4_values<R>(b[k], r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[k][i] += r[i];
            }
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(h[k][i], h[k][i], sum);
    sum = warp_sum(sum);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    sum = warp_sum(lane < warps ? red[lane] : 0.f);
    const float over = rsqrtf(sum / (float)p.width + p.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = column(k), n = p.width - c;
        // (all sixteen lanes of a scale take part in its maximum, those behind the row with zeros)
        const bool whole = p.vec && n >= 8, whole_out = p.vec_out && n >= 8;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 0.f;
        if (n > 0) {
            if (res) e4_store<R>(reinterpret_cast<R*>(p.residual_out) + row * p.residual_out_stride + c, h[k], n, whole);
            float w[8];
            if (!p.weight) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = 1.f;
            } else if (p.weight_type == 0) {
                e4_values<float>(e4_load<float>(reinterpret_cast<const float*>(p.weight) + c, n, whole), w);
            } else if (p.weight_type == 1) {
                e4_values<__half>(e4_load<__half>(reinterpret_cast<const __half*>(p.weight) + c, n, whole), w);
            } else {
                e4_values<__nv_bfloat16>(e4_load<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(p.weight) + c, n, whole), w);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (whole || i < n) y[i] = h[k][i] * over * (p.offset + w[i]);
        }
        if (p.scale) {
            float most = e4_most(y);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float s = e4_scale(most);
            if (n > 0) {
                e4_put(reinterpret_cast<uint8_t*>(p.out) + row * p.out_stride + c, e4_pack(y, 1.f / s), n, whole_out);
                if ((lane & 15) == 0) p.scale[row * p.groups + c / E4_GROUP] = s;
            }
        } else if (n > 0) {
            e4_store<E>(reinterpret_cast<E*>(p.out) + row * p.out_stride + c, y, n, whole_out);
        }
    }
}

struct E4Params {
    const void* x;
    long long x_stride;
    uint8_t* out;
    long long out_stride;
    float* scale;                    // [rows, or blocks of 128 rows][groups]
    int rows, width, groups;
    int vec;                         // eights of a row lie on 16-byte boundaries in x, on 8-byte ones in out
};

// a scale for 128 columns of a row: sixteen lanes.  Units of eight columns lie one behind another over the rows; a thread has U of them, a CTA apart
constexpr int E4_THREADS = 256, E4_UNITS = 2;
template <typename E>
__global__ void __launch_bounds__(E4_THREADS) e4_rows_kernel(const __grid_constant__ E4Params p) {
    pdl_wait();
    const unsigned per_row = (unsigned)p.groups * 16u;
    const unsigned long long first = (unsigned long long)blockIdx.x * (E4_THREADS * E4_UNITS) + threadIdx.x;
    E4Raw<E> a[E4_UNITS];
    unsigned row[E4_UNITS];
    int col[E4_UNITS];
#pragma unroll
    for (int u = 0; u < E4_UNITS; ++u) {
        const unsigned long long at = first + (unsigned long long)u * E4_THREADS;
        row[u] = at >> 32 ? (unsigned)(at / per_row) : (unsigned)at / per_row;
        col[u] = (int)(unsigned)(at - (unsigned long long)row[u] * per_row) * 8;
        if (row[u] < (unsigned)p.rows && col[u] < p.width)
            a[u] = e4_load<E>(reinterpret_cast<const E*>(p.x) + (long long)row[u] * p.x_stride + col[u], p.width - col[u], p.vec && p.width - col[u] >= 8);
    }
#pragma unroll
    for (int u = 0; u < E4_UNITS; ++u) {
        const bool real = row[u] < (unsigned)p.rows && col[u] < p.width;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (real) e4_values<E>(a[u], v);
        float most = e4_most(v);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float s = e4_scale(most);
        if (!real) continue;
        e4_put(p.out + (long long)row[u] * p.out_stride + col[u], e4_pack(v, 1.f / s), p.width - col[u], p.vec && p.width - col[u] >= 8);
        if ((threadIdx.x & 15) == 0) p.scale[(long long)row[u] * p.groups + col[u] / E4_GROUP] = s;
    }
}

// a scale for a block of 128 x 128: a CTA, in its registers; sixteen lanes along a row, sixteen rows at a time
template <typename E>
__global__ void __launch_bounds__(E4_THREADS) e4_blocks_kernel(const __grid_constant__ E4Params p) {
    __shared__ float red[E4_THREADS / 32];
    constexpr int ROWS = E4_THREADS / 16, N = E4_GROUP / ROWS;
    pdl_wait();
    const int g = blockIdx.x % p.groups, b = blockIdx.x / p.groups, c = g * E4_GROUP + (threadIdx.x & 15) * 8, n = p.width - c;
    const bool whole = p.vec && n >= 8;
    E4Raw<E> a[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long row = (long long)b * E4_GROUP + i * ROWS + (threadIdx.x >> 4);
        if (row < p.rows && n > 0) a[i] = e4_load<E>(reinterpret_cast<const E*>(p.x) + row * p.x_stride + c, n, whole);
    }
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long row = (long long)b * E4_GROUP + i * ROWS + (threadIdx.x >> 4);
        if (row >= p.rows || n <= 0) continue;
        float v[8];
        e4_values<E>(a[i], v);
        most = fmaxf(most, e4_most(v));
    }
    most = warp_max(most);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
    __syncthreads();
    most = 0.f;
#pragma unroll
    for (int i = 0; i < E4_THREADS / 32; ++i) most = fmaxf(most, red[i]);
    const float s = e4_scale(most), inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long row = (long long)b * E4_GROUP + i * ROWS + (threadIdx.x >> 4);
        if (row >= p.rows || n <= 0) continue;
        float v[8];
        e4_values<E>(a[i], v);
        e4_put(p.out + row * p.out_stride + c, e4_pack(v, inv), n, whole);
    }
    if (threadIdx.x == 0) p.scale[(long long)b * p.groups + g] = s;
}

}  // namespace b200

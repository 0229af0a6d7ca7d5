// Rows in 8-bit floating point (e4m3) with a scale for every 128 columns of a row, or for every block of 128 x 128: as they are, or behind a root-mean-square
// norm that first adds the residual:
//     h = x + residual (f32; handed on rounded to the residual's type),  y = h rsqrt(mean(h^2) + eps) (offset + weight)
//     s = max(max |y| over the group, 2^-100) / 448,  q = y / s
// s and y / s are f32, rounded to nearest, and q is the e4m3 number nearest to that.  (The floor keeps 1 / s a number; a group of zeros is zeros.)
//
// Bound: memory, each value read once and written once, as far as the instructions let it: two divisions for every scale in all of its lanes, conversions two values at a time, sixteen columns
// of a scale to a lane where no row has to stay.  Measured, with inputs larger than L2: rows of 4096 bf16 (14336 of them) 28 us, 6.3 TB/s, as a plain copy of these bytes (sixteen lanes of eight
// columns, two to a thread: 35); blocks 28 us, 6.3 TB/s (with a test at every load and widened values kept instead of made again: 65).
// Rows that start anywhere: a lane has every 32nd column, so that a warp's accesses are runs, all asked for at once (14336 rows of 4095 bf16 with a scale a row 88 us and blocks 62, of which
// eight neighbours a lane, one value at a time, took 141 and 112; 2539 rows of 1364 f16 6.9 and 12.6).
// A row of the norm stays in the registers of its CTA between the statistics and the outputs.  Few rows take a thread for every eight columns (latency; one row of 2560 1.9 us).  Many rows: CTAs
// that stay, sixteen columns a thread, with the next row on its way while one is worked on and the weights kept: 2048 rows of 4096, residual and all in bf16, 12.3 us, 4.8 TB/s (a CTA a row 15.7;
// a copy of as many bytes 11.0; values computed outside the condition behind which they are stored 15.6); rows of 4095 33 (48).
#pragma once
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "f32x2.cuh"
#include "float_types.cuh"

namespace b200 {

constexpr int E4_GROUP = 128;                    // columns of a scale
constexpr float E4_TOP = 448.f;                  // the largest number
constexpr int NORM_MAX_WIDTH = 32768;            // 512 threads of 64 columns

// eight values of a thread as they lie in memory.  EIGHTS: neighbours, on a boundary of 16 bytes.  Else: of 256 columns that a warp has, those of each 32 that are its lane's, so that a
// warp's accesses to rows that start anywhere are runs of 32 columns
template <typename E> struct E4Raw { uint4 u[sizeof(E) * 8 / 16]; };
__device__ __forceinline__ int e4_column(int i) { return (i >> 2) * 128 + (i & 3) * 32; }            // from the lane's first column
// eights: from p on.  Else: p[first + ...], of columns below `width`, whose last stands for those behind it (loads under a condition of their own take as long as one after the other)
template <bool EIGHTS, typename E>
__device__ __forceinline__ E4Raw<E> e4_load(const E* p, int first, int width) {
    E4Raw<E> r;
    if constexpr (EIGHTS) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p + first)[i];
    } else {
        E e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[min(first + e4_column(i), width - 1)];
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
        for (int i = 0; i < 8; ++i) v[i] = widened<E>(e[i]);
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
template <bool EIGHTS, typename E>
__device__ __forceinline__ void e4_store(E* p, int first, int width, const float (&v)[8]) {
    const E4Raw<E> r = e4_rounded<E>(v);
    if constexpr (EIGHTS) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) reinterpret_cast<uint4*>(p + first)[i] = r.u[i];
    } else {
        E e[8];
        memcpy(e, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (first + e4_column(i) < width) p[first + e4_column(i)] = e[i];
    }
}
// What a group's values are divided by: they become the f32 quotient as a division rounds it, to nearest, and that to nearest e4m3, so that the numbers are those that (y / s), converted
// anywhere else, has.  The reciprocal comes in two parts, 1 / s = high + low to 2^-45 of itself: with e = 1 - s high, low = high (e + e^2).  A quotient y high + y low is off by 2^-44 before it
// is rounded: as a division has it for every value of 16 bits (tried out), and for one of f32 but where y / s is that near (2^-30
// where low is denormal, for scales above 2^104) to the middle of two f32 numbers beside a tie.  (The product with a
// rounded reciprocal alone lay a step beside it where a value is on a tie of its group: 5 in 10 000 bf16 weights; 14336 x 4096 in blocks took 28.8 us with it where these take 29.4, and the norm of 2048 x 4096 12.4 and 12.3.)  high stays below 1 / s (the unit's is a step off at most): no low is
// negative, and zeros keep their signs.  An infinite scale makes zeros of numbers and NaN of infinities
struct E4Over { f32x2 high, low; };
__device__ __forceinline__ E4Over e4_over(float s) {
    float high;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(high) : "f"(s));
    high *= 1.f - 0x1p-22f;
    const float e = s < INFINITY ? fmaf(-s, high, 1.f) : 0.f, low = high * fmaf(e, e, e);
    return {pack2(high, high), pack2(low, low)};
}
__device__ __forceinline__ uint32_t e4_two(float a, float b, const E4Over& o) {
    const f32x2 y = pack2(a, b);
    // (satfinite: the group's largest may come out a hair above 448; NaN stays NaN)
    return __nv_cvt_float2_to_fp8x2(unpack2(fmadd2(y, o.high, prod2(y, o.low))), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4_four(const float* v, const E4Over& o) { return e4_two(v[0], v[1], o) | e4_two(v[2], v[3], o) << 16; }
__device__ __forceinline__ uint2 e4_pack(const float (&v)[8], const E4Over& o) { return make_uint2(e4_four(v, o), e4_four(v + 4, o)); }
// four values of a lane, 32 columns apart
__device__ __forceinline__ void e4_put(uint8_t* p, int first, int width, uint32_t q) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (first + 32 * i < width) p[first + 32 * i] = (uint8_t)(q >> (8 * i));
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
};

// E: x; R: residual and the sum that is handed on.  NV: eight values of a thread so many times; EIGHTS: neighbours, on 16-byte boundaries in all rows (out's, too: 8 of 8-bit
// ones); MANY: a CTA takes row after row
constexpr int NORM_MANY_THREADS = 256;
template <typename E, typename R, bool EIGHTS> constexpr int norm_many_per_sm() { return sizeof(E) == 4 || sizeof(R) == 4 || !EIGHTS ? 2 : 3; }         // CTAs of so many threads
template <typename E, typename R, int NV, bool EIGHTS, bool MANY>
__global__ void __launch_bounds__(MANY ? NORM_MANY_THREADS : (NV == 1 ? 1024 : 512), MANY ? norm_many_per_sm<E, R, EIGHTS>() : 1) rms_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float red[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const bool add = p.residual != nullptr;
    auto column = [&](int k) { return EIGHTS ? (k * (int)blockDim.x + tid) * 8 : (k * warps + warp) * 256 + lane; };
    // (a thread none of whose columns are there; others read the last one's)
    auto none = [&](int k) { return EIGHTS && column(k) >= p.width; };
    E4Raw<E> a[NV];
    E4Raw<R> b[NV];
    auto fetch = [&](int row) {
        const E* const x = reinterpret_cast<const E*>(p.x) + row * p.x_stride;
        const R* const res = reinterpret_cast<const R*>(p.residual) + row * p.residual_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (none(k)) continue;
            a[k] = e4_load<EIGHTS, E>(x, column(k), p.width);
            if (add) b[k] = e4_load<EIGHTS, R>(res, column(k), p.width);
        }
    };
    auto weights = [&](int k, float (&g)[8]) {   // offset + weight
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = 1.f;
        if (p.weight && !none(k)) {
            if (p.weight_type == B200RWKV_TYPE_F32) e4_values<float>(e4_load<EIGHTS, float>(reinterpret_cast<const float*>(p.weight), column(k), p.width), g);
            else if (p.weight_type == B200RWKV_TYPE_F16) e4_values<__half>(e4_load<EIGHTS, __half>(reinterpret_cast<const __half*>(p.weight), column(k), p.width), g);
            else e4_values<__nv_bfloat16>(e4_load<EIGHTS, __nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(p.weight), column(k), p.width), g);
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
            if (none(k)) {
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
            if (!EIGHTS) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[k][i] = column(k) + e4_column(i) < p.width ? h[k][i] : 0.f;
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
            const int c = column(k);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = 0.f;
            if (!none(k)) {
                if (add) e4_store<EIGHTS, R>(reinterpret_cast<R*>(p.residual_out) + row * p.residual_out_stride, c, p.width, h[k]);
                if (!EARLY) weights(k, g[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = h[k][i] * over * g[EARLY ? k : 0][i];
            }
            if (!p.scale) {
                if (!none(k)) e4_store<EIGHTS, E>(reinterpret_cast<E*>(p.out) + row * p.out_stride, c, p.width, y);
                continue;
            }
            uint8_t* const out = reinterpret_cast<uint8_t*>(p.out) + row * p.out_stride;
            float* const scale = p.scale + (long long)row * p.groups;
            if (EIGHTS) {                        // (all sixteen lanes of a scale take part in its maximum, those behind the row with zeros)
                float most = e4_most(y);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float s = e4_scale(most);
                if (!none(k)) {
                    *reinterpret_cast<uint2*>(out + c) = e4_pack(y, e4_over(s));
                    if ((lane & 15) == 0) scale[c / E4_GROUP] = s;
                }
            } else {                             // (a warp has two scales; behind the row its values are zeros)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = c + j * E4_GROUP;
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[4 * j + i] = at + 32 * i < p.width ? y[4 * j + i] : 0.f;
                    const float most = warp_max(fmaxf(fmaxf(fabsf(y[4 * j]), fabsf(y[4 * j + 1])), fmaxf(fabsf(y[4 * j + 2]), fabsf(y[4 * j + 3]))));
                    const float s = e4_scale(most);
                    e4_put(out, at, p.width, e4_four(y + 4 * j, e4_over(s)));
                    if (lane == 0 && at < p.width) scale[at / E4_GROUP] = s;
                }
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
    int wide;                        // sixteens of out lie on 16-byte boundaries
};

constexpr int E4_THREADS = 256, E4_PER_ROW = E4_GROUP / 16;         // lanes of a scale in a row
// A scale for 128 columns of a row.  EIGHTS: eight lanes of sixteen columns, which lie one behind another over the rows.  Else: a warp for two of them
template <bool EIGHTS, typename E>
__global__ void __launch_bounds__(E4_THREADS) e4_rows_kernel(const __grid_constant__ E4Params p) {
    pdl_wait();
    const unsigned per_row = EIGHTS ? (unsigned)p.groups * E4_PER_ROW : ((unsigned)p.groups + 1) / 2;
    const unsigned long long thread = (unsigned long long)blockIdx.x * E4_THREADS + threadIdx.x, at = EIGHTS ? thread : thread >> 5;
    const unsigned row = at >> 32 ? (unsigned)(at / per_row) : (unsigned)at / per_row, unit = (unsigned)(at - (unsigned long long)row * per_row);
    const E* const x = reinterpret_cast<const E*>(p.x) + (long long)row * p.x_stride;
    uint8_t* const out = p.out + (long long)row * p.out_stride;
    float* const scale = p.scale + (long long)row * p.groups;
    if (EIGHTS) {
        const int col = (int)unit * 16, n = row < (unsigned)p.rows ? p.width - col : 0;
        E4Raw<E> a[2];
        float v[2][8], most = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (n > 8 * j) a[j] = e4_load<true, E>(x, col + 8 * j, p.width);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
            if (n > 8 * j) e4_values<E>(a[j], v[j]);
            most = fmaxf(most, e4_most(v[j]));
        }
#pragma unroll
        for (int o = E4_PER_ROW / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float s = e4_scale(most);
        const E4Over over = e4_over(s);
        if (n <= 0) return;
        const uint2 q[2] = {e4_pack(v[0], over), e4_pack(v[1], over)};
        if (p.wide && n >= 16) {
            *reinterpret_cast<uint4*>(out + col) = make_uint4(q[0].x, q[0].y, q[1].x, q[1].y);
        } else {
            *reinterpret_cast<uint2*>(out + col) = q[0];
            if (n > 8) *reinterpret_cast<uint2*>(out + col + 8) = q[1];
        }
        if (threadIdx.x % E4_PER_ROW == 0) scale[col / E4_GROUP] = s;
    } else {
        if (row >= (unsigned)p.rows) return;     // (a warp as one)
        const int lane = threadIdx.x & 31, col = (int)unit * 2 * E4_GROUP + lane;
        float v[8];
        e4_values<E>(e4_load<false, E>(x, col, p.width), v);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int c = col + j * E4_GROUP;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = c + 32 * i < p.width ? v[4 * j + i] : 0.f;
            const float s = e4_scale(warp_max(fmaxf(fmaxf(fabsf(v[4 * j]), fabsf(v[4 * j + 1])), fmaxf(fabsf(v[4 * j + 2]), fabsf(v[4 * j + 3])))));
            e4_put(out, c, p.width, e4_four(v + 4 * j, e4_over(s)));
            if (lane == 0 && c < p.width) scale[c / E4_GROUP] = s;
        }
    }
}

// the same bits, of which the compiler knows nothing: what was made of them is made again instead of kept
template <typename E>
__device__ __forceinline__ void e4_anew(E4Raw<E>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; ++i) asm volatile("" : "+r"(r.u[i].x), "+r"(r.u[i].y), "+r"(r.u[i].z), "+r"(r.u[i].w));
}

// A scale for a block of 128 x 128: a CTA, in its registers.  EIGHTS: sixteen lanes along a row, sixteen rows at a time.  Else: a warp along a row.  Rows and columns that are not there
// read the last ones', which changes no maximum
template <bool EIGHTS, typename E>
__global__ void __launch_bounds__(E4_THREADS, EIGHTS && sizeof(E) == 2 ? 4 : 2) e4_blocks_kernel(const __grid_constant__ E4Params p) {
    __shared__ float red[E4_THREADS / 32];
    pdl_wait();
    const int g = blockIdx.x % p.groups, b = blockIdx.x / p.groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rows = min(E4_GROUP, p.rows - b * E4_GROUP), last = min(E4_GROUP, p.width - g * E4_GROUP) - (EIGHTS ? 8 : 1);      // of the block; the first column of its last eight
    const E* const x = reinterpret_cast<const E*>(p.x) + (long long)b * E4_GROUP * p.x_stride + (long long)g * E4_GROUP;
    uint8_t* const out = p.out + (long long)b * E4_GROUP * p.out_stride + (long long)g * E4_GROUP;
    auto scale_of = [&](float most) {
        most = warp_max(most);
        if (lane == 0) red[warp] = most;
        __syncthreads();
        most = 0.f;
#pragma unroll
        for (int i = 0; i < E4_THREADS / 32; ++i) most = fmaxf(most, red[i]);
        const float s = e4_scale(most);
        if (threadIdx.x == 0) p.scale[(long long)b * p.groups + g] = s;
        return s;
    };
    float most = 0.f;
    if (EIGHTS) {
        constexpr int ROWS = E4_THREADS / 16, N = E4_GROUP / ROWS;
        const int first = threadIdx.x >> 4, c = (threadIdx.x & 15) * 8;
        E4Raw<E> a[N];
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = e4_load<true, E>(x + min(first + i * ROWS, rows - 1) * p.x_stride, min(c, last), 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[8];
            e4_values<E>(a[i], v);
            most = fmaxf(most, e4_most(v));
            e4_anew(a[i]);
        }
        const E4Over over = e4_over(scale_of(most));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[8];
            e4_values<E>(a[i], v);
            if (first + i * ROWS < rows && c <= last) *reinterpret_cast<uint2*>(out + (first + i * ROWS) * p.out_stride + c) = e4_pack(v, over);
        }
    } else {
        constexpr int ROWS = E4_THREADS / 32, N = E4_GROUP / ROWS;
        E a[N][4];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[i][j] = x[min(warp + i * ROWS, rows - 1) * p.x_stride + min(lane + 32 * j, last)];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(widened<E>(a[i][j])));
        const E4Over over = e4_over(scale_of(most));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float v[4] = {widened<E>(a[i][0]), widened<E>(a[i][1]), widened<E>(a[i][2]), widened<E>(a[i][3])};
            if (warp + i * ROWS < rows) e4_put(out + (warp + i * ROWS) * p.out_stride, lane, last + 1, e4_four(v, over));
        }
    }
}

}  // namespace b200

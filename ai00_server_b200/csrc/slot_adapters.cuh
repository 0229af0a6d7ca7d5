// Adapters of slots in the steps of the RWKV models: what surrounds adapters.cuh's products.  A step with such slots runs its projections as ever; behind
// each launch the adapters are added to the outputs in place.  Projections that end in an activation (gate, channel-mix key and receptance) leave
// their sums in a scratch row instead, and the activation follows: in the adapters' kernel itself in steps of up to ADP_INLINE tokens, here in longer ones.
// Bound: four dependent launches a layer, 6 to 8 us each (8 layers of 7B widths, rank 16: a step of 16 slots 1061 us without adapters, 1549 with sixteen of them; with
// the activations in launches of their own 1592).
#pragma once
#include "operators.cuh"

namespace b200 {

constexpr int ADAPTER_POOL = 64;               // adapters a model holds at once

// adapter (place in the pool, -1: none) of every token and of every logits row of the step; rows behind the last: -2
struct AdapterIndexParams {
    MetaView meta;
    const int* slot_adapter;
    int *tok, *row;
    int rows, out_rows;
};
__global__ void adapter_index_kernel(const __grid_constant__ AdapterIndexParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    const int T = p.meta.T(), R = p.meta.R();
    if (i < p.rows) p.tok[i] = i < T ? p.slot_adapter[p.meta.tok_slot()[i]] : -2;
    if (i < p.out_rows) p.row[i] = i < R ? p.slot_adapter[p.meta.tok_slot()[p.meta.out_tok()[i]]] : -2;
}

// dst[r][i] = src[i][r], zero for r in [ranks, padded): `<name>.lora.0` as the converter writes it -> rows of k
__global__ void adapter_pack_a_kernel(const __half* __restrict__ src, __half* __restrict__ dst, int in, int ranks, int padded) {
    const size_t n = (size_t)padded * in;
    for (size_t e = (size_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (size_t)gridDim.x * blockDim.x) {
        const int r = (int)(e / in), i = (int)(e - (size_t)r * in);
        dst[e] = r < ranks ? src[(size_t)i * ranks + r] : __half(0.f);
    }
}
// `<name>.lora.1` [out, ranks] -> [out, padded]
__global__ void adapter_pack_b_kernel(const __half* __restrict__ src, __half* __restrict__ dst, int out, int ranks, int padded) {
    const size_t n = (size_t)out * padded;
    for (size_t e = (size_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (size_t)gridDim.x * blockDim.x) {
        const int o = (int)(e / padded), r = (int)(e - (size_t)o * padded);
        dst[e] = r < ranks ? src[(size_t)o * ranks + r] : __half(0.f);
    }
}
__global__ void adapter_slot_kernel(int* slot_adapter, int slot, int place) { slot_adapter[slot] = place; }

// sums of a projection -> its activation where the next launch reads it (f32 rows, or the A16 operand, split into halves at precision 1)
struct AdapterFinishParams {
    const float* src;            // [rows][N]
    const int* nrows;
    void* out;
    int N, act, a16, split;
    int ldo;                     // f32: floats between rows; A16: the operand's height
};
__global__ void __launch_bounds__(256) adapter_finish_kernel(const __grid_constant__ AdapterFinishParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int per = p.N / 8, total = per * *p.nrows;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
        const int m = i / per, n = (i - m * per) * 8;
        const float* s = p.src + (size_t)m * p.N + n;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
            const float4 x = *reinterpret_cast<const float4*>(s + k);
            v[k] = apply_act(x.x, p.act); v[k + 1] = apply_act(x.y, p.act); v[k + 2] = apply_act(x.z, p.act); v[k + 3] = apply_act(x.w, p.act);
        }
        if (!p.a16) {
            float* const o = reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n;
            *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
            continue;
        }
        __half* const o = reinterpret_cast<__half*>(p.out);
        uint4 hi, lo;
        if (p.split) {
            split_pack_h2(v[0], v[1], hi.x, lo.x); split_pack_h2(v[2], v[3], hi.y, lo.y);
            split_pack_h2(v[4], v[5], hi.z, lo.z); split_pack_h2(v[6], v[7], hi.w, lo.w);
            *reinterpret_cast<uint4*>(o + a16_index(m + 16, n, p.ldo)) = lo;
        } else {
            hi = make_uint4(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]), pack_h2(v[4], v[5]), pack_h2(v[6], v[7]));
        }
        *reinterpret_cast<uint4*>(o + a16_index(m, n, p.ldo)) = hi;
    }
}

}  // namespace b200

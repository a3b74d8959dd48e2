// Rows of keys or values to and from blocks of 64 tokens of one head
// (attend.h's layouts), a workgroup of 256 threads a block.
#pragma once

#include "attend.h"
#include "device.h"

namespace trit {

constexpr int BLOCK_THREADS = 256;

// The larger of a value and the one 32 (16) lanes away: a swap of two copies
// leaves a lane its own value in one and the other's in the other.
__device__ __forceinline__ float other_half_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_row_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// The largest over a wave.
__device__ __forceinline__ float wave_max(float v) {
    v = __builtin_fmaxf(v, dpp<DPP_XOR1>(v));
    v = __builtin_fmaxf(v, dpp<DPP_XOR2>(v));
    v = __builtin_fmaxf(v, dpp<DPP_HALF_MIRROR>(v));
    v = __builtin_fmaxf(v, dpp<DPP_MIRROR>(v));
    return other_half_max(other_row_max(v));
}

// A thread's share of a block: groups of 4 values that lie side by side in
// every layout. Keys: 4 dims of a token; values: 4 tokens of a dim.
template <int HDP>
struct BlockShare {
    static constexpr int GROUPS = BLOCK_TOKENS * HDP / 4 / BLOCK_THREADS;
    static constexpr int VALUES = 4 * GROUPS;
};
template <int HDP, bool V>
__device__ __forceinline__ void share_at(int group, int& token, int& e) {
    const int u = threadIdx.x + group * BLOCK_THREADS;
    token = V ? u / HDP * 4 : u / (HDP / 4);
    e = V ? u % HDP : u % (HDP / 4) * 4;
}
template <int HDP, bool V>
__device__ __forceinline__ int code_at(int token, int e) {
    return V ? v8_at<HDP>(token, e) : k8_at<HDP>(token, e);
}
template <int HDP, bool V>
__device__ __forceinline__ int half_at(int token, int e) {
    return V ? v16_at<HDP>(token, e) : k16_at<HDP>(token, e);
}

// f16 as a block holds it: what f16 does not hold as a finite value is NaN.
__device__ __forceinline__ _Float16 held(float v) {
    const _Float16 h = (_Float16)v;
    return __builtin_fabsf((float)h) < INFINITY ? h : (_Float16)NAN;
}

// The thread's share of the block whose token 0 is row `first` of `rows` (a
// head's columns; first may be negative), as f32; rows outside [0, count) and
// dims from hd on read some row and dim inside and are the caller's to
// replace. Every load is issued before any is used: under a condition each
// they would wait for each other.
template <int HDP, bool V>
__device__ __forceinline__ void load_share(const float* rows, long long stride, int first, int count, int hd,
                                           bool aligned, float (&v)[BlockShare<HDP>::VALUES]) {
    constexpr int G = BlockShare<HDP>::GROUPS;
    if (!V && aligned) {  // hd a multiple of 4
#pragma unroll
        for (int i = 0; i < G; ++i) {
            int tok, e;
            share_at<HDP, V>(i, tok, e);
            const int r = min(max(first + tok, 0), count - 1);
            const float4 x = gload_f4(rows + (size_t)r * stride + (e < hd ? e : 0));
            v[4 * i] = x.x;
            v[4 * i + 1] = x.y;
            v[4 * i + 2] = x.z;
            v[4 * i + 3] = x.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
        int tok, e;
        share_at<HDP, V>(i, tok, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = min(max(first + tok + (V ? j : 0), 0), count - 1), d = V ? e : e + j;
            v[4 * i + j] = *gmem(rows + (size_t)r * stride + (d < hd ? d : 0));
        }
    }
}

}  // namespace trit

// Shared by the sequence operators (scan_ops.hip, blocknorm_ops.hip, logprob_ops.hip): activations in fp32 / bf16 / fp16, four consecutive
// channels a lane, every sum, statistic and state in fp32; one rounding to the activations' type, at the store.
#pragma once
#include "../../include/lego_hip.h"
#include "common.hpp"

namespace lego {

template <typename T> using vec4 = T __attribute__((ext_vector_type(4)));

// channels c .. c + 3 of a row of `width`: one 16- / 8-byte load where the caller has shown the alignment (then width % 4 == 0), else one
// load a channel; channels outside the row read as 0
template <typename T, bool ALIGNED>
__device__ __forceinline__ f32x4 load4(const T* __restrict__ row, int c, int width) {
    if constexpr (ALIGNED) {
        if (c >= width) return f32x4{0.f, 0.f, 0.f, 0.f};
        return __builtin_convertvector(*reinterpret_cast<const vec4<T>*>(row + c), f32x4);
    } else {
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = c + k < width ? (float)row[c + k] : 0.f;
        return v;
    }
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void store4(T* __restrict__ row, int c, int width, f32x4 v) {
    if constexpr (ALIGNED) {
        if (c < width) *reinterpret_cast<vec4<T>*>(row + c) = __builtin_convertvector(v, vec4<T>);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < width) row[c + k] = (T)v[k];
    }
}

// 1 / (1 + e^-x) on the hardware exponential and reciprocal (each within 1 ulp); e^-x overflows to inf for x < -88 and gives 0
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * x));
}

inline bool aligned4(const void* p, int dtype) { return ((uintptr_t)p & (dtype == LEGO_F32 ? 15u : 7u)) == 0; }

}  // namespace lego

// one instantiation of BODY for the activations' type, named T there
#define LEGO_BY_TYPE(dtype, BODY)                                                                                                                  \
    do {                                                                                                                                           \
        if ((dtype) == LEGO_F32) { using T = float; BODY; }                                                                                        \
        else if ((dtype) == LEGO_BF16) { using T = __bf16; BODY; }                                                                                 \
        else { using T = _Float16; BODY; }                                                                                                         \
    } while (0)

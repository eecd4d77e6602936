// Shared by the sequence operators (scan_ops.hip, blocknorm_ops.hip, logprob_ops.hip): activations in fp32 / bf16 / fp16, a few
// consecutive channels a lane, every sum, statistic and state in fp32; one rounding to the activations' type, at the store.
#pragma once
#include "../../include/lego_hip.h"
#include "common.hpp"

namespace lego {

template <typename T, int N> using vec = T __attribute__((ext_vector_type(N)));

// Channels c .. c + N - 1 of a row of `width`, `at` bytes behind `base`; channels outside the row read as 0 and are not written.  `base` is the
// same for the wave (scalar registers) and `at` a 32-bit lane offset: a 64-bit address a lane would cost two registers for every access.
// Rows start anywhere (strides and odd widths leave 16-bit elements on 2-byte boundaries): the copies compile to ONE access at the element's
// alignment, which the hardware takes; only a row's last lane, where `width` is no multiple of N (FULL = false), goes element by element.
template <typename T, int N, bool FULL>
__device__ __forceinline__ vec<T, N> load_raw(const T* __restrict__ base, uint32_t at, int c, int width) {
    const T* p = reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + at);
    vec<T, N> v;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (T)0;
    if (FULL ? c < width : c + N <= width) __builtin_memcpy(&v, p, sizeof(v));
    else if (!FULL) {
#pragma unroll
        for (int k = 0; k < N - 1; ++k)
            if (c + k < width) v[k] = p[k];
    }
    return v;
}

template <typename T, int N, bool FULL>
__device__ __forceinline__ vec<float, N> load_at(const T* __restrict__ base, uint32_t at, int c, int width) {
    return __builtin_convertvector((load_raw<T, N, FULL>(base, at, c, width)), vec<float, N>);
}

template <typename T, int N, bool FULL>
__device__ __forceinline__ void store_at(T* __restrict__ base, uint32_t at, int c, int width, vec<float, N> v) {
    T* p = reinterpret_cast<T*>(reinterpret_cast<char*>(base) + at);
    const vec<T, N> o = __builtin_convertvector(v, vec<T, N>);
    if (FULL ? c < width : c + N <= width) __builtin_memcpy(p, &o, sizeof(o));
    else if (!FULL) {
#pragma unroll
        for (int k = 0; k < N - 1; ++k)
            if (c + k < width) p[k] = o[k];
    }
}

// the same of a row that begins at `row`
template <typename T, int N, bool FULL>
__device__ __forceinline__ vec<float, N> load(const T* __restrict__ row, int c, int width) {
    return load_at<T, N, FULL>(row, (uint32_t)(c * (int)sizeof(T)), c, width);
}
template <typename T, int N, bool FULL>
__device__ __forceinline__ void store(T* __restrict__ row, int c, int width, vec<float, N> v) {
    store_at<T, N, FULL>(row, (uint32_t)(c * (int)sizeof(T)), c, width, v);
}

// 1 / (1 + e^-x) on the hardware exponential and reciprocal (each within 1 ulp); e^-x overflows to inf for x < -88 and gives 0
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * x));
}

// the sum over the wave's 64 lanes, in every lane: shifts inside rows of 16 lanes, then across the rows, on the vector unit alone
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_shifted(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, true));
}
__device__ __forceinline__ float wave_total(float v) {
    v = add_shifted<0x111, 0xF>(v);                                    // row_shr:1, 2, 4, 8
    v = add_shifted<0x112, 0xF>(v);
    v = add_shifted<0x114, 0xF>(v);
    v = add_shifted<0x118, 0xF>(v);
    v = add_shifted<0x142, 0xA>(v);                                    // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
    v = add_shifted<0x143, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Channels c .. c + N - 1 of a row without a branch, for kernels that keep the next rows' loads in flight: channels behind the row read its end
// again (the caller leaves them out of its sums and does not store them).
template <typename T, int N, bool FULL>
__device__ __forceinline__ vec<T, N> load_some(const T* __restrict__ row, int c, int width) {
    vec<T, N> v;
    if constexpr (FULL) __builtin_memcpy(&v, row + min(c, width - N), sizeof(v));
    else
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = row[min(c + k, width - 1)];
    return v;
}

}  // namespace lego

// one instantiation of the statements behind `dtype` for the activations' type, named T there
#define LEGO_BY_TYPE(dtype, ...)                                                                                                                       \
    do {                                                                                                                                               \
        if ((dtype) == LEGO_F32) { using T = float; __VA_ARGS__; }                                                                                     \
        else if ((dtype) == LEGO_BF16) { using T = __bf16; __VA_ARGS__; }                                                                              \
        else { using T = _Float16; __VA_ARGS__; }                                                                                                      \
    } while (0)

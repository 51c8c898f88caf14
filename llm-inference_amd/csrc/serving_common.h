// serving_common.h -- what the kernels over packed sequences and the paged 4-bit cache share: element types, reductions
// inside a wave.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "cmhsa.h"
#include "cmhsa_packed.h"

namespace serving {

// A launch holds fewer than 2^32 threads: larger grids are refused here, so that no HIP error is left for the caller's next launch to find.
inline bool fits_a_launch(int64_t workgroups, int threads) { return workgroups * threads <= 0xffffffffLL; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// N consecutive elements (N * sizeof(T) a multiple of 16 bytes, 16-B aligned) as floats, and back: one rounding to nearest even
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T *p, float (&x)[N]) {
    constexpr int kPer = 16 / sizeof(T);
    static_assert(N % kPer == 0, "whole 16-byte pieces");
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
        typedef T vec __attribute__((ext_vector_type(kPer)));
        const vec v = reinterpret_cast<const vec *>(p)[i];
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[i * kPer + j] = (float)v[j];
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_floats(T *p, const float (&x)[N]) {
    constexpr int kPer = 16 / sizeof(T);
    static_assert(N % kPer == 0, "whole 16-byte pieces");
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
        typedef T vec __attribute__((ext_vector_type(kPer)));
        vec v;
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = (T)x[i * kPer + j];
        reinterpret_cast<vec *>(p)[i] = v;
    }
}

template <int kCtrl>
__device__ __forceinline__ float dpp_move(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kCtrl, 0xf, 0xf, false));
}
// over the four lanes of a quad, the result in each of them
__device__ __forceinline__ float quad_sum(float x) {
    x += dpp_move<0xB1>(x);            // quad_perm [1,0,3,2]
    return x + dpp_move<0x4E>(x);      // quad_perm [2,3,0,1]
}

// inclusive prefix sum over the 64 lanes (lane 63: the sum), in data-parallel moves
template <int kCtrl, int kRowMask>
__device__ __forceinline__ int add_moved(int x) { return x + __builtin_amdgcn_update_dpp(0, x, kCtrl, kRowMask, 0xf, false); }
__device__ __forceinline__ int prefix_sum(int x) {
    x = add_moved<0x111, 0xf>(x);      // row_shr 1, 2, 4, 8: within 16 lanes
    x = add_moved<0x112, 0xf>(x);
    x = add_moved<0x114, 0xf>(x);
    x = add_moved<0x118, 0xf>(x);
    x = add_moved<0x142, 0xa>(x);      // row_bcast 15: rows 1 and 3 get the sum of the row before
    return add_moved<0x143, 0xc>(x);   // row_bcast 31: rows 2 and 3 get the sum of the first two
}

__device__ __forceinline__ float wave_sum(float x) {
    x += dpp_move<0xB1>(x);            // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror: all 16 lanes of a row
    x += dpp_move<0x4E>(x);
    x += dpp_move<0x141>(x);
    x += dpp_move<0x140>(x);
    const int bits = __builtin_bit_cast(int, x);
    const int a = __builtin_amdgcn_readlane(bits, 0), b = __builtin_amdgcn_readlane(bits, 16), c = __builtin_amdgcn_readlane(bits, 32), d = __builtin_amdgcn_readlane(bits, 48);
    return (__builtin_bit_cast(float, a) + __builtin_bit_cast(float, b)) + (__builtin_bit_cast(float, c) + __builtin_bit_cast(float, d));
}
// the maximum over the 64 lanes of numbers that are not negative
__device__ __forceinline__ int wave_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, false));
    return max(max(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)), max(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(prefix_sum(x), 63); }

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return min(max(x, lo), hi); }

}  // namespace serving

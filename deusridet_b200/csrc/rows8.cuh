// rows8.cuh — quantising one row of the 8-bit pool, shared by the append kernels and the decode step.
#pragma once

#include "kv_common.cuh"
#include "sm100_primitives.cuh"

namespace drkv {

// Quantises the row of which each of its LANES lanes holds 8 elements; row: its index in the block's rows (K plane, then V
// plane, exponents in the same order).
template <int LANES>
__device__ __forceinline__ void quantise_row(const float (&x)[8], uint8_t* block, int64_t exponents, int row, int l, bool store) {
    // the maximum of |x|; NaN is passed over by the maximum, an infinity makes the row look again
    float top = fmax3(fmaxf(fabsf(x[0]), fabsf(x[1])), fabsf(x[2]), fabsf(x[3]));
    top = fmax3(fmax3(top, fabsf(x[4]), fabsf(x[5])), fabsf(x[6]), fabsf(x[7]));
    uint32_t amax = __float_as_uint(top == top ? top : 0.f);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (__any_sync(0xffffffffu, amax >= 0x7f800000u)) {
        amax = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t a = __float_as_uint(x[i]) & 0x7fffffffu;
            amax = max(amax, a < 0x7f800000u ? a : 0u);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    const int e = e4m3_row_exponent(amax);
    const float inv = exp2_int(-e);
    uint2 v;
    v.x = f32x4_to_e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    v.y = f32x4_to_e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    if (store) {
        *reinterpret_cast<uint2*>(block + (int64_t)row * (8 * LANES) + 8 * l) = v;
        if (l == 0) block[exponents + row] = (uint8_t)(e + 127);
    }
}

template <typename T>
__device__ __forceinline__ void unpack8(const Vec16& v, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = Elem<T>::unpack2(v.w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Rotates the row by the angles of append_rope_kernel, in fp32; c and s hold the cosines and sines of the lane's own 8 pairs
// (lanes past the rotated dims pass anything).  A shuffle within the row's lanes: rows are aligned groups of lanes.
__device__ __forceinline__ void rotate_row(float (&x)[8], const float* c, const float* s, int half, int l, bool live) {
    const int hl = half / 8;                                         // lanes of one rotated half (rotary_dim % 16 == 0)
    const bool first = l < hl, second = l >= hl && l < 2 * hl;
    const int lane = threadIdx.x & 31, other = lane + (first ? hl : second ? -hl : 0);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float o = __shfl_sync(0xffffffffu, x[i], other);
        if (live && (first || second)) {
            float y0, y1;
            rope_pair(first ? x[i] : o, first ? o : x[i], c[i], s[i], y0, y1);
            x[i] = first ? y0 : y1;
        }
    }
}

}  // namespace drkv

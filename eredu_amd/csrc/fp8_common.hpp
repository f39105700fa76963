// Linears in 8-bit floating point with block scales: what their kernels share.
//
// A group of values v (128 of a row, or 128 x 128 of a weight) becomes the
// scale s = a / 448, a = max|v| (at least 448 * 2^-126), and the codes
// e4m3(448 v / a).  Values of 16 bits and a have so few bits that the quotient
// is often a tie between two codes, so it has to be rounded from a quotient
// that is exact where it can be: with a = A 2^e, 1 <= A < 2, t = v * (448 2^-e) is exact
// for 16-bit v, q = t * rcp(A) is off by an f32 step or two, and
// q + (t - q A) rcp(A) is then t / A to f32's own rounding (so exact where
// the quotient has at most 24 bits).  Two FMAs a value, which hide behind the loads.
#pragma once

#include "../../include/eredu_fp8.h"
#include "eq_common.hpp"

namespace eq {

constexpr int kFp8Block = 128;
constexpr float kFp8Most = 448.f;
constexpr int64_t kFp8MaxCols = int64_t(1) << 22;
constexpr int64_t kFp8MaxGroups = int64_t(1) << 26;  // of 128 values of a row, of a call

// |v| of finite, infinite and NaN values in order, as bits.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest of the 16 lanes of a DPP row, in every lane: pairs, fours, then
// mirrored halves and rows (VALU alone, no LDS).
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0xB1, 0xf, 0xf, true)));   // quad_perm 1 0 3 2
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x4E, 0xf, 0xf, true)));   // quad_perm 2 3 0 1
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x141, 0xf, 0xf, true)));  // row_half_mirror
    return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x140, 0xf, 0xf, true)));  // row_mirror
}

struct Fp8Group {
    float up, part, inverse, scale;  // 448 2^-e, A, 1 / A, s
    bool finite;

    // most: abs_bits of the group's largest
    __device__ __forceinline__ explicit Fp8Group(uint32_t most) {
        finite = most < 0x7f800000u;
        const float a = finite ? fmaxf(__uint_as_float(most), kFp8Most * 0x1p-126f) : kFp8Most;
        const uint32_t bits = __float_as_uint(a);
        scale = finite ? a / kFp8Most : __uint_as_float(0x7fc00000u);
        up = ldexpf(kFp8Most, 127 - int(bits >> 23));
        part = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
        const float r = __builtin_amdgcn_rcpf(part);
        inverse = fmaf(fmaf(-part, r, 1.f), r, r);
    }
    __device__ __forceinline__ float code(float v) const {
        const float t = v * up, q = t * inverse;
        return finite ? fmaf(fmaf(-q, part, t), inverse, q) : 0.f;
    }
    // the codes of four values, the first in the low byte
    __device__ __forceinline__ uint32_t codes4(const float* v) const {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(code(v[0]), code(v[1]), 0, false);
        return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(code(v[2]), code(v[3]), lo, true));
    }
};

// Eight consecutive values, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const typename T::storage* p, float* v) {
    if constexpr (std::is_same<T, F32T>::value) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, BF16T>::value) {
                v[2 * i] = bf16_bits_to_f32(w[i] & 0xffffu);
                v[2 * i + 1] = bf16_bits_to_f32(w[i] >> 16);
            } else {
                v[2 * i] = f16_bits_to_f32(w[i] & 0xffffu);
                v[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(typename T::storage* p, const float* v) {
    if constexpr (std::is_same<T, F32T>::value) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, BF16T>::value) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            else w[i] = uint32_t(to_storage<T>(v[2 * i])) | uint32_t(to_storage<T>(v[2 * i + 1])) << 16;
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename T>
__device__ __forceinline__ float rounded(float v) {
    const typename T::storage s = to_storage<T>(v);
    return load_param<T>(&s, 0);
}

inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

// Host side: argument checks that several entry points share (false: the error is set).
bool fp8_cols_ok(const char* who, const char* name, int64_t cols);
bool fp8_rows_ok(const char* who, const char* name, const void* p, int64_t stride, int64_t cols, int64_t bytes);
bool fp8_scales_ok(const char* who, int64_t stride, int64_t rows, int64_t cols);

// eq_fp8_quantize after its checks.
void launch_fp8_quantize(void* codes, float* scales, int64_t scale_stride, const void* x, int64_t x_stride,
                         int64_t rows, int64_t cols, int dtype, hipStream_t st);

}  // namespace eq

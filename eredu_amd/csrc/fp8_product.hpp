// Products of rows in e4m3 codes: the matrix instructions and the arguments that
// their kernels share (fp8_matmul.hip: tiles; fp8_few.hip: few rows).
#pragma once

#include "fp8_common.hpp"

namespace eq {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Fp8Args {
    void* y;
    const uint8_t* x;
    const float* xs;
    int64_t x_stride, xs_stride;
    const uint8_t* w;
    const float* ws;
    int M, N, K, KB;  // KB: blocks of K
    int mtiles, ntiles, band;  // tiles
    int slots, parts;          // workgroups that run at once, and the most parts of K that a tile of the last pass makes
    float* part;               // the parts' sums
    // Grouped: tiles[i] = {expert, first, rows} of row tile i, the rows being order[first ..], {route, row of x};
    // tiles[mtiles].x: how many there are.  Expert -1: rows of zeros.
    const int4* tiles;
    const int2* order;
    const int32_t* rows;
    int64_t x_rows;
};

__device__ __forceinline__ f32x4 mfma128(u32x4 a0, u32x4 a1, u32x4 b0, u32x4 b1) {
    const i32x8 a = __builtin_bit_cast(i32x8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    const i32x8 b = __builtin_bit_cast(i32x8, __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
    // formats 0, 0: e4m3; scales 0: the form without scales
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{}, 0, 0, 0, 0, 0, 0);
}

// Eight codes as bf16.
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t lo, uint32_t hi) {
    const u32x4 v = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
    return __builtin_bit_cast(bf16x8, v);
}

// A lane's 32 codes of a row and block, as the matrix instruction takes them.
template <bool EXACT>
struct Operand;
template <>
struct Operand<false> {
    u32x4 c[2];
    __device__ __forceinline__ void take(u32x4 a, u32x4 b) { c[0] = a, c[1] = b; }
};
template <>
struct Operand<true> {
    bf16x8 c[4];
    __device__ __forceinline__ void take(u32x4 a, u32x4 b) {
        c[0] = codes_bf16(a[0], a[1]), c[1] = codes_bf16(a[2], a[3]);
        c[2] = codes_bf16(b[0], b[1]), c[3] = codes_bf16(b[2], b[3]);
    }
};
__device__ __forceinline__ f32x4 block_sums(const Operand<false>& a, const Operand<false>& b) {
    return mfma128(a.c[0], a.c[1], b.c[0], b.c[1]);
}
__device__ __forceinline__ f32x4 block_sums(const Operand<true>& a, const Operand<true>& b) {
    f32x4 d{};
#pragma unroll
    for (int i = 0; i < 4; i++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.c[i], b.c[i], d, 0, 0, 0);
    return d;
}

// VALS consecutive results of a row, n of them inside it.  Pieces of 16 bytes, at whatever place the row's length puts
// them (global stores need no alignment; 3103 x 2662 f32 of 96 columns took 52 us value by value, 15.5 in pieces side by side).
template <typename YT, int VALS>
__device__ __forceinline__ void store_run(typename YT::storage* p, const float* v, int n) {
    using S = typename YT::storage;
    constexpr int VEC = VALS < 16 / int(sizeof(S)) ? VALS : 16 / int(sizeof(S)), WORDS = VEC * int(sizeof(S)) / 4;
#pragma unroll
    for (int i = 0; i < VALS; i += VEC) {
        if (i + VEC <= n) {
            uint32_t w[WORDS];
#pragma unroll
            for (int e = 0; e < WORDS; e++) {
                if constexpr (std::is_same<YT, F32T>::value) w[e] = __float_as_uint(v[i + e]);
                else if constexpr (std::is_same<YT, BF16T>::value) w[e] = pack_bf16x2(v[i + 2 * e], v[i + 2 * e + 1]);
                else w[e] = uint32_t(to_storage<YT>(v[i + 2 * e])) | uint32_t(to_storage<YT>(v[i + 2 * e + 1])) << 16;
            }
            __builtin_memcpy(p + i, w, sizeof(w));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (i + e < n) store_out<YT>(p, i + e, v[i + e]);
        }
    }
}

// Few rows (fp8_few.hip): x of x_dtype, e4m3 codes or values that the kernel quantizes; with `ids`, a
// row and an expert for each of the routes (a.M of them).
struct Fp8Few {
    const void* x;
    int x_dtype;
    const int32_t* ids;
    int experts;
};
// Whether launch_fp8_few takes m rows (of routes: 1) of x_dtype without codes of them being made first.
bool fp8_few_takes(int64_t m, int64_t k, int x_dtype);
void launch_fp8_few(const Fp8Args& a, const Fp8Few& f, int y_dtype, hipStream_t st);

}  // namespace eq

// Values into e4m3 codes with block scales: rows as they are, behind the
// root-mean-square norm and behind silu(gate) * up, and weights.
//
//   s = max|v| / 448,  c = e4m3(448 v / max|v|)        (fp8_common.hpp)
//
// All of it is bound by memory: each value is read once, held in registers as
// f32 while its group's largest is found, and written once as a code.
#include "fp8_common.hpp"

namespace eq {
namespace {

// Sum over the block (blockDim.x a multiple of 64, at most 1024), the waves' sums in order.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
    for (int i = 0; i < int(blockDim.x >> 6); i++) t += red[i];
    return t;
}

constexpr float kLog2E = 1.44269504f, kLog2ELow = 1.92596300e-8f, kLn2 = 0.693147181f;  // log2 e in two parts

// 1 / (1 + e^-g): 2^(-g log2 e) with the rounding of the product put back, so that it is off by steps of f32 for gates from
// kFarGate on (by expf and a division the kernel took 76 us for 4096 x 14336 values, bound by the vector units).
__device__ __forceinline__ float sigmoid(float g) {
    const float t = -g * kLog2E, low = fmaf(-g, kLog2E, -t) - g * kLog2ELow, e = __builtin_amdgcn_exp2f(t);
    // (2^t = 0 and infinity, and an infinite g, have nothing to put back)
    const float exact = fabsf(t) < 126.f ? fmaf(e, low * kLn2, e) : e;
    return __builtin_amdgcn_rcpf(1.f + exact);
}

// silu(g) u of gates below kFarGate, where 1 / (1 + e^-g) nears the smallest normal f32 (behind it v_rcp_f32 gives 0) and is
// e^g but for 2^-124 of it.  Its power of two comes last, so that a large u finds all of its bits; it is off by
// the 2^x of one step, its correction and two products.
constexpr float kFarGate = -86.5f;
__device__ __forceinline__ float silu_mul_far(float g, float u) {
    const float c = g > -INFINITY ? fmaxf(g, -300.f) : g;  // (e^-300 of any u is below every code)
    const float t = c * kLog2E, low = fmaf(c, kLog2E, -t) + c * kLog2ELow, n = fmaxf(rintf(t), -500.f);
    const float e = __builtin_amdgcn_exp2f(t - n);
    return ldexpf(c * fmaf(e, low * kLn2, e) * 0x1p-9f * u, int(n) + 9);  // (300 sqrt 2 2^-9 < 1: no u overflows)
}

// Codes of 8 values of a lane whose group lies in its 16 lanes; `first` lanes write the scale.
__device__ __forceinline__ void put_group(const float* v, bool live, uint2* codes, float* scale, bool first) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) most = max(most, abs_bits(v[i]));
    const Fp8Group g(max16(live ? most : 0u));
    if (live) *codes = make_uint2(g.codes4(v), g.codes4(v + 4));
    if (first) *scale = g.scale;
}

// x, or silu(gate) * up: 16 lanes a group, eight values each; group i of the launch is row i / blocks.  Bound by
// memory: silu of 4096 x 14336 59.5 us (294 MB at 4.9 TB/s, a large copy 5.1), quantizing 4096 x 4096 12.5 us.
template <typename T, bool SILU>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                           int64_t scale_stride,
                                                           const typename T::storage* __restrict__ x, int64_t x_stride,
                                                           const typename T::storage* __restrict__ up,
                                                           int64_t up_stride, int rows, int cols, int blocks) {
    const uint32_t group = blockIdx.x * 16u + (threadIdx.x >> 4);
    const uint32_t row = group / uint32_t(blocks), block = group - row * uint32_t(blocks);
    const int lane = threadIdx.x & 15, at = int(block) * kFp8Block + lane * 8;
    const bool live = row < uint32_t(rows) && at < cols;
    float v[8] = {};
    if (live) {
        load8<T>(x + row * x_stride + at, v);
        if constexpr (SILU) {
            float u[8], g[8], least = 0.f;
            load8<T>(up + row * up_stride + at, u);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                g[i] = v[i], least = fminf(least, g[i]);
                v[i] = g[i] * sigmoid(g[i]) * u[i];
            }
            if (__builtin_expect(least < kFarGate, 0)) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = g[i] < kFarGate ? silu_mul_far(g[i], u[i]) : v[i];
            }
        }
    }
    put_group(v, live, reinterpret_cast<uint2*>(codes + int64_t(row) * cols + at), scales + block * scale_stride + row,
              lane == 0 && row < uint32_t(rows));
}

// Bound by memory (8192 x 4096 with a residual 46.3 us, 235 MB at 5.1 TB/s), a single row of 4096 by a launch, 2.8 us.
// One row a workgroup.  VPT > 0: a thread keeps its (at most VPT) pieces of
// eight values in registers between the two passes; 0: any length, read again.
template <typename T, int VPT>
__global__ __launch_bounds__(1024) void fp8_rms_norm_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                            int64_t scale_stride, typename T::storage* __restrict__ x,
                                                            const typename T::storage* __restrict__ residual,
                                                            const typename T::storage* __restrict__ weight, int dim,
                                                            float eps) {
    __shared__ float red[16];
    const int64_t row = blockIdx.x;
    const int pieces = dim / 8, padded = (pieces + 15) & ~15, step = blockDim.x;
    x += row * dim;
    residual = residual ? residual + row * dim : nullptr;
    codes += row * dim;
    scales += row;
    // the row's piece p, the residual added and written back
    auto fetch = [&](int p, float* v) __attribute__((always_inline)) {
        load8<T>(x + 8 * p, v);
        if (residual) {
            float r[8];
            load8<T>(residual + 8 * p, r);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = rounded<T>(v[i] + r[i]);
            store8<T>(x + 8 * p, v);
        }
    };
    auto squares = [&](const float* v) __attribute__((always_inline)) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) s = fmaf(v[i], v[i], s);
        return s;
    };
    auto put = [&](int p, float* v, const float* w, float inv) __attribute__((always_inline)) {
        const bool live = p < pieces;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = live ? w[i] * (v[i] * inv) : 0.f;
        put_group(v, live, reinterpret_cast<uint2*>(codes + 8 * p), scales + (p >> 4) * scale_stride,
                  (threadIdx.x & 15) == 0);
    };
    float ss = 0.f;
    if constexpr (VPT > 0) {
        float v[VPT][8], w[VPT][8];
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            const int p = threadIdx.x + j * step;
            if (p < pieces) {
                fetch(p, v[j]);
                load8<T>(weight + 8 * p, w[j]);
                ss += squares(v[j]);
            }
        }
        const float inv = 1.0f / sqrtf(block_sum(ss, red) / float(dim) + eps);
#pragma unroll
        for (int j = 0; j < VPT; j++) {
            const int p = threadIdx.x + j * step;
            if (p < padded) put(p, v[j], w[j], inv);  // (whole groups: 16 lanes go together)
        }
    } else {
        for (int p = threadIdx.x; p < pieces; p += step) {
            float v[8];
            fetch(p, v);
            ss += squares(v);
        }
        const float inv = 1.0f / sqrtf(block_sum(ss, red) / float(dim) + eps);
        for (int p = threadIdx.x; p < padded; p += step) {
            float v[8] = {}, w[8] = {};
            if (p < pieces) {
                load8<T>(x + 8 * p, v);  // (this thread's own values)
                load8<T>(weight + 8 * p, w);
            }
            put(p, v, w, inv);
        }
    }
}

// One 128 x 128 block a workgroup of 1024: row r of the block by 8 lanes of 16 values.  Bound by memory: 14336 x 4096 32.9 us,
// 176 MB at 5.4 TB/s.
template <typename T>
__global__ __launch_bounds__(1024) void fp8_quantize_weight_kernel(uint8_t* __restrict__ codes,
                                                                   float* __restrict__ scales,
                                                                   const typename T::storage* __restrict__ w, int rows,
                                                                   int cols, int row_blocks, int col_blocks) {
    __shared__ uint32_t red[16];
    const uint32_t cb = blockIdx.x % uint32_t(col_blocks), rest = blockIdx.x / uint32_t(col_blocks);
    const uint32_t rb = rest % uint32_t(row_blocks), bank = rest / uint32_t(row_blocks);
    const int row = int(rb) * kFp8Block + (threadIdx.x >> 3), col = int(cb) * kFp8Block + (threadIdx.x & 7) * 16;
    const bool live = row < rows && col < cols;
    const int64_t at = (int64_t(bank) * rows + row) * cols + col;
    float v[16] = {};
    uint32_t most = 0;
    if (live) {
        load8<T>(w + at, v);
        load8<T>(w + at + 8, v + 8);
#pragma unroll
        for (int i = 0; i < 16; i++) most = max(most, abs_bits(v[i]));
    }
    most = max16(most);
    most = max(most, uint32_t(__shfl_xor(int(most), 16)));
    most = max(most, uint32_t(__shfl_xor(int(most), 32)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) most = max(most, red[i]);
    const Fp8Group g(most);
    if (live)
        *reinterpret_cast<uint4*>(codes + at) =
            make_uint4(g.codes4(v), g.codes4(v + 4), g.codes4(v + 8), g.codes4(v + 12));
    if (threadIdx.x == 0) scales[blockIdx.x] = g.scale;
}

template <bool SILU>
void quantize_rows(void* codes, float* scales, int64_t scale_stride, const void* x, int64_t x_stride, const void* up,
                   int64_t up_stride, int64_t rows, int64_t cols, int dtype, hipStream_t st) {
    const int64_t blocks = fp8_blocks(cols), groups = rows * blocks;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        using S = typename T::storage;
        fp8_quantize_kernel<T, SILU><<<dim3(unsigned((groups + 15) / 16)), dim3(256), 0, st>>>(
            static_cast<uint8_t*>(codes), scales, scale_stride, static_cast<const S*>(x), x_stride,
            static_cast<const S*>(up), up_stride, int(rows), int(cols), int(blocks));
    });
}

int64_t dtype_bytes(int dtype) { return dtype == EQ_DTYPE_F32 ? 4 : 2; }

bool float_dtype_ok(const char* who, int dtype) {
    if (valid_dtype(dtype)) return true;
    set_error(std::string(who) + ": dtype must be f32, f16 or bf16");
    return false;
}

// (a launch has fewer than 2^32 threads: 16 to 64 a group)
bool groups_ok(const char* who, int64_t rows, int64_t cols) {
    if (rows >= 0 && rows < kFp8MaxGroups && rows * fp8_blocks(cols) < kFp8MaxGroups) return true;
    set_error(std::string(who) + ": rows * ceil(cols / 128) must be in [0, 2^26)");
    return false;
}

}  // namespace

bool fp8_cols_ok(const char* who, const char* name, int64_t cols) {
    if (cols > 0 && cols % 16 == 0 && cols < kFp8MaxCols) return true;
    set_error(std::string(who) + ": " + name + " must be a positive multiple of 16 below 2^22, got " + std::to_string(cols));
    return false;
}

bool fp8_rows_ok(const char* who, const char* name, const void* p, int64_t stride, int64_t cols, int64_t bytes) {
    if (!p) {
        set_error(std::string(who) + ": null pointer argument (" + name + ")");
        return false;
    }
    if (!aligned(p, 16) || stride * bytes % 16 != 0) {
        set_error(std::string(who) + ": rows of " + name + " must be 16-byte aligned");
        return false;
    }
    if (stride < cols || stride >= 2 * kFp8MaxCols) {
        set_error(std::string(who) + ": the row stride of " + name + " must be at least the row's length and below 2^23");
        return false;
    }
    return true;
}

bool fp8_scales_ok(const char* who, int64_t stride, int64_t rows, int64_t cols) {
    if (stride >= rows && stride <= INT64_MAX / 4 / fp8_blocks(cols)) return true;
    set_error(std::string(who) + ": scale_stride must be at least the number of rows");
    return false;
}

void launch_fp8_quantize(void* codes, float* scales, int64_t scale_stride, const void* x, int64_t x_stride,
                         int64_t rows, int64_t cols, int dtype, hipStream_t st) {
    quantize_rows<false>(codes, scales, scale_stride, x, x_stride, nullptr, 0, rows, cols, dtype, st);
}

}  // namespace eq

using namespace eq;

extern "C" int eq_fp8_quantize(void* codes, float* scales, int64_t scale_stride, const void* x, int64_t x_stride,
                               int64_t rows, int64_t cols, int dtype, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_fp8_quantize";
    if (!float_dtype_ok(who, dtype) || !fp8_cols_ok(who, "cols", cols) || !groups_ok(who, rows, cols)) return 1;
    if (rows == 0) return 0;
    if (!scales) {
        set_error(std::string(who) + ": null pointer argument (scales)");
        return 1;
    }
    if (!fp8_rows_ok(who, "codes", codes, cols, cols, 1) || !fp8_rows_ok(who, "x", x, x_stride, cols, dtype_bytes(dtype)) ||
        !fp8_scales_ok(who, scale_stride, rows, cols))
        return 1;
    launch_fp8_quantize(codes, scales, scale_stride, x, x_stride, rows, cols, dtype, reinterpret_cast<hipStream_t>(stream));
    return check_launch(who);
}

extern "C" int eq_fp8_quantize_weight(void* codes, float* scales, const void* w, int64_t count, int64_t rows,
                                      int64_t cols, int dtype, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_fp8_quantize_weight";
    if (!float_dtype_ok(who, dtype) || !fp8_cols_ok(who, "cols", cols)) return 1;
    if (rows < 0 || rows > INT32_MAX || count < 0 || count > INT32_MAX ||
        (count && fp8_blocks(rows) * fp8_blocks(cols) >= (int64_t(1) << 22) / count)) {
        set_error(std::string(who) + ": count and rows must be in [0, 2^31), blocks of 128 x 128 fewer than 2^22");
        return 1;
    }
    if (rows == 0 || count == 0) return 0;
    if (!scales) {
        set_error(std::string(who) + ": null pointer argument (scales)");
        return 1;
    }
    if (!fp8_rows_ok(who, "codes", codes, cols, cols, 1) || !fp8_rows_ok(who, "w", w, cols, cols, dtype_bytes(dtype))) return 1;
    const int64_t rb = fp8_blocks(rows), cb = fp8_blocks(cols);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        fp8_quantize_weight_kernel<T><<<dim3(unsigned(count * rb * cb)), dim3(1024), 0, reinterpret_cast<hipStream_t>(stream)>>>(
            static_cast<uint8_t*>(codes), scales, static_cast<const typename T::storage*>(w), int(rows), int(cols), int(rb),
            int(cb));
    });
    return check_launch(who);
}

extern "C" int eq_fp8_rms_norm(void* codes, float* scales, int64_t scale_stride, void* hidden, const void* residual,
                               const void* weight, int64_t rows, int64_t dim, float eps, int dtype, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_fp8_rms_norm";
    if (!float_dtype_ok(who, dtype) || !fp8_cols_ok(who, "dim", dim) || !groups_ok(who, rows, dim)) return 1;
    if (!(eps >= 0.f)) {
        set_error(std::string(who) + ": eps must be >= 0");
        return 1;
    }
    if (rows == 0) return 0;
    if (!scales) {
        set_error(std::string(who) + ": null pointer argument (scales)");
        return 1;
    }
    const int64_t bytes = dtype_bytes(dtype);
    if (!fp8_rows_ok(who, "codes", codes, dim, dim, 1) || !fp8_rows_ok(who, "hidden", hidden, dim, dim, bytes) ||
        (residual && !fp8_rows_ok(who, "residual", residual, dim, dim, bytes)) ||
        !fp8_rows_ok(who, "weight", weight, dim, dim, bytes) || !fp8_scales_ok(who, scale_stride, rows, dim))
        return 1;
    const int pieces = int(dim / 8);
    const int block = pieces >= 1024 ? 1024 : (pieces + 63) / 64 * 64;
    const int vpt = (pieces + block - 1) / block;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        using S = typename T::storage;
        auto go = [&](auto kern) {
            kern<<<dim3(unsigned(rows)), dim3(unsigned(block)), 0, reinterpret_cast<hipStream_t>(stream)>>>(
                static_cast<uint8_t*>(codes), scales, scale_stride, static_cast<S*>(hidden), static_cast<const S*>(residual),
                static_cast<const S*>(weight), int(dim), eps);
        };
        if (vpt == 1) go(fp8_rms_norm_kernel<T, 1>);
        else if (vpt == 2) go(fp8_rms_norm_kernel<T, 2>);
        else go(fp8_rms_norm_kernel<T, 0>);
    });
    return check_launch(who);
}

extern "C" int eq_fp8_silu_mul(void* codes, float* scales, int64_t scale_stride, const void* gate, int64_t gate_stride,
                               const void* up, int64_t up_stride, int64_t rows, int64_t cols, int dtype,
                               eq_stream_t stream) {
    clear_error();
    const char* who = "eq_fp8_silu_mul";
    if (!float_dtype_ok(who, dtype) || !fp8_cols_ok(who, "cols", cols) || !groups_ok(who, rows, cols)) return 1;
    if (rows == 0) return 0;
    if (!scales) {
        set_error(std::string(who) + ": null pointer argument (scales)");
        return 1;
    }
    const int64_t bytes = dtype_bytes(dtype);
    if (!fp8_rows_ok(who, "codes", codes, cols, cols, 1) || !fp8_rows_ok(who, "gate", gate, gate_stride, cols, bytes) ||
        !fp8_rows_ok(who, "up", up, up_stride, cols, bytes) || !fp8_scales_ok(who, scale_stride, rows, cols))
        return 1;
    quantize_rows<true>(codes, scales, scale_stride, gate, gate_stride, up, up_stride, rows, cols, dtype,
                        reinterpret_cast<hipStream_t>(stream));
    return check_launch(who);
}

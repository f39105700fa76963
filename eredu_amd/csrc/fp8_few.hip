// Products of few rows (at most 16, or one for each route) with e4m3 weights:
// bound by reading the weights once.
//
// A workgroup of 8 waves has 16 weight rows; wave v takes the blocks v, v + 8,
// .. of K, a block being one matrix instruction (fp8_matmul.hip).  A lane reads
// two pieces of 16 bytes of its weight row straight into the operand's
// registers, four blocks ahead of their use; the waves' sums are added through LDS in wave order.
// Rows of values are quantized by the workgroup into LDS while its first weights are on their way.
#include "fp8_product.hpp"

namespace eq {
namespace {

constexpr int kFewWaves = 8, kFewAhead = 4;
constexpr int kFewLds = 48 * 1024;  // codes of the rows, where the kernel makes them

struct F8T {};  // x in codes

template <typename XT, typename YT>
__global__ __launch_bounds__(64 * kFewWaves) void fp8_few_kernel(const Fp8Args args, const Fp8Few few) {
    constexpr bool CODED = std::is_same<XT, F8T>::value, EXACT = std::is_same<YT, F32T>::value;
    extern __shared__ __attribute__((aligned(16))) char shared[];  // codes [rows][128 KB], scales [rows][KB]
    __shared__ float sums[kFewWaves][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int l16 = lane & 15, quad = lane >> 4;
    const int N = args.N, K = args.K, KB = args.KB, n0 = blockIdx.x * 16;
    typename YT::storage* y = static_cast<typename YT::storage*>(args.y);

    // The rows of this workgroup: all of them, or route blockIdx.y's.
    int M = args.M, expert = 0;
    int64_t x_row = 0;
    if (few.ids) {
        const int r = blockIdx.y;
        M = 1;
        expert = few.ids[r];
        x_row = args.rows ? args.rows[r] : r;
        y += int64_t(r) * N;
        if (uint32_t(expert) >= uint32_t(few.experts) || x_row < 0 || x_row >= args.x_rows) {  // (the whole workgroup)
            if (int(threadIdx.x) < 16 && n0 + int(threadIdx.x) < N) store_out<YT>(y, n0 + threadIdx.x, 0.f);
            return;
        }
    }
    const int nblocks = (N + 127) / 128;
    const float* const wsp = args.ws + (int64_t(expert) * nblocks + n0 / 128) * KB;
    const int nrows = min(16, N - n0);
    const __amdgpu_buffer_rsrc_t wr =
        raw_rsrc(args.w + (int64_t(expert) * N + n0) * K, uint32_t(nrows) * uint32_t(K));
    const uint32_t a_off = l16 < nrows ? uint32_t(l16) * uint32_t(K) + 16u * quad : kOutOfRange;
    const uint8_t* const xp = CODED ? args.x + x_row * args.x_stride : nullptr;
    const float* const xsp = CODED ? args.xs + x_row : nullptr;
    const __amdgpu_buffer_rsrc_t xr = raw_rsrc(xp, CODED ? uint32_t(M - 1) * uint32_t(args.x_stride) + uint32_t(K) : 0u);
    const uint32_t b_off = l16 < M ? uint32_t(l16) * uint32_t(args.x_stride) + 16u * quad : kOutOfRange;
    float* const lds_scales = reinterpret_cast<float*>(shared + M * KB * 128);

    struct Block {
        u32x4 a[2], b[2];
        float sx, sw;
    };
    auto load = [&](Block& s, int kb) __attribute__((always_inline)) {
        const uint32_t k = uint32_t(kb) * 128u;
        const int left = K - int(k);  // pieces past K, and blocks past the last, are zeros
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool live = 16 * (quad + 4 * h) < left;
            s.a[h] = __builtin_amdgcn_raw_buffer_load_b128(wr, live ? a_off + 64u * h : kOutOfRange, k, 2);
            if constexpr (CODED) s.b[h] = __builtin_amdgcn_raw_buffer_load_b128(xr, live ? b_off + 64u * h : kOutOfRange, k, 0);
        }
        const int at = min(kb, KB - 1);
        s.sw = wsp[at];
        if constexpr (CODED) s.sx = l16 < M ? xsp[int64_t(at) * args.xs_stride + l16] : 0.f;
    };
    f32x4 acc{};
    auto add = [&](Block& s, int kb) __attribute__((always_inline)) {
        if constexpr (!CODED) {
            s.b[0] = s.b[1] = u32x4{};
            s.sx = 0.f;
            if (l16 < M) {
                const char* const row = shared + (l16 * KB + kb) * 128 + 16 * quad;
                s.b[0] = *reinterpret_cast<const u32x4*>(row);
                s.b[1] = *reinterpret_cast<const u32x4*>(row + 64);
                s.sx = lds_scales[l16 * KB + kb];
            }
        }
        Operand<EXACT> a, b;
        a.take(s.a[0], s.a[1]);
        b.take(s.b[0], s.b[1]);
        const f32x4 p = block_sums(a, b);
        const float scale = s.sx * s.sw;
#pragma unroll
        for (int r = 0; r < 4; r++) acc[r] = fmaf(scale, p[r], acc[r]);
    };

    Block s[kFewAhead];
#pragma unroll
    for (int i = 0; i < kFewAhead; i++) load(s[i], wave + kFewWaves * i);
    if constexpr (!CODED) {
        // 16 lanes a group of 128 values, eight each; what lies past K is a code of 0
        using S = typename XT::storage;
        const S* const x = static_cast<const S*>(few.x) + x_row * args.x_stride;
        const int groups = M * KB;
        for (int g = threadIdx.x >> 4; g < groups; g += 64 * kFewWaves / 16) {
            const int m = g / KB, at = (g - m * KB) * 128 + l16 * 8;
            float v[8] = {};
            if (at < K) load8<XT>(x + m * args.x_stride + at, v);
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) most = max(most, abs_bits(v[i]));
            const Fp8Group q(max16(most));
            *reinterpret_cast<uint2*>(shared + g * 128 + l16 * 8) = make_uint2(q.codes4(v), q.codes4(v + 4));
            if (l16 == 0) lds_scales[g] = q.scale;
        }
        lds_barrier();
    }
    for (int kb = wave; kb < KB; kb += kFewWaves * kFewAhead) {
#pragma unroll
        for (int i = 0; i < kFewAhead; i++) {
            const int at = kb + kFewWaves * i;
            if (at < KB) {
                add(s[i], at);
                load(s[i], at + kFewWaves * kFewAhead);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) sums[wave][l16][4 * quad + r] = acc[r];
    __syncthreads();
    const int m = threadIdx.x >> 4, n = n0 + l16;
    if (m < min(M, 16) && n < N) {
        float t = sums[0][m][l16];
#pragma unroll
        for (int i = 1; i < kFewWaves; i++) t += sums[i][m][l16];
        store_out<YT>(y, int64_t(m) * N + n, t);
    }
}

}  // namespace

bool fp8_few_takes(int64_t m, int64_t k, int x_dtype) {
    if (x_dtype == EQ_DTYPE_F8E4M3) return m <= 16;
    return m <= 4 && m * fp8_blocks(k) * 132 <= kFewLds;
}

void launch_fp8_few(const Fp8Args& a, const Fp8Few& f, int y_dtype, hipStream_t st) {
    const dim3 grid(unsigned((a.N + 15) / 16), f.ids ? unsigned(a.M) : 1u);
    const bool coded = f.x_dtype == EQ_DTYPE_F8E4M3;
    const size_t lds = coded ? 0 : size_t(f.ids ? 1 : a.M) * size_t(a.KB) * 132;
    with_dtype(y_dtype, [&](auto yt) {
        using YT = decltype(yt);
        if (coded) {
            fp8_few_kernel<F8T, YT><<<grid, dim3(64 * kFewWaves), 0, st>>>(a, f);
        } else {
            with_dtype(f.x_dtype, [&](auto xt) {
                fp8_few_kernel<decltype(xt), YT><<<grid, dim3(64 * kFewWaves), lds, st>>>(a, f);
            });
        }
    });
}

}  // namespace eq

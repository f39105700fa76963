// Products of few rows (at most 16, or one for each route) with e4m3 weights:
// bound by reading the weights once.
//
// A workgroup of WAVES waves has 16 NT weight rows; wave v takes the blocks v,
// v + WAVES, .. of K, a block being one matrix instruction a tile (fp8_matmul.hip), and
// the waves' sums are added through LDS in wave order.  Each wave brings its
// blocks into a ring of its own in LDS, AHEAD blocks before it needs them, and
// waits for none of the others.  (Straight into the operand's registers a load
// touches half a line of 16 rows, and 64 KiB took 1.7 us of a compute unit's address unit, this way 0.6.)
// Rows of values (at most 4) are quantized by the workgroup into LDS while its first weights are on their way.
//
// 8 waves, 16 rows and one block ahead leave room for more workgroups on a compute unit, which is worth
// more than a deeper ring (us in graphs; ahead 3 and 1: 16 rows of codes by 14336 x 4096 16.7, 13.0;
// a row of values by 14336 x 4096 13.3, 11.6; by 4096 x 4096 5.5, 5.4).  Where 64 rows to a workgroup of 4 waves
// fill the GPU, rows of codes are read a quarter as often (the first of those 11.1; 64 routes of 2048 x 768 24.9, 15.7).
#include "fp8_product.hpp"

namespace eq {
namespace {

constexpr int kFewLds = 48 * 1024;  // codes and scales of the rows, where the kernel makes them

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) const float lds_f32;

struct F8T {};  // x in codes

// ROWS8: loads of 8 rows of x (0: the kernel quantizes them).
template <typename XT, typename YT, int WAVES, int NT, int ROWS8, int AHEAD>
__global__ __launch_bounds__(64 * WAVES) void fp8_few_kernel(const Fp8Args args, const Fp8Few few) {
    constexpr bool CODED = std::is_same<XT, F8T>::value, EXACT = std::is_same<YT, F32T>::value;
    static_assert(CODED == (ROWS8 > 0), "rows in codes are loaded");
    constexpr int A_BYTES = NT * 2048, B_BYTES = ROWS8 * 1024, SLOT = A_BYTES + B_BYTES + (CODED ? 256 : 0);
    constexpr int LOADS = 2 * NT + ROWS8 + (CODED ? 1 : 0), RING = AHEAD + 1;
    constexpr int SUMS = WAVES * NT * 16 * 17 * 4, BYTES = WAVES * RING * SLOT;
    __shared__ __attribute__((aligned(16))) char ring[BYTES > SUMS ? BYTES : SUMS];  // and the sums, afterwards
    extern __shared__ __attribute__((aligned(16))) char coded[];                      // codes [rows][128 KB], scales [rows][KB]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int l16 = lane & 15, quad = lane >> 4;
    const int N = args.N, K = args.K, KB = args.KB, n0 = blockIdx.x * 16 * NT;
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
            if (int(threadIdx.x) < 16 * NT && n0 + int(threadIdx.x) < N) store_out<YT>(y, n0 + threadIdx.x, 0.f);
            return;
        }
    }
    const int nblocks = (N + 127) / 128;
    typedef __attribute__((address_space(4))) const float const_f32;
    const_f32* const wsp = (const_f32*)(args.ws + (int64_t(expert) * nblocks + n0 / 128) * KB);
    const int nrows = min(16 * NT, N - n0);
    const __amdgpu_buffer_rsrc_t wr = raw_rsrc(args.w + (int64_t(expert) * N + n0) * K, uint32_t(nrows) * uint32_t(K));
    const uint8_t* const xp = CODED ? args.x + x_row * args.x_stride : nullptr;
    const float* const xsp = CODED ? args.xs + x_row : nullptr;
    const __amdgpu_buffer_rsrc_t xr = raw_rsrc(xp, CODED ? uint32_t(M - 1) * uint32_t(args.x_stride) + uint32_t(K) : 0u);

    // Load i of the weights is rows 8 i ..: lane l has row l / 8 of them and the chunk that belongs in slot l % 8,
    // c ^ (row / 2) % 8, so that 16 rows are read at one chunk without bank conflicts.
    const int row8 = lane >> 3;
    uint32_t a_off[8], b_off[2];  // (the first 2 NT and ROWS8 used; bounds that depend on NT fail clang's host pass in a lambda)
    int chunk[2];                      // of even and odd loads
#pragma unroll
    for (int i = 0; i < 2; i++) chunk[i] = (lane & 7) ^ ((4 * i + (row8 >> 1)) & 7);
#pragma unroll
    for (int i = 0; i < 2 * NT; i++)
        a_off[i] = 8 * i + row8 < nrows ? uint32_t(8 * i + row8) * uint32_t(K) + 16u * chunk[i & 1] : kOutOfRange;
#pragma unroll
    for (int i = 0; i < 2; i++)
        b_off[i] = 8 * i + row8 < M ? uint32_t(8 * i + row8) * uint32_t(args.x_stride) + 16u * chunk[i] : kOutOfRange;
    lds_char* const mine = (lds_char*)ring + wave * RING * SLOT;
    auto load = [&](int kb, int slot) __attribute__((always_inline)) {
        const uint32_t k = uint32_t(kb) * 128u;
        const int left = K - int(k);  // chunks past K, and blocks past the last, are zeros
        lds_char* const to = mine + slot * SLOT;
#pragma unroll
        for (int i = 0; i < 2 * NT; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(to + i * 1024), 16,
                                                     16 * chunk[i & 1] < left ? a_off[i] : kOutOfRange, k, 0, 0);
        if constexpr (CODED) {
#pragma unroll
            for (int i = 0; i < ROWS8; i++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(to + A_BYTES + i * 1024), 16,
                                                         16 * chunk[i] < left ? b_off[i] : kOutOfRange, k, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(raw_rsrc(xsp + int64_t(min(kb, KB - 1)) * args.xs_stride, uint32_t(M) * 4u),
                                                     (lds_void*)(to + A_BYTES + B_BYTES), 4,
                                                     lane < M ? uint32_t(lane) * 4u : kOutOfRange, 0, 0, 0);
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) load(wave + WAVES * i, i);
    lds_f32* const lds_scales = (lds_f32*)((lds_char*)coded + M * KB * 128);
    if constexpr (!CODED) {
        // 16 lanes a group of 128 values, eight each; what lies past K is a code of 0
        using S = typename XT::storage;
        const S* const x = static_cast<const S*>(few.x) + x_row * args.x_stride;
        const int groups = M * KB;
        for (int g = threadIdx.x >> 4; g < groups; g += 64 * WAVES / 16) {
            const int m = g / KB, at = (g - m * KB) * 128 + l16 * 8;
            float v[8] = {};
            if (at < K) load8<XT>(x + m * args.x_stride + at, v);
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) most = max(most, abs_bits(v[i]));
            const Fp8Group q(max16(most));
            *reinterpret_cast<uint2*>(coded + g * 128 + l16 * 8) = make_uint2(q.codes4(v), q.codes4(v + 4));
            if (l16 == 0) *reinterpret_cast<float*>(coded + M * KB * 128 + g * 4) = q.scale;
        }
        lds_barrier();
    }

    f32x4 acc[NT] = {};
    const uint32_t at0 = uint32_t(l16 * 128 + ((quad ^ ((l16 >> 1) & 7)) << 4));  // chunks quad and quad + 4 of row l16
    int slot = 0;
#pragma unroll 1
    for (int kb = wave; kb < KB; kb += WAVES) {
        const float sw = wsp[kb];
        load(kb + WAVES * AHEAD, slot == 0 ? AHEAD : slot - 1);
        // this block has landed, the AHEAD after it may be on their way
        constexpr int LATER = LOADS * AHEAD;
        static_assert(LATER < 64, "vmcnt range");
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
        const lds_char* const from = mine + slot * SLOT;
        Operand<EXACT> a, b;
        float sx;
        if constexpr (CODED) {
            const lds_char* const row = from + A_BYTES;
            const u32x4 zero{};
            // (rows behind the loaded ones of x are zeros)
            const bool live = ROWS8 == 2 || l16 < 8;
            const uint32_t at = ROWS8 == 2 ? at0 : at0 & 1023u;
            const u32x4 lo = *(lds_u32x4*)(row + at), hi = *(lds_u32x4*)(row + (at ^ 64u));
            b.take(live ? lo : zero, live ? hi : zero);
            sx = *(lds_f32*)(from + A_BYTES + B_BYTES + l16 * 4);
        } else {
            u32x4 lo{}, hi{};
            sx = 0.f;
            if (l16 < M) {
                const lds_char* const row = (lds_char*)coded + (l16 * KB + kb) * 128 + 16 * quad;
                lo = *(lds_u32x4*)row, hi = *(lds_u32x4*)(row + 64);
                sx = lds_scales[l16 * KB + kb];
            }
            b.take(lo, hi);
        }
        const float scale = sx * sw;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            a.take(*(lds_u32x4*)(from + t * 2048 + at0), *(lds_u32x4*)(from + t * 2048 + (at0 ^ 64u)));
            const f32x4 p = block_sums(a, b);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[t][r] = fmaf(scale, p[r], acc[t][r]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (read, before the slot is loaded again)
        slot = slot == AHEAD ? 0 : slot + 1;
    }
    // Nothing is on its way into the ring when the sums take its place.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    float* const sums = reinterpret_cast<float*>(ring);  // [wave][tile][row of x][17]
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) sums[((wave * NT + t) * 16 + l16) * 17 + 4 * quad + r] = acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < M * NT * 16; i += 64 * WAVES) {
        const int m = i / (NT * 16), c = i % (NT * 16), n = n0 + c;
        if (n >= N) continue;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) t += sums[((w * NT + (c >> 4)) * 16 + m) * 17 + (c & 15)];
        store_out<YT>(y, int64_t(m) * N + n, t);
    }
}

}  // namespace

bool fp8_few_takes(int64_t m, int64_t k, int x_dtype) {
    if (x_dtype == EQ_DTYPE_F8E4M3) return m <= 16;
    return m <= 4 && m * fp8_blocks(k) * 132 <= kFewLds;
}

void launch_fp8_few(const Fp8Args& a, const Fp8Few& f, int y_dtype, hipStream_t st) {
    const int m = f.ids ? 1 : a.M;
    const unsigned routes = f.ids ? unsigned(a.M) : 1u;
    auto grid = [&](int rows) { return dim3(unsigned((a.N + rows - 1) / rows), routes); };
    // (of values, of which each workgroup makes its codes itself, there is nothing to read less often)
    const bool wide = f.x_dtype == EQ_DTYPE_F8E4M3 && int64_t((a.N + 63) / 64) * routes * 4 >= 3 * device_cu_count();
    with_dtype(y_dtype, [&](auto yt) {
        using YT = decltype(yt);
        if (f.x_dtype != EQ_DTYPE_F8E4M3)
            with_dtype(f.x_dtype, [&](auto xt) {
                fp8_few_kernel<decltype(xt), YT, 8, 1, 0, 1><<<grid(16), dim3(512), size_t(m) * size_t(a.KB) * 132, st>>>(a, f);
            });
        else if (wide && m <= 8) fp8_few_kernel<F8T, YT, 4, 4, 1, 1><<<grid(64), dim3(256), 0, st>>>(a, f);
        else if (wide) fp8_few_kernel<F8T, YT, 4, 4, 2, 1><<<grid(64), dim3(256), 0, st>>>(a, f);
        else if (m <= 8) fp8_few_kernel<F8T, YT, 8, 1, 1, 1><<<grid(16), dim3(512), 0, st>>>(a, f);
        else fp8_few_kernel<F8T, YT, 8, 1, 2, 1><<<grid(16), dim3(512), 0, st>>>(a, f);
    });
}

}  // namespace eq

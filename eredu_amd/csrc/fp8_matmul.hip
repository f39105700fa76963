// Products of rows in e4m3 codes with e4m3 weights, both with block scales:
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} cx[m, k] cw[n, k]
//
// A block of 128 columns is one v_mfma_f32_16x16x128_f8f6f4 (twice the rate of
// the 16x16x32 fp8 instruction).  Its sums start at zero and are added to the
// f32 accumulators with the scale: four FMAs a lane beside 32 cycles of matrix
// core, so half of the vector unit's time.  The weights are the A operand,
// whose rows are the result's: a lane has results of one activation row, so
// the scale is one register, sx sw, for all of its weight rows.  Which of the
// block's columns a lane's 32 bytes hold is the same for both operands, so it
// can be any of them.
//
// The e4m3 instructions (16x16x32 as well) line the products of 8 neighbouring
// columns up to the largest's exponent and keep 13 bits below it, cut off
// towards zero, before they are summed in f32 (measured with single products).
// That is 2^-13 of a product where the result's own rounding is 2^-9 or 2^-12 of
// the sum, so results of 16 bits take them.  f32 results take the codes as
// bf16, which holds them exactly, through v_mfma_f32_16x16x32_bf16: twice the cycles, and
// sums that are off by f32's rounding alone (of 128 products 7e-8 where the e4m3 ones are off by 5e-5).
#include <algorithm>

#include "fp8_product.hpp"

namespace eq {
namespace {

constexpr int kMostExperts = 4095;  // (two counters each in 64 KiB of LDS with room to spare)

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) const float lds_f32;

// How `tiles` tiles are dealt out to workgroups of which `slots` run at once, a pass: whole ones, but
// where half of the last pass's or more would have none, its tiles are taken in parts of K, `most` at
// the most, whose sums are joined by a kernel of their own.  Of routes the device alone knows how many tiles there are.
struct Passes {
    int whole, rest = 0, parts = 1;
    __host__ __device__ Passes(int tiles, int slots, int most) : whole(tiles) {
        if (most < 2 || tiles % slots == 0) return;
        const int left = tiles % slots, fit = slots / left;
        if (fit < 2) return;
        rest = left, whole = tiles - left, parts = fit < most ? fit : most;
    }
};

// Where tile `tile` of `used` row tiles by args.ntiles lies: in bands of `band` row tiles, column by column in
// each, so that the tiles that run at once are as many rows as columns and share their operands in the XCD's L2.
struct TileAt {
    int n0, first, mrows, expert = 0;  // first: row of x and y, or place in args.order
    __device__ __forceinline__ TileAt(const Fp8Args& args, int used, int tile, int cols, int rows) {
        const int band_at = tile / (args.band * args.ntiles), in_band = tile - band_at * args.band * args.ntiles;
        const int band_rows = min(args.band, used - band_at * args.band);
        const int tm = band_at * args.band + in_band % band_rows;
        n0 = in_band / band_rows * cols;
        if (args.tiles) {
            const int4 t = args.tiles[tm];
            expert = t.x, first = t.y, mrows = t.z;
        } else {
            first = tm * rows, mrows = min(rows, args.M - first);
        }
    }
};

// A lane's results of a row of a tile, the wave's from column `n` on, in pieces of 16 bytes of 16-bit results or f32.
template <typename YT, int NT>
__device__ __forceinline__ void store_rows(const Fp8Args& args, const TileAt& tile, int i, int n, int quad,
                                           const f32x4* v) {
    constexpr int PIECE = std::is_same<YT, F32T>::value ? 4 : 8;
    if (i >= tile.mrows) return;
    const int64_t row = args.tiles ? args.order[tile.first + i].x : tile.first + i;
    typename YT::storage* const y = static_cast<typename YT::storage*>(args.y) + row * args.N;
#pragma unroll
    for (int p = 0; p < 4 * NT / PIECE; p++) {
        float w[PIECE];
#pragma unroll
        for (int e = 0; e < PIECE; e++) w[e] = v[(PIECE * p + e) / 4][e % 4];
        const int at = n + PIECE * (4 * p + quad);
        store_run<YT, PIECE>(y + at, w, args.N - at);
    }
}

// WN x WM waves of NT x MT tiles of 16 x 16: 16 NT WN weight rows by 16 MT WM
// activation rows a workgroup.  Both operands go straight from memory to LDS,
// STAGES blocks of K deep.
//
// A lane's four results of a tile are consecutive, and its neighbours of the three other quads have the next ones:
// row i of a wave's A tile t is its weight row 16 t + i where results are f32, 64 consecutive bytes of a result row to
// a store, and 32 (t / 2) + 8 (i / 4) + 4 (t % 2) + i % 4 where two tiles make the 16 bytes of a lane.  (With
// all of a lane's results in one run a store touches each 64 bytes in quarters: f32 results of 2270 x 11264 x 512
// 51.5 us, this way 41.6; 16-bit ones the same.)
// A row's 128 bytes of a block lie in LDS in slots of 16, chunk c in slot c ^ key: 16 lanes read
// 16 rows at one chunk, LDS has 64 banks of 4 bytes (two rows), so the
// rows of one parity have to differ in their key: (row / 2) % 8 for the
// activations and where A's rows are consecutive, (row / 2) % 2 + 2 (row / 8 % 4) for A's rows of pairs
// (no bank conflict is counted).
//
// What bounds it: 4096 rows by 4096 take 60 us a pass of 256 tiles of 256 x 256 (12288 weight rows, three passes, 181 us;
// 16384, four, 242: 2.3 PFLOP/s), 14336 of them 225 (2.1 PFLOP/s; a library's unscaled fp8 product 217): half of the fourth
// pass is empty, and it takes 44.  In a pass the matrix cores are busy for 45 % of the cycles and the clock is at 1.95 GHz; the time
// follows the data (277 us with codes of more varied bits) and hardly the order of the tiles, which points at power:
// the instructions alone, from registers with the additions beside them, reach 3.6-3.9 PFLOP/s of such data, 4.7 of zeros.
// 512 x 14336 x 4096 (224 tiles of 256 x 128, 32.7 us, 1.8 PFLOP/s): by count 51 000 cycles of LDS a compute unit (39 000 of reads,
// at 128 bytes a cycle) beside 28 700 of matrix cores, of some 70 000.
// 8 us of a tile's 59 are its first loads and its stores.  Tried and not kept: the next block's operands read before
// the waves meet (the same there, small products 2 us slower), rotating the blocks' order from workgroup to
// workgroup and fetching ahead into L2 (the same or slower).
template <typename YT, int WN, int WM, int NT, int MT, int STAGES>
__global__ __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(1, 2))) void fp8_tile_kernel(
    const Fp8Args args) {
    constexpr int WAVES = WN * WM, TN = 16 * NT * WN, TM = 16 * MT * WM;
    constexpr int LA = TN / 8 / WAVES, LB = TM / 8 / WAVES;  // loads of 1 KiB (8 rows) a wave
    constexpr int LOADS = LA + LB + 1;                        // and one of scales
    static_assert(LA * 8 * WAVES == TN && LB * 8 * WAVES == TM && LA <= 8 && LB <= 8, "whole loads");
    static_assert(128 % (16 * NT) == 0, "a wave's weight rows have one scale");
    constexpr int SROWS = (TM + 63) & ~63, BUF = (TN + TM) * 128 + SROWS * 4;
    static_assert(64 * WAVES >= SROWS, "a scale load a wave");
    static_assert(STAGES >= 2 && STAGES <= 4, "buffers");
    constexpr bool EXACT = std::is_same<YT, F32T>::value;
    // (separate arrays, so that the compiler knows that a read of one does not wait for loads into another)
    __shared__ __attribute__((aligned(16))) char buf0[BUF], buf1[BUF], buf2[STAGES > 2 ? BUF : 16],
        buf3[STAGES > 3 ? BUF : 16];
    auto buf = [&](int i) __attribute__((always_inline)) {
        return i == 0 ? (lds_char*)buf0 : i == 1 ? (lds_char*)buf1 : i == 2 ? (lds_char*)buf2 : (lds_char*)buf3;
    };

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    const int wn = wave % WN, wm = wave / WN, l16 = lane & 15, quad = lane >> 4;
    const int N = args.N, K = args.K;

    // The workgroups of one XCD (id % 8) take a run of the whole tiles, then one of the last pass's parts.
    const int used = args.tiles ? args.tiles[args.mtiles].x : args.mtiles;
    const Passes passes(used * args.ntiles, args.slots, args.parts);
    const int whole = (passes.whole + 7) & ~7;
    const bool parted = int(blockIdx.x) >= whole;
    const int at = parted ? blockIdx.x - whole : blockIdx.x, total = parted ? passes.rest * passes.parts : passes.whole;
    const int run = (total + 7) >> 3, id = (at & 7) * run + (at >> 3);
    if ((at >> 3) >= run || id >= total) return;  // (the whole workgroup)
    const int split = parted ? id / passes.rest : 0, parts = parted ? passes.parts : 1;
    const TileAt tile(args, used, parted ? passes.whole + id - split * passes.rest : id, TN, TM);
    const int n0 = tile.n0, mrows = tile.mrows, expert = tile.expert;
    // Blocks of K: those of this part.
    const int k_begin = args.KB * split / parts, k_end = args.KB * (split + 1) / parts;

    const uint8_t* xp = args.x;
    const float* xsp = args.xs;
    uint32_t x_bytes = uint32_t((args.x_rows - 1) * args.x_stride + K);
    if (!args.tiles) {
        xp += tile.first * args.x_stride;
        xsp += tile.first;
        x_bytes = uint32_t(mrows - 1) * uint32_t(args.x_stride) + uint32_t(K);
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[t][j] = f32x4{};

    if (expert >= 0) {
        const int nrows = min(TN, N - n0);
        const __amdgpu_buffer_rsrc_t xr = raw_rsrc(xp, x_bytes);
        const __amdgpu_buffer_rsrc_t wr =
            raw_rsrc(args.w + (int64_t(expert) * N + n0) * K, uint32_t(nrows) * uint32_t(K));
        const int nblocks = (N + 127) / 128, nb = min((n0 + 16 * NT * wn) / 128, nblocks - 1);
        // (scalar loads, which the count of vector loads below leaves out)
        typedef __attribute__((address_space(4))) const float const_f32;
        const_f32* const wsp = (const_f32*)(args.ws + (int64_t(expert) * nblocks + nb) * args.KB);

        // Lane l of load i of a wave: row 8 (L wave + i) + l / 8 of the tile, the chunk that belongs in slot l % 8.
        uint32_t a_off[8], b_off[8], s_off;  // (the first LA and LB used)
        auto a_chunk = [&](int i) __attribute__((always_inline)) {
            const int row = 8 * (LA * wave + i) + (lane >> 3);
            return (lane & 7) ^ (EXACT ? (row >> 1) & 7 : ((row >> 1) & 1) | ((row >> 3) & 3) << 1);
        };
        auto b_chunk = [&](int i) __attribute__((always_inline)) {
            const int row = 8 * (LB * wave + i) + (lane >> 3);
            return (lane & 7) ^ ((row >> 1) & 7);
        };
        // the x row of tile row i, -1 past the tile's end
        auto x_row = [&](int i) __attribute__((always_inline)) {
            if (i >= mrows) return -1;
            if (!args.tiles) return i;
            return args.order[tile.first + i].y;
        };
#pragma unroll
        for (int i = 0; i < LA; i++) {
            const int row = 8 * (LA * wave + i) + (lane >> 3);
            a_off[i] = row < nrows ? uint32_t(row) * uint32_t(K) + 16u * a_chunk(i) : kOutOfRange;
        }
#pragma unroll
        for (int i = 0; i < LB; i++) {
            const int r = x_row(8 * (LB * wave + i) + (lane >> 3));
            b_off[i] = r >= 0 ? uint32_t(r) * uint32_t(args.x_stride) + 16u * b_chunk(i) : kOutOfRange;
        }
        const int s_wave = wave % (SROWS / 64);
        {
            const int r = x_row(64 * s_wave + lane);
            s_off = r >= 0 ? uint32_t(r) * 4u : kOutOfRange;
        }
        const uint32_t s_bytes = uint32_t(args.tiles ? args.x_rows : mrows) * 4u;

        // Load q of block kb into a buffer: weights, activations, scales.
        auto load = [&](lds_char* to, int kb, int q) __attribute__((always_inline)) {
            if (q < LA)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    wr, (__attribute__((address_space(3))) void*)(to + (LA * wave + q) * 1024), 16, a_off[q < LA ? q : 0],
                    uint32_t(kb) * 128u, 0, 0);
            else if (q < LA + LB)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    xr, (__attribute__((address_space(3))) void*)(to + TN * 128 + (LB * wave + q - LA) * 1024), 16,
                    b_off[q >= LA && q < LA + LB ? q - LA : 0], uint32_t(kb) * 128u, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    raw_rsrc(xsp + min(kb, args.KB - 1) * args.xs_stride, s_bytes),
                    (__attribute__((address_space(3))) void*)(to + (TN + TM) * 128 + s_wave * 256), 4, s_off, 0, 0, 0);
        };
        // Before the loads of block kb: of the last block the chunks past K, and behind the split's all, are zeros.
        auto limit = [&](int kb) __attribute__((always_inline)) {
            const int left = kb < k_end ? K - kb * 128 : 0;
            if (left >= 128) return;
#pragma unroll
            for (int i = 0; i < LA; i++) a_off[i] = 16 * a_chunk(i) < left ? a_off[i] : kOutOfRange;
#pragma unroll
            for (int i = 0; i < LB; i++) b_off[i] = 16 * b_chunk(i) < left ? b_off[i] : kOutOfRange;
        };

        // A: weight row of tile t is a_row + 16 t, or where results are pieces of eight a_row + 32 (t / 2) + 4 (t % 2);
        // B: activation row 16 (MT wm + j) + l16.  Chunks quad and quad + 4.
        const int a_row = 16 * NT * wn + (EXACT ? l16 : 8 * (l16 >> 2) + (l16 & 3));
        const int a_key = EXACT ? l16 >> 1 : ((l16 >> 1) & 1) | ((l16 >> 2) << 1);
        const uint32_t a_at = uint32_t(a_row * 128 + ((quad ^ a_key) << 4));
        const uint32_t b_at = uint32_t(TN * 128 + (16 * MT * wm + l16) * 128 + ((quad ^ ((l16 >> 1) & 7)) << 4));
        const uint32_t s_at = uint32_t((TN + TM) * 128 + (16 * MT * wm + l16) * 4);
        // Multiplies a block from one buffer while block kb is loaded into another, a load every EVERY matrix
        // instructions (over the first half of them; all at once before them cost 3 %).
        auto compute = [&](lds_char* from, float sw, lds_char* to, int kb) __attribute__((always_inline)) {
            constexpr int EVERY = NT * MT / 2 / LOADS > 1 ? NT * MT / 2 / LOADS : 1;
            Operand<EXACT> a[NT], b[2];
            float s[2];
            auto read_b = [&](int j) __attribute__((always_inline)) {
                b[j & 1].take(*(lds_u32x4*)(from + b_at + j * 2048), *(lds_u32x4*)(from + (b_at ^ 64u) + j * 2048));
                s[j & 1] = *(lds_f32*)(from + s_at + j * 64) * sw;
            };
            read_b(0);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int at = 128 * (EXACT ? 16 * t : 32 * (t / 2) + 4 * (t % 2));
                a[t].take(*(lds_u32x4*)(from + a_at + at), *(lds_u32x4*)(from + (a_at ^ 64u) + at));
            }
            // Tile i = NT j + t is multiplied while tile i - LAG's sums, which have arrived by then, are
            // scaled and added (a single wave: 72 cycles a tile with LAG 2, 38 with 3, 32 of them the matrix core's).
            constexpr int LAG = 3;
            f32x4 p[LAG + 1];
            float scale[LAG + 1];
#pragma unroll
            for (int i = 0; i < NT * MT + LAG; i++) {
                if (i < NT * MT) {
                    const int j = i / NT, t = i % NT;
                    if (t == 0 && j + 1 < MT) read_b(j + 1);
                    p[i % (LAG + 1)] = block_sums(a[t], b[j & 1]);
                    scale[i % (LAG + 1)] = s[j & 1];
                    if (i % EVERY == 0 && i / EVERY < LOADS) load(to, kb, i / EVERY);
                    if (i == NT * MT - 1) {
#pragma unroll
                        for (int q = (NT * MT - 1) / EVERY + 1; q < LOADS; q++) load(to, kb, q);
                    }
                }
                if (i >= LAG) {
                    const int j = (i - LAG) / NT, t = (i - LAG) % NT, q = (i - LAG) % (LAG + 1);
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[t][j][r] = fmaf(scale[q], p[q][r], acc[t][j][r]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // (the sums are done here: the compiler would else move the additions behind the
            // next block's branches, with a register for every product)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < MT; j++) asm volatile("" : "+v"(acc[t][j]));
        };
        // The oldest block on its way has landed and this wave's reads are done; then all waves'.
        auto turn = [&]() __attribute__((always_inline)) {
            constexpr int N = LOADS * (STAGES - 2);
            __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));  // vmcnt(N) lgkmcnt(0)
            asm volatile("s_barrier" ::: "memory");
        };

#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) {
            limit(k_begin + i);
#pragma unroll
            for (int q = 0; q < LOADS; q++) load(buf(i), k_begin + i, q);
        }
        float sw = wsp[k_begin];
        auto step = [&](int kb, int i) __attribute__((always_inline)) {
            const float next = wsp[min(kb + 1, k_end - 1)];
            turn();
            limit(kb + STAGES - 1);
            compute(buf(i), sw, buf((i + STAGES - 1) % STAGES), kb + STAGES - 1);
            sw = next;
        };
        int kb = k_begin;
        for (; kb + STAGES <= k_end; kb += STAGES) {
#pragma unroll
            for (int i = 0; i < STAGES; i++) step(kb + i, i);
        }
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++)
            if (kb + i < k_end) step(kb + i, i);
        __builtin_amdgcn_s_waitcnt(0x0070);  // (nothing is on its way to LDS when the workgroup ends)
    }

    if (parted) {
        f32x4* const part = reinterpret_cast<f32x4*>(args.part + int64_t(id) * (TN * TM)) + threadIdx.x;
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int t = 0; t < NT; t++) part[(j * NT + t) * 64 * WAVES] = acc[t][j];
        return;
    }
#pragma unroll
    for (int j = 0; j < MT; j++) {
        f32x4 v[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) v[t] = acc[t][j];
        store_rows<YT, NT>(args, tile, 16 * (MT * wm + j) + l16, n0 + 16 * NT * wn, quad, v);
    }
}

// The last pass's tiles: their parts' sums, in their order.  A workgroup has a 1 / MT of a tile, a thread what
// the tile's thread of its number had of it.  Bound by its chain of loads: 4.0 us for 7 parts of 77 x 4097, 4.7 behind
// 1554 routes of 4096.
template <typename YT, int WN, int WM, int NT, int MT>
__global__ __launch_bounds__(64 * WN * WM) void fp8_join_kernel(const Fp8Args args) {
    constexpr int WAVES = WN * WM, TN = 16 * NT * WN, TM = 16 * MT * WM;
    const int used = args.tiles ? args.tiles[args.mtiles].x : args.mtiles;
    const Passes passes(used * args.ntiles, args.slots, args.parts);
    const int i = blockIdx.x / MT, j = blockIdx.x - i * MT;
    if (i >= passes.rest || passes.parts == 1) return;
    const TileAt tile(args, used, passes.whole + i, TN, TM);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave % WN, wm = wave / WN;
    const int row = 16 * (MT * wm + j) + (lane & 15);
    if (row >= tile.mrows) return;
    const int64_t step = int64_t(passes.rest) * (TN * TM / 4);
    const f32x4* p = reinterpret_cast<const f32x4*>(args.part + int64_t(i) * (TN * TM)) + j * NT * 64 * WAVES + threadIdx.x;
    f32x4 v[NT] = {};
    int s = 0;
    auto add = [&](auto count) __attribute__((always_inline)) {  // several at once: their loads do not wait for each other
        constexpr int C = decltype(count)::value;
        f32x4 q[4][NT];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int t = 0; t < NT; t++) q[c][t] = p[(s + c) * step + t * 64 * WAVES];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) v[t][r] += q[c][t][r];
        s += C;
    };
    while (s + 4 <= passes.parts) add(std::integral_constant<int, 4>{});
    while (s < passes.parts) add(std::integral_constant<int, 1>{});
    store_rows<YT, NT>(args, tile, row, tile.n0 + 16 * NT * wn, lane >> 4, v);
}

// The routes of each expert side by side, and the row tiles that they make
// (fp8_tile_kernel's `tiles` and `order`).  Routes without an expert or a row come last, as expert -1.  An expert's
// routes stay in their order: which tile a route is in can decide in how many parts its products are summed.
// A workgroup places `chunk` routes (a multiple of 256).  It counts all of them, those before its own
// apart, so that it needs nothing of another one.  It places 64 after 64, whose order among themselves they find by
// comparing the bits of their experts' numbers.
// Neighbouring routes of one expert are counted by one of them (sorted routes would else queue for one counter).
// A chain of loads, counting, sums and stores bounds it, a launch of 2.5 us included: 4.2 us for 100 routes, 6.0 for 4096 of 128
// experts, 9.2 for 16384, 18 for 40000 (one workgroup for all, in any order: 4.0, 6.2, 17, 42).
__global__ __launch_bounds__(1024) void fp8_routes_kernel(int4* __restrict__ tiles, int2* __restrict__ order,
                                                          const int32_t* __restrict__ ids,
                                                          const int32_t* __restrict__ rows, int routes, int chunk,
                                                          int experts, int64_t x_rows, int tile_rows, int mtiles) {
    extern __shared__ int shared[];
    int* const before = shared;               // [experts + 1] routes of each expert before this workgroup's, then places
    int* const rest = shared + experts + 1;   // [experts + 1] the others
    __shared__ int sums[2][16], base[2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int begin = blockIdx.x * chunk, end = min(begin + chunk, routes);
    auto fetch = [&](int r, int& e, int& row) __attribute__((always_inline)) {
        r = min(r, routes - 1);
        e = ids[r];
        row = rows ? rows[r] : r;
    };
    // route r's counter (-1: no route)
    auto bucket = [&](int r, int e, int row) __attribute__((always_inline)) {
        if (r >= routes) return -1;
        return uint32_t(e) < uint32_t(experts) && row >= 0 && row < x_rows ? e : experts;
    };
    // The first of a run of lanes with one counter counts them all.
    auto add = [&](int* counters, int b) __attribute__((always_inline)) {
        const int ahead = __shfl_up(b, 1);
        const bool head = lane == 0 || b != ahead;
        const uint64_t heads = __ballot(head), behind = lane == 63 ? 0 : heads >> (lane + 1);
        const int run = behind ? __ffsll((unsigned long long)behind) : 64 - lane;
        if (head && b >= 0) atomicAdd(&counters[b], run);
    };
    constexpr int STEP = 4;  // steps of 1024 routes whose loads are on their way together
    for (int e = threadIdx.x; e <= experts; e += 1024) before[e] = rest[e] = 0;
    if (threadIdx.x < 2) base[threadIdx.x] = 0;
    int own, own_row;
    fetch(begin + threadIdx.x, own, own_row);
    __syncthreads();
#pragma unroll 1
    for (int r0 = 0; r0 < routes; r0 += 1024 * STEP) {  // (all lanes of a wave go together)
        int e[STEP], row[STEP];
#pragma unroll
        for (int i = 0; i < STEP; i++) fetch(r0 + 1024 * i + threadIdx.x, e[i], row[i]);
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            const int r = r0 + 1024 * i;
            if (r < routes) add(r + 64 * wave < begin ? before : rest, bucket(r + threadIdx.x, e[i], row[i]));
        }
    }
    __syncthreads();
    // running sums of routes and tiles over the experts, 1024 of them a step
#pragma unroll 1
    for (int e0 = 0; e0 <= experts; e0 += 1024) {
        const int e = e0 + threadIdx.x, own_at = e <= experts ? before[e] : 0, c = e <= experts ? own_at + rest[e] : 0;
        const int t = (c + tile_rows - 1) / tile_rows;
        int cs = c, ts = t;
        for (int o = 1; o < 64; o <<= 1) {
            const int cu = __shfl_up(cs, o), tu = __shfl_up(ts, o);
            if (lane >= o) cs += cu, ts += tu;
        }
        if (lane == 63) sums[0][wave] = cs, sums[1][wave] = ts;
        __syncthreads();
        int cb = base[0], tb = base[1];
#pragma unroll
        for (int i = 0; i < 15; i++) {
            const int cw = sums[0][i], tw = sums[1][i];
            if (i < wave) cb += cw, tb += tw;
        }
        __syncthreads();
        if (threadIdx.x == 1023) base[0] = cb + cs, base[1] = tb + ts;
        if (e <= experts) {
            before[e] = cb + cs - c + own_at;
            for (int i = blockIdx.x; i < t; i += gridDim.x)
                if (tb + ts - t + i < mtiles)  // (always: mtiles is what the routes can make)
                    tiles[tb + ts - t + i] =
                        make_int4(e < experts ? e : -1, cb + cs - c + i * tile_rows, min(tile_rows, c - i * tile_rows), 0);
        }
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) tiles[mtiles] = make_int4(base[1], 0, 0, 0);
    const int bits = 32 - __clz(experts);
#pragma unroll 1
    for (int r0 = begin; r0 < end; r0 += 256) {
        const int r = r0 + threadIdx.x;
        if (r0 > begin) fetch(r, own, own_row);
        const int b = wave < 4 ? bucket(r, own, own_row) : -1;
        uint64_t same = __ballot(b >= 0);
        for (int i = 0; i < bits; i++) {
            const bool bit = b >> i & 1;
            const uint64_t with = __ballot(bit);
            same &= bit ? with : ~with;
        }
        const int rank = __popcll(same & ((uint64_t(1) << lane) - 1));
        int at = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            if (wave == w && b >= 0) {
                at = before[b] + rank;
                if (rank == 0) before[b] = at + __popcll(same);
            }
            __syncthreads();
        }
        if (b >= 0) order[at] = make_int2(r, b < experts ? own_row : -1);
    }
}

template <typename YT, int WN, int WM, int NT, int MT, int STAGES>
void launch_tile(const Fp8Args& a, hipStream_t st) {
    // (of routes there are as many row tiles as a.mtiles or fewer)
    const int tiles = a.mtiles * a.ntiles;
    const Passes passes(tiles, a.slots, a.parts);
    const bool joined = a.tiles ? a.parts > 1 : passes.parts > 1;
    const int total = a.tiles ? tiles + (joined ? a.slots : 0) : ((passes.whole + 7) & ~7) + passes.rest * passes.parts;
    fp8_tile_kernel<YT, WN, WM, NT, MT, STAGES><<<dim3(unsigned(total + 7) / 8 * 8), dim3(64 * WN * WM), 0, st>>>(a);
    if (!joined) return;
    const int rest = a.tiles ? std::min(tiles, a.slots / 2) : passes.rest;
    fp8_join_kernel<YT, WN, WM, NT, MT><<<dim3(unsigned(rest * MT)), dim3(64 * WN * WM), 0, st>>>(a);
}

// The tile shapes, weight rows by activation rows, and what a workgroup of each took (measured over products
// of 32 .. 4096 rows): us before and after its blocks, us a block alone on its compute unit, and where two share one; of
// routes, whose weights are read by few workgroups each and come from memory, so many times as long where
// two buffers have only one block on its way (1554 routes to 8 experts of 4096 x 14336, 256 x 192: 1.6 us a block).
struct Shape {
    int cols, rows;
    float fixed, one, two, routed;  // two 0: a second one does not fit
};
constexpr Shape kShapes[] = {{256, 256, 8.f, 1.5f, 0.f, 1.25f}, {256, 192, 7.f, 1.2f, 0.f, 1.3f}, {256, 128, 5.f, .9f, 0.f, 1.f},
                             {128, 128, 2.f, .72f, 1.02f, 1.f}, {128, 96, 2.f, .5f, 0.f, 1.f},
                             {128, 64, 2.f, .38f, .58f, 1.f}, {128, 32, 2.f, .26f, 0.f, 1.f}};
constexpr int kWide = 3;  // the shapes of 256 weight rows: their f32 results would need more registers than there are
template <typename YT>
void launch_tiles(int shape, const Fp8Args& a, hipStream_t st) {
    if constexpr (!std::is_same<YT, F32T>::value) {
        if (shape == 0) launch_tile<YT, 4, 2, 4, 8, 2>(a, st);
        if (shape == 1) launch_tile<YT, 4, 2, 4, 6, 2>(a, st);
        if (shape == 2) launch_tile<YT, 4, 2, 4, 4, 3>(a, st);
    }
    if (shape == 3) launch_tile<YT, 2, 2, 4, 4, 2>(a, st);
    if (shape == 4) launch_tile<YT, 4, 1, 2, 6, 3>(a, st);
    if (shape == 5) launch_tile<YT, 4, 1, 2, 4, 3>(a, st);
    if (shape == 6) launch_tile<YT, 4, 1, 2, 2, 4>(a, st);
}

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

constexpr int kBand = 8;  // row tiles of a band
constexpr int64_t kMostTiles = (int64_t(1) << 23) - 4096;  // (fewer than 2^32 threads, with a pass of parts behind them)

// How a product is done, from its sizes and types alone (the scratch queries
// and the calls go by the same), and its scratch: lists of routes, the codes and scales of x, sums of splits.
struct Plan {
    bool few = false;  // fp8_few.hip's kernel, on x as it is where that takes it
    int shape = 0;     // else a tile of kShapes
    int64_t mtiles = 0, ntiles = 0, slots = 0, parts = 1;
    size_t tiles = 0, order = 0, codes = 0, scales = 0, part = 0;
    size_t bytes() const { return tiles + order + codes + scales + part; }
};

int64_t slots_of(const Shape& s) { return int64_t(s.two > 0.f ? 2 : 1) * device_cu_count() & ~int64_t(7); }

// Us that a product takes in `tiles` tiles of a shape, those of the last pass in `most` parts of K or
// fewer; what the tiles load comes from the caches at `rate` bytes a us, `bytes` of weights at 6 TB/s, which is
// overlapped with all but a quarter.  Of routes `tiles` is a guess.
double tiles_us(const Shape& s, int64_t tiles, int64_t blocks, int64_t most, double rate, double bytes, bool routed) {
    const int64_t slots = slots_of(s), cus = device_cu_count();
    auto took = [&](int64_t at_once, int64_t per) {
        return s.fixed + double(per) * (at_once > cus ? s.two : s.one) * (routed ? s.routed : 1.f);
    };
    const double unit = double(s.cols) * s.rows * 8. / 6e6;  // a part's sums, written and read (their kernel and its launch: 8)
    double us;
    if (routed && tiles > slots) {
        // half of the slots in the last pass, or a quarter in parts
        us = double(tiles) / double(slots) * took(slots, blocks);
        us += most > 1 ? took(cus, blocks / std::min<int64_t>(most, 4)) + 8. + double(slots) * unit : .5 * took(slots, blocks);
    } else {
        const Passes r{int(tiles), int(slots), int(most)};
        const int64_t parts = int64_t(r.rest) * r.parts;
        us = double(r.whole / slots) * took(slots, blocks);
        if (r.whole % slots) us += took(r.whole % slots, blocks);
        if (parts) us += took(parts, (blocks + r.parts - 1) / r.parts) + 8. + double(parts) * unit;
    }
    us = std::max(us, double(tiles * blocks) * double(s.cols + s.rows) * 128. / rate);
    const double read = bytes / 6e6;
    return std::max(us, read) + .25 * std::min(us, read);
}

// The shape of a product of m rows, in experts or not, its tiles and the parts of the last pass's.
void choose_tiles(Plan& p, int64_t m, int64_t n, int64_t k, int64_t experts, int y_dtype) {
    const int64_t blocks = fp8_blocks(k), used = experts ? std::min(experts, m) : 1;
    const double bytes = double(used) * double(n) * double(k);
    double best = 0.;
    for (int i = y_dtype == EQ_DTYPE_F32 ? kWide : 0; i < int(sizeof(kShapes) / sizeof(kShapes[0])); i++) {
        const Shape& s = kShapes[i];
        // (how the routes are spread is not known here: more than half a tile more for each expert; 17 TB/s where
        // neighbouring tiles share weights and activations, 11 with routes, measured)
        const int64_t mtiles = experts ? std::max(used, m / s.rows + used * 5 / 8) + 1 : (m + s.rows - 1) / s.rows;
        const int64_t tiles = mtiles * ((n + s.cols - 1) / s.cols);
        for (int64_t most = 1; most <= 16 && (most == 1 || blocks / most >= 4); most++) {  // (parts of four blocks or more)
            const double us = tiles_us(s, std::min(tiles, kMostTiles), blocks, most, experts ? 11e6 : 17e6, bytes, experts > 0);
            if (best > 0. && us >= best) continue;
            best = us, p.shape = i, p.parts = most;
        }
    }
    const Shape& s = kShapes[p.shape];
    p.mtiles = experts ? std::min(m, m / s.rows + experts + 1) : (m + s.rows - 1) / s.rows;
    p.ntiles = (n + s.cols - 1) / s.cols;
    p.slots = slots_of(s);
    if (p.parts > 1) {
        // (a pass's parts are as many as its slots or fewer)
        const int64_t tiles = std::min(p.mtiles * p.ntiles, kMostTiles);
        const Passes r{int(tiles), int(p.slots), int(p.parts)};
        const int64_t units = experts ? std::min(p.slots, tiles * p.parts) : r.rest * r.parts;
        p.part = round256(size_t(units) * size_t(s.cols * s.rows) * 4u);
    }
}

bool sizes_ok(const char* who, int64_t rows, int64_t n, int64_t k) {
    if (!fp8_cols_ok(who, "k", k)) return false;
    if (rows < 0 || n < 0 || rows >= (int64_t(1) << 30) || n >= (int64_t(1) << 30)) {
        set_error(std::string(who) + ": rows and n must be in [0, 2^30)");
        return false;
    }
    if (rows * fp8_blocks(k) >= kFp8MaxGroups) {
        set_error(std::string(who) + ": rows * ceil(k / 128) must be below 2^26");
        return false;
    }
    return true;
}

bool dtypes_ok(const char* who, int x_dtype, int y_dtype) {
    if (x_dtype != EQ_DTYPE_F8E4M3 && !valid_dtype(x_dtype)) {
        set_error(std::string(who) + ": x must be e4m3 codes, f32, f16 or bf16");
        return false;
    }
    if (!valid_dtype(y_dtype)) {
        set_error(std::string(who) + ": y must be f32, f16 or bf16");
        return false;
    }
    return true;
}

bool grid_ok(const char* who, const Plan& p) {
    if (p.mtiles * p.ntiles <= kMostTiles) return true;
    set_error(std::string(who) + ": more than 2^23 - 4096 tiles of the result");
    return false;
}

bool plan_product(const char* who, Plan& p, int64_t m, int64_t n, int64_t k, int x_dtype, int y_dtype) {
    if (!sizes_ok(who, m, n, k) || !dtypes_ok(who, x_dtype, y_dtype)) return false;
    // (what the kernel of few rows has operands for; 16 and 17 rows of codes by 4096 x 4096 6.9 and 14.9 us in graphs, by
    // 14336 x 4096 12.5 and 14.8: a tile of 128 x 32 to a workgroup leaves most of the GPU idle where n is small)
    p.few = m <= 16;
    if (p.few) p.mtiles = 1, p.ntiles = (n + 15) / 16;
    else choose_tiles(p, m, n, k, 0, y_dtype);
    if (x_dtype != EQ_DTYPE_F8E4M3 && !(p.few && fp8_few_takes(m, k, x_dtype))) {
        p.codes = round256(size_t(m) * size_t(k));
        p.scales = round256(size_t(m) * size_t(fp8_blocks(k)) * 4u);
    }
    return grid_ok(who, p);
}

// (offsets into the rows of x are 32 bits, kOutOfRange is none of them)
bool x_fits(const char* who, int64_t x_rows, int64_t stride) {
    if (x_rows * stride < int64_t(kOutOfRange)) return true;
    set_error(std::string(who) + ": the codes of x must be fewer than 3 * 2^30 bytes");
    return false;
}

bool plan_routes(const char* who, Plan& p, int64_t x_rows, int64_t experts, int64_t routes, int64_t n, int64_t k,
                 int x_dtype, int y_dtype) {
    if (!sizes_ok(who, routes, n, k) || !sizes_ok(who, x_rows, n, k) || !dtypes_ok(who, x_dtype, y_dtype)) return false;
    if (experts < 1 || experts > kMostExperts) {
        set_error(std::string(who) + ": experts must be in [1, " + std::to_string(kMostExperts) + "]");
        return false;
    }
    if (routes > 0 && n > 0) {
        if (x_rows < 1) {
            set_error(std::string(who) + ": x must have a row");
            return false;
        }
        if (!x_fits(who, x_rows, k)) return false;
    }
    // (a route to a workgroup costs no count of routes: 64 of them to some 35 of 128 experts of 768 x 2048 15.3 us; it reads an
    // expert's weight for each of its routes, though: 64 to 8 experts of 14336 x 4096 526 us, 66, in tiles, 103)
    p.few = routes <= 64;
    const bool plain = x_dtype == EQ_DTYPE_F8E4M3 || (p.few && fp8_few_takes(1, k, x_dtype));
    if (!plain) {
        p.codes = round256(size_t(x_rows) * size_t(k));
        p.scales = round256(size_t(x_rows) * size_t(fp8_blocks(k)) * 4u);
    }
    if (p.few) {
        p.mtiles = routes, p.ntiles = (n + 15) / 16;
        return grid_ok(who, p);
    }
    // (p.mtiles: a part tile for each expert that has one, and for the routes without)
    choose_tiles(p, routes, n, k, experts, y_dtype);
    p.tiles = round256(size_t(p.mtiles + 1) * sizeof(int4));
    p.order = round256(size_t(routes) * sizeof(int2));
    return grid_ok(who, p);
}

bool operands_ok(const char* who, const void* y, const void* x, int64_t x_stride, const float* x_scales,
                 int64_t scale_stride, const void* w, const float* w_scales, int64_t x_rows, int64_t k, int x_dtype,
                 int y_dtype) {
    const bool coded = x_dtype == EQ_DTYPE_F8E4M3;
    if (!y || !w_scales || (coded && !x_scales)) {
        set_error(std::string(who) + ": null pointer argument");
        return false;
    }
    if (!coded && x_scales) {
        set_error(std::string(who) + ": x_scales belong to codes");
        return false;
    }
    if (!aligned(y, y_dtype == EQ_DTYPE_F32 ? 4 : 2) || !aligned(w_scales, 4) || (coded && !aligned(x_scales, 4))) {
        set_error(std::string(who) + ": y and scales must be aligned to their values");
        return false;
    }
    return fp8_rows_ok(who, "x", x, x_stride, k, coded ? 1 : x_dtype == EQ_DTYPE_F32 ? 4 : 2) &&
           fp8_rows_ok(who, "w", w, k, k, 1) && (!coded || fp8_scales_ok(who, scale_stride, x_rows, k));
}

// The caller's scratch or the stream's workspace; null: the error is set.
char* scratch_of(WsHold& hold, const char* who, void* scratch, int64_t scratch_bytes, size_t need, hipStream_t st) {
    if (scratch) {
        if (scratch_bytes >= 0 && size_t(scratch_bytes) >= need && aligned(scratch, 256)) return static_cast<char*>(scratch);
        set_error(std::string(who) + ": needs " + std::to_string(need) + " bytes of 256-byte aligned scratch");
        return nullptr;
    }
    char* p = static_cast<char*>(ws_acquire(hold, nullptr, need, st));
    if (!p)
        set_error(std::string(who) + ": no workspace (its stream's workspace cannot grow while capturing: pass scratch, "
                  "or make one such call on the stream before capturing)");
    return p;
}

// x of a call: as it is, or quantized into scratch first where the plan says so; what its type is then.
int take_x(Fp8Args& a, char* scratch, const Plan& p, const void* x, int64_t x_stride, const float* x_scales,
           int64_t scale_stride, int64_t rows, int64_t k, int x_dtype, hipStream_t st) {
    if (!p.codes) {
        a.x = static_cast<const uint8_t*>(x), a.xs = x_scales, a.x_stride = x_stride, a.xs_stride = scale_stride;
        return x_dtype;
    }
    float* scales = reinterpret_cast<float*>(scratch + p.codes);
    launch_fp8_quantize(scratch, scales, rows, x, x_stride, rows, k, x_dtype, st);
    a.x = reinterpret_cast<const uint8_t*>(scratch), a.xs = scales, a.x_stride = k, a.xs_stride = rows;
    return EQ_DTYPE_F8E4M3;
}

}  // namespace
}  // namespace eq

using namespace eq;

extern "C" int64_t eq_fp8_matmul_scratch(int64_t m, int64_t n, int64_t k, int x_dtype, int y_dtype) {
    clear_error();
    Plan p;
    return plan_product("eq_fp8_matmul", p, m, n, k, x_dtype, y_dtype) ? int64_t(p.bytes()) : -1;
}

extern "C" int eq_fp8_matmul(void* y, const void* x, int64_t x_stride, const float* x_scales, int64_t scale_stride,
                             const void* w, const float* w_scales, int64_t m, int64_t n, int64_t k, int x_dtype,
                             int y_dtype, void* scratch, int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_fp8_matmul";
    Plan p;
    if (!plan_product(who, p, m, n, k, x_dtype, y_dtype)) return 1;
    if (m == 0 || n == 0) return 0;
    if (!operands_ok(who, y, x, x_stride, x_scales, scale_stride, w, w_scales, m, k, x_dtype, y_dtype)) return 1;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    WsHold hold;
    char* base = nullptr;
    if (p.bytes() && !(base = scratch_of(hold, who, scratch, scratch_bytes, p.bytes(), st))) return 1;
    Fp8Args a{};
    a.y = y;
    a.w = static_cast<const uint8_t*>(w);
    a.ws = w_scales;
    a.M = int(m), a.N = int(n), a.K = int(k), a.KB = int(fp8_blocks(k));
    a.mtiles = int(p.mtiles), a.ntiles = int(p.ntiles), a.band = kBand, a.slots = int(p.slots), a.parts = int(p.parts);
    x_dtype = take_x(a, base, p, x, x_stride, x_scales, scale_stride, m, k, x_dtype, st);
    if (p.few) {
        launch_fp8_few(a, Fp8Few{x, x_dtype, nullptr, 1}, y_dtype, st);
        return check_launch(who);
    }
    a.part = reinterpret_cast<float*>(base + p.bytes() - p.part);
    with_dtype(y_dtype, [&](auto t) { launch_tiles<decltype(t)>(p.shape, a, st); });
    return check_launch(who);
}

extern "C" int64_t eq_fp8_grouped_matmul_scratch(int64_t x_rows, int64_t experts, int64_t routes, int64_t n, int64_t k,
                                                 int x_dtype, int y_dtype) {
    clear_error();
    Plan p;
    return plan_routes("eq_fp8_grouped_matmul", p, x_rows, experts, routes, n, k, x_dtype, y_dtype) ? int64_t(p.bytes()) : -1;
}

extern "C" int eq_fp8_grouped_matmul(void* y, const void* x, int64_t x_stride, const float* x_scales,
                                     int64_t scale_stride, int64_t x_rows, const void* w, const float* w_scales,
                                     int64_t experts, const int32_t* ids, const int32_t* rows, int64_t routes,
                                     int64_t n, int64_t k, int x_dtype, int y_dtype, void* scratch,
                                     int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_fp8_grouped_matmul";
    Plan p;
    if (!plan_routes(who, p, x_rows, experts, routes, n, k, x_dtype, y_dtype)) return 1;
    if (routes == 0 || n == 0) return 0;
    if (!rows && x_rows != routes) {
        set_error(std::string(who) + ": without `rows` x must have a row for each route");
        return 1;
    }
    if (!ids || !aligned(ids, 4) || !aligned(rows, 4)) {
        set_error(std::string(who) + ": ids must be given, ids and rows aligned");
        return 1;
    }
    if (!operands_ok(who, y, x, x_stride, x_scales, scale_stride, w, w_scales, x_rows, k, x_dtype, y_dtype)) return 1;
    if (x_dtype == EQ_DTYPE_F8E4M3 && !x_fits(who, x_rows, x_stride)) return 1;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    WsHold hold;
    char* base = nullptr;
    if (p.bytes() && !(base = scratch_of(hold, who, scratch, scratch_bytes, p.bytes(), st))) return 1;
    Fp8Args a{};
    a.y = y;
    a.w = static_cast<const uint8_t*>(w);
    a.ws = w_scales;
    a.M = int(routes), a.N = int(n), a.K = int(k), a.KB = int(fp8_blocks(k));
    a.mtiles = int(p.mtiles), a.ntiles = int(p.ntiles), a.band = kBand, a.slots = int(p.slots), a.parts = int(p.parts);
    a.rows = rows, a.x_rows = x_rows;
    x_dtype = take_x(a, base + p.tiles + p.order, p, x, x_stride, x_scales, scale_stride, x_rows, k, x_dtype, st);
    if (p.few) {
        launch_fp8_few(a, Fp8Few{x, x_dtype, ids, int(experts)}, y_dtype, st);
        return check_launch(who);
    }
    a.tiles = reinterpret_cast<const int4*>(base);
    a.order = reinterpret_cast<const int2*>(base + p.tiles);
    // (64 workgroups at the most, each of which counts all routes)
    const int64_t chunk = (routes + 16383) / 16384 * 256;
    fp8_routes_kernel<<<dim3(unsigned((routes + chunk - 1) / chunk)), dim3(1024), size_t(2 * (experts + 1)) * 4u, st>>>(
        reinterpret_cast<int4*>(base), reinterpret_cast<int2*>(base + p.tiles), ids, rows, int(routes), int(chunk),
        int(experts), x_rows, kShapes[p.shape].rows, a.mtiles);
    a.part = reinterpret_cast<float*>(base + p.bytes() - p.part);
    with_dtype(y_dtype, [&](auto t) { launch_tiles<decltype(t)>(p.shape, a, st); });
    return check_launch(who);
}

// Attention over the paged 8-bit key/value cache (kv_common.hpp has the
// format, include/eredu_kv.h the rules).
#include <math.h>

#include "kv_common.hpp"

namespace eq {
namespace {

// The arithmetic, per wave and 64 tokens, for 16 * NR query rows (a row is one
// token and one of the query heads that share the KV head):
//
//   S^T = K . q^T on the int8 matrix cores.  K is the codes as they lie in the cache; q
//   is, per row, an integer of 16 bits of its largest magnitude, split into two
//   signed digits q = 256 hi + lo: the products are exact in 32 bits
//   (256 * 127 * 32512 < 2^31) and the digits' sums join by a shift before the
//   second product, S = sum lo c + 256 sum hi c.  No key is converted.
//   softmax: a row's score is S * f + const with f = scale * log2 e * (row's step) *
//   (page's step), one fma and one exp2 from the integer.
//   O^T += V^T . P^T in f16.  S^T comes out of the matrix cores with a lane
//   holding one query row and 4 tokens of each of 4 products; the 16 tokens of
//   a product are chosen as {16 a + 4 t + b}, so that lane group g holds the tokens
//   16 g .. 16 g + 15, whose probabilities are, in order, its operand of P^T: no
//   exchange between lanes, no LDS.  The operand of V^T for the same tokens is 16
//   consecutive bytes of one dimension, as a page holds them.
//   A value's code becomes f16 by a byte permute and one packed fma, which also
//   brings in its page's scale, as a power of two relative to the largest one
//   met (`base`): 1 + (c + 128) / 1024 -> c * 2^(5 + b - base), exact down
//   to 2^-29 of the largest page.
//
// The running maximum moves only when a score exceeds it by 2^8 (and base when
// a page's scale exceeds it): then, rarely, maxima are exchanged between the lane groups
// and O and l rescaled.  Probabilities are held as f16 of 2^6 exp2(score - m):
// at most 2^14, down to 2^-20 with all their bits.
constexpr float kProbBias = 6.f, kMaxSlack = 8.f;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

template <int D, int NR>
struct Rows {
    static constexpr int KS = D / 64, DT = D / 16;
    i32x4 hi[NR][KS], lo[NR][KS];  // the queries' digits: row lane % 16, dimensions 64 ks + 16 g ..
    float f[NR];                   // what turns their integer scores into exponents (NaN: a query that is not finite)
    int from[NR], until[NR];       // the tokens that they see
    f32x4 o[NR][DT];               // O^T: row lane % 16, dimensions 16 dt + 4 g ..
    float m[NR], l[NR];            // l: this lane group's part
    int base;                      // scale byte that o is relative to
};

// The query row at x (null: no row) turned by rot (null: not), as digits of
// its largest magnitude; s2 = scale * log2 e.
template <typename T, int D>
__device__ __forceinline__ void kv_query(const uint16_t* x, const float* rot, float s2, i32x4* hi, i32x4* lo, float& f) {
    constexpr int KS = D / 64;
    const int g = (threadIdx.x & 63) >> 4;
    float v[KS][16];
    uint32_t most = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        const int d0 = 64 * ks + 16 * g;
        if (x) {
            kv_load8<T>(x + d0, v[ks]);
            kv_load8<T>(x + d0 + 8, v[ks] + 8);
            if (rot) {
                float p[16];
                const bool first = d0 < D / 2;
                const int pd = first ? d0 + D / 2 : d0 - D / 2;
                const float* cs = rot + (first ? d0 : pd);
                kv_load8<T>(x + pd, p);
                kv_load8<T>(x + pd + 8, p + 8);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float a = v[ks][i] * cs[i], b = p[i] * cs[D / 2 + i];
                    v[ks][i] = first ? a - b : a + b;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[ks][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) most = max(most, __float_as_uint(v[ks][i]) & 0x7fffffffu);
    }
    most = max(most, uint32_t(__shfl_xor(int(most), 16)));
    most = max(most, uint32_t(__shfl_xor(int(most), 32)));
    const bool fine = most > 0u && most < 0x7f800000u;
    const int e = fine ? __builtin_amdgcn_frexp_expf(__uint_as_float(most)) : 0;
    const float mant = fine ? __builtin_amdgcn_frexp_mantf(__uint_as_float(most)) : 1.f;
    const float inv = 32512.f / mant;
    f = fine ? __builtin_amdgcn_ldexpf(mant * (s2 / 32512.f), e) : (most ? __uint_as_float(0x7fc00000u) : 0.f);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
#pragma unroll
        for (int w = 0; w < 4; w++) {
            uint32_t h = 0, l = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int q = fine ? int(rintf(__builtin_amdgcn_ldexpf(v[ks][4 * w + i], -e) * inv)) : 0;
                const int top = (q + 128) >> 8;
                h |= uint32_t(top & 0xff) << (8 * i);
                l |= uint32_t((q - 256 * top) & 0xff) << (8 * i);
            }
            hi[ks][w] = int(h), lo[ks][w] = int(l);
        }
    }
}

// 64 tokens: k(t, ks) and v(dt) give this lane's operands, kb and vb are its
// group's scale bytes, j0 its first token; dead: its page is missing.  EDGE: some row does not
// see some of the tokens.
template <bool EDGE, int D, int NR, typename KF, typename VF>
__device__ __forceinline__ void kv_tile(Rows<D, NR>& R, KF k, VF v, int kb, int vb, int j0, bool dead) {
    constexpr int KS = D / 64, DT = D / 16;
    i32x4 s[NR][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        i32x4 a[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) a[ks] = k(t, ks);
#pragma unroll
        for (int r = 0; r < NR; r++) {
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[ks], R.hi[r][ks], acc, 0, 0, 0);
            acc = acc << 8;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[ks], R.lo[r][ks], acc, 0, 0, 0);
            s[r][t] = acc;
        }
    }
    const bool nan = kb == 255 || vb == 255;
    const float kf = nan ? __uint_as_float(0x7fc00000u) : e8m0_to_f32(uint32_t(kb));
    const int ev = nan || dead ? 0 : vb;
    float f[NR], top[NR];
    int first[NR], seen[NR];
    bool need = ev > R.base;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        f[r] = R.f[r] * kf;
        if constexpr (EDGE) {
            first[r] = dead ? 16 : max(R.from[r] - j0, 0);
            seen[r] = max(min(R.until[r] - j0, 16) - first[r], 0);
#pragma unroll
            for (int n = 0; n < 16; n++)
                if (unsigned(n - first[r]) >= unsigned(seen[r])) s[r][n >> 2][n & 3] = INT32_MIN;
        }
        int mx = s[r][0][0];
#pragma unroll
        for (int n = 1; n < 16; n++) mx = max(mx, s[r][n >> 2][n & 3]);
        top[r] = float(mx) * f[r];
        if constexpr (EDGE) top[r] = seen[r] > 0 ? top[r] : -INFINITY;
        need |= top[r] > R.m[r] + kMaxSlack;
    }
    if (__any(need)) {
        const int up = max(max(__builtin_amdgcn_readlane(ev, 0), __builtin_amdgcn_readlane(ev, 16)),
                           max(__builtin_amdgcn_readlane(ev, 32), __builtin_amdgcn_readlane(ev, 48)));
        const int base = max(R.base, up);
        const float down = __builtin_amdgcn_ldexpf(1.f, R.base - base);
        R.base = base;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float mn = fmaxf(top[r], __shfl_xor(top[r], 16));
            mn = fmaxf(R.m[r], fmaxf(mn, __shfl_xor(mn, 32)));
            const float al = mn == R.m[r] ? 1.f : __builtin_amdgcn_exp2f(R.m[r] - mn);
            R.m[r] = mn;
            R.l[r] *= al;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) R.o[r][dt] *= al * down;
        }
    }
    h16x8 p[NR][2];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const float shift = kProbBias - R.m[r];
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 16; n += 4) {
            f32x4 e;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                e[i] = __builtin_amdgcn_exp2f(fmaf(float(s[r][n >> 2][i]), f[r], shift));
                if constexpr (EDGE) e[i] = unsigned(n + i - first[r]) < unsigned(seen[r]) ? e[i] : 0.f;
                sum += e[i];
            }
            const h16x4 h = __builtin_convertvector(e, h16x4);
#pragma unroll
            for (int i = 0; i < 4; i++) p[r][n >> 3][(n & 4) + i] = h[i];
        }
        R.l[r] += sum;
    }
    // 2^(15 + ev - base) in f16, subnormal below 2^-14
    const int x = 30 + ev - R.base;
    const uint16_t bits = uint16_t(x >= 1 ? x << 10 : (x >= -9 ? 1 << (9 + x) : 0));
    const _Float16 sc = __builtin_bit_cast(_Float16, bits);
    const h16x2 sc2 = {sc, sc}, off2 = sc2 * h16x2{_Float16(-1.125f), _Float16(-1.125f)};
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        const i32x4 w = v(dt);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            h16x8 a;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t c = uint32_t(w[2 * u + i]) ^ 0x80808080u;  // code + 128
                const h16x2 x0 = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x3c3c3c3cu, c, 0x04010400u));
                const h16x2 x1 = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x3c3c3c3cu, c, 0x04030402u));
                const h16x2 y0 = __builtin_elementwise_fma(x0, sc2, off2), y1 = __builtin_elementwise_fma(x1, sc2, off2);
                a[4 * i] = y0[0], a[4 * i + 1] = y0[1], a[4 * i + 2] = y1[0], a[4 * i + 3] = y1[1];
            }
#pragma unroll
            for (int r = 0; r < NR; r++) R.o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[r][u], R.o[r][dt], 0, 0, 0);
        }
    }
}

struct AttnCall {
    uint16_t* out;
    const uint16_t* q;
    int64_t q_stride;
    KvView c;
    KvBatch b;
    const float* rope;
    float s2;      // scale * log2 e
    int heads, group, tiles, splits, window;  // window 0: none
    bool causal;
    float* part;   // [row][head][split][D], normalised; null: one split
    float* lse;    // [row][head][split]
};

// The 64-token tiles that query tokens [i0, i1] of an entry see, and their
// share of one split.
struct TileRange {
    int begin, end;
};
__device__ __forceinline__ int kv_until(const AttnCall& A, const KvEntry& e, int i) {
    const int held = min(e.length, A.c.width << A.c.log2_page);
    return A.causal ? min(e.length - e.count + i + 1, held) : held;
}
__device__ __forceinline__ int kv_from(const AttnCall& A, const KvEntry& e, int i) {
    return A.window > 0 ? max(e.length - e.count + i + 1 - A.window, 0) : 0;
}
__device__ __forceinline__ TileRange kv_tiles(const AttnCall& A, const KvEntry& e, int i0, int i1) {
    TileRange t;
    t.begin = kv_from(A, e, i0) >> 6;
    t.end = max((max(kv_until(A, e, i1), 0) + 63) >> 6, t.begin);
    return t;
}
// Tiles of a split: at least one for each of a workgroup's waves.
__device__ __forceinline__ int kv_share(const AttnCall& A, const TileRange& t) {
    return max(4, (t.end - t.begin + A.splits - 1) / A.splits);
}

// Where a launch's workgroup works: the KV head varies fastest, so that one
// head's codes stay in one XCD's L2 where there are 8 of them.
struct Place {
    int kvh, split;
    KvEntry e;
    int first;  // row of the entry's rows * group that the tile begins with
};
template <int BM>
__device__ __forceinline__ bool kv_place(const AttnCall& A, Place& P) {
    const int id = blockIdx.x, per = A.c.kv_heads * A.tiles;
    P.kvh = id % A.c.kv_heads;
    P.split = id / per;
    int entry, place;
    const int group = A.group;
    // the last tiles first: in causal prompts they have the most to do
    if (!kv_locate(A.b, A.tiles - 1 - id % per / A.c.kv_heads, [&](int n) { return (n * group + BM - 1) / BM; }, entry, place))
        return false;
    P.e = kv_entry(A.c, A.b, entry);
    P.first = place * BM;
    return true;
}

// This lane's rows of the wave's tile, first .. first + 16 NR - 1.
template <typename T, int D, int NR>
__device__ __forceinline__ void kv_begin(const AttnCall& A, const Place& P, int first, Rows<D, NR>& R) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int row = first + 16 * r + (lane & 15), i = row / A.group;
        const bool live = i < P.e.count;
        const int pos = P.e.length - P.e.count + i;
        R.from[r] = live ? kv_from(A, P.e, i) : 0;
        R.until[r] = live ? kv_until(A, P.e, i) : 0;
        const bool sees = live && R.from[r] < R.until[r];
        const uint16_t* x = A.q + int64_t(P.e.start + i) * A.q_stride + int64_t(P.kvh * A.group + row % A.group) * D;
        kv_query<T, D>(sees ? x : nullptr, sees && A.rope && pos >= 0 ? A.rope + int64_t(pos) * D : nullptr, A.s2,
                       R.hi[r], R.lo[r], R.f[r]);
        R.m[r] = -INFINITY;
        R.l[r] = 0.f;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) R.o[r][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    R.base = 0;
}

// 4 dimensions of one row: the output, or its part of one split.
template <typename T, int D>
__device__ __forceinline__ void kv_store4(const AttnCall& A, const Place& P, int row, int d, f32x4 o) {
    const int i = row / A.group, h = P.kvh * A.group + row % A.group;
    const int64_t at = int64_t(P.e.start + i) * A.heads + h;
    if (A.part) {
        *reinterpret_cast<f32x4*>(A.part + (at * A.splits + P.split) * D + d) = o;
    } else {
        uint16_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = to_storage<T>(o[j]);
        *reinterpret_cast<uint2*>(A.out + at * D + d) = make_uint2(w[0] | uint32_t(w[1]) << 16, w[2] | uint32_t(w[3]) << 16);
    }
}
__device__ __forceinline__ void kv_store_lse(const AttnCall& A, const Place& P, int row, float lse) {
    const int i = row / A.group, h = P.kvh * A.group + row % A.group;
    A.lse[(int64_t(P.e.start + i) * A.heads + h) * A.splits + P.split] = lse;
}

// --------------------------------------------------- few rows: a stream of tokens
//
// 16 rows a workgroup, whose 4 waves take the split's tiles in turn, each
// with a softmax of its own, joined at the end.  Operands go from memory to
// registers as the matrix cores take them, the next tile's under way while one is computed.

template <int D>
struct Tile {
    i32x4 k[4][D / 64], v[D / 16];
    int kb, vb;
    bool dead;
};

template <int D>
__device__ __forceinline__ void kv_fetch(const AttnCall& A, const Place& P, int tile, int ida, int idg, Tile<D>& t) {
    const int lane = threadIdx.x & 63, g = lane >> 4, a = (lane & 15) >> 2, T = 1 << A.c.log2_page;
    t.dead = idg < 0;
    const int64_t pa = int64_t(max(ida, 0)) * A.c.kv_heads + P.kvh, pg = int64_t(max(idg, 0)) * A.c.kv_heads + P.kvh;
    t.kb = A.c.ks[pg];
    t.vb = A.c.vs[pg];
    const int8_t* k = A.c.k + (pa * T + ((tile * 64 + 16 * a) & (T - 1)) + (lane & 3)) * D + 16 * g;
    const int8_t* v = A.c.v + (pg * D + (lane & 15)) * T + ((tile * 64 + 16 * g) & (T - 1));
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int ks = 0; ks < D / 64; ks++) t.k[i][ks] = *reinterpret_cast<const i32x4*>(k + 4 * i * D + 64 * ks);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) t.v[dt] = *reinterpret_cast<const i32x4*>(v + 16 * dt * T);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void kv_stream_kernel(const AttnCall A) {
    constexpr int NR = 1, BM = 16, DC = D < 128 ? D : 128;
    __shared__ float os[4][16][DC + 4];
    __shared__ float ms[4][16], ls[4][16];
    __shared__ int bs[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    Place P;
    if (!kv_place<BM>(A, P)) return;
    const int rows = min(BM, P.e.count * A.group - P.first);
    const TileRange all = kv_tiles(A, P.e, P.first / A.group, (P.first + rows - 1) / A.group);
    const int share = kv_share(A, all), begin = all.begin + P.split * share, end = min(all.end, begin + share);
    if (P.split > 0 && begin >= end) return;
    Rows<D, NR> R;
    kv_begin<T, D, NR>(A, P, P.first, R);
    // tiles [clear_from, clear_until) are seen whole by every row there is
    const int clear_from = (kv_from(A, P.e, (P.first + rows - 1) / A.group) + 63) >> 6, clear_until = max(kv_until(A, P.e, P.first / A.group), 0) >> 6;

    auto page = [&](int tile, int block) { return kv_page(A.c, P.e.seq, (tile * 64 + 16 * block) >> A.c.log2_page); };
    const int a = (lane & 15) >> 2;
    int tile = begin + wave;
    if (tile < end) {
        Tile<D> cur, nxt;
        kv_fetch<D>(A, P, tile, page(tile, a), page(tile, g), cur);
        int ida = page(tile + 4, a), idg = page(tile + 4, g);
        auto step = [&](Tile<D>& now, Tile<D>& next) __attribute__((always_inline)) {
            const bool more = tile + 4 < end;
            if (more) {
                kv_fetch<D>(A, P, tile + 4, ida, idg, next);
                ida = page(tile + 8, a), idg = page(tile + 8, g);
            }
            auto k = [&](int t, int ks) __attribute__((always_inline)) { return now.k[t][ks]; };
            auto v = [&](int dt) __attribute__((always_inline)) { return now.v[dt]; };
            if (tile >= clear_from && tile < clear_until && !__any(now.dead))
                kv_tile<false, D, NR>(R, k, v, now.kb, now.vb, tile * 64 + 16 * g, false);
            else
                kv_tile<true, D, NR>(R, k, v, now.kb, now.vb, tile * 64 + 16 * g, now.dead);
            tile += 4;
            return more;
        };
        while (step(cur, nxt) && step(nxt, cur)) {
        }
    }
    // join the four waves' states
    float l = R.l[0];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) ms[wave][lane] = R.m[0], ls[wave][lane] = l;
    if (lane == 0) bs[wave] = R.base;
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += DC) {
        if (d0) __syncthreads();
#pragma unroll
        for (int dt = 0; dt < DC / 16; dt++)
            *reinterpret_cast<f32x4*>(&os[wave][lane & 15][16 * dt + 4 * g]) = R.o[0][d0 / 16 + dt];
        __syncthreads();
        const int row = tid >> 4;
        if (row < rows) {
            float m = -INFINITY, sum = 0.f, w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) m = fmaxf(m, ms[i][row]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float up = ms[i][row] == m ? 1.f : __builtin_amdgcn_exp2f(ms[i][row] - m);
                sum += ls[i][row] * up;
                w[i] = up;
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] *= inv;
            if (A.part && d0 == 0 && (tid & 15) == 0)
                kv_store_lse(A, P, P.first + row, sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum));
            for (int d = 4 * (tid & 15); d < DC; d += 64) {
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(&os[i][row][d]);
#pragma unroll
                    for (int j = 0; j < 4; j++) o[j] += __builtin_amdgcn_ldexpf(x[j] * w[i], bs[i] - 132);
                }
                kv_store4<T, D>(A, P, P.first + row, d0 + d, o);
            }
        }
    }
}

// ------------------------------------------ many rows: blocks of rows over shared tiles
//
// 64 * NR rows a workgroup, 16 * NR for each of its 4 waves, all over the same
// tokens: a tile's 64 keys and values go from memory straight to LDS once for the
// workgroup, one tile ahead, and each wave takes its operands from there.
// 16-byte pieces of a row are swapped by an exclusive or with bits of the row, so
// that the 8 lanes of a read lie in different banks: keys (row = token 16 a + 4 t + b,
// read for all a and b at once) by b and a's low bit, values (row = dimension) by its
// next bits.
template <int D>
__device__ __forceinline__ int kv_key_swap(int token) {
    return D >= 128 ? (token & 3) | (token >> 2 & 4) : (token >> 1 & 1) | (token >> 3 & 2);
}
__device__ __forceinline__ int kv_value_swap(int d) { return d >> 1 & 3; }

typedef __attribute__((address_space(3))) char lds_char;

// A wave's share of a tile: 64 lanes' pieces land side by side, so the swap is
// in the addresses they come from.  idg: this lane group's page, idv: that of the
// lane's value pieces.
template <int D>
__device__ __forceinline__ void kv_stage(const AttnCall& A, const Place& P, int tile, int idg, int idv, lds_char* kbuf,
                                         lds_char* vbuf) {
    constexpr int KP = D / 16;  // 16-byte pieces of a key
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, T = 1 << A.c.log2_page;
#pragma unroll
    for (int j = 0; j < D / 64; j++) {
        const int p = (j * 4 + wave) * 64 + lane, token = p / KP, c = (p % KP) ^ kv_key_swap<D>(token);
        const int block = __builtin_amdgcn_readfirstlane(token >> 4);  // (a wave's 1024 / D tokens lie in one block)
        const int id = __builtin_amdgcn_readlane(idg, 16 * block);
        const int8_t* src = A.c.k + ((int64_t(max(id, 0)) * A.c.kv_heads + P.kvh) * T + ((tile * 64 + token) & (T - 1))) * D + 16 * c;
        __builtin_amdgcn_global_load_lds(
            const_cast<int8_t*>(src), (__attribute__((address_space(3))) void*)(kbuf + (j * 4 + wave) * 1024), 16, 0, 0);
    }
    const int g = (lane & 3) ^ kv_value_swap(lane >> 2);
    const int8_t* src0 = A.c.v + (int64_t(max(idv, 0)) * A.c.kv_heads + P.kvh) * D * T + ((tile * 64 + 16 * g) & (T - 1));
#pragma unroll
    for (int j = 0; j < D / 64; j++) {
        const int d = (j * 4 + wave) * 16 + (lane >> 2);
        __builtin_amdgcn_global_load_lds(
            const_cast<int8_t*>(src0 + d * T), (__attribute__((address_space(3))) void*)(vbuf + (j * 4 + wave) * 1024), 16, 0, 0);
    }
}

template <typename T, int D, int NR>
__global__ __launch_bounds__(256) void kv_block_kernel(const AttnCall A) {
    constexpr int BM = 64 * NR;
    __shared__ __attribute__((aligned(16))) char k0[64 * D], k1[64 * D], v0[64 * D], v1[64 * D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    Place P;
    if (!kv_place<BM>(A, P)) return;
    const int rows = min(BM, P.e.count * A.group - P.first);
    const TileRange all = kv_tiles(A, P.e, P.first / A.group, (P.first + rows - 1) / A.group);
    const int share = kv_share(A, all), begin = all.begin + P.split * share, end = min(all.end, begin + share);
    if (P.split > 0 && begin >= end) return;
    // this wave's rows, the tiles that any of them sees and those that all see whole
    const int first = P.first + 16 * NR * wave, mine = min(16 * NR, rows - 16 * NR * wave);
    Rows<D, NR> R;
    kv_begin<T, D, NR>(A, P, first, R);
    int see_from = 0, see_until = 0, clear_from = 0, clear_until = 0;
    if (mine > 0) {
        const int i0 = first / A.group, i1 = (first + mine - 1) / A.group;
        const TileRange t = kv_tiles(A, P.e, i0, i1);
        see_from = t.begin, see_until = t.end;
        clear_from = (kv_from(A, P.e, i1) + 63) >> 6, clear_until = max(kv_until(A, P.e, i0), 0) >> 6;
    }
    const int gv = (lane & 3) ^ kv_value_swap(lane >> 2);
    auto page = [&](int tile, int block) { return kv_page(A.c, P.e.seq, (tile * 64 + 16 * block) >> A.c.log2_page); };
    if (begin < end) {
        int idg = page(begin, g), idv = page(begin, gv);
        int kb, vb, kbn, vbn, idn = idg;
        auto scales = [&](int id, int& x, int& y) __attribute__((always_inline)) {
            const int64_t at = int64_t(max(id, 0)) * A.c.kv_heads + P.kvh;
            x = A.c.ks[at], y = A.c.vs[at];
        };
        scales(idg, kbn, vbn);
        kv_stage<D>(A, P, begin, idg, idv, (lds_char*)k0, (lds_char*)v0);
        int tile = begin;
        if (tile + 1 < end) idg = page(tile + 1, g), idv = page(tile + 1, gv);
        auto step = [&](const char* kc, const char* vc, char* kn, char* vn) __attribute__((always_inline)) {
            __syncthreads();  // this tile is there, and the other buffers are read
            const bool dead = idn < 0;
            kb = kbn, vb = vbn;
            const bool more = tile + 1 < end;
            if (more) {
                scales(idg, kbn, vbn);
                idn = idg;
                const int sg = idg, sv = idv;
                if (tile + 2 < end) idg = page(tile + 2, g), idv = page(tile + 2, gv);
                kv_stage<D>(A, P, tile + 1, sg, sv, (lds_char*)kn, (lds_char*)vn);
            }
            if (tile >= see_from && tile < see_until) {
                auto k = [&](int t, int ks) __attribute__((always_inline)) {
                    const int token = 4 * (lane & 12) + 4 * t + (lane & 3);
                    return *reinterpret_cast<const i32x4*>(kc + token * D + 16 * ((4 * ks + g) ^ kv_key_swap<D>(token)));
                };
                auto v = [&](int dt) __attribute__((always_inline)) {
                    const int d = 16 * dt + (lane & 15);
                    return *reinterpret_cast<const i32x4*>(vc + d * 64 + 16 * (g ^ kv_value_swap(d)));
                };
                if (tile >= clear_from && tile < clear_until && !__any(dead))
                    kv_tile<false, D, NR>(R, k, v, kb, vb, tile * 64 + 16 * g, false);
                else
                    kv_tile<true, D, NR>(R, k, v, kb, vb, tile * 64 + 16 * g, dead);
            }
            tile++;
            return more;
        };
        while (step(k0, v0, k1, v1) && step(k1, v1, k0, v0)) {
        }
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        float l = R.l[r];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int row = 16 * r + (lane & 15);
        if (row >= mine) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (A.part && g == 0) kv_store_lse(A, P, first + row, l == 0.f ? -INFINITY : R.m[r] + __builtin_amdgcn_logf(l));
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) {
            f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = __builtin_amdgcn_ldexpf(R.o[r][dt][j] * inv, R.base - 132);
            kv_store4<T, D>(A, P, first + row, 16 * dt + 4 * g, o);
        }
    }
}

// One wave for each row and head: its splits' parts, weighed by their sums.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttnCall A, int bm) {
    const int lane = threadIdx.x & 63, u = blockIdx.x * 4 + (threadIdx.x >> 6), h = u % A.heads;
    int entry, i;
    if (u / A.heads >= A.b.total || !kv_locate(A.b, u / A.heads, [](int n) { return n; }, entry, i)) return;
    const KvEntry e = kv_entry(A.c, A.b, entry);
    const int row = i * A.group + h % A.group, first = row / bm * bm, rows = min(bm, e.count * A.group - first);
    const TileRange t = kv_tiles(A, e, first / A.group, (first + rows - 1) / A.group);
    const int share = kv_share(A, t), parts = (t.end - t.begin + share - 1) / share;
    const int64_t at = int64_t(e.start + i) * A.heads + h;
    constexpr int V = D / 64;
    float m = -INFINITY, sum = 0.f, o[V] = {};
    for (int s0 = 0; s0 < parts; s0 += 64) {
        const float mine = s0 + lane < parts ? A.lse[at * A.splits + s0 + lane] : -INFINITY;
        float top = mine;
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
        const float mn = fmaxf(m, top), al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        float w = s0 + lane < parts ? (mine == mn ? 1.f : __builtin_amdgcn_exp2f(mine - mn)) : 0.f;
        if (mine == -INFINITY) w = 0.f;
        sum = sum * al + wave_sum(w);
#pragma unroll
        for (int j = 0; j < V; j++) o[j] *= al;
        const int n = min(64, parts - s0);
        for (int s = 0; s < n; s++) {
            const float ws = __shfl(w, s);
            const float* p = A.part + (at * A.splits + s0 + s) * D + lane * V;
#pragma unroll
            for (int j = 0; j < V; j++) o[j] = fmaf(ws, p[j], o[j]);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < V; j++) A.out[at * D + lane * V + j] = to_storage<T>(o[j] * inv);
}

bool attention_sizes_ok(const char* who, const eq_kv_cache* c, int n_heads, int64_t n, int64_t total) {
    if (n_heads <= 0 || n_heads > 65535 || n_heads % c->kv_heads != 0) {
        set_error(std::string(who) + ": n_heads must be a multiple of kv_heads, at most 65535");
        return false;
    }
    if (n < 0 || n > (1 << 20) || total < 0 || total > INT32_MAX / 2 || total * n_heads > INT32_MAX) {
        set_error(std::string(who) + ": need 0 <= n <= 2^20 sequences and 0 <= total * n_heads < 2^31");
        return false;
    }
    return true;
}

// Which kernel, how many rows a workgroup, how many splits: from the call's
// sizes alone (lengths are on the device; the table's width bounds them).
struct Plan {
    int rows;    // of a workgroup: 16 (stream), 64 or 128 (block)
    int64_t tiles;
    int splits;
    size_t part_bytes, lse_bytes;
};
Plan plan_attention(const eq_kv_cache* c, int n_heads, int64_t n, int64_t total, bool ragged) {
    Plan p;
    const int64_t group = n_heads / c->kv_heads, rows = n ? total * group / n : 0;  // of a sequence and KV head, on average
    p.rows = rows <= 48 ? 16 : (rows <= 64 || c->head_dim > 128 ? 64 : 128);
    p.tiles = ragged ? total * group / p.rows + n : n * ((total / (n ? n : 1) * group + p.rows - 1) / p.rows);
    const int64_t groups = p.tiles * c->kv_heads, cap = (c->width * c->page_tokens + 63) / 64;
    int64_t splits = groups ? (2 * device_cu_count() + groups - 1) / groups : 1;
    if (splits > (cap + 3) / 4) splits = (cap + 3) / 4;
    if (splits > 1024) splits = 1024;
    p.splits = splits < 1 ? 1 : int(splits);
    p.part_bytes = p.splits > 1 ? size_t(total) * n_heads * p.splits * c->head_dim * 4 : 0;
    p.lse_bytes = p.splits > 1 ? (size_t(total) * n_heads * p.splits * 4 + 255) & ~size_t(255) : 0;
    return p;
}

}  // namespace
}  // namespace eq

using namespace eq;

extern "C" int64_t eq_kv_attention_scratch(const eq_kv_cache* cache, int n_heads, int64_t n, int64_t total, bool ragged) {
    clear_error();
    const char* who = "eq_kv_attention_scratch";
    if (!kv_cache_ok(who, cache) || !attention_sizes_ok(who, cache, n_heads, n, total)) return -1;
    const Plan p = plan_attention(cache, n_heads, n, total, ragged);
    return int64_t(p.part_bytes + p.lse_bytes);
}

extern "C" int eq_kv_attention(void* out, const void* q, int64_t q_stride, int n_heads, const eq_kv_cache* cache,
                               int64_t layer, const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total,
                               float scale, bool causal, int64_t window, const float* rope, int64_t rope_positions,
                               int dtype, void* scratch, int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_attention";
    if (!kv_cache_ok(who, cache) || !kv_batch_ok(who, cache, layer, seqs, n, cu, total) ||
        !attention_sizes_ok(who, cache, n_heads, n, total) || !kv_rope_ok(who, cache, rope, rope_positions))
        return 1;
    if (dtype != EQ_DTYPE_BF16 && dtype != EQ_DTYPE_F16) {
        set_error("eq_kv_attention: q and out must be bfloat16 or float16");
        return 1;
    }
    if (window < 0 || (window > 0 && !causal)) {
        set_error("eq_kv_attention: window must be 0, or positive with causal");
        return 1;
    }
    if (!(scale >= 0.f) || !(scale < INFINITY)) {
        set_error("eq_kv_attention: scale must be finite and not negative");
        return 1;
    }
    if (n == 0 || total == 0) return 0;
    const int D = cache->head_dim;
    if (!out || !q || !aligned(out, 16) || !aligned(q, 16) || q_stride % 8 || q_stride < int64_t(n_heads) * D) {
        set_error("eq_kv_attention: q and out must be 16-byte aligned, q_stride a multiple of 8 and at least "
                  "n_heads * head_dim");
        return 1;
    }
    const Plan plan = plan_attention(cache, n_heads, n, total, cu != nullptr);
    const int64_t blocks = plan.tiles * cache->kv_heads * plan.splits;
    if (blocks >= (1 << 24)) {  // a grid of under 2^32 threads
        set_error("eq_kv_attention: too many rows");
        return 1;
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    AttnCall A;
    A.part = A.lse = nullptr;
    if (plan.splits > 1) {
        const size_t need = plan.part_bytes + plan.lse_bytes;
        if (scratch && (scratch_bytes < 0 || size_t(scratch_bytes) < need || !aligned(scratch, 256))) {
            set_error("eq_kv_attention: needs " + std::to_string(need) + " bytes of 256-byte aligned scratch");
            return 1;
        }
        char* ws = static_cast<char*>(scratch ? scratch : ws_acquire(nullptr, need, st));
        if (!ws) {
            set_error("eq_kv_attention: no workspace (its stream's workspace cannot grow while capturing: pass "
                      "scratch, or make one such call on the stream before capturing)");
            return 1;
        }
        A.lse = reinterpret_cast<float*>(ws);
        A.part = reinterpret_cast<float*>(ws + plan.lse_bytes);
    }
    A.out = static_cast<uint16_t*>(out);
    A.q = static_cast<const uint16_t*>(q);
    A.q_stride = q_stride;
    A.c = kv_view(cache, layer);
    A.b = kv_batch(seqs, n, cu, total);
    A.rope = rope;
    A.s2 = scale * 1.44269504088896340736f;
    A.heads = n_heads;
    A.group = n_heads / cache->kv_heads;
    A.tiles = int(plan.tiles);
    A.splits = plan.splits;
    A.window = int(window < kKvMaxLength ? window : kKvMaxLength);
    A.causal = causal;
    const dim3 grid{unsigned(blocks)}, join(unsigned((total * n_heads + 3) / 4));
    auto go = [&](auto t, auto d) {
        typedef decltype(t) T;
        constexpr int DIM = decltype(d)::value;
        if (plan.rows == 16) kv_stream_kernel<T, DIM><<<grid, dim3(256), 0, st>>>(A);
        else if (plan.rows == 64) kv_block_kernel<T, DIM, 1><<<grid, dim3(256), 0, st>>>(A);
        else if constexpr (DIM <= 128) kv_block_kernel<T, DIM, 2><<<grid, dim3(256), 0, st>>>(A);
        if (plan.splits > 1) kv_join_kernel<T, DIM><<<join, dim3(256), 0, st>>>(A, plan.rows);
    };
    auto with_d = [&](auto t) {
        if (D == 64) go(t, std::integral_constant<int, 64>{});
        else if (D == 128) go(t, std::integral_constant<int, 128>{});
        else go(t, std::integral_constant<int, 256>{});
    };
    if (dtype == EQ_DTYPE_BF16) with_d(BF16T{});
    else with_d(F16T{});
    return check_launch(who);
}

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
//   is, per row, an integer of 24 bits of its largest magnitude, split into three
//   signed digits q = 256 hi + mid + low / 256: the products are exact
//   and the digits' sums join in f32.  No key is converted.  Two digits, 16 bits, are as good as
//   three but where a row's products with a page are large (Fine): there alone the third is multiplied.
//   softmax: a row's score is S * f + const with f = scale * log2 e * (row's step) *
//   (page's step), one fma and one exp2.
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
// Probabilities are held as f16 of exp2(score + b), b = 6 less the maximum that was
// met: at most 2^14, down to 2^-20 with all their bits.  b moves only when a score would pass
// that (and base when a page's scale exceeds it): then, rarely, maxima are exchanged between the lane
// groups and O and l rescaled.
constexpr float kProbBias = 6.f, kMaxSlack = 8.f;
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: floats next to it are whole numbers

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

// Over the wave.
template <typename F>
__device__ __forceinline__ int kv_wave(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
    return f(f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             f(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// When two digits, 16 bits of a row's largest magnitude, will do.  A query is off by at most half of their unit u, a
// score with a page's codes c by 0.29 u |c| in the mean, where |c| is 25 to 35 sqrt(D) for normal values
// (73 sqrt(D) for codes spread evenly over a byte).  Where u in exponents, f * (page step), is at most 2^-15 /
// sqrt(D), a probability is so off by 2e-4 for the usual codes, as much as an output that is rounded to
// f16 (2.1e-4 in the mean, at most 4.9e-4); bf16 rounds 8 times as coarsely and gets 4 times the limit.  Normal queries and
// keys whose scores spread by 1.5 stay under half of it.  With two digits everywhere, one channel of the
// queries 30, 100 and 300 times the others (and the keys' as much smaller) made f16 outputs 1.8, 4.4 and 13 times as far
// off as rounding alone; so it is 1.4 times, as without such a channel.  Where the third digit is needed it costs as
// much again as the matrix cores take for one: 2048 queries over 32768 tokens 1.64 ms instead of 1.19, a token
// after 131071 87 us instead of 69, seven prompts 155 instead of 113.
template <typename T, int D>
struct Fine {
    static constexpr int exponent = std::is_same<T, F16T>::value ? -15 : -13;
    // the limit as frexp has it
    static constexpr int e = D == 64 ? exponent - 2 : exponent - 3;
    static constexpr float mant = D == 128 ? 0.70710678f : 0.5f;
    // The smallest scale byte of a page with which a row of factor f > 0 is over it.
    static __device__ __forceinline__ int from(float f) {
        return 127 + e - __builtin_amdgcn_frexp_expf(f) + (mant >= __builtin_amdgcn_frexp_mantf(f) ? 1 : 0);
    }
};

template <int D, int NR>
struct Rows {
    static constexpr int KS = D / 64, DT = D / 16;
    i32x4 hi[NR][KS], mid[NR][KS];  // the queries' digits: row lane % 16, dimensions 64 ks + 16 g ..
    int fine;                      // key scale bytes from here on take the third digit too (the same for the wave)
    float f[NR];                   // what turns their integer scores into exponents (NaN: a query that is not finite)
    int from[NR], until[NR];       // the tokens that they see
    f32x4 o[NR][DT];               // O^T: row lane % 16, dimensions 16 dt + 4 g ..
    float b[NR], l[NR];            // b: inf before the first token; l: this lane group's part
    int base;                      // scale byte that o is relative to
};

// A query row's values and angles as this lane has them on the way: dimensions
// 64 ks + 16 g .. of the row, and the angles of the pairs that they are in (the other
// of a pair is the lane's own 64-group ks + D / 128, or lane group g + 2's where D = 64).
template <int D>
struct RawQuery {
    static constexpr int KS = D / 64, AS = D >= 128 ? D / 128 : 1;
    uint4 x[KS][2];
    float4 cs[AS][4], sn[AS][4];
};
template <int D>
__device__ __forceinline__ void kv_query_load(const uint16_t* x, const float* rot, RawQuery<D>& q) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int ks = 0; ks < D / 64; ks++) {
        const uint4* p = reinterpret_cast<const uint4*>(x + 64 * ks + 16 * g);
        q.x[ks][0] = p[0], q.x[ks][1] = p[1];
    }
    if (!rot) return;
#pragma unroll
    for (int i = 0; i < RawQuery<D>::AS; i++) {
        const float4* p = reinterpret_cast<const float4*>(rot + (D >= 128 ? 64 * i + 16 * g : 16 * (g & 1)));
#pragma unroll
        for (int j = 0; j < 4; j++) q.cs[i][j] = p[j], q.sn[i][j] = p[D / 8 + j];
    }
}

// Four values of a row as three signed digits of whole numbers, inv times the values: the lower bytes of q + 128 +
// 256 * 128 are their digits plus 128, the third the highest digit.
__device__ __forceinline__ void kv_digits(const float* v, float inv, int& hi, int& mid, int& low) {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = uint32_t(int(rintf(v[i] * inv))) + 0x8080u;
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05040100u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05040100u);
    hi = int(__builtin_amdgcn_perm(__builtin_amdgcn_perm(x[3], x[2], 0x0c0c0602u), __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u), 0x05040100u));
    mid = int(__builtin_amdgcn_perm(b, a, 0x07050301u) ^ 0x80808080u);
    low = int(__builtin_amdgcn_perm(b, a, 0x06040200u) ^ 0x80808080u);
}

// The row turned (where it has angles), as multiples of its largest magnitude / (256 * 32512); f: what a product of
// the middle digit's unit with a page's codes is worth in exponents, before the page's scale (s2 = scale *
// log2 e; NaN where the row is not finite, and its digits are any).  sees: whether there is a row that sees
// anything.  keep(ks, digits) gets the lowest ones.
template <typename T, int D, typename KF>
__device__ __forceinline__ void kv_query(const RawQuery<D>& q, bool sees, bool turn, float s2, i32x4* hi, i32x4* mid, float& f, KF keep) {
    constexpr int KS = D / 64;
    float v[KS][16];
    uint32_t most = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t w[4] = {q.x[ks][i].x, q.x[ks][i].y, q.x[ks][i].z, q.x[ks][i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[ks][8 * i + 2 * j] = kv_to_f32<T>(w[j] & 0xffffu);
                v[ks][8 * i + 2 * j + 1] = kv_to_f32<T>(w[j] >> 16);
            }
        }
    if (turn) {  // (the same for the whole wave)
        if constexpr (D >= 128) {
#pragma unroll
            for (int i = 0; i < KS / 2; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float cs = (&q.cs[i][j >> 2].x)[j & 3], sn = (&q.sn[i][j >> 2].x)[j & 3];
                    const float a = v[i][j], b = v[i + KS / 2][j];
                    v[i][j] = a * cs - b * sn;
                    v[i + KS / 2][j] = b * cs + a * sn;
                }
        } else {
            const bool first = (threadIdx.x & 63) < 32;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float cs = (&q.cs[0][j >> 2].x)[j & 3], sn = (&q.sn[0][j >> 2].x)[j & 3];
                const float a = v[0][j], b = __shfl_xor(a, 32), x = a * cs, y = b * sn;
                v[0][j] = first ? x - y : x + y;
            }
        }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int i = 0; i < 16; i++) most = max(most, __float_as_uint(v[ks][i]) & 0x7fffffffu);
    most = max(most, uint32_t(__shfl_xor(int(most), 16)));
    most = max(most, uint32_t(__shfl_xor(int(most), 32)));
    if (!sees) most = 0u;  // (a row that sees nothing is zero)
    const bool fine = most > 0u && most < 0x7f800000u;
    float top = __uint_as_float(most), down = 1.f;
    if (__any(fine && top < 0x1p-100f)) {  // (256 * 32512 / top may be no f32)
        const float up = fine && top < 0x1p-100f ? 0x1p64f : 1.f;
        down = 1.f / up, top *= up;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int i = 0; i < 16; i++) v[ks][i] *= up;
    }
    const float inv = fine ? 256.f * 32512.f / top : 0.f;
    f = fine ? top * (s2 / 32512.f) * down : (most ? __uint_as_float(0x7fc00000u) : 0.f);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        i32x4 low;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            int h, m, l;
            kv_digits(v[ks] + 4 * w, inv, h, m, l);
            hi[ks][w] = h, mid[ks][w] = m, low[w] = l;
        }
        keep(ks, low);
    }
}

// The lane, made anew where it is asked for (an address that is seldom used would else keep a register).
__device__ __forceinline__ int kv_lane() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(l));
    return l;
}

// The scores of 64 tokens: s[r][t][i] is row r's with token 4 t + i
// of this lane group's 16, plus kMagic; k(t, ks) gives the operands.  The products of a digit
// stay below 2^22 (256 * 127 * 128), so sums that begin with the bits of 1.5 * 2^23
// are that float plus the sum, and no score is converted (v_cvt_f32_i32 takes as long as two
// or three fmas: 83 ns for 16 in a loop, where 16 fmas take 39).
template <int D, int NR, typename KF>
__device__ __forceinline__ void kv_scores(const Rows<D, NR>& R, KF k, f32x4 (&s)[NR][4]) {
    constexpr int KS = D / 64;
    constexpr int M = 0x4b400000;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        i32x4 a[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) a[ks] = k(t, ks);
#pragma unroll
        for (int r = 0; r < NR; r++) {
            i32x4 hi = {M, M, M, M}, mid = {M, M, M, M};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[ks], R.hi[r][ks], hi, 0, 0, 0);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[ks], R.mid[r][ks], mid, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) s[r][t][i] = fmaf(__int_as_float(hi[i]) - kMagic, 256.f, __int_as_float(mid[i]));
        }
    }
}

// The same scores with the third digit, as exponents by kf, this lane group's page step: rounded once, so that
// scores of any size stay below their maximum.  (A sum next to kMagic is a whole number, one far from it
// rounded as f32 rounds it: neither loses what is added here.)
template <int D, int NR, typename KF, typename LF>
__device__ __forceinline__ void kv_scores_fine(const Rows<D, NR>& R, KF k, float kf, LF low, f32x4 (&s)[NR][4]) {
    constexpr int M = 0x4b400000;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        i32x4 l[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) l[r] = i32x4{M, M, M, M};
#pragma unroll
        for (int ks = 0; ks < D / 64; ks++) {
            const i32x4 a = k(t, ks);
#pragma unroll
            for (int r = 0; r < NR; r++) l[r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, low(r, ks), l[r], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[r][t][i] = fmaf(__int_as_float(l[r][i]) - kMagic, 1.f / 256, s[r][t][i] - kMagic) * (R.f[r] * kf);
        __builtin_amdgcn_sched_barrier(0);  // (seldom done: no registers for more than one product at a time)
    }
}

template <int NR>
__device__ __forceinline__ void kv_tops(const f32x4 (&s)[NR][4], float (&top)[NR]) {
#pragma unroll
    for (int r = 0; r < NR; r++) {
        top[r] = s[r][0][0];
#pragma unroll
        for (int n = 1; n < 16; n++) top[r] = fmaxf(top[r], s[r][n >> 2][n & 3]);
    }
}

// The softmax of those scores: the probabilities p, their sums, and the
// states so far brought to the tile's maximum (if that moves) and base.  kf is
// this lane group's page step (NaN: the key's scale byte or the value's is 255), j0 its first
// token; dead: its page is missing; base: the largest value scale byte so far,
// this tile's included.  fine (the same for the wave): the tile takes the third digit, k(t, ks) and low(r, ks) give
// its operands.  (It shares the masks' branch: with one more on the way from the products to the exponents cross
// attention took 37.6 us instead of 31.4.)  edge (the same for the wave): some row does not see some of the
// tokens; these are left out of the maximum, and their exponents are -inf.
template <int D, int NR, typename KF, typename LF>
__device__ __forceinline__ void kv_softmax(Rows<D, NR>& R, f32x4 (&s)[NR][4], bool fine, KF k, LF low, float kf, int j0, bool dead,
                                           bool edge, int base, h16x8 (&p)[NR][2]) {
    constexpr int DT = D / 16;
    float f[NR], top[NR], shift[NR];
    int first[NR], seen[NR];
    bool need = base > R.base;
    float zero = kMagic;  // what stands for 0 in the scores
#pragma unroll
    for (int r = 0; r < NR; r++) first[r] = 0, seen[r] = 16, f[r] = R.f[r] * kf;
    if (edge | fine) {
        if (fine) {
            kv_scores_fine<D, NR>(R, k, kf, low, s);
            zero = 0.f;
#pragma unroll
            for (int r = 0; r < NR; r++) f[r] = 1.f;
        }
        if (edge) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                first[r] = dead ? 16 : max(R.from[r] - j0, 0);
                seen[r] = max(min(R.until[r] - j0, 16) - first[r], 0);
#pragma unroll
                for (int n = 0; n < 16; n++)
                    if (unsigned(n - first[r]) >= unsigned(seen[r])) s[r][n >> 2][n & 3] = -INFINITY;
            }
        }
    }
    kv_tops<NR>(s, top);
#pragma unroll
    for (int r = 0; r < NR; r++) {
        shift[r] = fmaf(-zero, f[r], R.b[r]);
        need |= seen[r] > 0 && fmaf(top[r], f[r], shift[r]) > kProbBias + kMaxSlack;
    }
    if (__any(need)) {
        const float down = __builtin_amdgcn_ldexpf(1.f, R.base - base);
        R.base = base;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float mn = seen[r] > 0 ? (top[r] - zero) * f[r] : -INFINITY;
            mn = fmaxf(mn, __shfl_xor(mn, 16));
            mn = fmaxf(mn, __shfl_xor(mn, 32));
            const float b = fminf(R.b[r], kProbBias - mn), al = b == R.b[r] ? 1.f : __builtin_amdgcn_exp2f(b - R.b[r]);
            R.b[r] = b;
            shift[r] = fmaf(-zero, f[r], b);
            R.l[r] *= al;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) R.o[r][dt] *= al * down;
        }
    }
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int n = 0; n < 16; n++) s[r][n >> 2][n & 3] = fmaf(s[r][n >> 2][n & 3], f[r], shift[r]);
    if (edge) {
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int n = 0; n < 16; n++)
                if (unsigned(n - first[r]) >= unsigned(seen[r])) s[r][n >> 2][n & 3] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[r][t][i] = __builtin_amdgcn_exp2f(s[r][t][i]);
                sum += s[r][t][i];
            }
            const h16x4 h = __builtin_convertvector(s[r][t], h16x4);
#pragma unroll
            for (int i = 0; i < 4; i++) p[r][t >> 1][(t & 1) * 4 + i] = h[i];
        }
        R.l[r] += sum;
    }
}

// What a page's codes become f16 by: 1 + (c + 128) / 1024 times `mul`, plus `add`,
// is c * 2^(5 + vb - base); subnormal below 2^-29 of base, and 0 at last.
struct Convert {
    h16x2 mul, add;
    __device__ __forceinline__ Convert(int vb, int base) {
        const int ex = 30 + vb - base;
        const uint16_t bits = uint16_t(ex >= 1 ? ex << 10 : (ex >= -9 ? 1 << (9 + ex) : 0));
        const _Float16 m = __builtin_bit_cast(_Float16, bits);
        mul = h16x2{m, m};
        add = mul * h16x2{_Float16(-1.125f), _Float16(-1.125f)};
    }
    // 8 codes
    __device__ __forceinline__ h16x8 operator()(uint32_t w0, uint32_t w1) const {
        h16x8 a;
        const uint32_t w[2] = {w0 ^ 0x80808080u, w1 ^ 0x80808080u};  // code + 128
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const h16x2 x0 = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x3c3c3c3cu, w[i], 0x04010400u));
            const h16x2 x1 = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x3c3c3c3cu, w[i], 0x04030402u));
            const h16x2 y0 = __builtin_elementwise_fma(x0, mul, add), y1 = __builtin_elementwise_fma(x1, mul, add);
            a[4 * i] = y0[0], a[4 * i + 1] = y0[1], a[4 * i + 2] = y1[0], a[4 * i + 3] = y1[1];
        }
        return a;
    }
};

// v(dt, u): this lane's 8 values of dimension 16 dt + lane % 16, tokens 8 u .. of its group's 16.
template <int D, int NR, typename VF>
__device__ __forceinline__ void kv_values(Rows<D, NR>& R, const h16x8 (&p)[NR][2], VF v) {
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const h16x8 a = v(dt, u);
#pragma unroll
            for (int r = 0; r < NR; r++) R.o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[r][u], R.o[r][dt], 0, 0, 0);
        }
    }
}

// The largest of four lane groups' values, in a scalar register.
__device__ __forceinline__ int kv_group_max(int v) {
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

struct AttnCall {
    uint16_t* out;
    const uint16_t* q;
    int64_t q_stride;
    KvView c;
    KvBatch b;
    const float* rope;
    float s2;      // scale * log2 e
    int heads, rows, tiles, splits, window;  // rows: of a workgroup; window 0: none
    unsigned group;
    bool causal;
    int groups;    // kv_stream_kernel's workgroups
    int slot_rows;  // rows of its slots: as many as a unit may have
    float* part;   // kv_block_kernel: [row][head][split][D], normalised; null: one split.  kv_stream_kernel: [slot][row][D]
    float* lse;    // [row][head][split], or [slot][row]
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
// Tiles of a split of a block's, at least 4.
__device__ __forceinline__ int kv_share(const AttnCall& A, const TileRange& t) {
    return max(4, (t.end - t.begin + A.splits - 1) / A.splits);
}
// Whether a block's first split does all of it and writes it out.  2 or 3 splits
// are those of many rows, whose parts cost more than up to 16 tiles take longer in one: 4 prompts of 512
// tokens, 16 heads of 64 dimensions, take 27 us so, 35 with all blocks split.  (Without a mask all blocks of a
// sequence see the same, and looking costs the join 2 us.)
__device__ __forceinline__ bool kv_whole(const AttnCall& A, const TileRange& t) {
    return A.splits == 1 || (A.causal && t.end - t.begin <= (A.splits <= 3 ? 16 : 4));
}

// Where a launch's workgroup works: the KV head varies fastest, so that one
// head's codes stay in one XCD's L2 where there are 8 of them.
struct Place {
    int kvh, split;  // split: of kv_block_kernel
    KvEntry e;
    int first;  // row of the entry's rows * group that the tile begins with
};

// Of causal batches the blocks that see most come first, whichever sequence they
// are of (16 prompts of 256 tokens 45.9 us in the sequences' order, 43.5 so; seven of 213 to 2299 tokens
// 128 and 124): the last block to begin is a short one.  A lane has an entry, whose blocks are
// the levels [off, off + blocks) of BM rows from its first token on; unit u is the one with u
// before it when the levels are gone through from the last.
template <int BM>
__device__ __forceinline__ bool kv_place_by_level(const AttnCall& A, int u, Place& P) {
    const int lane = threadIdx.x & 63;
    KvEntry mine{-1, 0, 0, 0};
    if (lane < A.b.n) mine = kv_entry(A.c, A.b, lane);
    const int blocks = (mine.count * int(A.group) + BM - 1) / BM;
    const int off = int(min(int64_t(max(mine.length - mine.count, 0)) * A.group / BM, int64_t(1) << 29)), end = off + blocks;
    const auto sum = [](int a, int b) { return a + b; };
    if (u >= kv_wave(blocks, sum)) return false;
    int lo = 0, hi = kv_wave(end, [](int a, int b) { return max(a, b); }), before = 0;
    while (hi - lo > 1) {  // at level lo or behind it there are more than u blocks, at hi or behind it `before`, not more
        const int mid = (lo + hi) >> 1, n = kv_wave(min(max(end - mid, 0), blocks), sum);
        if (n > u) lo = mid;
        else hi = mid, before = n;
    }
    const bool at = lo >= off && lo < end;
    const uint64_t all = __ballot(at);
    const int rank = __popcll(all & ((uint64_t(1) << lane) - 1));
    const int l = __ffsll((unsigned long long)__ballot(at && rank == u - before)) - 1;
    P.e = KvEntry{__builtin_amdgcn_readlane(mine.seq, l), __builtin_amdgcn_readlane(mine.start, l),
                  __builtin_amdgcn_readlane(mine.count, l), __builtin_amdgcn_readlane(mine.length, l)};
    P.first = (lo - __builtin_amdgcn_readlane(off, l)) * BM;
    return true;
}

template <int BM>
__device__ __forceinline__ bool kv_place(const AttnCall& A, Place& P) {
    const int id = blockIdx.x, per = A.c.kv_heads * A.tiles, u = id % per / A.c.kv_heads;
    P.kvh = id % A.c.kv_heads;
    P.split = id / per;
    if (A.causal && A.b.n > 1 && A.b.n <= 64) return kv_place_by_level<BM>(A, u, P);
    int entry, place;
    const int group = A.group;
    // (the last blocks first: of one causal prompt they have the most to do)
    if (!kv_locate(A.b, A.tiles - 1 - u, [&](int n) { return (n * group + BM - 1) / BM; }, entry, place)) return false;
    const KvEntry e = kv_entry(A.c, A.b, entry);
    P.e = KvEntry{__builtin_amdgcn_readfirstlane(e.seq), __builtin_amdgcn_readfirstlane(e.start),
                  __builtin_amdgcn_readfirstlane(e.count), __builtin_amdgcn_readfirstlane(e.length)};
    P.first = place * BM;
    return true;
}

// This lane's rows of the wave's tile, first .. first + 16 NR - 1: what they
// see and the loads of their queries (of the entry's first row where there is none, in bounds
// and not used), then the rest.
template <int D, int NR>
struct RowLoads {
    RawQuery<D> q[NR];
    bool sees[NR];
};
template <int D, int NR>
__device__ __forceinline__ void kv_begin_loads(const AttnCall& A, const Place& P, int first, Rows<D, NR>& R, RowLoads<D, NR>& W) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const unsigned row = first + 16 * r + (lane & 15);
        const int i = row / A.group, ii = i < P.e.count ? i : 0;
        const int pos = P.e.length - P.e.count + ii;
        R.from[r] = i < P.e.count ? kv_from(A, P.e, i) : 0;
        R.until[r] = i < P.e.count ? kv_until(A, P.e, i) : 0;
        W.sees[r] = R.from[r] < R.until[r];
        const uint16_t* x = A.q + int64_t(P.e.start + ii) * A.q_stride + int64_t(P.kvh * A.group + (row - i * A.group)) * D;
        // (a position that has pages is inside the table of angles; any other is not used)
        kv_query_load<D>(x, A.rope ? A.rope + int64_t(kv_clamp(pos, 0, (A.c.width << A.c.log2_page) - 1)) * D : nullptr, W.q[r]);
    }
}
template <int D, int NR>
__device__ __forceinline__ void kv_nothing(Rows<D, NR>& R) {  // no tokens yet
#pragma unroll
    for (int r = 0; r < NR; r++) {
        R.b[r] = INFINITY;
        R.l[r] = 0.f;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) R.o[r][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    R.base = 0;
}
// (keep(r, ks, digits) gets the rows' lowest digits)
template <typename T, int D, int NR, typename KF>
__device__ __forceinline__ void kv_begin(const AttnCall& A, Rows<D, NR>& R, const RowLoads<D, NR>& W, KF keep) {
    int fine = 256;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        kv_query<T, D>(W.q[r], W.sees[r], A.rope != nullptr, A.s2, R.hi[r], R.mid[r], R.f[r],
                       [&](int ks, const i32x4& low) __attribute__((always_inline)) { keep(r, ks, low); });
        if (R.f[r] > 0.f) fine = min(fine, Fine<T, D>::from(R.f[r]));
    }
    R.fine = kv_wave(fine, [](int a, int b) { return min(a, b); });
    kv_nothing<D, NR>(R);
}

// A row's output, and 4 dimensions of it, or of its part of one split.
template <int D>
__device__ __forceinline__ uint16_t* kv_out(const AttnCall& A, const Place& P, int row) {
    const int i = unsigned(row) / A.group, h = P.kvh * A.group + unsigned(row) % A.group;
    return A.out + (int64_t(P.e.start + i) * A.heads + h) * D;
}
template <typename T>
__device__ __forceinline__ uint2 kv_pack4(f32x4 o) {
    uint16_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = to_storage<T>(o[j]);
    return make_uint2(w[0] | uint32_t(w[1]) << 16, w[2] | uint32_t(w[3]) << 16);
}
template <typename T, int D>
__device__ __forceinline__ void kv_store4(const AttnCall& A, const Place& P, int row, int d, f32x4 o) {
    *reinterpret_cast<uint2*>(kv_out<D>(A, P, row) + d) = kv_pack4<T>(o);
}
template <int D>
__device__ __forceinline__ void kv_store_part4(const AttnCall& A, const Place& P, int row, int d, f32x4 o) {
    const int i = unsigned(row) / A.group, h = P.kvh * A.group + unsigned(row) % A.group;
    const int64_t at = int64_t(P.e.start + i) * A.heads + h;
    *reinterpret_cast<f32x4*>(A.part + (at * A.splits + P.split) * D + d) = o;
}
__device__ __forceinline__ void kv_store_lse(const AttnCall& A, const Place& P, int row, float lse) {
    const int i = unsigned(row) / A.group, h = P.kvh * A.group + unsigned(row) % A.group;
    A.lse[(int64_t(P.e.start + i) * A.heads + h) * A.splits + P.split] = lse;
}

// --------------------------------------------------- few rows: a stream of tokens
//
// 16 rows at a time, each wave by itself.  Operands go from memory to registers as
// the matrix cores take them.
//
// The work is the list of all tiles: of all entries, their blocks of 16 rows,
// KV heads and 64-token tiles, in that order.  Each of the launch's waves takes
// an equal run of it, whatever the sequences' lengths, and works off the units
// (a block of rows and a KV head) in it one by one.  A unit that lies in one run
// is written out; of the others a run has its first and its last, at most, and
// these go to two slots of the wave, to be joined by kv_stream_join_kernel.
// Memory bounds it where contexts are long (one row over 131071 tokens, 8 KV heads of 128
// dimensions: 268 MB in 54 us with pages of 64, 5.0 TB/s, 63 us with pages of 128, whose tiles are
// not contiguous; 48 sequences of 17 .. 8191: 121 MB in 31.7 us), the trips to
// lengths, table, scales and first tile, about 5 us, where they are short (1025 tokens: 8.0 us).

constexpr int kStreamRows = 16;

// An entry's tiles: [begin, end) are those that any of its rows sees, `tiles`
// their number, at least 1 (rows that see nothing are written too), and `all`
// that of all its units together.  (A plan bounds their sum below 2^31.)
struct Units {
    int begin, end, tiles, all;
};
__device__ __forceinline__ Units kv_units(const AttnCall& A, const KvEntry& e) {
    Units u = {0, 0, 0, 0};
    if (e.count > 0) {
        const TileRange t = kv_tiles(A, e, 0, e.count - 1);
        u.begin = t.begin, u.end = t.end;
        u.tiles = max(t.end - t.begin, 1);
        u.all = (e.count * A.group + kStreamRows - 1) / kStreamRows * A.c.kv_heads * u.tiles;
    }
    return u;
}

// The list of tiles, as a wave knows it.  Up to 64 entries: a lane has one and
// the tiles before it, and the rest is exchanges between lanes.  More: thread t
// goes through the entries t * per .. (t + 1) * per - 1 and LDS has what the
// other waves need, up to 256 entries themselves.
struct TileListLds {
    KvEntry entries[256];
    int sums[4], found[4], found_entry[4];
};
struct TileList {
    TileListLds& lds;
    KvEntry mine;
    int before, own, all;  // tiles before this lane's (thread's) entries, of them, and of all

    __device__ __forceinline__ TileList(const AttnCall& A, TileListLds& L) : lds(L) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        mine = KvEntry{-1, 0, 0, 0};
        own = 0;
        if (A.b.n <= 64) {
            if (lane < A.b.n) {
                mine = kv_entry(A.c, A.b, lane);
                own = kv_units(A, mine).all;
            }
        } else {
            const int per = (A.b.n + 255) / 256;
            for (int i = threadIdx.x * per; i < min(A.b.n, int(threadIdx.x + 1) * per); i++) {
                const KvEntry e = kv_entry(A.c, A.b, i);
                if (per == 1) L.entries[i] = e;
                own += kv_units(A, e).all;
            }
        }
        int upto = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(upto, o);
            if (lane >= o) upto += t;
        }
        before = upto - own;
        all = __builtin_amdgcn_readlane(upto, 63);
        if (A.b.n <= 64) return;
        if (lane == 63) L.sums[wave] = upto;
        if (threadIdx.x < 4) L.found[threadIdx.x] = L.found_entry[threadIdx.x] = 0;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            if (w < wave) before += L.sums[w];
            all += L.sums[w];
        }
    }
    // entry i, the same for all lanes of the wave
    __device__ __forceinline__ KvEntry entry(const AttnCall& A, int i) const {
        if (A.b.n <= 64)
            return KvEntry{__builtin_amdgcn_readlane(mine.seq, i), __builtin_amdgcn_readlane(mine.start, i),
                           __builtin_amdgcn_readlane(mine.count, i), __builtin_amdgcn_readlane(mine.length, i)};
        const KvEntry e = A.b.n <= 256 ? lds.entries[i] : kv_entry(A.c, A.b, i);
        return KvEntry{__builtin_amdgcn_readfirstlane(e.seq), __builtin_amdgcn_readfirstlane(e.start),
                       __builtin_amdgcn_readfirstlane(e.count), __builtin_amdgcn_readfirstlane(e.length)};
    }
    // tiles before entry i (all threads of the workgroup call this)
    __device__ __forceinline__ int tiles_before(const AttnCall& A, int i) {
        if (A.b.n <= 64) return __builtin_amdgcn_readlane(before, i);
        const int per = (A.b.n + 255) / 256;
        if (i / per == int(threadIdx.x)) {
            int at = before;
            for (int k = threadIdx.x * per; k < i; k++) at += kv_units(A, per == 1 ? lds.entries[k] : kv_entry(A.c, A.b, k)).all;
            lds.found[0] = at;
        }
        __syncthreads();
        return __builtin_amdgcn_readfirstlane(lds.found[0]);
    }
    // the entry of tile first + wave * step, and the tiles before it (all threads of the workgroup call this)
    __device__ __forceinline__ int find(const AttnCall& A, int first, int step, int& base) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pos = first + wave * step;
        if (A.b.n <= 64) {
            const uint64_t at = __ballot(before <= pos && pos < before + own);
            const int i = at ? __ffsll((unsigned long long)at) - 1 : 0;
            base = __builtin_amdgcn_readlane(before, i);
            return i;
        }
        const int per = (A.b.n + 255) / 256;
        int at = before;
        for (int i = threadIdx.x * per; i < min(A.b.n, int(threadIdx.x + 1) * per); i++) {
            const int n = per == 1 ? own : kv_units(A, kv_entry(A.c, A.b, i)).all;
#pragma unroll
            for (int w = 0; w < 4; w++)
                if (at <= first + w * step && first + w * step < at + n) lds.found[w] = at, lds.found_entry[w] = i;
            at += n;
        }
        __syncthreads();
        base = __builtin_amdgcn_readfirstlane(lds.found[wave]);
        return __builtin_amdgcn_readfirstlane(lds.found_entry[wave]);
    }
};
__device__ __forceinline__ int kv_run(const AttnCall& A, int all) { return max(1, int(unsigned(all + 4 * A.groups - 1) / unsigned(4 * A.groups))); }

// (Keys and values have one set of registers each: the next tile's keys are
// requested when the scores are done, its values when the values are, so 2 or
// 3 waves fit a SIMD and cover each other's waits.)
template <int D>
struct Tile {
    i32x4 k[4][D / 64], v[D / 16];
};

template <int D>
__device__ __forceinline__ const int8_t* kv_keys(const AttnCall& A, const Place& P, int tile, int id, int lane) {
    const int g = lane >> 4, a = (lane & 15) >> 2, T = 1 << A.c.log2_page;
    return A.c.k + ((int64_t(max(id, 0)) * A.c.kv_heads + P.kvh) * T + ((tile * 64 + 16 * a) & (T - 1)) + (lane & 3)) * D + 16 * g;
}
template <int D>
__device__ __forceinline__ void kv_fetch_keys(const AttnCall& A, const Place& P, int tile, int id, Tile<D>& t) {
    const int8_t* k = kv_keys<D>(A, P, tile, id, threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int ks = 0; ks < D / 64; ks++) t.k[i][ks] = *reinterpret_cast<const i32x4*>(k + 4 * i * D + 64 * ks);
}
template <int D>
__device__ __forceinline__ void kv_fetch_values(const AttnCall& A, const Place& P, int tile, int id, Tile<D>& t) {
    const int lane = threadIdx.x & 63, g = lane >> 4, T = 1 << A.c.log2_page;
    const int8_t* v = A.c.v + ((int64_t(max(id, 0)) * A.c.kv_heads + P.kvh) * D + (lane & 15)) * T + ((tile * 64 + 16 * g) & (T - 1));
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++, v += 16 * T) t.v[dt] = *reinterpret_cast<const i32x4*>(v);
}

template <typename T, int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void kv_stream_kernel(const AttnCall A) {
    constexpr int NR = 1, BM = kStreamRows, KS = D / 64;
    __shared__ TileListLds lds;
    __shared__ i32x4 digits[4 * KS * 64];  // each lane's own lowest ones
    i32x4* const low = digits + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * KS * 64;
    const int lane = threadIdx.x & 63, g = lane >> 4, a = (lane & 15) >> 2;
    TileList list(A, lds);
    const int run = kv_run(A, list.all), wid = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (blockIdx.x * 4 * int64_t(run) >= list.all) return;
    int base, entry = list.find(A, blockIdx.x * 4 * run, run, base);
    const int start = int(min(int64_t(wid) * run, int64_t(list.all))), stop = min(start + run, list.all);
    if (start >= stop) return;
    int pos = start;
    Place P;
    P.split = 0;
    auto enter = [&]() __attribute__((always_inline)) {
        P.e = list.entry(A, entry);
        return kv_units(A, P.e);
    };
    Units U = enter();
    // (offsets that cover rows many times over may list more tiles than an int counts: then no entry need
    // have this one, and the first, which find gives, need not have a row)
    if (unsigned(pos - base) >= unsigned(U.all)) return;
    while (true) {
        const int local = pos - base, unit = unsigned(local) / unsigned(U.tiles), tile0 = local - unit * U.tiles;
        const int tiles = min(U.tiles - tile0, stop - pos);
        const int block = unsigned(unit) / unsigned(A.c.kv_heads);
        P.kvh = unit - block * A.c.kv_heads;
        P.first = block * BM;
        const int rows = min(BM, P.e.count * A.group - P.first), end = min(U.begin + tile0 + tiles, U.end);
        // tiles [clear_from, clear_until) are seen whole by every row there is
        const int clear_from = (kv_from(A, P.e, unsigned(P.first + rows - 1) / A.group) + 63) >> 6,
                  clear_until = max(kv_until(A, P.e, unsigned(P.first) / A.group), 0) >> 6;
        // (table entries and scale bytes are looked at a tile after they are requested, so
        // that nothing waits for them)
        const int seq = max(P.e.seq, 0);
        auto table = [&](int tile, int block) __attribute__((always_inline)) {
            return kv_page_entry(A.c, seq, (tile * 64 + 16 * block) >> A.c.log2_page);
        };
        auto scales = [&](int id, int& x, int& y) __attribute__((always_inline)) {
            const int64_t at = int64_t(max(id, 0)) * A.c.kv_heads + P.kvh;
            x = A.c.ks[at], y = A.c.vs[at];
        };
        Rows<D, NR> R;
        RowLoads<D, NR> W;
        int tile = U.begin + tile0, kb, vb;
        int ea = table(tile, a), eg = table(tile, g);
        kv_begin_loads<D, NR>(A, P, P.first, R, W);
        __builtin_amdgcn_sched_barrier(0);
        // (a unit without tiles, of rows that see nothing, reads some page and uses none of it)
        Tile<D> t;
        int idg = kv_page_of(A.c, eg), ida = kv_page_of(A.c, ea);
        kv_fetch_keys<D>(A, P, tile, ida, t);
        scales(idg, kb, vb);
        ea = table(tile + 1, a), eg = table(tile + 1, g);
        __builtin_amdgcn_sched_barrier(0);
        kv_begin<T, D, NR>(A, R, W, [&](int, int ks, const i32x4& x) __attribute__((always_inline)) {
            low[64 * ks + lane] = x;
        });  // (while the first keys are under way)
        __builtin_amdgcn_sched_barrier(0);
        kv_fetch_values<D>(A, P, tile, idg, t);
        for (; tile < end; tile++) {
            const bool more = tile + 1 < end;
            const bool fine = kv_group_max(kb) >= R.fine;
            const float kf = kb == 255 || vb == 255 ? __uint_as_float(0x7fc00000u) : e8m0_to_f32(uint32_t(kb));
            f32x4 s[NR][4];
            kv_scores<D, NR>(R, [&](int i, int ks) __attribute__((always_inline)) { return t.k[i][ks]; }, s);
            int kbn = 0, vbn = 0, idn = -1, idk = ida;
            if (more) {
                idn = kv_page_of(A.c, eg), ida = kv_page_of(A.c, ea);
                kv_fetch_keys<D>(A, P, tile + 1, ida, t);
                scales(idn, kbn, vbn);
                ea = table(tile + 2, a), eg = table(tile + 2, g);
            }
            const bool dead = idg < 0;
            const int ev = vb == 255 || dead ? 0 : vb, top = max(R.base, kv_group_max(ev));
            h16x8 p[NR][2];
            // (the third digit reads the tile's keys again: their registers have the next one's)
            kv_softmax<D, NR>(R, s, fine, [&](int i, int ks) __attribute__((always_inline)) {
                return *reinterpret_cast<const i32x4*>(kv_keys<D>(A, P, tile, idk, kv_lane()) + 4 * i * D + 64 * ks);
            }, [&](int, int ks) __attribute__((always_inline)) { return low[64 * ks + kv_lane()]; }, kf, tile * 64 + 16 * g, dead,
                              tile < clear_from || tile >= clear_until || __any(dead), top, p);
            const Convert to(ev, top);
            kv_values<D, NR>(R, p, [&](int dt, int u) __attribute__((always_inline)) {
                return to(uint32_t(t.v[dt][2 * u]), uint32_t(t.v[dt][2 * u + 1]));
            });
            if (more) kv_fetch_values<D>(A, P, tile + 1, idn, t);
            idg = idn, kb = kbn, vb = vbn;
        }
        // a unit of several runs goes to a slot
        const bool part = tiles < U.tiles;
        const int slot = 2 * wid + (pos == start ? 0 : 1), row = lane & 15;
        float l = R.l[0];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (row < rows) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (part && g == 0) A.lse[slot * A.slot_rows + row] = l == 0.f ? -INFINITY : __builtin_amdgcn_logf(l) - R.b[0];
#pragma unroll
            for (int dt = 0; dt < D / 16; dt++) {
                f32x4 o;
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = __builtin_amdgcn_ldexpf(R.o[0][dt][j] * inv, R.base - 132);
                if (part) *reinterpret_cast<f32x4*>(A.part + (int64_t(slot) * A.slot_rows + row) * D + 16 * dt + 4 * g) = o;
                else kv_store4<T, D>(A, P, P.first + row, 16 * dt + 4 * g, o);
            }
        }
        pos += tiles;
        if (pos >= stop) return;
        while (pos - base >= U.all) {  // on to the next entry that has rows
            base += U.all;
            if (++entry >= A.b.n) return;
            U = enter();
        }
    }
}

// 4 lanes' worth of one state: (m, sum, o) in every lane of a set of D / 4
// lanes, joined over the sets of W waves (state of set 0 on return; only the
// threads t < D / 4 go on).
template <int D, int W>
struct Joiner {
    static constexpr int LANES = D / 4, SETS = 64 * W / LANES;
    f32x4 os[W == 1 ? 1 : SETS][LANES];
    float ms[W], sums[W == 1 ? 1 : SETS];

    __device__ __forceinline__ bool join(int t, float m, float& sum, f32x4& o) {
        const int set = t / LANES;
        float top = m;
#pragma unroll
        for (int w = LANES; w < 64; w <<= 1) top = fmaxf(top, __shfl_xor(top, w));
        if constexpr (W > 1) {
            if ((t & 63) == 0) ms[t >> 6] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, ms[w]);
        }
        const float al = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
        sum *= al;
        o *= al;
        if constexpr (W > 1) {
            os[set][t % LANES] = o;
            if (t % LANES == 0) sums[set] = sum;
            __syncthreads();
            if (t >= LANES) return false;
            sum = sums[0];
            o = os[0][t];
#pragma unroll
            for (int s = 1; s < SETS; s++) {
                sum += sums[s];
                o += os[s][t];
            }
            return true;
        } else {
#pragma unroll
            for (int w = LANES; w < 64; w <<= 1) {
                sum += __shfl_xor(sum, w);
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] += __shfl_xor(o[i], w);
            }
            return t < LANES;
        }
    }
};

// 4 states (exponents e, -inf: nothing; parts x) into a running one.
__device__ __forceinline__ void kv_merge4(const float (&e)[4], const f32x4 (&x)[4], float& m, float& sum, f32x4& o) {
    const float mn = fmaxf(m, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])));
    const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    sum *= al;
    o *= al;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (e[j] == -INFINITY) continue;
        const float w = __builtin_amdgcn_exp2f(e[j] - mn);  // (NaN for a NaN)
        sum += w;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = fmaf(w, x[j][i], o[i]);
    }
}

template <typename T, int D>
__device__ __forceinline__ void kv_out4(const AttnCall& A, int64_t at, int t, float sum, f32x4 o) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = to_storage<T>(o[i] * inv);
    *reinterpret_cast<uint2*>(A.out + at * D + 4 * t) = make_uint2(w[0] | uint32_t(w[1]) << 16, w[2] | uint32_t(w[3]) << 16);
}

// The units that lie in several runs of kv_stream_kernel: for each row (of the rows
// that entries cover) and query head a wave, or a workgroup of 4, or of 16 (at most 64
// entries, which TileList keeps within a wave): the fewer rows, the more parts a unit has.
template <typename T, int D, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void kv_stream_join_kernel(const AttnCall A) {
    __shared__ Joiner<D, W> J;
    __shared__ TileListLds lds;
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x, u = blockIdx.x;
    const int h = W == 1 ? __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6)) : blockIdx.y;
    int entry, i;
    if (!kv_locate(A.b, u, [](int n) { return n; }, entry, i)) return;
    TileList list(A, lds);
    const int run = kv_run(A, list.all), base = list.tiles_before(A, entry);
    if (W == 1 && h >= A.heads) return;
    const KvEntry e = list.entry(A, entry);
    const Units U = kv_units(A, e);
    const int row = i * A.group + unsigned(h) % A.group;
    const int S = base + (row / kStreamRows * A.c.kv_heads + int(unsigned(h) / A.group)) * U.tiles;
    // (offsets that cover rows many times over may list more tiles than an int counts: no slot behind the last)
    const unsigned slots = 4 * A.groups;
    const int w0 = min(unsigned(S) / unsigned(run), slots - 1), w1 = min(unsigned(S + U.tiles - 1) / unsigned(run), slots - 1);
    if (w0 == w1) return;  // written out
    constexpr int LANES = D / 4, SETS = 64 * W / LANES;
    const int set = t / LANES;
    float m = -INFINITY, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int b = w0; b <= w1; b += 4 * SETS) {
        f32x4 x[4];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int w = b + j * SETS + set;
            const bool is = w <= w1;
            const int64_t slot = int64_t(2 * (is ? w : w0) + (w == w0 && S != w0 * run ? 1 : 0)) * A.slot_rows + row % kStreamRows;
            f[j] = is ? A.lse[slot] : -INFINITY;
            x[j] = is ? reinterpret_cast<const f32x4*>(A.part + slot * D)[t % LANES] : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        kv_merge4(f, x, m, sum, o);
    }
    if (J.join(t, m, sum, o)) kv_out4<T, D>(A, int64_t(e.start + i) * A.heads + h, t, sum, o);
}

// ------------------------------------------ many rows: blocks of rows over shared tiles
//
// 16 * NR * NW rows a workgroup, 16 * NR for each of its NW waves, all over the same
// tokens.  A tile's keys and values go through registers, where the values become f16
// once for the workgroup (a wave converting them for itself had 3/8 of its vector
// instructions for that), to LDS, one tile ahead, and each wave takes its operands from there.
// (Keys loaded straight to LDS took the same time, and could not be held back.)  What bounds it most is a
// SIMD's vector and matrix instructions, which hardly overlap: 2048 rows over 32768 tokens, 32 heads on 8
// of 128 dimensions, 1.18 ms, 900 TFLOP/s, the matrix cores busy 36 % of the cycles and the vector unit, but for
// their instructions' issue, 52 %; a block's life before its first tile and after its last is about 9 us.  16-byte pieces of a row are swapped by
// an exclusive or with bits of the row, so that the lanes that a read or a write takes
// together (16 of them, of two lane groups) lie in different banks: a key's (row =
// token 16 a + 4 t + b, read for all a and b at once) by bits of a and b, a value's
// (row = dimension, pieces 4 u + g of the 8 tokens 16 g + 8 u ..) by its low bits.
template <int D>
__device__ __forceinline__ int kv_key_swap(int token) {
    if (D == 64) return -(token >> 4) & 3;
    if (D == 128) return (token & 3) | (token >> 2 & 4);
    return (token & 3) | (token >> 2 & 12);
}
__device__ __forceinline__ int kv_value_swap(int d) { return (d & 1) | (d >> 1 & 2) | (d << 1 & 4); }

// A tile's keys and values are 4 D pieces each; piece p = j * threads + thread of
// the keys is in a page (a scalar: a wave's 1024 / D tokens lie in one block of 16) at an
// offset that is the same for every tile.
template <int D>
__device__ __forceinline__ int kv_key_offset(int p, int T) {
    constexpr int KP = D / 16;  // 16-byte pieces of a key
    return (p / KP & (T - 1)) * D + 16 * (p % KP);
}
template <int D>
__device__ __forceinline__ int kv_key_place(int p) {
    constexpr int KP = D / 16;
    return p / KP * KP + ((p % KP) ^ kv_key_swap<D>(p / KP));
}
// The page of a wave's pieces, the first of them piece p; id: of this lane's group.
template <int D>
__device__ __forceinline__ const int8_t* kv_key_page(const AttnCall& A, const Place& P, int tile, int idg, int p) {
    const int T = 1 << A.c.log2_page, id = __builtin_amdgcn_readlane(idg, p / D * 16);  // of token block p / D
    return A.c.k + ((int64_t(max(id, 0)) * A.c.kv_heads + P.kvh) * T + (tile * 64 & (T - 1))) * D;
}

// NW waves of 16 * NR rows; WPS of them to a SIMD.
template <typename T, int D, int NR, int NW, int WPS>
__global__ __launch_bounds__(64 * NW, WPS) void kv_block_kernel(const AttnCall A) {
    constexpr int BM = 16 * NR * NW, THREADS = 64 * NW, PT = 4 * D / THREADS;
    static_assert(PT * THREADS == 4 * D, "whole pieces a thread");
    constexpr int PITCH = D + 8;  // of an output row in LDS: 16 rows' 8 bytes are in different banks
    __shared__ i32x4 lds[24 * D];
    static_assert(BM * PITCH * 2 <= 24 * D * 16, "the output fits where the tiles were");
    // the queries' lowest digits, each lane's own: as many in LDS as leave a CU its workgroups, as registers
    // are short (all, but for 64 rows of 128 dimensions half of them: held in registers they all spill)
    constexpr int KS = D / 64;
    constexpr int SPARE = (160 * 1024 / (4 * WPS / NW) - 24 * D * 16) / (THREADS * 16), IN_LDS = SPARE < NR * KS ? SPARE : NR * KS;
    __shared__ i32x4 digits[NW * IN_LDS * 64];
    i32x4* const low_lds = digits + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * IN_LDS * 64;
    i32x4 low_regs[NR * KS - IN_LDS + 1];
    i32x4 *const k0 = lds, *const k1 = lds + 4 * D;
    h16x8 *const v0 = reinterpret_cast<h16x8*>(lds + 8 * D), *const v1 = v0 + 8 * D;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    Place P;
    if (!kv_place<BM>(A, P)) return;
    const int rows = min(BM, P.e.count * int(A.group) - P.first);
    const TileRange all = kv_tiles(A, P.e, unsigned(P.first) / A.group, unsigned(P.first + rows - 1) / A.group);
    const bool part = !kv_whole(A, all);
    if (!part && P.split > 0) return;
    const int share = kv_share(A, all), begin = all.begin + P.split * share, end = part ? min(all.end, begin + share) : all.end;
    if (part && begin >= end) {
        if (tid < rows) kv_store_lse(A, P, P.first + tid, -INFINITY);
        return;
    }
    // this wave's rows, the tiles that any of them sees and those that all see whole
    const int first = P.first + 16 * NR * wave, mine = min(16 * NR, rows - 16 * NR * wave);
    Rows<D, NR> R;
    int see_from = 0, see_until = 0, clear_from = 0, clear_until = 0;
    if (mine > 0) {
        const int i0 = unsigned(first) / A.group, i1 = unsigned(first + mine - 1) / A.group;
        const TileRange t = kv_tiles(A, P.e, i0, i1);
        see_from = t.begin, see_until = t.end;
        clear_from = (kv_from(A, P.e, i1) + 63) >> 6, clear_until = max(kv_until(A, P.e, i0), 0) >> 6;
    }
    const int page_tokens = 1 << A.c.log2_page;
    int ofs[PT];
#pragma unroll
    for (int j = 0; j < PT; j++) ofs[j] = kv_key_offset<D>(j * THREADS + tid, page_tokens);
    // of the values, piece p is the 16 tokens 16 (p % 4) .. of dimension p / 4
    const int gv = lane & 3, dv = tid >> 2;
    // (table entries and scale bytes are looked at a step after they are requested, so that nothing
    // waits for them; begin < end: there is a sequence)
    auto table = [&](int tile, int block) __attribute__((always_inline)) {
        return kv_page_entry(A.c, P.e.seq, (tile * 64 + 16 * block) >> A.c.log2_page);
    };
    if (begin < end) {
        int tile = begin, base = 0, base_next = 0;
        int eg = table(tile, g), ev = table(tile, gv), idn, idv, kb, vb, kbn, vbn, vbv;
        RowLoads<D, NR> W;
        kv_begin_loads<D, NR>(A, P, first, R, W);
        i32x4 raw[PT], rawk[PT];
        // requests tile `t` (table entries eg, ev): its scales, values and keys
        auto request = [&](int t) __attribute__((always_inline)) {
            idn = kv_page_of(A.c, eg), idv = kv_page_of(A.c, ev);
            const int64_t at = int64_t(max(idn, 0)) * A.c.kv_heads + P.kvh, av = int64_t(max(idv, 0)) * A.c.kv_heads + P.kvh;
            const int next = min(t + 1, end - 1);
            eg = table(next, g), ev = table(next, gv);
            kbn = A.c.ks[at], vbn = A.c.vs[at], vbv = A.c.vs[av];
            const int8_t* src = A.c.v + (av * D + dv) * page_tokens + ((t * 64 + 16 * gv) & (page_tokens - 1));
#pragma unroll
            for (int j = 0; j < PT; j++) raw[j] = *reinterpret_cast<const i32x4*>(src + THREADS / 4 * j * page_tokens);
#pragma unroll
            for (int j = 0; j < PT; j++)
                rawk[j] = *reinterpret_cast<const i32x4*>(kv_key_page<D>(A, P, t, idn, j * THREADS + 64 * wave) + unsigned(ofs[j]));
        };
        // its values as f16
        auto convert = [&](i32x4* kbuf, h16x8* vbuf) __attribute__((always_inline)) {
            base_next = max(base, kv_group_max(idn < 0 || vbn == 255 ? 0 : vbn));
#pragma unroll
            for (int j = 0; j < PT; j++) kbuf[kv_key_place<D>(j * THREADS + tid)] = rawk[j];
            const Convert to(idv < 0 || vbv == 255 ? 0 : vbv, base_next);
#pragma unroll
            for (int j = 0; j < PT; j++) {
                const int d = dv + THREADS / 4 * j;
                vbuf[8 * d + (gv ^ kv_value_swap(d))] = to(uint32_t(raw[j][0]), uint32_t(raw[j][1]));
                vbuf[8 * d + ((4 + gv) ^ kv_value_swap(d))] = to(uint32_t(raw[j][2]), uint32_t(raw[j][3]));
            }
        };
        request(tile);
        kv_begin<T, D, NR>(A, R, W, [&](int r, int ks, const i32x4& x) __attribute__((always_inline)) {
            if (r * KS + ks < IN_LDS) low_lds[(r * KS + ks) * 64 + lane] = x;
            else low_regs[r * KS + ks - IN_LDS] = x;
        });  // (while the first tile is on its way)
        convert(k0, v0);
        auto step = [&](const i32x4* kc, const h16x8* vc, i32x4* kn, h16x8* vn) __attribute__((always_inline)) {
            __syncthreads();  // this tile is there, and the other buffers are read
            const bool dead = idn < 0, more = tile + 1 < end;
            kb = kbn, vb = vbn, base = base_next;
            if (more) request(tile + 1);
            if (tile >= see_from && tile < see_until) {
                const bool fine = kv_group_max(kb) >= R.fine;
                const float kf = kb == 255 || vb == 255 ? __uint_as_float(0x7fc00000u) : e8m0_to_f32(uint32_t(kb));
                f32x4 s[NR][4];
                auto keys = [&](int t, int ks) __attribute__((always_inline)) {
                    const int token = 4 * (lane & 12) + 4 * t + (lane & 3);
                    return kc[token * (D / 16) + ((4 * ks + g) ^ kv_key_swap<D>(token))];
                };
                kv_scores<D, NR>(R, keys, s);
                h16x8 p[NR][2];
                kv_softmax<D, NR>(R, s, fine, keys, [&](int r, int ks) __attribute__((always_inline)) {
                    return r * KS + ks < IN_LDS ? low_lds[(r * KS + ks) * 64 + kv_lane()] : low_regs[r * KS + ks - IN_LDS];
                }, kf, tile * 64 + 16 * g, dead,
                                  tile < clear_from || tile >= clear_until || __any(dead), base, p);
                kv_values<D, NR>(R, p, [&](int dt, int u) __attribute__((always_inline)) {
                    const int d = 16 * dt + (lane & 15);
                    return vc[8 * d + ((4 * u + g) ^ kv_value_swap(d))];
                });
            }
            if (more) convert(kn, vn);
            tile++;
            return more;
        };
        while (step(k0, v0, k1, v1) && step(k1, v1, k0, v0)) {
        }
    } else {
        kv_nothing<D, NR>(R);
    }
    __syncthreads();  // the last tile is read
    uint16_t* turn = reinterpret_cast<uint16_t*>(lds) + wave * 16 * NR * PITCH;
#pragma unroll
    for (int r = 0; r < NR; r++) {
        float l = R.l[r];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int row = 16 * r + (lane & 15);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (part && g == 0 && row < mine) kv_store_lse(A, P, first + row, l == 0.f ? -INFINITY : __builtin_amdgcn_logf(l) - R.b[r]);
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) {
            f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = __builtin_amdgcn_ldexpf(R.o[r][dt][j] * inv, R.base - 132);
            if (!part) *reinterpret_cast<uint2*>(turn + row * PITCH + 16 * dt + 4 * g) = kv_pack4<T>(o);
            else if (row < mine) kv_store_part4<D>(A, P, first + row, 16 * dt + 4 * g, o);
        }
    }
    if (part) return;
    __syncthreads();
    // whole rows at once (32 prompts of 128 tokens: 38.6 us with 8-byte stores from the registers, 37.7 so)
    constexpr int LANES = D / 8, AT = 64 / LANES;
#pragma unroll
    for (int i = 0; i < 16 * NR; i += AT) {
        const int row = i + lane / LANES, d = lane % LANES * 8;
        if (row < mine) *reinterpret_cast<i32x4*>(kv_out<D>(A, P, first + row) + d) = *reinterpret_cast<const i32x4*>(turn + row * PITCH + d);
    }
}

// The splits of one row and head, weighed by their sums; a split that had
// nothing to do has lse = -inf and its part is not used.  W waves (1, or 4 where
// there are many splits); D / 4 lanes take one split's part, and the parts are
// requested with the sums, before any weight is known, 4 splits ahead.
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttnCall A) {
    __shared__ Joiner<D, W> J;
    constexpr int LANES = D / 4, SETS = 64 * W / LANES;
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    // (grid: rows by heads, or by 4 heads)
    const int h = W == 1 ? blockIdx.y * 4 + (threadIdx.x >> 6) : blockIdx.y;
    if (h >= A.heads) return;
    int entry, i;
    if (!kv_locate(A.b, blockIdx.x, [](int n) { return n; }, entry, i)) return;
    int start, count;
    kv_rows(A.b, entry, start, count);
    if (A.causal) {
        const KvEntry e = kv_entry(A.c, A.b, entry);
        const unsigned first = (unsigned(i) * A.group + unsigned(h) % A.group) / A.rows * A.rows;
        const unsigned last = min(first + A.rows, unsigned(count) * A.group) - 1;
        if (kv_whole(A, kv_tiles(A, e, first / A.group, last / A.group))) return;  // written out
    }
    const int64_t at = int64_t(start + i) * A.heads + h;
    const float* lse = A.lse + at * A.splits;
    const f32x4* part = reinterpret_cast<const f32x4*>(A.part + at * A.splits * D) + t % LANES;
    const int set = t / LANES;
    float m = -INFINITY, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < A.splits; s0 += 4 * SETS) {
        f32x4 x[4];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int s = s0 + j * SETS + set;
            f[j] = s < A.splits ? lse[s] : -INFINITY;
            x[j] = s < A.splits ? part[int64_t(s) * LANES] : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        kv_merge4(f, x, m, sum, o);
    }
    if (J.join(t, m, sum, o)) kv_out4<T, D>(A, at, t, sum, o);
}

// (n and total are looked at before: kv_rows_ok)
bool attention_sizes_ok(const char* who, const eq_kv_cache* c, int n_heads, int64_t total) {
    if (n_heads <= 0 || n_heads > 65535 || n_heads % c->kv_heads != 0) {
        set_error(std::string(who) + ": n_heads must be a multiple of kv_heads, at most 65535");
        return false;
    }
    if (total * n_heads > INT32_MAX) {
        set_error(std::string(who) + ": need 0 <= n <= 2^16 sequences and 0 <= total * n_heads < 2^31");
        return false;
    }
    return true;
}

// Which kernel, how many rows a workgroup, how many splits: from the call's
// sizes alone (lengths and offsets are on the device; the table's width bounds them), so of a ragged batch by
// its rows on average: a prompt of 2000 rows beside one row after 65536 tokens takes 1.71 ms in one call, whose
// row is one workgroup's a KV head, 71 and 33 us in two.
struct Plan {
    int rows;    // of a workgroup: 16 (stream), 64 or 128 (block)
    int64_t tiles;
    int splits;  // of a block's tokens
    int groups;  // workgroups of a stream
    int slot_rows;  // of a stream's slots
    int join_waves;  // of a stream's rows: 16, 4 or 1
    size_t part_bytes, lse_bytes;
};
Plan plan_attention(const eq_kv_cache* c, int n_heads, int64_t n, int64_t total, bool ragged) {
    Plan p = {};
    const int64_t group = n_heads / c->kv_heads, rows = n ? total * group / n : 0;  // of a sequence and KV head, on average
    const int64_t cap = (c->width * c->page_tokens + 63) / 64;
    auto blocks = [&](int bm) {
        return ragged ? total * group / bm + n : n * ((total / (n ? n : 1) * group + bm - 1) / bm);
    };
    const int64_t most = blocks(kStreamRows) * c->kv_heads;  // units of a stream (over 2^31 tiles are not listed)
    // blocks, and (of a ragged batch, whose blocks are bounded by one a sequence too many) those of even sequences
    auto likely = [&](int bm) { return n * ((rows + bm - 1) / bm) * c->kv_heads; };
    p.rows = 128;
    if (rows <= 48 && most < INT32_MAX / cap) p.rows = kStreamRows;
    else if (rows <= 64) p.rows = 64;
    // 64 rows use a tile for half as many products (2048 rows over 4000 tokens of 128 dimensions: 114 us,
    // 98 with 128), but fill the CUs with fewer (2 prompts of 128 tokens, 16 heads of 128 dimensions: 9.7 us, 15.2
    // with 128; 512 rows over 8000 tokens lose by it, 61.6 and 57.6) and waste fewer (150 rows in 192: 44 us, in
    // 256 57); at 256 dimensions, where they need the LDS of 128, they lose always (37 us, 29)
    else if (c->head_dim <= 128 && (2 * likely(128) <= device_cu_count() || 7 * likely(64) < 12 * likely(128))) p.rows = 64;
    p.tiles = blocks(p.rows);
    if (p.rows == kStreamRows) {
        const int64_t runs = (most * cap + 3) / 4;  // at least a tile for each of 4 waves
        p.splits = 1;
        p.groups = int(runs < 2 * device_cu_count() ? runs : 2 * device_cu_count());
        // few rows have many parts: 256 parts take 16 waves 2.7 us instead of 4 waves 6 us, 17 parts 4.7 instead
        // of 3.9.  Many have few: 7200 rows take a wave each 6.3 us instead of 18.5 with 4 waves, 640 rows 7.2 instead of 5.4
        const int64_t joins = total * n_heads;
        p.join_waves = n <= 64 && joins <= 2 * device_cu_count() && cap > 64 ? 16 : (joins <= 4 * device_cu_count() ? 4 : 1);
        // (a decode step of 4 heads a group fills a quarter of 16 rows: 8.4 MB at 128 dimensions instead of 33.8)
        const int64_t unit = (ragged || !n ? total : total / n) * group;
        p.slot_rows = int(unit < kStreamRows ? unit : kStreamRows);
        p.part_bytes = size_t(p.groups) * 8 * p.slot_rows * c->head_dim * 4;
        p.lse_bytes = (size_t(p.groups) * 8 * p.slot_rows * 4 + 255) & ~size_t(255);
        return p;
    }
    // as many splits as come nearest to filling the CUs once (300 queries over 8000 tokens, 80 blocks: 560
    // workgroups 95 us, 480 79 us); of 128 rows two workgroups fit a CU, of 64 three or, at 64 dimensions, four, at 256 one
    const int fit = c->head_dim > 128 ? 1 : p.rows == 128 ? 2 : c->head_dim == 128 ? 3 : 4;
    const int64_t units = likely(p.rows);
    int64_t splits = units ? (fit * device_cu_count() + units / 2) / units : 1;
    if (splits > (cap + 3) / 4) splits = (cap + 3) / 4;
    if (splits > 1024) splits = 1024;
    p.splits = splits < 1 ? 1 : int(splits);
    p.groups = 0;
    p.part_bytes = p.splits > 1 ? size_t(total) * n_heads * p.splits * c->head_dim * 4 : 0;
    p.lse_bytes = p.splits > 1 ? (size_t(total) * n_heads * p.splits * 4 + 255) & ~size_t(255) : 0;
    return p;
}

// Workgroups of a plan's block kernel, and threads of one.
int64_t plan_blocks(const eq_kv_cache* c, const Plan& p) { return p.rows == kStreamRows ? 0 : p.tiles * c->kv_heads * p.splits; }
int plan_threads(const eq_kv_cache* c, const Plan& p) { return p.rows == 128 && c->head_dim > 128 ? 512 : 256; }

// Grids of under 2^32 threads a side, of the blocks and of the joins (a row's heads lie in y); a stream's own is small.
bool plan_ok(const char* who, const eq_kv_cache* c, const Plan& p, int64_t total) {
    if (total < (1 << 24) && plan_blocks(c, p) * plan_threads(c, p) < int64_t(1) << 32) return true;
    set_error(std::string(who) + ": too many rows");
    return false;
}

}  // namespace
}  // namespace eq

using namespace eq;

extern "C" int64_t eq_kv_attention_scratch(const eq_kv_cache* cache, int n_heads, int64_t n, int64_t total, bool ragged) {
    clear_error();
    const char* who = "eq_kv_attention_scratch";
    if (!kv_cache_ok(who, cache) || !kv_rows_ok(who, n, total, !ragged) || !attention_sizes_ok(who, cache, n_heads, total)) return -1;
    const Plan p = plan_attention(cache, n_heads, n, total, ragged);
    if (!plan_ok(who, cache, p, total)) return -1;
    return int64_t(p.part_bytes + p.lse_bytes);
}

extern "C" int eq_kv_attention(void* out, const void* q, int64_t q_stride, int n_heads, const eq_kv_cache* cache,
                               int64_t layer, const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total,
                               float scale, bool causal, int64_t window, const float* rope, int64_t rope_positions,
                               int dtype, void* scratch, int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_attention";
    if (!kv_cache_ok(who, cache) || !kv_batch_ok(who, cache, layer, seqs, n, cu, total) ||
        !attention_sizes_ok(who, cache, n_heads, total) || !kv_rope_ok(who, cache, rope, rope_positions))
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
    if (!plan_ok(who, cache, plan, total)) return 1;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    WsHold hold;
    AttnCall A;
    A.part = A.lse = nullptr;
    if (plan.part_bytes) {
        const size_t need = plan.part_bytes + plan.lse_bytes;
        if (scratch && (scratch_bytes < 0 || size_t(scratch_bytes) < need || !aligned(scratch, 256))) {
            set_error("eq_kv_attention: needs " + std::to_string(need) + " bytes of 256-byte aligned scratch");
            return 1;
        }
        char* ws = static_cast<char*>(scratch ? scratch : ws_acquire(hold, nullptr, need, st));
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
    A.rows = plan.rows;
    A.tiles = int(plan.tiles);
    A.splits = plan.splits;
    A.groups = plan.groups;
    A.slot_rows = plan.slot_rows;
    A.window = int(window < kKvMaxLength ? window : kKvMaxLength);
    A.causal = causal;
    const dim3 grid{unsigned(plan_blocks(cache, plan))};
    auto go = [&](auto t, auto d) {
        typedef decltype(t) T;
        constexpr int DIM = decltype(d)::value;
        if (plan.rows == kStreamRows) {
            kv_stream_kernel<T, DIM><<<dim3(unsigned(plan.groups)), dim3(256), 0, st>>>(A);
            const dim3 rows{unsigned(total), unsigned(n_heads)};
            if (plan.join_waves == 16) kv_stream_join_kernel<T, DIM, 16><<<rows, dim3(1024), 0, st>>>(A);
            else if (plan.join_waves == 4) kv_stream_join_kernel<T, DIM, 4><<<rows, dim3(256), 0, st>>>(A);
            else kv_stream_join_kernel<T, DIM, 1><<<dim3(unsigned(total), unsigned((n_heads + 3) / 4)), dim3(256), 0, st>>>(A);
            return;
        }
        // 128 rows are 4 waves of 32 up to 128 dimensions (2048 queries over 32768 tokens of 128: 1.19 ms;
        // 8 of 16, whose registers spill at four to a SIMD, 1.33), 8 of 16 at 256, where 4 waves of 32 do not
        // fit and 64 rows to a workgroup read every key twice as often (0.60 ms against 1.05)
        if (plan.rows == 64) kv_block_kernel<T, DIM, 1, 4, DIM == 64 ? 4 : DIM == 128 ? 3 : 1><<<grid, dim3(256), 0, st>>>(A);
        else if constexpr (DIM <= 128) kv_block_kernel<T, DIM, 2, 4, 2><<<grid, dim3(256), 0, st>>>(A);
        else kv_block_kernel<T, DIM, 1, 8, 2><<<grid, dim3(512), 0, st>>>(A);
        if (plan.splits > 16) kv_join_kernel<T, DIM, 4><<<dim3(unsigned(total), unsigned(n_heads)), dim3(256), 0, st>>>(A);
        else if (plan.splits > 1) kv_join_kernel<T, DIM, 1><<<dim3(unsigned(total), unsigned((n_heads + 3) / 4)), dim3(256), 0, st>>>(A);
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

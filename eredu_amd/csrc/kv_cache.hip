// The paged 8-bit key/value cache: writing new tokens, reading them back, and
// its pages -- growing, sharing, freeing and compacting (kv_common.hpp has the
// format, include/eredu_kv.h the rules; the attention is in kv_attention.hip).
//
// All of these move bytes: append reads 2 bytes and writes 1 a value (10000 tokens of 8 heads
// of 128 dimensions 18 us, 3.4 TB/s), read the reverse (14 us, 4.4 TB/s), extend and
// compact read and write whole pages (335 MB in 50 us); fork, shrink and free are trips to the tables: a fork
// to 15 sequences of 31 pages 3.7 us, 16 sequences shrunk 2.5, 15 freed 1.6 to 4.
#include "kv_common.hpp"

namespace eq {

// ------------------------------------------------------------------ host side

bool kv_cache_ok(const char* name, const eq_kv_cache* c) {
    const std::string who(name);
    auto bad = [&](const char* what) {
        set_error(who + ": " + what);
        return false;
    };
    if (!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !c->tables || !c->lengths || !c->refs ||
        !c->missing)
        return bad("null pointer argument");
    const int T = c->page_tokens, D = c->head_dim;
    if (T < 16 || T > kKvMaxPage || (T & (T - 1))) return bad("page_tokens must be 16, 32, 64 or 128");
    if (D != 64 && D != 128 && D != 256) return bad("head_dim must be 64, 128 or 256");
    if (c->kv_heads <= 0 || c->kv_heads > 65535) return bad("kv_heads must be in [1, 65535]");
    if (c->layers <= 0 || c->layers > INT32_MAX || c->pages <= 0 || c->pages > INT32_MAX - 64 || c->sequences <= 0 ||
        c->sequences > INT32_MAX || c->width <= 0 || c->width > kKvMaxLength / T)
        return bad("layers, pages, sequences and width must be positive, width * page_tokens at most 2^30");
    if (c->sequences * c->width >= int64_t(1) << 31) return bad("tables must have fewer than 2^31 entries");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16)) return bad("codes must be 16-byte aligned");
    return true;
}

bool kv_rows_ok(const char* name, int64_t n, int64_t total, bool even) {
    if (n < 0 || total < 0 || n > kKvMaxEntries || total > INT32_MAX / 2 || (n == 0 && total != 0)) {
        set_error(std::string(name) + ": need 0 <= n <= 2^16 sequences and 0 <= total < 2^30 rows");
        return false;
    }
    if (n > 0 && even && total % n != 0) {
        set_error(std::string(name) + ": without offsets the rows must divide evenly among the sequences");
        return false;
    }
    return true;
}

bool kv_batch_ok(const char* name, const eq_kv_cache* c, int64_t layer, const int32_t* seqs, int64_t n,
                 const int32_t* cu, int64_t total) {
    const std::string who(name);
    if (layer < 0 || layer >= c->layers) {
        set_error(who + ": layer " + std::to_string(layer) + " outside [0, " + std::to_string(c->layers) + ")");
        return false;
    }
    if (!kv_rows_ok(name, n, total, !cu)) return false;
    if (n > 0 && !seqs) {
        set_error(who + ": null pointer argument");
        return false;
    }
    return true;
}

bool kv_rope_ok(const char* name, const eq_kv_cache* c, const float* rope, int64_t positions) {
    if (!rope) return true;
    if (positions < c->width * c->page_tokens || !aligned(rope, 16)) {
        set_error(std::string(name) + ": the rotation table must be 16-byte aligned and cover width * page_tokens "
                  "positions");
        return false;
    }
    return true;
}

KvView kv_view(const eq_kv_cache* c, int64_t layer) {
    const int64_t codes = c->pages * c->kv_heads * c->page_tokens * c->head_dim, scales = c->pages * c->kv_heads;
    KvView v;
    v.k = c->k_codes + layer * codes;
    v.v = c->v_codes + layer * codes;
    v.ks = c->k_scales + layer * scales;
    v.vs = c->v_scales + layer * scales;
    v.tables = c->tables;
    v.lengths = c->lengths;
    v.pages = int(c->pages);
    v.sequences = int(c->sequences);
    v.width = int(c->width);
    v.kv_heads = c->kv_heads;
    v.log2_page = __builtin_ctz(unsigned(c->page_tokens));
    return v;
}

KvBatch kv_batch(const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total) {
    return KvBatch{seqs, cu, int(n), int(cu || n == 0 ? 0 : total / n), int(total)};
}

namespace {

// ------------------------------------------------------------ append and read

// Pages that `count` consecutive tokens can lie in, wherever they begin.
__host__ __device__ __forceinline__ int kv_spanned(int count, int log2_page) {
    return count > 0 ? ((count + (1 << log2_page) - 2) >> log2_page) + 1 : 0;
}
// Their sum over a batch, or more: sum((c + T - 2) / T + 1) <= total / T + 2 n.
int64_t kv_page_units(const KvBatch& b, int log2_page) {
    return b.cu ? (int64_t(b.total) >> log2_page) + 2 * int64_t(b.n) : int64_t(b.n) * kv_spanned(b.each, log2_page);
}

// The smallest byte in [1, 254] with most <= 127 * 2^(byte - 127), `most` given
// by its bits: 127 * 2^(b - 127) has exponent field b + 6 and fraction
// 0x7e0000.  255 for infinities and NaN.
__device__ __forceinline__ int kv_byte(uint32_t bits) {
    if (bits >= 0x7f800000u) return 255;
    return kv_clamp(int(bits >> 23) - 6 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0), 1, 254);
}

// 2^(127 - b): what a page's values are multiplied by before they are rounded.
__device__ __forceinline__ float kv_inverse(int b) {
    return __uint_as_float(b >= 254 ? 0x00400000u : unsigned(254 - b) << 23);
}

__device__ __forceinline__ uint32_t kv_code(float x, float inv) { return uint32_t(int(rintf(x * inv))) & 0xffu; }

// The four codes of a word in a scale 2^k (k <= 0) times as large: f = 2^-k.
__device__ __forceinline__ uint32_t kv_rescale4(uint32_t w, float f) {
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) o |= (uint32_t(int(rintf(float(int8_t(w >> (8 * i))) * f))) & 0xffu) << (8 * i);
    return o;
}

// This call's tokens in one page of one entry.
struct KvSpan {
    int page;         // -1: missing
    int from, until;  // places [from, until) of the page; empty: nothing to do
    int row;          // of the token at `from`
    int position;     // and its position
};

__device__ __forceinline__ KvSpan kv_span(const KvView& c, const KvEntry& e, int place) {
    const int first = e.length - e.count, index = (first >> c.log2_page) + place, base = index << c.log2_page;
    KvSpan s;
    s.from = max(first - base, 0);
    s.until = min(e.length - base, 1 << c.log2_page);
    s.position = base + s.from;
    s.row = e.start + s.position - first;
    s.page = s.from < s.until && e.seq >= 0 ? kv_page(c, e.seq, index) : -1;
    return s;
}

// 8 values at dimension d0 < D / 2 of a row and the 8 that they pair with, as
// loaded with the angles of theirs, and turned.
struct KvPairs {
    uint4 a, b;
    float4 cs[2], sn[2];

    __device__ __forceinline__ void load(const uint16_t* x, int d0, int D, const float* rot) {
        a = *reinterpret_cast<const uint4*>(x + d0);
        b = *reinterpret_cast<const uint4*>(x + d0 + D / 2);
        if (!rot) return;
        const float4* p = reinterpret_cast<const float4*>(rot + d0);
        cs[0] = p[0], cs[1] = p[1], sn[0] = p[D / 8], sn[1] = p[D / 8 + 1];
    }
    template <typename T>
    __device__ __forceinline__ void values(bool turn, float (&f)[16]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f[2 * i] = kv_to_f32<T>(w[i] & 0xffffu);
            f[2 * i + 1] = kv_to_f32<T>(w[i] >> 16);
        }
        if (!turn) return;
        const float c[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
        const float n[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w, sn[1].x, sn[1].y, sn[1].z, sn[1].w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float u = f[i] * c[i] - f[8 + i] * n[i];
            f[8 + i] = f[8 + i] * c[i] + f[i] * n[i];
            f[i] = u;
        }
    }
};

__device__ __forceinline__ uint32_t kv_most(const float (&f)[16]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
}

// 4 rows of 4 bytes <-> 4 columns.
__device__ __forceinline__ void kv_turn4(const uint32_t r0, const uint32_t r1, const uint32_t r2, const uint32_t r3, uint32_t (&c)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(r1, r0, 0x05010400u), b = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
    const uint32_t d = __builtin_amdgcn_perm(r3, r2, 0x05010400u), e = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
    c[0] = __builtin_amdgcn_perm(d, a, 0x05040100u), c[1] = __builtin_amdgcn_perm(d, a, 0x07060302u);
    c[2] = __builtin_amdgcn_perm(e, b, 0x05040100u), c[3] = __builtin_amdgcn_perm(e, b, 0x07060302u);
}

// The bytes of a word of 4 places, from place t on, that lie in [from, until).
__device__ __forceinline__ uint32_t kv_places(int t, int from, int until) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) m |= t + i >= from && t + i < until ? 0xffu << (8 * i) : 0u;
    return m;
}

// Grid (page units, kv_heads, keys | values), NT threads: one page of one
// head.  The page's new rows are read for their largest magnitude and, where
// that is one round of 2 pieces a thread (64 tokens of 128 dimensions), stay in registers for
// their codes; else they are read again, from L2.  Values turn in LDS, by 4 x 4
// bytes, to be written along the tokens, 16 of a dimension at once.
// 6 waves a SIMD: 80 registers instead of 117 cover more of the loads' trips, 10000
// tokens 20.1 -> 18.0 us.
constexpr int kAppendItems = 2;

template <typename T, int D, int NT>
__global__ __launch_bounds__(NT, 6) void kv_append_kernel(KvView c, KvBatch b, const uint16_t* __restrict__ k,
                                                        const uint16_t* __restrict__ v, int64_t k_stride,
                                                        int64_t v_stride, const float* __restrict__ rope) {
    extern __shared__ __attribute__((aligned(16))) uint8_t turn[];  // values: [token][D + 4]
    __shared__ uint32_t red[NT / 64];
    const int tid = threadIdx.x, head = blockIdx.y, log2_page = c.log2_page, page_tokens = 1 << log2_page;
    const bool values = blockIdx.z != 0;
    int entry, place;
    if (!kv_locate(b, blockIdx.x, [&](int n) { return kv_spanned(n, log2_page); }, entry, place)) return;
    const KvEntry e = kv_entry(c, b, entry);
    if (e.seq < 0) return;
    const KvSpan s = kv_span(c, e, place);
    constexpr int groups = D / 16, pitch = D + 4;
    const int items = max(s.until - s.from, 0) * groups;
    const uint16_t* x = (values ? v + int64_t(s.row) * v_stride : k + int64_t(s.row) * k_stride) + int64_t(head) * D;
    const int64_t stride = values ? v_stride : k_stride;
    // (the rows are read whether or not the page is there: they are rows of this call; the angles only
    // of positions that have a page)
    const float* rot = rope && !values && s.page >= 0 ? rope + int64_t(s.position) * D : nullptr;
    KvPairs raw[kAppendItems];
#pragma unroll
    for (int j = 0; j < kAppendItems; j++) {
        const int it = tid + NT * j, t = it / groups;
        if (it < items) raw[j].load(x + int64_t(t) * stride, it % groups * 8, D, rot ? rot + int64_t(t) * D : nullptr);
    }
    bool later = false;  // another entry names this sequence
    for (int j = entry + 1 + tid; j < b.n; j += NT) later |= b.seqs[j] == e.seq;
    if (__syncthreads_or(later) || s.page < 0) return;
    uint8_t* scale = (values ? c.vs : c.ks) + int64_t(s.page) * c.kv_heads + head;
    const int was = s.from > 0 ? *scale : 0;

    const bool held = items <= NT * kAppendItems;
    uint32_t most = 0;
    float f[kAppendItems][16];
#pragma unroll
    for (int j = 0; j < kAppendItems; j++)
        if (tid + NT * j < items) {
            raw[j].values<T>(rot != nullptr, f[j]);
            most = max(most, kv_most(f[j]));
        }
    for (int it = tid + NT * kAppendItems; it < items; it += NT) {
        const int t = it / groups;
        KvPairs r;
        float y[16];
        r.load(x + int64_t(t) * stride, it % groups * 8, D, rot ? rot + int64_t(t) * D : nullptr);
        r.values<T>(rot != nullptr, y);
        most = max(most, kv_most(y));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, uint32_t(__shfl_xor(int(most), o)));
    if ((tid & 63) == 0) red[tid >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; w++) most = max(most, red[w]);
    const int now = max(kv_byte(most), was);
    if (tid == 0) *scale = uint8_t(now);
    const bool move = s.from > 0 && was < now && now != 255;  // the page's older codes change their step
    const float down = __uint_as_float(unsigned(max(127 + was - now, 0)) << 23);
    const float inv = kv_inverse(now);

    int8_t* codes = (values ? c.v : c.k) + (int64_t(s.page) * c.kv_heads + head) * page_tokens * D;
    auto put = [&](int it, const float (&y)[16]) __attribute__((always_inline)) {
        const int t = it / groups, d0 = it % groups * 8;
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (now != 255) {
#pragma unroll
            for (int i = 0; i < 16; i++) w[i >> 2] |= kv_code(y[i], inv) << (8 * (i & 3));
        }
        if (values) {
            uint32_t* p = reinterpret_cast<uint32_t*>(turn + t * pitch + d0);
            p[0] = w[0], p[1] = w[1];
            p = reinterpret_cast<uint32_t*>(turn + t * pitch + d0 + D / 2);
            p[0] = w[2], p[1] = w[3];
        } else {
            int8_t* row = codes + (s.from + t) * D + d0;
            *reinterpret_cast<uint2*>(row) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2*>(row + D / 2) = make_uint2(w[2], w[3]);
        }
    };
#pragma unroll
    for (int j = 0; j < kAppendItems; j++)
        if (tid + NT * j < items) put(tid + NT * j, f[j]);
    if (!held) {
        for (int it = tid + NT * kAppendItems; it < items; it += NT) {
            const int t = it / groups;
            KvPairs r;
            float y[16];
            r.load(x + int64_t(t) * stride, it % groups * 8, D, rot ? rot + int64_t(t) * D : nullptr);
            r.values<T>(rot != nullptr, y);
            put(it, y);
        }
    }
    if (!values) {
        if (move) {
            uint4* p = reinterpret_cast<uint4*>(codes);
            for (int i = tid; i < s.from * D / 16; i += NT) {
                const uint4 o = p[i];
                p[i] = make_uint4(kv_rescale4(o.x, down), kv_rescale4(o.y, down), kv_rescale4(o.z, down),
                                  kv_rescale4(o.w, down));
            }
        }
        return;
    }
    __syncthreads();
    // 16 places of 4 dimensions: older codes, then new ones, then what was there
    const int first = move ? 0 : s.from >> 4, blocks = ((s.until + 15) >> 4) - first;
    for (int it = tid; it < blocks * (D / 4); it += NT) {
        const int d4 = it / blocks, t0 = (first + it - d4 * blocks) * 16;
        uint32_t n[4][4];  // [dimension][4 places]
#pragma unroll
        for (int q = 0; q < 4; q++) {
            uint32_t r[4], col[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = t0 + 4 * q + i;
                r[i] = t >= s.from && t < s.until ? *reinterpret_cast<const uint32_t*>(turn + (t - s.from) * pitch + 4 * d4) : 0u;
            }
            kv_turn4(r[0], r[1], r[2], r[3], col);
#pragma unroll
            for (int i = 0; i < 4; i++) n[i][q] = col[i];
        }
        uint4* p = reinterpret_cast<uint4*>(codes + int64_t(4 * d4) * page_tokens + t0);
        const bool whole = t0 >= s.from && t0 + 16 <= s.until;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint4* at = reinterpret_cast<uint4*>(reinterpret_cast<int8_t*>(p) + i * page_tokens);
            if (!whole) {
                const uint4 o = *at;
                const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t fresh = kv_places(t0 + 4 * q, s.from, s.until), old = kv_places(t0 + 4 * q, 0, s.from);
                    uint32_t keep = w[q];
                    if (move) keep = (keep & ~old) | (kv_rescale4(keep, down) & old);
                    n[i][q] = (n[i][q] & fresh) | (keep & ~fresh);
                }
            }
            *at = make_uint4(n[i][0], n[i][1], n[i][2], n[i][3]);
        }
    }
}

// Grid (page units, kv_heads, keys | values), NT threads: the rows of one page
// and head; values turn in LDS, by 4 x 4 bytes.
template <typename T, int D, int NT>
__global__ __launch_bounds__(NT) void kv_read_kernel(typename T::storage* __restrict__ k,
                                                      typename T::storage* __restrict__ v, KvView c, KvBatch b) {
    extern __shared__ __attribute__((aligned(16))) uint8_t turn[];  // values: [token][D + 4]
    const int tid = threadIdx.x, head = blockIdx.y, log2_page = c.log2_page, page_tokens = 1 << log2_page;
    const bool values = blockIdx.z != 0;
    int entry, place;
    if (!kv_locate(b, blockIdx.x, [&](int n) { return kv_spanned(n, log2_page); }, entry, place)) return;
    const KvEntry e = kv_entry(c, b, entry);
    const KvSpan s = kv_span(c, e, place);
    if (s.from >= s.until) return;
    typename T::storage* out = (values ? v : k) + (int64_t(s.row) * c.kv_heads + head) * D;
    const int64_t stride = int64_t(c.kv_heads) * D;
    constexpr int groups = D / 8, pitch = D + 4;
    const int items = (s.until - s.from) * groups;
    const bool here = s.page >= 0;
    const int64_t at = (int64_t(here ? s.page : 0) * c.kv_heads + head);
    const int8_t* codes = (values ? c.v : c.k) + at * page_tokens * D;
    const float scale = here ? e8m0_to_f32((values ? c.vs : c.ks)[at]) : 0.f;
    if (values && here) {
        const int first = s.from >> 4, blocks = ((s.until + 15) >> 4) - first;
        for (int it = tid; it < blocks * (D / 4); it += NT) {
            const int d4 = it / blocks, t0 = (first + it - d4 * blocks) * 16;
            const int8_t* p = codes + int64_t(4 * d4) * page_tokens + t0;
            uint4 o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = *reinterpret_cast<const uint4*>(p + i * page_tokens);
            const uint32_t w[4][4] = {{o[0].x, o[0].y, o[0].z, o[0].w}, {o[1].x, o[1].y, o[1].z, o[1].w},
                                      {o[2].x, o[2].y, o[2].z, o[2].w}, {o[3].x, o[3].y, o[3].z, o[3].w}};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint32_t row[4];
                kv_turn4(w[0][q], w[1][q], w[2][q], w[3][q], row);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = t0 + 4 * q + i;
                    if (t >= s.from && t < s.until) *reinterpret_cast<uint32_t*>(turn + (t - s.from) * pitch + 4 * d4) = row[i];
                }
            }
        }
        __syncthreads();
    }
    constexpr int kAtOnce = 4;  // pieces of 8 codes a thread requests before it writes one
    for (int base = tid; base < items; base += kAtOnce * NT) {
        uint2 w[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int it = base + NT * u, t = it / groups, d0 = it % groups * 8;
            w[u] = make_uint2(0u, 0u);
            if (!here || it >= items) continue;
            if (values) {
                const uint32_t* p = reinterpret_cast<const uint32_t*>(turn + t * pitch + d0);
                w[u] = make_uint2(p[0], p[1]);
            } else {
                w[u] = *reinterpret_cast<const uint2*>(codes + (s.from + t) * D + d0);
            }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int it = base + NT * u, t = it / groups, d0 = it % groups * 8;
            if (it >= items) continue;
            alignas(16) typename T::storage o[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                o[i] = to_storage<T>(here ? float(int8_t((i < 4 ? w[u].x : w[u].y) >> (8 * (i & 3)))) * scale : 0.f);
            uint4* to = reinterpret_cast<uint4*>(out + t * stride + d0);
#pragma unroll
            for (int i = 0; i < int(sizeof(o) / 16); i++) to[i] = reinterpret_cast<const uint4*>(o)[i];
        }
    }
}

// ------------------------------------------------------------------ the pages

// What a page kernel works on; the integers live in the call's scratch.
struct KvPages {
    int32_t* tables;
    int32_t* lengths;
    int32_t* refs;
    int32_t* missing;
    int pages, sequences, width, log2_page;
};

// One workgroup of 1024 decides where pages go, the copies and tables follow
// in a launch of their own.
constexpr int kPlanThreads = 1024;

struct KvPlanScratch {
    uint64_t* bits;   // [words]: which pages are live
    int32_t* before;  // [words + 1]: live pages before each word
    int32_t* list;    // [pages]: free pages by rank (extend); holes by rank (compact)
    int32_t* map;     // [pages]: movers by rank, then where pages went (compact); writers (extend)
    int32_t* keeper;  // [pages] (extend); movers (compact)
    int32_t* claim;   // [sequences]
    int32_t* offset;  // [n]: rank of an entry's first page, bit 30: it copies its last one first
    int32_t* moves;   // [2 * max(n, pages)]: (from, to)
    int32_t* count;   // [1]: of moves
};

__device__ __forceinline__ int32_t agent_load(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive sum over the workgroup's threads; `all` gets the total.
__device__ __forceinline__ int block_exclusive(int v, int* red, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(upto, o);
        if (lane >= o) upto += t;
    }
    __syncthreads();  // red of the call before is read
    if (lane == 63) red[wave] = upto;
    __syncthreads();
    int base = 0;
    all = 0;
    for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w < wave) base += red[w];
        all += red[w];
    }
    return base + upto - v;
}

// Which pages are live, and how many before each word of 64; returns their number.
__device__ __forceinline__ int kv_survey(const KvPages& c, uint64_t* bits, int32_t* before, int* red) {
    const int words = (c.pages + 63) >> 6, lane = threadIdx.x & 63;
    for (int w = threadIdx.x >> 6; w < words; w += kPlanThreads / 64) {
        const int p = w * 64 + lane;
        const uint64_t live = __ballot(p < c.pages && c.refs[p] > 0);
        if (lane == 0) bits[w] = live;
    }
    __syncthreads();
    int carry = 0;
    for (int base = 0; base < words; base += kPlanThreads) {
        const int w = base + threadIdx.x;
        int all;
        const int ex = block_exclusive(w < words ? __popcll(bits[w]) : 0, red, all);
        if (w < words) before[w] = carry + ex;
        carry += all;
    }
    __syncthreads();
    return carry;
}

__device__ __forceinline__ int live_before(const uint64_t* bits, const int32_t* before, int p) {
    return before[p >> 6] + __popcll(bits[p >> 6] & ((uint64_t(1) << (p & 63)) - 1));
}

// The free pages of rank below `most`, in order.
__device__ __forceinline__ void kv_list_free(const KvPages& c, const uint64_t* bits, const int32_t* before, int most, int32_t* list) {
    for (int p = threadIdx.x; p < c.pages; p += kPlanThreads) {
        if (bits[p >> 6] >> (p & 63) & 1) continue;
        const int rank = p - live_before(bits, before, p);
        if (rank < most) list[rank] = p;
    }
}

// An entry's sequence and growth, false where it does nothing: no such
// sequence, no tokens, or a later entry names it too.
__device__ __forceinline__ bool kv_grows(const KvPages& c, const KvBatch& b, const KvPlanScratch& s, int i, int& seq,
                                         int& length, int& count) {
    int start;
    kv_rows(b, i, start, count);
    seq = b.seqs[i];
    if (unsigned(seq) >= unsigned(c.sequences) || count <= 0 || agent_load(s.claim + seq) != i) return false;
    length = kv_clamp(c.lengths[seq], 0, kKvMaxLength);
    count = min(count, kKvMaxLength - length);
    return true;
}

// The page that holds a sequence's last token if there is room behind it.
__device__ __forceinline__ int kv_open_page(const KvPages& c, int seq, int length) {
    const int index = length >> c.log2_page;
    if ((length & ((1 << c.log2_page) - 1)) == 0 || index >= c.width) return -1;
    const int id = c.tables[int64_t(seq) * c.width + index];
    return unsigned(id) < unsigned(c.pages) ? id : -1;
}

// Adds to the cache's count, which stays where an int ends (2^16 entries may each lack 2^26 pages).
__device__ __forceinline__ void kv_count_missing(const KvPages& c, uint64_t lack) {
    if (lack) *c.missing = int32_t(min(uint64_t(max(*c.missing, 0)) + lack, uint64_t(INT32_MAX)));
}

// Gives an entry its pages, free ones from rank `at` on (list: by rank); from: the page it copies first, or -1.
__device__ __forceinline__ void kv_grow(const KvPages& c, const KvPlanScratch& s, int seq, int length, int count, int from, int at,
                                        int free_pages, const int32_t* list, int* copies, uint64_t* lack) {
    const int T = 1 << c.log2_page;
    int32_t* row = c.tables + int64_t(seq) * c.width;
    int none = 0;
    if (from >= 0) {
        const int to = at < free_pages ? list[at] : -1;
        at++;
        if (to >= 0) {
            const int m = atomicAdd(copies, 1);
            s.moves[2 * m] = from;
            s.moves[2 * m + 1] = to;
            c.refs[to] = 1;
        } else {
            none++;
        }
        atomicSub(c.refs + from, 1);
        row[length >> c.log2_page] = to;
    }
    const int have = (length + T - 1) >> c.log2_page, need = (length + count + T - 1) >> c.log2_page;
    for (int w = have; w < min(need, c.width); w++, at++) {
        const int page = at < free_pages ? list[at] : -1;
        if (page >= 0) c.refs[page] = 1;
        else none++;
        row[w] = page;
    }
    none += need - max(have, min(need, c.width));
    c.lengths[seq] = length + count;
    if (none) atomicAdd(reinterpret_cast<unsigned long long*>(lack), (unsigned long long)none);
}

__global__ __launch_bounds__(kPlanThreads) void kv_extend_plan_kernel(KvPages c, KvBatch b, KvPlanScratch s) {
    __shared__ int red[kPlanThreads / 64];
    __shared__ uint64_t lack;
    __shared__ int copies;
    const int tid = threadIdx.x, T = 1 << c.log2_page;
    if (tid == 0) lack = 0, copies = 0;
    int32_t* writers = s.map;
    // of the entries that name a sequence the last counts
    for (int i = tid; i < b.n; i += kPlanThreads) {
        const int seq = b.seqs[i];
        if (unsigned(seq) >= unsigned(c.sequences)) continue;
        s.claim[seq] = -1;
        const int open = kv_open_page(c, seq, kv_clamp(c.lengths[seq], 0, kKvMaxLength));
        if (open >= 0) writers[open] = 0, s.keeper[open] = -1;
    }
    __syncthreads();
    for (int i = tid; i < b.n; i += kPlanThreads)
        if (unsigned(b.seqs[i]) < unsigned(c.sequences)) atomicMax(s.claim + b.seqs[i], i);
    __syncthreads();
    // who writes to a shared page, and the last of them (sums and maxima: any order gives the same)
    for (int i = tid; i < b.n; i += kPlanThreads) {
        int seq, length, count;
        if (!kv_grows(c, b, s, i, seq, length, count)) continue;
        const int open = kv_open_page(c, seq, length);
        if (open >= 0) {
            atomicAdd(writers + open, 1);
            atomicMax(s.keeper + open, i);
        }
    }
    const int live = kv_survey(c, s.bits, s.before, red), free_pages = c.pages - live;
    // how many pages each entry takes, and from which free one on
    int carry = 0;
    for (int base = 0; base < b.n; base += kPlanThreads) {
        const int i = base + tid;
        int seq, length, count, take = 0;
        bool copy = false;
        if (i < b.n && kv_grows(c, b, s, i, seq, length, count)) {
            const int open = kv_open_page(c, seq, length);
            copy = open >= 0 && (c.refs[open] > agent_load(writers + open) || agent_load(s.keeper + open) != i);
            take = min((length + count + T - 1) >> c.log2_page, c.width) - min((length + T - 1) >> c.log2_page, c.width) +
                   (copy ? 1 : 0);
        }
        int all;
        const int at = carry + block_exclusive(take, red, all);
        if (i < b.n) s.offset[i] = min(at, kKvMaxLength - 1) | (copy ? 1 << 30 : 0);
        carry = min(carry, kKvMaxLength - all) + all;
    }
    kv_list_free(c, s.bits, s.before, carry, s.list);
    __syncthreads();
    for (int i = tid; i < b.n; i += kPlanThreads) {
        int seq, length, count;
        if (!kv_grows(c, b, s, i, seq, length, count)) continue;
        kv_grow(c, s, seq, length, count, s.offset[i] >> 30 ? kv_open_page(c, seq, length) : -1, s.offset[i] & ((1 << 30) - 1), free_pages, s.list, &copies, &lack);
    }
    __syncthreads();
    if (tid == 0) {
        s.count[0] = copies;
        kv_count_missing(c, lack);
    }
}

// The same for few entries and pages, an entry a thread: who names a sequence
// last and who writes to a page is found by looking through the entries in LDS, and pages are
// counted and listed there, so that nothing goes to memory and back but what the
// tables say (16 entries: 6.0 us, the kernel above 7.4; compaction's plan likewise 2.9 and 4.6).
constexpr int kFewEntries = 256, kFewPages = 64 * kPlanThreads, kFewTaken = 4096;

__global__ __launch_bounds__(kPlanThreads) void kv_extend_few_kernel(KvPages c, KvBatch b, KvPlanScratch s) {
    __shared__ int red[kPlanThreads / 64];
    __shared__ uint64_t lack;
    __shared__ int copies;
    __shared__ uint64_t bits[kFewPages / 64];
    __shared__ int32_t before[kFewPages / 64], seqs[kFewEntries], opens[kFewEntries], list[kFewTaken];
    const int tid = threadIdx.x, T = 1 << c.log2_page;
    if (tid == 0) lack = 0, copies = 0;
    int seq = -1, length = 0, count = 0, open = -1, refs = 0;
    if (tid < b.n) {
        int start;
        kv_rows(b, tid, start, count);
        seq = b.seqs[tid];
        if (unsigned(seq) >= unsigned(c.sequences)) seq = -1;
        if (seq >= 0) {
            length = kv_clamp(c.lengths[seq], 0, kKvMaxLength);
            open = kv_open_page(c, seq, length);
            if (open >= 0) refs = c.refs[open];
        }
        seqs[tid] = seq;
    }
    const int free_pages = c.pages - kv_survey(c, bits, before, red);
    bool grows = seq >= 0 && count > 0;
    if (grows)
        for (int j = tid + 1; j < b.n; j++) grows &= seqs[j] != seq;
    count = min(count, kKvMaxLength - length);
    if (tid < b.n) opens[tid] = grows ? open : -1;
    __syncthreads();
    bool copy = false;
    int take = 0;
    if (grows) {
        if (open >= 0) {
            int writers = 0, keeper = 0;
            for (int j = 0; j < b.n; j++)
                if (opens[j] == open) writers++, keeper = j;
            copy = refs > writers || keeper != tid;
        }
        take = min((length + count + T - 1) >> c.log2_page, c.width) - min((length + T - 1) >> c.log2_page, c.width) + (copy ? 1 : 0);
    }
    int all;
    const int at = block_exclusive(take, red, all);
    const bool near = all <= kFewTaken;
    if (near) kv_list_free(c, bits, before, all, list);
    else kv_list_free(c, bits, before, all, s.list);
    __syncthreads();
    if (grows) {
        if (near) kv_grow(c, s, seq, length, count, copy ? open : -1, at, free_pages, list, &copies, &lack);
        else kv_grow(c, s, seq, length, count, copy ? open : -1, at, free_pages, s.list, &copies, &lack);
    }
    __syncthreads();
    if (tid == 0) {
        s.count[0] = copies;
        kv_count_missing(c, lack);
    }
}

template <bool kFew>
__global__ __launch_bounds__(kPlanThreads) void kv_compact_plan_kernel(KvPages c, KvPlanScratch s) {
    __shared__ int red[kPlanThreads / 64];
    __shared__ uint64_t near_bits[kFew ? kFewPages / 64 : 1];
    __shared__ int32_t near_before[kFew ? kFewPages / 64 : 1];
    uint64_t* bits = kFew ? near_bits : s.bits;
    int32_t* before = kFew ? near_before : s.before;
    const int tid = threadIdx.x, live = kv_survey(c, bits, before, red);
    const int stay = live < c.pages ? live_before(bits, before, live) : live;  // live pages before page `live`
    int32_t* movers = s.keeper;
    for (int p = tid; p < c.pages; p += kPlanThreads) {
        const bool is = bits[p >> 6] >> (p & 63) & 1;
        const int rank = live_before(bits, before, p);
        s.map[p] = p;
        if (is && p >= live) movers[rank - stay] = p;
        if (!is && p < live) s.list[p - rank] = p;
    }
    __syncthreads();
    for (int r = tid; r < live - stay; r += kPlanThreads) {
        const int from = movers[r], to = s.list[r];
        s.map[from] = to;
        s.moves[2 * r] = from;
        s.moves[2 * r + 1] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (tid == 0) s.count[0] = live - stay;
}

// Copies the pages of the move list, all layers, 16 KiB a step; then (map not
// null) the tables' entries follow their pages.  (Loads that pass the caches by take 335 MB, read and written, in
// 65 us and 15 copies of one page in 21, these 50 and 13: a page is read more than once.  32 KiB a step: 53.)
constexpr int kMoveStep = 16384;
__global__ __launch_bounds__(256) void kv_move_kernel(KvPages c, int8_t* k, int8_t* v, uint8_t* ks, uint8_t* vs,
                                                      int layers, int kv_heads, int64_t page_bytes,
                                                      const int32_t* __restrict__ moves,
                                                      const int32_t* __restrict__ count,
                                                      const int32_t* __restrict__ map) {
    constexpr int kVecs = kMoveStep / 4096;
    const int steps = int((page_bytes + kMoveStep - 1) / kMoveStep), tid = threadIdx.x;
    const int64_t units = int64_t(*count) * layers * 2 * steps;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int step = int(u % steps), half = int(u / steps % 2);
        const int64_t ml = u / steps / 2, layer = ml % layers;
        const int m = int(ml / layers);
        const int64_t from = layer * c.pages + moves[2 * m], to = layer * c.pages + moves[2 * m + 1];
        int8_t* codes = half ? v : k;
        const uint4* src = reinterpret_cast<const uint4*>(codes + from * page_bytes + int64_t(step) * kMoveStep);
        uint4* dst = reinterpret_cast<uint4*>(codes + to * page_bytes + int64_t(step) * kMoveStep);
        const int vecs = int(min(int64_t(kMoveStep), page_bytes - int64_t(step) * kMoveStep) / 16);
        uint4 t[kVecs];
        if (vecs == kMoveStep / 16) {
#pragma unroll
            for (int i = 0; i < kVecs; i++) t[i] = src[tid + 256 * i];
#pragma unroll
            for (int i = 0; i < kVecs; i++) store_stream16(dst + tid + 256 * i, t[i]);
        } else {
            for (int i = tid; i < vecs; i += 256) dst[i] = src[i];
        }
        if (step == 0) {
            uint8_t* scales = half ? vs : ks;
            for (int h = tid; h < kv_heads; h += 256) scales[to * kv_heads + h] = scales[from * kv_heads + h];
        }
    }
    if (!map) return;
    const int64_t entries = int64_t(c.sequences) * c.width;
    for (int64_t i = int64_t(blockIdx.x) * 256 + tid; i < entries; i += int64_t(gridDim.x) * 256) {
        const int id = c.tables[i];
        if (unsigned(id) < unsigned(c.pages) && map[id] != id) c.tables[i] = map[id];
    }
}

// One workgroup per pair: the source's row and length as they are, and one
// reference more for each of its pages.
__global__ __launch_bounds__(256) void kv_fork_take_kernel(KvPages c, const int32_t* __restrict__ src,
                                                           const int32_t* __restrict__ dst, int n, int32_t* rows) {
    const int i = blockIdx.x, from = src[i], to = dst[i], tid = threadIdx.x;
    bool later = false;
    for (int j = i + 1 + tid; j < n; j += 256) later |= dst[j] == to;
    const bool off = __syncthreads_or(later) || unsigned(from) >= unsigned(c.sequences) ||
                     unsigned(to) >= unsigned(c.sequences);
    int32_t* row = rows + int64_t(i) * (c.width + 1);
    if (tid == 0) row[c.width] = off ? -1 : kv_clamp(c.lengths[from], 0, kKvMaxLength);
    if (off) return;
    for (int w = tid; w < c.width; w += 256) {
        const int id = c.tables[int64_t(from) * c.width + w];
        row[w] = id;
        if (unsigned(id) < unsigned(c.pages)) atomicAdd(c.refs + id, 1);
    }
}

__global__ __launch_bounds__(256) void kv_fork_give_kernel(KvPages c, const int32_t* __restrict__ dst,
                                                           const int32_t* __restrict__ rows) {
    const int i = blockIdx.x, to = dst[i];
    const int32_t* row = rows + int64_t(i) * (c.width + 1);
    if (row[c.width] < 0) return;
    for (int w = threadIdx.x; w < c.width; w += 256) {
        const int old = c.tables[int64_t(to) * c.width + w];
        if (unsigned(old) < unsigned(c.pages)) atomicSub(c.refs + old, 1);
        c.tables[int64_t(to) * c.width + w] = row[w];
    }
    if (threadIdx.x == 0) c.lengths[to] = row[c.width];
}

// Both in one launch where one workgroup holds all pairs' rows (the wait between two
// launches is most of their time: 15 pairs of 31 pages 3.7 us, 6.1 in two).
constexpr int kFewRows = 4096;

__global__ __launch_bounds__(kPlanThreads) void kv_fork_few_kernel(KvPages c, const int32_t* __restrict__ src,
                                                                   const int32_t* __restrict__ dst, int n) {
    constexpr int EACH = kFewRows / kPlanThreads;
    __shared__ int32_t from[kFewEntries], to[kFewEntries];
    const int tid = threadIdx.x;
    int mine = -1, length = 0;
    if (tid < n) {
        mine = src[tid], to[tid] = dst[tid];
        if (unsigned(mine) >= unsigned(c.sequences) || unsigned(to[tid]) >= unsigned(c.sequences)) mine = -1;
        if (mine >= 0) length = kv_clamp(c.lengths[mine], 0, kKvMaxLength);
    }
    __syncthreads();
    if (tid < n) {
        for (int j = tid + 1; j < n; j++)
            if (to[j] == to[tid]) mine = -1;
        from[tid] = mine;
    }
    __syncthreads();
    int32_t *at[EACH], id[EACH];
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const int it = tid + k * kPlanThreads, i = it / c.width, w = it - i * c.width;
        at[k] = nullptr;
        if (i >= n || from[i] < 0) continue;
        at[k] = c.tables + int64_t(to[i]) * c.width + w;
        id[k] = c.tables[int64_t(from[i]) * c.width + w];
        const int old = *at[k];
        if (unsigned(id[k]) < unsigned(c.pages)) atomicAdd(c.refs + id[k], 1);
        if (unsigned(old) < unsigned(c.pages)) atomicSub(c.refs + old, 1);
    }
    __syncthreads();  // every row and length is read
#pragma unroll
    for (int k = 0; k < EACH; k++)
        if (at[k]) *at[k] = id[k];
    if (mine >= 0) c.lengths[to[tid]] = length;
}

// One workgroup per entry: the length, and the pages behind the tokens that stay.
__global__ __launch_bounds__(256) void kv_shrink_kernel(KvPages c, const int32_t* __restrict__ seqs,
                                                        const int32_t* __restrict__ counts, int count, int n) {
    const int i = blockIdx.x, seq = seqs[i], tid = threadIdx.x, T = 1 << c.log2_page;
    bool later = false;
    for (int j = i + 1 + tid; j < n; j += 256) later |= seqs[j] == seq;
    const bool is = unsigned(seq) < unsigned(c.sequences);
    const int length = is ? kv_clamp(c.lengths[seq], 0, kKvMaxLength) : 0;
    if (__syncthreads_or(later) || !is) return;  // (and every thread has the length)
    const int rest = length - kv_clamp(counts ? counts[i] : count, 0, length);
    int32_t* row = c.tables + int64_t(seq) * c.width;
    for (int w = ((rest + T - 1) >> c.log2_page) + tid; w < c.width; w += 256) {
        const int id = row[w];
        if (unsigned(id) < unsigned(c.pages)) atomicSub(c.refs + id, 1);
        row[w] = -1;
    }
    if (tid == 0) c.lengths[seq] = rest;
}

// One workgroup per sequence; the exchange lets one of several entries that
// name a sequence give up each page.
__global__ __launch_bounds__(256) void kv_free_kernel(KvPages c, const int32_t* __restrict__ seqs) {
    const int seq = seqs[blockIdx.x];
    if (unsigned(seq) >= unsigned(c.sequences)) return;
    for (int w = threadIdx.x; w < c.width; w += 256) {
        const int id = atomicExch(c.tables + int64_t(seq) * c.width + w, -1);
        if (unsigned(id) < unsigned(c.pages)) atomicSub(c.refs + id, 1);
    }
    if (threadIdx.x == 0) c.lengths[seq] = 0;
}

KvPages pages_of(const eq_kv_cache* c) {
    return KvPages{c->tables,           c->lengths,       c->refs,          c->missing, int(c->pages),
                   int(c->sequences), int(c->width), __builtin_ctz(unsigned(c->page_tokens))};
}

// The plan's arrays in `base` (null: only their size).
size_t plan_scratch(const eq_kv_cache* c, int64_t n, char* base, KvPlanScratch* s) {
    size_t at = 0;
    auto take = [&](auto*& p, int64_t count) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
        at += (size_t(count) * sizeof(*p) + 255) & ~size_t(255);
    };
    KvPlanScratch t;
    const int64_t words = (c->pages + 63) / 64;
    take(t.bits, words);
    take(t.before, words + 1);
    take(t.list, c->pages);
    take(t.map, c->pages);
    take(t.keeper, c->pages);
    take(t.claim, c->sequences);
    take(t.offset, n);
    take(t.moves, 2 * (n > c->pages ? n : c->pages));
    take(t.count, 1);
    if (s) *s = t;
    return at;
}

size_t pages_scratch_bytes(const eq_kv_cache* c, int64_t n) {
    const size_t plan = plan_scratch(c, n, nullptr, nullptr), fork = size_t(n) * size_t(c->width + 1) * 4;
    return plan > fork ? plan : fork;
}

char* scratch_for(WsHold& hold, const char* who, void* scratch, int64_t scratch_bytes, size_t need, hipStream_t st) {
    if (scratch) {
        if (scratch_bytes < 0 || size_t(scratch_bytes) < need || !aligned(scratch, 256)) {
            set_error(std::string(who) + ": needs " + std::to_string(need) + " bytes of 256-byte aligned scratch");
            return nullptr;
        }
        return static_cast<char*>(scratch);
    }
    void* p = ws_acquire(hold, nullptr, need, st);
    if (!p)
        set_error(std::string(who) + ": no workspace (its stream's workspace cannot grow while capturing: pass "
                  "scratch, or make one such call on the stream before capturing)");
    return static_cast<char*>(p);
}

bool kv_count_ok(const char* who, int64_t n) {
    if (n >= 0 && n <= kKvMaxEntries) return true;
    set_error(std::string(who) + ": need 0 <= n <= 2^16");
    return false;
}

bool kv_list_ok(const char* who, const int32_t* a, const int32_t* b, int64_t n) {
    if (!kv_count_ok(who, n)) return false;
    if (n > 0 && (!a || !b)) {
        set_error(std::string(who) + ": null pointer argument");
        return false;
    }
    return true;
}

// Head dimension and threads of a workgroup that has one page of one head: as many
// as a page has 16-byte pieces (10000 tokens in pages of 16, 128 dimensions: append 20 us with 128 threads, 29 with
// 256, read 16 and 21; in pages of 64 with 128 threads read 15, with 256 14).
template <typename F>
void with_page(const eq_kv_cache* c, F f) {
    const int pieces = c->page_tokens * c->head_dim / 16;
    auto threads = [&](auto d) {  // (the smallest page, of 16 tokens, has as many pieces as the head has dimensions)
        constexpr int D = decltype(d)::value;
        if constexpr (D <= 64) {
            if (pieces <= 64) return f(d, std::integral_constant<int, 64>{});
        }
        if constexpr (D <= 128) {
            if (pieces <= 128) return f(d, std::integral_constant<int, 128>{});
        }
        f(d, std::integral_constant<int, 256>{});
    };
    if (c->head_dim == 64) threads(std::integral_constant<int, 64>{});
    else if (c->head_dim == 128) threads(std::integral_constant<int, 128>{});
    else threads(std::integral_constant<int, 256>{});
}

// Of at most `moves` pages.
void launch_moves(const eq_kv_cache* c, const KvPlanScratch& s, int64_t moves, const int32_t* map, hipStream_t st) {
    // (no more workgroups than a small cache has work for: a launch that moves nothing is a launch)
    const int64_t page = int64_t(c->kv_heads) * c->page_tokens * c->head_dim, entries = map ? c->sequences * c->width / 1024 : 0;
    const int64_t steps = (moves < c->pages ? moves : c->pages) * c->layers * 2 * ((page + kMoveStep - 1) / kMoveStep);
    const int64_t most = steps > entries ? steps : entries + 1, grid = most < 8192 ? most : 8192;
    kv_move_kernel<<<dim3(unsigned(grid)), dim3(256), 0, st>>>(pages_of(c), c->k_codes, c->v_codes, c->k_scales, c->v_scales,
                                                     int(c->layers), c->kv_heads,
                                                     int64_t(c->kv_heads) * c->page_tokens * c->head_dim, s.moves,
                                                     s.count, map);
}

}  // namespace
}  // namespace eq

using namespace eq;

extern "C" int eq_kv_append(const eq_kv_cache* cache, int64_t layer, const void* k, const void* v, int64_t k_stride,
                            int64_t v_stride, const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total,
                            const float* rope, int64_t rope_positions, int dtype, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_append";
    if (!kv_cache_ok(who, cache) || !kv_batch_ok(who, cache, layer, seqs, n, cu, total) ||
        !kv_rope_ok(who, cache, rope, rope_positions))
        return 1;
    if (dtype != EQ_DTYPE_BF16 && dtype != EQ_DTYPE_F16) {
        set_error("eq_kv_append: k and v must be bfloat16 or float16");
        return 1;
    }
    if (n == 0 || total == 0) return 0;
    if (!k || !v) {
        set_error("eq_kv_append: null pointer argument");
        return 1;
    }
    const int D = cache->head_dim;
    const int64_t row = int64_t(cache->kv_heads) * D;
    if (!aligned(k, 16) || !aligned(v, 16) || k_stride % 8 || v_stride % 8 || k_stride < row || v_stride < row) {
        set_error("eq_kv_append: k and v must be 16-byte aligned, their row strides multiples of 8 and at least "
                  "kv_heads * head_dim");
        return 1;
    }
    const KvView c = kv_view(cache, layer);
    const KvBatch b = kv_batch(seqs, n, cu, total);
    const int64_t units = kv_page_units(b, c.log2_page);
    if (units >= (1 << 24)) {  // a grid of under 2^32 threads
        set_error("eq_kv_append: too many rows");
        return 1;
    }
    const size_t lds = size_t(cache->page_tokens) * (D + 4);
    const dim3 grid(unsigned(units), unsigned(cache->kv_heads), 2);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto of = [&](auto t) {
        typedef decltype(t) T;
        with_page(cache, [&](auto d, auto nt) {
            kv_append_kernel<T, decltype(d)::value, decltype(nt)::value><<<grid, dim3(decltype(nt)::value), lds, st>>>(
                c, b, static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_stride, v_stride, rope);
        });
    };
    if (dtype == EQ_DTYPE_BF16) of(BF16T{});
    else of(F16T{});
    return check_launch(who);
}

extern "C" int eq_kv_read(void* k, void* v, const eq_kv_cache* cache, int64_t layer, const int32_t* seqs, int64_t n,
                          const int32_t* cu, int64_t total, int dtype, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_read";
    if (!kv_cache_ok(who, cache) || !kv_batch_ok(who, cache, layer, seqs, n, cu, total)) return 1;
    if (!valid_dtype(dtype)) {
        set_error("eq_kv_read: invalid dtype code");
        return 1;
    }
    if (n == 0 || total == 0) return 0;
    if (!k || !v || !aligned(k, 16) || !aligned(v, 16)) {
        set_error("eq_kv_read: k and v must be 16-byte aligned");
        return 1;
    }
    const KvView c = kv_view(cache, layer);
    const KvBatch b = kv_batch(seqs, n, cu, total);
    const int64_t units = kv_page_units(b, c.log2_page);
    if (units >= (1 << 24)) {  // a grid of under 2^32 threads
        set_error("eq_kv_read: too many rows");
        return 1;
    }
    const int D = cache->head_dim;
    const size_t lds = size_t(cache->page_tokens) * (D + 4);
    const dim3 grid(unsigned(units), unsigned(cache->kv_heads), 2);
    with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        with_page(cache, [&](auto d, auto nt) {
            kv_read_kernel<T, decltype(d)::value, decltype(nt)::value>
                <<<grid, dim3(decltype(nt)::value), lds, reinterpret_cast<hipStream_t>(stream)>>>(
                    static_cast<typename T::storage*>(k), static_cast<typename T::storage*>(v), c, b);
        });
    });
    return check_launch(who);
}

extern "C" int64_t eq_kv_pages_scratch(const eq_kv_cache* cache, int64_t n) {
    clear_error();
    if (!kv_cache_ok("eq_kv_pages_scratch", cache) || !kv_count_ok("eq_kv_pages_scratch", n))
        return -1;
    return int64_t(pages_scratch_bytes(cache, n));
}

extern "C" int eq_kv_extend(const eq_kv_cache* cache, const int32_t* seqs, int64_t n, const int32_t* cu, int64_t count,
                            void* scratch, int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_extend";
    if (!kv_cache_ok(who, cache) || !kv_list_ok(who, seqs, seqs, n)) return 1;
    if (!cu && (count < 0 || count > kKvMaxLength)) {
        set_error("eq_kv_extend: count must be in [0, 2^30]");
        return 1;
    }
    if (n == 0 || (!cu && count == 0)) return 0;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    WsHold hold;
    char* base = scratch_for(hold, who, scratch, scratch_bytes, pages_scratch_bytes(cache, n), st);
    if (!base) return 1;
    KvPlanScratch s;
    plan_scratch(cache, n, base, &s);
    const KvBatch b{seqs, cu, int(n), int(count), INT32_MAX};
    if (n <= kFewEntries && cache->pages <= kFewPages) kv_extend_few_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(pages_of(cache), b, s);
    else kv_extend_plan_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(pages_of(cache), b, s);
    launch_moves(cache, s, n, nullptr, st);
    return check_launch(who);
}

extern "C" int eq_kv_fork(const eq_kv_cache* cache, const int32_t* src, const int32_t* dst, int64_t n, void* scratch,
                          int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_fork";
    if (!kv_cache_ok(who, cache) || !kv_list_ok(who, src, dst, n)) return 1;
    if (n == 0) return 0;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    WsHold hold;
    char* base = scratch_for(hold, who, scratch, scratch_bytes, pages_scratch_bytes(cache, n), st);
    if (!base) return 1;
    int32_t* rows = reinterpret_cast<int32_t*>(base);
    const KvPages c = pages_of(cache);
    if (n <= kFewEntries && n * cache->width <= kFewRows) {
        kv_fork_few_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(c, src, dst, int(n));
    } else {
        kv_fork_take_kernel<<<dim3(unsigned(n)), dim3(256), 0, st>>>(c, src, dst, int(n), rows);
        kv_fork_give_kernel<<<dim3(unsigned(n)), dim3(256), 0, st>>>(c, dst, rows);
    }
    return check_launch(who);
}

extern "C" int eq_kv_shrink(const eq_kv_cache* cache, const int32_t* seqs, int64_t n, const int32_t* counts, int64_t count,
                            eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_shrink";
    if (!kv_cache_ok(who, cache) || !kv_list_ok(who, seqs, seqs, n)) return 1;
    if (!counts && (count < 0 || count > kKvMaxLength)) {
        set_error("eq_kv_shrink: count must be in [0, 2^30]");
        return 1;
    }
    if (n == 0) return 0;
    kv_shrink_kernel<<<dim3(unsigned(n)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream)>>>(pages_of(cache), seqs, counts,
                                                                                                 int(count), int(n));
    return check_launch(who);
}

extern "C" int eq_kv_free(const eq_kv_cache* cache, const int32_t* seqs, int64_t n, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_free";
    if (!kv_cache_ok(who, cache) || !kv_list_ok(who, seqs, seqs, n)) return 1;
    if (n == 0) return 0;
    kv_free_kernel<<<dim3(unsigned(n)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream)>>>(pages_of(cache), seqs);
    return check_launch(who);
}

extern "C" int eq_kv_compact(const eq_kv_cache* cache, void* scratch, int64_t scratch_bytes, eq_stream_t stream) {
    clear_error();
    const char* who = "eq_kv_compact";
    if (!kv_cache_ok(who, cache)) return 1;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    WsHold hold;
    char* base = scratch_for(hold, who, scratch, scratch_bytes, pages_scratch_bytes(cache, 0), st);
    if (!base) return 1;
    KvPlanScratch s;
    plan_scratch(cache, 0, base, &s);
    if (cache->pages <= kFewPages) kv_compact_plan_kernel<true><<<dim3(1), dim3(kPlanThreads), 0, st>>>(pages_of(cache), s);
    else kv_compact_plan_kernel<false><<<dim3(1), dim3(kPlanThreads), 0, st>>>(pages_of(cache), s);
    launch_moves(cache, s, cache->pages, s.map, st);
    return check_launch(who);
}

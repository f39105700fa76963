// Attention over the paged 8-bit key/value cache (kv_common.hpp has the
// format, include/eredu_kv.h the rules).
#include <math.h>

#include "kv_common.hpp"

namespace eq {
namespace {

// One workgroup per row and query head: 256 tokens a step, a thread each for
// the scores, then a thread for each dimension for the values.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_attention_simple_kernel(uint16_t* __restrict__ out, const uint16_t* __restrict__ q,
                                                          int64_t q_stride, KvView c, KvBatch b, float scale,
                                                          bool causal, int64_t window, const float* __restrict__ rope,
                                                          int heads) {
    __shared__ float qs[D], p[256], vs[256];
    __shared__ float red[8];
    const int tid = threadIdx.x, h = blockIdx.y, kvh = h / (heads / c.kv_heads), T0 = 1 << c.log2_page;
    int entry, place;
    if (!kv_locate(b, blockIdx.x, [](int n) { return n; }, entry, place)) return;
    const KvEntry e = kv_entry(c, b, entry);
    const int row = e.start + place, pos = e.length - e.count + place;
    for (int d = tid; d < D / 2; d += 256) {
        const uint16_t* x = q + int64_t(row) * q_stride + int64_t(h) * D;
        float u = kv_to_f32<T>(x[d]), v = kv_to_f32<T>(x[d + D / 2]);
        if (rope && pos >= 0) {
            const float cs = rope[int64_t(pos) * D + d], sn = rope[int64_t(pos) * D + D / 2 + d];
            const float t = u * cs - v * sn;
            v = v * cs + u * sn;
            u = t;
        }
        qs[d] = u, qs[d + D / 2] = v;
    }
    __syncthreads();
    const int len = min(e.length, c.width << c.log2_page);
    const int hi = causal ? min(pos + 1, len) : len;
    const int lo = causal && window > 0 ? int(max(int64_t(0), int64_t(pos) + 1 - window)) : 0;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int base = lo / 256 * 256; base < hi; base += 256) {
        const int j = base + tid;
        const int page = j >= lo && j < hi ? kv_page(c, e.seq, j >> c.log2_page) : -1;
        float s = -INFINITY;
        vs[tid] = 0.f;
        if (page >= 0) {
            const int64_t at = int64_t(page) * c.kv_heads + kvh;
            const int8_t* kr = c.k + (at * T0 + (j & (T0 - 1))) * D;
            float a = 0.f;
            for (int d = 0; d < D; d++) a = fmaf(qs[d], float(kr[d]), a);
            s = a * e8m0_to_f32(c.ks[at]) * scale;
            vs[tid] = e8m0_to_f32(c.vs[at]);
            if (vs[tid] != vs[tid]) s = vs[tid];
        }
        float mx = s;
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float al = m == mn ? 1.f : expf(m - mn);
        const float pe = page >= 0 ? expf(s - (mn == -INFINITY ? 0.f : mn)) : 0.f;
        p[tid] = pe;
        float sum = pe;
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
        if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
        __syncthreads();
        l = l * al + (red[4] + red[5] + red[6] + red[7]);
        m = mn;
        o *= al;
        if (tid < D) {
            for (int t = max(lo - base, 0); t < min(256, hi - base); t++) {
                const int pg = kv_page(c, e.seq, (base + t) >> c.log2_page);
                if (pg < 0) continue;
                const int64_t at = int64_t(pg) * c.kv_heads + kvh;
                o = fmaf(p[t], vs[t] * float(c.v[(at * D + tid) * T0 + ((base + t) & (T0 - 1))]), o);
            }
        }
        __syncthreads();
    }
    if (tid < D) {
        const float r = l == 0.f ? 0.f : o / l;
        out[(int64_t(row) * heads + h) * D + tid] = to_storage<T>(r);
    }
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

}  // namespace
}  // namespace eq

using namespace eq;

extern "C" int64_t eq_kv_attention_scratch(const eq_kv_cache* cache, int n_heads, int64_t n, int64_t total, bool ragged) {
    clear_error();
    const char* who = "eq_kv_attention_scratch";
    if (!kv_cache_ok(who, cache) || !attention_sizes_ok(who, cache, n_heads, n, total)) return -1;
    return 0;
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
    const KvView c = kv_view(cache, layer);
    const KvBatch b = kv_batch(seqs, n, cu, total);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto go = [&](auto kern) {
        kern<<<dim3(unsigned(total), unsigned(n_heads)), dim3(256), 0, st>>>(
            static_cast<uint16_t*>(out), static_cast<const uint16_t*>(q), q_stride, c, b, scale, causal, window, rope, n_heads);
    };
    auto with_d = [&](auto t) {
        typedef decltype(t) T;
        if (D == 64) go(kv_attention_simple_kernel<T, 64>);
        else if (D == 128) go(kv_attention_simple_kernel<T, 128>);
        else go(kv_attention_simple_kernel<T, 256>);
    };
    if (dtype == EQ_DTYPE_BF16) with_d(BF16T{});
    else with_d(F16T{});
    return check_launch(who);
}

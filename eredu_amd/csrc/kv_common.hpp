// The paged 8-bit key/value cache: what its kernels share.
//
// A page holds T = 2^t tokens of every layer and KV head: int8 codes, keys as
// [T][D] and values as [D][T] (so that 16 tokens of one dimension are one
// 16-byte load, the operand of P.V), and for keys and values one E8M0 byte b
// each: value = code * 2^(b - 127), b = 255 = NaN.  Powers of two make
// quantizing, growing a page's scale and reading back exact but for the one
// rounding to the code.
//
// Everything read from device memory that is used as an index is checked where
// it is used: a page id outside [0, pages) is a missing page, a sequence id
// outside [0, sequences) is no sequence, lengths and offsets are clamped.
#pragma once

#include "../../include/eredu_kv.h"
#include "eq_common.hpp"

namespace eq {

constexpr int kKvMaxPage = 128;
constexpr int kKvMaxLength = 1 << 30;  // of a sequence, and of width * page
constexpr int kKvMaxEntries = 1 << 16;  // of a call (every workgroup goes through them)

struct KvView {
    int8_t* k;          // this layer's pages
    int8_t* v;
    uint8_t* ks;
    uint8_t* vs;
    const int32_t* tables;
    const int32_t* lengths;
    int pages, sequences, width, kv_heads, log2_page;
};

// The tokens of a call: sequence entry i has rows [start, start + count) and
// its new tokens are the last `count` of its `length` tokens.
struct KvBatch {
    const int32_t* seqs;
    const int32_t* cu;  // null: every entry has `each` rows
    int n, each, total;
};

struct KvEntry {
    int seq, start, count, length;  // seq -1: no sequence (length 0)
};

__device__ __forceinline__ int kv_clamp(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ void kv_rows(const KvBatch& b, int i, int& start, int& count) {
    if (b.cu) {
        start = kv_clamp(b.cu[i], 0, b.total);
        count = kv_clamp(b.cu[i + 1], start, b.total) - start;
    } else {
        start = i * b.each;
        count = b.each;
    }
}

__device__ __forceinline__ KvEntry kv_entry(const KvView& c, const KvBatch& b, int i) {
    KvEntry e;
    kv_rows(b, i, e.start, e.count);
    const int s = b.seqs[i];
    e.seq = unsigned(s) < unsigned(c.sequences) ? s : -1;
    e.length = e.seq >= 0 ? kv_clamp(c.lengths[e.seq], 0, kKvMaxLength) : 0;
    return e;
}

// The entry whose units hold unit `u`, and the unit's place in it; units(count)
// is an entry's number of units.  False past the last one.  All lanes of the
// wave take part and get the same answer (ragged batches: 64 entries a step).
template <typename F>
__device__ __forceinline__ bool kv_locate(const KvBatch& b, int u, F units, int& entry, int& place) {
    if (!b.cu) {
        const int per = units(b.each);
        entry = per ? u / per : b.n;
        place = u - entry * per;
        return entry < b.n;
    }
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < b.n; base += 64) {
        int start, count, mine = 0;
        if (base + lane < b.n) {
            kv_rows(b, base + lane, start, count);
            mine = units(count);
        }
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(upto, o);
            if (lane >= o) upto += t;
        }
        const uint64_t past = __ballot(upto > u);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            entry = __builtin_amdgcn_readfirstlane(base + l);
            place = __builtin_amdgcn_readfirstlane(u - __shfl(upto - mine, l));
            return true;
        }
        u -= __shfl(upto, 63);
    }
    return false;
}

__device__ __forceinline__ int kv_page(const KvView& c, int seq, int index) {
    if (seq < 0 || unsigned(index) >= unsigned(c.width)) return -1;
    const int id = c.tables[int64_t(seq) * c.width + index];
    return unsigned(id) < unsigned(c.pages) ? id : -1;
}

// The same in two halves, so that nothing waits for the entry before it is
// used: the table entry of a page index of a sequence (index >= 0; behind the table: its
// last entry, whose tokens there are not), and the page it names.
__device__ __forceinline__ int kv_page_entry(const KvView& c, int seq, int index) {
    return c.tables[int64_t(seq) * c.width + min(index, c.width - 1)];
}
__device__ __forceinline__ int kv_page_of(const KvView& c, int entry) { return unsigned(entry) < unsigned(c.pages) ? entry : -1; }

template <typename T> __device__ __forceinline__ float kv_to_f32(uint32_t bits);
template <> __device__ __forceinline__ float kv_to_f32<BF16T>(uint32_t b) { return bf16_bits_to_f32(b); }
template <> __device__ __forceinline__ float kv_to_f32<F16T>(uint32_t b) { return f16_bits_to_f32(b); }

// Host side: argument checks of every entry point, and the views they make.
bool kv_cache_ok(const char* who, const eq_kv_cache* c);
bool kv_rows_ok(const char* who, int64_t n, int64_t total, bool even);  // even: no offsets
bool kv_batch_ok(const char* who, const eq_kv_cache* c, int64_t layer, const int32_t* seqs, int64_t n,
                 const int32_t* cu, int64_t total);
bool kv_rope_ok(const char* who, const eq_kv_cache* c, const float* rope, int64_t positions);
KvView kv_view(const eq_kv_cache* c, int64_t layer);
KvBatch kv_batch(const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total);

}  // namespace eq

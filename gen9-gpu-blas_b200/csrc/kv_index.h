// kv_index.h -- index arithmetic of the paged key-value cache, plain functions for host and device alike, so that the
// bounds rules (pages outside the pool, lengths past the table, offsets past 32 bits) are checked on the CPU
// (tests/test_kv_cpu.py compiles this file with the host compiler).
#pragma once
#include <cstdint>
#include <cstring>
#ifdef __CUDACC__
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD static inline
#endif

namespace g9kv {

// Division of 0 <= k < 2^31 by a fixed page size: q = k·mul >> sh with mul = ⌈2^sh / page⌉, sh = 32 + ⌈log2 page⌉, exact for
// all k below 2^31 (mul·page - 2^sh < page <= 2^(sh - 32)); mul < 2^33, so the product stays below 2^64.
struct PageDiv {
    uint64_t mul;
    int sh, page;
};
KV_HD PageDiv page_div(int page) {
    PageDiv d;
    int lg = 0;
    while (((int64_t)1 << lg) < page) lg++;
    d.page = page;
    d.sh = 32 + lg;
    d.mul = lg == 31 ? 0 : ((((uint64_t)1 << d.sh) + (uint64_t)page - 1) / (uint64_t)page);
    if (lg == 31) {          // pages above 2^30 slots: one page spans every slot below it, plain division below
        d.sh = 0;
    }
    return d;
}
KV_HD int page_quot(const PageDiv &d, int k) { return d.sh ? (int)(((uint64_t)(uint32_t)k * d.mul) >> d.sh) : k / d.page; }

// Slots a token sees: [0, seen) with seen = vis + dvis·t held to [0, cap].
KV_HD int seen_slots(int vis, int dvis, int t, int cap) {
    int64_t v = (int64_t)vis + (int64_t)dvis * t;
    if (v < 0) v = 0;
    return v < cap ? (int)v : cap;
}
// The first slot inside a window of `window` slots that ends at `seen` (window 0: none).
KV_HD int first_slot(int seen, int window) { return window > 0 && seen > window ? seen - window : 0; }

// A page number as the kernels use it: -1 unless 0 <= place < mp and the table's entry lies in the pool.
KV_HD int page_id(const int *table, int64_t ts, int s, int place, int mp, int n_pages) {
    if (place < 0 || place >= mp) return -1;
    const int id = table[(int64_t)s * ts + place];
    return id >= 0 && id < n_pages ? id : -1;
}

// Offset of a slot's row in the pool, in elements.
KV_HD int64_t row_at(int id, int slot, int g, int64_t sp, int64_t sk, int64_t sh) {
    return (int64_t)id * sp + (int64_t)slot * sk + (int64_t)g * sh;
}

// Order-preserving bits of a weight (larger weight, larger number): NaN is 0, -0 equals +0, everything below 0xFFFFFFFF.
KV_HD uint32_t weight_key(float w) {
    uint32_t u;
#ifdef __CUDA_ARCH__
    u = __float_as_uint(w);
#else
    std::memcpy(&u, &w, 4);
#endif
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
    if (u == 0x80000000u) u = 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// The same for a page score in 64 bits: NaN is 0, every other score is above 0 and below 2^64 - 1.
KV_HD uint64_t score_key(double x) {
    uint64_t u;
#ifdef __CUDA_ARCH__
    u = (uint64_t)__double_as_longlong(x);
#else
    std::memcpy(&u, &x, 8);
#endif
    if ((u & 0x7fffffffffffffffull) > 0x7ff0000000000000ull) return 0ull;
    if (u == 0x8000000000000000ull) u = 0ull;
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

}  // namespace g9kv

// Host build of the paged cache's index arithmetic (gen9-gpu-blas_b200/csrc/kv_index.h) for test_kv_cpu.py.
#include "kv_index.h"

extern "C" {
int kv_quot(int page, int k) {
    const g9kv::PageDiv d = g9kv::page_div(page);
    return g9kv::page_quot(d, k);
}
// number of k in [first, first + count·step) for which the quotient is wrong
int64_t kv_quot_wrong(int page, int64_t first, int64_t count, int64_t step) {
    const g9kv::PageDiv d = g9kv::page_div(page);
    int64_t bad = 0;
    for (int64_t i = 0; i < count; i++) {
        const int64_t k = first + i * step;
        if (k < 0 || k > 0x7fffffff) continue;
        bad += g9kv::page_quot(d, (int)k) != (int)(k / page);
    }
    return bad;
}
int kv_seen(int vis, int step, int t, int cap) { return g9kv::seen_slots(vis, step, t, cap); }
int kv_first(int seen, int window) { return g9kv::first_slot(seen, window); }
int kv_page(const int *table, int64_t ts, int s, int place, int mp, int n_pages) {
    return g9kv::page_id(table, ts, s, place, mp, n_pages);
}
int64_t kv_row(int id, int slot, int g, int64_t sp, int64_t sk, int64_t sh) { return g9kv::row_at(id, slot, g, sp, sk, sh); }
uint32_t kv_wkey(float w) { return g9kv::weight_key(w); }
uint64_t kv_skey(double x) { return g9kv::score_key(x); }
}

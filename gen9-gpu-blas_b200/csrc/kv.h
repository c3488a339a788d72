// kv.h -- state and checks shared by the paged-cache operators (kv.cu, kv_attn.cu). Not installed.
#pragma once
#include "gen9blas_kv.h"
#include "internal.h"
#include "kv_index.h"
#include <vector>

#pragma GCC visibility push(hidden)

// A workspace: one buffer and zeroed arrival counters (every call leaves the counters it used at zero), grown as calls
// need. Blocks outgrown stay allocated in a workspace of the caller's own, because captured graphs may hold them.
struct gen9blas_kv_ws {
    unsigned magic = 0;
    int dev = -1;
    bool keep = true;                 // outgrown blocks stay until kv_ws_free
    void *buf = nullptr;
    size_t n = 0;
    unsigned *cnt = nullptr;
    size_t cnt_n = 0;
    cudaStream_t last = nullptr;      // stream of the last call
    bool used = false;
    std::vector<void *> old;
};

namespace g9 {

constexpr unsigned kKvWsMagic = 0x67396b76u;

// The cache as the kernels take it.
struct KvDev {
    int D, HKV, page, n_pages, mp, ns, cap;   // cap = mp·page slots per stream
    __half *K, *V, *bounds;
    long long kp, kk, kh, vp, vk, vh;
    const int *table;
    long long ts;
    g9kv::PageDiv div;
};

// One call: its stream and the capture that is in (0: none).
struct KvCall {
    DevState *d = nullptr;
    cudaStream_t st = nullptr;
    unsigned long long capture = 0;
};

// Starts a call: checks the cache's description and the shape (H = HKV for calls without query heads), then the device
// and the stream. Returns 0, GEN9BLAS_DECLINED or an error; a cache without streams or slots returns 0 with ns = 0.
int kv_begin(const gen9blas_kv_cache *c, int H, int sync, const char *who, KvDev *dev, KvCall *call);
// What a call writes must not overlap itself: rows of acc and pos (used: either given), and of the pool. Strides have to nest:
// each at least what the dimensions with smaller ones span. 0 or an error.
int kv_marks_apart(const gen9blas_kv_cache *c, bool used, int64_t ms, int64_t mh, const char *who);
int kv_rows_apart(const gen9blas_kv_cache *c, const char *who);
// p is device or managed memory of the current device.
int kv_operand(const KvCall &call, const void *p, const char *who, const char *name);
// The workspace of a call: at least `bytes` (NULL allowed for 0) and `counters` zeroed words.
int kv_workspace(gen9blas_kv_ws *ws, const KvCall &call, const char *who, size_t bytes, size_t counters, void **buf,
                 unsigned **cnt);
// Workspaces past this are refused as out of memory, so that sizes do not overflow.
constexpr long long kKvMost = 1LL << 46;
int kv_too_large(const char *who);
// Ends a call: waits if sync, else records what was written for the no-wait ledger.
int kv_finish(const KvCall &call, int sync, const QueuedWrite *w, int n);

}  // namespace g9
#pragma GCC visibility pop

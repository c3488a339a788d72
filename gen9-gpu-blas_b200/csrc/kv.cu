// kv.cu -- the paged key-value cache (include/gen9blas_kv.h): argument checks and workspaces, cache writes, page selection
// and eviction by accumulated attention weight. Attention over the pages is in kv_attn.cu. No counterpart in the
// reference, whose attention (lib/gen9blas_ml.h:122-149) reads one contiguous cache per stream.
#include "kv.h"
#include "common.cuh"
#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

using namespace g9;
using namespace g9kv;

// ---------------------------------------------------------------------------------------------- checks, workspaces
namespace g9 {

// Elements from the pool's base to the end of its last row; -1 if that passes 2^62.
static long long pool_span(const gen9blas_kv_cache *c, int64_t sp, int64_t sk, int64_t sh) {
    const __int128 n = (__int128)(c->n_pages - 1) * sp + (__int128)(c->page - 1) * sk + (__int128)(c->HKV - 1) * sh + c->D;
    return n > ((__int128)1 << 62) ? -1 : (long long)n;
}

static bool shape_ok(int D, int H, int HKV) { return D >= 8 && D <= 256 && D % 8 == 0 && HKV >= 1 && H >= HKV && H % HKV == 0; }

int kv_begin(const gen9blas_kv_cache *c, int H, int sync, const char *who, KvDev *k, KvCall *call) {
    G.status = 0;
    G.err[0] = 0;
    if (!c) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: no cache", who);
    if (!shape_ok(c->D, H ? H : c->HKV, c->HKV)) return GEN9BLAS_DECLINED;
    if (c->page < 1 || c->n_pages < 0 || c->mp < 0 || c->ns < 0 || c->ts < 0)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: page = %d, n_pages = %d, mp = %d, ns = %d, ts = %lld", who, c->page,
                    c->n_pages, c->mp, c->ns, (long long)c->ts);
    if ((long long)c->mp * c->page > INT_MAX - 64)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %d pages of %d slots per stream pass 2^31 slots", who, c->mp, c->page);
    if ((long long)c->ns * c->HKV > INT_MAX)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %d streams of %d heads pass 2^31 rows", who, c->ns, c->HKV);
    *k = KvDev{};
    k->ns = c->ns;
    if (c->n_pages > 0) {
        const int64_t st[6] = {c->kp, c->kk, c->kh, c->vp, c->vk, c->vh};
        for (int64_t s : st)
            if (s < 0 || s % 8) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: a stride of K or V is no multiple of 8 elements", who);
        if (!c->K || !c->V) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: no K or V", who);
        if (((uintptr_t)c->K | (uintptr_t)c->V | (uintptr_t)c->bounds) & 15)
            return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: K, V or bounds is not 16-byte aligned", who);
        const long long ks = pool_span(c, c->kp, c->kk, c->kh), vs = pool_span(c, c->vp, c->vk, c->vh);
        if (ks < 0 || vs < 0 || (size_t)ks * 2 > c->k_bytes || (size_t)vs * 2 > c->v_bytes)
            return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: the pool's last row passes k_bytes = %zu or v_bytes = %zu", who,
                        c->k_bytes, c->v_bytes);
    }
    if (c->ns > 0 && c->mp > 0 && !c->table) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: no table", who);
    k->D = c->D;
    k->HKV = c->HKV;
    k->page = c->page;
    k->n_pages = c->n_pages;
    k->mp = c->mp;
    k->cap = c->mp * c->page;
    k->K = (__half *)c->K;
    k->V = (__half *)c->V;
    k->bounds = (__half *)c->bounds;
    k->kp = c->kp;
    k->kk = c->kk;
    k->kh = c->kh;
    k->vp = c->vp;
    k->vk = c->vk;
    k->vh = c->vh;
    k->table = c->table;
    k->ts = c->ts;
    k->div = page_div(c->page);
    if (int e = begin_op()) return e;
    call->d = dev_state();
    call->st = stream();
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    G9_CU(cudaStreamIsCapturing(call->st, &cs));
    call->capturing = cs != cudaStreamCaptureStatusNone;
    if (call->capturing && sync)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: sync = 1 while the stream is being captured", who);
    if (c->n_pages > 0) {
        G9_TRY(kv_operand(*call, c->K, who, "K"));
        G9_TRY(kv_operand(*call, c->V, who, "V"));
        if (c->bounds) G9_TRY(kv_operand(*call, c->bounds, who, "bounds"));
    }
    if (c->ns > 0 && c->mp > 0) G9_TRY(kv_operand(*call, c->table, who, "table"));
    return 0;
}

int kv_operand(const KvCall &call, const void *p, const char *who, const char *name) {
    cudaPointerAttributes a;
    if (!p) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: no %s", who, name);
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        a.type = cudaMemoryTypeUnregistered;
    }
    if (a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == call.d->dev)) return 0;
    if (a.type == cudaMemoryTypeDevice)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %s is memory of device %d, the current device is %d", who, name, a.device,
                    call.d->dev);
    return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %s is not device or managed memory", who, name);
}

// The library's own workspace of each device.
static gen9blas_kv_ws g_ws[kMaxDevices];

int kv_workspace(gen9blas_kv_ws *ws, const KvCall &call, const char *who, size_t bytes, size_t counters, void **buf,
                 unsigned **cnt) {
    const bool own = ws == nullptr;
    if (own) {
        if (call.capturing)
            return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: a captured call needs a workspace (gen9blas_kv_ws_create)", who);
        ws = &g_ws[call.d->dev];
        ws->magic = kKvWsMagic;
        ws->keep = false;
    }
    if (ws->magic != kKvWsMagic) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: not a workspace", who);
    if (ws->dev < 0) ws->dev = call.d->dev;
    if (ws->dev != call.d->dev)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: the workspace belongs to device %d, the current device is %d", who, ws->dev,
                    call.d->dev);
    const bool grow = ws->n < bytes || ws->cnt_n < counters;
    if (call.capturing) {
        if (grow)
            return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: the workspace is too small and cannot grow during a capture: make a call "
                        "of this shape before it", who);
    } else {
        // calls of one workspace run in order: one on another stream waits for everything queued so far
        if (ws->used && ws->last != call.st) G9_CU(cudaDeviceSynchronize());
        ws->used = true;
        ws->last = call.st;
    }
    auto bigger = [&](void **p, size_t *have, size_t want, bool zero) -> int {
        want = (want + want / 4 + 0xFFFF) & ~(size_t)0xFFFF;   // a quarter more, in 64 KiB: growing lengths grow it rarely
        void *fresh = nullptr;
        size_t got = 0;
        if (*p && !ws->keep) {
            G9_CU(cudaStreamSynchronize(call.st));
            G9_CU(cudaFree(*p));
            *p = nullptr;
            *have = 0;
        }
        if (ws->keep && *p) {
            try {
                ws->old.push_back(*p);
            } catch (const std::bad_alloc &) {
                return fail(GEN9BLAS_ERR_OUT_OF_MEMORY, "%s: host memory", who);
            }
            *p = nullptr;
            *have = 0;
        }
        G9_TRY(ensure_buffer(&fresh, &got, want));
        if (zero) G9_CU(cudaMemsetAsync(fresh, 0, got, call.st));
        *p = fresh;
        *have = got;
        return 0;
    };
    if (ws->n < bytes) G9_TRY(bigger(&ws->buf, &ws->n, bytes, false));
    if (ws->cnt_n < counters) {
        void *p = ws->cnt;
        size_t have = ws->cnt_n * sizeof(unsigned);
        ws->cnt = nullptr;
        ws->cnt_n = 0;
        G9_TRY(bigger(&p, &have, counters * sizeof(unsigned), true));
        ws->cnt = (unsigned *)p;
        ws->cnt_n = have / sizeof(unsigned);
    }
    *buf = ws->buf;
    *cnt = ws->cnt;
    return 0;
}

int kv_finish(const KvCall &call, int sync, const KvWrite *w, int n) {
    if (call.capturing) {
        // a replay writes without passing here: later calls of this library treat any range as possibly being written
        call.d->queued_overflow = true;
        return 0;
    }
    if (sync) {
        G9_CU(cudaStreamSynchronize(call.st));
        queued_writes_clear(call.d);
        return check_dev_err(call.d);
    }
    for (int i = 0; i < n; i++)
        if (w[i].p) queued_writes_add(call.d, w[i].p, w[i].bytes, call.st);
    return 0;
}

}  // namespace g9

namespace {

constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------------------------- cache writes
struct AppendArgs {
    KvDev c;
    int nt, tp;               // new tokens (padded), pages they can touch per stream
    const float *K, *V;
    long long kt, kh, ks, vt, vh, vs;
    const int *len, *cnt, *pos0;
    float *acc;
    int *pos;
    long long ms, mh;
    int v4;                   // rows of K and V are 16-byte aligned
    unsigned *bad;
};

__device__ __forceinline__ float4 row4(const float *p, int v4) {
    return v4 ? __ldg(reinterpret_cast<const float4 *>(p)) : make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
}
__device__ __forceinline__ uint2 half4(float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    return make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}
__device__ __forceinline__ __half2 as_h2(unsigned x) { return *reinterpret_cast<const __half2 *>(&x); }
__device__ __forceinline__ unsigned as_u(__half2 x) { return *reinterpret_cast<const unsigned *>(&x); }

// One CTA per (page that may be touched, head, stream); its warps take the page's new rows in turn, a lane four elements
// (or two times four, D > 128) of each row, and keep the elements' least and largest value for the bounds.
__global__ void __launch_bounds__(256) kv_append_k(AppendArgs a) {
    __shared__ uint2 red[8][2][2][32];   // [warp][least, largest][four-element group of the lane][lane]
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int s = blockIdx.z, g = blockIdx.y;
    const long long n0 = max(a.len[s], 0);
    const int cn = a.cnt ? min(max(a.cnt[s], 0), a.nt) : a.nt;
    const long long place = n0 / c.page + blockIdx.x;
    const long long k0 = max(n0, place * c.page), k1 = min(n0 + cn, (place + 1) * c.page);
    if (k0 >= k1) return;
    const int id = place < c.mp ? page_id(c.table, c.ts, s, (int)place, c.mp, c.n_pages) : -1;
    if (id < 0) {
        if (threadIdx.x == 0 && a.bad) *(volatile unsigned *)a.bad = 1u;
        return;
    }
    const int i0 = (int)(k0 - place * c.page);
    const __half2 top = __half2half2(__ushort_as_half(0x7c00)), low = __half2half2(__ushort_as_half(0xfc00));
    __half2 mn[2][2] = {{top, top}, {top, top}}, mx[2][2] = {{low, low}, {low, low}};
    __half *kd = c.K + row_at(id, 0, g, c.kp, c.kk, c.kh), *vd = c.V + row_at(id, 0, g, c.vp, c.vk, c.vh);
    const int rows = (int)(k1 - k0);
    const long long t0 = k0 - n0;
    const float *ksrc = a.K + s * a.ks + g * a.kh, *vsrc = a.V + s * a.vs + g * a.vh;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int d = 4 * lane + 128 * j;
        if (d >= c.D) break;
#pragma unroll 4
        for (int r = warp; r < rows; r += nw) {
            const uint2 kv = half4(row4(ksrc + (t0 + r) * a.kt + d, a.v4)), vv = half4(row4(vsrc + (t0 + r) * a.vt + d, a.v4));
            *reinterpret_cast<uint2 *>(kd + (long long)(i0 + r) * c.kk + d) = kv;
            *reinterpret_cast<uint2 *>(vd + (long long)(i0 + r) * c.vk + d) = vv;
            mn[j][0] = __hmin2(mn[j][0], as_h2(kv.x));
            mn[j][1] = __hmin2(mn[j][1], as_h2(kv.y));
            mx[j][0] = __hmax2(mx[j][0], as_h2(kv.x));
            mx[j][1] = __hmax2(mx[j][1], as_h2(kv.y));
        }
    }
    if (a.acc || a.pos) {
        const long long m0 = s * a.ms + g * a.mh;
        const int p0 = a.pos0 ? a.pos0[s] : (int)n0;
        for (int r = threadIdx.x; r < rows; r += blockDim.x) {
            if (a.acc) a.acc[m0 + k0 + r] = 0.0f;
            if (a.pos) a.pos[m0 + k0 + r] = p0 + (int)(t0 + r);
        }
    }
    if (!c.bounds) return;
    if (nw > 1) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            red[warp][0][j][lane] = make_uint2(as_u(mn[j][0]), as_u(mn[j][1]));
            red[warp][1][j][lane] = make_uint2(as_u(mx[j][0]), as_u(mx[j][1]));
        }
        __syncthreads();
        if (warp > 0) return;
        for (int w = 1; w < nw; w++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint2 x = red[w][0][j][lane], y = red[w][1][j][lane];
                mn[j][0] = __hmin2(mn[j][0], as_h2(x.x));
                mn[j][1] = __hmin2(mn[j][1], as_h2(x.y));
                mx[j][0] = __hmax2(mx[j][0], as_h2(y.x));
                mx[j][1] = __hmax2(mx[j][1], as_h2(y.y));
            }
    }
    __half *b = c.bounds + ((long long)id * c.HKV + g) * 2 * c.D;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int d = 4 * lane + 128 * j;
        if (d >= c.D) break;
        uint2 *lo = reinterpret_cast<uint2 *>(b + d), *hi = reinterpret_cast<uint2 *>(b + c.D + d);
        if (i0 > 0) {   // the page held rows before
            const uint2 x = *lo, y = *hi;
            mn[j][0] = __hmin2(mn[j][0], as_h2(x.x));
            mn[j][1] = __hmin2(mn[j][1], as_h2(x.y));
            mx[j][0] = __hmax2(mx[j][0], as_h2(y.x));
            mx[j][1] = __hmax2(mx[j][1], as_h2(y.y));
        }
        *lo = make_uint2(as_u(mn[j][0]), as_u(mn[j][1]));
        *hi = make_uint2(as_u(mx[j][0]), as_u(mx[j][1]));
    }
}

// ---------------------------------------------------------------------------------------------- page selection
struct SelectArgs {
    KvDev c;
    int G, H, nq, dvis, first, last, nsel;
    const float *Q;
    long long qt, qh, qs;
    const int *vis;
    unsigned long long *key;   // [row (s, t, g)][mp]
    int *sel;
};

// Scores: one CTA of 128 threads per (64 pages, row (s, t, g)). The 64 pages' bounds pass through shared memory; thread i
// sums half of the head's elements of page i % 64 for every query head in 64 bits.
constexpr int SEL_PAGES = 64;
__global__ void __launch_bounds__(128) kv_score_k(SelectArgs a) {
    extern __shared__ __align__(16) uint8_t sel_sm[];
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const long long row = blockIdx.y;
    const int g = (int)(row % c.HKV);
    const long long st = row / c.HKV;
    const int t = (int)(st % a.nq), s = (int)(st / a.nq);
    const int have = (seen_slots(a.vis[s], a.dvis, t, c.cap) + c.page - 1) / c.page;
    const int p0 = blockIdx.x * SEL_PAGES;
    if (p0 >= have) return;
    double *q = reinterpret_cast<double *>(sel_sm);                 // [G][D]
    const int pitch = 2 * c.D * 2 + 16;                             // bytes of a page's bounds, padded
    uint8_t *bs = sel_sm + (size_t)a.G * c.D * sizeof(double);     // [64][pitch]
    double *part = reinterpret_cast<double *>(bs + (size_t)SEL_PAGES * pitch);   // [64]
    for (int i = threadIdx.x; i < a.G * c.D; i += blockDim.x) {
        const int h = i / c.D, d = i - h * c.D;
        q[i] = (double)a.Q[s * a.qs + t * a.qt + (long long)(g * a.G + h) * a.qh + d];
    }
    const int cpr = c.D / 4;   // 16-byte chunks of one page's bounds
    for (int i = threadIdx.x; i < SEL_PAGES * cpr; i += blockDim.x) {
        const int p = i / cpr, ch = i - p * cpr;
        const int id = p0 + p < have ? page_id(c.table, c.ts, s, p0 + p, c.mp, c.n_pages) : -1;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (id >= 0) v = __ldg(reinterpret_cast<const uint4 *>(c.bounds + ((long long)id * c.HKV + g) * 2 * c.D) + ch);
        *reinterpret_cast<uint4 *>(bs + p * pitch + ch * 16) = v;
    }
    __syncthreads();
    const int p = threadIdx.x & (SEL_PAGES - 1), part_no = threadIdx.x / SEL_PAGES;
    const int d0 = part_no ? (c.D / 2 + 1) / 2 * 2 : 0, d1 = part_no ? c.D : (c.D / 2 + 1) / 2 * 2;
    const __half2 *lo = reinterpret_cast<const __half2 *>(bs + p * pitch), *hi = lo + c.D / 2;
    double best = -INFINITY;
    bool nan = false;
    for (int h = 0; h < a.G; h++) {
        double x = 0.0;
        const double *qh = q + h * c.D;
        for (int d = d0; d < d1; d += 2) {
            const float2 l = __half22float2(lo[d / 2]), u = __half22float2(hi[d / 2]);
            const double q0 = qh[d], q1 = qh[d + 1];
            x = fma(q0, (double)(q0 >= 0.0 ? u.x : l.x), x);
            x = fma(q1, (double)(q1 >= 0.0 ? u.y : l.y), x);
        }
        if (part_no) part[p] = x;
        __syncthreads();
        if (!part_no) {
            x += part[p];
            nan = nan || x != x;
            best = fmax(best, x);
        }
        __syncthreads();
    }
    if (part_no || p0 + p >= have) return;
    const int at = p0 + p;
    unsigned long long key = nan ? 0ull : score_key(best);
    if (page_id(c.table, c.ts, s, at, c.mp, c.n_pages) < 0) key = 0ull;
    if (at < a.first || at >= have - a.last) key = ~0ull;
    a.key[row * c.mp + at] = key;
}

// The nsel largest keys of a row (ties: lowest place), ascending by place: the threshold by radix selection over 8-bit
// digits from the top, then one ordered pass. One CTA per row.
__device__ __forceinline__ int block_scan_incl(int v, int *sh, int *total) {   // blockDim.x = 1024 at most, multiple of 32
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kAll, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[w] = x;
    __syncthreads();
    if (w == 0) {
        int y = lane < nw ? sh[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(kAll, y, o);
            if (lane >= o) y += z;
        }
        sh[lane] = y;
    }
    __syncthreads();
    *total = sh[nw - 1];
    return x + (w ? sh[w - 1] : 0);
}

__global__ void __launch_bounds__(512) kv_choose_k(SelectArgs a) {
    __shared__ int hist[256], scan[32];
    __shared__ int sh_digit, sh_above, sh_in;
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const long long row = blockIdx.x;
    const long long st = row / c.HKV;
    const int t = (int)(st % a.nq), s = (int)(st / a.nq);
    const int have = (seen_slots(a.vis[s], a.dvis, t, c.cap) + c.page - 1) / c.page;
    int *out = a.sel + row * a.nsel;
    if (have <= a.nsel) {
        for (int i = threadIdx.x; i < a.nsel; i += blockDim.x) out[i] = i < have ? i : -1;
        return;
    }
    const unsigned long long *key = a.key + row * c.mp;
    unsigned long long prefix = 0, mask = 0;
    int need = a.nsel;          // how many of the keys that share the prefix are still to be taken
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < have; i += blockDim.x) {
            const unsigned long long k = key[i];
            if ((k & mask) == prefix) atomicAdd(&hist[(int)(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x < 32) {   // lane l holds digits 255 - 8l .. 248 - 8l, from the top
            int v[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) sum += v[j] = hist[255 - 8 * (int)threadIdx.x - j];
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(kAll, incl, o);
                if ((int)threadIdx.x >= o) incl += y;
            }
            int above = incl - sum;
            if (above < need && incl >= need) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (above + v[j] >= need) {
                        sh_digit = 255 - 8 * (int)threadIdx.x - j;
                        sh_above = above;
                        sh_in = v[j];
                        break;
                    }
                    above += v[j];
                }
            }
        }
        __syncthreads();
        need -= sh_above;
        prefix |= (unsigned long long)sh_digit << shift;
        mask |= 255ull << shift;
        const bool whole = sh_in == need;   // every key of this prefix is taken: no further digit matters
        __syncthreads();
        if (whole) break;
    }
    // taken: keys above the prefix (masked), and the first `need` that share it
    int base = 0, eq_base = 0;
    for (int i0 = 0; i0 < have; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const unsigned long long k = i < have ? key[i] & mask : 0ull;
        const bool eq = i < have && k == prefix;
        int total_eq, total;
        const int eq_rank = block_scan_incl(eq, scan, &total_eq) + eq_base;
        const bool take = i < have && (k > prefix || (eq && eq_rank <= need));
        const int at = block_scan_incl(take, scan, &total) + base;
        if (take) out[at - 1] = i;
        base += total;
        eq_base += total_eq;
    }
}

// ---------------------------------------------------------------------------------------------- eviction
struct EvictArgs {
    KvDev c;
    const int *len;
    int keep, first, recent;
    float *acc;
    int *pos;
    long long ms, mh;
    int *src;        // [row (s, g)][keep]: the slot that moves into slot k, or -1
    int *holes;      // [row][keep]: given-up slots below keep
    int *used;       // [row]: slots in use
    int *len_out;
};

constexpr int EV_BINS = 2048;
// Which slots stay, and where the movers go: one CTA per row (s, g). The threshold key by radix selection over digits of
// 11, 11 and 10 bits, then one ordered pass: below `keep` the given-up slots are listed, from there on the j-th staying
// slot becomes the source of the j-th of them.
__global__ void __launch_bounds__(1024) kv_rank_k(EvictArgs a) {
    __shared__ int hist[EV_BINS];
    __shared__ int scan[32];
    __shared__ int sh_digit, sh_above, sh_in, sh_new;
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const int row = blockIdx.x, s = row / c.HKV, g = row - s * c.HKV;
    const int n = min(max(a.len[s], 0), c.cap), keep = a.keep;
    if (threadIdx.x == 0) a.used[row] = n;
    if (n <= keep) return;
    const float *acc = a.acc + s * a.ms + g * a.mh;
    const int *pos = a.pos ? a.pos + s * a.ms + g * a.mh : nullptr;
    int *src = a.src + (long long)row * keep, *holes = a.holes + (long long)row * keep;
    if (threadIdx.x == 0) sh_new = INT_MIN;
    __syncthreads();
    int newest = n - 1;
    if (pos) {
        int m = INT_MIN;
        for (int k = threadIdx.x; k < n; k += blockDim.x) m = max(m, pos[k]);
        m = __reduce_max_sync(kAll, m);
        if ((threadIdx.x & 31) == 0) atomicMax(&sh_new, m);
        __syncthreads();
        newest = sh_new;
    }
    const long long old = (long long)newest - a.recent;
    auto key_of = [&](int k) -> unsigned {
        const int p = pos ? pos[k] : k;
        return p < a.first || p > old ? kAll : weight_key(acc[k]);
    };
    unsigned prefix = 0, mask = 0;
    int need = keep;
    for (int d = 0; d < 3; d++) {
        const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < EV_BINS; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        for (int k = threadIdx.x; k < n; k += blockDim.x) {
            const unsigned x = key_of(k);
            if ((x & mask) == prefix) atomicAdd(&hist[(x >> shift) & ((1u << bits) - 1)], 1);
        }
        __syncthreads();
        // thread i: bins 2047 - 2i and 2046 - 2i, from the top
        const int b0 = EV_BINS - 1 - 2 * (int)threadIdx.x;
        const int v0 = hist[b0], v1 = hist[b0 - 1];
        int total;
        const int incl = block_scan_incl(v0 + v1, scan, &total);
        const int above = incl - v0 - v1;
        if (above < need && incl >= need) {
            const bool second = above + v0 < need;
            sh_digit = second ? b0 - 1 : b0;
            sh_above = second ? above + v0 : above;
            sh_in = second ? v1 : v0;
        }
        __syncthreads();
        need -= sh_above;
        prefix |= (unsigned)sh_digit << shift;
        mask |= ((1u << bits) - 1) << shift;
        const bool whole = sh_in == need;
        __syncthreads();
        if (whole) break;
    }
    int eq_base = 0, out_base = 0;
    for (int k0 = 0; k0 < keep; k0 += blockDim.x) {
        const int k = k0 + threadIdx.x;
        const bool in = k < keep;
        const unsigned x = in ? key_of(k) & mask : 0u;
        const bool eq = in && x == prefix;
        int total_eq, total;
        const int eq_rank = block_scan_incl(eq, scan, &total_eq) + eq_base;
        const bool hole = in && !(x > prefix || (eq && eq_rank <= need));
        const int at = block_scan_incl(hole, scan, &total) + out_base;
        if (in) src[k] = -1;
        if (hole) holes[at - 1] = k;
        eq_base += total_eq;
        out_base += total;
    }
    __syncthreads();   // the list of holes is written
    int in_base = 0;
    for (int k0 = keep; k0 < n; k0 += blockDim.x) {
        const int k = k0 + threadIdx.x;
        const bool in = k < n;
        const unsigned x = in ? key_of(k) & mask : 0u;
        const bool eq = in && x == prefix;
        int total_eq, total;
        const int eq_rank = block_scan_incl(eq, scan, &total_eq) + eq_base;
        const bool stay = in && (x > prefix || (eq && eq_rank <= need));
        const int at = block_scan_incl(stay, scan, &total) + in_base;
        if (stay && at <= out_base) src[holes[at - 1]] = k;
        eq_base += total_eq;
        in_base += total;
    }
}

// The moves: one warp per (page below keep, row). lpr lanes carry a row, 16 bytes each; the bounds of a page that got or
// lost rows are taken over the rows it now holds, the movers' from their sources.
__global__ void __launch_bounds__(256) kv_move_k(EvictArgs a, int pages, int lpr) {
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const int lane = threadIdx.x & 31;
    const long long w = blockIdx.x * 8LL + (threadIdx.x >> 5);
    const long long row = w / pages;
    if (row >= (long long)c.ns * c.HKV) return;
    const int place = (int)(w % pages), s = (int)(row / c.HKV), g = (int)(row % c.HKV);
    const int n = a.used[row], keep = a.keep;
    if (place == 0 && g == 0 && lane == 0) a.len_out[s] = min(n, keep);
    if (n <= keep) return;
    const int k0 = place * c.page, rows = min(c.page, keep - k0);
    if (rows <= 0) return;
    const int *src = a.src + row * keep + k0;
    bool any = false;
    for (int i = lane; i < rows; i += 32) any = any || src[i] >= 0;
    any = __any_sync(kAll, any);
    const bool cut = rows < c.page;   // the page held slots at and above keep
    if (!any && !cut) return;
    const int id = page_id(c.table, c.ts, s, place, c.mp, c.n_pages);
    if (any) {
        float *acc = a.acc + s * a.ms + g * a.mh;
        int *pos = a.pos ? a.pos + s * a.ms + g * a.mh : nullptr;
        for (int i = lane; i < rows; i += 32) {
            const int k = src[i];
            if (k < 0) continue;
            acc[k0 + i] = acc[k];
            if (pos) pos[k0 + i] = pos[k];
        }
    }
    if (id < 0) return;
    const int rpw = 32 / lpr, sub = lane / lpr, ch = lane - sub * lpr;
    const bool live = ch * 8 < c.D;
    const bool bounds = c.bounds != nullptr;
    __half2 mn[4], mx[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        mn[j] = __half2half2(__ushort_as_half(0x7c00));
        mx[j] = __half2half2(__ushort_as_half(0xfc00));
    }
#pragma unroll 4
    for (int i = sub; i < rows; i += rpw) {
        const int k = src[i];
        int from = -1, slot = i;
        if (k >= 0) {
            const int pl = page_quot(c.div, k);
            from = page_id(c.table, c.ts, s, pl, c.mp, c.n_pages);
            slot = k - pl * c.page;
        }
        if (!live || (!bounds && from < 0)) continue;
        const int rid = from >= 0 ? from : id;
        if (from < 0) slot = i;
        const uint4 kv = *reinterpret_cast<const uint4 *>(c.K + row_at(rid, slot, g, c.kp, c.kk, c.kh) + ch * 8);
        if (from >= 0) {
            const uint4 vv = *reinterpret_cast<const uint4 *>(c.V + row_at(rid, slot, g, c.vp, c.vk, c.vh) + ch * 8);
            *reinterpret_cast<uint4 *>(c.K + row_at(id, i, g, c.kp, c.kk, c.kh) + ch * 8) = kv;
            *reinterpret_cast<uint4 *>(c.V + row_at(id, i, g, c.vp, c.vk, c.vh) + ch * 8) = vv;
        }
        const unsigned x[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mn[j] = __hmin2(mn[j], as_h2(x[j]));
            mx[j] = __hmax2(mx[j], as_h2(x[j]));
        }
    }
    if (!bounds) return;
    for (int o = lpr; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mn[j] = __hmin2(mn[j], as_h2(__shfl_xor_sync(kAll, as_u(mn[j]), o)));
            mx[j] = __hmax2(mx[j], as_h2(__shfl_xor_sync(kAll, as_u(mx[j]), o)));
        }
    if (sub || !live) return;
    __half *b = c.bounds + ((long long)id * c.HKV + g) * 2 * c.D + ch * 8;
    *reinterpret_cast<uint4 *>(b) = make_uint4(as_u(mn[0]), as_u(mn[1]), as_u(mn[2]), as_u(mn[3]));
    *reinterpret_cast<uint4 *>(b + c.D) = make_uint4(as_u(mx[0]), as_u(mx[1]), as_u(mx[2]), as_u(mx[3]));
}

// bytes that the acc or pos rows of all heads and streams span
size_t marks_bytes(const KvDev &c, int64_t ms, int64_t mh) {
    return ((size_t)std::max(c.ns - 1, 0) * (size_t)std::max<int64_t>(ms, 0) + (size_t)(c.HKV - 1) * (size_t)std::max<int64_t>(mh, 0) +
            (size_t)c.cap) * 4;
}
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace

// ---------------------------------------------------------------------------------------------- entry points
extern "C" {

GEN9BLAS_API int gen9blas_kv_supported(int D, int H, int HKV) { return shape_ok(D, H, HKV) ? 1 : 0; }

GEN9BLAS_API void *gen9blas_get_stream(void) { return G.user_stream_set ? (void *)G.user_stream : nullptr; }

GEN9BLAS_API gen9blas_kv_ws *gen9blas_kv_ws_create(void) {
    if (begin_op()) return nullptr;
    gen9blas_kv_ws *ws = new (std::nothrow) gen9blas_kv_ws;
    if (!ws) {
        fail(GEN9BLAS_ERR_OUT_OF_MEMORY, "kv_ws_create: host memory");
        return nullptr;
    }
    ws->magic = kKvWsMagic;
    return ws;
}

GEN9BLAS_API void gen9blas_kv_ws_free(gen9blas_kv_ws *ws) {
    if (!ws || ws->magic != kKvWsMagic || gen9blas_init()) return;
    if (ws->dev >= 0) {
        int cur = -1;
        cudaGetDevice(&cur);
        cudaSetDevice(ws->dev);
        cudaDeviceSynchronize();
        for (void *p : ws->old) cudaFree(p);
        cudaFree(ws->buf);
        cudaFree(ws->cnt);
        cudaSetDevice(cur);
        cudaGetLastError();
    }
    ws->magic = 0;
    delete ws;
}

GEN9BLAS_API int gen9blas_kv_append(const gen9blas_kv_cache *c, int nt, const float *K, int64_t kt, int64_t kh, int64_t ks,
                                    const float *V, int64_t vt, int64_t vh, int64_t vs, const int *len, const int *cnt,
                                    float *acc, int *pos, int64_t ms, int64_t mh, const int *pos0, int sync, int *bad) {
    const char *who = "kv_append";
    AppendArgs a{};
    KvCall call;
    if (bad) *bad = 0;
    if (int e = kv_begin(c, 0, sync, who, &a.c, &call)) return e;
    if (c->ns == 0 || nt <= 0) return 0;
    if (c->ns > 65535 || c->HKV > 65535)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %d streams of %d heads in one call", who, c->ns, c->HKV);
    G9_TRY(kv_operand(call, K, who, "K (new)"));
    G9_TRY(kv_operand(call, V, who, "V (new)"));
    G9_TRY(kv_operand(call, len, who, "len"));
    if (cnt) G9_TRY(kv_operand(call, cnt, who, "cnt"));
    if (acc) G9_TRY(kv_operand(call, acc, who, "acc"));
    if (pos) G9_TRY(kv_operand(call, pos, who, "pos"));
    if (pos && pos0) G9_TRY(kv_operand(call, pos0, who, "pos0"));
    a.nt = nt;
    a.tp = (nt - 1) / c->page + 2;   // nt slots from anywhere in a page
    a.K = K;
    a.V = V;
    a.kt = kt;
    a.kh = kh;
    a.ks = ks;
    a.vt = vt;
    a.vh = vh;
    a.vs = vs;
    a.len = len;
    a.cnt = cnt;
    a.pos0 = pos ? pos0 : nullptr;
    a.acc = acc;
    a.pos = pos;
    a.ms = ms;
    a.mh = mh;
    a.v4 = (((uintptr_t)K | (uintptr_t)V) & 15) == 0 && ((kt | kh | ks | vt | vh | vs) & 3) == 0;
    volatile unsigned *flag = (volatile unsigned *)call.d->err_host + 2;   // read back by a waiting call
    if (sync) {
        a.bad = call.d->err_dev + 2;
        *flag = 0;
    }
    const int per = std::min(nt, c->page);
    const int warps = std::min(8, std::max(1, (per + 3) / 4));
    G9_CU(launch_pdl(kv_append_k, dim3((unsigned)a.tp, (unsigned)c->HKV, (unsigned)c->ns), dim3(32 * warps), 0, call.st, a));
    G9_TRY(launched("kv_append"));
    const size_t marks = marks_bytes(a.c, ms, mh);
    const KvWrite w[4] = {{c->K, c->k_bytes}, {c->V, c->v_bytes}, {acc, marks}, {pos, marks}};
    G9_TRY(kv_finish(call, sync, w, 4));
    if (sync && bad) *bad = (int)*flag;
    return 0;
}

GEN9BLAS_API int gen9blas_kv_select(const gen9blas_kv_cache *c, int H, int nq, const float *Q, int64_t qt, int64_t qh,
                                    int64_t qs, const int *vis, int dvis, int first, int last, int nsel, int *sel,
                                    gen9blas_kv_ws *ws, int sync) {
    const char *who = "kv_select";
    SelectArgs a{};
    KvCall call;
    if (H < 1) return GEN9BLAS_DECLINED;
    if (c && (first < 0 || last < 0 || dvis < 0 || nsel < 0))
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: first = %d, last = %d, nsel = %d, dvis = %d", who, first, last, nsel, dvis);
    if (c && c->n_pages > 0 && !c->bounds) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: the cache has no bounds", who);
    if (int e = kv_begin(c, H, sync, who, &a.c, &call)) return e;
    if (c->ns == 0 || nq <= 0 || nsel == 0) return 0;
    const long long rows = (long long)c->ns * nq * c->HKV;
    if (rows > 65535) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %lld rows (stream, token, head) in one call", who, rows);
    G9_TRY(kv_operand(call, Q, who, "Q"));
    G9_TRY(kv_operand(call, vis, who, "vis"));
    G9_TRY(kv_operand(call, sel, who, "sel"));
    a.G = H / c->HKV;
    a.H = H;
    a.nq = nq;
    a.dvis = dvis;
    a.first = first;
    a.last = last;
    a.nsel = nsel;
    a.Q = Q;
    a.qt = qt;
    a.qh = qh;
    a.qs = qs;
    a.vis = vis;
    a.sel = sel;
    void *buf = nullptr;
    unsigned *cnt = nullptr;
    G9_TRY(kv_workspace(ws, call, who, std::max<size_t>((size_t)rows * c->mp * 8, 256), 0, &buf, &cnt));
    a.key = (unsigned long long *)buf;
    const size_t smem = (size_t)a.G * c->D * 8 + (size_t)SEL_PAGES * (4 * c->D + 16) + SEL_PAGES * 8;
    if (smem > 227 * 1024) return GEN9BLAS_DECLINED;
    static bool attr[kMaxDevices] = {};
    G9_CU(smem_limit_once(kv_score_k, 227 * 1024, attr));
    if (c->mp > 0) {
        G9_CU(launch_pdl(kv_score_k, dim3((unsigned)((c->mp + SEL_PAGES - 1) / SEL_PAGES), (unsigned)rows), dim3(128), smem,
                         call.st, a));
        G9_TRY(launched("kv_score"));
    }
    G9_CU(launch_pdl(kv_choose_k, dim3((unsigned)rows), dim3(512), 0, call.st, a));
    G9_TRY(launched("kv_choose"));
    const KvWrite w[1] = {{sel, (size_t)rows * nsel * 4}};
    return kv_finish(call, sync, w, 1);
}

GEN9BLAS_API int gen9blas_kv_evict(const gen9blas_kv_cache *c, const int *len, int keep, int first, int recent, float *acc,
                                   int *pos, int64_t ms, int64_t mh, int *len_out, gen9blas_kv_ws *ws, int sync) {
    const char *who = "kv_evict";
    EvictArgs a{};
    KvCall call;
    if (c && (keep < 1 || first < 0 || recent < 0 || (long long)first + recent > keep))
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: keep = %d, first = %d, recent = %d", who, keep, first, recent);
    if (int e = kv_begin(c, 0, sync, who, &a.c, &call)) return e;
    if (c->ns == 0) return 0;
    G9_TRY(kv_operand(call, len, who, "len"));
    G9_TRY(kv_operand(call, len_out, who, "len_out"));
    G9_TRY(kv_operand(call, acc, who, "acc"));
    if (pos) G9_TRY(kv_operand(call, pos, who, "pos"));
    const long long rows = (long long)c->ns * c->HKV;
    const int keep_in = std::min(keep, a.c.cap);        // no stream holds more
    a.len = len;
    a.keep = std::max(keep_in, 1);
    a.first = first;
    a.recent = recent;
    a.acc = acc;
    a.pos = pos;
    a.ms = ms;
    a.mh = mh;
    a.len_out = len_out;
    void *buf = nullptr;
    unsigned *cnt = nullptr;
    const size_t list = up256((size_t)rows * a.keep * 4);
    G9_TRY(kv_workspace(ws, call, who, 2 * list + up256((size_t)rows * 4), 0, &buf, &cnt));
    a.src = (int *)buf;
    a.holes = (int *)((char *)buf + list);
    a.used = (int *)((char *)buf + 2 * list);
    G9_CU(launch_pdl(kv_rank_k, dim3((unsigned)rows), dim3(1024), 0, call.st, a));
    G9_TRY(launched("kv_rank"));
    const int pages = (a.keep + c->page - 1) / c->page;
    const int lpr = c->D <= 64 ? 8 : c->D <= 128 ? 16 : 32;
    const long long warps = rows * pages;
    if ((warps + 7) / 8 > INT_MAX) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %lld pages in one call", who, warps);
    G9_CU(launch_pdl(kv_move_k, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, call.st, a, pages, lpr));
    G9_TRY(launched("kv_move"));
    const size_t marks = marks_bytes(a.c, ms, mh);
    const KvWrite w[4] = {{c->K, c->k_bytes}, {c->V, c->v_bytes}, {acc, marks}, {pos, marks}};
    return kv_finish(call, sync, w, 4);
}

}  // extern "C"

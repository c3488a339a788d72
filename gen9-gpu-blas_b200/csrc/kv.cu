// kv.cu -- the paged key-value cache (include/gen9blas_kv.h): argument checks and workspaces, cache writes, page selection
// and eviction by accumulated attention weight. Attention over the pages is in kv_attn.cu. No counterpart in the
// reference, whose attention (lib/gen9blas_ml.h:122-149) reads one contiguous cache per stream.
#include "kv.h"
#include "common.cuh"
#include "kv_plan.cuh"
#include "mma_sync.cuh"
#include "sm100.cuh"
#include <cooperative_groups.h>
#include <algorithm>
#include <cfloat>
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
    if ((long long)c->mp * c->page > INT_MAX - 65536)   // slots are counted in 32 bits, in steps of up to 6144
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
    if (!gen9blas_init() && !dev_state_if_ready(G.cur_dev)) {   // setting the device up allocates, which would end a capture
        const cudaStream_t st = c->stream ? (cudaStream_t)c->stream : G.user_stream_set ? G.user_stream : nullptr;
        cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
        if (st && cudaStreamIsCapturing(st, &cs) != cudaSuccess) cudaGetLastError();
        if (cs != cudaStreamCaptureStatusNone)
            return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: the first call on a device cannot be captured: make one before, with the "
                        "workspace (gen9blas_kv_ws_create) of the captured one", who);
    }
    if (int e = begin_op()) return e;
    call->d = dev_state();
    call->st = c->stream ? (cudaStream_t)c->stream : stream();
    call->capture = capture_of(call->st);
    if (call->capture == kCaptureUnknown)   // a launch would end that other capture, too
        return fail(GEN9BLAS_ERR, "%s: the capture of the call's stream has failed, or that of a stream which synchronises with it "
                    "is under way", who);
    if (call->capture && sync)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: sync = 1 while the stream is being captured", who);
    if (c->n_pages > 0) {
        G9_TRY(kv_operand(*call, c->K, who, "K"));
        G9_TRY(kv_operand(*call, c->V, who, "V"));
        if (c->bounds) G9_TRY(kv_operand(*call, c->bounds, who, "bounds"));
    }
    if (c->ns > 0 && c->mp > 0) G9_TRY(kv_operand(*call, c->table, who, "table"));
    return 0;
}

// Whether rows of `row` elements, n[i] of them `st[i]` apart in each of the dimensions, share no element: the strides nest, each
// at least what the rows of the dimensions with smaller ones span together.
static bool rows_nest(int dims, const long long *n, const int64_t *st, long long row) {
    bool done[3] = {};
    __int128 span = row;
    for (int k = 0; k < dims; k++) {
        int at = -1;
        for (int i = 0; i < dims; i++)
            if (!done[i] && (at < 0 || st[i] < st[at])) at = i;
        done[at] = true;
        if (n[at] <= 1) continue;
        if (st[at] < span) return false;
        span += (__int128)(n[at] - 1) * st[at];
    }
    return true;
}

int kv_marks_apart(const gen9blas_kv_cache *c, bool used, int64_t ms, int64_t mh, const char *who) {
    if (!c || !used) return 0;
    const long long cap = (long long)c->mp * c->page, n[2] = {c->ns, c->HKV};
    const int64_t st[2] = {ms, mh};
    if (!rows_nest(2, n, st, cap))
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: rows of acc or pos overlap: strides %lld and %lld, %lld slots", who,
                    (long long)ms, (long long)mh, cap);
    return 0;
}

int kv_rows_apart(const gen9blas_kv_cache *c, const char *who) {
    if (!c || c->n_pages <= 0) return 0;
    const long long n[3] = {c->n_pages, c->page, c->HKV};
    const int64_t ks[3] = {c->kp, c->kk, c->kh}, vs[3] = {c->vp, c->vk, c->vh};
    if (!rows_nest(3, n, ks, c->D) || !rows_nest(3, n, vs, c->D))
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: rows of K or V overlap: strides %lld, %lld, %lld and %lld, %lld, %lld elements", who,
                    (long long)c->kp, (long long)c->kk, (long long)c->kh, (long long)c->vp, (long long)c->vk, (long long)c->vh);
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
        if (call.capture)
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
    if (call.capture) {
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

int kv_too_large(const char *who) { return fail(GEN9BLAS_ERR_OUT_OF_MEMORY, "%s: the call's workspace passes 2^46 bytes", who); }

int kv_finish(const KvCall &call, int sync, const QueuedWrite *w, int n) {
    if (sync) {
        G9_CU(cudaStreamSynchronize(call.st));
        queued_writes_clear(call.d, call.st);
        return check_dev_err(call.d);
    }
    queued_writes_add(call.d, w, n, call.st, call.capture);
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

__device__ __forceinline__ __half2 as_h2(unsigned x) { return *reinterpret_cast<const __half2 *>(&x); }
__device__ __forceinline__ unsigned as_u(__half2 x) { return *reinterpret_cast<const unsigned *>(&x); }
// eight F32 elements as FP16, to nearest even
__device__ __forceinline__ uint4 row8(const float *p, int v4) {
    float x[8];
    if (v4) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __ldg(p + i);
    }
    return make_uint4(as_u(__floats2half2_rn(x[0], x[1])), as_u(__floats2half2_rn(x[2], x[3])), as_u(__floats2half2_rn(x[4], x[5])),
                      as_u(__floats2half2_rn(x[6], x[7])));
}
// the elements' least and largest of two pairs of 8
__device__ __forceinline__ uint4 least8(uint4 x, uint4 y) {
    return make_uint4(as_u(__hmin2(as_h2(x.x), as_h2(y.x))), as_u(__hmin2(as_h2(x.y), as_h2(y.y))),
                      as_u(__hmin2(as_h2(x.z), as_h2(y.z))), as_u(__hmin2(as_h2(x.w), as_h2(y.w))));
}
__device__ __forceinline__ uint4 largest8(uint4 x, uint4 y) {
    return make_uint4(as_u(__hmax2(as_h2(x.x), as_h2(y.x))), as_u(__hmax2(as_h2(x.y), as_h2(y.y))),
                      as_u(__hmax2(as_h2(x.z), as_h2(y.z))), as_u(__hmax2(as_h2(x.w), as_h2(y.w))));
}
__device__ __forceinline__ uint4 shfl8(uint4 x, int o) {
    return make_uint4(__shfl_xor_sync(kAll, x.x, o), __shfl_xor_sync(kAll, x.y, o), __shfl_xor_sync(kAll, x.z, o),
                      __shfl_xor_sync(kAll, x.w, o));
}

// One CTA per (page that may be touched, head, stream); its warps take the page's new rows in turn, lpr lanes a row, eight
// elements a lane, and keep the elements' least and largest value for the bounds. Bound by memory: the rows read once in
// FP32 and written once in FP16: 16.9 µs for 81 MB, with four rounds of rows in flight per warp at four CTAs per SM (eight bytes a
// lane instead of sixteen 18.5; two rounds at five CTAs 21.8, their registers spilled).
__global__ void __launch_bounds__(256, 4) kv_append_k(const __grid_constant__ AppendArgs a, int lpr) {
    __shared__ uint4 red[8][2][32];   // [warp][least, largest][lane]
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
    const int i0 = (int)(k0 - place * c.page), rows = (int)(k1 - k0);
    const long long t0 = k0 - n0;
    const int rpw = 32 / lpr, sub = lane / lpr, d = (lane - sub * lpr) * 8;   // rows of a warp at once, this lane's row and elements
    const bool live = d < c.D;
    uint4 mn = make_uint4(0x7c007c00u, 0x7c007c00u, 0x7c007c00u, 0x7c007c00u);
    uint4 mx = make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
    __half *kd = c.K + row_at(id, i0, g, c.kp, c.kk, c.kh) + d, *vd = c.V + row_at(id, i0, g, c.vp, c.vk, c.vh) + d;
    const float *ksrc = a.K + s * a.ks + g * a.kh + t0 * a.kt + d, *vsrc = a.V + s * a.vs + g * a.vh + t0 * a.vt + d;
    if (live) {
#pragma unroll 4
        for (int r = warp * rpw + sub; r < rows; r += nw * rpw) {
            const uint4 kv = row8(ksrc + r * a.kt, a.v4), vv = row8(vsrc + r * a.vt, a.v4);
            *reinterpret_cast<uint4 *>(kd + r * c.kk) = kv;
            *reinterpret_cast<uint4 *>(vd + r * c.vk) = vv;
            mn = least8(mn, kv);
            mx = largest8(mx, kv);
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
    for (int o = lpr; o < 32; o <<= 1) {
        mn = least8(mn, shfl8(mn, o));
        mx = largest8(mx, shfl8(mx, o));
    }
    if (nw > 1) {
        red[warp][0][lane] = mn;
        red[warp][1][lane] = mx;
        __syncthreads();
        if (warp > 0) return;
        for (int w = 1; w < nw; w++) {
            mn = least8(mn, red[w][0][lane]);
            mx = largest8(mx, red[w][1][lane]);
        }
    }
    if (sub || !live) return;
    uint4 *lo = reinterpret_cast<uint4 *>(c.bounds + ((long long)id * c.HKV + g) * 2 * c.D + d);
    uint4 *hi = reinterpret_cast<uint4 *>(c.bounds + (((long long)id * c.HKV + g) * 2 + 1) * c.D + d);
    if (i0 > 0) {   // the page held rows before
        mn = least8(mn, *lo);
        mx = largest8(mx, *hi);
    }
    *lo = mn;
    *hi = mx;
}

// ---------------------------------------------------------------------------------------------- page selection
// Two kernels. kv_score_k reads the bounds once and scores every page in FP32 on the tensor cores; kv_choose_k takes the
// nsel best of a row, and where the FP32 scores cannot tell which side of the border a page lies on (they differ by less
// than twice their error bound) it computes those pages' scores again in 64 bits: the choice is the one of the 64-bit
// scores. Scoring everything in 64 bits took 118 µs at 16 streams × 8 heads × 2048 pages of D 128 (101 MB of bounds), its
// conversions and FP64 multiply-adds the limit.
struct SelectArgs {
    KvDev c;
    int G, H, nq, dvis, first, last, nsel;
    int hg, tiles, tg, zt, zs;      // 8-head groups of a token, row tiles (token, group) in all, at once in a CTA, in all of a unit
                                    // (whole tokens; more than tg only where one token's groups are more), units of a head
    int unit_steps;                 // most steps of a unit: ⌈mp / 16⌉
    PageDiv by_zs;
    const float *Q;
    long long qt, qh, qs;
    const int *vis;
    float *score;               // [row (s, t, g)][mp]: FP32 scores; kv_choose_k overwrites those that it decided by hand
    float *l1;                  // [(s, t, h)]: sum of |q|
    float *peak;                // [(s, g, z)][unit_steps]: largest |bound| of a step; infinity where a score is not finite
    unsigned long long *key;    // [row][mp]: 64-bit keys of pages decided by hand, where they are many
    int *sel;
    unsigned *err;              // the device's error word
};

__device__ __forceinline__ int pages_seen(const SelectArgs &a, int s, int t) {
    const int n = seen_slots(a.vis[s], a.dvis, t, a.c.cap);
    return n / a.c.page + (n % a.c.page != 0);
}

__device__ __forceinline__ void bulk_row(void *dst, const void *src, unsigned bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                     sm100::smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
                 : "memory");
}
constexpr uint64_t SWAIT_NS = 2000000000ull;   // a row that has not landed after 2 s is an error
constexpr int SCOST = 8;   // steps that a CTA reads in the time of a segment's latencies
constexpr int SW = 4, SPAGES = 16, SNST = 2;   // warps of a CTA, pages of a step, stages of a warp's ring: two, so that an SM
// holds 12 warps (D = 128), because a step computes about as long as its copy takes (three stages took 5.5 µs longer at 101 MB)
template <int DP>
struct ScoreCfg {
    static constexpr int PITCH = DP * 2 * 2 + 16;                   // a page's lower and upper row; 16 bytes more spread the banks
    static constexpr int STAGE = SPAGES * PITCH;
    static constexpr int RING = SW * SNST * STAGE;
    static constexpr int QF = 2 * (DP / 16) * 32 * 16;              // fragments of one row tile: q < 0 and q > 0
    static constexpr int TG = DP == 256 ? 1 : DP == 128 ? 4 : 8;    // row tiles a CTA holds at most
    static constexpr int BARS = SW * SNST * 8;
    static constexpr int smem(int tg) { return RING + BARS + tg * (QF + 8 * 4); }
};

// Score of (page, query head): Σ_d max(q_d·lo_d, q_d·hi_d) = Σ min(q, 0)·lo + Σ max(q, 0)·hi, a product of the bounds (A, 16
// pages × 16 elements, FP16 as they are) with the two halves of the query (B, 8 heads) in two FP16 parts each, as in
// attn_paged_k. Units are (stream, head, tokens whose tiles of 8 heads shared memory holds at once); a CTA's run (kv_plan.cuh)
// is a stretch of steps of 16 pages, of which its four warps take every fourth through rings of their own. A page's score is
// the largest over the heads of a token; where one token has more tiles than fit, the CTA reads its pages again for the next
// ones. Bound by the reading of the bounds.
template <int DP>
__global__ void __launch_bounds__(SW * 32) kv_score_k(const __grid_constant__ SelectArgs a) {
    using C = ScoreCfg<DP>;
    constexpr int KT = DP / 16, PITCH = C::PITCH;
    extern __shared__ __align__(128) uint8_t ss[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(ss + C::RING);
    uint4 *qf = reinterpret_cast<uint4 *>(ss + C::RING + C::BARS);                       // [tile][half][kt][lane]
    float *qinv = reinterpret_cast<float *>(ss + C::RING + C::BARS + a.tg * C::QF);      // [tile][8]
    __shared__ int quit;
    const KvDev &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    uint8_t *wring = ss + warp * SNST * C::STAGE;
    uint64_t *bar = bars + warp * SNST;
    if (lane < SNST) sm100::mbar_init(bar + lane, 1);
    sm100::fence_barrier_init();
    if (tid == 0) quit = 0;
    // what lies behind a row shorter than the tiles is multiplied by zeros: it has to be finite
    for (int i = lane; i < SNST * SPAGES; i += 32)
        for (int e = c.D * 4; e < PITCH; e += 16) *reinterpret_cast<uint4 *>(wring + i * PITCH + e) = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
    pdl_next();
    pdl_wait();
    const int kts = (c.D + 15) / 16, inner = c.HKV * a.zs;
    const unsigned wbase = sm100::smem_u32(wring);
    unsigned copied = 0, used = 0;   // copies of this warp so far, and those it has waited for: copy n goes to stage n % SNST,
                                     // in the barrier's phase n / SNST
    const int arow = (lane & 7) + ((lane >> 3) & 1) * 8, acol = lane >> 4;
    bool ok = true;
    auto wait = [&]() {
        ok = ok && sm100::mbar_wait(bar + used % SNST, used / SNST & 1, &quit, SWAIT_NS);
        used++;
    };
    auto unit_steps = [&](int s) { return max(1, (pages_seen(a, s, a.nq - 1) + SPAGES - 1) / SPAGES); };
    const Run run = find_run(c.ns, inner, SCOST, SW, unit_steps);
    int s = run.outer, pre = run.pre;
    for (int at = run.lo; at < run.hi && ok;) {
        const int nv = unit_steps(s) + SCOST, iu = (at - pre) / nv;
        if (iu >= inner) {
            pre += nv * inner;
            s++;
            continue;
        }
        const int us = pre + iu * nv, sb = max(at - us - SCOST, 0), se = min(run.hi - us, nv) - SCOST;
        at = us + nv;
        if (se <= 0) break;   // the run ends before the unit's first step
        const int g = page_quot(a.by_zs, iu), z = iu - g * a.zs;
        const int z0 = z * a.zt, z1 = min(z0 + a.zt, a.tiles);
        const int have = pages_seen(a, s, (z1 - 1) / a.hg);   // of the unit's last token; steps go by the call's last
        float *peaks = a.peak + (((long long)s * c.HKV + g) * a.zs + z) * a.unit_steps;
        const int my = se > sb + warp ? (se - sb - warp + SW - 1) / SW : 0;
        auto id_of = [&](int i) {
            const int p = (sb + warp + SW * i) * SPAGES + (lane & 15);
            return i < my && p < have ? page_id(c.table, c.ts, s, p, c.mp, c.n_pages) : -1;
        };
        // one bulk copy per page, both rows (lane l < 16: page l); a page that is missing keeps what its place held before
        auto copy = [&](int i, int id) {
            if (i >= my) return;
            const int st = copied % SNST;
            const unsigned here = __ballot_sync(kAll, lane < SPAGES && id >= 0);
            if (lane == 0) sm100::mbar_arrive_expect_tx(bar + st, __popc(here) * c.D * 4);
            __syncwarp();
            if (here >> lane & 1u)
                bulk_row(wring + st * C::STAGE + lane * PITCH, c.bounds + ((long long)id * c.HKV + g) * 2 * c.D, c.D * 4, bar + st);
            copied++;
        };
        __syncthreads();   // every warp has left the last unit's fragments
        for (int tile0 = z0; tile0 < z1 && ok; tile0 += a.tg) {
            const int ntile = min(a.tg, z1 - tile0);
            if (tile0 > z0) __syncthreads();   // every warp has left the last tiles' fragments
            int ids[SNST];   // page numbers of the steps i .. i + SNST - 1; the last is the next to be copied
#pragma unroll
            for (int i = 0; i < SNST; i++) ids[i] = id_of(i);
#pragma unroll
            for (int i = 0; i < SNST - 1; i++) copy(i, ids[i]);
            // ---- query fragments: a warp prepares every fourth row of the tiles
            for (int r = warp; r < ntile * 8; r += SW) {
                const int tile = tile0 + (r >> 3), t = tile / a.hg, h = (tile - t * a.hg) * 8 + (r & 7);
                const bool live = h < a.G;
                const float *qp = a.Q + s * a.qs + t * a.qt + (long long)(g * a.G + (live ? h : 0)) * a.qh;
                float x[DP / 32], big = 0.0f, l1 = 0.0f;
#pragma unroll
                for (int i = 0; i < DP / 64; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int d = 64 * i + 2 * lane + j;
                        const float v = live && d < c.D ? qp[d] : 0.0f;
                        x[2 * i + j] = v;
                        big = fmaxf(big, fabsf(v));
                        l1 += fabsf(v);
                    }
                for (int i = 16; i > 0; i >>= 1) {
                    big = fmaxf(big, __shfl_xor_sync(kAll, big, i));
                    l1 += __shfl_xor_sync(kAll, l1, i);
                }
                int ex = 0;
                if (big > 0.0f) ex = min(max(140 - (int)((__float_as_uint(big) >> 23) & 0xffu), -126), 126);
                const float up = at_pow2(ex);
                if (lane == 0) {
                    qinv[r] = at_pow2(-ex);
                    if (live && sb == 0) a.l1[((long long)s * a.nq + t) * a.H + g * a.G + h] = l1;
                }
#pragma unroll
                for (int i = 0; i < DP / 64; i++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        float y0 = x[2 * i] * up, y1 = x[2 * i + 1] * up;
                        y0 = half ? fmaxf(y0, 0.0f) : fminf(y0, 0.0f);
                        y1 = half ? fmaxf(y1, 0.0f) : fminf(y1, 0.0f);
                        unsigned h2, l2;
                        at_split(y0, y1, h2, l2);
                        const int d = 64 * i + 2 * lane, kt = d >> 4, dd = d & 15;
                        unsigned *f = reinterpret_cast<unsigned *>(qf + (((r >> 3) * 2 + half) * KT + kt) * 32 + (r & 7) * 4 + ((dd & 7) >> 1));
                        f[dd >> 3] = h2;
                        f[2 + (dd >> 3)] = l2;
                    }
            }
            __syncthreads();
            for (int i = 0; i < my; i++) {
                const unsigned lo = wbase + used % SNST * C::STAGE, hi = lo + c.D * 2;
                wait();
                if (!__all_sync(kAll, ok)) {
                    ok = false;
                    break;
                }
                copy(i + SNST - 1, ids[SNST - 1]);   // into the stage before this one, which every lane has left
                const int step = sb + warp + SW * i, p = step * SPAGES + gq;
                const bool in0 = __shfl_sync(kAll, ids[0], gq) >= 0, in1 = __shfl_sync(kAll, ids[0], gq + 8) >= 0;
                float top[2] = {-INFINITY, -INFINITY};
                __half2 pk0 = __half2half2(__ushort_as_half(0)), pk1 = pk0;
                bool wild = false;
                for (int tile = 0; tile < ntile; tile++) {
                    float sc[4][4] = {};   // lower and upper bounds, by the queries' first and second parts: four chains, not one
                    const uint4 *q0 = qf + tile * 2 * KT * 32 + lane, *q1 = q0 + KT * 32;
#pragma unroll
                    for (int kt = 0; kt < KT; kt++) {
                        if (kt >= kts) break;
                        const unsigned off = arow * PITCH + kt * 32 + acol * 16;
                        unsigned l4[4], u4[4];
                        at_ldsm(lo + off, l4);
                        at_ldsm(hi + off, u4);
                        if (tile == 0) {   // registers 0 and 2: page gq, 1 and 3: page gq + 8
                            pk0 = __hmax2(__hmax2(pk0, __hmax2(__habs2(as_h2(l4[0])), __habs2(as_h2(l4[2])))),
                                          __hmax2(__habs2(as_h2(u4[0])), __habs2(as_h2(u4[2]))));
                            pk1 = __hmax2(__hmax2(pk1, __hmax2(__habs2(as_h2(l4[1])), __habs2(as_h2(l4[3])))),
                                          __hmax2(__habs2(as_h2(u4[1])), __habs2(as_h2(u4[3]))));
                        }
                        const uint4 f = q0[kt * 32], h = q1[kt * 32];
                        at_mma(sc[0], l4, f.x, f.y);
                        at_mma(sc[1], u4, h.x, h.y);
                        at_mma(sc[2], l4, f.z, f.w);
                        at_mma(sc[3], u4, h.z, h.w);
                    }
                    const int t = (tile0 + tile) / a.hg, hb = (tile0 + tile - t * a.hg) * 8;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if (hb + 2 * tq + j >= a.G) continue;
                        const float inv = qinv[tile * 8 + 2 * tq + j];
                        const float x0 = ((sc[0][j] + sc[1][j]) + (sc[2][j] + sc[3][j])) * inv;
                        const float x1 = ((sc[0][2 + j] + sc[1][2 + j]) + (sc[2][2 + j] + sc[3][2 + j])) * inv;
                        wild = wild || (in0 && !(fabsf(x0) < INFINITY)) || (in1 && !(fabsf(x1) < INFINITY));
                        top[0] = fmaxf(top[0], x0);
                        top[1] = fmaxf(top[1], x1);
                    }
                    if ((tile0 + tile) % a.hg != a.hg - 1 && tile != ntile - 1) continue;   // more heads of this token follow
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        top[e] = fmaxf(top[e], __shfl_xor_sync(kAll, top[e], 1));
                        top[e] = fmaxf(top[e], __shfl_xor_sync(kAll, top[e], 2));
                    }
                    if (tq == 0) {
                        float *out = a.score + (((long long)s * a.nq + t) * c.HKV + g) * c.mp;
                        const bool more = tile0 > z0;   // the token's earlier groups have left their largest
                        if (p < have) out[p] = in0 ? (more ? fmaxf(out[p], top[0]) : top[0]) : -INFINITY;
                        if (p + 8 < have) out[p + 8] = in1 ? (more ? fmaxf(out[p + 8], top[1]) : top[1]) : -INFINITY;
                    }
                    top[0] = top[1] = -INFINITY;
                }
                if (!in0) pk0 = __half2half2(__ushort_as_half(0));
                if (in1) pk0 = __hmax2(pk0, pk1);
                // FP16 bits of positive numbers keep their order
                const unsigned top16 = __reduce_max_sync(kAll, max(as_u(pk0) & 0xffffu, as_u(pk0) >> 16));
                wild = __any_sync(kAll, wild);
                if (lane == 0) {
                    const float pk = wild ? INFINITY : __half2float(__ushort_as_half((unsigned short)top16));
                    peaks[step] = tile0 > z0 ? fmaxf(peaks[step], pk) : pk;
                }
#pragma unroll
                for (int k = 0; k + 1 < SNST; k++) ids[k] = ids[k + 1];
                ids[SNST - 1] = id_of(i + SNST);
                __syncwarp();   // every lane has read this stage
            }
        }
    }
    if (!ok) {   // a copy that has not landed: what is in flight is waited for, again with a limit
        ok = true;
        while (used < copied) wait();
        if (lane == 0) {
            quit = 1;
            *(volatile unsigned *)a.err = kDevErrWaitTimeout;
        }
    }
}

__device__ __forceinline__ int block_scan_incl(int v, int *sh, int *total) {   // whole CTA, at most 1024 threads
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
    int y = lane < nw ? sh[lane] : 0, before = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(kAll, y, o);
        if (lane >= o) y += z;
    }
    *total = __shfl_sync(kAll, y, 31);
    before = __shfl_sync(kAll, y, max(w - 1, 0));
    return x + (w ? before : 0);
}

constexpr int NLIST = 64;
struct NthKey {   // shared memory of nth_key
    uint32_t buf[2][4][32];
    uint32_t list[NLIST];
    int n, found[3];
    uint32_t pub[2][3];   // this CTA's part of a sum over the cluster, by turns
};

// Who shares the keys: one CTA, or the CTAs of a cluster, which add up through each other's shared memory.
struct Solo {
    __device__ void range(NthKey &, uint32_t &, uint32_t &, int &) {}
    __device__ void add(NthKey &, uint32_t &, uint32_t &, uint32_t &) {}
    __device__ NthKey *home(NthKey &sh) { return &sh; }
    __device__ void sync() { __syncthreads(); }
};
struct Cluster {
    cooperative_groups::cluster_group g;
    int size, rank, turn;
    __device__ Cluster() : g(cooperative_groups::this_cluster()), size((int)g.num_blocks()), rank((int)g.block_rank()), turn(0) {}
    // Publishes three words of this CTA and returns lane's CTA's ones (nothing for lanes past the cluster). A word is written
    // again two turns later, behind a barrier that every reader of this turn has passed.
    __device__ bool all(NthKey &sh, uint32_t a, uint32_t b, uint32_t c, uint32_t (&out)[3]) {
        if (threadIdx.x == 0) {
            sh.pub[turn][0] = a;
            sh.pub[turn][1] = b;
            sh.pub[turn][2] = c;
        }
        g.sync();
        const int lane = threadIdx.x & 31;
        if (lane < size) {
            const uint32_t *p = g.map_shared_rank(&sh.pub[turn][0], lane);
            out[0] = p[0];
            out[1] = p[1];
            out[2] = p[2];
        }
        turn ^= 1;
        return lane < size;
    }
    __device__ void range(NthKey &sh, uint32_t &lo, uint32_t &hi, int &top) {
        if (size == 1) return;
        uint32_t v[3];
        const bool in = all(sh, lo, hi, (uint32_t)top, v);
        lo = __reduce_min_sync(kAll, in ? v[0] : kAll);
        hi = __reduce_max_sync(kAll, in ? v[1] : 0u);
        top = __reduce_add_sync(kAll, in ? (int)v[2] : 0);
    }
    __device__ void add(NthKey &sh, uint32_t &a, uint32_t &b, uint32_t &c) {
        if (size == 1) return;
        uint32_t v[3];
        const bool in = all(sh, a, b, c, v);
        a = __reduce_add_sync(kAll, in ? v[0] : 0u);
        b = __reduce_add_sync(kAll, in ? v[1] : 0u);
        c = __reduce_add_sync(kAll, in ? v[2] : 0u);
    }
    __device__ NthKey *home(NthKey &sh) { return size == 1 ? &sh : g.map_shared_rank(&sh, 0); }
    __device__ void sync() {
        if (size == 1) __syncthreads();
        else g.sync();
    }
};

// The m-th largest of n keys (n >= m >= 1), how many are larger and how many as large. A range of keys is cut into four a
// round, by the counts of the keys at least as large as each of three borders (added up in the warps, through shared memory
// and over the cluster), from the least and the largest key on, until at most NLIST keys lie in it; those are ranked directly.
// Keys of all ones stand above the range. This CTA holds `mine` of the keys: thread t the keys t, t + NT, ... in reg (anything
// past the end); keys beyond R·NT come from `more` in every round. Scores and weights fill their range evenly enough for about
// three rounds; it takes 16 at most. (Radix selection with shared-memory histograms took 3 to 4 µs a digit here, for the
// crowding of keys in few bins, its scans and four barriers each; cutting from the top bit on 0.7 µs a round, eight rounds.)
template <int NT, int R, typename Team, typename More>
__device__ __forceinline__ uint32_t nth_key(Team &team, const uint32_t (&reg)[R], int mine, int n, int m, NthKey &sh, More more,
                                            int *larger, int *equal) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    constexpr int W = NT / 32;
    uint32_t lo = kAll, hi = 0;
    int top = 0;
    auto range = [&](uint32_t k) {
        top += k == kAll;
        lo = min(lo, k);
        hi = k == kAll ? hi : max(hi, k);
    };
#pragma unroll
    for (int i = 0; i < R; i++)
        if ((int)threadIdx.x + i * NT < mine) range(reg[i]);
    for (int i = R * NT + threadIdx.x; i < mine; i += NT) range(more(i));
    lo = __reduce_min_sync(kAll, lo);
    hi = __reduce_max_sync(kAll, hi);
    top = __reduce_add_sync(kAll, top);
    if (lane == 0) {
        sh.buf[0][0][w] = lo;
        sh.buf[0][1][w] = hi;
        sh.buf[0][2][w] = top;
    }
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    lo = __reduce_min_sync(kAll, lane < W ? sh.buf[0][0][lane] : kAll);
    hi = __reduce_max_sync(kAll, lane < W ? sh.buf[0][1][lane] : 0u);
    top = __reduce_add_sync(kAll, lane < W ? (int)sh.buf[0][2][lane] : 0);
    team.range(sh, lo, hi, top);
    if (top >= m) {
        *larger = 0;
        *equal = top;
        return kAll;
    }
    int above = top, in = n - top;   // keys above hi, keys in [lo, hi]
    for (int round = 1; in > NLIST && lo < hi; round++) {
        const uint32_t d = hi - lo, a1 = lo + (d >> 2) + 1, a2 = lo + (d >> 1) + 1, a3 = lo + (d >> 1) + (d >> 2) + 1;
        uint32_t c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t k = (int)threadIdx.x + i * NT < mine ? reg[i] : 0u;   // a1 > 0
            c1 += k >= a1;
            c2 += k >= a2;
            c3 += k >= a3;
        }
        for (int i = R * NT + threadIdx.x; i < mine; i += NT) {
            const uint32_t k = more(i);
            c1 += k >= a1;
            c2 += k >= a2;
            c3 += k >= a3;
        }
        uint32_t (&buf)[4][32] = sh.buf[round & 1];
        c1 = __reduce_add_sync(kAll, c1);
        c2 = __reduce_add_sync(kAll, c2);
        c3 = __reduce_add_sync(kAll, c3);
        if (lane == 0) {
            buf[0][w] = c1;
            buf[1][w] = c2;
            buf[2][w] = c3;
        }
        __syncthreads();
        c1 = __reduce_add_sync(kAll, lane < W ? buf[0][lane] : 0u);
        c2 = __reduce_add_sync(kAll, lane < W ? buf[1][lane] : 0u);
        c3 = __reduce_add_sync(kAll, lane < W ? buf[2][lane] : 0u);
        team.add(sh, c1, c2, c3);
        const int all = in + above;   // keys of at least lo
        if ((int)c3 >= m) {
            lo = a3;
            in = (int)c3 - above;
        } else if ((int)c2 >= m) {
            lo = a2;
            hi = a3 - 1;
            in = (int)(c2 - c3);
            above = (int)c3;
        } else if ((int)c1 >= m) {
            lo = a1;
            hi = a2 - 1;
            in = (int)(c1 - c2);
            above = (int)c2;
        } else {
            hi = a1 - 1;
            in = all - (int)c1;
            above = (int)c1;
        }
    }
    if (in > NLIST) {   // equal keys
        *larger = above;
        *equal = in;
        return lo;
    }
    NthKey *home = team.home(sh);
    auto put = [&](uint32_t k) {
        if (k >= lo && k <= hi) {
            const int at = atomicAdd(&home->n, 1);
            if (at < NLIST) home->list[at] = k;   // never more
        }
    };
#pragma unroll
    for (int i = 0; i < R; i++)
        if ((int)threadIdx.x + i * NT < mine) put(reg[i]);
    for (int i = R * NT + threadIdx.x; i < mine; i += NT) put(more(i));
    team.sync();
    if (home != &sh) {
        if ((int)threadIdx.x < in) sh.list[threadIdx.x] = home->list[threadIdx.x];
        __syncthreads();
    }
    // four threads a key of the list: how many are larger, how many at least as large; the r-th is where fewer than r are
    // larger and at least r as large
    static_assert(NT >= 4 * NLIST, "a quad of threads per key");
    const int r = m - above, i = threadIdx.x >> 2;
    if (threadIdx.x < 4 * NLIST) {
        const uint32_t k = i < in ? sh.list[i] : 0u;
        int g = 0, e = 0;
#pragma unroll 4
        for (int j = threadIdx.x & 3; j < in; j += 4) {
            g += sh.list[j] > k;
            e += sh.list[j] >= k;
        }
        g += __shfl_xor_sync(kAll, g, 1);
        e += __shfl_xor_sync(kAll, e, 1);
        g += __shfl_xor_sync(kAll, g, 2);
        e += __shfl_xor_sync(kAll, e, 2);
        if ((threadIdx.x & 3) == 0 && i < in && g < r && e >= r) {   // equal keys write the same
            sh.found[0] = (int)k;
            sh.found[1] = g;
            sh.found[2] = e;
        }
    }
    __syncthreads();
    *larger = above + sh.found[1];
    *equal = sh.found[2] - sh.found[1];
    return (uint32_t)sh.found[0];
}

// Places of the hits of a CTA's items in order of their index (item i·NT + thread): exclusive sums, in place, of the counts of
// the (round, warp) pairs in cnt, N <= blockDim.x of them. Returns the total.
template <int N>
__device__ __forceinline__ int scan_counts(int *cnt, int *scan) {
    __syncthreads();   // the counts are written
    const int v = (int)threadIdx.x < N ? cnt[threadIdx.x] : 0;
    int total;
    const int x = block_scan_incl(v, scan, &total) - v;
    if ((int)threadIdx.x < N) cnt[threadIdx.x] = x;
    __syncthreads();
    return total;
}

// Adds one to hist[bin] for the lanes with in: lanes of a warp with the same bin together.
__device__ __forceinline__ void hist_add(int *hist, int bin, bool in) {
    const unsigned live = __ballot_sync(kAll, in);
    if (!in) return;
    const unsigned same = __match_any_sync(live, bin);
    if ((int)(threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&hist[bin], __popc(same));
}

// Finds the bin that holds the need-th item from the top, how many lie above it and how many in it. hist: 2·blockDim bins.
__device__ __forceinline__ void pick_bin(const int *hist, int need, int *scan, int *out) {
    const int b0 = 2 * (int)blockDim.x - 1 - 2 * (int)threadIdx.x, v0 = hist[b0], v1 = hist[b0 - 1];
    int total;
    const int incl = block_scan_incl(v0 + v1, scan, &total), above = incl - v0 - v1;
    if (above < need && incl >= need) {
        const bool second = above + v0 < need;
        out[0] = second ? b0 - 1 : b0;
        out[1] = second ? above + v0 : above;
        out[2] = second ? v1 : v0;
    }
    __syncthreads();
}

// A page's score in 64 bits, by one warp: the key of the largest over the heads h0 .. h1 - 1 (0: NaN, or no page). Both
// products are taken, each exact: where a bound is not finite the sign of the query's element does not tell the larger.
__device__ __forceinline__ unsigned long long exact_key(const SelectArgs &a, int s, int t, int g, int place, int h0, int h1) {
    const KvDev &c = a.c;
    const int lane = threadIdx.x & 31;
    const int id = page_id(c.table, c.ts, s, place, c.mp, c.n_pages);
    if (id < 0) return 0ull;
    const __half *lo = c.bounds + ((long long)id * c.HKV + g) * 2 * c.D, *hi = lo + c.D;
    double best = -INFINITY;
    bool nan = false;
    for (int h = h0; h < h1; h++) {
        const float *q = a.Q + s * a.qs + t * a.qt + (long long)(g * a.G + h) * a.qh;
        double x = 0.0;
#pragma unroll 4
        for (int d = lane; d < c.D; d += 32) {
            const double v = (double)q[d], y = v * (double)__half2float(lo[d]), z = v * (double)__half2float(hi[d]);
            x += y >= z || y != y ? y : z;
        }
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
        nan = nan || x != x;
        best = fmax(best, x);
    }
    return nan ? 0ull : score_key(best);
}

constexpr int CLIST = 512;   // pages decided by hand in shared memory
// One CTA per row (s, t, g). Keys are the FP32 scores' order-preserving bits (pages that are always taken above all); tau is
// the nsel-th largest. With E the bound of a score's error, a page above tau + 2E is taken, one below tau - 2E is not: nsel pages
// have scores of at least tau - E, and fewer than nsel more than tau + E. The pages between are ranked by their 64-bit scores.
// CR: scores a thread holds in registers, as many as the table's pages need (more are read again where they are used).
template <int CT, int CR>
__global__ void __launch_bounds__(CT) kv_choose_k(const __grid_constant__ SelectArgs a) {
    constexpr int CBITS = CT == 256 ? 9 : CT == 512 ? 10 : 11;   // of a digit of the 64-bit keys: 2·CT bins
    __shared__ NthKey nth;
    __shared__ int hist[2 * CT], scan[32], got[3];
    __shared__ int order[CR * CT / 32];
    __shared__ unsigned taken[CR * CT / 32];   // pages decided by hand, of those that registers hold
    __shared__ float red[2][CT / 32];
    __shared__ int list[CLIST];
    __shared__ unsigned long long lkey[CLIST];
    __shared__ unsigned char lnan[CLIST];
    __shared__ int sure, nlist;
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const int row = blockIdx.x, st = row / c.HKV, g = row - st * c.HKV;
    const int s = st / a.nq, t = st - s * a.nq;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int have = pages_seen(a, s, t), m = a.nsel;
    int *out = a.sel + (long long)row * m;
    if (have <= m) {
        for (int i = tid; i < m; i += CT) out[i] = i < have ? i : -1;
        return;
    }
    float *score = a.score + (long long)row * c.mp;
    auto always = [&](int p) { return p < a.first || p >= have - a.last; };
    auto key_of = [&](int p, float x) { return always(p) ? kAll : weight_key(x); };
    float x[CR];
#pragma unroll
    for (int i = 0; i < CR; i++) x[i] = tid + i * CT < have ? __ldcg(score + tid + i * CT) : 0.0f;
    // ---- E = 2^-15 · max |q|_1 · max |bound| (2^-14 for D > 128): each of a chain's D/16 tensor-core steps adds 17 numbers, each
    // cut off at worst 2^-23 below the largest, 2^-18.9 of what bounds the chain's sums; those bounds of the two chains of the
    // queries' first parts add up to |q|_1·|bound|, so that 8 steps at D = 128 make 2^-15.9. The second parts' chains are 2^-11 of
    // that, what those parts leave out 2^-21, the sums and the scale in FP32 2^-22. 2^-126 more covers what scores and E itself lose
    // where they fall below FP32's normal numbers.
    float big = 0.0f, l1 = 0.0f;
    {
        const float *peak = a.peak + (((long long)s * c.HKV + g) * a.zs + t * a.hg / a.zt) * a.unit_steps;
        for (int i = tid; i < (have + SPAGES - 1) / SPAGES; i += CT) big = fmaxf(big, __ldcg(peak + i));
        for (int h = tid; h < a.G; h += CT) l1 = fmaxf(l1, __ldcg(a.l1 + (long long)st * a.H + g * a.G + h));
        for (int o = 16; o > 0; o >>= 1) {
            big = fmaxf(big, __shfl_xor_sync(kAll, big, o));
            l1 = fmaxf(l1, __shfl_xor_sync(kAll, l1, o));
        }
        if (tid == 0) nlist = sure = 0;
        if (lane == 0) {
            red[0][warp] = big;
            red[1][warp] = l1;
        }
    }
    // ---- tau
    uint32_t key[CR];
#pragma unroll
    for (int i = 0; i < CR; i++) key[i] = tid + i * CT < have ? key_of(tid + i * CT, x[i]) : 0u;
    for (int i = tid; i < CR * CT / 32; i += CT) taken[i] = 0;
    int larger, equal;
    Solo solo;
    const uint32_t at = nth_key<CT, CR>(solo, key, have, have, m, nth, [&](int i) { return key_of(i, __ldcg(score + i)); }, &larger, &equal);
    for (int w = 0; w < CT / 32; w++) {
        big = fmaxf(big, red[0][w]);
        l1 = fmaxf(l1, red[1][w]);
    }
    const float E = (c.D > 128 ? 0x1p-14f : 0x1p-15f) * l1 * big + 0x1p-126f;
    const bool full = at == kAll;   // enough pages that are always taken: the lowest of them
    const float tau = __uint_as_float(at & 0x80000000u ? at & 0x7fffffffu : ~at);
    const bool know = E < INFINITY && at != 0u && !full;   // otherwise every page that is not always taken is ranked by hand
    // finite, so that pages taken by hand (infinity, see decide) lie above it; scores are finite where E is
    const float above = know ? fminf(tau + 2.0f * E, FLT_MAX) : FLT_MAX, below = know ? tau - 2.0f * E : -INFINITY;
    // 1: taken for sure, 0: not, -1: between
    auto side = [&](int i, float y) { return always(i) || (know && y > above) ? 1 : !know || y >= below ? -1 : 0; };
    auto decide = [&](int i, bool take) {
        if (i >= CR * CT) score[i] = take ? INFINITY : -INFINITY;
        else if (take) atomicOr(&taken[i >> 5], 1u << (i & 31));
    };
    if (!full) {
        int mine = 0;
        auto look = [&](int i, float y) {
            const int w = side(i, y);
            mine += w > 0;
            if (w < 0) {
                const int slot = atomicAdd(&nlist, 1);
                if (slot < CLIST) list[slot] = i;
            }
        };
#pragma unroll
        for (int i = 0; i < CR; i++)
            if (tid + i * CT < have) look(tid + i * CT, x[i]);
        for (int i = CR * CT + tid; i < have; i += CT) look(i, __ldcg(score + i));
        mine = __reduce_add_sync(kAll, mine);
        if (lane == 0) atomicAdd(&sure, mine);
        __syncthreads();
        const int r = m - sure, nb = nlist;   // r >= 1 of the nb pages between are taken
        if (nb <= CLIST) {
            if (nb > r) {   // a warp per (page, query head)
                for (int i = tid; i < nb; i += CT) {
                    lkey[i] = 0ull;
                    lnan[i] = 0;
                }
                __syncthreads();
                for (int i = warp; i < nb * a.G; i += CT / 32) {
                    const int e = i / a.G;
                    const unsigned long long k = exact_key(a, s, t, g, list[e], i - e * a.G, i - e * a.G + 1);
                    if (lane == 0) {
                        if (k) atomicMax(&lkey[e], k);
                        else lnan[e] = 1;
                    }
                }
            }
            __syncthreads();
            if (nb > r) {   // a NaN of one head makes the page's score NaN
                for (int i = tid; i < nb; i += CT)
                    if (lnan[i]) lkey[i] = 0ull;
                __syncthreads();
            }
            for (int i = tid; i < nb; i += CT) {
                int better = 0;
                if (nb > r)
                    for (int j = 0; j < nb; j++)
                        better += lkey[j] > lkey[i] || (lkey[j] == lkey[i] && list[j] < list[i]);
                decide(list[i], better < r);
            }
        } else {   // very many: 64-bit keys of all of them, and radix selection over these
            unsigned long long *wide = a.key + (long long)row * c.mp;
            for (int i = warp; i < have; i += CT / 32) {
                const bool in = side(i, __ldcg(score + i)) < 0;
                const unsigned long long k = in ? exact_key(a, s, t, g, i, 0, a.G) : 0ull;
                // a page of the list has a key of at least 1, so that 0 marks the others; NaN and missing pages get 1
                if (lane == 0) wide[i] = in ? max(k, 1ull) : 0ull;
            }
            __syncthreads();
            unsigned long long pre = 0, msk = 0;
            int left = r;
            for (int shift = 64 - CBITS; shift > -CBITS; shift -= CBITS) {   // 2·CT bins
                const int sh = max(shift, 0), bits = min(CBITS + shift, CBITS);
                for (int i = tid; i < 2 * CT; i += CT) hist[i] = 0;
                __syncthreads();
                for (int i = tid; i < (have + CT - 1) / CT * CT; i += CT) {
                    const unsigned long long k = i < have ? wide[i] : 0ull;
                    hist_add(hist, (int)(k >> sh) & ((1 << bits) - 1), k != 0ull && (k & msk) == pre);
                }
                __syncthreads();
                pick_bin(hist, left, scan, got);
                left -= got[1];
                pre |= (unsigned long long)got[0] << sh;
                msk |= (unsigned long long)((1 << bits) - 1) << sh;
                __syncthreads();
            }
            int eq0 = 0;
            for (int i0 = 0; i0 < have; i0 += CT) {   // ties: the lowest places
                const int i = i0 + tid;
                const unsigned long long k = i < have ? wide[i] : 0ull;
                int total;
                const int rank = block_scan_incl(k != 0ull && k == pre, scan, &total) + eq0;
                if (k != 0ull) decide(i, k > pre || (k == pre && rank <= left));
                eq0 += total;
            }
        }
        __syncthreads();   // the decided scores are written
    }
    // ---- the taken pages in order, CR·CT at a time
    int base = 0;
    for (int i0 = 0; i0 < have && base < m; i0 += CR * CT) {
        unsigned hit[CR];
#pragma unroll
        for (int i = 0; i < CR; i++) {
            const int p = i0 + i * CT + tid;
            bool take = p < have && always(p);
            if (p < have && !full) {
                if (i0 == 0) take = take || (know && x[i] > above) || (taken[p >> 5] >> (p & 31) & 1u);
                else take = take || __ldcg(score + p) > above;
            }
            hit[i] = __ballot_sync(kAll, take);
            if (lane == 0) order[i * (CT / 32) + warp] = __popc(hit[i]);
        }
        const int total = scan_counts<CR * CT / 32>(order, scan);
#pragma unroll
        for (int i = 0; i < CR; i++) {
            const int slot = base + order[i * (CT / 32) + warp] + __popc(hit[i] & ((1u << lane) - 1u));
            if ((hit[i] >> lane & 1u) && slot < m) out[slot] = i0 + i * CT + tid;
        }
        base += total;
        __syncthreads();   // the sums are read before the next counts land on them
    }
}

// ---------------------------------------------------------------------------------------------- eviction
struct EvictArgs {
    KvDev c;
    const int *len;
    int keep, first, recent, pages;
    float *acc;
    int *pos;
    long long ms, mh;
    int *src;        // [row (s, g)][keep]: the slot that moves into slot k, or -1
    int *holes;      // [row][keep]: given-up slots below keep
    int *flag;       // [row][pages]: the page loses or gets a row
    int *todo;       // [row][pages]: those pages
    int *used;       // [row][2]: slots in use, pages to do
    int *len_out;
};

// Which slots stay, and where the movers go: a cluster of 1 to 8 CTAs per row (s, g), a stretch of the slots each. The threshold
// is the keep-th largest key; then an ordered pass over the slots, ER·ET at a time: below `keep` the given-up slots are listed
// and their pages marked, from there on the j-th staying slot becomes the source of the j-th of them. A CTA of ET threads
// holds ER slots a thread in registers, those beyond are read again where they are used. As few threads as the table's slots
// need (256 rows of 2064 slots took 61 µs with 1024 threads of 16, most of them idle), and clusters for long rows (64 rows of
// 16384 slots: 31 µs with a CTA of 1024 threads each).
template <int ET, int ER>
__global__ void __launch_bounds__(ET) kv_rank_k(const __grid_constant__ EvictArgs a) {
    __shared__ NthKey nth;
    __shared__ int order[ER * ET / 32], scan[32], sh_new;
    constexpr int PAIRS = ER * ET / 32;
    Cluster team;
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const int row = blockIdx.x / team.size, s = row / c.HKV, g = row - s * c.HKV;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = min(max(a.len[s], 0), c.cap), keep = a.keep;
    const int per = ((n + team.size - 1) / team.size + 31) / 32 * 32;
    const int from = min(team.rank * per, n), mine = min(per, n - from);   // this CTA's slots: [from, from + mine)
    if (tid == 0) {
        if (team.rank == 0) {
            a.used[2 * row] = n;
            a.used[2 * row + 1] = 0;
        }
        sh_new = INT_MIN;
    }
    if (n <= keep) return;
    const float *acc = a.acc + s * a.ms + g * a.mh;
    const int *pos = a.pos ? a.pos + s * a.ms + g * a.mh : nullptr;
    int *src = a.src + (long long)row * keep, *holes = a.holes + (long long)row * keep, *flag = a.flag + (long long)row * a.pages;
    for (int i = team.rank * ET + tid; i < a.pages; i += team.size * ET) flag[i] = 0;
    uint32_t key[ER];   // the weight's key, then that with the sure ones on top
    int newest = n - 1;
    if (pos) {
        int p[ER], m = INT_MIN;
#pragma unroll
        for (int i = 0; i < ER; i++) p[i] = tid + i * ET < mine ? __ldg(pos + from + tid + i * ET) : INT_MIN;
#pragma unroll
        for (int i = 0; i < ER; i++) key[i] = tid + i * ET < mine ? weight_key(__ldg(acc + from + tid + i * ET)) : 0u;
#pragma unroll
        for (int i = 0; i < ER; i++) m = max(m, p[i]);
        for (int k = ER * ET + tid; k < mine; k += ET) m = max(m, __ldg(pos + from + k));
        m = __reduce_max_sync(kAll, m);
        __syncthreads();   // sh_new is set
        if (lane == 0) atomicMax(&sh_new, m);
        __syncthreads();
        uint32_t none = 0, big = (uint32_t)sh_new ^ 0x80000000u;   // unsigned order
        int zero = 0;
        team.range(nth, none, big, zero);
        newest = (int)(big ^ 0x80000000u);
#pragma unroll
        for (int i = 0; i < ER; i++)
            if (tid + i * ET < mine && (p[i] < a.first || p[i] > (long long)newest - a.recent)) key[i] = kAll;
    } else {
#pragma unroll
        for (int i = 0; i < ER; i++) {
            const int k = from + tid + i * ET;
            key[i] = tid + i * ET >= mine ? 0u : k < a.first || k > (long long)newest - a.recent ? kAll : weight_key(__ldg(acc + k));
        }
    }
    const long long old = (long long)newest - a.recent;
    auto key_of = [&](int k) -> uint32_t {
        const int p = pos ? __ldg(pos + k) : k;
        return p < a.first || p > old ? kAll : weight_key(__ldg(acc + k));
    };
    int larger, equal;
    const uint32_t last = nth_key<ET, ER>(team, key, mine, n, keep, nth, [&](int i) { return key_of(from + i); }, &larger, &equal);
    const int need = keep - larger;   // of the `equal` keys at the threshold the first `need` stay
    // sum of v over the CTA; then the sum over the earlier CTAs of the cluster
    auto cta_sum = [&](int v) {
        int total;
        block_scan_incl(v, scan, &total);
        return total;
    };
    auto earlier = [&](int a0, int a1, int *b0, int *b1) {
        uint32_t v[3];
        const bool in = team.all(nth, (uint32_t)a0, (uint32_t)a1, 0u, v) && lane < team.rank;
        *b0 = __reduce_add_sync(kAll, in ? (int)v[0] : 0);
        *b1 = __reduce_add_sync(kAll, in ? (int)v[1] : 0);
    };
    int eq_before = 0, eq_base = 0;
    if (equal != need && team.size > 1) {
        int e = 0;
#pragma unroll
        for (int i = 0; i < ER; i++) e += tid + i * ET < mine && key[i] == last;
        for (int i = ER * ET + tid; i < mine; i += ET) e += key_of(from + i) == last;
        int none;
        earlier(cta_sum(e), 0, &eq_before, &none);
    }
    // which of the slots from + i0 + i·ET + tid stay, bit i; advances eq_base
    auto staying = [&](int i0) -> unsigned {
        if (i0 > 0 || mine > ER * ET) {
#pragma unroll
            for (int i = 0; i < ER; i++) key[i] = i0 + i * ET + tid < mine ? key_of(from + i0 + i * ET + tid) : 0u;
        }
        unsigned stays = 0;
        if (equal == need) {
#pragma unroll
            for (int i = 0; i < ER; i++) stays |= (unsigned)(key[i] >= last && i0 + i * ET + tid < mine) << i;
            return stays;
        }
        unsigned eq[ER];
#pragma unroll
        for (int i = 0; i < ER; i++) {
            eq[i] = __ballot_sync(kAll, i0 + i * ET + tid < mine && key[i] == last);
            if (lane == 0) order[i * (ET / 32) + warp] = __popc(eq[i]);
        }
        const int total = scan_counts<PAIRS>(order, scan);
#pragma unroll
        for (int i = 0; i < ER; i++) {
            const int rank = eq_base + order[i * (ET / 32) + warp] + __popc(eq[i] & ((1u << lane) - 1u));
            stays |= (unsigned)(i0 + i * ET + tid < mine && (key[i] > last || (key[i] == last && rank < need))) << i;
        }
        eq_base += total;
        __syncthreads();   // the sums are read before the next counts land on them
        return stays;
    };
    int holes_n = 0, moved = 0;   // before this CTA's slots, then before the next of them
    if (per <= ER * ET) {         // (every CTA of the cluster) all slots in registers: the counts of both kinds share a scan
        eq_base = eq_before;
        const unsigned stays = staying(0);
        unsigned hole[ER], mover[ER];
#pragma unroll
        for (int i = 0; i < ER; i++) {
            const int k = from + i * ET + tid;
            const bool in = i * ET + tid < mine, stay = stays >> i & 1u;
            hole[i] = __ballot_sync(kAll, in && k < keep && !stay);
            mover[i] = __ballot_sync(kAll, in && k >= keep && stay);
            if (lane == 0) order[i * (ET / 32) + warp] = __popc(hole[i]) | __popc(mover[i]) << 16;   // at most ER·ET of each
            if (in && k < keep) src[k] = -1;
        }
        const int total = scan_counts<PAIRS>(order, scan);
        if (team.size > 1) earlier(total & 0xffff, total >> 16, &holes_n, &moved);
#pragma unroll
        for (int i = 0; i < ER; i++)
            if (hole[i] >> lane & 1u) {
                const int k = from + i * ET + tid;
                holes[holes_n + (order[i * (ET / 32) + warp] & 0xffff) + __popc(hole[i] & ((1u << lane) - 1u))] = k;
                flag[page_quot(c.div, k)] = 1;
            }
        team.sync();   // every hole is listed
#pragma unroll
        for (int i = 0; i < ER; i++)
            if (mover[i] >> lane & 1u) {
                const int at = moved + (order[i * (ET / 32) + warp] >> 16) + __popc(mover[i] & ((1u << lane) - 1u));
                if (at < keep) src[__ldcg(holes + at)] = from + i * ET + tid;
            }
    } else {
        if (team.size > 1) {
            int h = 0, m = 0;
            eq_base = eq_before;
            for (int i0 = 0; i0 < mine; i0 += ER * ET) {
                const unsigned stays = staying(i0);
#pragma unroll
                for (int i = 0; i < ER; i++) {
                    const int k = from + i0 + i * ET + tid;
                    h += i0 + i * ET + tid < mine && k < keep && !(stays >> i & 1u);
                    m += k >= keep && (stays >> i & 1u);
                }
            }
            h = cta_sum(h);
            m = cta_sum(m);
            earlier(h, m, &holes_n, &moved);
        }
        const int moved_base = moved;
        eq_base = eq_before;
        // two rounds over the slots: the holes, then -- once every CTA of the cluster has listed its own -- the movers
        for (int phase = 0; phase < 2; phase++) {
            if (phase) {
                eq_base = eq_before;
                moved = moved_base;
                team.sync();
            }
            for (int i0 = 0; i0 < mine; i0 += ER * ET) {
                // slots on one side of keep only have work in one of the phases
                if (phase ? from + min(i0 + ER * ET, mine) <= keep : from + i0 >= keep) {
                    if (equal != need) staying(i0);
                    continue;
                }
                const unsigned stays = staying(i0);
                unsigned hit[ER];
#pragma unroll
                for (int i = 0; i < ER; i++) {
                    const int k = from + i0 + i * ET + tid;
                    const bool in = i0 + i * ET + tid < mine, stay = stays >> i & 1u;
                    hit[i] = __ballot_sync(kAll, in && (phase ? k >= keep && stay : k < keep && !stay));
                    if (lane == 0) order[i * (ET / 32) + warp] = __popc(hit[i]);
                    if (!phase && in && k < keep) src[k] = -1;
                }
                const int total = scan_counts<PAIRS>(order, scan);
#pragma unroll
                for (int i = 0; i < ER; i++) {
                    const int k = from + i0 + i * ET + tid;
                    if (!(hit[i] >> lane & 1u)) continue;
                    const int at = (phase ? moved : holes_n) + order[i * (ET / 32) + warp] + __popc(hit[i] & ((1u << lane) - 1u));
                    if (phase) {
                        if (at < keep) src[__ldcg(holes + at)] = k;
                    } else {
                        holes[at] = k;
                        flag[page_quot(c.div, k)] = 1;
                    }
                }
                if (phase) moved += total;
                else holes_n += total;
                __syncthreads();   // the sums are read before the next counts land on them
            }
        }
    }
    team.sync();   // every page is marked, every CTA's shared memory read
    if (team.rank) return;
    // the pages that change: those with holes, and the one that held slots on both sides of keep
    int base = 0;
    for (int i0 = 0; i0 < a.pages; i0 += ER * ET) {
        unsigned hit[ER];
#pragma unroll
        for (int i = 0; i < ER; i++) {
            const int p = i0 + i * ET + tid;
            hit[i] = __ballot_sync(kAll, p < a.pages && (__ldcg(flag + p) || (p == a.pages - 1 && keep % c.page)));
            if (lane == 0) order[i * (ET / 32) + warp] = __popc(hit[i]);
        }
        const int total = scan_counts<PAIRS>(order, scan);
#pragma unroll
        for (int i = 0; i < ER; i++)
            if (hit[i] >> lane & 1u)
                a.todo[(long long)row * a.pages + base + order[i * (ET / 32) + warp] + __popc(hit[i] & ((1u << lane) - 1u))] = i0 + i * ET + tid;
        base += total;
        __syncthreads();
    }
    if (tid == 0) a.used[2 * row + 1] = base;
}

// The moves: the CTAs of a row (`ctas` of them) take its changed pages in turn, a page to `team` warps (1 or all four), which
// take its rows 4·32 / lpr at a time; lpr lanes carry a row, 16 bytes each, by asynchronous copies into a place of the lane's
// own in shared memory and out from there. The bounds of a page are taken over the rows it now holds, the movers' from their
// sources. Every source lies at or above keep and every target below, so that the order of the moves does not matter. Bound by
// memory, rows in and out, and by issuing: ranking and moves of 8 × 8 heads, 16384 -> 8192 slots in pages of 32 (335 MB) take 83.5 µs
// with four rows of a lane in flight and ten CTAs per SM (nine 86.4, but 20.9 against 21.4 µs where a few of 2064 slots go; places
// worked out for those four rows at a time 87.1; a row at a time through registers, twelve CTAs, 95.6). Pages of more than 32
// slots take the whole CTA, or 64 rows come one after the other.
constexpr int MT = 128, MCTAS = 10, MR = 4;   // threads of a CTA, CTAs of an SM, rows of a lane at once
__device__ __forceinline__ void async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(sm100::smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }
__global__ void __launch_bounds__(MT, MCTAS) kv_move_k(const __grid_constant__ EvictArgs a, int ctas, int lpr, int team) {
    __shared__ uint4 buf[MT / 32][MR][2][32];   // [warp][row of the lane][K, V][lane]; then [warp][0][least, largest][lane]
    pdl_next();
    pdl_wait();
    const KvDev &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / ctas, part = blockIdx.x - row * ctas;
    const int s = row / c.HKV, g = row - s * c.HKV, keep = a.keep;
    if (part == 0 && g == 0 && tid == 0) a.len_out[s] = min(a.used[2 * row], keep);
    const int todo = a.used[2 * row + 1], teams = MT / 32 / team, mate = warp % team;
    const int rpw = 32 / lpr, sub = lane / lpr, ch = lane - sub * lpr;   // rows of a warp at once, this lane's row, its 16 bytes
    const bool live = ch * 8 < c.D, bounds = c.bounds != nullptr;
    const int step = MR * rpw, span = team > 1 ? step : 32;   // rows of a warp at once; rows whose places are worked out at once
    for (int w = part * teams + warp / team; w < todo; w += ctas * teams) {
        const int place = a.todo[(long long)row * a.pages + w];
        const int k0 = place * c.page, rows = min(c.page, keep - k0);
        const int *src = a.src + (long long)row * keep + k0;
        const int id = page_id(c.table, c.ts, s, place, c.mp, c.n_pages);
        float *acc = a.acc + s * a.ms + g * a.mh;
        int *pos = a.pos ? a.pos + s * a.ms + g * a.mh : nullptr;
        for (int i = mate * 32 + lane; i < rows; i += team * 32) {
            const int k = src[i];
            if (k < 0) continue;
            acc[k0 + i] = acc[k];
            if (pos) pos[k0 + i] = pos[k];
        }
        if (id < 0) continue;
        uint4 mn = make_uint4(0x7c007c00u, 0x7c007c00u, 0x7c007c00u, 0x7c007c00u);   // +inf, -inf
        uint4 mx = make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
        for (int r0 = mate * span; r0 < rows; r0 += team * span) {
            // lane: the source of row r0 + lane, offsets in the pools (V: -1 where the row stays)
            long long ko = 0, vo = -1;
            if (lane < span && r0 + lane < rows) {
                const int k = __ldg(src + r0 + lane), pl = page_quot(c.div, max(k, 0));
                const int from = k >= 0 ? page_id(c.table, c.ts, s, pl, c.mp, c.n_pages) : -1;
                ko = from >= 0 ? row_at(from, k - pl * c.page, g, c.kp, c.kk, c.kh) : row_at(id, r0 + lane, g, c.kp, c.kk, c.kh);
                if (from >= 0) vo = row_at(from, k - pl * c.page, g, c.vp, c.vk, c.vh);
            }
            __half *kd = c.K + row_at(id, r0, g, c.kp, c.kk, c.kh) + ch * 8, *vd = c.V + row_at(id, r0, g, c.vp, c.vk, c.vh) + ch * 8;
            const int here = min(span, rows - r0);
            const unsigned moves = __ballot_sync(kAll, vo >= 0);   // by row
            // MR rows of each lane at once into this warp's shared memory, each lane its own 16 bytes of them, then out from there
            for (int i0 = 0; i0 < here; i0 += step) {
#pragma unroll
                for (int j = 0; j < MR; j++) {
                    const int i = i0 + j * rpw + sub;
                    const long long kr = __shfl_sync(kAll, ko, i), vr = __shfl_sync(kAll, vo, i);
                    if (i >= here || !live) continue;
                    if (bounds || vr >= 0) async16(&buf[warp][j][0][lane], c.K + kr + ch * 8);
                    if (vr >= 0) async16(&buf[warp][j][1][lane], c.V + vr + ch * 8);
                }
                async_wait();
#pragma unroll
                for (int j = 0; j < MR; j++) {
                    const int i = i0 + j * rpw + sub;
                    if (i >= here || !live || (!bounds && !(moves >> i & 1u))) continue;
                    const uint4 kv = buf[warp][j][0][lane];
                    if (moves >> i & 1u) {
                        *reinterpret_cast<uint4 *>(kd + (long long)i * c.kk) = kv;
                        *reinterpret_cast<uint4 *>(vd + (long long)i * c.vk) = buf[warp][j][1][lane];
                    }
                    if (!bounds) continue;
                    mn = least8(mn, kv);
                    mx = largest8(mx, kv);
                }
            }
        }
        if (!bounds) continue;
        for (int o = lpr; o < 32; o <<= 1) {
            mn = least8(mn, shfl8(mn, o));
            mx = largest8(mx, shfl8(mx, o));
        }
        if (team > 1) {   // the whole CTA: every warp is here
            buf[warp][0][0][lane] = mn;
            buf[warp][0][1][lane] = mx;
            __syncthreads();
            if (warp == 0)
                for (int i = 1; i < team; i++) {
                    mn = least8(mn, buf[i][0][0][lane]);
                    mx = largest8(mx, buf[i][0][1][lane]);
                }
            __syncthreads();   // the partial bounds are read before the next page's land on them
        }
        if (mate == 0 && sub == 0 && live) {
            __half *b = c.bounds + ((long long)id * c.HKV + g) * 2 * c.D + ch * 8;
            *reinterpret_cast<uint4 *>(b) = mn;
            *reinterpret_cast<uint4 *>(b + c.D) = mx;
        }
    }
}

// bytes that the acc or pos rows of all heads and streams span
size_t marks_bytes(const KvDev &c, int64_t ms, int64_t mh) {
    return ((size_t)std::max(c.ns - 1, 0) * (size_t)std::max<int64_t>(ms, 0) + (size_t)(c.HKV - 1) * (size_t)std::max<int64_t>(mh, 0) +
            (size_t)c.cap) * 4;
}
size_t bounds_bytes(const KvDev &c) { return (size_t)c.n_pages * (size_t)c.HKV * 2 * (size_t)c.D * sizeof(__half); }
// A cluster of `size` CTAs per row, with programmatic stream serialization as launch_pdl.
template <int ET, int ER>
int rank_launch(const EvictArgs &a, const KvCall &call, long long rows, int size) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * size));
    cfg.blockDim = dim3(ET);
    cfg.stream = call.st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)size;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    G9_CU(cudaLaunchKernelEx(&cfg, kv_rank_k<ET, ER>, a));
    return launched("kv_rank");
}

// One wave of CTAs, as many as shared memory lets an SM hold, and no more than there can be runs.
template <int DP>
int score_launch(const SelectArgs &a, const KvCall &call, long long most) {
    using C = ScoreCfg<DP>;
    static bool attr[kMaxDevices] = {};
    const int smem = C::smem(a.tg), per = std::max(1, 227 * 1024 / (smem + 1024 + 64));
    G9_CU(smem_limit_once(kv_score_k<DP>, C::smem(C::TG), attr));
    const unsigned ctas = (unsigned)std::min<long long>(most, (long long)std::min(per, 4) * call.d->sm_count);
    G9_CU(launch_pdl(kv_score_k<DP>, dim3(ctas), dim3(SW * 32), smem, call.st, a));
    return launched("kv_score");
}

// lanes that carry a row, 16 bytes each
int row_lanes(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }
size_t up256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace

// ---------------------------------------------------------------------------------------------- entry points
extern "C" {

GEN9BLAS_API int gen9blas_kv_supported(int D, int H, int HKV) { return shape_ok(D, H, HKV) ? 1 : 0; }

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
    G9_TRY(kv_rows_apart(c, who));
    G9_TRY(kv_marks_apart(c, acc || pos, ms, mh, who));
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
    a.tp = std::min((nt - 1) / c->page, c->mp - 1) + 2;   // nt slots from anywhere in a page; one behind the table tells bad
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
    const int lpr = row_lanes(c->D), per = std::min(nt, c->page) * lpr / 32;   // rounds of one warp over a page's rows
    const int warps = std::min(8, std::max(1, (per + 3) / 4));
    G9_CU(launch_pdl(kv_append_k, dim3((unsigned)a.tp, (unsigned)c->HKV, (unsigned)c->ns), dim3(32 * warps), 0, call.st, a, lpr));
    G9_TRY(launched("kv_append"));
    const size_t marks = marks_bytes(a.c, ms, mh);
    // positions and lengths are no early reader's operand; the bounds can be one, as the weights of a product
    const QueuedWrite w[4] = {{c->K, c->k_bytes}, {c->V, c->v_bytes}, {acc, marks}, {c->bounds, bounds_bytes(a.c)}};
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
    if (rows > INT_MAX)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %lld rows (stream, token, head) in one call", who, rows);
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
    a.hg = (a.G + 7) / 8;
    const long long tiles = (long long)nq * a.hg;
    const int dp = c->D <= 64 ? 64 : c->D <= 128 ? 128 : 256;
    // a CTA reads its pages once for as many row tiles as its shared memory holds
    const long long tg = std::min<long long>(tiles, dp == 64 ? ScoreCfg<64>::TG : dp == 128 ? ScoreCfg<128>::TG : ScoreCfg<256>::TG);
    const long long zt = a.hg > tg ? a.hg : tg / a.hg * a.hg, zs = (tiles + zt - 1) / zt;
    a.tiles = (int)tiles;
    a.tg = (int)std::min(tg, zt);
    a.zt = (int)zt;
    a.zs = (int)zs;
    a.by_zs = page_div((int)zs);
    a.unit_steps = std::max(1, (c->mp + SPAGES - 1) / SPAGES);
    const long long units = (long long)c->ns * c->HKV * zs;
    if (units * (a.unit_steps + SCOST) > INT_MAX / 2)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %lld rows of up to %d pages pass 2^30 steps in one call", who, rows, c->mp);
    if ((__int128)rows * c->mp * 12 + (__int128)c->ns * nq * H * 4 > kKvMost) return kv_too_large(who);
    const size_t score = up256((size_t)rows * c->mp * 4), key = up256((size_t)rows * c->mp * 8),
                 l1 = up256((size_t)c->ns * nq * H * 4), peak = up256((size_t)units * a.unit_steps * 4);
    void *buf = nullptr;
    unsigned *cnt = nullptr;
    G9_TRY(kv_workspace(ws, call, who, score + key + l1 + peak, 0, &buf, &cnt));
    a.score = (float *)buf;
    a.err = call.d->err_dev;
    a.key = (unsigned long long *)((char *)buf + score);
    a.l1 = (float *)((char *)buf + score + key);
    a.peak = (float *)((char *)buf + score + key + l1);
    if (c->mp > 0) {
        const long long most = (units * (a.unit_steps + SCOST) + SW - 1) / SW;
        if (dp == 64) G9_TRY(score_launch<64>(a, call, most));
        else if (dp == 128) G9_TRY(score_launch<128>(a, call, most));
        else G9_TRY(score_launch<256>(a, call, most));
    }
    const dim3 grid((unsigned)rows);
    // Threads of a row: 512; 1024 for long rows that all fit on the GPU (scoring and choosing of 128 rows of 2048 pages 37.0 µs,
    // 39.8 with 512, 41.6 with 256; 512 rows of 1500 pages 118, 104 and 153; 8 rows of 1250 pages 15.7, 14.7 and 16.7); 256
    // where they hold all (8 rows of 256 pages 11.1, 12.3 with 512). Rows longer than the registers hold read the rest again in
    // every round.
    const auto choose = [&](auto kernel, int threads) -> int {
        G9_CU(launch_pdl(kernel, grid, dim3((unsigned)threads), 0, call.st, a));
        return launched("kv_choose");
    };
    if (c->mp <= 256) G9_TRY(choose(kv_choose_k<256, 1>, 256));
    else if (c->mp <= 1024) G9_TRY(choose(kv_choose_k<512, 2>, 512));
    else if (rows <= call.d->sm_count && c->mp > 1536) {
        if (c->mp <= 2048) G9_TRY(choose(kv_choose_k<1024, 2>, 1024));
        else if (c->mp <= 4096) G9_TRY(choose(kv_choose_k<1024, 4>, 1024));
        else G9_TRY(choose(kv_choose_k<1024, 8>, 1024));
    } else if (c->mp <= 2048) G9_TRY(choose(kv_choose_k<512, 4>, 512));
    else G9_TRY(choose(kv_choose_k<512, 16>, 512));
    return kv_finish(call, sync, nullptr, 0);   // page places are no early reader's operand
}

GEN9BLAS_API int gen9blas_kv_evict(const gen9blas_kv_cache *c, const int *len, int keep, int first, int recent, float *acc,
                                   int *pos, int64_t ms, int64_t mh, int *len_out, gen9blas_kv_ws *ws, int sync) {
    const char *who = "kv_evict";
    EvictArgs a{};
    KvCall call;
    if (c && (keep < 1 || first < 0 || recent < 0 || (long long)first + recent > keep))
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: keep = %d, first = %d, recent = %d", who, keep, first, recent);
    G9_TRY(kv_rows_apart(c, who));
    G9_TRY(kv_marks_apart(c, true, ms, mh, who));
    if (int e = kv_begin(c, 0, sync, who, &a.c, &call)) return e;
    if (c->ns == 0) return 0;
    G9_TRY(kv_operand(call, len, who, "len"));
    G9_TRY(kv_operand(call, len_out, who, "len_out"));
    if (a.c.cap > 0) G9_TRY(kv_operand(call, acc, who, "acc"));
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
    a.pages = (a.keep - 1) / c->page + 1;
    if ((__int128)rows * (a.keep + a.pages) * 8 > kKvMost) return kv_too_large(who);
    const size_t list = up256((size_t)rows * a.keep * 4), pages = up256((size_t)rows * a.pages * 4);
    G9_TRY(kv_workspace(ws, call, who, 2 * list + 2 * pages + up256((size_t)rows * 8), 0, &buf, &cnt));
    a.src = (int *)buf;
    a.holes = (int *)((char *)buf + list);
    a.flag = (int *)((char *)buf + 2 * list);
    a.todo = (int *)((char *)buf + 2 * list + pages);
    a.used = (int *)((char *)buf + 2 * list + 2 * pages);
    // Clusters that hold a row's slots in registers, and larger ones while the GPU has SMs to spare for rows of 1024 slots a CTA;
    // rows of up to 8192 slots still go to one CTA of 1024 threads (256 rows of 8000: 71 µs against 89 with two of 512), as
    // do stretches beyond what eight CTAs of 512 hold (8 rows of 60000: 65 µs against 104).
    int size = 1;
    auto more = [&]() {
        if (rows * size * 2 <= call.d->sm_count && a.c.cap > 2048 * size) return true;
        return a.c.cap > 512 * 12 * size && (size > 1 || a.c.cap > 1024 * 8);
    };
    while (size < 8 && more()) size *= 2;
    if (rows * size > INT_MAX) size = 1;
    const int per = (a.c.cap + size - 1) / size;
    if (size == 1 && per <= 256 * 4) G9_TRY((rank_launch<256, 4>(a, call, rows, 1)));
    else if (per <= 512 * 6) G9_TRY((rank_launch<512, 6>(a, call, rows, size)));
    else if (per <= 512 * 9) G9_TRY((rank_launch<512, 9>(a, call, rows, size)));
    else if (per <= 512 * 12) G9_TRY((rank_launch<512, 12>(a, call, rows, size)));
    else G9_TRY((rank_launch<1024, 8>(a, call, rows, size)));
    const int team = c->page > 32 ? MT / 32 : 1, teams = MT / 32 / team;
    // a page per team, as many as can change (each mover changes one, and the last may lose slots), up to four waves of CTAs
    const long long most = std::min<long long>(a.pages, (long long)a.c.cap - a.keep + 1);
    const long long ctas = std::max<long long>(1, std::min<long long>((most + teams - 1) / teams, 4LL * MCTAS * call.d->sm_count / rows));
    const int lpr = row_lanes(c->D);
    G9_CU(launch_pdl(kv_move_k, dim3((unsigned)(rows * ctas)), dim3(MT), 0, call.st, a, (int)ctas, lpr, team));
    G9_TRY(launched("kv_move"));
    const size_t marks = marks_bytes(a.c, ms, mh);
    const QueuedWrite w[4] = {{c->K, c->k_bytes}, {c->V, c->v_bytes}, {acc, marks}, {c->bounds, bounds_bytes(a.c)}};
    return kv_finish(call, sync, w, 4);
}

}  // extern "C"

// kv_attn.cu -- attention over the paged key-value cache (gen9blas_attn_paged, include/gen9blas_kv.h): decoding and draft
// tokens, the whole cache, a window of it or chosen pages, with the weights each slot receives on request.
#include "kv.h"
#include "kv_plan.cuh"
#include "mma_sync.cuh"
#include "sm100.cuh"
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

using namespace g9;
using namespace g9kv;

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int AW = 4;        // warps of a CTA
constexpr int AKEYS = 16;    // keys of a step

// Units: a head's queries of one stream -- (stream s, key-value head g, tile of at most 8·NT rows (token, query head)) --
// or, with chosen pages, of one token. `outer` counts streams, or (stream, token) pairs; unit u = outer·inner + g·tiles +
// tile. Steps of 16 keys are counted over all units in order, fewer than 2^31 in all.
// 352 bytes: the size of a kernel's parameters moves the host's time for its launch (a call through g9kv 11.7 µs; 12.1 with 344 or
// 360 bytes, 12.7 with 384).
struct alignas(16) PagedArgs {
    KvDev c;
    int H, G, nq, dvis, window;
    int qn;                   // tokens of a unit: nq, or 1 with chosen pages
    int tiles, inner, outer;  // row tiles, HKV·tiles, streams (· nq)
    PageDiv by_g, by_tiles;
    const float *Q;
    long long qt, qh, qs;
    int q2, o4;               // pairs of a query's elements are 8-byte aligned, fours of an output's 16-byte
    const int *vis, *sel;
    int nsel, sel_steps;      // chosen pages per unit, their steps
    int *list;                // room for the entries that count: nsel for each unit, one more for each (CTA, unit)
    float qscale;             // scale · log2 e
    float *O, *lse;
    float *part;              // partial results, slot (CTA + unit)
    unsigned *cnt;            // arrivals per unit, zero before and after each launch
    float *score;             // scores in base 2 [(s, t, h)][score_row], NULL without weights
    long long score_row;
    float *lse2;              // log2 of the sum of 2^score, [(s, t, h)], with weights
};

static_assert(sizeof(PagedArgs) == 352, "see above");

constexpr float PSCALE = 64.0f;   // of the weights as FP16

// 2^x, results below 2^-126 as 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the larger one, NaN if either is
__device__ __forceinline__ float max_nan(float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}
__device__ __forceinline__ void cp16(unsigned dst, const void *src, int bytes) {   // bytes 16, or 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

template <int DP, int NT, bool W>
struct PagedCfg {
    static constexpr int ROWS = 8 * NT;                         // query rows of a unit
    static constexpr int STAGE = AKEYS * DP * 2 * 2;            // bytes of a warp's stage: K rows, V rows
    // Resident CTAs of an SM, held to by registers and shared memory: as many warps as fit serve the latencies of a step better
    // than deeper rings of fewer (D 128: three CTAs of two stages against two of three 24.9 and 26.2 µs at 8 streams of 4096
    // keys, 31.5 and 35.5 at 64 chosen pages of 16, two row tiles 185 and 201 at 64 streams of 4096; D 64: four of three against
    // two of six 79 and 107 µs at 2 streams of 131071 keys). Two row tiles of D 64: three of two 15.9 µs at 16 windows of 2048
    // keys and 114 at 64 streams of 8192, three of four 16.6 and 115, four of three 17.7 and 111, two of six 17.9 and 140.
    static constexpr int CTAS = DP == 256 ? 1 : DP == 64 && NT == 1 ? 4 : 3;
    static constexpr int NST = CTAS == 3 ? 2 : 3;
    static constexpr int RING = AW * NST * STAGE;
    static constexpr int QF = NT == 1 ? 0 : DP / 16 * NT * 32 * 16;   // query fragments, hi and lo (NT = 1: registers)
    static constexpr int KIDX = AW * NST * AKEYS * 4;
    static constexpr int ROWOFF = AW * AKEYS * 16;
    static constexpr int SMEM = RING + QF + KIDX + ROWOFF + ROWS * 4;
    // Steps that a CTA reads in the time of a segment's latencies: found with D 128 and one row tile (see where the run is cut). A
    // step of D 64 is half the bytes and one of D 256 twice; their own numbers have not been measured.
    static constexpr int COST = 16;
};

// Steps of one outer index: its slots [k0, k1) from the first visible one on, held to a multiple of a step; at least one,
// so that every unit is finished by some CTA.
template <bool SEL>
__device__ __forceinline__ int outer_steps(const PagedArgs &a, int o, int &k0, int &k1) {
    if constexpr (SEL) {
        k0 = 0;
        k1 = a.nsel * a.c.page;
        return a.sel_steps;
    }
    const int v = a.vis[o];
    k1 = seen_slots(v, a.dvis, a.nq - 1, a.c.cap);
    k0 = a.window > 0 ? first_slot(seen_slots(v, a.dvis, 0, a.c.cap), a.window) / AKEYS * AKEYS : 0;
    return max(1, (k1 - k0 + AKEYS - 1) / AKEYS);
}

// A list of chosen pages: an entry counts if it names a place of the table above every earlier entry that does, so that each page
// counts once, and in key order.
__device__ __forceinline__ int named(int e, int mp) { return e >= 0 && e < mp ? e : -1; }
// Whether the first n entries are as a selection leaves them, ascending places and what names none behind: then each that names a
// place counts. By a whole CTA of NT threads; a barrier.
template <int NT>
__device__ __forceinline__ bool list_plain(const int *sel, int n, int mp) {
    int odd = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i + 1 < n; i += NT) {
        const int x = sel[i], y = sel[i + 1];
        odd |= (int)(y >= 0) & (int)(y < mp) & (int)(x < 0 | x >= y);
    }
    return !__syncthreads_or(odd);
}
// Entry i + lane of any list, -1 where it does not count or i + lane >= n; by a whole warp.
__device__ __forceinline__ int list_counts(const int *sel, int i, int n, int mp) {
    const int lane = threadIdx.x & 31, e = i + lane < n ? named(sel[i + lane], mp) : -1;
    int top = -1, x = e;
    for (int k = lane; k < i; k += 32) top = max(top, named(sel[k], mp));
    top = __reduce_max_sync(kAll, top);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kAll, x, o);
        if (lane >= o) x = max(x, y);
    }
    const int before = __shfl_up_sync(kAll, x, 1);
    return e > max(top, lane ? before : -1) ? e : -1;
}

// The score, in base 2, of query row q (its place among all (s, t, h)) and a key row in shared memory, whose 16-byte pieces are
// exchanged by `swap`: element by element.
__device__ __forceinline__ float plain_score(const PagedArgs &a, int q, const uint8_t *key, int swap) {
    const int h = q % a.H, st = q / a.H, t = st % a.nq, s = st / a.nq;
    const float *qp = a.Q + s * a.qs + t * a.qt + h * a.qh;
    float x = 0.0f;
#pragma unroll 1
    for (int d = 0; d < a.c.D; d++) x = fmaf(qp[d], __half2float(reinterpret_cast<const __half *>(key)[((d >> 3) ^ swap) * 8 + (d & 7)]), x);
    return x * a.qscale;
}

// The same as a call, where the loop's code in line would cost the kernel registers (windows of D 64: 22.5 µs, 24.6 in line; D 256
// with two row tiles: 144.6 in line, 149.4 with the call).
__device__ __noinline__ float plain_score_call(const PagedArgs &a, int q, const uint8_t *key, int swap) { return plain_score(a, q, key, swap); }

// Elements d .. d + 3 of output row q from the sum L of its weights, the greatest score M and the sums x of PSCALE-fold weights.
__device__ __forceinline__ void paged_out(const PagedArgs &a, long long q, int d, float M, float L, float4 x) {
    const bool none = L == 0.0f;   // the row sees nothing
    const float f = none ? 0.0f : 1.0f / PSCALE / L;
    if (d < a.c.D) {
        float *out = a.O + q * a.c.D + d;
        if (a.o4) {
            *reinterpret_cast<float4 *>(out) = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
        } else {
            out[0] = x.x * f;
            out[1] = x.y * f;
            out[2] = x.z * f;
            out[3] = x.w * f;
        }
    }
    if (d == 0 && (a.lse || a.lse2)) {
        const float l2 = none ? -INFINITY : M + log2f(L);
        if (a.lse) a.lse[q] = l2 * 0.693147180559945309f;
        if (a.lse2) a.lse2[q] = l2;
    }
}

template <int DP, int NT, bool W, bool SEL>
__global__ void __launch_bounds__(AW * 32, PagedCfg<DP, NT, W>::CTAS) attn_paged_k(const __grid_constant__ PagedArgs a) {
    using C = PagedCfg<DP, NT, W>;
    constexpr int ROWS = C::ROWS, NST = C::NST, KT = DP / 16, PITCH = DP * 2;
    extern __shared__ __align__(128) uint8_t pa_sm[];
    __shared__ bool sh_last;
    __shared__ const int *sh_sel[AW];   // the unit's list, for each warp (a register pair less in the loop)
    uint8_t *ring = pa_sm;
    uint4 *qf = reinterpret_cast<uint4 *>(pa_sm + C::RING);               // [kt][nt][lane]: hi, hi, lo, lo
    int *kidx_all = reinterpret_cast<int *>(pa_sm + C::RING + C::QF);     // [warp][stage][16]: slot, INT_MAX if not visible
    longlong2 *off_all = reinterpret_cast<longlong2 *>(pa_sm + C::RING + C::QF + C::KIDX);   // [warp][16]: row offsets
    float *qinv = reinterpret_cast<float *>(pa_sm + C::RING + C::QF + C::KIDX + C::ROWOFF);   // [row]
    const KvDev &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- this CTA's run of steps. Counting a segment's latencies in (about 6 µs, COST steps; see kv_plan.cuh) took 8 streams of
    // 4096 keys from 32.4 to 26.3 µs and one stream of 1000 keys from 14.1 to 9.6.
    const Run run = find_run(a.outer, a.inner, C::COST, AW, [&](int o) {
        int k0, k1;
        return outer_steps<SEL>(a, o, k0, k1);
    });
    const int lo = run.lo, hi = run.hi, chunk = run.chunk, b = blockIdx.x;
    int outer = run.outer, pre = run.pre;

    uint8_t *wring = ring + warp * NST * C::STAGE;
    const unsigned wbase = sm100::smem_u32(wring);
    int *kidx = kidx_all + warp * NST * AKEYS;
    longlong2 *roff = off_all + warp * AKEYS;
    const int arow = (lane & 7) + ((lane >> 3) & 1) * 8, acol = lane >> 4;          // ldmatrix: K rows as A
    const int vrow = (lane & 7) + (lane >> 4) * 8, vcol = (lane >> 3) & 1;          // ldmatrix.trans: Vᵀ as A

    for (int at = lo; at < hi;) {
        int k0, k1;
        const int n = outer_steps<SEL>(a, outer, k0, k1), nv = n + C::COST, iu = (at - pre) / nv;
        if (iu >= a.inner) {
            pre += nv * a.inner;
            outer++;
            continue;
        }
        const int u = outer * a.inner + iu, us = pre + iu * nv, rs0 = us + C::COST;   // the unit's run, its first step in it
        const int sb = max(at - rs0, 0), se = min(hi - rs0, n);
        at = us + nv;
        if (se <= 0) break;   // this CTA's run ends before the unit's first step
        // the unit's nsl slots, one a CTA, follow one another from slot0 on in key order
        const int slot = b + u, slot0 = rs0 / chunk + u, nsl = (rs0 + n - 1) / chunk + u - slot0 + 1;
        const int g = page_quot(a.by_tiles, iu), row0 = (iu - g * a.tiles) * ROWS;
        const int s = SEL ? outer / a.nq : outer, t0 = SEL ? outer - s * a.nq : 0;
        const int live_rows = min(ROWS, a.qn * a.G - row0);
        const int vs = a.vis[s];
        if constexpr (SEL) {   // the entries that count, from this segment's first one to its last
            const int *sel = a.sel + ((long long)outer * c.HKV + g) * a.nsel;
            const int e0 = page_quot(c.div, sb * AKEYS), e1 = min(a.nsel, page_quot(c.div, se * AKEYS - 1) + 1);
            if (!list_plain<AW * 32>(sel, e1, c.mp)) {   // a copy: segments that follow one another share an entry at most
                int *own = a.list + (long long)u * a.nsel + slot;
                for (int e = e0 + 32 * warp; e < e1; e += 32 * AW) {
                    const int place = list_counts(sel, e, e1, c.mp);
                    if (e + lane < e1) own[e + lane] = place;
                }
                __syncthreads();
                sel = own;
            }
            if (lane == 0) sh_sel[warp] = sel;
            __syncwarp();
        }
        // lane r: row r of the unit -- the slots it sees, its query head's place among all (s, t, h)
        const int my_row = row0 + (lane < live_rows ? lane : 0), my_t = t0 + page_quot(a.by_g, my_row);
        const int my_h = g * a.G + my_row - (my_t - t0) * a.G;
        const int my_q = (s * a.nq + my_t) * a.H + my_h;
        const int my_see = seen_slots(vs, a.dvis, my_t, c.cap), my_from = first_slot(my_see, a.window);
        // slots that some row of the unit sees lie in [kmin, kmax), those that every row sees in [kmin_all, kmax_all)
        const int kmax_all = __shfl_sync(kAll, my_see, 0), kmax = __shfl_sync(kAll, my_see, live_rows - 1);
        const int kmin = __shfl_sync(kAll, my_from, 0), kmin_all = __shfl_sync(kAll, my_from, live_rows - 1);

        const int my = se > sb + warp ? (se - sb - warp + AW - 1) / AW : 0;
        // ---- this warp's i-th step: where its 16 rows lie (lane l < 16: row l), and their copies into stage i % NST
        struct Where {
            long long ko, vo;   // offsets in the pools, -1: no such row
            int k;              // its slot, INT_MAX
        };
        auto locate = [&](int i) -> Where {
            const int j = k0 + (sb + warp + AW * i) * AKEYS + (lane & 15);
            int k = INT_MAX, place = -1, slot_in = 0;
            if (i < my) {
                if constexpr (SEL) {
                    const int e = page_quot(c.div, j);
                    slot_in = j - e * c.page;
                    if (e < a.nsel) place = sh_sel[warp][e];
                    k = (int)((unsigned)place * c.page + slot_in);   // read only below mp places
                } else if (j >= kmin && j < kmax) {
                    place = page_quot(c.div, j);
                    slot_in = j - place * c.page;
                    k = j;
                }
            }
            const int id = page_id(c.table, c.ts, s, place, c.mp, c.n_pages);
            if (id < 0 || k >= kmax) return {-1, 0, INT_MAX};
            return {row_at(id, slot_in, g, c.kp, c.kk, c.kh), row_at(id, slot_in, g, c.vp, c.vk, c.vh), k};
        };
        auto copy = [&](int i, const Where &w) {
            if (i < my) {
                const int stage = i % NST;
                if (lane < 16) {
                    kidx[stage * AKEYS + lane] = w.k;
                    roff[lane] = make_longlong2(w.ko, w.vo);
                }
                __syncwarp();
                const unsigned kd = wbase + stage * C::STAGE, vd = kd + AKEYS * PITCH;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int row = q * 4 + (lane >> 3);
                    const longlong2 ro = roff[row];
#pragma unroll
                    for (int h = 0; h < DP / 64; h++) {
                        const int ch = (lane & 7) + 8 * h;
                        const int bytes = ro.x >= 0 && ch * 8 < c.D ? 16 : 0;
                        const unsigned off = row * PITCH + ((ch ^ (row & 7)) << 4);
                        cp16(kd + off, bytes ? c.K + ro.x + ch * 8 : c.K, bytes);
                        cp16(vd + off, bytes ? c.V + ro.y + ch * 8 : c.V, bytes);
                    }
                }
                __syncwarp();   // the offsets are read before the next step's land on them
            }
            cp_commit();
        };
        // the queries and the places of the first steps are requested together, then the steps themselves
        float qx[NT == 1 ? KT : 1][4];
        if constexpr (NT == 1) {   // lane: row gq, elements 16kt + 2tq + {0, 1} and + {8, 9}
            const int src = gq < live_rows ? gq : 0;
            const float *qp = a.Q + s * a.qs + __shfl_sync(kAll, my_t, src) * a.qt + __shfl_sync(kAll, my_h, src) * a.qh;
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = 16 * kt + 2 * tq + 8 * e;
                    float2 v = make_float2(0.0f, 0.0f);
                    if (gq < live_rows && d < c.D)
                        v = a.q2 ? __ldg(reinterpret_cast<const float2 *>(qp + d)) : make_float2(__ldg(qp + d), __ldg(qp + d + 1));
                    qx[kt][2 * e] = v.x;
                    qx[kt][2 * e + 1] = v.y;
                }
        }
        Where first[NST - 1];
#pragma unroll
        for (int i = 0; i < NST - 1; i++) first[i] = locate(i);
#pragma unroll
        for (int i = 0; i < NST - 1; i++) copy(i, first[i]);
        Where next = locate(NST - 1);

        // ---- query fragments (B of the scores), two FP16 parts of each row's query · 2^ex, 2^ex such that its largest
        // element lies in [2^13, 2^14): both parts keep their bits
        auto up_of = [](float big) {
            return big > 0.0f ? min(max(140 - (int)((__float_as_uint(big) >> 23) & 0xffu), -126), 126) : 0;
        };
        unsigned qr[NT == 1 ? KT : 1][4];   // NT = 1: the fragments of all tiles in registers
        float inv[NT][2];
        if constexpr (NT == 1) {
            float big = 0.0f;
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    qx[kt][e] *= a.qscale;
                    big = fmaxf(big, fabsf(qx[kt][e]));
                }
            big = fmaxf(big, __shfl_xor_sync(kAll, big, 1));
            big = fmaxf(big, __shfl_xor_sync(kAll, big, 2));
            const int ex = up_of(big);
            const float up = at_pow2(ex), down = at_pow2(-ex);
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int e = 0; e < 2; e++) at_split(qx[kt][2 * e] * up, qx[kt][2 * e + 1] * up, qr[kt][e], qr[kt][2 + e]);
            inv[0][0] = __shfl_sync(kAll, down, 8 * tq);
            inv[0][1] = __shfl_sync(kAll, down, 8 * tq + 4);
        } else {
            // each warp prepares every fourth row, all of them requested first
            constexpr int RW = ROWS / AW;
            float x[RW][DP / 32];
#pragma unroll
            for (int k = 0; k < RW; k++) {
                const int r = warp + AW * k, src = r < live_rows ? r : 0;
                const float *qp = a.Q + s * a.qs + __shfl_sync(kAll, my_t, src) * a.qt + __shfl_sync(kAll, my_h, src) * a.qh;
#pragma unroll
                for (int i = 0; i < DP / 64; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int d = 64 * i + 2 * lane + j;
                        x[k][2 * i + j] = r < live_rows && d < c.D ? __ldg(qp + d) : 0.0f;
                    }
            }
#pragma unroll
            for (int k = 0; k < RW; k++) {
                const int r = warp + AW * k;
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < DP / 32; i++) {
                    x[k][i] *= a.qscale;
                    big = fmaxf(big, fabsf(x[k][i]));
                }
                for (int i = 16; i > 0; i >>= 1) big = fmaxf(big, __shfl_xor_sync(kAll, big, i));
                const int ex = up_of(big);
                const float up = at_pow2(ex);
                if (lane == 0) qinv[r] = at_pow2(-ex);
#pragma unroll
                for (int i = 0; i < DP / 64; i++) {
                    unsigned h2, l2;
                    at_split(x[k][2 * i] * up, x[k][2 * i + 1] * up, h2, l2);
                    const int d = 64 * i + 2 * lane, kt = d >> 4, dd = d & 15;
                    unsigned *f = reinterpret_cast<unsigned *>(qf + (kt * NT + (r >> 3)) * 32 + (r & 7) * 4 + ((dd & 7) >> 1));
                    f[dd >> 3] = h2;
                    f[2 + (dd >> 3)] = l2;
                }
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) inv[nt][j] = qinv[8 * nt + 2 * tq + j];
        }
        // this lane's score columns: rows 8nt + 2tq + j, and the slots they see
        int see[NT][2], from[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int r = 8 * nt + 2 * tq + j;
                see[nt][j] = __shfl_sync(kAll, my_see, r);
                from[nt][j] = __shfl_sync(kAll, my_from, r);
                if (r >= live_rows) see[nt][j] = 0;
            }

        float *srow[2];   // one tile: the rows' scores
        if constexpr (W && NT == 1) {
#pragma unroll
            for (int j = 0; j < 2; j++) srow[j] = a.score + (long long)__shfl_sync(kAll, my_q, 2 * tq + j) * a.score_row;
        }
        float m[NT][2], l[NT][2], o[KT][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -FLT_MAX;   // no score yet: the first seen one passes it
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < KT; dt++) o[dt][nt][0] = o[dt][nt][1] = o[dt][nt][2] = o[dt][nt][3] = 0.0f;
        }
        for (int i = 0; i < my; i++) {
            cp_wait<NST - 2>();
            __syncwarp();          // every lane's part of this stage has landed; the stage before it is free
            copy(i + NST - 1, next);
            next = locate(i + NST);
            const int stage = i % NST;
            const unsigned kb = wbase + stage * C::STAGE, vb = kb + AKEYS * PITCH;
            // The tensor cores truncate as they accumulate, so the chains are kept short: the queries' second parts apart from the
            // first, and with one tile the first parts in two halves (an output's error against 64 bits at 7861 keys, D 128:
            // 1.1e-6 of its norm with one chain, 6.1e-7 with two, 3.9e-7 with three, at the same speed; three for two tiles
            // spill registers).
            constexpr int HALF = NT == 1 ? KT / 2 : KT;
            float sc[NT][4] = {}, s2[NT][4] = {}, sl[NT][4] = {};
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
                unsigned af[4];
                at_ldsm(kb + arow * PITCH + (((2 * kt + acol) ^ (arow & 7)) << 4), af);
                if constexpr (NT == 1) {
                    at_mma(kt < HALF ? sc[0] : s2[0], af, qr[kt][0], qr[kt][1]);
                    at_mma(sl[0], af, qr[kt][2], qr[kt][3]);
                } else {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const uint4 f = qf[(kt * NT + nt) * 32 + lane];
                        at_mma(sc[nt], af, f.x, f.y);
                        at_mma(sl[nt], af, f.z, f.w);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[nt][e] += HALF < KT ? s2[nt][e] + sl[nt][e] : sl[nt][e];
            const int ka = kidx[stage * AKEYS + gq], kc = kidx[stage * AKEYS + gq + 8];
            // sc[nt][2e + j]: key gq + 8e, row 8nt + 2tq + j. Most steps are seen by every row as a whole.
            const bool whole = __all_sync(kAll, min(ka, kc) >= kmin_all && max(ka, kc) < kmax_all);
            if (!whole) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if (ka >= see[nt][j] || ka < from[nt][j]) sc[nt][j] = -INFINITY;
                        if (kc >= see[nt][j] || kc < from[nt][j]) sc[nt][2 + j] = -INFINITY;
                    }
            }
            // For the weights. With one tile before the scores are looked at (8 streams of 8192 keys 51.0 µs, 51.9 behind that), with two
            // behind it (D 128, 64 streams of 4096 keys 208 µs, 214 before it).
            auto keep_scores = [&]() {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int r = 8 * nt + 2 * tq + j, at0 = k0 + (sb + warp + AW * i) * AKEYS + gq;
                        float *sr = NT == 1 ? srow[j] : a.score + (long long)__shfl_sync(kAll, my_q, r) * a.score_row;
                        if (r < live_rows && at0 < k1) sr[at0] = sc[nt][j] * inv[nt][j];
                        if (r < live_rows && at0 + 8 < k1) sr[at0 + 8] = sc[nt][2 + j] * inv[nt][j];
                    }
            };
            if constexpr (W && NT == 1) keep_scores();
            // Weights are 2^(score - m) with m a greatest score of before: it is raised, and the sums scaled down, only when
            // a score passes it by more than 8, so that most steps need no maximum over the lanes.
            float p[NT][2][2];   // of (key gq + 8e, row 8nt + 2tq + j), at most 2^8
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    p[nt][0][j] = fmaf(sc[nt][j], inv[nt][j], -m[nt][j]);
                    p[nt][1][j] = fmaf(sc[nt][2 + j], inv[nt][j], -m[nt][j]);
                    over = over || !(max_nan(p[nt][0][j], p[nt][1][j]) <= 8.0f);   // also NaN
                }
            if (__any_sync(kAll, over)) {
                // An infinite element of a key meets the query's two parts separately, and infinity times a part of zero is NaN:
                // what came out as NaN is computed again by the formula, for a score of -inf has no weight.
                bool nan = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) nan = nan || sc[nt][e] != sc[nt][e];
                if (__any_sync(kAll, nan)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {   // key gq + 8·(e / 2), row 8nt + 2tq + e % 2
                            const int r = 8 * nt + 2 * tq + (e & 1), q = __shfl_sync(kAll, my_q, r);
                            if (sc[nt][e] != sc[nt][e] && r < live_rows)
                                sc[nt][e] = (DP == 256 ? plain_score : plain_score_call)(a, q, wring + stage * C::STAGE + (gq + 8 * (e >> 1)) * PITCH, gq) / inv[nt][e & 1];
                        }
                    if constexpr (W && NT == 1) keep_scores();
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float mx = fmaxf(sc[nt][j], sc[nt][2 + j]);
                        mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 16));
                        const float mn = fmaxf(m[nt][j], mx * inv[nt][j]), alpha = ex2(m[nt][j] - mn);
                        m[nt][j] = mn;
                        l[nt][j] *= alpha;
                        p[nt][0][j] = fmaf(sc[nt][j], inv[nt][j], -mn);
                        p[nt][1][j] = fmaf(sc[nt][2 + j], inv[nt][j], -mn);
#pragma unroll
                        for (int dt = 0; dt < KT; dt++) {
                            o[dt][nt][j] *= alpha;
                            o[dt][nt][2 + j] *= alpha;
                        }
                    }
            }
            if constexpr (W && NT == 2) keep_scores();
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    p[nt][0][j] = ex2(p[nt][0][j]);
                    p[nt][1][j] = ex2(p[nt][1][j]);
                    l[nt][j] += p[nt][0][j] + p[nt][1][j];
                }
            // A slot that some rows see and others do not has weight 0 for the others, but 0·V is not 0 where V is not
            // finite: such rows of V (a sound cache has none) are added to the rows that see them by hand, then cleared.
            if (!whole) {
                // element 2·lane (and + 1) of 64 of each row: which of the 16 rows hold something that is not finite
                unsigned wild = 0;
#pragma unroll
                for (int kk = 0; kk < AKEYS; kk++)
#pragma unroll
                    for (int h = 0; h < DP / 64; h++) {
                        const unsigned w = reinterpret_cast<const unsigned *>(wring + stage * C::STAGE + (AKEYS + kk) * PITCH)[32 * h + lane];
                        if ((w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u) wild |= 1u << kk;
                    }
                wild = __reduce_or_sync(kAll, wild);
                while (wild) {
                    const int kk = __ffs(wild) - 1, key = kidx[stage * AKEYS + kk];
                    wild &= wild - 1;
                    if (key == INT_MAX || (key >= kmin_all && key < kmax_all)) continue;
                    __half *vp = reinterpret_cast<__half *>(wring + stage * C::STAGE + (AKEYS + kk) * PITCH);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float lo_p = __shfl_sync(kAll, p[nt][0][j], (kk & 7) * 4 + tq);
                            const float hi_p = __shfl_sync(kAll, p[nt][1][j], (kk & 7) * 4 + tq);
                            if (key >= see[nt][j] || key < from[nt][j]) continue;
                            const float w = (kk < 8 ? lo_p : hi_p) * PSCALE;
#pragma unroll
                            for (int dt = 0; dt < KT; dt++) {
                                o[dt][nt][j] += w * __half2float(vp[((2 * dt) ^ (kk & 7)) * 8 + gq]);
                                o[dt][nt][2 + j] += w * __half2float(vp[((2 * dt + 1) ^ (kk & 7)) * 8 + gq]);
                            }
                        }
                    __syncwarp();
                    for (int d = lane; d < DP; d += 32) vp[d] = __ushort_as_half(0);
                    __syncwarp();
                }
            }
            // the weights times 2^6 in two FP16 parts: what a weight loses is below 2^-31 of the greatest, whose weight is at
            // least 1
            unsigned bh[NT][2], bl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                unsigned h0, l0, h1, l1;
                at_split(p[nt][0][0] * PSCALE, p[nt][0][1] * PSCALE, h0, l0);
                at_split(p[nt][1][0] * PSCALE, p[nt][1][1] * PSCALE, h1, l1);
                bh[nt][0] = at_movt(h0);
                bh[nt][1] = at_movt(h1);
                bl[nt][0] = at_movt(l0);
                bl[nt][1] = at_movt(l1);
            }
            // The step's products start from zero and join the running sums by rounded FP32 operations: the tensor cores
            // truncate as they accumulate, which over hundreds of steps in a row would pass FP32's own rounding.
#pragma unroll
            for (int dt = 0; dt < KT; dt++) {
                unsigned af[4];
                at_ldsm_t(vb + vrow * PITCH + (((2 * dt + vcol) ^ (vrow & 7)) << 4), af);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    at_mma(x, af, bh[nt][0], bh[nt][1]);
                    at_mma(x, af, bl[nt][0], bl[nt][1]);
                    o[dt][nt][0] += x[0];
                    o[dt][nt][1] += x[1];
                    o[dt][nt][2] += x[2];
                    o[dt][nt][3] += x[3];
                }
            }
        }
        cp_wait<0>();
        // ---- merge the warps: into the outputs, or into this CTA's slot if other CTAs have parts of the unit too
        __syncthreads();   // every warp has left its stages
        constexpr int OP = DP + 4;
        float *mw = reinterpret_cast<float *>(ring), *lw = mw + AW * ROWS, *ow = lw + AW * ROWS;   // [warp][row], [warp][row][OP]
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = l[nt][j];
                x += __shfl_xor_sync(kAll, x, 4);
                x += __shfl_xor_sync(kAll, x, 8);
                x += __shfl_xor_sync(kAll, x, 16);
                const int r = 8 * nt + 2 * tq + j;
                if (r >= live_rows) continue;
                if (gq == 0) {
                    mw[warp * ROWS + r] = m[nt][j];
                    lw[warp * ROWS + r] = x;
                }
#pragma unroll
                for (int dt = 0; dt < KT; dt++) {
                    ow[(warp * ROWS + r) * OP + 16 * dt + gq] = o[dt][nt][j];
                    ow[(warp * ROWS + r) * OP + 16 * dt + gq + 8] = o[dt][nt][2 + j];
                }
            }
        __syncthreads();
        constexpr int PR = DP + 4;
        float *pslot = a.part + (long long)slot * ROWS * PR;   // a slot's row: greatest score, sum, 2 words, the D sums
        // each thread: elements d .. d + 3 of rows tid / (DP / 4), + RS, ...
        constexpr int RS = AW * 32 / (DP / 4);
        const int d = tid % (DP / 4) * 4;
        for (int r0 = 0; r0 < live_rows; r0 += RS) {
            const int r = min(r0 + tid / (DP / 4), ROWS - 1);
            const long long q = __shfl_sync(kAll, my_q, r);
            if (r >= live_rows) continue;
            float M = -INFINITY, L = 0.0f;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < AW; w++) M = fmaxf(M, mw[w * ROWS + r]);
            const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < AW; w++) {
                const float f = exp2f(mw[w * ROWS + r] - ref);
                const float4 y = *reinterpret_cast<const float4 *>(ow + (w * ROWS + r) * OP + d);
                L = fmaf(lw[w * ROWS + r], f, L);
                x = make_float4(fmaf(y.x, f, x.x), fmaf(y.y, f, x.y), fmaf(y.z, f, x.z), fmaf(y.w, f, x.w));
            }
            if (nsl == 1) {
                paged_out(a, q, d, M, L, x);
            } else {
                *reinterpret_cast<float4 *>(pslot + r * PR + 4 + d) = x;
                if (d == 0) *reinterpret_cast<float2 *>(pslot + r * PR) = make_float2(M, L);
            }
        }
        __syncthreads();   // the merge area is read, every slot word written
        if (nsl == 1) continue;
        if (tid == 0) {   // releases the CTA's slot (ordered before by the barrier), acquires the other CTAs'
            unsigned before;
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.cnt + u) : "memory");
            sh_last = before + 1u == (unsigned)nsl;
        }
        __syncthreads();
        if (!sh_last) continue;
        // The unit's last CTA adds up the slots in key order, SW slots of RB rows a thread at a time with their loads in flight
        // together. (A kernel of its own for it was slower: 30.1 µs against 27.8 at 8 streams of 4096 keys, the wait between
        // the kernels.)
        const float *pb = a.part + (long long)slot0 * ROWS * PR;
        constexpr int RB = NT == 1 ? 1 : 2, SW = 16 / RB;
        for (int r0 = 0; r0 < live_rows; r0 += RS * RB) {
            int r[RB];
            long long q[RB];
            float M[RB], L[RB];
            float4 x[RB];
#pragma unroll
            for (int k = 0; k < RB; k++) {
                r[k] = min(r0 + RS * k + tid / (DP / 4), ROWS - 1);
                q[k] = __shfl_sync(kAll, my_q, r[k]);
                M[k] = -INFINITY;
                L[k] = 0.0f;
                x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            for (int j0 = 0; j0 < nsl; j0 += SW) {
                float2 ml[RB][SW];
                float4 y[RB][SW];
#pragma unroll
                for (int k = 0; k < RB; k++)
#pragma unroll
                    for (int j = 0; j < SW; j++) {
                        ml[k][j] = make_float2(-INFINITY, 0.0f);
                        y[k][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (j0 + j < nsl && r[k] < live_rows) {
                            const float *p = pb + ((j0 + j) * ROWS + r[k]) * PR;
                            ml[k][j] = __ldcg(reinterpret_cast<const float2 *>(p));
                            y[k][j] = __ldcg(reinterpret_cast<const float4 *>(p + 4 + d));
                        }
                    }
#pragma unroll
                for (int k = 0; k < RB; k++) {
                    float mn = M[k];
#pragma unroll
                    for (int j = 0; j < SW; j++) mn = fmaxf(mn, ml[k][j].x);
                    const float ref = mn == -INFINITY ? 0.0f : mn, al = exp2f(M[k] - ref);
                    M[k] = mn;
                    L[k] *= al;
                    x[k] = make_float4(x[k].x * al, x[k].y * al, x[k].z * al, x[k].w * al);
#pragma unroll
                    for (int j = 0; j < SW; j++) {
                        const float f = exp2f(ml[k][j].x - ref);
                        L[k] = fmaf(ml[k][j].y, f, L[k]);
                        x[k] = make_float4(fmaf(y[k][j].x, f, x[k].x), fmaf(y[k][j].y, f, x[k].y), fmaf(y[k][j].z, f, x[k].z),
                                           fmaf(y[k][j].w, f, x[k].w));
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < RB; k++)
                if (r[k] < live_rows) paged_out(a, q[k], d, M[k], L[k], x[k]);
        }
        if (tid == 0) a.cnt[u] = 0u;   // the next call finds the counter at zero
    }
}

// The softmax weight of a score; a row whose scores are all -inf has none.
__device__ __forceinline__ float weight(float score, float l2) { return l2 == -INFINITY ? 0.0f : exp2f(score - l2); }

// acc[k] += Σ over tokens and the head's queries of 2^(score − lse2), in a fixed order. Without chosen pages a thread per
// four slots (a slot without a page has scores of -inf and gains 0); with them one CTA per (stream, head) walks the tokens
// one after the other, because their choices overlap.
__global__ void __launch_bounds__(256) kv_weigh_k(const __grid_constant__ PagedArgs a, float *acc, long long ms, long long mh, int v4) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const KvDev &c = a.c;
    const int sg = blockIdx.y, s = sg / c.HKV, g = sg - s * c.HKV;
    float *row = acc + s * ms + g * mh;
    const int vs = a.vis[s];
    if (!a.sel) {
        const int k = (blockIdx.x * 256 + threadIdx.x) * 4;
        const int k0 = first_slot(seen_slots(vs, a.dvis, 0, c.cap), a.window), k1 = seen_slots(vs, a.dvis, a.nq - 1, c.cap);
        if (k >= k1 || k + 3 < k0) return;
        const bool whole = v4 && k >= k0 && k + 3 < k1;
        float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f), sum = w;
        if (whole) w = *reinterpret_cast<const float4 *>(row + k);   // together with the scores
        for (int t = 0; t < a.nq; t++) {
            const int see = seen_slots(vs, a.dvis, t, c.cap), from = first_slot(see, a.window);
            if (k >= see || k + 3 < from) continue;
            const long long q = ((long long)s * a.nq + t) * a.H + g * a.G;
#pragma unroll 4
            for (int h = 0; h < a.G; h++) {
                const float l2 = __ldcg(a.lse2 + q + h);
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.score + (q + h) * a.score_row + k));
                // scores outside [from, see) were not written for this token where its whole step lies outside
                if (k >= from) sum.x += weight(x.x, l2);
                if (k + 1 >= from && k + 1 < see) sum.y += weight(x.y, l2);
                if (k + 2 >= from && k + 2 < see) sum.z += weight(x.z, l2);
                if (k + 3 >= from && k + 3 < see) sum.w += weight(x.w, l2);
            }
        }
        // Slots that gain nothing stay as they are, bit for bit; those behind the last one seen or before the first, which are
        // other calls' to write, are not written at all.
        auto gain = [](float w, float x) { return x == 0.0f ? w : w + x; };
        if (whole) {
            *reinterpret_cast<float4 *>(row + k) = make_float4(gain(w.x, sum.x), gain(w.y, sum.y), gain(w.z, sum.z), gain(w.w, sum.w));
        } else {
            if (sum.x != 0.0f) row[k] += sum.x;
            if (sum.y != 0.0f) row[k + 1] += sum.y;
            if (sum.z != 0.0f) row[k + 2] += sum.z;
            if (sum.w != 0.0f) row[k + 3] += sum.w;
        }
        return;
    }
    const int n = a.nsel * c.page;
    for (int t = 0; t < a.nq; t++) {
        const int see = seen_slots(vs, a.dvis, t, c.cap);
        const int *sel = a.sel + (((long long)s * a.nq + t) * c.HKV + g) * a.nsel;
        const long long q = ((long long)s * a.nq + t) * a.H + g * a.G;
        auto add = [&](int j, int e, int place) {   // no other thread has this slot: a page counts once
            if (page_id(c.table, c.ts, s, place, c.mp, c.n_pages) < 0) return;
            const int k = place * c.page + j - e * c.page;
            if (k >= see) return;
            float sum = 0.0f;
            for (int h = 0; h < a.G; h++) sum += weight(__ldcg(a.score + (q + h) * a.score_row + j), __ldcg(a.lse2 + q + h));
            row[k] += sum;
        };
        if (list_plain<256>(sel, a.nsel, c.mp)) {
            for (int j = threadIdx.x; j < n; j += 256) {
                const int e = page_quot(c.div, j);
                add(j, e, sel[e]);
            }
        } else {   // a warp per 32 entries, page by page
            for (int e0 = threadIdx.x & ~31; e0 < a.nsel; e0 += 256) {
                const int mine = list_counts(sel, e0, a.nsel, c.mp);
                for (int x = 0; x < min(32, a.nsel - e0); x++) {
                    const int place = __shfl_sync(kAll, mine, x);
                    for (int i = threadIdx.x & 31; place >= 0 && i < c.page; i += 32) add((e0 + x) * c.page + i, e0 + x, place);
                }
            }
        }
        __syncthreads();   // the next token may choose the same pages
    }
}

template <int DP, int NT, bool W, bool SEL>
int paged_one(const PagedArgs &a, const KvCall &call, bool plan, int *ctas) {
    using C = PagedCfg<DP, NT, W>;
    static bool attr[kMaxDevices] = {};
    static int occ[kMaxDevices] = {};
    if (plan) {   // the resident CTAs of the device
        G9_CU(smem_limit_once(attn_paged_k<DP, NT, W, SEL>, C::SMEM, attr));
        if (!occ[call.d->dev])
            G9_CU(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ[call.d->dev], attn_paged_k<DP, NT, W, SEL>, AW * 32, C::SMEM));
        *ctas = std::max(occ[call.d->dev], 1) * call.d->sm_count;
        return 0;
    }
    // Not launched early: the CTAs fill an SM's registers, and one that finds a CTA of the kernel before among them leaves a hole
    // too small for the last one, which then waits for a whole run (8 streams of 4193 to 8193 keys behind an append 53 µs
    // against 42, the same with weights 62 against 48). Without a wave to fill, starting early saves 0.5 µs.
    attn_paged_k<DP, NT, W, SEL><<<(unsigned)*ctas, AW * 32, C::SMEM, call.st>>>(a);
    return launched("attn_paged");
}

// Chosen pages have kernels of their own: what they take of the registers slows the others (D 128, two row tiles, weights 207 -> 224 µs).
template <int DP, int NT>
int paged_either(const PagedArgs &a, const KvCall &call, bool weights, bool plan, int *ctas) {
    if (a.sel) return weights ? paged_one<DP, NT, true, true>(a, call, plan, ctas) : paged_one<DP, NT, false, true>(a, call, plan, ctas);
    return weights ? paged_one<DP, NT, true, false>(a, call, plan, ctas) : paged_one<DP, NT, false, false>(a, call, plan, ctas);
}

// The kernel of a padded head size and a number of 8-row tiles; plan: only its resident CTAs.
int paged(int dp, int nt, const PagedArgs &a, const KvCall &call, bool weights, bool plan, int *ctas) {
    if (dp == 64)
        return nt == 1 ? paged_either<64, 1>(a, call, weights, plan, ctas) : paged_either<64, 2>(a, call, weights, plan, ctas);
    if (dp == 128)
        return nt == 1 ? paged_either<128, 1>(a, call, weights, plan, ctas) : paged_either<128, 2>(a, call, weights, plan, ctas);
    return nt == 1 ? paged_either<256, 1>(a, call, weights, plan, ctas) : paged_either<256, 2>(a, call, weights, plan, ctas);
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace

extern "C" {

GEN9BLAS_API int gen9blas_attn_paged(const gen9blas_kv_cache *c, int H, int nq, const float *Q, int64_t qt, int64_t qh,
                                     int64_t qs, const int *vis, int dvis, int window, const int *sel, int nsel, float scale,
                                     float *O, float *lse, float *acc, int64_t ms, int64_t mh, gen9blas_kv_ws *ws, int sync) {
    const char *who = "attn_paged";
    PagedArgs a{};
    KvCall call;
    if (H < 1) return GEN9BLAS_DECLINED;
    if (c && (dvis < 0 || window < 0 || nsel < 0 || (sel && window > 0)))
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: dvis = %d, window = %d, nsel = %d%s", who, dvis, window, nsel,
                    sel && window > 0 ? ": chosen pages and a window together" : "");
    if (c && sel && (long long)nsel * c->page > INT_MAX - 64)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %d chosen pages of %d slots pass 2^31", who, nsel, c->page);
    G9_TRY(kv_marks_apart(c, acc != nullptr, ms, mh, who));
    if (int e = kv_begin(c, H, sync, who, &a.c, &call)) return e;
    if (c->ns == 0 || nq <= 0) return 0;
    G9_TRY(kv_operand(call, Q, who, "Q"));
    G9_TRY(kv_operand(call, vis, who, "vis"));
    G9_TRY(kv_operand(call, O, who, "O"));
    if (sel) G9_TRY(kv_operand(call, sel, who, "sel"));
    if (lse) G9_TRY(kv_operand(call, lse, who, "lse"));
    if (acc) G9_TRY(kv_operand(call, acc, who, "acc"));
    a.H = H;
    a.G = H / c->HKV;
    a.nq = nq;
    a.dvis = dvis;
    a.window = window;
    a.Q = Q;
    a.qt = qt;
    a.qh = qh;
    a.qs = qs;
    a.vis = vis;
    a.sel = sel;
    a.nsel = sel ? nsel : 0;
    a.sel_steps = std::max(1, (int)(((long long)a.nsel * c->page + AKEYS - 1) / AKEYS));
    a.qscale = scale * 1.44269504088896341f;
    a.O = O;
    a.lse = lse;
    a.qn = sel ? 1 : nq;
    const long long rows = (long long)a.qn * a.G;
    const int dp = c->D <= 64 ? 64 : c->D <= 128 ? 128 : 256;
    // Sixteen rows a unit, or eight with the keys read once for each eight, while that is little to read (one stream of 4096
    // keys, 16 rows, D 128: 16.1 µs against 20.3; 16 streams of 1000 keys 27.2 against 24.7; two and four tokens of 8 heads
    // in 16 windows of 2048 keys, D 64: 12.6 and 17.2 against 13.9 and 15.9). Units of 32 rows were slower at every shape
    // (32 heads, 8 streams of 8192 keys 35 µs against 27; 4 tokens in the windows 20.6) but long ones of D 64 (64 streams of
    // 8192 keys, 32 rows: 105 against 115).
    const long long slots = sel ? (long long)nsel * c->page : std::min<long long>(a.c.cap, window > 0 ? (long long)window + (long long)dvis * nq : a.c.cap);
    const bool little = (__int128)c->ns * c->HKV * ((rows + 7) / 8) * slots * c->D * 4 <= 48 << 20;
    const int nt = rows <= 8 || little ? 1 : 2;
    const long long tiles = (rows + 8 * nt - 1) / (8 * nt), outer = (long long)c->ns * (sel ? nq : 1);
    // never more steps than this; they and the (s, t, h) rows are counted in 32 bits
    const long long per = (sel ? a.sel_steps : (a.c.cap + AKEYS - 1) / AKEYS + 1) + PagedCfg<64, 1, false>::COST;
    if ((__int128)outer * tiles * c->HKV * per > INT_MAX / 2 || (__int128)c->ns * nq * H > INT_MAX)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %lld (stream, token) rows of up to %lld slots pass 2^30 steps in one call", who,
                    (long long)c->ns * nq, (long long)per * AKEYS);
    a.tiles = (int)tiles;
    a.inner = (int)tiles * c->HKV;
    a.outer = (int)outer;
    a.by_g = page_div(a.G);
    a.by_tiles = page_div(a.tiles);
    a.o4 = ((uintptr_t)O & 15) == 0;
    a.q2 = ((uintptr_t)Q & 7) == 0 && ((qt | qh | qs) & 1) == 0;
    const long long units = outer * a.inner;
    int ctas = 1;
    G9_TRY(paged(dp, nt, a, call, acc != nullptr, true, &ctas));
    // never more CTAs than steps there can be
    ctas = (int)std::min<long long>(ctas, (units * per + AW - 1) / AW);
    if (acc && (long long)c->ns * c->HKV > 65535)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: weights of %lld (stream, head) rows in one call", who, (long long)c->ns * c->HKV);
    if (((__int128)ctas + units) * 8 * nt * (dp + 4) * 4 > kKvMost) return kv_too_large(who);
    const size_t part = up256((size_t)(ctas + units) * 8 * nt * (dp + 4) * 4);
    const long long heads = (long long)c->ns * nq * H;
    a.score_row = ((sel ? (long long)a.nsel * c->page : a.c.cap) + 3) / 4 * 4;   // rows of whole float4
    const size_t lse2 = acc ? up256((size_t)heads * 4) : 0;
    if (acc && (__int128)heads * a.score_row * 4 > kKvMost) return kv_too_large(who);
    const size_t score = acc ? up256((size_t)heads * a.score_row * 4) : 0;
    if ((__int128)units * a.nsel * 4 > kKvMost) return kv_too_large(who);
    const size_t list = sel ? up256(((size_t)units * a.nsel + ctas + units) * 4) : 0;
    void *buf = nullptr;
    G9_TRY(kv_workspace(ws, call, who, part + lse2 + score + list, (size_t)units, &buf, &a.cnt));
    if (sel) a.list = (int *)((char *)buf + part + lse2 + score);
    a.part = (float *)buf;
    if (c->n_pages == 0) a.c.K = a.c.V = (__half *)buf;   // named by copies of no bytes
    if (acc) {
        a.lse2 = (float *)((char *)buf + part);
        a.score = (float *)((char *)buf + part + lse2);
    }
    G9_TRY(paged(dp, nt, a, call, acc != nullptr, false, &ctas));
    if (acc && a.score_row > 0) {
        const dim3 grid(sel ? 1u : (unsigned)((a.c.cap + 1023) / 1024), (unsigned)(c->ns * c->HKV));
        const int v4 = ((uintptr_t)acc & 15) == 0 && ((ms | mh) & 3) == 0;
        G9_CU(launch_pdl(kv_weigh_k, grid, dim3(256), 0, call.st, a, acc, (long long)ms, (long long)mh, v4));
        G9_TRY(launched("kv_weigh"));
    }
    const size_t marks = ((size_t)(c->ns - 1) * (size_t)std::max<int64_t>(ms, 0) +
                          (size_t)(c->HKV - 1) * (size_t)std::max<int64_t>(mh, 0) + (size_t)a.c.cap) * 4;
    const QueuedWrite w[3] = {{O, (size_t)heads * c->D * 4}, {lse, (size_t)heads * 4}, {acc, marks}};
    return kv_finish(call, sync, w, 3);
}

}  // extern "C"

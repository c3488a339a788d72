// kv_attn.cu -- attention over the paged key-value cache (gen9blas_attn_paged, include/gen9blas_kv.h): decoding and draft
// tokens, the whole cache, a window of it or chosen pages, with the weights each slot receives on request.
#include "kv.h"
#include "mma_sync.cuh"
#include "sm100.cuh"
#include <algorithm>
#include <climits>
#include <cmath>

using namespace g9;
using namespace g9kv;

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int AW = 4;        // warps of a CTA
constexpr int AKEYS = 16;    // keys of a step

// Units: a head's queries of one stream -- (stream s, key-value head g, tile of at most 8·NT rows (token, query head)) --
// or, with chosen pages, of one token. `outer` counts streams, or (stream, token) pairs; unit u = outer·inner + (tile, g).
struct PagedArgs {
    KvDev c;
    int H, G, nq, dvis, window;
    int qn;                   // tokens of a unit: nq, or 1 with chosen pages
    int tiles, inner, outer;  // row tiles, HKV·tiles, streams (· nq)
    const float *Q;
    long long qt, qh, qs;
    const int *vis, *sel;
    int nsel, sel_steps;      // chosen pages per unit, their steps
    float qscale;             // scale · log2 e
    float *O, *lse;
    float *part;              // partial results, slot (CTA + unit)
    unsigned *cnt;            // arrivals per unit, zero before and after each launch
    float *score;             // scores in base 2 [(s, t, h)][score_row], NULL without weights
    long long score_row;
    float *lse2;              // log2 of the sum of 2^score, [(s, t, h)], with weights
};

__device__ __forceinline__ void cp16(unsigned dst, const void *src, int bytes) {   // bytes 16, or 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

template <int DP, int NT>
struct PagedCfg {
    static constexpr int ROWS = 8 * NT;                         // query rows of a unit
    static constexpr int STAGE = AKEYS * DP * 2 * 2;            // bytes of a warp's stage: K rows, V rows
    static constexpr int NST = DP == 64 ? 6 : 3;
    static constexpr int RING = AW * NST * STAGE;
    static constexpr int QF = DP / 16 * NT * 32 * 16;           // query fragments, hi and lo
    static constexpr int KIDX = AW * NST * AKEYS * 4;
    static constexpr int SMEM = RING + QF + KIDX + ROWS * 4;
    static constexpr int CTAS = DP == 256 ? 1 : 2;
};

// Steps of one outer index: its slots from the first visible one, held to a multiple of a step; at least one, so that
// every unit is finished by some CTA.
__device__ __forceinline__ int outer_steps(const PagedArgs &a, int o, int &k0, int &k1) {
    if (a.sel) {
        k0 = 0;
        k1 = a.nsel * a.c.page;
        return a.sel_steps;
    }
    const int v = a.vis[o];
    k1 = seen_slots(v, a.dvis, a.nq - 1, a.c.cap);
    k0 = first_slot(seen_slots(v, a.dvis, 0, a.c.cap), a.window) / AKEYS * AKEYS;
    return max(1, (k1 - k0 + AKEYS - 1) / AKEYS);
}

template <int DP, int NT>
__global__ void __launch_bounds__(AW * 32, PagedCfg<DP, NT>::CTAS) attn_paged_k(const __grid_constant__ PagedArgs a) {
    using C = PagedCfg<DP, NT>;
    constexpr int ROWS = C::ROWS, NST = C::NST, KT = DP / 16, PITCH = DP * 2;
    extern __shared__ __align__(128) uint8_t pa_sm[];
    uint8_t *ring = pa_sm;
    uint4 *qf = reinterpret_cast<uint4 *>(pa_sm + C::RING);               // [kt][nt][lane]: hi, hi, lo, lo
    int *kidx_all = reinterpret_cast<int *>(pa_sm + C::RING + C::QF);     // [warp][stage][16]: slot, INT_MAX if not visible
    float *qinv = reinterpret_cast<float *>(pa_sm + C::RING + C::QF + C::KIDX);   // [row]
    __shared__ long long sh_tot[AW];
    __shared__ long long sh_pre;
    __shared__ int sh_outer;
    __shared__ bool sh_last;
    const KvDev &c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- this CTA's steps [lo, hi) of all T, and the outer index that holds lo
    long long T = 0;
    if (a.sel) {
        T = (long long)a.outer * a.inner * a.sel_steps;
    } else {
        long long mine = 0;
        for (int o = tid; o < a.outer; o += AW * 32) {
            int k0, k1;
            mine += (long long)outer_steps(a, o, k0, k1) * a.inner;
        }
        for (int i = 16; i > 0; i >>= 1) mine += __shfl_xor_sync(kAll, mine, i);
        if (lane == 0) sh_tot[warp] = mine;
        __syncthreads();
        for (int w = 0; w < AW; w++) T += sh_tot[w];
    }
    const long long B = min((long long)gridDim.x, (T + AW - 1) / AW), b = blockIdx.x;
    if (b >= B) return;
    const long long lo = b * T / B, hi = (b + 1) * T / B;
    if (a.sel) {
        if (tid == 0) {
            const long long per = (long long)a.inner * a.sel_steps;
            sh_outer = (int)(lo / per);
            sh_pre = lo / per * per;
        }
    } else {
        long long run = 0;
        for (int o0 = 0; o0 < a.outer; o0 += AW * 32) {
            const int o = o0 + tid;
            long long n = 0;
            if (o < a.outer) {
                int k0, k1;
                n = (long long)outer_steps(a, o, k0, k1) * a.inner;
            }
            long long x = n;
            for (int i = 1; i < 32; i <<= 1) {
                const long long y = __shfl_up_sync(kAll, x, i);
                if (lane >= i) x += y;
            }
            __syncthreads();
            if (lane == 31) sh_tot[warp] = x;
            __syncthreads();
            long long before = run;
            for (int w = 0; w < warp; w++) before += sh_tot[w];
            if (lo >= before + x - n && lo < before + x) {
                sh_outer = o;
                sh_pre = before + x - n;
            }
            for (int w = 0; w < AW; w++) run += sh_tot[w];
            if (lo < run) break;
        }
    }
    __syncthreads();
    int outer = sh_outer;
    long long pre = sh_pre;   // steps before this outer index

    uint8_t *wring = ring + warp * NST * C::STAGE;
    const unsigned wbase = sm100::smem_u32(wring);
    int *kidx = kidx_all + warp * NST * AKEYS;
    const int arow = (lane & 7) + ((lane >> 3) & 1) * 8, acol = lane >> 4;          // ldmatrix: K rows as A
    const int vrow = (lane & 7) + (lane >> 4) * 8, vcol = (lane >> 3) & 1;          // ldmatrix.trans: Vᵀ as A

    for (long long at = lo; at < hi;) {
        int k0, k1;
        const int n = outer_steps(a, outer, k0, k1);
        const long long in = (at - pre) / n;
        if (in >= a.inner) {
            pre += (long long)n * a.inner;
            outer++;
            continue;
        }
        const int iu = (int)in;
        const long long u = (long long)outer * a.inner + iu, rs0 = pre + (long long)iu * n;
        const int sb = (int)(at - rs0), se = (int)(min(hi, rs0 + n) - rs0);
        at = rs0 + se;
        const int g = iu / a.tiles, row0 = (iu - g * a.tiles) * ROWS;
        const int s = a.sel ? outer / a.nq : outer, t0 = a.sel ? outer - s * a.nq : 0;
        const int live_rows = min(ROWS, a.qn * a.G - row0);
        const int vs = a.vis[s];
        const int *sel = a.sel ? a.sel + ((long long)outer * c.HKV + g) * a.nsel : nullptr;
        // slots that some row of the unit sees lie in [kmin, kmax), those that every row sees in [kmin_all, kmax_all)
        const int tf = t0 + row0 / a.G, tl = t0 + (row0 + live_rows - 1) / a.G;
        const int kmax_all = seen_slots(vs, a.dvis, tf, c.cap), kmax = seen_slots(vs, a.dvis, tl, c.cap);
        const int kmin = first_slot(kmax_all, a.window), kmin_all = first_slot(kmax, a.window);

        // ---- query fragments: each warp prepares every fourth row
        for (int r = warp; r < ROWS; r += AW) {
            const bool live = r < live_rows;
            const int t = t0 + (live ? (row0 + r) / a.G : 0), h = g * a.G + (live ? (row0 + r) % a.G : 0);
            const float *qp = a.Q + s * a.qs + t * a.qt + h * a.qh;
            float x[DP / 32], big = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 64; i++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int d = 64 * i + 2 * lane + j;
                    x[2 * i + j] = live && d < c.D ? qp[d] * a.qscale : 0.0f;
                    big = fmaxf(big, fabsf(x[2 * i + j]));
                }
            }
            for (int i = 16; i > 0; i >>= 1) big = fmaxf(big, __shfl_xor_sync(kAll, big, i));
            int ex = 0;   // the row's largest |q| · 2^ex lies in [2^13, 2^14): both FP16 parts keep their bits
            if (big > 0.0f) ex = min(max(140 - (int)((__float_as_uint(big) >> 23) & 0xffu), -126), 126);
            const float up = at_pow2(ex);
            if (lane == 0) qinv[r] = at_pow2(-ex);
#pragma unroll
            for (int i = 0; i < DP / 64; i++) {
                unsigned h2, l2;
                at_split(x[2 * i] * up, x[2 * i + 1] * up, h2, l2);
                const int d = 64 * i + 2 * lane, kt = d >> 4, dd = d & 15;
                unsigned *f = reinterpret_cast<unsigned *>(qf + (kt * NT + (r >> 3)) * 32 + (r & 7) * 4 + ((dd & 7) >> 1));
                f[dd >> 3] = h2;
                f[2 + (dd >> 3)] = l2;
            }
        }
        // this lane's score columns: rows 8nt + 2tq + j, and the slots they see
        int see[NT][2], from[NT][2];
        float *srow[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int r = 8 * nt + 2 * tq + j;
                see[nt][j] = from[nt][j] = 0;
                srow[nt][j] = nullptr;
                if (r < live_rows) {
                    const int t = t0 + (row0 + r) / a.G, h = g * a.G + (row0 + r) % a.G;
                    see[nt][j] = seen_slots(vs, a.dvis, t, c.cap);
                    from[nt][j] = first_slot(see[nt][j], a.window);
                    if (a.score) srow[nt][j] = a.score + (((long long)s * a.nq + t) * a.H + h) * a.score_row;
                }
            }
        __syncthreads();
        float inv[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) inv[nt][j] = qinv[8 * nt + 2 * tq + j];

        const int my = se > sb + warp ? (se - sb - warp + AW - 1) / AW : 0;
        // ---- copies of this warp's i-th step into stage i % NST
        auto issue = [&](int i) {
            if (i < my) {
                const int stage = i % NST, j = k0 + (sb + warp + AW * i) * AKEYS + (lane & 15);
                long long ko = -1, vo = 0;
                int k = INT_MAX;
                if (sel) {
                    const int e = page_quot(c.div, j), slot = j - e * c.page;
                    if (e < a.nsel) {
                        const int place = sel[e];
                        if (place >= 0 && (e == 0 || place > sel[e - 1])) {
                            const int id = page_id(c.table, c.ts, s, place, c.mp, c.n_pages);
                            const int kk = place * c.page + slot;   // id < 0 when place is not below mp
                            if (id >= 0 && kk < kmax) {
                                k = kk;
                                ko = row_at(id, slot, g, c.kp, c.kk, c.kh);
                                vo = row_at(id, slot, g, c.vp, c.vk, c.vh);
                            }
                        }
                    }
                } else if (j >= kmin && j < kmax) {
                    const int place = page_quot(c.div, j), slot = j - place * c.page;
                    const int id = page_id(c.table, c.ts, s, place, c.mp, c.n_pages);
                    if (id >= 0) {
                        k = j;
                        ko = row_at(id, slot, g, c.kp, c.kk, c.kh);
                        vo = row_at(id, slot, g, c.vp, c.vk, c.vh);
                    }
                }
                if (lane < 16) kidx[stage * AKEYS + lane] = k;
                const unsigned kd = wbase + stage * C::STAGE, vd = kd + AKEYS * PITCH;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int row = q * 4 + (lane >> 3);
                    const long long kr = __shfl_sync(kAll, ko, row), vr = __shfl_sync(kAll, vo, row);
#pragma unroll
                    for (int h = 0; h < DP / 64; h++) {
                        const int ch = (lane & 7) + 8 * h;
                        const int bytes = kr >= 0 && ch * 8 < c.D ? 16 : 0;
                        const unsigned off = row * PITCH + ((ch ^ (row & 7)) << 4);
                        cp16(kd + off, bytes ? c.K + kr + ch * 8 : c.K, bytes);
                        cp16(vd + off, bytes ? c.V + vr + ch * 8 : c.V, bytes);
                    }
                }
            }
            cp_commit();
        };

        float m[NT][2], l[NT][2], o[KT][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < KT; dt++) o[dt][nt][0] = o[dt][nt][1] = o[dt][nt][2] = o[dt][nt][3] = 0.0f;
        }
        for (int i = 0; i < NST - 1; i++) issue(i);
        for (int i = 0; i < my; i++) {
            cp_wait<NST - 2>();
            __syncwarp();          // every lane's part of this stage has landed; the stage before it is free
            issue(i + NST - 1);
            const int stage = i % NST;
            const unsigned kb = wbase + stage * C::STAGE, vb = kb + AKEYS * PITCH;
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
                unsigned af[4];
                at_ldsm(kb + arow * PITCH + (((2 * kt + acol) ^ (arow & 7)) << 4), af);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const uint4 f = qf[(kt * NT + nt) * 32 + lane];
                    at_mma(sc[nt], af, f.x, f.y);
                    at_mma(sc[nt], af, f.z, f.w);
                }
            }
            const int ka = kidx[stage * AKEYS + gq], kc = kidx[stage * AKEYS + gq + 8];
            float p[NT][2][2], alpha[NT][2];   // weight of (key gq or gq + 8, row 8nt + 2tq + j)
            bool moved = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float x0 = ka < see[nt][j] && ka >= from[nt][j] ? sc[nt][j] * inv[nt][j] : -INFINITY;
                    const float x1 = kc < see[nt][j] && kc >= from[nt][j] ? sc[nt][2 + j] * inv[nt][j] : -INFINITY;
                    if (srow[nt][j]) {
                        const int at0 = k0 + (sb + warp + AW * i) * AKEYS + gq;
                        if (at0 < k1) srow[nt][j][at0] = x0;
                        if (at0 + 8 < k1) srow[nt][j][at0 + 8] = x1;
                    }
                    float mx = fmaxf(x0, x1);
                    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 16));
                    const float mn = fmaxf(m[nt][j], mx), ref = mn == -INFINITY ? 0.0f : mn;
                    alpha[nt][j] = exp2f(m[nt][j] - ref);
                    moved = moved || mn != m[nt][j];
                    m[nt][j] = mn;
                    p[nt][0][j] = exp2f(x0 - ref);
                    p[nt][1][j] = exp2f(x1 - ref);
                    l[nt][j] = fmaf(l[nt][j], alpha[nt][j], p[nt][0][j] + p[nt][1][j]);
                }
            if (__any_sync(kAll, moved)) {
#pragma unroll
                for (int dt = 0; dt < KT; dt++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        o[dt][nt][0] *= alpha[nt][0];
                        o[dt][nt][1] *= alpha[nt][1];
                        o[dt][nt][2] *= alpha[nt][0];
                        o[dt][nt][3] *= alpha[nt][1];
                    }
            }
            // A slot that some rows see and others do not has weight 0 for the others, but 0·V is not 0 where V is not
            // finite: such rows of V (a sound cache has none) are added to the rows that see them by hand, then cleared.
            const bool odd = (ka != INT_MAX && (ka < kmin_all || ka >= kmax_all)) ||
                             (kc != INT_MAX && (kc < kmin_all || kc >= kmax_all));
            if (__any_sync(kAll, odd)) {
                for (int kk = 0; kk < AKEYS; kk++) {
                    const int key = kidx[stage * AKEYS + kk];
                    if (key == INT_MAX || (key >= kmin_all && key < kmax_all)) continue;
                    __half *vp = reinterpret_cast<__half *>(wring + stage * C::STAGE + (AKEYS + kk) * PITCH);
                    bool wild = false;
                    for (int d = lane; d < DP; d += 32) wild = wild || (__half_as_ushort(vp[d]) & 0x7c00) == 0x7c00;
                    if (!__any_sync(kAll, wild)) continue;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float lo_p = __shfl_sync(kAll, p[nt][0][j], (kk & 7) * 4 + tq);
                            const float hi_p = __shfl_sync(kAll, p[nt][1][j], (kk & 7) * 4 + tq);
                            if (key >= see[nt][j] || key < from[nt][j]) continue;
                            const float w = (kk < 8 ? lo_p : hi_p) * 16384.0f;
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
            // weights of up to 1 as up to 2^14, in two FP16 parts: what a weight loses is below 2^-39 of the largest
            unsigned bh[NT][2], bl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                unsigned h0, l0, h1, l1;
                at_split(p[nt][0][0] * 16384.0f, p[nt][0][1] * 16384.0f, h0, l0);
                at_split(p[nt][1][0] * 16384.0f, p[nt][1][1] * 16384.0f, h1, l1);
                bh[nt][0] = at_movt(h0);
                bh[nt][1] = at_movt(h1);
                bl[nt][0] = at_movt(l0);
                bl[nt][1] = at_movt(l1);
            }
#pragma unroll
            for (int dt = 0; dt < KT; dt++) {
                unsigned af[4];
                at_ldsm_t(vb + vrow * PITCH + (((2 * dt + vcol) ^ (vrow & 7)) << 4), af);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    at_mma(o[dt][nt], af, bh[nt][0], bh[nt][1]);
                    at_mma(o[dt][nt], af, bl[nt][0], bl[nt][1]);
                }
            }
        }
        cp_wait<0>();
        // ---- merge the warps (and other CTAs' parts of the unit, if any)
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
        const long long b0 = cta_of(rs0, T, B), b1 = cta_of(rs0 + n - 1, T, B);
        const int nsl = (int)(b1 - b0 + 1);
        constexpr int SLOT = ROWS * (DP + 2);
        float *pslot = a.part + (b + u) * SLOT;
        // row r, element d of the result from sum L, greatest M and the sum x of 2^14-fold weights
        auto finish = [&](int r, int d, float M, float L, float x) {
            const int t = t0 + (row0 + r) / a.G, h = g * a.G + (row0 + r) % a.G;
            const long long q = ((long long)s * a.nq + t) * a.H + h;
            const bool none = M == -INFINITY;
            if (d < c.D) a.O[q * c.D + d] = none ? 0.0f : x * (1.0f / 16384.0f) / L;
            if (d == 0) {
                const float l2 = none ? -INFINITY : M + log2f(L);
                if (a.lse) a.lse[q] = l2 * 0.693147180559945309f;
                if (a.lse2) a.lse2[q] = l2;
            }
        };
        for (int i = tid; i < live_rows * DP; i += AW * 32) {
            const int r = i / DP, d = i - r * DP;
            float M = mw[r];
#pragma unroll
            for (int w = 1; w < AW; w++) M = fmaxf(M, mw[w * ROWS + r]);
            const float ref = M == -INFINITY ? 0.0f : M;
            float L = 0.0f, x = 0.0f;
#pragma unroll
            for (int w = 0; w < AW; w++) {
                const float f = exp2f(mw[w * ROWS + r] - ref);
                L = fmaf(lw[w * ROWS + r], f, L);
                x = fmaf(ow[(w * ROWS + r) * OP + d], f, x);
            }
            if (nsl == 1) {
                finish(r, d, M, L, x);
            } else {
                pslot[r * (DP + 2) + 2 + d] = x;
                if (d == 0) {
                    pslot[r * (DP + 2)] = M;
                    pslot[r * (DP + 2) + 1] = L;
                }
            }
        }
        __syncthreads();   // the merge area is read, every slot word written
        if (nsl == 1) continue;
        if (tid == 0) {
            __threadfence();   // release of the CTA's slot (ordered before by the barrier)
            sh_last = atomicAdd(a.cnt + u, 1u) + 1u == (unsigned)nsl;
            __threadfence();   // acquire of the other CTAs' slots
        }
        __syncthreads();
        if (!sh_last) continue;
        const float *pb = a.part + (b0 + u) * SLOT;   // the unit's slots follow one another in key order
        float *wm = reinterpret_cast<float *>(ring), *hm = wm + (size_t)nsl * live_rows, *hl = hm + ROWS;   // [row][slot] weights
        for (int r = warp; r < live_rows; r += AW) {
            float M = -INFINITY, L = 0.0f;
            for (int j = lane; j < nsl; j += 32) M = fmaxf(M, __ldcg(pb + (long long)j * SLOT + r * (DP + 2)));
            for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, i));
            const float ref = M == -INFINITY ? 0.0f : M;
            for (int j = lane; j < nsl; j += 32) {
                const float *p = pb + (long long)j * SLOT + r * (DP + 2);
                const float f = exp2f(__ldcg(p) - ref);
                wm[r * nsl + j] = f;
                L = fmaf(__ldcg(p + 1), f, L);
            }
            for (int i = 16; i > 0; i >>= 1) L += __shfl_xor_sync(kAll, L, i);
            if (lane == 0) {
                hm[r] = M;
                hl[r] = L;
            }
        }
        __syncthreads();
        for (int i = tid; i < live_rows * DP; i += AW * 32) {
            const int r = i / DP, d = i - r * DP;
            const float *p = pb + r * (DP + 2) + 2 + d;
            float x = 0.0f;
#pragma unroll 8
            for (int j = 0; j < nsl; j++) x = fmaf(__ldcg(p + (long long)j * SLOT), wm[r * nsl + j], x);
            finish(r, d, hm[r], hl[r], x);
        }
        if (tid == 0) a.cnt[u] = 0u;   // the next call finds the counter at zero
        __syncthreads();               // the weights are read before the next unit's copies land on them
    }
}

// The softmax weight of score `at` of a row; a row whose scores are all -inf has none.
__device__ __forceinline__ float weight(const PagedArgs &a, long long row, int at) {
    const float l2 = __ldcg(a.lse2 + row);
    return l2 == -INFINITY ? 0.0f : exp2f(__ldcg(a.score + row * a.score_row + at) - l2);
}

// acc[k] += Σ over tokens and the head's queries of 2^(score − lse2), in a fixed order. Without chosen pages a thread per
// slot; with them one CTA per (stream, head) walks the tokens one after the other, because their choices overlap.
__global__ void __launch_bounds__(256) kv_weigh_k(const __grid_constant__ PagedArgs a, float *acc, long long ms, long long mh) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const KvDev &c = a.c;
    const long long sg = blockIdx.y;
    const int s = (int)(sg / c.HKV), g = (int)(sg % c.HKV);
    float *row = acc + s * ms + g * mh;
    const int vs = a.vis[s];
    if (!a.sel) {
        const int k = blockIdx.x * 256 + threadIdx.x;
        if (k >= seen_slots(vs, a.dvis, a.nq - 1, c.cap)) return;
        if (page_id(c.table, c.ts, s, page_quot(c.div, k), c.mp, c.n_pages) < 0) return;
        float sum = 0.0f;
        for (int t = 0; t < a.nq; t++) {
            const int see = seen_slots(vs, a.dvis, t, c.cap);
            if (k >= see || k < first_slot(see, a.window)) continue;
            const long long q = ((long long)s * a.nq + t) * a.H + g * a.G;
            for (int h = 0; h < a.G; h++) sum += weight(a, q + h, k);
        }
        row[k] += sum;
        return;
    }
    const int n = a.nsel * c.page;
    for (int t = 0; t < a.nq; t++) {
        const int see = seen_slots(vs, a.dvis, t, c.cap);
        const int *sel = a.sel + (((long long)s * a.nq + t) * c.HKV + g) * a.nsel;
        const long long q = ((long long)s * a.nq + t) * a.H + g * a.G;
        for (int j = threadIdx.x; j < n; j += 256) {
            const int e = page_quot(c.div, j), place = sel[e];
            if (place < 0 || (e > 0 && place <= sel[e - 1])) continue;
            if (page_id(c.table, c.ts, s, place, c.mp, c.n_pages) < 0) continue;
            const int k = place * c.page + j - e * c.page;
            if (k >= see) continue;
            float sum = 0.0f;
            for (int h = 0; h < a.G; h++) sum += weight(a, q + h, j);
            row[k] += sum;
        }
        __syncthreads();   // the next token may choose the same pages
    }
}

template <int DP, int NT>
int paged_run(const PagedArgs &a, const KvCall &call, bool plan, int *ctas) {
    using C = PagedCfg<DP, NT>;
    static bool attr[kMaxDevices] = {};
    static int occ[kMaxDevices] = {};
    G9_CU(smem_limit_once(attn_paged_k<DP, NT>, C::SMEM, attr));
    if (!occ[call.d->dev])
        G9_CU(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ[call.d->dev], attn_paged_k<DP, NT>, AW * 32, C::SMEM));
    // the last CTA of a unit keeps a weight for each of its slots and rows where the copies landed
    const long long fit = C::RING / 4 / C::ROWS - 4;
    *ctas = (int)std::min<long long>((long long)std::max(occ[call.d->dev], 1) * call.d->sm_count, fit);
    if (plan) return 0;
    return 0;
}

template <int DP, int NT>
int paged_launch(const PagedArgs &a, const KvCall &call, int ctas) {
    using C = PagedCfg<DP, NT>;
    G9_CU(launch_pdl(attn_paged_k<DP, NT>, dim3((unsigned)ctas), dim3(AW * 32), C::SMEM, call.st, a));
    return launched("attn_paged");
}

template <int DP, int NT>
int paged_either(const PagedArgs &a, const KvCall &call, bool plan, int *ctas) {
    return plan ? paged_run<DP, NT>(a, call, true, ctas) : paged_launch<DP, NT>(a, call, *ctas);
}

int paged(int dp, int nt, const PagedArgs &a, const KvCall &call, bool plan, int *ctas) {
    if (dp == 64) {
        if (nt == 1) return paged_either<64, 1>(a, call, plan, ctas);
        if (nt == 2) return paged_either<64, 2>(a, call, plan, ctas);
        return paged_either<64, 4>(a, call, plan, ctas);
    }
    if (dp == 128) {
        if (nt == 1) return paged_either<128, 1>(a, call, plan, ctas);
        if (nt == 2) return paged_either<128, 2>(a, call, plan, ctas);
        return paged_either<128, 4>(a, call, plan, ctas);
    }
    if (nt == 1) return paged_either<256, 1>(a, call, plan, ctas);
    return paged_either<256, 2>(a, call, plan, ctas);
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
    const int nt = rows <= 8 ? 1 : rows <= 16 || dp == 256 ? 2 : 4;
    const long long tiles = (rows + 8 * nt - 1) / (8 * nt), outer = (long long)c->ns * (sel ? nq : 1);
    if (tiles * c->HKV > INT_MAX || outer > INT_MAX || outer * tiles * c->HKV > INT_MAX)
        return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: %lld row tiles in one call", who, outer * tiles * c->HKV);
    a.tiles = (int)tiles;
    a.inner = (int)tiles * c->HKV;
    a.outer = (int)outer;
    const long long units = outer * a.inner;
    int ctas = 1;
    G9_TRY(paged(dp, nt, a, call, true, &ctas));
    // never more CTAs than steps there can be
    const long long most = units * (sel ? a.sel_steps : std::max<long long>(1, (a.c.cap + AKEYS - 1) / AKEYS + 1));
    ctas = (int)std::min<long long>(ctas, (most + AW - 1) / AW);
    const size_t part = up256((size_t)(ctas + units) * 8 * nt * (dp + 2) * 4);
    const long long heads = (long long)c->ns * nq * H;
    a.score_row = sel ? (long long)a.nsel * c->page : a.c.cap;
    const size_t lse2 = acc ? up256((size_t)heads * 4) : 0;
    if (acc && (__int128)heads * a.score_row * 4 > ((__int128)1 << 46))
        return fail(GEN9BLAS_ERR_OUT_OF_MEMORY, "%s: weights of %lld rows of %lld slots", who, heads, a.score_row);
    const size_t score = acc ? (size_t)heads * a.score_row * 4 : 0;
    void *buf = nullptr;
    G9_TRY(kv_workspace(ws, call, who, part + lse2 + score, (size_t)units, &buf, &a.cnt));
    a.part = (float *)buf;
    if (acc) {
        a.lse2 = (float *)((char *)buf + part);
        a.score = (float *)((char *)buf + part + lse2);
    }
    G9_TRY(paged(dp, nt, a, call, false, &ctas));
    if (acc && a.score_row > 0) {
        const long long sg = (long long)c->ns * c->HKV;
        if (sg > 65535) return fail(GEN9BLAS_ERR_INVALID_ARG, "%s: weights of %lld (stream, head) rows in one call", who, sg);
        const dim3 grid(sel ? 1u : (unsigned)((a.c.cap + 255) / 256), (unsigned)sg);
        G9_CU(launch_pdl(kv_weigh_k, grid, dim3(256), 0, call.st, a, acc, (long long)ms, (long long)mh));
        G9_TRY(launched("kv_weigh"));
    }
    const size_t marks = ((size_t)(c->ns - 1) * (size_t)std::max<int64_t>(ms, 0) +
                          (size_t)(c->HKV - 1) * (size_t)std::max<int64_t>(mh, 0) + (size_t)a.c.cap) * 4;
    const KvWrite w[3] = {{O, (size_t)heads * c->D * 4}, {lse, (size_t)heads * 4}, {acc, marks}};
    return kv_finish(call, sync, w, 3);
}

}  // extern "C"

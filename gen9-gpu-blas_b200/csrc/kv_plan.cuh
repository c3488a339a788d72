// kv_plan.cuh -- the split of a paged-cache kernel's work over one wave of CTAs (kv_attn.cu, kv.cu). Units (a head of a stream
// and a tile of its queries) have numbers of steps that only the device knows; `inner` units in a row share an `outer`
// index (a stream) and its number of steps. All units' steps in a row are cut into equal runs, one a CTA, which a CTA takes a
// segment of a unit at a time. A segment costs a CTA some latencies besides its steps (row data, first copies, merge), so
// each unit is counted `cost` steps longer than it is, at its start: a CTA that begins a unit in the middle of its run gets
// that much less to read, and short units begin a run of their own.
#pragma once
#include <cuda_runtime.h>

namespace g9kv {

struct Run {
    int lo, hi;       // this CTA's run, in counted steps; empty: lo >= hi
    int chunk;        // length of a run, a multiple of `warps`
    int outer, pre;   // the outer index that holds lo, the counted steps before it
};

// Every warp works the run out for itself. steps(o): steps of outer index o, at least 1; all counted steps stay below 2^30.
template <typename Steps>
__device__ __forceinline__ Run find_run(int outers, int inner, int cost, int warps, Steps steps) {
    const unsigned all = 0xffffffffu;
    const int lane = threadIdx.x & 31, b = blockIdx.x;
    int T = 0, n0 = 0;   // counted steps in all; of outer index `lane`
    for (int o = lane; o < outers; o += 32) {
        const int n = (steps(o) + cost) * inner;
        if (o == lane) n0 = n;
        T += n;
    }
    T = __reduce_add_sync(all, T);
    Run r;
    r.chunk = (int)(((unsigned)T + gridDim.x - 1) / gridDim.x + warps - 1) / warps * warps;
    r.outer = r.pre = 0;
    if ((long long)b * r.chunk >= T) {
        r.lo = r.hi = 0;
        return r;
    }
    r.lo = b * r.chunk;
    r.hi = min(r.lo + r.chunk, T);
    for (int o0 = 0;; o0 += 32) {
        const int n = o0 + lane < outers ? (o0 ? (steps(o0 + lane) + cost) * inner : n0) : 0;
        int x = n;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const int y = __shfl_up_sync(all, x, i);
            if (lane >= i) x += y;
        }
        const unsigned past = __ballot_sync(all, r.pre + x > r.lo);   // lo < T: found before the indices run out
        if (past) {
            const int l = __ffs(past) - 1;
            r.outer = o0 + l;
            r.pre += __shfl_sync(all, x - n, l);
            return r;
        }
        r.pre += __shfl_sync(all, x, 31);
    }
}

}  // namespace g9kv

"""GPU parity of the paged key-value cache (include/gen9blas_kv.h through gen9-gpu-blas_b200/g9kv.py) against the 64-bit
NumPy forms of oracle/kv_ref.py: cache writes, attention over pages, page selection, eviction, and a decoding loop of all
four. Layout operations are compared bit for bit; attention within the bound of `attend_close`."""
import ctypes
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import kv_ref  # noqa: E402

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def kv(gpu_lib):
    import g9kv
    return g9kv


def make(rng, lens, page, heads, D, spare=3, layout="phsd", extra=0, poison=False, holes=()):
    """A cache on host and device: streams of `lens` slots (room for `extra` more), random pages, optional NaN in every slot
    that is not in use, `holes`: (stream, place) without a page."""
    ns = len(lens)
    mp = max(1, max(-(-(n + extra) // page) for n in lens))
    pool = ns * mp + spare
    K = rng.standard_normal((pool, heads, page, D)).astype(np.float16)
    V = rng.standard_normal((pool, heads, page, D)).astype(np.float16)
    table = rng.permutation(pool)[:ns * mp].reshape(ns, mp).astype(np.int32)
    for s, n in enumerate(lens):
        table[s, -(-(n + extra) // page):] = -1
    for s, o in holes:
        table[s, o] = -1
    if poison:
        free = np.ones((pool, page), bool)
        for s, n in enumerate(lens):
            for k in range(n):
                if table[s, k // page] >= 0:
                    free[table[s, k // page], k % page] = False
        K.transpose(0, 2, 1, 3)[free] = np.nan
        V.transpose(0, 2, 1, 3)[free] = np.inf
    bounds = np.zeros((pool, heads, 2, D), np.float16)
    for s, n in enumerate(lens):
        for o in range(-(-n // page)):
            p, m = table[s, o], min(page, n - o * page)
            if p >= 0:
                bounds[p, :, 0], bounds[p, :, 1] = K[p, :, :m].min(1), K[p, :, :m].max(1)
    host = {"K": K, "V": V, "bounds": bounds, "table": table}
    if layout == "phsd":
        dev = [torch.from_numpy(x.copy()).cuda() for x in (K, V)]
    elif layout == "pshd":      # slots outside the heads, as a contiguous cache of rows of all heads
        dev = [torch.from_numpy(x.transpose(0, 2, 1, 3).copy()).cuda().permute(0, 2, 1, 3) for x in (K, V)]
    else:                       # padded rows, K and V interleaved in one buffer
        both = torch.zeros(pool, heads, page, 2, D + 8, dtype=torch.float16, device="cuda")
        both[..., 0, :D] = torch.from_numpy(K).cuda()
        both[..., 1, :D] = torch.from_numpy(V).cuda()
        dev = [both[..., 0, :D], both[..., 1, :D]]
    return host, dev[0], dev[1], torch.from_numpy(table).cuda(), torch.from_numpy(bounds.copy()).cuda()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def attend_close(got, ref, D):
    """Element-wise bound. A score (natural units) is off by at most e = spread·(2^-21 + (D + 4)·2^-24): the query's two FP16
    parts drop less than 2^-22 of it, D + 4 FP32 roundings follow (products, sums, scale), the base-2 exponent adds as
    much as |x|·2^-24 again; a weight is then off by 2e and an output by that share of sum w|v|, besides the roundings of
    exp2 (2^-22) and of up to 16 FP32 additions in a row in each of the two sums (2^-20 each at these lengths, whose steps
    are split over the CTAs)."""
    O, lse, _, spread, mass = ref
    e = spread * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
    o, l = got[0].cpu().numpy().astype(np.float64), got[1].cpu().numpy().astype(np.float64)
    tol = (2 * e[..., None] + 2.0 ** -19 + 2.0 ** -22) * mass + 1e-30
    assert np.all(np.abs(o - O) <= tol), float(np.max(np.abs(o - O) / tol))
    dead = np.isneginf(lse)
    assert np.array_equal(dead, np.isneginf(l))
    assert np.all(np.abs(l[~dead] - lse[~dead]) <= (e + 2.0 ** -20 + 2.0 ** -22 * (1 + np.abs(lse)))[~dead])
    assert np.all(o[dead] == 0)


# ------------------------------------------------------------------------------------------------ cache writes
@pytest.mark.parametrize("page,heads,D,nt,layout", [(16, 2, 128, 1, "phsd"), (8, 3, 64, 21, "pshd"), (5, 1, 80, 7, "both"),
                                                    (64, 2, 256, 70, "phsd"), (1, 2, 8, 3, "pshd")])
def test_append(kv, page, heads, D, nt, layout):
    rng = np.random.default_rng(page + D)
    lens, count = [0, 1, page, 3 * page - 1], [nt, max(nt - 1, 0), 0, nt + 5]
    host, K, V, table, bounds = make(rng, lens, page, heads, D, extra=nt + 1, layout=layout)
    cap = table.shape[1] * page
    acc = rng.random((4, heads, cap)).astype(np.float32)
    pos = rng.integers(0, 99, (4, heads, cap)).astype(np.int32)
    k, v = (rng.standard_normal((4, nt, heads, D)).astype(np.float32) for _ in range(2))
    k[0, 0, 0, 0], v[0, 0, 0, 1] = 1e6, -1e6             # beyond FP16: infinities, as a plain conversion gives
    dacc, dpos = torch.from_numpy(acc).cuda(), torch.from_numpy(pos).cuda()
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    for pos0, cnt in ((None, count), ([5, 6, 7, 2 ** 30], None)):
        fine = kv_ref.append(host, k, v, lens, cnt, acc, pos, pos0)
        got = cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints(lens),
                           count=None if cnt is None else ints(cnt), acc=dacc, pos=dpos,
                           pos0=None if pos0 is None else ints(pos0), wait=True)
        assert got == fine
        for name, x in (("K", K), ("V", V), ("bounds", bounds)):
            assert np.array_equal(x.cpu().numpy(), host[name], equal_nan=True), name
        assert np.array_equal(dacc.cpu().numpy(), acc) and np.array_equal(dpos.cpu().numpy(), pos)


def test_append_strided_source_and_bad_pages(kv):
    rng = np.random.default_rng(5)
    heads, D, page = 2, 64, 8
    host, K, V, table, _ = make(rng, [6, 4, 0], page, heads, D, extra=8, holes=[(1, 1)])
    host["bounds"] = None
    table[2, 0] = 2 ** 31 - 1
    host["table"] = table.cpu().numpy()
    wide = torch.randn(3, heads, 10, D + 3, device="cuda")       # head-major, odd row pitch: no 16-byte rows
    k = wide[:, :, :9, :D].permute(0, 2, 1, 3)
    v = wide[:, :, 1:, 2:D + 2].permute(0, 2, 1, 3)
    cache = kv.PagedKV(K, V, table)
    assert cache.append(k, v, ints([6, 4, -3]), wait=True) is False
    assert kv_ref.append(host, k.cpu().numpy(), v.cpu().numpy(), [6, 4, -3]) is False
    assert np.array_equal(K.cpu().numpy(), host["K"]) and np.array_equal(V.cpu().numpy(), host["V"])
    assert cache.append(k[:, :1], v[:, :1], ints([2 ** 31 - 1, 0, 9 * page]), count=ints([1, -1, 1]), wait=True) is False
    assert np.array_equal(K.cpu().numpy(), host["K"])
    assert cache.append(k[:, :0], v[:, :0], ints([0, 0, 0]), wait=True) is True


# ------------------------------------------------------------------------------------------------ attention
CASES = [   # lens, page, heads, group, D, tokens, window, layout
    ([1, 40, 0, 100], 16, 2, 4, 128, 1, 0, "phsd"),
    ([257, 31, 1000], 16, 2, 8, 64, 1, 0, "pshd"),
    ([37, 500, 3], 24, 1, 1, 128, 1, 0, "both"),
    ([700, 65], 32, 2, 3, 80, 1, 100, "phsd"),
    ([90, 333], 7, 2, 7, 96, 3, 0, "phsd"),
    ([500, 17, 64], 64, 1, 4, 128, 4, 33, "pshd"),
    ([130, 0, 1], 1, 1, 2, 256, 2, 0, "phsd"),
    ([300], 128, 2, 16, 256, 1, 0, "phsd"),
    ([1500], 16, 2, 4, 128, 9, 0, "phsd"),          # 36 rows of a head: five units (units of two tiles: test_kv_large_gpu.py)
    ([64, 200], 48, 1, 5, 8, 13, 10, "phsd"),
    ([200] * 40, 16, 2, 4, 64, 1, 0, "phsd"),       # more units than CTAs split evenly over
    ([2000, 0, 0, 5, 0, 1999], 16, 4, 4, 128, 1, 0, "phsd"),
    ([60], 16, 1, 80, 64, 1, 0, "phsd"),            # one key-value head under 80 query heads
    ([300], 32, 2, 2, 64, 40, 0, "pshd"),           # a short prompt in one call
    ([3 * i % 41 for i in range(100)], 8, 2, 4, 64, 1, 0, "phsd"),
    ([70, 9, 33], 8, 1, 3, 200, 2, 12, "both"),
]


@pytest.mark.parametrize("lens,page,heads,group,D,nq,window,layout", CASES)
@pytest.mark.parametrize("weights", [False, True])
def test_attend(kv, lens, page, heads, group, D, nq, window, layout, weights):
    rng = np.random.default_rng(len(lens) * 1000 + page + D + nq)
    host, K, V, table, _ = make(rng, [n + nq - 1 if n else 0 for n in lens], page, heads, D, layout=layout, poison=True)
    vis = np.array(lens) - (nq - 1) * (np.array(lens) == 0)      # an empty stream stays empty for every token
    q = (rng.standard_normal((len(lens), nq, heads * group, D)) * 2).astype(np.float32)
    acc0 = rng.random((len(lens), heads, table.shape[1] * page)).astype(np.float32)
    acc = torch.from_numpy(acc0).cuda() if weights else None
    cache = kv.PagedKV(K, V, table)
    ref = kv_ref.attend(host, q, vis, window=window)
    got = cache.attend(torch.from_numpy(q).cuda(), ints(vis), window=window, acc=acc, lse=True)
    attend_close(got, ref, D)
    if weights:
        e = ref[3].max() * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
        a = acc.cpu().numpy()
        assert np.all(np.abs(a - (acc0 + ref[2])) <= (4 * e + 2.0 ** -19 + nq * group * 2.0 ** -24) * ref[2] +
                      2.0 ** -23 * (acc0 + ref[2]))
        assert np.array_equal(a[ref[2] == 0], acc0[ref[2] == 0])
        again = torch.from_numpy(acc0).cuda()
        cache.attend(torch.from_numpy(q).cuda(), ints(vis), window=window, acc=again)
        assert torch.equal(acc, again)          # the same bits each time


@pytest.mark.parametrize("nq,page,group,D", [(1, 16, 4, 128), (3, 5, 2, 64), (2, 32, 9, 128)])
def test_attend_chosen_pages(kv, nq, page, group, D):
    rng = np.random.default_rng(nq + page)
    lens, heads, m = [400, 33, 2, 0], 2, 6
    host, K, V, table, _ = make(rng, [n + nq - 1 if n else 0 for n in lens], page, heads, D, poison=True, holes=[(0, 3)])
    vis = np.array(lens) - (nq - 1) * (np.array(lens) == 0)
    mp = table.shape[1]
    sel = np.sort(rng.integers(0, mp, (4, nq, heads, m)), axis=-1).astype(np.int32)   # with doubles: counted once
    sel[0, 0, 0] = [0, 3, 3, mp - 1, -1, -1]
    sel[0, 0, 1] = [-1, 2, mp, mp + 5, 2 ** 31 - 1, -2 ** 31]
    sel[1, 0, 0] = -1
    q = rng.standard_normal((4, nq, heads * group, D)).astype(np.float32)
    ref = kv_ref.attend(host, q, vis, sel=sel)
    acc = torch.zeros(4, heads, mp * page, device="cuda")
    got = kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints(vis), sel=torch.from_numpy(sel).cuda(), acc=acc,
                                         lse=True)
    attend_close(got, ref, D)
    e = ref[3].max() * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
    assert np.all(np.abs(acc.cpu().numpy() - ref[2]) <= (4 * e + 2.0 ** -19 + nq * group * 2.0 ** -23) * ref[2] + 1e-30)
    none = kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints(vis), sel=torch.empty(4, nq, heads, 0, dtype=torch.int32,
                                                                                              device="cuda"))
    assert not none.any()


def test_attend_scales_and_strides(kv):
    """Queries from tiny to large (the power-of-two scaling of the FP16 parts), a strided query, another scale."""
    rng = np.random.default_rng(8)
    host, K, V, table, _ = make(rng, [300, 50], 16, 2, 64)
    for mul, scale in ((1e-30, None), (1e-3, 0.7), (40.0, None), (1e4, 1e-4)):
        wide = torch.randn(2, 8, 1, 70, device="cuda") * mul
        q = wide[:, :, :, 3:67].permute(0, 2, 1, 3)
        ref = kv_ref.attend(host, q.cpu().numpy(), [300, 50], scale=scale)
        attend_close(kv.PagedKV(K, V, table).attend(q, ints([300, 50]), scale=scale, lse=True), ref, 64)


def test_attend_one_dominating_and_many_small_weights(kv):
    """One slot takes nearly all of the weight, thousands share the rest: their sum has to survive."""
    rng = np.random.default_rng(12)
    n, D = 6000, 128
    host, K, V, table, _ = make(rng, [n], 16, 1, D)
    host["K"] *= np.float16(0.05)
    p = host["table"][0, 0]
    host["K"][p, 0, 3] = 1.0
    q = np.full((1, 1, 4, D), 0.9, np.float32)
    K.copy_(torch.from_numpy(host["K"]))
    attend_close(kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints([n]), lse=True), kv_ref.attend(host, q, [n]), D)


def test_attend_draft_tokens_with_wild_values_ahead(kv):
    """Values that only later draft tokens see (or that an earlier token's window has left) are infinite or NaN: the
    others' results stay as they are."""
    rng = np.random.default_rng(9)
    lens, D, nq, window = [130, 47], 64, 5, 20
    host, K, V, table, _ = make(rng, [n + nq - 1 for n in lens], 16, 2, D)
    q = torch.randn(2, nq, 8, D, device="cuda")
    for w in (0, window):
        clean = kv.PagedKV(K, V, table).attend(q, ints(lens), window=w)
        K2, V2 = K.clone(), V.clone()
        for s, n in enumerate(lens):
            for k, bad in ((n + 2, float("inf")), (n + 3, float("nan")), (n - window + 1, float("-inf"))):
                p, i = table[s, k // 16].item(), k % 16
                V2[p, :, i] = bad
        got = kv.PagedKV(K2, V2, table).attend(q, ints(lens), window=w)
        for s, n in enumerate(lens):
            for t in range(nq):
                seen = range(max(0, n + t - w) if w else 0, n + t)
                wild = [k for k in (n + 2, n + 3, n - window + 1) if k in seen]
                if wild:
                    assert not torch.isfinite(got[s, t]).any()
                else:
                    assert torch.equal(got[s, t], clean[s, t])


def test_attend_wild_keys(kv):
    """A seen key that is NaN or infinite spoils the heads that see it and no others."""
    rng = np.random.default_rng(10)
    host, K, V, table, _ = make(rng, [40, 40, 40], 8, 2, 64)
    q = torch.rand(3, 1, 4, 64, device="cuda") + 0.1
    base = kv.PagedKV(K, V, table).attend(q, ints([40, 40, 33]))
    K[table[0, 2].long(), 0, 3, 5] = float("nan")
    K[table[1, 1].long(), 1, 2] = float("inf")
    K[table[2, 4].long(), 1, 1:] = float("nan")          # behind the last slot seen
    out = kv.PagedKV(K, V, table).attend(q, ints([40, 40, 33]))
    assert torch.isnan(out[0, 0, :2]).all() and torch.equal(out[0, 0, 2:], base[0, 0, 2:])
    assert not torch.isfinite(out[1, 0, 2:]).any() and torch.equal(out[1, 0, :2], base[1, 0, :2])
    assert torch.equal(out[2], base[2])


def test_attend_long_cache_past_32_bit_offsets(kv):
    """Pages whose offset in the pool passes 2^31 elements (and 2^32 bytes), checked against the same pages moved down."""
    page, heads, D, n = 64, 8, 128, 700
    pool = 2 ** 31 // (page * heads * D) + 40
    K = torch.zeros(pool, heads, page, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    mp = -(-n // page)
    low, high = torch.arange(mp, device="cuda"), torch.arange(pool - mp, pool, device="cuda")
    for X in (K, V):
        X[low] = torch.randn(mp, heads, page, D, device="cuda").half()
        X[high] = X[low]
    q = torch.randn(1, 1, 32, D, device="cuda")
    got = [kv.PagedKV(K, V, t[None].int()).attend(q, ints([n])) for t in (low, high)]
    assert torch.equal(got[0], got[1]) and got[0].abs().max() > 0
    k = torch.randn(1, 3, heads, D, device="cuda")
    kv.PagedKV(K, V, high[None].int()).append(k, -k, ints([n]))
    assert torch.equal(K[pool - 1, :, n % page:n % page + 3], k[0].half().transpose(0, 1))
    assert torch.equal(V[pool - 1, :, n % page:n % page + 3], -k[0].half().transpose(0, 1))


def test_attend_equals_the_contiguous_cache(kv, gpu_lib):
    """Pages in order are the contiguous cache of gen9blas_attn_dec: the two agree."""
    rng = np.random.default_rng(14)
    n, D, heads, H = 515, 128, 2, 8
    host, K, V, table, _ = make(rng, [n], 16, heads, D)
    rows = [torch.from_numpy(np.concatenate([host[x][p] for p in host["table"][0]], axis=1)[:, :n].copy()).cuda() for x in "KV"]
    q = torch.randn(1, 1, H, D, device="cuda")
    O = torch.empty(1, 1, H, D, device="cuda")
    vis = ints([n])
    torch.cuda.synchronize()
    size = rows[0].numel() * 2
    assert gpu_lib.attn_dec(D, H, heads, 1, 1, n, q.data_ptr(), H * D, D, H * D, rows[0].data_ptr(), D, n * D, heads * n * D, size,
                            rows[1].data_ptr(), D, n * D, heads * n * D, size, O.data_ptr(), D ** -0.5, vis.data_ptr(), 0, 0,
                            1) == 0, gpu_lib.error()
    ref = kv_ref.attend(host, q.cpu().numpy(), [n])
    out, lse = kv.PagedKV(K, V, table).attend(q, vis, lse=True)
    attend_close((out, lse), ref, D)
    attend_close((O, lse), ref, D)


def test_streams_that_share_pages(kv):
    rng = np.random.default_rng(15)
    host, K, V, table, _ = make(rng, [200, 150, 90], 16, 2, 64)
    table[1, :5] = table[0, :5]
    table[2, :5] = table[0, :5]
    host["table"] = table.cpu().numpy()
    q = rng.standard_normal((3, 1, 8, 64)).astype(np.float32)
    attend_close(kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints([200, 150, 90]), lse=True),
                 kv_ref.attend(host, q, [200, 150, 90]), 64)


# ------------------------------------------------------------------------------------------------ selection
@pytest.mark.parametrize("lens,page,heads,group,D,nq,m,first,last", [
    ([400, 17, 0, 1], 16, 2, 4, 128, 1, 8, 1, 1), ([1000, 999], 8, 1, 1, 64, 3, 20, 2, 3), ([300], 5, 2, 7, 80, 2, 1, 0, 0),
    ([3000], 4, 1, 2, 256, 1, 100, 0, 1), ([90], 16, 3, 8, 8, 1, 3, 5, 5), ([64 * 130], 64, 1, 4, 128, 1, 64, 1, 1),
    ([200], 8, 1, 72, 64, 2, 5, 1, 1), ([333, 20], 16, 1, 16, 256, 2, 7, 1, 1), ([500], 16, 2, 4, 128, 7, 9, 1, 1),
    ([700, 701], 16, 1, 12, 128, 5, 4, 0, 0), ([9000], 8, 1, 4, 128, 1, 600, 1, 1)])
def test_select(kv, lens, page, heads, group, D, nq, m, first, last):
    rng = np.random.default_rng(D + page)
    host, K, V, table, bounds = make(rng, [n + nq - 1 if n else 0 for n in lens], page, heads, D)
    vis = np.array(lens) - (nq - 1) * (np.array(lens) == 0)
    q = rng.standard_normal((len(lens), nq, heads * group, D)).astype(np.float32)
    got = kv.PagedKV(K, V, table, bounds=bounds).select(torch.from_numpy(q).cuda(), ints(vis), m, first=first, last=last)
    assert np.array_equal(got.cpu().numpy(), kv_ref.select(host, q, vis, m, first=first, last=last))


def test_select_ties_nan_and_missing_pages(kv):
    rng = np.random.default_rng(21)
    host, K, V, table, bounds = make(rng, [320, 320], 8, 2, 64, holes=[(0, 9)])
    b = host["bounds"]
    t = host["table"]
    b[t[0, 10:30]] = b[t[0, 10]]                       # twenty equal pages
    b[t[1, 5], 0, :, 3] = np.nan
    b[t[1, 6], 0, 1] = np.inf
    bounds.copy_(torch.from_numpy(b))
    q = np.abs(rng.standard_normal((2, 1, 4, 64))).astype(np.float32) + 0.1
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    for m in (1, 2, 7, 15, 39, 40, 41):
        got = cache.select(torch.from_numpy(q).cuda(), ints([320, 320]), m, first=1, last=0).cpu().numpy()
        assert np.array_equal(got, kv_ref.select(host, q, [320, 320], m, first=1, last=0)), m


def test_select_near_ties_follow_the_exact_order(kv):
    """Pages whose scores differ by less than FP32 can tell: a constant part of 2^14, differences of 2^-28."""
    D, n = 64, 60
    K = torch.zeros(n, 1, 1, D, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(2)
    bounds = np.zeros((n, 1, 2, D), np.float16)
    bounds[:, 0, 1, 0] = 128.0
    bounds[:, 0, 1, 1] = rng.permutation(n) * 2.0 ** -20
    q = np.zeros((1, 1, 1, D), np.float32)
    q[..., 0], q[..., 1] = 128.0, 2.0 ** -8
    table = ints(np.arange(n)[None])
    host = {"K": K.cpu().numpy(), "V": K.cpu().numpy(), "bounds": bounds, "table": table.cpu().numpy()}
    got = kv.PagedKV(K, K, table, bounds=torch.from_numpy(bounds).cuda()).select(torch.from_numpy(q).cuda(), ints([n]), 10, first=0,
                                                                                last=0)
    assert np.array_equal(got.cpu().numpy(), kv_ref.select(host, q, [n], 10, first=0, last=0))


def test_select_a_nan_of_one_head_ranks_the_page_last(kv):
    """Infinite bounds against a query element of zero: NaN for that head, +inf or a number for the others of its group."""
    rng = np.random.default_rng(31)
    n, D = 40, 64
    K = torch.zeros(n, 1, 1, D, dtype=torch.float16, device="cuda")
    bounds = np.sort(rng.standard_normal((n, 1, 2, D)).astype(np.float16), axis=2)
    bounds[3::5, 0, 1, 0] = np.inf
    bounds[4::10, 0, 0, 1] = -np.inf
    bounds[9, 0, 0, 2], bounds[9, 0, 1, 2] = np.inf, -np.inf     # a page all of whose keys are NaN there
    q = rng.standard_normal((1, 3, 4, D)).astype(np.float32)
    q[:, :, :, 0] = [[[0.0, 1.0, -1.0, 2.0], [1.0, 1.0, 2.0, 3.0], [-1.0, -2.0, -1.0, -3.0]]]
    q[:, :, :, 1] = [[[1.0, 1.0, 1.0, 1.0], [1.0, 0.0, 1.0, -1.0], [-1.0, -2.0, -1.0, -3.0]]]
    table = np.arange(n, dtype=np.int32)[None]
    host = {"K": K.cpu().numpy(), "V": K.cpu().numpy(), "bounds": bounds, "table": table}
    cache = kv.PagedKV(K, K, ints(table), bounds=torch.from_numpy(bounds).cuda())
    for m in (1, 3, 10, 30, 35):
        got = cache.select(torch.from_numpy(q).cuda(), ints([n - 2]), m, first=0, last=0).cpu().numpy()
        with np.errstate(invalid="ignore"):
            assert np.array_equal(got, kv_ref.select(host, q, [n - 2], m, first=0, last=0)), m


@pytest.mark.parametrize("size", [1e-44, 3e-42, 1e-38, 1e-30, 1e30, 3e38])
def test_select_with_queries_at_the_ends_of_float32(kv, size):
    """Scores that FP32 rounds to a few units of its least number, or to infinity, still rank as their 64-bit values."""
    rng = np.random.default_rng(32)
    host, K, V, table, bounds = make(rng, [16 * 60], 16, 2, 64)
    q = (np.clip(rng.standard_normal((1, 1, 4, 64)), -1, 1) * size).astype(np.float32)
    got = kv.PagedKV(K, V, table, bounds=bounds).select(torch.from_numpy(q).cuda(), ints([16 * 60]), 12, first=0, last=0)
    assert np.array_equal(got.cpu().numpy(), kv_ref.select(host, q, [16 * 60], 12, first=0, last=0))


@pytest.mark.parametrize("n,m", [(3000, 700), (600, 30)])
def test_select_many_equal_pages(kv, n, m):
    """Hundreds of pages with the same bounds, some infinite or missing: the lowest places of the equal ones."""
    rng = np.random.default_rng(22)
    K = torch.zeros(n, 2, 1, 64, dtype=torch.float16, device="cuda")
    kinds = rng.standard_normal((3, 2, 2, 64)).astype(np.float16)
    kinds.sort(axis=2)
    bounds = kinds[rng.integers(0, 3, n)]
    table = np.arange(n, dtype=np.int32)[None].copy()
    q = rng.standard_normal((1, 1, 4, 64)).astype(np.float32)
    for step in range(3):
        if step == 1:
            table[0, ::17] = -1
        if step == 2:
            bounds[5::31, :, 1, 3] = np.inf
            bounds[6::31, :, :, 3] = np.nan
        host = {"K": K.cpu().numpy(), "V": K.cpu().numpy(), "bounds": bounds, "table": table}
        got = kv.PagedKV(K, K, ints(table), bounds=torch.from_numpy(bounds).cuda()).select(torch.from_numpy(q).cuda(), ints([n]), m)
        assert np.array_equal(got.cpu().numpy(), kv_ref.select(host, q, [n], m)), step


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("lens,keep,page,heads,D,first,recent,layout", [
    ([50, 33, 32, 0, 5], 32, 16, 2, 128, 2, 4, "phsd"), ([100], 1, 8, 1, 64, 0, 0, "pshd"), ([100, 99], 37, 5, 3, 80, 4, 30, "both"),
    ([513], 512, 64, 2, 256, 0, 1, "phsd"), ([70, 10], 500, 16, 1, 8, 4, 4, "phsd"), ([3000, 2999], 1500, 32, 2, 64, 4, 32, "phsd"),
    ([20000, 13001, 400], 9000, 16, 1, 8, 4, 32, "phsd"), ([60000], 30001, 64, 2, 8, 4, 32, "pshd"), ([7000] * 30, 6990, 100, 2, 8, 0, 9, "phsd")])
@pytest.mark.parametrize("with_pos", [False, True])
def test_evict(kv, lens, keep, page, heads, D, first, recent, layout, with_pos):
    rng = np.random.default_rng(keep + page)
    host, K, V, table, bounds = make(rng, lens, page, heads, D, layout=layout)
    cap = table.shape[1] * page
    acc = np.round(rng.exponential(size=(len(lens), heads, cap)), 2).astype(np.float32)      # with ties
    pos = rng.permuted(np.tile(np.arange(cap, dtype=np.int32), (len(lens), heads, 1)), axis=-1) if with_pos else None
    dacc, dpos = torch.from_numpy(acc.copy()).cuda(), torch.from_numpy(pos.copy()).cuda() if with_pos else None
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    n = ints(lens)
    got = cache.evict(n, keep, dacc, dpos, first=first, recent=recent, out=n)               # lengths in place
    want = kv_ref.evict(host, lens, keep, acc, pos, first=first, recent=recent)
    assert np.array_equal(got.cpu().numpy(), want)
    assert np.array_equal(dacc.cpu().numpy(), acc)
    assert pos is None or np.array_equal(dpos.cpu().numpy(), pos)
    for name, x in (("K", K), ("V", V), ("bounds", bounds)):
        assert np.array_equal(x.cpu().numpy(), host[name]), name


def test_evict_odd_weights_and_bad_pages(kv):
    """NaN, infinite, negative and all-equal weights; a stream with a missing page; lengths past the table and below 0."""
    rng = np.random.default_rng(31)
    lens, keep, page, heads = [60, 60, 64, 64, 64], 20, 8, 2
    host, K, V, table, bounds = make(rng, lens, page, heads, 64, holes=[(2, 1), (2, 6)])
    acc = rng.standard_normal((5, heads, 64)).astype(np.float32)
    acc[0, 0, ::3], acc[0, 1, 5:9] = np.nan, np.inf
    acc[1] = 0.0
    acc[1, 1, ::2] = -0.0
    acc[3] = np.nan
    lens2 = [60, 60, 64, 2 ** 31 - 1, -5]
    dacc = torch.from_numpy(acc.copy()).cuda()
    got = kv.PagedKV(K, V, table, bounds=bounds).evict(ints(lens2), keep, dacc, first=1, recent=2)
    assert np.array_equal(got.cpu().numpy(), kv_ref.evict(host, lens2, keep, acc, None, first=1, recent=2))
    assert np.array_equal(dacc.cpu().numpy(), acc, equal_nan=True)
    for name, x in (("K", K), ("V", V), ("bounds", bounds)):
        assert np.array_equal(x.cpu().numpy(), host[name]), name


# ------------------------------------------------------------------------------------------------ together
def test_decoding_loop(kv):
    """A short serving loop with all operators: prompts enter, tokens are decoded with weights, pages are chosen, the cache is
    thinned and decoding goes on over the reordered slots."""
    rng = np.random.default_rng(40)
    heads, group, D, page, ns = 2, 4, 64, 8, 3
    lens = np.array([30, 0, 17])
    host, K, V, table, bounds = make(rng, list(lens), page, heads, D, extra=40)
    cap = table.shape[1] * page
    acc, pos = np.zeros((ns, heads, cap), np.float32), np.tile(np.arange(cap, dtype=np.int32), (ns, heads, 1))
    dacc, dpos = torch.from_numpy(acc.copy()).cuda(), torch.from_numpy(pos.copy()).cuda()
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    n, at = lens.copy(), lens.copy()
    dn = ints(n)
    for step in range(12):
        nt = 5 if step == 0 else 1
        k, v = (rng.standard_normal((ns, nt, heads, D)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((ns, nt, heads * group, D)).astype(np.float32)
        tk, tv, tq = (torch.from_numpy(x).cuda() for x in (k, v, q))
        cache.append(tk, tv, dn, acc=dacc, pos=dpos, pos0=ints(at))
        kv_ref.append(host, k, v, n, None, acc, pos, at)
        ref = kv_ref.attend(host, q, n + 1)
        got = cache.attend(tq, dn + 1, acc=dacc, lse=True)
        attend_close(got, ref, D)
        acc += ref[2].astype(np.float32)
        sel = cache.select(tq, dn + 1, 3)
        want = kv_ref.select(host, q, n + 1, 3)
        assert np.array_equal(sel.cpu().numpy(), want)
        attend_close(cache.attend(tq, dn + 1, sel=sel, lse=True), kv_ref.attend(host, q, n + 1, sel=want), D)
        n, at, dn = n + nt, at + nt, dn + nt
        if step in (4, 9, 10):
            acc = dacc.cpu().numpy().copy()             # the same weights on both sides: the order below is theirs
            dn = cache.evict(dn, 20, dacc, dpos, first=2, recent=6)
            n = kv_ref.evict(host, n, 20, acc, pos, first=2, recent=6)
            assert np.array_equal(dn.cpu().numpy(), n) and np.array_equal(dpos.cpu().numpy(), pos)
            assert np.array_equal(dacc.cpu().numpy(), acc)
    for name, x in (("K", K), ("V", V), ("bounds", bounds)):
        assert np.array_equal(x.cpu().numpy(), host[name]), name


def test_captured_step_follows_its_lengths(kv):
    """append, select and attend captured once and replayed: lengths and tables are read on the device. Two graphs with a
    workspace each, an eager call between the replays."""
    rng = np.random.default_rng(41)
    heads, group, D, page, ns = 2, 4, 128, 16, 2
    host, K, V, table, bounds = make(rng, [100, 45], page, heads, D, extra=30)
    host["bounds"] = bounds.cpu().numpy().copy()
    n = ints([100, 45])
    k, v = (torch.zeros(ns, 1, heads, D, device="cuda") for _ in range(2))
    q = torch.zeros(ns, 1, heads * group, D, device="cuda")
    acc = torch.zeros(ns, heads, table.shape[1] * page, device="cuda")
    eager = kv.PagedKV(K, V, table, bounds=bounds)
    with pytest.raises(RuntimeError, match="workspace"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            try:
                eager.attend(q, n)
            finally:
                k.add_(0)                 # the capture holds something, and ends
    graphs = []
    for _ in range(2):
        cache = kv.PagedKV(K, V, table, bounds=bounds, workspace=kv.Workspace())
        with pytest.raises(RuntimeError, match="grow"):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                try:
                    cache.attend(q, n)
                finally:
                    k.add_(0)
        K0, V0, b0 = K.clone(), V.clone(), bounds.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):     # one call of each shape before the capture
            cache.append(k, v, n, count=torch.zeros_like(n))
            cache.select(q, n + 1, 2)
            cache.attend(q, n + 1, acc=acc)
            cache.attend(q, n + 1, sel=cache.select(q, n + 1, 2))
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.append(k, v, n)
            see = n + 1
            sel = cache.select(q, see, 2)
            out, lse = cache.attend(q, see, acc=acc, lse=True)
            part, plse = cache.attend(q, see, sel=sel, lse=True)
            n.add_(1)
        assert torch.equal(K, K0) and torch.equal(V, V0) and torch.equal(bounds, b0)     # nothing ran
        graphs.append((g, cache, sel, out, lse, part, plse))
    acc.zero_()
    size = np.array([100, 45])
    total = np.zeros(acc.shape)
    for step in range(20):
        g, cache, sel, out, lse, part, plse = graphs[step % 2]
        kn, vn = (rng.standard_normal((ns, 1, heads, D)).astype(np.float32) for _ in range(2))
        qn = rng.standard_normal((ns, 1, heads * group, D)).astype(np.float32)
        k.copy_(torch.from_numpy(kn))
        v.copy_(torch.from_numpy(vn))
        q.copy_(torch.from_numpy(qn))
        g.replay()
        kv_ref.append(host, kn, vn, size)
        ref = kv_ref.attend(host, qn, size + 1)
        attend_close((out, lse), ref, D)
        total += ref[2]
        want = kv_ref.select(host, qn, size + 1, 2)
        assert np.array_equal(sel.cpu().numpy(), want)
        attend_close((part, plse), kv_ref.attend(host, qn, size + 1, sel=want), D)
        size = size + 1
        if step % 5 == 0:
            attend_close(eager.attend(q, n, lse=True), ref, D)
    assert np.array_equal(n.cpu().numpy(), size)
    assert np.allclose(acc.cpu().numpy(), total, rtol=1e-4)


def test_calls_on_several_streams(kv):
    """One cache object and the library's own workspace, calls on two streams in turn."""
    rng = np.random.default_rng(42)
    host, K, V, table, _ = make(rng, [900, 700], 16, 2, 64)
    cache = kv.PagedKV(K, V, table)
    qs = [torch.randn(2, 1, 8, 64, device="cuda") for _ in range(6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cache.attend(q, ints([900, 700]), lse=True))
    torch.cuda.synchronize()
    for q, got in zip(qs, outs):
        attend_close(got, kv_ref.attend(host, q.cpu().numpy(), [900, 700]), 64)


def test_nothing_to_do(kv):
    """No streams, no tokens, no pages, no pool: empty or zero results, nothing read."""
    z = dict(device="cuda", dtype=torch.float16)
    K = torch.zeros(0, 2, 16, 64, **z)
    b = torch.zeros(0, 2, 2, 64, **z)
    q = torch.randn(3, 2, 4, 64, device="cuda")
    for table in (torch.full((3, 5), 7, dtype=torch.int32, device="cuda"), torch.zeros(3, 0, dtype=torch.int32, device="cuda")):
        cache = kv.PagedKV(K, K, table, bounds=b)
        acc = torch.ones(3, 2, cache.slots, device="cuda")
        out, lse = cache.attend(q, ints([50, 0, 3]), lse=True, acc=acc)
        assert not out.any() and torch.isneginf(lse).all() and (acc == 1).all()
        got = cache.select(q, ints([50, 0, 3]), 3).cpu().numpy()
        have = np.minimum([[50, 51], [0, 1], [3, 4]], cache.slots)
        assert np.array_equal((got >= 0).sum(-1), np.minimum(-(-have // 16), 3)[:, :, None].repeat(2, 2))
        assert cache.append(q[:, :, :2], q[:, :, :2], ints([0, 1, 2]), wait=True) is False
        assert cache.evict(ints([60, 2, 9]), 8, acc).tolist() == [min(8, cache.slots), min(2, cache.slots), min(8, cache.slots)]
    K = torch.randn(4, 2, 16, 64, **z)
    none = kv.PagedKV(K, K, torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
    assert none.attend(q[:0], ints([])).shape == (0, 2, 4, 64)
    one = kv.PagedKV(K, K, ints([[1, 2]]))
    assert one.attend(q[:1, :0], ints([9])).shape == (1, 0, 4, 64)


def test_workspace_of_its_own(kv):
    """A workspace grows with the calls, serves several caches in turn and ends without its caches."""
    rng = np.random.default_rng(44)
    ws = kv.Workspace()
    for n, D in ((50, 64), (4000, 128), (100, 256)):
        host, K, V, table, _ = make(rng, [n, n // 2], 16, 2, D)
        q = rng.standard_normal((2, 1, 8, D)).astype(np.float32)
        acc = torch.zeros(2, 2, table.shape[1] * 16, device="cuda")
        got = kv.PagedKV(K, V, table, workspace=ws).attend(torch.from_numpy(q).cuda(), ints([n, n // 2]), acc=acc, lse=True)
        attend_close(got, kv_ref.attend(host, q, [n, n // 2]), D)
    cache = kv.PagedKV(K, V, table, workspace=ws)
    ws.free()
    ws.free()
    with pytest.raises(ValueError, match="freed"):
        cache.attend(torch.from_numpy(q).cuda(), ints([n, n // 2]))


def test_refusals_on_the_device(kv, gpu_lib):
    rng = np.random.default_rng(43)
    host, K, V, table, bounds = make(rng, [20], 8, 2, 64)
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    q = torch.randn(1, 1, 4, 64, device="cuda")
    n = ints([20])
    for bad in (dict(q=q.double()), dict(q=q[..., :60]), dict(q=q.cpu()), dict(visible=n.long()), dict(visible=n.cpu()),
                dict(acc=torch.zeros(1, 2, 5, device="cuda")), dict(out=torch.zeros(1, 1, 4, 64)),
                dict(sel=torch.zeros(1, 1, 1, 4, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            cache.attend(**{"q": q, "visible": n, **bad})
    with pytest.raises(ValueError):
        cache.attend(torch.randn(1, 1, 3, 64, device="cuda"), n)           # 3 query heads over 2
    with pytest.raises(RuntimeError, match="bounds"):
        kv.PagedKV(K, V, table).select(q, n, 2)
    wide = 2 ** 32 + 4                                                     # 4 in 32 bits
    for call in (lambda: cache.attend(q, n, window=wide), lambda: cache.attend(q, n, step=wide),
                 lambda: cache.select(q, n, 2, first=wide), lambda: cache.evict(n, wide, torch.zeros(1, 2, 32, device="cuda")),
                 lambda: cache.evict(n, 8, torch.zeros(1, 2, 32, device="cuda"), recent=wide)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="overlap"):
        cache.attend(q, n, acc=torch.zeros(1, 1, 32, device="cuda").expand(1, 2, 32))
    hostv = (ctypes.c_int * 4)(20)
    args = (4, 1, q.data_ptr(), 256, 64, 256, ctypes.addressof(hostv), 1, 0, None, 0, 0.125, q.data_ptr(), None, None, 0, 0, None, 0)
    assert kv._fn["attn_paged"](cache._c, *args) == -3 and b"vis" in kv._fn["error"]()
    torch.cuda.synchronize()


def test_queued_write_is_seen_by_the_contiguous_attention(kv, gpu_lib):
    """append queued, then gen9blas_attn_dec on the same memory, whose first copies may precede the wait on the kernel
    before: the ledger of queued writes keeps them behind."""
    D, heads, n = 128, 2, 512
    K = torch.zeros(1, heads, n, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    q = torch.randn(1, 1, 8, D, device="cuda")
    O = torch.empty(1, 1, 8, D, device="cuda")
    cache = kv.PagedKV(K, V, ints([[0]]))
    vis, zero = ints([n]), ints([0])
    torch.cuda.synchronize()
    for it in range(5):
        k, v = (torch.randn(1, n, heads, D, device="cuda") for _ in range(2))
        cache.append(k, v, zero)
        assert gpu_lib.set_stream(torch.cuda.current_stream().cuda_stream or 1) == 0
        size = K.numel() * 2
        assert gpu_lib.attn_dec(D, 8, heads, 1, 1, n, q.data_ptr(), 8 * D, D, 8 * D, K.data_ptr(), D, n * D, heads * n * D, size,
                                V.data_ptr(), D, n * D, heads * n * D, size, O.data_ptr(), D ** -0.5, vis.data_ptr(), 0, 0,
                                0) == 0
        assert gpu_lib.set_stream(None) == 0
        torch.cuda.synchronize()
        host = {"K": k.half().cpu().numpy().transpose(0, 2, 1, 3), "V": v.half().cpu().numpy().transpose(0, 2, 1, 3),
                "table": np.zeros((1, 1), np.int32), "bounds": None}
        ref = kv_ref.attend(host, q.cpu().numpy(), [n])
        _, lse = cache.attend(q, vis, lse=True)
        attend_close((O, lse), ref, D)


def test_waiting_on_one_stream_keeps_the_writes_queued_on_another(kv, gpu_lib):
    """As above, with a waiting call on another stream between the write and the read: the write is still in the ledger."""
    D, heads, n = 128, 2, 4096
    K = torch.zeros(1, heads, n, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    q = torch.randn(1, 1, 8, D, device="cuda")
    O = torch.empty(1, 1, 8, D, device="cuda")
    cache = kv.PagedKV(K, V, ints([[0]]))
    small = torch.zeros(2, 1, heads, 16, D, dtype=torch.float16, device="cuda")
    other = kv.PagedKV(small[0], small[1], ints([[0]]))
    one = torch.randn(1, 1, heads, D, device="cuda")
    vis, zero = ints([n]), ints([0])
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for it in range(5):
        k, v = (torch.randn(1, n, heads, D, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            for _ in range(20):
                cache.append(k, v, zero)
        with torch.cuda.stream(b):
            assert other.append(one, one, zero, wait=True) is True
        with torch.cuda.stream(a):
            cache.append(k, v, zero)
        assert gpu_lib.set_stream(a.cuda_stream) == 0
        size = K.numel() * 2
        status = gpu_lib.attn_dec(D, 8, heads, 1, 1, n, q.data_ptr(), 8 * D, D, 8 * D, K.data_ptr(), D, n * D, heads * n * D, size,
                                  V.data_ptr(), D, n * D, heads * n * D, size, O.data_ptr(), D ** -0.5, vis.data_ptr(), 0, 0, 0)
        assert gpu_lib.set_stream(None) == 0
        torch.cuda.synchronize()
        assert status == 0
        host = {"K": k.half().cpu().numpy().transpose(0, 2, 1, 3), "V": v.half().cpu().numpy().transpose(0, 2, 1, 3),
                "table": np.zeros((1, 1), np.int32), "bounds": None}
        _, lse = cache.attend(q, vis, lse=True)
        attend_close((O, lse), kv_ref.attend(host, q.cpu().numpy(), [n]), D)


def test_append_of_more_tokens_than_the_table_holds(kv):
    """The launch covers the table and one page behind it; what passes it is dropped and told."""
    heads, D, page = 1, 8, 4
    K, V = (torch.zeros(3, heads, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    cache = kv.PagedKV(K, V, ints([[0, 1], [2, -1]]))
    k = torch.arange(1, 1 + 2 * 1000 * D, device="cuda", dtype=torch.float32).reshape(2, 1000, 1, D) / 64
    assert cache.append(k, -k, ints([3, 0]), count=ints([5, 4]), wait=True) is True
    assert cache.append(k, -k, ints([3, 0]), wait=True) is False
    want = torch.zeros(3, page, D)
    flat = k[:, :, 0].cpu().half().float()
    want[0, 3], want[1], want[2] = flat[0, 0], flat[0, 1:5], flat[1, :4]
    assert torch.equal(K[:, 0].cpu().float(), want) and torch.equal(V[:, 0].cpu().float(), -want)
    for at in (8, 9, 2 ** 31 - 1):                                    # behind the table altogether
        assert cache.append(k, k, ints([at, at]), wait=True) is False
    assert torch.equal(K[:, 0].cpu().float(), want)


def test_two_graphs_with_their_own_workspaces_at_once(kv):
    """Replayed on two streams with nothing between them: each gives what its calls gave before the capture. The workspaces'
    objects are gone by then; their memory stays, because captured calls have used it."""
    rng = np.random.default_rng(41)
    graphs = []
    for k in range(2):
        lens = [900 + 300 * k, 1200, 5]
        _, K, V, table, bounds = make(rng, lens, 16, 2, 64, extra=8)
        cache = kv.PagedKV(K, V, table, bounds=bounds, workspace=kv.Workspace())
        q, vis = torch.randn(3, 2, 8, 64, device="cuda"), ints([n - 1 for n in lens])
        acc = torch.zeros(3, 2, table.shape[1] * 16, device="cuda")

        def step(cache=cache, q=q, vis=vis, acc=acc):
            out, lse = cache.attend(q, vis, lse=True, acc=acc)
            sel = cache.select(q, vis, 9)
            return out, lse, sel, cache.attend(q, vis, sel=sel)
        first = [x.clone() for x in step()]
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        graphs.append((graph, stream, out, first, (K, V, table, bounds, q, vis, acc)))     # the workspace: no one's any more
        del step, cache
    torch.cuda.synchronize()
    for _ in range(50):
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, first, _ in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@pytest.mark.parametrize("vis,step,window", [([2 ** 31 - 1, -2 ** 31, 100], 1, 0), ([2 ** 31 - 1] * 3, 2 ** 31 - 1, 0),
                                             ([-5, 0, 2 ** 31 - 1], 2 ** 31 - 1, 2 ** 31 - 1), ([100, 100, 100], 0, 1)])
def test_counts_at_the_ends_of_their_type(kv, vis, step, window):
    rng = np.random.default_rng(42)
    host, K, V, table, bounds = make(rng, [100, 100, 100], 10, 2, 64)
    q = rng.standard_normal((3, 2, 4, 64)).astype(np.float32)
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    attend_close(cache.attend(torch.from_numpy(q).cuda(), ints(vis), step=step, window=window, lse=True),
                 kv_ref.attend(host, q, vis, step=step, window=window), 64)
    got = cache.select(torch.from_numpy(q).cuda(), ints(vis), 4, step=step)
    assert np.array_equal(got.cpu().numpy(), kv_ref.select(host, q, vis, 4, step=step))
    acc = torch.rand(3, 2, 100, device="cuda")
    before = K.clone()
    assert cache.evict(ints(vis), 2 ** 31 - 1, acc).tolist() == [min(max(v, 0), 100) for v in vis]
    assert torch.equal(K, before)


@pytest.mark.parametrize("call", ["append", "evict"])
@pytest.mark.parametrize("tokens", [1, 16])
def test_queued_bounds_are_seen_by_a_product_with_them(kv, gpu_lib, call, tokens):
    """Bounds as the weights of an FP16 product (a caller's own page scores) right behind the call that writes them: the
    product's first loads may precede its wait on the kernel before, unless the ledger of queued writes holds the bounds.
    The product's FP32 sums of exact products over D = 64 are off by 64 roundings of the sum of their absolute values, and its
    FP16 result by half a step more."""
    D, heads, page, mp, ns = 64, 2, 16, 512, 4
    K = torch.zeros(ns * mp, heads, page, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    bounds = torch.zeros(ns * mp, heads, 2, D, dtype=torch.float16, device="cuda")
    table = ints(np.arange(ns * mp).reshape(ns, mp))
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    n = mp * page
    full, zero = ints([n] * ns), ints([0] * ns)
    A = torch.randn(tokens, D, device="cuda").half()
    rows = ns * mp * heads * 2
    C = torch.empty(tokens, rows, dtype=torch.float16, device="cuda")
    acc = torch.rand(ns, heads, n, device="cuda")
    for it in range(4):
        k = torch.randn(ns, n, heads, D, device="cuda") + it
        if call == "evict":
            cache.append(k, k, zero)
        torch.cuda.synchronize()
        assert gpu_lib.set_stream(torch.cuda.current_stream().cuda_stream or 1) == 0
        gpu_lib.set_nowait(1)
        try:
            if call == "append":
                cache.append(k, k, zero)
            else:
                cache.evict(full, n // 2, acc)
            status = gpu_lib.gemm(0, 0, 1, tokens, rows, D, 1.0, A.data_ptr(), D, bounds.data_ptr(), D, 0.0, C.data_ptr(), rows)
        finally:
            gpu_lib.set_nowait(0)
            assert gpu_lib.set_stream(None) == 0
        torch.cuda.synchronize()
        assert status == 0, gpu_lib.error()
        W = bounds.reshape(rows, D).double()
        ref, mass = A.double() @ W.T, A.double().abs() @ W.abs().T
        assert bool(((C.double() - ref).abs() <= mass * D * 2.0 ** -24 + ref.abs() * 2.0 ** -11 + 2.0 ** -24).all()), it


def test_writes_of_more_streams_than_the_ledger_holds(kv, gpu_lib):
    """Appends on 40 streams at once, each read back by the contiguous attention of its stream; twice."""
    D, heads, n = 128, 1, 256
    streams = [torch.cuda.Stream() for _ in range(40)]
    K = torch.zeros(40, 1, heads, n, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    q, O = torch.randn(40, 1, 1, 4, D, device="cuda"), torch.empty(40, 1, 1, 4, D, device="cuda")
    table, zero, vis = ints([[0]]), ints([0]), ints([n])
    caches = [kv.PagedKV(K[i], V[i], table) for i in range(40)]
    for it in range(2):
        k, v = (torch.randn(40, 1, n, heads, D, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        try:
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    for _ in range(3):
                        caches[i].append(k[i], v[i], zero)
            for i, st in enumerate(streams):
                assert gpu_lib.set_stream(st.cuda_stream) == 0
                size = K[i].numel() * 2
                assert gpu_lib.attn_dec(D, 4, heads, 1, 1, n, q[i].data_ptr(), 4 * D, D, 4 * D, K[i].data_ptr(), D, n * D, n * D, size,
                                        V[i].data_ptr(), D, n * D, n * D, size, O[i].data_ptr(), D ** -0.5, vis.data_ptr(), 0, 0,
                                        1) == 0, gpu_lib.error()
        finally:
            assert gpu_lib.set_stream(None) == 0
        torch.cuda.synchronize()
        for i in range(0, 40, 7):
            host = {"K": k[i].half().cpu().numpy().transpose(0, 2, 1, 3), "V": v[i].half().cpu().numpy().transpose(0, 2, 1, 3),
                    "table": np.zeros((1, 1), np.int32), "bounds": None}
            ref = kv_ref.attend(host, q[i].cpu().numpy(), [n])
            attend_close((O[i], torch.from_numpy(ref[1])), ref, D)


def _dec(gpu_lib, K, V, q, O, n, vis):
    """gen9blas_attn_dec of all keys of a contiguous [1, heads, n, D] cache on torch's current stream, queued."""
    heads, D = K.shape[1], K.shape[3]
    H, size = q.shape[2], K.numel() * 2
    assert gpu_lib.set_stream(torch.cuda.current_stream().cuda_stream or 1) == 0
    try:
        return gpu_lib.attn_dec(D, H, heads, 1, 1, n, q.data_ptr(), H * D, D, H * D, K.data_ptr(), D, n * D, heads * n * D, size,
                                V.data_ptr(), D, n * D, heads * n * D, size, O.data_ptr(), D ** -0.5, vis.data_ptr(), 0, 0, 0)
    finally:
        assert gpu_lib.set_stream(None) == 0


@pytest.mark.parametrize("where", ["captured", "beside a capture"])
def test_a_write_in_the_queue_does_not_end_a_capture(kv, gpu_lib, where):
    """append queued outside of a capture; then the contiguous attention of the same memory, itself captured, or called on
    another stream while a capture runs: the ledger has an entry for its keys and must not ask for its event there."""
    D, heads, n = 128, 2, 4096
    K = torch.zeros(1, heads, n, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    q, O, x = torch.randn(1, 1, 8, D, device="cuda"), torch.zeros(1, 1, 8, D, device="cuda"), torch.zeros(1, device="cuda")
    cache, vis, zero = kv.PagedKV(K, V, ints([[0]])), ints([n]), ints([0])
    k, v = (torch.randn(1, n, heads, D, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert _dec(gpu_lib, K, V, q, O, n, vis) == 0          # buffers and kernels are there before the capture
    with torch.cuda.stream(side):
        assert _dec(gpu_lib, K, V, q, O, n, vis) == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    if where == "captured":
        cache.append(k, v, zero)
        with torch.cuda.graph(graph):
            x.add_(1)
            assert _dec(gpu_lib, K, V, q, O, n, vis) == 0, gpu_lib.error()
        assert not O.any()
    else:
        with torch.cuda.stream(side):
            cache.append(k, v, zero)
        with torch.cuda.graph(graph):
            x.add_(1)
            with torch.cuda.stream(side):
                assert _dec(gpu_lib, K, V, q, O, n, vis) == 0, gpu_lib.error()
    graph.replay()
    torch.cuda.synchronize()
    assert x.item() == 1
    host = {"K": k.half().cpu().numpy().transpose(0, 2, 1, 3), "V": v.half().cpu().numpy().transpose(0, 2, 1, 3),
            "table": np.zeros((1, 1), np.int32), "bounds": None}
    ref = kv_ref.attend(host, q.cpu().numpy(), [n])
    attend_close((O, torch.from_numpy(ref[1])), ref, D)


def test_captured_writes_are_seen_by_captured_early_readers(kv, gpu_lib):
    """append, the contiguous attention of the same memory and a product with the bounds, captured into one graph: at each replay
    the readers wait for that replay's writes. Two graphs of the same calls, replayed in turn."""
    D, heads, n = 64, 2, 4096
    K = torch.zeros(1, heads, n, D, dtype=torch.float16, device="cuda")
    V = torch.zeros_like(K)
    bounds = torch.zeros(1, heads, 2, D, dtype=torch.float16, device="cuda")
    q, O = torch.randn(1, 1, 8, D, device="cuda"), torch.zeros(1, 1, 8, D, device="cuda")
    A, C = torch.randn(2, D, device="cuda").half(), torch.zeros(2, heads * 2, dtype=torch.float16, device="cuda")
    k, v = (torch.zeros(1, n, heads, D, device="cuda") for _ in range(2))
    cache, vis, zero = kv.PagedKV(K, V, ints([[0]]), bounds=bounds), ints([n]), ints([0])

    def step():
        cache.append(k, v, zero)
        assert _dec(gpu_lib, K, V, q, O, n, vis) == 0, gpu_lib.error()
        assert gpu_lib.set_stream(torch.cuda.current_stream().cuda_stream or 1) == 0
        gpu_lib.set_nowait(1)
        try:
            assert gpu_lib.gemm(0, 0, 1, 2, heads * 2, D, 1.0, A.data_ptr(), D, bounds.data_ptr(), D, 0.0, C.data_ptr(), heads * 2) == 0
        finally:
            gpu_lib.set_nowait(0)
            assert gpu_lib.set_stream(None) == 0
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step()
    for it in range(6):
        kn, vn = (torch.randn(1, n, heads, D, device="cuda") + it for _ in range(2))
        k.copy_(kn)
        v.copy_(vn)
        graphs[it % 2].replay()
        torch.cuda.synchronize()
        host = {"K": kn.half().cpu().numpy().transpose(0, 2, 1, 3), "V": vn.half().cpu().numpy().transpose(0, 2, 1, 3),
                "table": np.zeros((1, 1), np.int32), "bounds": None}
        ref = kv_ref.attend(host, q.cpu().numpy(), [n])
        attend_close((O, torch.from_numpy(ref[1])), ref, D)
        W = torch.stack([kn[0].half().amin(0), kn[0].half().amax(0)], 1).reshape(heads * 2, D).double()   # FP16 products, as above
        want, mass = A.double() @ W.T, A.double().abs() @ W.abs().T
        assert bool(((C.double() - want).abs() <= mass * D * 2.0 ** -24 + want.abs() * 2.0 ** -11 + 2.0 ** -24).all()), it


def _unordered(rng, mp, m, kind):
    """Lists of m entries whose pages come twice, out of order or between entries that name no page."""
    if kind == "short":
        return [[3, -1, 3], [5, 2, 5], [5, 3, 4, 5], [mp, 3, 2 ** 31 - 1, 4], [-1, -2 ** 31, 2, 2], [0, 0, 1, 0, 1, 2], [7, 6, 5, 4, 3, 8]]
    x = np.sort(rng.integers(0, mp, m)).astype(np.int64)
    back = rng.integers(1, m, m // 8)
    x[back] = x[rng.integers(0, back)]                                  # an earlier one again
    x[rng.integers(0, m, m // 8)] = rng.choice([-1, mp, 2 ** 31 - 1, -2 ** 31], m // 8)
    return x


@pytest.mark.parametrize("page,group,D,nq,m,kind", [(16, 4, 64, 2, 6, "short"), (1, 2, 64, 2, 6, "short"), (5, 12, 128, 1, 6, "short"),
                                                    (64, 4, 256, 1, 6, "short"), (16, 4, 128, 3, 100, "long"), (3, 9, 64, 1, 200, "long"),
                                                    (1, 1, 64, 1, 700, "long"), (128, 4, 64, 2, 40, "long")])
def test_lists_that_name_a_page_twice(kv, page, group, D, nq, m, kind):
    """A page counts once wherever its other mentions stand; its weights are added once, and the same bits each time."""
    rng = np.random.default_rng(page + m)
    heads, mp = 2, max(10, m)
    host, K, V, table, _ = make(rng, [mp * page - nq, mp * page - nq - 3], page, heads, D, extra=nq)
    assert table.shape[1] == mp
    sel = np.full((2, nq, heads, m), -1, np.int32)
    flat = sel.reshape(-1, m)
    for i in range(len(flat)):
        x = _unordered(rng, mp, m, kind)
        x = x[(i + page) % len(x)] if kind == "short" else x
        flat[i, :len(x)] = x
    vis = np.array([mp * page - nq, mp * page - nq - 3])
    q = rng.standard_normal((2, nq, heads * group, D)).astype(np.float32)
    ref = kv_ref.attend(host, q, vis, sel=sel)
    accs = []
    for _ in range(3):
        acc = torch.zeros(2, heads, mp * page, device="cuda")
        got = kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints(vis), sel=torch.from_numpy(sel).cuda(), acc=acc, lse=True)
        attend_close(got, ref, D)
        accs.append(acc)
    assert torch.equal(accs[0], accs[1]) and torch.equal(accs[0], accs[2])
    e = ref[3].max() * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
    assert np.all(np.abs(accs[0].cpu().numpy() - ref[2]) <= (4 * e + 2.0 ** -19 + nq * group * 2.0 ** -23) * ref[2] + 1e-30)


@pytest.mark.parametrize("nq,step,window", [(1, 1, 0), (3, 1, 5), (2, 20, 7)])
def test_weights_leave_slots_that_no_token_sees_as_they_were(kv, nq, step, window):
    """Bit for bit, a negative zero among them: behind the last slot seen, before and between the windows, without a page."""
    rng = np.random.default_rng(50)
    host, K, V, table, _ = make(rng, [64, 50], 8, 2, 64, holes=[(0, 1), (1, 4)])
    q = rng.standard_normal((2, nq, 8, 64)).astype(np.float32)
    acc = torch.full((2, 2, 64), -0.0, device="cuda")
    vis = [13, 34]
    kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints(vis), step=step, window=window, acc=acc)
    W = kv_ref.attend(host, q, vis, step=step, window=window)[2]
    bits = acc.cpu().numpy().view(np.int32)
    assert np.all(bits[W == 0] == -2 ** 31) and np.all(acc.cpu().numpy()[W > 0] > 0)


def test_tensors_that_require_a_gradient_are_refused(kv):
    """The operators give none: rather an error than a gradient that is lost without a word. Without gradients they serve."""
    rng = np.random.default_rng(51)
    _, K, V, table, bounds = make(rng, [40], 8, 2, 64)
    n, q, k = ints([30]), torch.randn(1, 1, 4, 64, device="cuda"), torch.randn(1, 1, 2, 64, device="cuda")
    cache = kv.PagedKV(K, V, table, bounds=bounds)
    want, pages = cache.attend(q, n), cache.select(q, n, 2)
    wq, wk = q.clone().requires_grad_(), k.clone().requires_grad_()
    for call in (lambda: cache.attend(wq, n), lambda: cache.attend(wq * 2, n), lambda: cache.select(wq, n, 2),
                 lambda: cache.append(wk, k, n), lambda: cache.append(k, wk, n)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    leaf = kv.PagedKV(K.clone().requires_grad_(), V, table, bounds=bounds)
    with pytest.raises(ValueError, match="gradient"):
        leaf.attend(q, n)
    with torch.no_grad():
        assert torch.equal(cache.attend(wq, n), want) and torch.equal(cache.select(wq, n, 2), pages)
        assert torch.equal(leaf.attend(q, n), want) and not cache.attend(wq, n).requires_grad
        cache.append(wk, wk, n)
    with torch.inference_mode():
        cache.attend(wq, n)
    assert torch.equal(cache.attend(wq.detach(), n), cache.attend(q, n))


def test_a_workspace_collected_during_a_capture_does_not_end_it(kv):
    """Freeing waits for the device, which a capture does not allow: it is put off to the next workspace."""
    rng = np.random.default_rng(52)
    host, K, V, table, _ = make(rng, [40], 16, 1, 64)
    q, n = torch.randn(1, 1, 4, 64, device="cuda"), ints([40])
    kept, other = (kv.PagedKV(K, V, table, workspace=kv.Workspace()) for _ in range(2))
    want = kept.attend(q, n)
    assert torch.equal(other.attend(q, n), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = kept.attend(q, n)
        del other
        assert len(kv._dead) == 1
        second = kept.attend(q, n)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)
    kv.Workspace()
    assert not kv._dead
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(second, want)


def test_the_legacy_stream_beside_a_blocking_stream_s_capture(kv, gpu_lib):
    """A call on the legacy stream is refused while a stream that synchronises with it is captured, and the capture goes on."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    rng = np.random.default_rng(53)
    _, K, V, table, _ = make(rng, [40], 16, 1, 64)
    cache = kv.PagedKV(K, V, table, workspace=kv.Workspace())
    q, k, n, x = torch.randn(1, 1, 4, 64, device="cuda"), torch.randn(1, 1, 1, 64, device="cuda"), ints([40]), torch.zeros(64, device="cuda")
    want, zero = cache.attend(q, n), ints([0])
    before = K.clone()
    torch.cuda.synchronize()
    err, stream = rt.cudaStreamCreate()
    assert err == 0
    try:
        assert rt.cudaStreamBeginCapture(stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed)[0] == 0
        assert rt.cudaMemsetAsync(x.data_ptr(), 1, 256, stream)[0] == 0
        for call in (lambda: cache.append(k, k, zero, count=zero), lambda: kv._fn["attn_paged"](cache._ref, 4, 1, q.data_ptr(), 256, 64, 256,
                     n.data_ptr(), 1, 0, None, 0, 0.125, q.data_ptr(), None, None, 0, 0, cache.workspace.handle, 0)):
            try:
                assert call() not in (0, None)
            except RuntimeError as e:
                assert "capture" in str(e)
        err, graph = rt.cudaStreamEndCapture(stream)
        assert err == 0                                       # the capture has not been ended by the calls
        assert rt.cudaGraphDestroy(graph)[0] == 0
    finally:
        rt.cudaStreamDestroy(stream)
    torch.cuda.synchronize()
    assert torch.equal(cache.attend(q, n), want) and torch.equal(K, before) and not x.any()

"""GPU parity of the paged key-value cache at sizes that take other kernels than small ones do: two tiles of query rows a unit
(attn_paged), rows of slots and of pages that the registers of a CTA or of a cluster do not hold (kv_evict, kv_select).
References in 64 bits: oracle/kv_ref.py, or whole-array NumPy forms of the same definitions where its slot-by-slot ones
would take minutes."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import kv_ref  # noqa: E402
from test_kv_gpu import attend_close, ints, make  # noqa: E402

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def kv(gpu_lib):
    import g9kv
    return g9kv


# ------------------------------------------------------------------------------------------------ two row tiles
def wide_table(host, table, slots):
    """The same cache with a table of `slots` slots: places behind those in use have no page."""
    page = host["K"].shape[2]
    mp = -(-slots // page)
    out = np.full((table.shape[0], mp), -1, np.int32)
    out[:, :table.shape[1]] = host["table"]
    host["table"] = out
    return torch.from_numpy(out.copy()).cuda()


def two_tiles(ns, heads, rows, slots, dim):
    """Units of two tiles of eight rows are for what reads more than 48 MiB with one (attn_paged); by the table's room."""
    return rows > 8 and ns * heads * -(-rows // 8) * slots * dim * 4 > 48 << 20


@pytest.mark.parametrize("lens,room,page,heads,group,D,nq,window", [
    ([300, 0, 41], 30000, 16, 2, 4, 128, 3, 0),          # 12 rows of a head: one unit, its second tile half full
    ([300, 17], 60000, 24, 2, 5, 64, 4, 0),              # 20 rows: a whole unit and one of four rows
    ([200, 33], 30000, 7, 1, 12, 256, 1, 0),
    ([90, 250], 40000, 32, 2, 9, 200, 2, 0),
    ([260], 120000, 16, 1, 16, 80, 3, 0),
    ([14000, 13400, 40], 14016, 32, 2, 6, 128, 2, 13000),   # windows long enough to count as much
    ([9000, 8100], 9008, 16, 3, 10, 64, 3, 8500)])
@pytest.mark.parametrize("weights", [False, True])
def test_attend_with_two_row_tiles(kv, lens, room, page, heads, group, D, nq, window, weights):
    assert two_tiles(len(lens), heads, group * nq, min(room, window + nq) if window else room, D)
    rng = np.random.default_rng(len(lens) * 1000 + page + D + nq)
    host, K, V, table, _ = make(rng, [n + nq - 1 if n else 0 for n in lens], page, heads, D, poison=True)
    table = wide_table(host, table, room)
    vis = np.array(lens) - (nq - 1) * (np.array(lens) == 0)
    q = (rng.standard_normal((len(lens), nq, heads * group, D)) * 2).astype(np.float32)
    acc0 = rng.random((len(lens), heads, table.shape[1] * page)).astype(np.float32)
    acc = torch.from_numpy(acc0).cuda() if weights else None
    ref = kv_ref.attend(host, q, vis, window=window)
    cache = kv.PagedKV(K, V, table)
    attend_close(cache.attend(torch.from_numpy(q).cuda(), ints(vis), window=window, acc=acc, lse=True), ref, D)
    if weights:     # the bound of test_attend: a weight is off by 2e and its own roundings, their sum by one rounding each
        e = ref[3].max() * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
        a = acc.cpu().numpy()
        assert np.all(np.abs(a - (acc0 + ref[2])) <= (4 * e + 2.0 ** -19 + nq * group * 2.0 ** -24) * ref[2] + 2.0 ** -23 * (acc0 + ref[2]))
        assert np.array_equal(a[ref[2] == 0], acc0[ref[2] == 0])
        again = torch.from_numpy(acc0).cuda()
        cache.attend(torch.from_numpy(q).cuda(), ints(vis), window=window, acc=again)
        assert torch.equal(acc, again)


@pytest.mark.parametrize("group,D,nq,m,page", [(12, 128, 2, 200, 32), (9, 64, 1, 220, 64), (16, 256, 1, 110, 32)])
def test_attend_chosen_pages_with_two_row_tiles(kv, group, D, nq, m, page):
    rng = np.random.default_rng(group)
    lens, heads = [m * page + 900, m * page, 70, 9000], 2
    assert two_tiles(4, heads, group, m * page, D)
    host, K, V, table, _ = make(rng, [n + nq - 1 for n in lens], page, heads, D, poison=True, holes=[(0, 3)])
    mp = table.shape[1]
    sel = np.full((4, nq, heads, m), -1, np.int32)
    for s in range(4):
        for t in range(nq):
            for g in range(heads):
                n = rng.integers(m // 2, m + 1)
                sel[s, t, g, :n] = np.sort(rng.permutation(mp)[:n])
    q = rng.standard_normal((4, nq, heads * group, D)).astype(np.float32)
    ref = kv_ref.attend(host, q, lens, sel=sel)
    acc = torch.zeros(4, heads, mp * page, device="cuda")
    attend_close(kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints(lens), sel=torch.from_numpy(sel).cuda(), acc=acc,
                                                lse=True), ref, D)
    e = ref[3].max() * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
    assert np.all(np.abs(acc.cpu().numpy() - ref[2]) <= (4 * e + 2.0 ** -19 + nq * group * 2.0 ** -23) * ref[2] + 1e-30)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_draft_tokens_with_wild_values_ahead_in_two_row_tiles(kv, D):
    """Values that only later draft tokens see are infinite or NaN: the others' results stay as they are."""
    rng = np.random.default_rng(9)
    lens, nq, heads, room = [130, 47], 5, 2, 8000000 // D
    assert two_tiles(2, heads, 4 * nq, room, D)
    host, K, V, table, _ = make(rng, [n + nq - 1 for n in lens], 16, heads, D)
    table = wide_table(host, table, room)
    q = torch.randn(2, nq, 8, D, device="cuda")
    clean = kv.PagedKV(K, V, table).attend(q, ints(lens))
    for s, n in enumerate(lens):
        for k, bad in ((n + 2, float("inf")), (n + 3, float("nan"))):
            V[table[s, k // 16].item(), :, k % 16] = bad
    got = kv.PagedKV(K, V, table).attend(q, ints(lens))
    assert torch.equal(got[:, :3], clean[:, :3]) and not torch.isfinite(got[:, 3:]).any()


# ------------------------------------------------------------------------------------------------ eviction of long rows
def evict_ref(K, V, bounds, table, lens, keep, acc, pos, first, recent):
    """As kv_ref.evict, by whole arrays; in place."""
    page, heads = K.shape[2], K.shape[1]
    for s, n in enumerate(lens):
        if n <= keep:
            continue
        for g in range(heads):
            at = np.arange(n) if pos is None else pos[s, g, :n].astype(np.int64)
            sure = (at < first) | (at > at.max() - recent)
            w = acc[s, g, :n].astype(np.float64)
            rank = np.lexsort((np.arange(n), -np.where(np.isnan(w), 0.0, w), np.where(sure, 0, np.where(np.isnan(w), 2, 1))))
            stay = np.zeros(n, bool)
            stay[rank[:keep]] = True
            holes, movers = np.flatnonzero(~stay[:keep]), np.flatnonzero(stay[keep:]) + keep
            to, come = table[s, holes // page], table[s, movers // page]
            K[to, g, holes % page] = K[come, g, movers % page]
            V[to, g, holes % page] = V[come, g, movers % page]
            acc[s, g, holes] = acc[s, g, movers]
            if pos is not None:
                pos[s, g, holes] = pos[s, g, movers]
            changed = set(holes // page) | ({(keep - 1) // page} if keep % page else set())
            for o in changed:
                rows = K[table[s, o], g, :min(page, keep - o * page)]
                bounds[table[s, o], g] = np.stack([rows.min(0), rows.max(0)])


@pytest.mark.parametrize("lens,keep,page,heads", [([70000], 33333, 16, 1), ([70000, 20000, 65536, 65537], 65536, 64, 1),
                                                  ([140000, 139999], 60001, 48, 1), ([70001] * 3, 69990, 16, 2), ([270000], 7, 128, 1)])
@pytest.mark.parametrize("with_pos", [False, True])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long_rows(kv, lens, keep, page, heads, with_pos, ties):
    """More slots than eight CTAs hold in registers. Ties: few different weights, the border among thousands of equal ones."""
    rng = np.random.default_rng(keep + page)
    host, K, V, table, bounds = make(rng, lens, page, heads, 8)
    cap = table.shape[1] * page
    acc = rng.exponential(size=(len(lens), heads, cap)).astype(np.float32)
    if ties:
        acc = np.floor(acc * 2)
        acc[:, :, 5::1000] = np.nan
    pos = rng.permuted(np.tile(np.arange(cap, dtype=np.int32), (len(lens), heads, 1)), axis=-1) if with_pos else None
    dacc, dpos = torch.from_numpy(acc.copy()).cuda(), torch.from_numpy(pos.copy()).cuda() if with_pos else None
    got = kv.PagedKV(K, V, table, bounds=bounds).evict(ints(lens), keep, dacc, dpos, first=min(3, keep // 2), recent=min(30, keep // 2))
    evict_ref(host["K"], host["V"], host["bounds"], host["table"], lens, keep, acc, pos, min(3, keep // 2), min(30, keep // 2))
    assert got.tolist() == [min(n, keep) for n in lens]
    assert np.array_equal(dacc.cpu().numpy(), acc, equal_nan=True)
    assert pos is None or np.array_equal(dpos.cpu().numpy(), pos)
    for name, x in (("K", K), ("V", V), ("bounds", bounds)):
        assert np.array_equal(x.cpu().numpy(), host[name]), name


# ------------------------------------------------------------------------------------------------ selection over long rows
def select_ref(bounds, table, q, have, m, first, last):
    """As kv_ref.select for one page per slot, by whole arrays: every stream sees `have` pages."""
    ns, nq, H, D = q.shape
    heads = bounds.shape[1]
    out = np.full((ns, nq, heads, m), -1, np.int32)
    place = np.arange(have)
    for s in range(ns):
        ids = table[s, :have]
        inside = (ids >= 0) & (ids < bounds.shape[0])
        b = bounds[np.where(inside, ids, 0)].astype(np.float64)
        for t in range(nq):
            for g in range(heads):
                qd = q[s, t, g * (H // heads):(g + 1) * (H // heads)].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    score = np.stack([np.maximum(x * b[:, g, 0], x * b[:, g, 1]).sum(-1) for x in qd])
                gone = ~inside | np.isnan(score).any(0)
                kind = np.where((place < first) | (place >= have - last), 0, np.where(gone, 2, 1))
                best = np.sort(np.lexsort((place, -np.where(kind == 1, score.max(0), 0.0), kind))[:m])
                out[s, t, g, :len(best)] = best
    return out


@pytest.mark.parametrize("n,m,ns,heads,group", [
    (1800, 64, 1, 2, 4), (2049, 100, 80, 2, 1), (5000, 3000, 1, 1, 4), (9000, 600, 1, 2, 4), (20000, 64, 2, 1, 4), (20000, 19990, 1, 1, 2),
    (8193, 8192, 1, 2, 1), (9000, 50, 75, 2, 1)])
@pytest.mark.parametrize("kind", ["distinct", "equal", "gone"])
def test_select_long_rows(kv, n, m, ns, heads, group, kind):
    """Pages of one slot, more than the registers of a CTA hold (8192); with `equal`, three kinds of pages only, so that thousands
    lie at the border; with `gone`, pages without a place, NaN and infinite bounds as well."""
    rng = np.random.default_rng(n + m)
    D = 8
    K = torch.zeros(n, heads, 1, D, dtype=torch.float16, device="cuda")
    if kind == "distinct":
        bounds = rng.standard_normal((n, heads, 2, D)).astype(np.float16)
    else:
        bounds = rng.standard_normal((3, heads, 2, D)).astype(np.float16)[rng.integers(0, 3, n)]
    bounds.sort(axis=2)
    table = np.stack([rng.permutation(n) for _ in range(ns)]).astype(np.int32)
    if kind == "gone":
        table[:, 3::17] = -1
        table[:, n - 5] = n
        bounds[5::31, :, 1, 3] = np.inf
        bounds[6::31, :, :, 3] = np.nan
    q = rng.standard_normal((ns, 1, heads * group, D)).astype(np.float32)
    got = kv.PagedKV(K, K, ints(table), bounds=torch.from_numpy(bounds).cuda()).select(torch.from_numpy(q).cuda(), ints([n] * ns), m,
                                                                                       first=2, last=3)
    assert np.array_equal(got.cpu().numpy(), select_ref(bounds, table, q, n, m, 2, 3))


def by_slots(host):
    """The same cache in pages of one slot."""
    K, page = host["K"], host["K"].shape[2]
    out = {x: host[x].transpose(0, 2, 1, 3).reshape(-1, K.shape[1], 1, K.shape[3]) for x in "KV"}
    t = host["table"].astype(np.int64)
    out["table"] = np.where(t[:, :, None] >= 0, t[:, :, None] * page + np.arange(page), -1).reshape(len(t), -1).astype(np.int32)
    return out


@pytest.mark.parametrize("group,D,nq,room", [(4, 128, 1, 0), (3, 80, 4, 0), (4, 256, 2, 0), (4, 64, 5, 120000), (12, 128, 1, 30000), (5, 256, 3, 30000)])
@pytest.mark.parametrize("chosen", [False, True])
def test_scores_of_minus_infinity_have_no_weight(kv, group, D, nq, room, chosen):
    """Keys with elements of -inf (and +inf against a negative query): their scores are -inf, whatever the parts of the query that
    meet them, and their slots are as if they were not seen. Query elements there from normal ones to ones that fall below all
    FP16 parts; a row all of whose scores are -inf gives 0 and -inf."""
    rng = np.random.default_rng(group + D)
    lens, heads, page = [300, 40, 16], 2, 16
    host, K, V, table, _ = make(rng, [n + nq - 1 for n in lens], page, heads, D)
    if room and not chosen:
        table = wide_table(host, table, room)
        assert two_tiles(3, heads, group * nq, room, D)
    q = rng.standard_normal((3, nq, heads * group, D)).astype(np.float32)
    q[..., 5] = np.abs(q[..., 5]) + 0.1
    q[..., 6] = -2.0 ** -10                               # exact in one part: the second part is zero
    q[..., 7] = 1e-12
    ref = by_slots(host)
    gone = [sorted(rng.permutation(n)[:n // 3]) for n in lens[:2]] + [range(lens[2])]
    for s, ks in enumerate(gone):
        for k in ks:
            p, i = host["table"][s, k // page], k % page
            d = rng.choice([5, 6, 7])
            K[int(p), :, i, int(d)] = float("inf") if d == 6 else -float("inf")
            if k % 3 == 0:
                K[int(p), :, i, 5] = -float("inf")
            ref["table"][s, k] = -1
    for s, n in enumerate(lens):
        ref["table"][s, n:] = -1
    sel = None
    rsel = None
    if chosen:
        mp = host["table"].shape[1]
        sel = np.full((3, nq, heads, 9), -1, np.int32)
        for i in np.ndindex(3, nq, heads):
            m = rng.integers(1, 10)
            sel[i][:m] = np.sort(rng.permutation(mp)[:m])
        rsel = np.where(sel[..., None] >= 0, sel[..., None] * page + np.arange(page), -1).reshape(3, nq, heads, -1)
    vis = [lens[0], lens[1], lens[2]]
    want = kv_ref.attend(ref, q, vis, step=0, sel=rsel)
    acc = torch.full((3, heads, table.shape[1] * page), 0.25, device="cuda")
    got = kv.PagedKV(K, V, table).attend(torch.from_numpy(q).cuda(), ints(vis), step=0, acc=acc, lse=True,
                                         sel=None if sel is None else torch.from_numpy(sel).cuda())
    attend_close(got, want, D)
    assert np.isneginf(want[1][2]).all() and not got[0][2].any()
    a, W = acc.cpu().numpy(), np.zeros(acc.shape)
    W[:, :, :want[2].shape[2]] = want[2]
    e = want[3].max() * (2.0 ** -21 + (D + 4) * 2.0 ** -24)
    assert np.all(np.abs(a - (0.25 + W)) <= (4 * e + 2.0 ** -19 + nq * group * 2.0 ** -23) * W + 2.0 ** -23 * (0.25 + W))
    assert np.all(a[W == 0] == 0.25)


@pytest.mark.parametrize("q,hi", [(float(np.finfo(np.float32).max), 1.0), (-float(np.finfo(np.float32).max), -1.0), (3e38, 1.0)])
@pytest.mark.parametrize("n,m", [(9000, 8500), (9000, 9), (20000, 19000), (600, 550)])
def test_select_long_rows_with_scores_at_the_end_of_float32(kv, q, hi, n, m):
    """Equal scores near FP32's largest number, where the border plus the error bound of the scores passes it: every place of the
    list is written, the lowest ones. Some pages lie below by a step of FP16."""
    D = 8
    K = torch.zeros(n, 1, 1, D, dtype=torch.float16, device="cuda")
    bounds = np.zeros((n, 1, 2, D), np.float16)
    bounds[:, 0, :, 0] = hi
    low = np.arange(7, n, 100)
    bounds[low, 0, :, 0] = hi * (1 - 2.0 ** -11)
    qs = np.zeros((1, 1, 1, D), np.float32)
    qs[..., 0] = q
    out = torch.full((1, 1, 1, m), -7, dtype=torch.int32, device="cuda")
    table = np.arange(n, dtype=np.int32)[None]
    got = kv.PagedKV(K, K, ints(table), bounds=torch.from_numpy(bounds).cuda()).select(torch.from_numpy(qs).cuda(), ints([n]), m, first=0,
                                                                                       last=0, out=out)
    assert np.array_equal(got.cpu().numpy(), select_ref(bounds, table, qs, n, m, 0, 0))

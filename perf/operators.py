"""Timed cases of the paged key-value cache: cache writes, attention over pages, page selection and eviction.

Each case is one call on a cache of a decoder's layer: FP16 keys and values in pages of a shared pool, a table of page
numbers for each stream, F32 activations. `run` computes a case by elementary torch operations, or, with `own` set, by
the library's paged-cache calls (gen9-gpu-blas_b200/g9kv.py). Sizes follow this repository's decoding benchmark
(32 query heads over 8 key-value heads of 128, 8 streams of 4096 keys) and spread around it.
"""
import math
import os
import sys

import torch

own = False

_DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    base = {"heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # one decoding step of a mid-size batch writes its new keys and values (latency: 32 rows per head)
        {"name": "append one token", "op": "append", "streams": 32, "keys": 2000, "new": 1, "page": 16, **base},
        # four prompts of uneven length enter the cache at once
        {"name": "append prompts", "op": "append", "streams": 4, "keys": 100, "new": 2000, "page": 32, **base},
        # a single chat's decoding step: latency
        {"name": "attend one stream", "op": "attend", "streams": 1, "new": 1, "keys": 1000, "page": 16, "window": 0,
         "weights": False, "chosen": 0, **base},
        # this repository's decoding benchmark, in pages and with uneven lengths
        {"name": "attend batch", "op": "attend", "streams": 8, "new": 1, "keys": 4096, "page": 32, "window": 0,
         "weights": False, "chosen": 0, **base},
        # two long documents, an odd number of keys
        {"name": "attend long", "op": "attend", "streams": 2, "new": 1, "keys": 131071, "page": 64, "window": 0,
         "weights": False, "chosen": 0, **base},
        # four drafted tokens checked at once in a smaller model with a sliding window, pages that are no power of two
        {"name": "attend drafts in a window", "op": "attend", "streams": 16, "new": 4, "keys": 5000, "page": 24,
         "window": 2048, "weights": False, "chosen": 0, "heads": 16, "kv_heads": 2, "dim": 64},
        # a decoding step that also keeps count of the attention each key receives
        {"name": "attend with weights", "op": "attend", "streams": 8, "new": 1, "keys": 8192, "page": 16, "window": 0,
         "weights": True, "chosen": 0, **base},
        # a decoding step over 64 chosen pages of each long stream
        {"name": "attend chosen pages", "op": "attend", "streams": 16, "new": 1, "keys": 65536, "page": 32, "window": 0,
         "weights": False, "chosen": 64, **base},
        # the choice of pages for one stream (latency) and for a batch of long ones
        {"name": "select one stream", "op": "select", "streams": 1, "new": 1, "keys": 20000, "page": 16, "chosen": 64, **base},
        {"name": "select batch", "op": "select", "streams": 16, "new": 1, "keys": 65536, "page": 32, "chosen": 64, **base},
        # a cache at its budget drops the few slots by which each stream has outgrown it
        {"name": "evict a few", "op": "evict", "streams": 32, "keys": 2064, "keep": 2048, "page": 16, **base},
        # prompts cut to half their length before decoding
        {"name": "evict half", "op": "evict", "streams": 8, "keys": 16384, "keep": 8192, "page": 32, **base},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv_heads = rng.choice([1, 2, 4, 8])
    c = {"op": rng.choice(["append", "attend", "attend", "attend", "select", "evict"]),
         "kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), "dim": rng.choice([64, 80, 96, 128, 128, 128]),
         "page": rng.choice([8, 16, 16, 24, 32, 64, 128]), "streams": _log(rng, 1, 40)}
    room = 2 * 131071 * 8 * 128 // (c["streams"] * kv_heads * c["dim"])   # keys a stream may have: the largest listed cache
    c["keys"] = _log(rng, 16, min(200000, room))
    if c["op"] == "append":
        c["new"] = rng.choice([1, 1, 2, 5, _log(rng, 6, 2000)])
        c["keys"] = min(c["keys"], 8192)
        while c["streams"] * c["new"] * kv_heads * c["dim"] > 4 * 2000 * 8 * 128:
            c["new"] = max(1, c["new"] // 2)
    elif c["op"] == "attend":
        c["new"] = rng.choice([1, 1, 1, 2, 3, 5])
        c["window"] = rng.choice([0, 0, 0, _log(rng, 8, 8192)])
        c["weights"] = rng.random() < 0.3
        c["chosen"] = 0 if c["window"] else rng.choice([0, 0, _log(rng, 1, 100)])
        while c["new"] * c["keys"] * c["heads"] * c["streams"] > 2 * 131071 * 32:
            c["keys"] = max(16, c["keys"] // 2)
        while c["chosen"] > 1 and c["streams"] * c["new"] * kv_heads * c["chosen"] * c["page"] * c["dim"] > room * c["streams"] * kv_heads * c["dim"]:
            c["chosen"] //= 2
    elif c["op"] == "select":
        c["new"] = rng.choice([1, 1, 2, 4])
        c["chosen"] = _log(rng, 1, 200)
        while c["new"] * c["keys"] // c["page"] * c["heads"] * c["streams"] > 16 * 2048 * 32:
            c["keys"] = max(16, c["keys"] // 2)
    else:
        while c["streams"] * c["keys"] * kv_heads * c["dim"] > 8 * 16384 * 8 * 128:
            c["keys"] = c["keys"] // 2
        c["keys"] = max(64, c["keys"])
        c["keep"] = max(48, int(c["keys"] * rng.uniform(0.2, 1.0)))
    return c


def _lengths(c):
    """Slots in use for each stream before the call: uneven, by the case alone."""
    n, keys = c["streams"], c["keys"]
    if c["op"] == "evict" and 0 < keys - c["keep"] <= 64:   # outgrown by a few
        return [keys - (s * 5) % (keys - c["keep"] + 1) for s in range(n)]
    return [keys - (s * 37 * keys // 101) % (keys // 2 + 1) for s in range(n)]


def _counts(c):
    """Tokens that each stream of an append really brings (the batch is padded to `new`)."""
    return [c["new"] - (s * 29 * c["new"] // 97) % (c["new"] // 2 + 1) for s in range(c["streams"])]


_FIRST, _RECENT = 4, 32   # of an eviction: attention sinks and the newest tokens stay


def prepare(case, seed):
    c = case
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    ns, hk, d, page, h = c["streams"], c["kv_heads"], c["dim"], c["page"], c["heads"]
    lens = _lengths(c)
    most = max(lens) + (c["new"] if c["op"] in ("append", "attend", "select") else 0)
    mp = -(-most // page) + 1
    used = ns * mp
    pool = used + 7
    f16 = dict(device=_DEV, dtype=torch.float16)
    # keys of a page resemble each other, as keys of neighbouring tokens do
    K = torch.randn(pool, hk, page, d, generator=g, **f16)
    K += torch.randn(pool, hk, 1, d, generator=g, **f16)
    V = torch.randn(pool, hk, page, d, generator=g, **f16)
    table = torch.randperm(pool, generator=g, device=_DEV)[:used].view(ns, mp).to(torch.int32)
    ends = torch.tensor(lens, device=_DEV, dtype=torch.int32)
    blank = torch.arange(mp, device=_DEV)[None] * page >= (ends[:, None] + (c.get("new", 0)))
    table = torch.where(blank, torch.full_like(table, -1), table)      # pages not given out yet
    s = {"case": c, "K": K, "V": V, "table": table, "lens": ends, "mp": mp}
    slot = torch.arange(mp * page, device=_DEV)
    if c["op"] == "append":
        n = c["new"]
        s["k"] = torch.randn(ns, n, hk, d, generator=g, device=_DEV)
        s["v"] = torch.randn(ns, n, hk, d, generator=g, device=_DEV)
        s["count"] = torch.tensor(_counts(c), device=_DEV, dtype=torch.int32)
        s["bounds"] = _all_bounds(K, table, ends, page)
        s["acc"] = torch.rand(ns, hk, mp * page, generator=g, device=_DEV)
        s["pos"] = slot.to(torch.int32).expand(ns, hk, -1).contiguous()
        s["pos0"] = ends + 11
    elif c["op"] == "attend":
        n = c["new"]
        s["q"] = torch.randn(ns, n, h, d, generator=g, device=_DEV) * 1.5
        s["visible"] = ends + 1
        if c["chosen"]:
            s["sel"] = _some_pages(c, ends, mp, n, g)
        if c["weights"]:
            s["acc"] = torch.rand(ns, hk, mp * page, generator=g, device=_DEV)
    elif c["op"] == "select":
        n = c["new"]
        s["q"] = torch.randn(ns, n, h, d, generator=g, device=_DEV) * 1.5
        s["visible"] = ends + 1
        s["bounds"] = _all_bounds(K, table, ends + n, page)
    else:
        # few keys hold most of the weight
        acc = torch.exp(2.0 * torch.randn(ns, hk, mp * page, generator=g, device=_DEV))
        pos = slot.to(torch.int32).expand(ns, hk, -1) * 2
        s["meta0"] = torch.stack([acc.view(torch.int32), pos])   # weights and positions before the call
        s["meta"] = s["meta0"].clone()
        s["bounds"] = _all_bounds(K, table, ends, page)
    return s


def _all_bounds(K, table, ends, page):
    """Least and largest key of every page in use, over its slots in use: [pool, heads, 2, dim]."""
    pool, hk, _, d = K.shape
    ns, mp = table.shape
    b = torch.zeros(pool, hk, 2, d, device=K.device, dtype=K.dtype)
    for s in range(ns):
        n = -(-int(ends[s]) // page)
        ids = table[s, :n].long()
        inside = torch.arange(n * page, device=K.device).view(n, 1, page, 1) < ends[s]
        k = K[ids]
        b[ids, :, 0] = torch.where(inside, k, torch.full_like(k, math.inf)).amin(2)
        b[ids, :, 1] = torch.where(inside, k, torch.full_like(k, -math.inf)).amax(2)
    return b


def _some_pages(c, ends, mp, n, g):
    """A choice of pages as a selection gives it: ascending, the first and the last among them, -1 behind."""
    ns, hk, m = c["streams"], c["kv_heads"], c["chosen"]
    t = torch.arange(n, device=_DEV)
    have = -(-(ends[:, None] + 1 + t) // c["page"])                       # pages that a token sees
    at = torch.arange(mp, device=_DEV)
    score = torch.rand(ns, n, hk, mp, generator=g, device=_DEV)
    score = torch.where((at == 0) | (at == have[:, :, None, None] - 1), score + 1, score)
    score = torch.where(at < have[:, :, None, None], score, score - 10)
    best = score.topk(min(m, mp), -1)
    ids = torch.where(best.values > -5, best.indices, mp).sort(-1).values
    ids = torch.nn.functional.pad(ids, (0, m - ids.shape[-1]), value=mp)
    return torch.where(ids < mp, ids, -1).to(torch.int32)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "select": _own_select, "evict": _own_evict}[op](s)
    return {"append": _append, "attend": _attend, "select": _select, "evict": _evict}[op](s)


def _cache(s):
    """The library's cache object over the state's pool, made at the first call and kept, as a server keeps it."""
    if "cache" not in s:
        at = os.path.join(os.getcwd(), "gen9-gpu-blas_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import g9kv
        s["cache"] = g9kv.PagedKV(s["K"], s["V"], s["table"], bounds=s.get("bounds"))
    return s["cache"]


def _own_append(s):
    _cache(s).append(s["k"], s["v"], s["lens"], count=s["count"], acc=s["acc"], pos=s["pos"], pos0=s["pos0"])
    return s["K"], s["V"], s["bounds"], s["acc"], s["pos"]


def _own_attend(s):
    c = s["case"]
    out, lse = _cache(s).attend(s["q"], s["visible"], window=c["window"], sel=s.get("sel"), acc=s.get("acc"), lse=True)
    return out, lse, s.get("acc")


def _own_select(s):
    return _cache(s).select(s["q"], s["visible"], s["case"]["chosen"], first=1, last=1)


def _own_evict(s):
    s["meta"].copy_(s["meta0"])
    acc, pos = s["meta"][0].view(torch.float32), s["meta"][1]
    n = _cache(s).evict(s["lens"], s["case"]["keep"], acc, pos, first=_FIRST, recent=_RECENT)
    return n, s["K"], s["V"], acc, pos, s["bounds"]


def _append(s):
    K, V, c = s["K"], s["V"], s["case"]
    page, ns, n = c["page"], c["streams"], c["new"]
    t = torch.arange(n, device=_DEV)
    live = t < s["count"][:, None]
    slot = s["lens"][:, None].long() + t
    st, tt = live.nonzero(as_tuple=True)
    sl = slot[st, tt]
    pg, at = s["table"][st, sl // page].long(), sl % page
    K[pg, :, at] = s["k"][st, tt].half()
    V[pg, :, at] = s["v"][st, tt].half()
    # bounds of the touched pages: anew over the slots in use, which is what they are when kept from the start
    touched = st * s["mp"] + sl // page
    touched = touched.unique()
    u, o = touched // s["mp"], touched % s["mp"]
    ids = s["table"][u, o].long()
    inside = (o[:, None] * page + torch.arange(page, device=_DEV) < (s["lens"] + s["count"])[u][:, None])[:, None, :, None]
    k = K[ids]
    s["bounds"][ids, :, 0] = torch.where(inside, k, torch.full_like(k, math.inf)).amin(2)
    s["bounds"][ids, :, 1] = torch.where(inside, k, torch.full_like(k, -math.inf)).amax(2)
    s["acc"][st, :, sl] = 0.0
    s["pos"][st, :, sl] = (s["pos0"][st] + tt.to(torch.int32))[:, None]
    return K, V, s["bounds"], s["acc"], s["pos"]


def _seen(s, keys):
    """[streams, new, keys]: whether a token sees a slot."""
    c = s["case"]
    vt = s["visible"][:, None] + torch.arange(c["new"], device=_DEV)
    k = torch.arange(keys, device=_DEV)
    seen = k < vt[:, :, None]
    if c.get("window"):
        seen = seen & (k >= vt[:, :, None] - c["window"])
    return seen


def _rows(s, pool):
    """The slots of every stream in order, in 32 bits: [streams, kv heads, slots, dim]."""
    got = pool[s["table"].clamp(min=0).long()]
    ns, mp, hk, page, d = got.shape
    return got.permute(0, 2, 1, 3, 4).reshape(ns, hk, mp * page, d).float()


def _attend(s):
    c, q = s["case"], s["q"]
    ns, n, h, d = q.shape
    hk, page = c["kv_heads"], c["page"]
    grp = h // hk
    if c["chosen"]:
        # the chosen pages of every (token, kv head) alone
        sel = s["sel"].permute(0, 2, 1, 3)                                           # [ns, hk, n, m]
        m = sel.shape[-1]
        ids = torch.gather(s["table"].long()[:, None, None].expand(ns, hk, n, -1), 3, sel.clamp(min=0).long())
        heads = torch.arange(hk, device=_DEV)[None, :, None, None]
        k = s["K"][ids, heads].reshape(ns, hk, n, m * page, d).float()
        v = s["V"][ids, heads].reshape(ns, hk, n, m * page, d).float()
        slot = (sel[..., None].long() * page + torch.arange(page, device=_DEV)).reshape(ns, hk, n, m * page)
        vt = (s["visible"][:, None] + torch.arange(n, device=_DEV))[:, None, :, None]
        seen = ((sel >= 0)[..., None].expand(-1, -1, -1, -1, page).reshape(slot.shape) & (slot < vt))[:, :, :, None]
        qq = q.view(ns, n, hk, grp, d).permute(0, 2, 1, 3, 4)                         # [ns, hk, n, grp, d]
    else:
        k, v = _rows(s, s["K"])[:, :, None], _rows(s, s["V"])[:, :, None]
        seen = _seen(s, k.shape[3])[:, None, :, None].expand(-1, -1, -1, grp, -1).reshape(ns, 1, 1, n * grp, -1)
        qq = q.view(ns, n, hk, grp, d).permute(0, 2, 1, 3, 4).reshape(ns, hk, 1, n * grp, d)
    x = (qq @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    out = (w @ v).reshape(ns, hk, n, grp, d).permute(0, 2, 1, 3, 4).reshape(ns, n, h, d)
    lse = (torch.log(total) + top).reshape(ns, hk, n, grp).permute(0, 2, 1, 3).reshape(ns, n, h)
    if c["weights"]:
        if c["chosen"]:
            per = torch.where(seen, w, torch.zeros_like(w)).sum(3)
            s["acc"].scatter_add_(2, slot.clamp(min=0).reshape(ns, hk, -1), per.reshape(ns, hk, -1))
        else:
            s["acc"] += w.sum((2, 3))
    return out.contiguous(), lse.contiguous(), s.get("acc")


def _select(s):
    c, q = s["case"], s["q"]
    ns, n, h, d = q.shape
    hk, page, m = c["kv_heads"], c["page"], c["chosen"]
    b = s["bounds"][s["table"].clamp(min=0).long()].double()                          # [ns, mp, hk, 2, d]
    lo, hi = (b[:, :, :, i].permute(0, 2, 3, 1)[:, :, None] for i in (0, 1))          # [ns, hk, 1, d, mp]
    qq = q.double().view(ns, n, hk, h // hk, d).permute(0, 2, 1, 3, 4)
    score = (qq.clamp(min=0) @ hi + qq.clamp(max=0) @ lo).amax(3)                     # [ns, hk, n, mp]
    mp = score.shape[-1]
    have = (-(-(s["visible"][:, None] + torch.arange(n, device=_DEV)) // page))[:, None, :, None]
    at = torch.arange(mp, device=_DEV)
    score = torch.where((at < 1) | (at >= have - 1), torch.full_like(score, math.inf), score)
    score = torch.where(at < have, score, torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :m]
    order = torch.where(torch.arange(order.shape[-1], device=_DEV) < have, order, mp).sort(-1).values
    order = torch.nn.functional.pad(order, (0, m - order.shape[-1]), value=mp)
    return torch.where(order < mp, order, -1).to(torch.int32).permute(0, 2, 1, 3).contiguous()


def _evict(s):
    s["meta"].copy_(s["meta0"])
    acc, pos = s["meta"][0].view(torch.float32), s["meta"][1]
    c, K, V, n = s["case"], s["K"], s["V"], s["lens"]
    page, hk, keep, ns = c["page"], c["kv_heads"], c["keep"], c["streams"]
    slots = acc.shape[-1]
    at = torch.arange(slots, device=_DEV)
    used = at < n[:, None, None]
    newest = torch.where(used, pos, torch.full_like(pos, -1)).amax(-1, keepdim=True)
    kept = (pos < _FIRST) | (pos > newest - _RECENT)
    key = torch.where(used, torch.where(kept, torch.full_like(acc, math.inf), acc), torch.full_like(acc, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    stay = torch.zeros_like(used.expand(ns, hk, -1)).scatter_(2, order, True) & used
    stay = torch.where((n > keep)[:, None, None], stay, used)
    room = min(keep, max(1, slots - keep))
    hole = (at < keep) & used & ~stay
    move = (at >= keep) & stay
    far = torch.full_like(at, slots)
    dst = torch.where(hole, at, far).sort(-1).values[..., :room]
    src = torch.where(move, at, far).sort(-1).values[..., :room]
    u, g, j = ((dst < slots) & (src < slots)).nonzero(as_tuple=True)
    dst, src = dst[u, g, j], src[u, g, j]
    dp, sp = s["table"][u, dst // page].long(), s["table"][u, src // page].long()
    K[dp, g, dst % page] = K[sp, g, src % page]
    V[dp, g, dst % page] = V[sp, g, src % page]
    acc[u, g, dst] = acc[u, g, src]
    pos[u, g, dst] = pos[u, g, src]
    left = torch.minimum(n, torch.full_like(n, keep))
    have = -(-left // page)
    mp = s["mp"]
    o = torch.arange(mp, device=_DEV)
    u, o = ((o < have[:, None]) & (n > keep)[:, None]).nonzero(as_tuple=True)
    ids = s["table"][u, o].long()
    inside = (o[:, None] * page + torch.arange(page, device=_DEV) < left[u][:, None])[:, None, :, None]
    k = K[ids]
    s["bounds"][ids, :, 0] = torch.where(inside, k, torch.full_like(k, math.inf)).amin(2)
    s["bounds"][ids, :, 1] = torch.where(inside, k, torch.full_like(k, -math.inf)).amax(2)
    return left, K, V, acc, pos, s["bounds"]


# ------------------------------------------------------------------------------------------------ work and exact values
def work(case):
    c = case
    ns, hk, d, page, h = c["streams"], c["kv_heads"], c["dim"], c["page"], c["heads"]
    lens = _lengths(c)
    row = hk * d
    if c["op"] == "append":
        counts = _counts(c)
        touched = sum((n + k - 1) // page - n // page + 1 for n, k in zip(lens, counts))
        new = sum(counts)
        return {"bytes": new * row * 2 * (4 + 2) + touched * row * 2 * 2 * 2 + new * hk * 8, "flops": 2 * new * row}
    if c["op"] == "attend":
        seen = pairs = 0
        for n in lens:
            for t in range(c["new"]):
                vt = n + 1 + t
                k = vt
                if c["chosen"]:
                    have = -(-vt // page)
                    k = vt if have <= c["chosen"] else (c["chosen"] - 1) * page + (vt - 1) % page + 1
                elif c["window"]:
                    k = min(vt, c["window"])
                pairs += k
                if c["chosen"]:
                    seen += k                      # every token chooses its own pages
            if not c["chosen"]:
                last = n + c["new"]
                seen += min(last, c["window"] + c["new"] - 1) if c["window"] else last
        q = ns * c["new"] * h * d * 4
        return {"bytes": seen * row * 2 * 2 + 2 * q + (seen * hk * 8 if c["weights"] else 0), "flops": 4 * pairs * h * d}
    if c["op"] == "select":
        pages = sum(-(-(n + c["new"]) // page) for n in lens)
        per = sum(-(-(n + 1 + t) // page) for n in lens for t in range(c["new"]))
        return {"bytes": pages * row * 2 * 2 + ns * c["new"] * (h * d * 4 + hk * c["chosen"] * 4), "flops": 2 * per * h * d}
    keep, total = c["keep"], 0
    for n in lens:
        over = max(0, n - keep)
        moved = keep * over / n
        changed = page * (keep / page) * (1 - (1 - over / n) ** page)      # slots of pages that get another row
        total += n * 8 + moved * (d * 8 + 16) + (changed * d * 2 + changed / page * d * 4 if over else 0)
    return {"bytes": hk * total, "flops": 0}


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    ns, hk, d, page, h = c["streams"], c["kv_heads"], c["dim"], c["page"], c["heads"]
    lens = _lengths(c)
    K, V, table = s["K"], s["V"], s["table"]
    if c["op"] == "append":
        for u, (n, cnt) in enumerate(zip(lens, _counts(c))):
            for o in range(n // page, (n + cnt - 1) // page + 1):
                p, a, b = int(table[u, o]), max(n, o * page), min(n + cnt, (o + 1) * page)
                K[p, :, a - o * page:b - o * page] = s["k"][u, a - n:b - n].transpose(0, 1).to(torch.float16)
                V[p, :, a - o * page:b - o * page] = s["v"][u, a - n:b - n].transpose(0, 1).to(torch.float16)
                s["bounds"][p, :, 0] = K[p, :, :b - o * page].amin(1)
                s["bounds"][p, :, 1] = K[p, :, :b - o * page].amax(1)
            s["acc"][u, :, n:n + cnt] = 0
            s["pos"][u, :, n:n + cnt] = torch.arange(cnt, device=_DEV, dtype=torch.int32) + n + 11
        return K.double(), V.double(), s["bounds"].double(), s["acc"].double(), None
    if c["op"] == "attend":
        new, grp = c["new"], h // hk
        out = torch.zeros(ns, new, h, d, device=_DEV, dtype=torch.float64)
        lse = torch.full((ns, new, h), -math.inf, device=_DEV, dtype=torch.float64)
        acc = s["acc"].double() if c["weights"] else None
        sel = s["sel"].tolist() if c["chosen"] else None
        if c["chosen"] and ns * new * hk > 2000:
            return None
        for u in range(ns):
            pages = -(-(lens[u] + new) // page)
            for g in range(hk):
                ids = table[u, :pages].long()
                k64 = K[ids, g].double().reshape(-1, d)
                v64 = V[ids, g].double().reshape(-1, d)
                for t in range(new):
                    vt = lens[u] + 1 + t
                    at = torch.arange(max(0, vt - c["window"]) if c["window"] else 0, vt, device=_DEV)
                    if sel:
                        mine = torch.tensor([o for o in sel[u][t][g] if o >= 0], device=_DEV)
                        at = (mine[:, None] * page + torch.arange(page, device=_DEV)).reshape(-1)
                        at = at[at < vt]
                    if not len(at):
                        continue
                    x = s["q"][u, t, g * grp:(g + 1) * grp].double() @ k64[at].T / math.sqrt(d)
                    p = torch.softmax(x, -1)
                    out[u, t, g * grp:(g + 1) * grp] = p @ v64[at]
                    lse[u, t, g * grp:(g + 1) * grp] = torch.logsumexp(x, -1)
                    if acc is not None:
                        acc[u, g, at] += p.sum(0)
        return out, lse, acc
    if c["op"] == "select":
        return None            # whole numbers only
    if ns * hk > 600:
        return None
    acc, pos = s["meta0"][0].view(torch.float32).clone(), s["meta0"][1].clone()
    keep = c["keep"]
    for u, n in enumerate(lens):
        if n <= keep:
            continue
        for g in range(hk):
            a, p = acc[u, g, :n].double(), pos[u, g, :n]
            sure = (p < _FIRST) | (p > p.max() - _RECENT)
            rank = torch.where(sure, a + 1e30, a)
            best = torch.topk(rank, keep).indices
            stays = torch.zeros(n, dtype=torch.bool, device=_DEV)
            stays[best] = True
            holes = torch.nonzero(~stays[:keep]).flatten()
            movers = torch.nonzero(stays[keep:]).flatten() + keep
            to, come = table[u, holes // page].long(), table[u, movers // page].long()
            K[to, g, holes % page] = K[come, g, movers % page]
            V[to, g, holes % page] = V[come, g, movers % page]
            acc[u, g, holes] = acc[u, g, movers]
            pos[u, g, holes] = pos[u, g, movers]
        kept = [int(x) for x in table[u, :-(-keep // page)].tolist()]
        whole = torch.tensor(kept[:keep // page], device=_DEV, dtype=torch.long)
        s["bounds"][whole, :, 0], s["bounds"][whole, :, 1] = K[whole].amin(2), K[whole].amax(2)
        if keep % page:
            s["bounds"][kept[-1], :, 0] = K[kept[-1], :, :keep % page].amin(1)
            s["bounds"][kept[-1], :, 1] = K[kept[-1], :, :keep % page].amax(1)
    return None, K.double(), V.double(), acc.double(), None, s["bounds"].double()

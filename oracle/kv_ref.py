"""Plain 64-bit NumPy forms of the paged key-value cache operators (include/gen9blas_kv.h): test infrastructure.

A cache is a dict: K, V float16 [pages, heads, page, D], bounds float16 [pages, heads, 2, D] or None, table int32
[streams, mp]. Slots are walked one by one from the definitions; nothing here shares code with the library."""
import numpy as np


def place_of(cache, s, k):
    """(page, slot in it) of slot k of stream s, or None."""
    page = cache["K"].shape[2]
    if k < 0 or k // page >= cache["table"].shape[1]:
        return None
    p = int(cache["table"][s, k // page])
    return (p, k % page) if 0 <= p < cache["K"].shape[0] else None


def seen(cache, vis, step, t):
    return int(min(max(int(vis) + step * t, 0), cache["table"].shape[1] * cache["K"].shape[2]))


def visible_slots(cache, s, vis, step, t, window=0, sel=None):
    """Slots that token t of stream s sees, in order; sel: the list of places for one (token, head)."""
    n, page = seen(cache, vis, step, t), cache["K"].shape[2]
    if sel is None:
        ks = range(max(0, n - window) if window else 0, n)
    else:
        ks, top = [], -1
        for e in sel:
            if top < e < cache["table"].shape[1]:       # above every earlier one that counts: each page once
                ks += [k for k in range(e * page, (e + 1) * page) if k < n]
                top = e
    return [k for k in ks if place_of(cache, s, k) is not None]


def attend(cache, q, vis, step=1, scale=None, window=0, sel=None):
    """(O, lse, weights [s, heads, slots], spread): spread[s, t, h] bounds sum_d |q_d k_d| · scale over the seen keys and
    mass[s, t, h, d] = sum_k w_k |v_kd|, for error bounds."""
    K, V = cache["K"].astype(np.float64), cache["V"].astype(np.float64)
    ns, nq, H, D = q.shape
    hkv = K.shape[1]
    slots = cache["table"].shape[1] * K.shape[2]
    scale = D ** -0.5 if scale is None else scale
    O = np.zeros(q.shape)
    lse = np.full((ns, nq, H), -np.inf)
    W = np.zeros((ns, hkv, slots))
    spread, mass = np.zeros((ns, nq, H)), np.zeros(q.shape)
    for s in range(ns):
        for t in range(nq):
            for g in range(hkv):
                ks = visible_slots(cache, s, vis[s], step, t, window, None if sel is None else sel[s, t, g])
                if not ks:
                    continue
                at = [place_of(cache, s, k) for k in ks]
                k64 = np.stack([K[p, g, i] for p, i in at])
                v64 = np.stack([V[p, g, i] for p, i in at])
                for h in range(g * (H // hkv), (g + 1) * (H // hkv)):
                    qd = q[s, t, h].astype(np.float64)
                    x = k64 @ qd * scale
                    top = x.max()
                    e = np.exp(x - top)
                    w = e / e.sum()
                    O[s, t, h] = w @ v64
                    lse[s, t, h] = top + np.log(e.sum())
                    W[s, g, ks] += w
                    spread[s, t, h] = (np.abs(k64) @ np.abs(qd)).max() * abs(scale)
                    mass[s, t, h] = w @ np.abs(v64)
    return O, lse, W, spread, mass


def select(cache, q, vis, nsel, step=1, first=1, last=1):
    ns, nq, H, D = q.shape
    page, mp = cache["K"].shape[2], cache["table"].shape[1]
    hkv = cache["K"].shape[1]
    out = np.full((ns, nq, hkv, nsel), -1, np.int32)
    for s in range(ns):
        for t in range(nq):
            have = -(-seen(cache, vis[s], step, t) // page)
            for g in range(hkv):
                rank = []
                for o in range(have):
                    p = int(cache["table"][s, o])
                    if o < first or o >= have - last:
                        key = (2, 0.0)
                    elif not 0 <= p < cache["K"].shape[0]:
                        key = (0, 0.0)
                    else:
                        lo, hi = cache["bounds"][p, g].astype(np.float64)
                        sc = []
                        for h in range(g * (H // hkv), (g + 1) * (H // hkv)):
                            qd = q[s, t, h].astype(np.float64)
                            sc.append(float(np.sum(np.maximum(qd * lo, qd * hi))))
                        key = (0, 0.0) if any(np.isnan(sc)) else (1, max(sc))
                    rank.append((-key[0], -key[1], o))
                best = sorted(o for _, _, o in sorted(rank)[:nsel])
                out[s, t, g, :len(best)] = best
    return out


def _bounds_of(rows):
    return np.stack([rows.min(0), rows.max(0)])


def append(cache, k, v, length, count=None, acc=None, pos=None, pos0=None):
    """In place; returns whether every token found a page."""
    ns, nt, hkv, D = k.shape
    fine = True
    for s in range(ns):
        n = max(int(length[s]), 0)
        for t in range(nt if count is None else min(max(int(count[s]), 0), nt)):
            at = place_of(cache, s, n + t)
            if at is None:
                fine = False
                continue
            p, i = at
            for g in range(hkv):
                with np.errstate(over="ignore"):
                    cache["K"][p, g, i] = k[s, t, g].astype(np.float16)
                    cache["V"][p, g, i] = v[s, t, g].astype(np.float16)
                if cache["bounds"] is not None:
                    row = cache["K"][p, g, i]
                    b = cache["bounds"][p, g]
                    cache["bounds"][p, g] = np.stack([row, row]) if i == 0 else np.stack([np.minimum(b[0], row),
                                                                                             np.maximum(b[1], row)])
                if acc is not None:
                    acc[s, g, n + t] = 0
                if pos is not None:
                    pos[s, g, n + t] = t + (n if pos0 is None else int(pos0[s]))
    return fine


def evict(cache, length, keep, acc, pos=None, first=0, recent=0):
    """In place; returns the new lengths."""
    ns, page, hkv = cache["table"].shape[0], cache["K"].shape[2], cache["K"].shape[1]
    cap = cache["table"].shape[1] * page
    out = np.zeros(ns, np.int32)
    for s in range(ns):
        n = min(max(int(length[s]), 0), cap)
        out[s] = min(n, keep)
        if n <= keep:
            continue
        for g in range(hkv):
            at = np.arange(n) if pos is None else pos[s, g, :n].astype(np.int64)
            sure = (at < first) | (at > at.max() - recent)
            w = acc[s, g, :n].astype(np.float64)
            rank = sorted(range(n), key=lambda k: (0, 0.0, k) if sure[k] else (2, 0.0, k) if np.isnan(w[k]) else (1, -w[k], k))
            stay = set(rank[:keep])
            holes = [k for k in range(keep) if k not in stay]
            movers = [k for k in range(keep, n) if k in stay]
            assert len(holes) == len(movers)
            for a, b in zip(holes, movers):
                to, come = place_of(cache, s, a), place_of(cache, s, b)
                if to is not None and come is not None:
                    cache["K"][to[0], g, to[1]] = cache["K"][come[0], g, come[1]]
                    cache["V"][to[0], g, to[1]] = cache["V"][come[0], g, come[1]]
                acc[s, g, a] = acc[s, g, b]
                if pos is not None:
                    pos[s, g, a] = pos[s, g, b]
            if cache["bounds"] is not None:
                for o in range(-(-keep // page)):
                    rows = min(page, keep - o * page)
                    p = place_of(cache, s, o * page)
                    if p is not None and (rows < page or any(o * page <= k < o * page + rows for k in holes)):
                        cache["bounds"][p[0], g] = _bounds_of(cache["K"][p[0], g, :rows])
    return out

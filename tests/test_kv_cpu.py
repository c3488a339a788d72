"""CPU checks of the paged key-value cache: the index arithmetic of csrc/kv_index.h through a host build (pages outside
the pool, lengths past the table, offsets past 32 bits, the division by the page size, the split of the steps), the
refusals of the C entry points that need no GPU, and the 64-bit reference forms of oracle/kv_ref.py on small caches."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import PKG, ROOT

sys.path.insert(0, os.path.join(ROOT, "oracle"))
import kv_ref  # noqa: E402

INT_MAX = 2 ** 31 - 1


@pytest.fixture(scope="module")
def idx(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv") / "kv_index.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", os.path.join(PKG, "csrc"),
                    os.path.join(ROOT, "tests", "kv_index_host.cpp"), "-o", so], check=True)
    d = ctypes.CDLL(so)
    i, l, p = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
    for name, args, res in (("kv_quot", [i, i], i), ("kv_quot_wrong", [i, l, l, l], l), ("kv_seen", [i] * 4, i),
                            ("kv_first", [i, i], i), ("kv_page", [p, l, i, i, i, i], i), ("kv_row", [i, i, i, l, l, l], l),
                            ("kv_wkey", [ctypes.c_float], ctypes.c_uint32), ("kv_skey", [ctypes.c_double], ctypes.c_uint64)):
        f = getattr(d, name)
        f.argtypes, f.restype = args, res
    return d


@pytest.mark.parametrize("page", [1, 2, 3, 5, 7, 8, 16, 24, 31, 100, 255, 1000, 4096, 65535, 2 ** 20 + 7, 2 ** 30, INT_MAX - 64])
def test_page_quotient(idx, page):
    assert idx.kv_quot_wrong(page, 0, 20000, 1) == 0
    assert idx.kv_quot_wrong(page, INT_MAX - 20000, 20001, 1) == 0
    assert idx.kv_quot_wrong(page, 0, 100000, 21473) == 0
    for m in (1, 2, 1000, INT_MAX // page):          # at and beside multiples of the page
        assert idx.kv_quot_wrong(page, m * page - 2, 5, 1) == 0


def test_seen_slots_are_held_to_the_table(idx):
    assert idx.kv_seen(5, 1, 3, 100) == 8
    assert idx.kv_seen(-7, 1, 3, 100) == 0
    assert idx.kv_seen(INT_MAX, INT_MAX, INT_MAX, 100) == 100
    assert idx.kv_seen(-INT_MAX, 0, 0, 100) == 0
    assert idx.kv_first(10, 0) == 0 and idx.kv_first(10, 3) == 7 and idx.kv_first(10, 11) == 0


def test_pages_outside_the_pool_are_none(idx):
    table = np.array([[0, 4, -1, 5, 2147483647, -2147483648]], np.int32)
    got = [idx.kv_page(table.ctypes.data, 6, 0, o, 6, 5) for o in range(-1, 8)]
    assert got == [-1, 0, 4, -1, -1, -1, -1, -1, -1]


def test_row_offsets_pass_32_bits(idx):
    assert idx.kv_row(3_000_000, 15, 7, 16 * 8 * 128, 128, 16 * 128) == 3_000_000 * 16 * 8 * 128 + 15 * 128 + 7 * 16 * 128
    assert idx.kv_row(INT_MAX, 0, 0, 2 ** 20, 0, 0) == INT_MAX * 2 ** 20


def test_keys_keep_the_order(idx):
    w = [-np.inf, -3e38, -1.5, -1e-45, 0.0, 1e-45, 1e-3, 1.0, 1.0000001, 3e38, np.inf]
    keys = [idx.kv_wkey(x) for x in w]
    assert keys == sorted(keys) and len(set(keys)) == len(keys) and 0 < keys[0] and keys[-1] < 0xFFFFFFFF
    assert idx.kv_wkey(-0.0) == idx.kv_wkey(0.0) and idx.kv_wkey(np.nan) == 0 == idx.kv_wkey(-np.nan)
    x = [-np.inf, -1e308, -1.0, -5e-324, 0.0, 5e-324, 1.0, 1.0000000000000002, 1e308, np.inf]
    keys = [idx.kv_skey(v) for v in x]
    assert keys == sorted(keys) and len(set(keys)) == len(keys) and 0 < keys[0] and keys[-1] < 2 ** 64 - 1
    assert idx.kv_skey(-0.0) == idx.kv_skey(0.0) and idx.kv_skey(np.nan) == 0


# ------------------------------------------------------------------------------------------------ refusals, no GPU
@pytest.fixture(scope="module")
def kv():
    import g9kv
    return g9kv


def _cache(kv, buf, **over):
    """A description of a sound cache of 4 pages over host memory (refusals come before any operand is looked at)."""
    base = (ctypes.addressof(buf) + 63) // 64 * 64
    f = dict(D=64, HKV=2, page=8, n_pages=4, K=base, kp=1024, kk=64, kh=512, k_bytes=8192, V=base + 8192, vp=1024, vk=64,
             vh=512, v_bytes=8192, bounds=base + 16384, table=base + 32768, ts=4, mp=4, ns=2)
    f.update(over)
    return kv._Cache(**f)


@pytest.mark.parametrize("over,status", [
    (dict(D=60), 1), (dict(D=264), 1), (dict(D=0), 1), (dict(HKV=0), 1), (dict(HKV=3), 1),
    (dict(page=0), -3), (dict(n_pages=-1), -3), (dict(mp=-1), -3), (dict(ns=-1), -3), (dict(ts=-1), -3),
    (dict(kk=60), -3), (dict(vp=-1024), -3), (dict(K=None), -3), (dict(V=None), -3), (dict(k_bytes=8190), -3),
    (dict(v_bytes=0), -3), (dict(table=None), -3), (dict(mp=2 ** 30, page=4), -3), (dict(ns=2 ** 30, HKV=4, kh=0, vh=0), -3),
    (dict(kp=2 ** 62), -3), (dict(), -5)])
def test_caches_that_are_refused(kv, over, status):
    if kv._fn["init"]() == 0:
        pytest.skip("a GPU is present: host memory would be refused for another reason")
    buf = ctypes.create_string_buffer(40000)
    c = _cache(kv, buf, **over)
    q = ctypes.addressof(buf)
    got = kv._fn["attn_paged"](c, 4, 1, q, 256, 64, 256, q, 1, 0, None, 0, 1.0, q, None, None, 0, 0, None, 0)
    assert got == status, kv._fn["error"]()
    if status == -3:
        assert kv._fn["error"]()


def test_arguments_that_are_refused(kv):
    buf = ctypes.create_string_buffer(40000)
    c, q = _cache(kv, buf), ctypes.addressof(buf)
    attn = kv._fn["attn_paged"]
    assert attn(None, 4, 1, q, 256, 64, 256, q, 1, 0, None, 0, 1.0, q, None, None, 0, 0, None, 0) == -3
    assert attn(c, 0, 1, q, 256, 64, 256, q, 1, 0, None, 0, 1.0, q, None, None, 0, 0, None, 0) == 1
    assert attn(c, 3, 1, q, 256, 64, 256, q, 1, 0, None, 0, 1.0, q, None, None, 0, 0, None, 0) == 1     # not a multiple of 2
    assert attn(c, 4, 1, q, 256, 64, 256, q, -1, 0, None, 0, 1.0, q, None, None, 0, 0, None, 0) == -3   # step
    assert attn(c, 4, 1, q, 256, 64, 256, q, 1, -2, None, 0, 1.0, q, None, None, 0, 0, None, 0) == -3   # window
    assert attn(c, 4, 1, q, 256, 64, 256, q, 1, 5, q, 2, 1.0, q, None, None, 0, 0, None, 0) == -3       # window and sel
    assert attn(c, 4, 1, q, 256, 64, 256, q, 1, 0, q, -1, 1.0, q, None, None, 0, 0, None, 0) == -3      # nsel
    assert attn(c, 4, 1, q, 256, 64, 256, q, 1, 0, q, 2 ** 29, 1.0, q, None, None, 0, 0, None, 0) == -3
    select = kv._fn["kv_select"]
    assert select(c, 4, 1, q, 256, 64, 256, q, 1, -1, 0, 4, q, None, 0) == -3
    assert select(c, 4, 1, q, 256, 64, 256, q, 1, 0, 0, -4, q, None, 0) == -3
    assert select(_cache(kv, buf, bounds=None), 4, 1, q, 256, 64, 256, q, 1, 0, 0, 4, q, None, 0) == -3
    evict = kv._fn["kv_evict"]
    assert evict(c, q, 0, 0, 0, q, None, 0, 0, q, None, 0) == -3
    assert evict(c, q, 8, 5, 4, q, None, 0, 0, q, None, 0) == -3
    assert kv._fn["kv_append"](_cache(kv, buf, K=c.K + 2), 1, q, 1, 1, 1, q, 1, 1, 1, q, None, None, None, 0, 0, None, 0,
                               None) == -3
    assert kv._fn["kv_supported"](128, 32, 8) == 1 and kv._fn["kv_supported"](128, 32, 5) == 0


def test_what_a_call_writes_must_not_overlap_itself(kv):
    """Broadcast rows (stride 0) or rows closer than their length, of the pool, acc or pos, where a call writes them."""
    buf = ctypes.create_string_buffer(40000)
    c, q = _cache(kv, buf), ctypes.addressof(buf)
    append, evict, attn = kv._fn["kv_append"], kv._fn["kv_evict"], kv._fn["attn_paged"]
    tokens = (1, q, 64, 64, 64, q, 64, 64, 64, q, None)
    for over in (dict(kp=0), dict(kh=0), dict(kk=56), dict(vh=0), dict(vp=32), dict(vk=0)):
        bad = _cache(kv, buf, **over)
        assert append(bad, *tokens, None, None, 0, 0, None, 0, None) == -3 and b"overlap" in kv._fn["error"]()
        assert evict(bad, q, 8, 0, 0, q, None, 64, 32, q, None, 0) == -3 and b"overlap" in kv._fn["error"]()
    for ms, mh in ((0, 32), (31, 32), (64, 0), (64, 31)):
        assert append(c, *tokens, q, None, ms, mh, None, 0, None) == -3 and b"overlap" in kv._fn["error"]()
        assert append(c, *tokens, None, q, ms, mh, None, 0, None) == -3 and b"overlap" in kv._fn["error"]()
        assert evict(c, q, 8, 0, 0, q, None, ms, mh, q, None, 0) == -3 and b"overlap" in kv._fn["error"]()
        assert attn(c, 4, 1, q, 256, 64, 256, q, 1, 0, None, 0, 1.0, q, None, q, ms, mh, None, 0) == -3 and b"overlap" in kv._fn["error"]()


def test_strides_that_are_long_enough_each_but_overlap_together(kv):
    """Rows of one dimension lie apart, but some of two dimensions are the same; layouts whose strides nest are not refused."""
    buf = ctypes.create_string_buffer(40000)
    c, q = _cache(kv, buf), ctypes.addressof(buf)
    append, evict, attn = kv._fn["kv_append"], kv._fn["kv_evict"], kv._fn["attn_paged"]
    tokens = (1, q, 64, 64, 64, q, 64, 64, 64, q, None)

    def overlap(status):
        return status == -3 and b"overlap" in kv._fn["error"]()
    for over in (dict(kp=64), dict(kk=64, kh=64), dict(vp=512), dict(vh=64), dict(kp=1016), dict(vp=64, vk=256, vh=128)):
        bad = _cache(kv, buf, **over)
        assert overlap(append(bad, *tokens, None, None, 0, 0, None, 0, None)), over
        assert overlap(evict(bad, q, 8, 0, 0, q, None, 64, 32, q, None, 0)), over
    for over in (dict(kk=128, kh=64), dict(kp=64, kk=256, kh=2048), dict(vk=72, vh=576, vp=1152, v_bytes=16384), dict(kp=0, n_pages=1)):
        assert not overlap(append(_cache(kv, buf, **{**dict(k_bytes=16384, v_bytes=16384), **over}), *tokens, None, None, 0, 0, None, 0,
                                  None)), over
    for ms, mh in ((32, 32), (63, 32), (32, 63), (48, 40)):
        assert overlap(append(c, *tokens, q, None, ms, mh, None, 0, None))
        assert overlap(append(c, *tokens, None, q, ms, mh, None, 0, None))
        assert overlap(evict(c, q, 8, 0, 0, q, None, ms, mh, q, None, 0))
        assert overlap(attn(c, 4, 1, q, 256, 64, 256, q, 1, 0, None, 0, 1.0, q, None, q, ms, mh, None, 0))
    for ms, mh in ((64, 32), (32, 64), (100, 40), (33, 70)):
        assert not overlap(append(c, *tokens, q, None, ms, mh, None, 0, None))
    one = _cache(kv, buf, ns=1)
    assert not overlap(append(one, *tokens, q, None, 0, 32, None, 0, None)) and overlap(append(one, *tokens, q, None, 0, 31, None, 0, None))


def test_python_face_checks_types(kv):
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="float16"):
        kv.PagedKV(torch.zeros(2, 1, 4, 8), torch.zeros(2, 1, 4, 8), torch.zeros(1, 1, dtype=torch.int32))


# ------------------------------------------------------------------------------------------------ the reference forms
def test_reference_attention_of_one_slot_returns_its_value():
    rng = np.random.default_rng(3)
    K = rng.standard_normal((3, 1, 4, 8)).astype(np.float16)
    cache = {"K": K, "V": (2 * K).astype(np.float16), "bounds": None, "table": np.array([[2, -1], [1, 7]], np.int32)}
    q = rng.standard_normal((2, 2, 2, 8)).astype(np.float32)
    O, lse, W, _, _ = kv_ref.attend(cache, q, [1, 0])
    assert np.array_equal(O[0, 0, 0], cache["V"][2, 0, 0].astype(np.float64))
    assert np.all(O[1, 0] == 0) and np.all(lse[1, 0] == -np.inf)
    assert np.allclose(O[1, 1, 0], cache["V"][1, 0, 0]) and np.isclose(W[0].sum(), 4)
    # pages that are missing hide their slots
    assert kv_ref.visible_slots(cache, 0, 8, 1, 0) == [0, 1, 2, 3] == kv_ref.visible_slots(cache, 1, 8, 1, 0)
    assert kv_ref.visible_slots(cache, 0, 3, 1, 0, window=2) == [1, 2]
    assert kv_ref.visible_slots(cache, 0, 8, 1, 0, sel=[0, 0, -1]) == [0, 1, 2, 3]


def test_reference_lists_count_a_page_once():
    cache = {"K": np.zeros((9, 1, 2, 8), np.float16), "table": np.arange(8, dtype=np.int32)[None]}

    def places(sel):
        ks = kv_ref.visible_slots(cache, 0, 16, 1, 0, sel=sel)
        assert ks == sorted(set(ks)) and len(ks) % 2 == 0
        return [k // 2 for k in ks[::2]]
    assert places([3, -1, 3]) == [3] and places([5, 2, 5]) == [5] and places([5, 3, 4, 5, 6]) == [5, 6]
    assert places([8, 3, 2 ** 31 - 1, 4, -2 ** 31, 4, 7]) == [3, 4, 7] and places([-1, 0, 0, 1]) == [0, 1] and places([]) == []


def test_reference_eviction_keeps_the_heaviest():
    cache = {"K": np.arange(24, dtype=np.float16).reshape(3, 1, 8, 1).repeat(8, 3), "table": np.array([[2, 0]], np.int32)}
    cache["V"] = -cache["K"]
    cache["bounds"] = np.zeros((3, 1, 2, 8), np.float16)
    acc = np.array([[[1, 9, 2, 8, 3, 7, 4, 6, 5, 9.5, 0, 0, 0, 0, 0, 0]]], np.float32)
    pos = np.arange(16, dtype=np.int32).reshape(1, 1, 16)
    n = kv_ref.evict(cache, [12], 4, acc, pos, first=1, recent=1)
    assert list(n) == [4] and list(pos[0, 0, :4]) == [0, 1, 9, 11]
    assert list(cache["K"][2, 0, :4, 0]) == [16, 17, 1, 3]
    assert list(cache["bounds"][2, 0, :, 0]) == [1, 17]

"""CPU checks of the ledger of queued writes (csrc/ledger.h) through a host build with scripted streams: which ranges may still be
written, what a full ledger answers, and that it opens again."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import PKG, ROOT


@pytest.fixture(scope="module")
def dll(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("ledger") / "ledger.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", os.path.join(PKG, "csrc"),
                    os.path.join(ROOT, "tests", "ledger_host.cpp"), "-o", so], check=True)
    d = ctypes.CDLL(so)
    d.led_overlap.argtypes = [ctypes.c_uint64, ctypes.c_uint64]
    d.led_end.argtypes = [ctypes.c_int, ctypes.c_long]
    d.led_open.restype = ctypes.c_long
    return d


@pytest.fixture
def led(dll):
    dll.led_new(64)

    class Led:
        end, clear, overlap = staticmethod(dll.led_end), staticmethod(dll.led_clear), staticmethod(lambda lo, n=8: bool(dll.led_overlap(lo, n)))
        waits, open, can_record = staticmethod(dll.led_waits), staticmethod(dll.led_open), staticmethod(dll.led_can_record)
        ranges, lost = dll.led_ranges(), dll.led_lost()

        @staticmethod
        def call(st, *ranges):
            lo = (ctypes.c_uint64 * len(ranges))(*[r[0] for r in ranges])
            n = (ctypes.c_uint64 * len(ranges))(*[r[1] for r in ranges])
            dll.led_call(st, len(ranges), lo, n)
    return Led


def test_a_range_is_held_until_its_call_has_ended(led):
    led.call(0, (1000, 100), (5000, 10), (0, 7), (9000, 0))
    assert led.overlap(1000) and led.overlap(1092, 8) and led.overlap(990, 11) and led.overlap(5009, 1)
    assert not led.overlap(1100) and not led.overlap(990, 10) and not led.overlap(0, 8) and not led.overlap(9000)
    led.end(0, 1)
    assert not led.overlap(1000, 10000)


def test_waiting_for_a_stream_forgets_its_writes_only(led):
    led.call(0, (1000, 100))
    led.call(1, (1000, 100), (3000, 10))
    led.clear(0)
    assert led.overlap(1050) and led.overlap(3000)
    led.clear(1)
    assert not led.overlap(0, 10 ** 6)


def test_a_later_call_of_the_range_is_waited_for(led):
    led.call(0, (1000, 100))
    led.call(0, (1050, 100))
    led.end(0, 1)
    assert led.overlap(1000)          # one entry, up to the second call
    led.end(0, 1)
    assert not led.overlap(1000)


@pytest.mark.parametrize("wait", ["events", "streams"])
def test_a_ledger_that_two_streams_overflowed_opens_again(led, wait):
    for i in range(led.ranges):
        led.call(0, (10 ** 6 * (i + 1), 10))
    led.call(1, (7, 1))
    led.call(2, (9, 1))
    led.call(2, (11, 1))
    assert led.overlap(3) and led.waits() == 0      # any range may be one of those without an entry
    for st in (1, 2):
        assert led.overlap(3)
        led.clear(st) if wait == "streams" else led.end(st, led.open(st))
    assert not led.overlap(3) and led.overlap(10 ** 6)
    led.clear(0)
    assert not led.overlap(0, 10 ** 9)
    led.call(1, (500, 10))                          # and works as before
    assert led.overlap(505, 1) and not led.overlap(400)


def test_the_overflow_of_a_stream_that_is_never_waited_for_ends_with_its_work(led):
    for i in range(led.ranges):
        led.call(0, (10 ** 6 * (i + 1), 10))
    led.call(1, (7, 1))
    led.call(1, (9, 1))
    led.end(1, 1)
    assert led.overlap(3)
    led.end(1, 1)
    assert not led.overlap(3)


def test_more_overflowing_streams_than_are_kept_are_waited_for(led):
    for i in range(led.ranges):
        led.call(0, (10 ** 6 * (i + 1), 10))
    for st in range(1, led.lost + 1):
        led.call(st, (100 * st, 1))
    assert led.waits() == 0
    led.call(led.lost + 1, (3, 1))
    assert led.waits() == 1 and led.open(led.lost + 1) == 0
    led.end(1, 1)
    led.call(led.lost + 2, (3, 1))                  # the room of the stream whose work has ended
    assert led.waits() == 1
    for st in range(led.lost + 3):
        led.end(st, led.open(st))
    assert not led.overlap(0, 10 ** 9)


def test_where_no_event_can_be_recorded_the_call_is_waited_for(led):
    led.can_record(0)
    led.call(0, (1000, 100))
    assert led.waits() == 1 and not led.overlap(1000)
    led.can_record(1)
    led.call(0, (1000, 100))
    assert led.waits() == 1 and led.overlap(1000)


def test_a_full_ledger_widens_entries_of_the_same_stream(led):
    for i in range(led.ranges):
        led.call(0, (1000 * (i + 1), 10))
    led.call(0, (500, 10))
    assert led.waits() == 0 and led.overlap(500) and led.overlap(700) and not led.overlap(100)
    led.end(0, 10 ** 6)
    assert not led.overlap(0, 10 ** 9)


def test_random_calls_never_miss_an_open_write(led):
    """Against every write kept by itself: a range with an open write is never called free, and all is free in the end."""
    rng = random.Random(5)
    open_ = [[] for _ in range(64)]
    for step in range(6000):
        st = rng.randrange(rng.choice([2, 8, 40]))
        what = rng.random()
        if what < 0.55:
            ranges = [(rng.randrange(1, 10 ** 5), rng.randrange(1, 300)) for _ in range(rng.randrange(1, 5))]
            led.call(st, *ranges)
            open_[st].append(ranges)
        elif what < 0.75 and open_[st]:
            led.end(st, 1)
            open_[st].pop(0)
        elif what < 0.78:
            led.clear(st)
            open_[st].clear()
        for x in range(64):                          # the ledger may have waited for a stream
            del open_[x][:len(open_[x]) - led.open(x)]
        lo, n = rng.randrange(1, 10 ** 5), rng.randrange(1, 300)
        if any(a < lo + n and lo < a + b for calls in open_ for ranges in calls for a, b in ranges):
            assert led.overlap(lo, n), step
    for x in range(64):
        led.end(x, led.open(x))
    assert not led.overlap(0, 10 ** 9)


# ------------------------------------------------------------------------------------------------ captured calls
@pytest.fixture
def cap(dll):
    dll.cap_new()
    dll.cap_call.argtypes = [ctypes.c_uint64, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    dll.cap_overlap.argtypes = [ctypes.c_uint64] * 3

    class Cap:
        captures, ranges = dll.cap_captures(), dll.cap_ranges()

        @staticmethod
        def call(capture, *ranges):
            lo = (ctypes.c_uint64 * len(ranges))(*[r[0] for r in ranges])
            n = (ctypes.c_uint64 * len(ranges))(*[r[1] for r in ranges])
            dll.cap_call(capture, len(ranges), lo, n)

        @staticmethod
        def overlap(capture, lo, n=8):
            return bool(dll.cap_overlap(lo, n, capture))
    return Cap


def test_a_captured_write_counts_in_its_capture_alone(cap):
    cap.call(7, (1000, 100), (5000, 10), (0, 9), (8000, 0))
    assert cap.overlap(7, 1092) and cap.overlap(7, 5000) and not cap.overlap(7, 1100) and not cap.overlap(7, 8000)
    assert not cap.overlap(8, 1000)             # another graph's calls read early, whatever this one wrote
    cap.call(8, (3000, 10))
    assert cap.overlap(8, 3000) and not cap.overlap(8, 1000) and not cap.overlap(7, 3000) and cap.overlap(7, 1000)


def test_more_captured_ranges_than_are_kept(cap):
    rng = random.Random(3)
    ranges = [(rng.randrange(1, 10 ** 6), rng.randrange(1, 100)) for _ in range(4 * cap.ranges)]
    for i, r in enumerate(ranges):
        cap.call(1, r)
        assert all(cap.overlap(1, lo, n) for lo, n in ranges[:i + 1])
    assert not cap.overlap(1, 2 * 10 ** 6)


def test_more_captures_than_are_kept(cap):
    for c in range(1, 3 * cap.captures):
        assert not cap.overlap(c, 1000)         # a new capture starts open, however many there were
        cap.call(c, (1000, 10))
        assert cap.overlap(c, 1000) and not cap.overlap(c, 2000)
    assert cap.overlap(1, 2000)                 # one that went: it may have written anything
    cap.call(1, (1, 1))
    assert cap.overlap(1, 2000) and not cap.overlap(3 * cap.captures - 1, 2000)


def test_a_capture_in_use_stays_while_others_come(cap):
    for c in range(2, 5 * cap.captures):
        cap.call(1, (1000, 10))
        cap.call(c, (2000, 10))
    assert cap.overlap(1, 1000) and not cap.overlap(1, 2000)

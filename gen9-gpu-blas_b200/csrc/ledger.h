// ledger.h -- the ledger of queued writes: which device ranges calls that were queued without a wait may still write. A kernel
// that reads an input before griddepcontrol.wait asks it first. Plain C++ over a few operations on events and streams, so that
// its rules are checked on the CPU (tests/test_ledger_cpu.py compiles this file with a scripted Api).
#pragma once
#include <cstddef>
#include <cstdint>

namespace g9 {

struct QueuedWrite {
    const void *p;   // NULL: none
    size_t bytes;
};

// Api: Stream and Event types (a default Event is "not made yet") and, all static,
//   bool record(Event &, Stream)   records the event behind all work queued on the stream so far (makes it on first use); false: cannot
//   bool done(Event)               whether that work has ended (false also where it cannot tell), asked while a Quiet is alive
//   Quiet                          such questions do no harm in its scope
//   void wait(Stream)              waits for the stream
template <typename Api>
class QueuedLedger {
    using Stream = typename Api::Stream;
    using Event = typename Api::Event;

public:
    static constexpr int kRanges = 32;
    static constexpr int kLost = 16;

    // The ranges of one call, queued on st just now. They share one event, recorded for the first of them.
    void add(const QueuedWrite *w, int n, Stream st) {
        int ev = -1;
        for (int k = 0; k < n; k++) {
            if (!w[k].p || !w[k].bytes) continue;
            if (ev < 0) {
                for (ev = 0; used_[ev]; ev++) {}   // one event more than there are entries
                if (!Api::record(ev_[ev], st)) return lost(st);
            }
            const uintptr_t lo = (uintptr_t)w[k].p, hi = lo + w[k].bytes;
            const int i = slot(lo, hi, st);
            if (i < 0) return lost(st);
            Entry &e = e_[i];
            if (i == n_) {
                n_++;
                e.lo = lo;
                e.hi = hi;
                e.st = st;
            } else {
                used_[e.ev]--;
                if (lo < e.lo) e.lo = lo;
                if (hi > e.hi) e.hi = hi;
            }
            e.ev = ev;
            used_[ev]++;
        }
    }

    // Whether overlap() has to look at events.
    bool touches(const void *p, size_t bytes) const {
        const uintptr_t lo = (uintptr_t)p, hi = lo + bytes;
        for (int i = 0; i < n_; i++)
            if (lo < e_[i].hi && e_[i].lo < hi) return true;
        return lost_n_ > 0;
    }

    // st has been waited for: its writes are done.
    void clear(Stream st) {
        for (int i = n_ - 1; i >= 0; i--)
            if (e_[i].st == st) drop(i);
        for (int i = lost_n_ - 1; i >= 0; i--)
            if (lost_[i].st == st) lost_drop(i);
    }

    // Whether queued work may still write some of [p, p + bytes): by the entries, or always while a write without one is under way.
    bool overlap(const void *p, size_t bytes) {
        if (!touches(p, bytes)) return false;
        const typename Api::Quiet quiet;
        for (int i = lost_n_ - 1; i >= 0; i--)
            if (Api::done(lost_[i].ev)) lost_drop(i);
        if (lost_n_) return true;
        const uintptr_t lo = (uintptr_t)p, hi = lo + bytes;
        for (int i = n_ - 1; i >= 0; i--) {
            if (!(lo < e_[i].hi && e_[i].lo < hi)) continue;
            if (!Api::done(ev_[e_[i].ev])) return true;
            drop(i);
        }
        return false;
    }

private:
    // An entry holds writes of one stream, up to its event.
    struct Entry {
        uintptr_t lo, hi;
        Stream st;
        int ev;
    };
    struct Lost {
        Stream st;
        Event ev{};
    };
    Entry e_[kRanges];
    int n_ = 0;
    Event ev_[kRanges + 1]{};
    int used_[kRanges + 1] = {};   // entries that hold the event
    Lost lost_[kLost]{};           // streams with writes that found no entry, each with an event behind the last of them
    int lost_n_ = 0;

    // The entry that takes a range of stream st: one that it overlaps or touches, a free one, or, where all are taken, that
    // of the stream which grows least. -1: all belong to other streams.
    int slot(uintptr_t lo, uintptr_t hi, Stream st) {
        for (int i = 0; i < n_; i++)
            if (lo <= e_[i].hi && e_[i].lo <= hi && e_[i].st == st) return i;
        if (n_ == kRanges) forget_ended();
        if (n_ < kRanges) return n_;
        int best = -1;
        size_t least = SIZE_MAX;
        for (int i = 0; i < n_; i++) {
            if (e_[i].st != st) continue;
            const size_t grown = lo < e_[i].lo ? e_[i].lo - lo : hi > e_[i].hi ? hi - e_[i].hi : 0;
            if (grown < least) {
                least = grown;
                best = i;
            }
        }
        return best;
    }

    // Drops the entries whose calls have ended, asking once for each call.
    void forget_ended() {
        const typename Api::Quiet quiet;
        for (int ev = 0; ev <= kRanges; ev++) {
            if (!used_[ev] || !Api::done(ev_[ev])) continue;
            for (int i = n_ - 1; i >= 0; i--)
                if (e_[i].ev == ev) drop(i);
        }
    }

    // The last entry takes the place of one that is dropped.
    void drop(int i) {
        used_[e_[i].ev]--;
        e_[i] = e_[--n_];
    }
    void lost_drop(int i) {
        const Lost gone = lost_[i];
        lost_[i] = lost_[--lost_n_];
        lost_[lost_n_] = gone;   // its event is kept for the next one
    }

    // A write on st that has no entry: overlap() answers true until it has ended. Where that could not be told, it is waited for.
    void lost(Stream st) {
        const typename Api::Quiet quiet;
        for (int i = lost_n_ - 1; i >= 0; i--)
            if (Api::done(lost_[i].ev)) lost_drop(i);
        int i = 0;
        while (i < lost_n_ && lost_[i].st != st) i++;
        if (i == kLost || !Api::record(lost_[i].ev, st)) return Api::wait(st);
        lost_[i].st = st;
        if (i == lost_n_) lost_n_++;
    }
};

// The ranges that captured calls write, by the capture's number: within its graph a kernel may start before the one ahead of it
// has ended. A replay as a whole starts and ends in its stream's order, so that a record matters to calls of the same capture
// alone, and its end needs no event. The latest kCaptures captures are kept; one older than those that went is answered for
// as if it wrote everything (numbers rise; where they did not, that is what a new capture would get).
class CaptureLedger {
public:
    static constexpr int kCaptures = 32;
    static constexpr int kRanges = 24;

    void add(const QueuedWrite *w, int n, unsigned long long capture) {
        if (lost(capture)) return;
        Record &r = record(capture);
        for (int k = 0; k < n; k++) {
            if (!w[k].p || !w[k].bytes) continue;
            const uintptr_t lo = (uintptr_t)w[k].p, hi = lo + w[k].bytes;
            int best = 0;
            size_t least = SIZE_MAX;
            for (int i = 0; i < r.n; i++) {   // 0: overlapping or touching
                const size_t far = lo > r.hi[i] ? lo - r.hi[i] : r.lo[i] > hi ? r.lo[i] - hi : 0;
                if (far < least) {
                    least = far;
                    best = i;
                }
            }
            if (least > 0 && r.n < kRanges) {
                best = r.n++;
                r.lo[best] = lo;
                r.hi[best] = hi;
            } else {                          // full: the nearest one grows over what lies between
                if (lo < r.lo[best]) r.lo[best] = lo;
                if (hi > r.hi[best]) r.hi[best] = hi;
            }
        }
    }

    // Whether the answer of overlap() depends on the capture.
    bool touches(const void *p, size_t bytes) const {
        const uintptr_t lo = (uintptr_t)p, hi = lo + bytes;
        for (int i = 0; i < n_; i++)
            for (int k = 0; k < r_[i].n; k++)
                if (lo < r_[i].hi[k] && r_[i].lo[k] < hi) return true;
        return gone_ > 0;
    }

    bool overlap(const void *p, size_t bytes, unsigned long long capture) const {
        if (lost(capture)) return true;
        const uintptr_t lo = (uintptr_t)p, hi = lo + bytes;
        for (int i = 0; i < n_; i++) {
            if (r_[i].capture != capture) continue;
            for (int k = 0; k < r_[i].n; k++)
                if (lo < r_[i].hi[k] && r_[i].lo[k] < hi) return true;
        }
        return false;
    }

private:
    struct Record {
        unsigned long long capture, used;   // used: when a range was last added
        int n;
        uintptr_t lo[kRanges], hi[kRanges];
    };
    Record r_[kCaptures];
    int n_ = 0;
    unsigned long long clock_ = 0, gone_ = 0;   // gone_: the highest number of those that went

    bool lost(unsigned long long capture) const {
        if (capture > gone_) return false;
        for (int i = 0; i < n_; i++)
            if (r_[i].capture == capture) return false;
        return true;
    }
    Record &record(unsigned long long capture) {
        int at = 0;
        for (int i = 0; i < n_; i++) {
            if (r_[i].capture == capture) {
                r_[i].used = ++clock_;
                return r_[i];
            }
            if (r_[i].used < r_[at].used) at = i;
        }
        if (n_ < kCaptures) at = n_++;
        else if (r_[at].capture > gone_) gone_ = r_[at].capture;
        r_[at].capture = capture;
        r_[at].used = ++clock_;
        r_[at].n = 0;
        return r_[at];
    }
};

}  // namespace g9

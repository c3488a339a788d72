// Host build of csrc/ledger.h for tests/test_ledger_cpu.py: streams are numbers, work ends when the test says so.
#include "ledger.h"
#include <cstdlib>
#include <vector>

namespace {

struct Script {
    struct Event {
        int stream = -1;
        long behind = -1;   // works of the stream before it
    };
    static std::vector<long> queued, ended;   // works of a stream
    static std::vector<int> waits;
    static bool can_record;
    using Stream = int;
    static bool record(Event &e, Stream st) {
        if (!can_record) return false;
        e = {st, queued[st]};
        return true;
    }
    static int quiet;
    struct Quiet {
        Quiet() { quiet++; }
        ~Quiet() { quiet--; }
    };
    static bool done(const Event &e) {
        if (quiet != 1) std::abort();   // asked outside of the scope that keeps it harmless
        return ended[e.stream] >= e.behind;
    }
    static void wait(Stream st) {
        waits.push_back(st);
        ended[st] = queued[st];
    }
};
std::vector<long> Script::queued, Script::ended;
std::vector<int> Script::waits;
bool Script::can_record = true;
int Script::quiet = 0;
g9::QueuedLedger<Script> *ledger = nullptr;

}  // namespace

extern "C" {
void led_new(int streams) {
    delete ledger;
    ledger = new g9::QueuedLedger<Script>;
    Script::queued.assign(streams, 0);
    Script::ended.assign(streams, 0);
    Script::waits.clear();
    Script::can_record = true;
}
void led_can_record(int on) { Script::can_record = on; }
// one call on st that writes n ranges
void led_call(int st, int n, const uint64_t *lo, const uint64_t *bytes) {
    std::vector<g9::QueuedWrite> w;
    for (int i = 0; i < n; i++) w.push_back({(const void *)lo[i], (size_t)bytes[i]});
    Script::queued[st]++;
    ledger->add(w.data(), n, st);
}
void led_end(int st, long works) { Script::ended[st] += works; }
long led_open(int st) { return Script::queued[st] - Script::ended[st]; }
void led_clear(int st) {
    Script::ended[st] = Script::queued[st];
    ledger->clear(st);
}
int led_overlap(uint64_t lo, uint64_t bytes) { return ledger->overlap((const void *)lo, bytes); }
int led_waits() { return (int)Script::waits.size(); }
int led_ranges() { return g9::QueuedLedger<Script>::kRanges; }
int led_lost() { return g9::QueuedLedger<Script>::kLost; }
}

namespace {
g9::CaptureLedger *captured = nullptr;
}
extern "C" {
void cap_new() {
    delete captured;
    captured = new g9::CaptureLedger;
}
void cap_call(uint64_t capture, int n, const uint64_t *lo, const uint64_t *bytes) {
    std::vector<g9::QueuedWrite> w;
    for (int i = 0; i < n; i++) w.push_back({(const void *)lo[i], (size_t)bytes[i]});
    captured->add(w.data(), n, capture);
}
int cap_overlap(uint64_t lo, uint64_t bytes, uint64_t capture) { return captured->overlap((const void *)lo, bytes, capture); }
int cap_captures() { return g9::CaptureLedger::kCaptures; }
int cap_ranges() { return g9::CaptureLedger::kRanges; }
}

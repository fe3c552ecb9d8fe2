// Every order of events of the hand-off between the copying warps and the issuer of the 4-bit product by pairs of CTAs, waits that
// give up at any point among them, with the rule of csrc/fp4_handoff.h. Prints how many states it saw, and how many of them
// have no way on though the issuer has not come to its end.
//
// A copying warp: waits (until the MMAs of step i - STAGES are done; may give up at any time, and then waits for nothing but the
// rule), arrives at the barrier of its stage, goes on to step i + CP. The issuer: at a tile's first step waits for the epilogue (may
// give up), arrives at the step's barrier and stays until two arrivals are in, its own or not, then counts the step as taken and,
// unless it gave up, issues the MMAs.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <tuple>
#include <vector>

#include "fp4_handoff.h"

using hn::fp4g::Handoff;
constexpr int S = Handoff::STAGES, CP = Handoff::CP;

struct State {
    int step[CP];           // of each copying warp
    bool failed[CP];
    int count[S];           // arrivals at each barrier, 0 or 1
    bool inside;            // the issuer's arrival for `taken` is in, and it waits
    bool released;          // ... and the barrier has completed
    bool issuer_failed;
    int taken, issued;      // steps the issuer has passed; whose MMAs it issued
    bool operator<(const State &o) const { return key() < o.key(); }
    std::vector<int> key() const {
        std::vector<int> k;
        for (int i = 0; i < CP; ++i) { k.push_back(step[i]); k.push_back(failed[i]); }
        for (int i = 0; i < S; ++i) k.push_back(count[i]);
        for (int v : {(int)inside, (int)released, (int)issuer_failed, taken, issued}) k.push_back(v);
        return k;
    }
};

static int steps, tile;

// an arrival at barrier b; two complete it
static void arrive(State &s, int b) {
    if (++s.count[b] < 2) return;
    s.count[b] = 0;
    if (s.inside && s.taken % S == b) s.released = true;
}

static std::vector<State> next(const State &s) {
    std::vector<State> out;
    for (int w = 0; w < CP; ++w) {
        const int i = s.step[w];
        if (i >= steps) continue;
        if (!s.failed[w]) {
            State t = s;
            t.failed[w] = true;
            out.push_back(t);
        }
        if (s.failed[w] ? s.taken >= Handoff::taken_before(i) : s.issued > i - S) {
            State t = s;
            t.step[w] += CP;
            arrive(t, i % S);
            out.push_back(t);
        }
    }
    if (s.taken < steps) {
        if (!s.inside) {
            if (s.taken % tile == 0 && !s.issuer_failed) {
                State t = s;
                t.issuer_failed = true;
                out.push_back(t);
            }
            State t = s;
            t.inside = true;
            t.released = false;
            arrive(t, s.taken % S);
            out.push_back(t);
        } else if (s.released) {
            State t = s;
            t.inside = false;
            ++t.taken;
            if (!s.issuer_failed) t.issued = t.taken;
            out.push_back(t);
        }
    }
    return out;
}

int main(int argc, char **argv) {
    steps = argc > 1 ? atoi(argv[1]) : 13;
    tile = argc > 2 ? atoi(argv[2]) : 4;
    State first = {};
    for (int w = 0; w < CP; ++w) first.step[w] = w;
    std::set<State> seen = {first};
    std::vector<State> todo = {first};
    long stuck = 0, ends = 0;
    while (!todo.empty()) {
        const State s = todo.back();
        todo.pop_back();
        const std::vector<State> n = next(s);
        if (n.empty()) ++(s.taken < steps ? stuck : ends);
        for (const State &t : n)
            if (seen.insert(t).second) todo.push_back(t);
    }
    printf("states %zu, ends %ld, stuck %ld\n", seen.size(), ends, stuck);
    return stuck == 0 && ends > 0 ? 0 : 1;
}

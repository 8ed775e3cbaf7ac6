// The extents of the experts' plan from its entries alone: the parts of its words one behind the other, every entry in one
// workgroup's share.  CPU only; prints "ok <checks>" or what failed.
#include <cstdio>
#include <random>
#include <vector>

#include "../tr-infer_amd/csrc/geometry.hpp"

using namespace trk::geo;
typedef unsigned long long u64;

static u64 checks = 0;
static bool bad(bool ok, const char* what, unsigned a, unsigned b, unsigned c) {
    checks++;
    if (!ok) printf("%s at %u %u %u\n", what, a, b, c);
    return !ok;
}

int main() {
    std::mt19937 rng(11);
    const unsigned T = 1024;  // entries that a workgroup's threads take at once
    for (int i = 0; i < 20000; i++) {
        const unsigned m = 9 + rng() % (i % 3 ? 300 : 20000), slots = 1 + rng() % 32, E = 1 + rng() % 1024;
        const u64 n = (u64)m * slots;
        const unsigned rows = plan_rows(m, slots, E), wgs = plan_workgroups(m, slots);
        if (bad(rows == 32 || rows == 64 || rows == 128, "rows of a tile", m, slots, E)) return 1;
        // entries dealt to experts by halves, until one is left with the rest: few full tiles, many ragged ones
        std::vector<u64> load(E);
        u64 left = n;
        for (unsigned e = 0; e < E && left; e++) load[e] = e + 1 == E ? left : (left + 1) / 2, left -= load[e];
        u64 tiles = 0;
        for (u64 l : load) tiles += l / rows + (l % rows ? 1 : 0);
        const u64 head = 4, entries = head + n, first_tile = plan_tile_at(m, slots), counts = plan_counts_at(m, slots, E);
        if (bad(first_tile >= entries && first_tile % 4 == 0, "tiles behind the entries", m, slots, E)) return 1;
        if (bad(counts >= first_tile + 4 * tiles, "counts behind the last tile", m, slots, E)) return 1;
        if (bad(plan_words(m, slots, E) >= counts + (wgs > 1 ? (u64)wgs * E : 0), "words", m, slots, E)) return 1;
        // each workgroup takes `per` rounds of T entries, as the launcher reckons them
        const u64 per = (n + (u64)wgs * T - 1) / ((u64)wgs * T);
        u64 seen = 0;
        for (unsigned w = 0; w < wgs; w++) {
            const u64 from = (u64)w * per * T, to = from + per * T;
            seen += from >= n ? 0 : (to < n ? to : n) - from;
        }
        if (bad(seen == n && (u64)wgs * per * T <= 0xffffffffull, "entries of the workgroups", m, slots, E)) return 1;
    }
    // the largest that is taken
    for (unsigned slots : {1u, 7u, 32u}) {
        const unsigned m = 0x7fffffffu / slots, wgs = plan_workgroups(m, slots);
        const u64 n = (u64)m * slots, per = (n + (u64)wgs * T - 1) / ((u64)wgs * T);
        if (bad((u64)wgs * per * T >= n && (u64)wgs * per * T <= 0xffffffffull, "the largest", m, slots, 0)) return 1;
    }
    printf("ok %llu\n", checks);
    return 0;
}

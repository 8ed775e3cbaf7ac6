// The rules that choose the int8 products' forms, at sizes where the forms were timed, and the plan's extents over a sweep
// of sizes and loads.  CPU only; prints "ok <checks>" or what failed.
#include <cstdio>
#include <random>
#include <vector>

#include "../tr-infer_amd/csrc/geometry.hpp"

using namespace trk::geo;

static unsigned long long checks = 0;
static bool bad(bool ok, const char* what, unsigned a, unsigned b, unsigned c) {
    checks++;
    if (!ok) printf("%s at %u %u %u\n", what, a, b, c);
    return !ok;
}

int main() {
    // m, rows, k -> the form that was fastest, or within a tenth of it
    const struct {
        unsigned m, rows, k, form;
    } timed[] = {{4096, 12288, 2560, I8_TILE_256}, {8192, 8192, 8192, I8_TILE_256}, {1600, 6000, 4096, I8_TILE_256},
                 {2048, 4096, 4096, I8_TILE_128},  {512, 12288, 2560, I8_TILE_128}, {1600, 6000, 512, I8_TILE_128},
                 {256, 12288, 2560, I8_TILE_64},   {128, 12288, 2560, I8_TILE_64},  {64, 12288, 2560, I8_TILE_64},
                 {1024, 2048, 2048, I8_TILE_64},   {400, 2560, 4096, I8_TILE_64},   {32, 12288, 2560, I8_TILE_32},
                 {1, 12288, 2560, I8_TILE_32},     {77, 5003, 1999, I8_TILE_32},    {512, 1024, 4096, I8_TILE_32},
                 {1, 2560, 2560, I8_STRIP},        {16, 2560, 10240, I8_STRIP},     {1, 5000, 512, I8_STRIP},
                 {16, 320, 512, I8_STRIP}};
    for (const auto& t : timed)
        if (bad(gemm_i8_form(t.m, t.rows, t.k, t.k, t.k) == (I8Form)t.form, "form", t.m, t.rows, t.k)) return 1;
    // rows too far apart for 32-bit offsets never go to the tiles
    if (bad(gemm_i8_form(4096, 12288, 2560, 1u << 23, 2560) == I8_STRIP, "far weights", 0, 0, 0)) return 1;
    if (bad(gemm_i8_form(4096, 12288, 2560, 2560, 1u << 23) == I8_STRIP, "far rows", 0, 0, 0)) return 1;
    if (bad(i8_tile_addresses(2048, 2048, 2097151) && !i8_tile_addresses(2048, 2048, 2097152), "addresses", 0, 0, 0)) return 1;
    if (bad(!i8_tile_addresses(1u << 23, 2048, 9), "address of weights", 0, 0, 0)) return 1;
    // a plan's tiles under any load fit what it is sized for, and its parts do not overlap
    std::mt19937 rng(5);
    for (int i = 0; i < 20000; i++) {
        const unsigned m = 1 + rng() % (i % 3 ? 300 : 20000), slots = 1 + rng() % 32, E = 1 + rng() % 1024;
        const unsigned rows = plan_rows(m, slots, E);
        std::vector<unsigned> load(E);
        const unsigned long long n = (unsigned long long)m * slots;
        unsigned long long left = n;
        for (unsigned e = 0; e < E && left; e++) {  // from one entry each to all on one
            const unsigned long long most = i % 2 ? left : 1 + rng() % (2 * n / E + 1);
            load[e] = (unsigned)(e + 1 == E ? left : most < left ? most : left);
            left -= load[e];
        }
        unsigned long long tiles = 0;
        for (unsigned e = 0; e < E; e++) tiles += (load[e] + rows - 1) / rows;
        if (bad(tiles <= plan_tiles(m, slots, E, rows), "tiles", m, slots, E)) return 1;
        if (bad(plan_tile_at(m, slots) >= 4 + n && plan_tile_at(m, slots) % 4 == 0, "tile words", m, slots, E)) return 1;
        const unsigned wgs = plan_workgroups(m, slots);
        if (bad(plan_words(m, slots, E) >= plan_counts_at(m, slots, E) + (wgs > 1 ? wgs * E : 0), "count words", m, slots, E))
            return 1;
        if (bad(wgs >= 1 && wgs <= 64, "plan workgroups", m, slots, E)) return 1;
    }
    printf("ok %llu\n", checks);
    return 0;
}

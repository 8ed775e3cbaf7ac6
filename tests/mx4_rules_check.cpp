// The rules that choose the 4-bit products' forms, at sizes where the forms were timed.  CPU only; prints "ok <checks>" or what
// failed.
#include <cstdio>

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
    } timed[] = {{1, 512, 512, I8_STRIP},         {1, 12288, 2560, I8_STRIP},      {4, 5003, 8192, I8_STRIP},
                 {16, 2560, 8192, I8_STRIP},      {200, 512, 2560, I8_STRIP},      {33, 5003, 2560, I8_TILE_32},
                 {400, 2560, 2560, I8_TILE_32},   {100, 5003, 512, I8_TILE_64},    {64, 12288, 2560, I8_TILE_64},
                 {4096, 512, 8192, I8_TILE_64},   {200, 2560, 8192, I8_TILE_64},   {800, 12288, 2560, I8_TILE_128},
                 {4096, 2560, 2560, I8_TILE_128}, {512, 12288, 2560, I8_TILE_128}, {4096, 12288, 512, I8_TILE_256},
                 {4096, 12288, 2560, I8_TILE_256}};
    for (const auto& t : timed) {
        const unsigned nb = (t.k + 31) / 32;
        if (bad(gemm_mx4_form(t.m, t.rows, nb, 16 * nb, 16 * nb, nb, nb) == (I8Form)t.form, "form", t.m, t.rows, t.k)) return 1;
    }
    // rows too far apart for 32-bit offsets never go to the tiles
    for (int i = 0; i < 4; i++) {
        const unsigned long long far = 1u << 23, ld[4] = {i == 0 ? far : 1280, i == 1 ? far : 1280, i == 2 ? far : 80, i == 3 ? far : 80};
        if (bad(gemm_mx4_form(4096, 12288, 80, ld[0], ld[1], ld[2], ld[3]) == I8_STRIP, "far rows", i, 0, 0)) return 1;
    }
    if (bad(!layer_routes_apart(704) && layer_routes_apart(1408), "routes", 0, 0, 0)) return 1;
    if (bad(layer_down_waves(128, 11) == 12 && layer_down_waves(1024, 11) == 8 && layer_down_waves(1024, 64) == 4 && layer_down_waves(128, 2) == 4, "waves", 0, 0, 0))
        return 1;
    printf("ok %llu\n", checks);
    return 0;
}

// Which kernel a 4-bit product's size takes: a line of input each, a line of output.  CPU only.
//   gemm m rows k        -> strip, 64x32, 64x64, 128x128 or 256x256 (rows of whole blocks)
//   up m slots E rows    -> the experts' tile: entries, "narrow" or "wide", and at 128 entries "once" or "again" (whether the
//   down m slots E rows     weights are loaded past the caches' order)
#include <cstdio>
#include <cstring>

#include "../tr-infer_amd/csrc/geometry.hpp"

using namespace trk::geo;

int main() {
    char op[8];
    unsigned a, b, c, d;
    while (scanf("%7s", op) == 1) {
        if (!strcmp(op, "gemm")) {
            if (scanf("%u %u %u", &a, &b, &c) != 3) return 1;
            const unsigned nb = (c + 31) / 32, lds = (nb + 3) / 4 * 4;
            static const char* const names[] = {"strip", "64x32", "64x64", "128x128", "256x256"};
            printf("%s\n", names[gemm_mx4_form(a, b, nb, 16 * nb, 16 * nb, lds, lds)]);
            continue;
        }
        const bool up = !strcmp(op, "up");
        if ((!up && strcmp(op, "down")) || scanf("%u %u %u %u", &a, &b, &c, &d) != 4) return 1;
        const unsigned rows = plan_rows(a, b, c);
        const bool narrow = experts_width(up ? 2 * d : d, plan_tiles(a, b, c, rows), false) == X_NARROW;
        printf("%u %s%s\n", rows, narrow ? "narrow" : "wide",
               rows < 128 ? "" : experts_once(a, b, c, up ? 64 : 128) ? " once" : " again");
    }
    return 0;
}

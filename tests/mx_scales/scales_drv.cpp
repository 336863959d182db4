// Host driver: the reads of a many-row MXFP4 product's scales (csrc/mx_scales.h), for
// every group of every K up to the number given, in buffers that end where the rows do.
// Built with the address sanitizer, which reports a read past them.
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "mx_scales.h"

using namespace apus;

static int bad = 0;
#define CHECK(c)                                                              \
    do {                                                                      \
        if (!(c) && bad++ < 10) printf("K %d stage %d G %d group %d: %s\n", K, stage, G, grp, #c); \
    } while (0)

// as the kernels bring a group's scales: `per` stages to 16 of them
static void group(int K, int stage, int G, int grp) {
    const KShare sh = k_share(K, stage, G, grp);
    const uint32_t ks = K / 32, s0 = sh.k0 / 32, rows = 3;
    const int left = (K - sh.k0 + stage - 1) / stage, own = sh.nk < left ? sh.nk : left, per = 512 / stage;
    CHECK(sh.k0 < K && sh.k0 % stage == 0);
    uint8_t *const buf = (uint8_t *)malloc(rows * ks);   // (16-byte aligned)
    for (uint32_t i = 0; i < rows * ks; i++) buf[i] = (uint8_t)(i * 37 + 11);
    for (uint32_t r = 0; r < rows; r++) {
        const uint8_t *const row = buf + r * ks;
        if (scales_whole(ks, s0, buf, nullptr)) {
            uint8_t v[16];
            memcpy(v, row + s0, 16);
            CHECK(((uintptr_t)row + s0) % 16 == 0 && s0 + 16 <= ks);
        }
        for (int c = 0; c < (own + per - 1) / per; c++) {
            RowScales f;
            f.load(row, s0 + 16 * c, ks);
            for (uint32_t i = 0; i < 16; i++) {
                const uint32_t at = s0 + 16 * c + i;
                CHECK((uint8_t)(f.v[i / 4] >> (i % 4 * 8)) == (at < ks ? row[at] : 0));
            }
        }
    }
    free(buf);
}

int main(int argc, char **argv) {
    const int last = argc > 1 ? atoi(argv[1]) : 8192;
    for (int K = 32; K <= last; K += 32)
        for (int stage = 64; stage <= 256; stage *= 4)
            for (int G = 1; G <= 2; G++) {
                if (G == 2 && K <= stage) continue;      // (halves need a stage each)
                for (int grp = 0; grp < G; grp++) group(K, stage, G, grp);
            }
    printf("%s\n", bad ? "FAILED" : "ok");
    return bad != 0;
}

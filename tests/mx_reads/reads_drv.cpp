// Host driver: what the MXFP4 products read (csrc/mx_reads.h), in buffers that end where
// the operands do: the scales of every group of every K up to the number given, the rows
// of every tile. Built with the address sanitizer, which reports a read past them.
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "mx_reads.h"

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
    const int own = (sh.n + stage - 1) / stage, per = 512 / stage;
    CHECK(sh.n > 0 && sh.k0 % stage == 0 && (grp == 0) == (sh.k0 == 0));
    CHECK(sh.k0 + sh.n == (grp == G - 1 ? K : k_share(K, stage, G, 1).k0));       // all of K, once
    CHECK(sh.nk == k_share(K, stage, G, 0).nk && own <= sh.nk);                   // (as many barriers)
    CHECK((sh.nk - 1) * stage <= sh.n);                                           // whole, but for the last
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

// the tiles of workgroups of `tiles` 16 rows; a load adds a uniform offset of up to the
// last step's, which has to stay under the tile's bytes
static void tiles_of(int total, int tiles) {
    const int K = 416, stage = 128, G = tiles, grp = total, pitch = K / 2;
    for (int r0 = 0; r0 < total; r0 += 16 * tiles)
        for (int t = 0; t < tiles; t++) {
            const Rows16 r = rows16(r0 + 16 * t, total);
            CHECK(r.n >= 1 && r.n <= 16 && r.first >= 0 && r.first + r.n <= total);
            CHECK(r0 + 16 * t >= total || (r.first == r0 + 16 * t && r.first + r.n == (total < r.first + 16 ? total : r.first + 16)));
            for (int k = 0; k < K; k += stage) CHECK(k / 2 < r.n * pitch);
        }
}

int main(int argc, char **argv) {
    const int last = argc > 1 ? atoi(argv[1]) : 8192;
    for (int K = 32; K <= last; K += 32)
        for (int stage = 64; stage <= 256; stage *= 4)
            for (int G = 1; G <= 2; G++) {
                if (G == 2 && K <= stage) continue;      // (halves need a stage each)
                for (int grp = 0; grp < G; grp++) group(K, stage, G, grp);
            }
    for (int total = 1; total <= 300; total++)
        for (int tiles = 1; tiles <= 4; tiles++) tiles_of(total, tiles);
    printf("%s\n", bad ? "FAILED" : "ok");
    return bad != 0;
}

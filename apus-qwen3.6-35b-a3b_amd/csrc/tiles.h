// tiles.h -- the order in which a GEMM's workgroups take its output tiles.
#pragma once
#include <hip/hip_runtime.h>

namespace apus {

// Workgroup -> (output tile, row tile). Workgroups are dealt round-robin
// to the 8 XCDs (id % 8), each XCD running its ids in order, so XCD x gets
// tiles x q .. x q + q - 1 (q an eighth of the tiles) of an order in which
// the 32 tiles that an XCD runs together share operand tiles, which stay in
// that XCD's L2 while they walk K in step: with 8 or more row tiles, blocks
// of 4 output x 8 row tiles (12 distinct operand tiles instead of 18 with
// whole row-tile columns); with fewer, an output tile's row tiles one after
// the other. Every XCD has the same number of tiles to within one (whole
// 4 x 8 blocks dealt to XCDs left half of the chip idle below 8 blocks:
// 2048 outputs x 512 rows, K = 4096, 34.7 us, now 17.4).
__host__ __device__ inline int tile_grid(int nbo, int nbm) { return (nbo * nbm + 7) / 8 * 8; }
__host__ __device__ inline void tile_of(int id, int nbo, int nbm, int &ob, int &mb) {
    const int n = nbo * nbm, q = (n + 7) / 8, t = (id % 8) * q + id / 8;
    if (t >= n) {
        ob = nbo;                                  // past the last tile
        mb = 0;
        return;
    }
    if (nbm < 8) {
        ob = t / nbm;
        mb = t % nbm;
        return;
    }
    // bands of 8 row tiles; in a band, blocks of 4 output tiles, row fastest
    const int band = t / (8 * nbo), rows = min(8, nbm - 8 * band);
    const int p = t - 8 * nbo * band;
    const int blk = p / (4 * rows), w = min(4, nbo - 4 * blk), e = p - 4 * rows * blk;
    ob = 4 * blk + e % w;
    mb = 8 * band + e / w;
}

}  // namespace apus

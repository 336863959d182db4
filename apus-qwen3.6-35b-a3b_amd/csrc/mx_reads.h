// mx_reads.h -- which rows, k and scales the MXFP4 products read. Host code too: the
// reads are checked against the operands' ends on the CPU.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace apus {

// The 16 rows from `first` of `total`: those there are. With none left the last row
// again, for a tile whose products are not stored: a buffer of no bytes would end before
// the uniform offset that its loads add, which the bounds check is not made for.
struct Rows16 {
    int first, n;
};
__host__ __device__ inline Rows16 rows16(int first, int total) {
    const int left = total - first;
    return left > 0 ? Rows16{first, left < 16 ? left : 16} : Rows16{total - 1, 1};
}

// Group grp of G (1 or 2) of a many-row product: n of the K elements, from k0 on, in nk
// stages of `stage`. All but the last of a group's stages are whole: the kernels mask
// what lies past its k in the last one only. With K in halves, an odd number of stages
// leaves the first half one less, which it takes as one past its k.
struct KShare {
    int k0, n, nk;
};
__host__ __device__ inline KShare k_share(int K, int stage, int G, int grp) {
    const int all = (K + stage - 1) / stage, nk = (all + G - 1) / G, half = all / 2 * stage;
    return G == 1 ? KShare{0, K, nk} : grp == 0 ? KShare{0, half, nk} : KShare{half, K - half, nk};
}

// The first 16 scales of a group, from scale s0 of rows of ks on, are copied to LDS as
// they are: rows, start and bases in whole 16 bytes, so that the row has 16 from there.
__host__ __device__ inline bool scales_whole(uint32_t ks, uint32_t s0, const uint8_t *ws, const uint8_t *xs) {
    return (ks | s0 | (uint32_t)(uintptr_t)ws | (uint32_t)(uintptr_t)xs) % 16 == 0;
}

// Scales p .. p + 15 (512 k) of a row's ks, for a thread to bring, zeros past the row's
// end; p < ks. So many at a time because a load whose lanes read different rows takes
// the address unit a clock a lane, however little each lane reads: 8 bytes a row and
// stage took it as long as the codes.
struct RowScales {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 v;
    __host__ __device__ __forceinline__ void load(const uint8_t *row, uint32_t p, uint32_t ks) {
        if (ks >= 16) {                                  // (the row's last 16 bytes and a shift)
            const uint32_t at = p < ks - 16 ? p : ks - 16, past = p - at;
            __builtin_memcpy(&v, row + at, 16);          // (rows may begin at any byte)
            if (past) v = __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, v) >> (8 * (past & 15)));
        } else {
            v = u32x4{};
            for (uint32_t i = p; i < ks; i++) v[(i - p) / 4] |= (uint32_t)row[i] << ((i - p) % 4 * 8);
        }
    }
};

}  // namespace apus

// mx.h -- host checks shared by the MXFP4 and mixture-of-experts entry points.
// These check their arguments before they look for a device, so that a bad
// call is refused the same way with and without one.
#pragma once
#include "apus_rt.h"

namespace apus {

int mx_check_dims(size_t M, size_t O, size_t K);   // sizes under 2^31, K in whole blocks
int mx_ready();                                    // ensure_ready, on the calling thread's device

// A block of nb bytes and M rows (first row, bytes between rows, bytes of a row) share bytes.
inline bool block_overlaps(const void *b, size_t nb, const void *rows, size_t pitch, size_t n, size_t M) {
    const uintptr_t b0 = (uintptr_t)b, r0 = (uintptr_t)rows;
    const size_t i = b0 < r0 + n ? 0 : (b0 - r0 - n) / pitch + 1;    // the first row that ends past b0
    return i < M && r0 + i * pitch < b0 + nb;
}

// y = x w^T: M rows, O outputs, K inner elements; x is bf16 rows of pitch ldx, or,
// with xs, MXFP4
struct MxProduct {
    const uint8_t *w, *ws;
    const void *x;
    const uint8_t *xs;
    size_t ldx;
    uint16_t *y;
    size_t ldy;
    int M, O, K;
};
// products for many rows (mx_wide.hip): shape 2, tiles of 128 x 128, two a CU; 3, the
// same, one a CU, with K in two halves side by side; 4, 256 x 256; 5 (bf16 activations
// only), 256 outputs x 128 rows, two a CU
int mx_gemm_wide(const MxProduct &a, int shape);
// of so many 256 x 256 tiles, those that go in quarters, as the last workgroups
size_t mx_quarters(size_t tiles);

}  // namespace apus

#define APUS_ENABLED()                                                       \
    do {                                                                     \
        int r_ = ::apus::check_enabled();                                    \
        if (r_ != ::apus::kOk) return r_;                                    \
    } while (0)

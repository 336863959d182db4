// mx.h -- host checks shared by the MXFP4 and mixture-of-experts entry points.
// These check their arguments before they look for a device, so that a bad
// call is refused the same way with and without one.
#pragma once
#include "apus_rt.h"

namespace apus {

int mx_check_dims(size_t M, size_t O, size_t K);   // sizes under 2^31, K in whole blocks
int mx_ready();                                    // ensure_ready, on the calling thread's device

// products for many rows (mx_wide.hip): tiles of 128 x 128 (shape 2) or 256 x 256
// (shape 4)
int mx_gemm_wide(const uint8_t *w, const uint8_t *ws, const uint8_t *x, const uint8_t *xs,
                 uint16_t *y, size_t ldy, int M, int O, int K, int shape);
int mx_gemm_wide16(const uint8_t *w, const uint8_t *ws, const uint16_t *x, size_t ldx, uint16_t *y,
                   size_t ldy, int M, int O, int K, int shape);

}  // namespace apus

#define APUS_ENABLED()                                                       \
    do {                                                                     \
        int r_ = ::apus::check_enabled();                                    \
        if (r_ != ::apus::kOk) return r_;                                    \
    } while (0)

// mxfp4.hip -- MXFP4 (mx_dev.h) beside the bf16 projections: quantisation of
// bf16 rows, the values back, and products y[m][o] = rnd(sum_k w[o][k]
// x[m][k]) with MXFP4 weights and bf16 or MXFP4 activations.
//
// Layouts: codes [rows][K / 2], scales [rows][K / 32], both dense; bf16
// operands have rows of any pitch. K is a multiple of 32.
#include <stdint.h>

#include <algorithm>

#include "../../include/apus_hip.h"
#include "apus_dev.h"
#include "apus_host.h"
#include "mx.h"
#include "mx_dev.h"

using namespace apus;

namespace {

// 8 elements of row r, chunk c (of K / 8): the address of each operand.
// Dense rows are one long row.
struct Pos {
    size_t r, c;
};
__device__ __forceinline__ Pos pos_of(size_t i, size_t per_row, bool dense) {
    if (dense) return {0, i};
    const size_t r = i / per_row;
    return {r, i - r * per_row};
}

// A thread quantises 8 elements, four neighbours a block. The block's scale
// is 2^(floor(log2 max|x|) - 2), e2m1's largest exponent being 2, from the
// exponent field of the largest code (a subnormal maximum: the smallest scale,
// 2^-127); the hardware conversion rounds to nearest even and saturates at 6.
// A block with an infinity or NaN gets scale 255 (NaN) and zero codes.
__global__ __launch_bounds__(256) void k_mx_quantize(const uint16_t *__restrict__ x, size_t ldx,
                                                     uint8_t *__restrict__ codes,
                                                     uint8_t *__restrict__ scales, size_t n8,
                                                     size_t per_row, bool dense) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n8; i += (size_t)gridDim.x * 256) {
        const Pos p = pos_of(i, per_row, dense);
        const u32x4 v = *reinterpret_cast<const u32x4 *>(x + p.r * ldx + p.c * 8);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) m = max(m, max(v[j] & 0x7fffu, (v[j] >> 16) & 0x7fffu));
        // (the four threads of a block are a quad, all active: n8 % 4 == 0)
        m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));
        m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));
        const uint32_t e = m >> 7;
        const uint32_t s = e == 255 ? 255 : (uint32_t)max((int)e - 2, 0);
        const float sc = __uint_as_float(s << 23);
        // (scalars first: a bit cast of a vector's element reads element 0)
        const uint32_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v0), sc, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v1), sc, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v2), sc, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v3), sc, 3);
        reinterpret_cast<uint32_t *>(codes)[i] = s == 255 ? 0 : c;
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
    }
}

__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t *__restrict__ codes,
                                                       const uint8_t *__restrict__ scales,
                                                       uint16_t *__restrict__ x, size_t ldx,
                                                       size_t n8, size_t per_row, bool dense) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n8; i += (size_t)gridDim.x * 256) {
        const Pos p = pos_of(i, per_row, dense);
        const mx_bf16x8 v = mx_widen(reinterpret_cast<const uint32_t *>(codes)[i], scales[i >> 2]);
        *reinterpret_cast<mx_bf16x8 *>(x + p.r * ldx + p.c * 8) = v;
    }
}

// ---- products of few rows --------------------------------------------------
// A workgroup forms 16 outputs x 16 rows; its 4 wavefronts take every fourth
// step of 128 k, and their partial sums meet in LDS.
template <bool XMX>
__global__ __launch_bounds__(256) void k_mx_gemm_few(const uint8_t *__restrict__ w,
                                                     const uint8_t *__restrict__ ws,
                                                     const void *__restrict__ x,
                                                     const uint8_t *__restrict__ xs, size_t ldx,
                                                     uint16_t *__restrict__ y, size_t ldy, int M,
                                                     int O, int K, int nbo) {
    __shared__ mx_f32x4 red[4][64];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = (blockIdx.x % nbo) * 16, m0 = (blockIdx.x / nbo) * 16;
    // (outputs past O and rows past M repeat the last one; they are not stored)
    const auto wr = WMx::row(w, ws, (size_t)min(o0 + r, O - 1), K, g);
    const size_t m = (size_t)min(m0 + r, M - 1);
    mx_f32x4 acc{};
    for (int k = wave * 128; k < K; k += 512) {
        WMx::Frag wf;
        WMx::load(wf, wr, k, K);
        if constexpr (XMX) {
            const auto xr = WMx::row(x, xs, m, K, g);
            WMx::Frag xf;
            WMx::load(xf, xr, k, K);
            acc = mfma16_mx(wf, xf, acc);
        } else {
            const auto xr = XBf16<WMx>::row((const uint16_t *)x, ldx, m, g);
            XBf16<WMx>::Frag xf;
            XBf16<WMx>::load(xf, xr, k, K);
#pragma unroll
            for (int j = 0; j < 4; j++)
                acc = mfma16(WMx::operand(wf, j), __builtin_bit_cast(mx_bf16x8, xf.v[j]), acc);
        }
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    acc = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    if (m0 + r >= M) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int o = o0 + 4 * g + i;
        if (o < O) y[(size_t)(m0 + r) * ldy + o] = f2bf(acc[i]);
    }
}

// the y of an empty sum
__global__ __launch_bounds__(256) void k_mx_zero_rows(uint16_t *__restrict__ y, size_t ldy, size_t O,
                                                      size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256)
        y[i / O * ldy + i % O] = 0;
}

unsigned stream_grid(size_t threads) {
    return (unsigned)std::min<size_t>((threads + 255) / 256, (size_t)cu_count() * 32);
}

// Two sets of M rows (first row, bytes between rows, bytes of a row) share
// bytes. Rows of one pitch may interleave (column slices of one buffer);
// otherwise the sets' extents decide.
bool rows_overlap(const void *a, size_t pa, size_t na, const void *b, size_t pb, size_t nb, size_t M) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    const uintptr_t a1 = a0 + (M - 1) * pa + na, b1 = b0 + (M - 1) * pb + nb;
    if (a1 <= b0 || b1 <= a0) return false;
    if (pa != pb) return true;
    const size_t off = (b0 >= a0 ? b0 - a0 : pa - (a0 - b0) % pa) % pa;
    return off < na || off + nb > pa;
}

int gemm_check(const uint8_t *w, const uint8_t *ws, const void *x, const uint8_t *xs, size_t ldx,
               const uint16_t *y, size_t ldy, size_t M, size_t O, size_t K) {
    if (int r = mx_check_dims(M, O, K)) return r;
    if (M == 0 || O == 0) return kOk;
    if (!y) return set_error(kErrArgument, "NULL output");
    if (ldy < O) return set_error(kErrArgument, "output rows of %zu elements with pitch %zu", O, ldy);
    if ((uintptr_t)y % 2) return set_error(kErrArgument, "misaligned output");
    if (K == 0) return kOk;
    if (!w || !ws || !x) return set_error(kErrArgument, "NULL operand");
    if ((uintptr_t)w % 16) return set_error(kErrUnsupported, "MXFP4 codes need 16-byte alignment");
    const size_t mxk = K / 2, mxs = K / kMxBlock;
    if (xs) {
        if ((uintptr_t)x % 16)
            return set_error(kErrUnsupported, "MXFP4 codes need 16-byte alignment");
        if (rows_overlap(x, mxk, mxk, y, ldy * 2, O * 2, M) ||
            rows_overlap(xs, mxs, mxs, y, ldy * 2, O * 2, M))
            return set_error(kErrArgument, "the output overlaps the activations");
    } else {
        if ((uintptr_t)x % 16 || ldx % 8)
            return set_error(kErrUnsupported, "activation rows need 16-byte alignment (pitch %zu)", ldx);
        if (ldx < K) return set_error(kErrArgument, "rows of %zu elements with pitch %zu", K, ldx);
        if (rows_overlap(x, ldx * 2, K * 2, y, ldy * 2, O * 2, M))
            return set_error(kErrArgument, "the output overlaps the activations");
    }
    return kOk;
}

template <bool XMX>
int gemm_run(const uint8_t *w, const uint8_t *ws, const void *x, const uint8_t *xs, size_t ldx,
             uint16_t *y, size_t ldy, size_t M, size_t O, size_t K) {
    if (M == 0 || O == 0) return kOk;
    if (K == 0) {
        k_mx_zero_rows<<<stream_grid(M * O), 256, 0, stream()>>>(y, ldy, O, M * O);
        return launch_check("k_mx_zero_rows");
    }
    const unsigned nbo = cdiv(O, 16), nbm = cdiv(M, 16);
    if ((size_t)nbo * nbm > 0x7fffffffu) return set_error(kErrUnsupported, "MXFP4 gemm too large");
    APUS_TIMED("k_mx_gemm_few", k_mx_gemm_few<XMX><<<nbo * nbm, 256, 0, stream()>>>(
                                    w, ws, x, xs, ldx, y, ldy, (int)M, (int)O, (int)K, (int)nbo));
    return launch_check("k_mx_gemm_few");
}

}  // namespace

namespace apus {

int mx_check_dims(size_t M, size_t O, size_t K) {
    if (M > 0x7fffffffu || O > 0x7fffffffu || K > 0x7fffffffu)
        return set_error(kErrUnsupported, "MXFP4 dims past 2^31");
    if (K % kMxBlock)
        return set_error(kErrUnsupported, "MXFP4 rows come in blocks of %d (K=%zu)", kMxBlock, K);
    return kOk;
}

int mx_ready() {
    APUS_READY();
    int dev = -1;
    APUS_HIP_TRY(hipGetDevice(&dev));
    if (dev != current_device())
        return set_error(kErrArgument, "the calling thread's device is %d, the library's %d", dev,
                         current_device());
    return kOk;
}

}  // namespace apus

extern "C" {

int apus_hip_mxfp4_quantize(const uint16_t *x, size_t ldx, uint8_t *codes, uint8_t *scales,
                            size_t M, size_t K) {
    APUS_ENABLED();
    if (int r = mx_check_dims(M, 0, K)) return r;
    if (M && K) {
        if (!x || !codes || !scales) return set_error(kErrArgument, "NULL operand");
        if (ldx < K) return set_error(kErrArgument, "rows of %zu elements with pitch %zu", K, ldx);
        if ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)codes % 16)
            return set_error(kErrUnsupported, "MXFP4 quantisation needs 16-byte aligned rows and codes");
        if (rows_overlap(x, ldx * 2, K * 2, codes, K / 2, K / 2, M) ||
            rows_overlap(x, ldx * 2, K * 2, scales, K / kMxBlock, K / kMxBlock, M) ||
            rows_overlap(codes, M * K / 2, M * K / 2, scales, M * K / kMxBlock, M * K / kMxBlock, 1))
            return set_error(kErrArgument, "overlapping operands");
    }
    if (int r = mx_ready()) return r;
    if (!M || !K) return kOk;
    const size_t n8 = M * (K / 8);
    APUS_TIMED("k_mx_quantize", k_mx_quantize<<<stream_grid(n8), 256, 0, stream()>>>(
                                    x, ldx, codes, scales, n8, K / 8, ldx == K || M == 1));
    return launch_check("k_mx_quantize");
}

int apus_hip_mxfp4_dequantize(const uint8_t *codes, const uint8_t *scales, uint16_t *x, size_t ldx,
                              size_t M, size_t K) {
    APUS_ENABLED();
    if (int r = mx_check_dims(M, 0, K)) return r;
    if (M && K) {
        if (!x || !codes || !scales) return set_error(kErrArgument, "NULL operand");
        if (ldx < K) return set_error(kErrArgument, "rows of %zu elements with pitch %zu", K, ldx);
        if ((uintptr_t)x % 16 || ldx % 8 || (uintptr_t)codes % 16)
            return set_error(kErrUnsupported, "MXFP4 dequantisation needs 16-byte aligned rows and codes");
        if (rows_overlap(x, ldx * 2, K * 2, codes, K / 2, K / 2, M) ||
            rows_overlap(x, ldx * 2, K * 2, scales, K / kMxBlock, K / kMxBlock, M))
            return set_error(kErrArgument, "overlapping operands");
    }
    if (int r = mx_ready()) return r;
    if (!M || !K) return kOk;
    const size_t n8 = M * (K / 8);
    APUS_TIMED("k_mx_dequantize", k_mx_dequantize<<<stream_grid(n8), 256, 0, stream()>>>(
                                      codes, scales, x, ldx, n8, K / 8, ldx == K || M == 1));
    return launch_check("k_mx_dequantize");
}

int apus_hip_mxfp4_gemm_dev(const uint8_t *w, const uint8_t *ws, const uint16_t *x, size_t ldx,
                            uint16_t *y, size_t ldy, size_t M, size_t O, size_t K) {
    APUS_ENABLED();
    if (int r = gemm_check(w, ws, x, nullptr, ldx, y, ldy, M, O, K)) return r;
    if (int r = mx_ready()) return r;
    return gemm_run<false>(w, ws, x, nullptr, ldx, y, ldy, M, O, K);
}

int apus_hip_mxfp4_gemm_mx_dev(const uint8_t *w, const uint8_t *ws, const uint8_t *x,
                               const uint8_t *xs, uint16_t *y, size_t ldy, size_t M, size_t O,
                               size_t K) {
    APUS_ENABLED();
    if (M && O && K && !xs) return set_error(kErrArgument, "NULL operand");
    if (int r = gemm_check(w, ws, x, xs, 0, y, ldy, M, O, K)) return r;
    if (int r = mx_ready()) return r;
    return gemm_run<true>(w, ws, x, xs, 0, y, ldy, M, O, K);
}

}  // extern "C"

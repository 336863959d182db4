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
#include "mx_reads.h"

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
// A block with an infinity or NaN gets scale 255 (NaN) and zero codes. Bytes: 12352
// rows of 2048 in 12.9 us, 64 MB, 5.0 TB/s; one row 1.2 us, all launch.
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

// 8 elements a thread, their scale read with them. 12352 rows of 2048: 9.8 us.
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
// A workgroup forms 16 RT outputs x 16 NT rows; its 8 wavefronts take every
// eighth pair of steps of 128 k, and their partial sums meet in LDS. A pair's loads are all
// on their way before the first is used; with more than 32 rows of bf16 activations, a
// step's (there are no registers for more). Rows come along their length and
// become operands in LDS of the wavefront's own (mx_dev.h): loaded by each lane for
// itself the product of 37 rows took 10.5 us, now 7.1. XR: the loads of four
// rows that a tile of bf16 activations has (1 for up to 4 rows).
// Bound by the latency of these rounds of loads, one after the other: 1 row x 12352
// outputs, K 2048, one round, 5.6 us for 13.5 MB; 37 rows x 2048 x 4096, four, on half the
// CUs, 7.1 us; 64 rows of MXFP4 x 2048 x 4096, two, on half the CUs, 5.6 us.
constexpr int kFewWaves = 8;

template <bool XMX, int RT, int NT, int XR>
__global__ __launch_bounds__(64 * kFewWaves) void k_mx_gemm_few(const uint8_t *__restrict__ w,
                                                                const uint8_t *__restrict__ ws,
                                                                const void *__restrict__ x,
                                                                const uint8_t *__restrict__ xs, size_t ldx,
                                                                uint16_t *__restrict__ y, size_t ldy, int M,
                                                                int O, int K, int nbo) {
    constexpr int S = !XMX && NT > 2 ? 1 : 2;            // steps in flight (registers)
    constexpr int XT = XMX ? WMx::kTile : RowsBf16::kTile;
    constexpr int PART = RT * 1024 + XT > RT * NT * 1024 ? RT * 1024 + XT : RT * NT * 1024;
    __shared__ __attribute__((aligned(16))) char sm[kFewWaves * PART];
    using X = XBf16<WMx>;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = (blockIdx.x % nbo) * 16 * RT, m0 = (blockIdx.x / nbo) * 16 * NT;
    char *const mine = sm + wave * PART, *const mx = mine + RT * 1024;
    // (outputs past O and rows past M read as zero or as the last one, and are not stored)
    WMx::Tile wt[RT], xt[NT];
    i32x4 xb[NT];
    uint32_t xl[NT][4];
    const uint32_t pitch = (uint32_t)ldx * 2;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const Rows16 o = rows16(o0 + 16 * t, O);
        wt[t] = WMx::tile(w, ws, o.first, o.n, K);
    }
#pragma unroll
    for (int u = 0; u < NT; u++) {
        const Rows16 m = rows16(m0 + 16 * u, M);
        if constexpr (XMX) {
            xt[u] = WMx::tile(x, xs, m.first, m.n, K);
        } else {
            xb[u] = dma_rsrc((const uint16_t *)x + (size_t)m.first * ldx, (m.n - 1) * pitch + K * 2);
#pragma unroll
            for (int i = 0; i < 4; i++) xl[u][i] = 4 * i + g < m.n ? (4 * i + g) * pitch : kPast - 256;
        }
    }
    const auto wl = WMx::raw_lane(lane, K);
    const int steps = (K + 127) / 128;
    mx_f32x4 acc[RT][NT] = {};
    for (int st = wave * 2; st < steps; st += st & 1 || S == 2 ? kFewWaves * 2 - (S == 1) : 1) {
        WMx::Raw fw[S][RT], fq[S][NT];
        RowsBf16::Raw fx[S][NT];
#pragma unroll
        for (int s = 0; s < S; s++) {
#pragma unroll
            for (int t = 0; t < RT; t++) WMx::load_raw(fw[s][t], wt[t], wl, st + s, K);
#pragma unroll
            for (int u = 0; u < NT; u++) {
                if constexpr (XMX) WMx::load_raw(fq[s][u], xt[u], wl, st + s, K);
                else X::load_raw<XR>(fx[s][u], xb[u], xl[u], st + s, K);
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < S; s++) {
            WMx::Frag f[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                WMx::put(mine + t * 1024, fw[s][t], lane);
                WMx::get(f[t], mine + t * 1024, fw[s][t], lane);
            }
#pragma unroll
            for (int u = 0; u < NT; u++) {
                if constexpr (XMX) {
                    WMx::Frag q;
                    WMx::put(mx, fq[s][u], lane);
                    WMx::get(q, mx, fq[s][u], lane);
#pragma unroll
                    for (int t = 0; t < RT; t++) acc[t][u] = mfma16_mx(f[t], q, acc[t][u]);
                } else {
                    RowsBf16::put(mx, fx[s][u], lane);
                    mx_bf16x8 v[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = X::piece(mx, j, lane);
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int t = 0; t < RT; t++)
                            acc[t][u] = mfma16(WMx::operand(f[t], j), v[j], acc[t][u]);
                }
            }
        }
    }
    // [wave][row tile][tile]
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int u = 0; u < NT; u++) *reinterpret_cast<mx_f32x4 *>(mine + (t * NT + u) * 1024 + lane * 16) = acc[t][u];
    __syncthreads();
    // a thread finishes 4 outputs of a row, a row's outputs side by side
    const bool vec = ((ldy | (size_t)O) & 3) == 0 && ((uintptr_t)y & 7) == 0;
    for (int e = threadIdx.x; e < RT * NT * 64; e += 64 * kFewWaves) {
        const int q = e % (4 * RT), r = e / (4 * RT), o = o0 + 4 * q, m = m0 + r;
        if (m >= M || o >= O) continue;
        const char *p = sm + (q / 4 * NT + r / 16) * 1024 + (q % 4 * 16 + r % 16) * 16;
        mx_f32x4 s = *reinterpret_cast<const mx_f32x4 *>(p);
#pragma unroll
        for (int v = 1; v < kFewWaves; v++) s += *reinterpret_cast<const mx_f32x4 *>(p + v * PART);
        uint16_t *yo = y + (size_t)m * ldy + o;
        if (vec) {
            *reinterpret_cast<ushort4 *>(yo) = make_ushort4(f2bf(s[0]), f2bf(s[1]), f2bf(s[2]), f2bf(s[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (o + i < O) yo[i] = f2bf(s[i]);
        }
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

// 32-bit offsets reach 256 rows of activations or codes
constexpr size_t kMxMaxPitch = (size_t)1 << 21;
// elements of a matrix with its gaps (no extent overflows, tiles count in 32 bits)
constexpr size_t kMxMaxElements = (size_t)1 << 40;

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
    if (ldy > kMxMaxElements / M) return set_error(kErrUnsupported, "%zu output rows of pitch %zu", M, ldy);
    if ((uintptr_t)y % 2) return set_error(kErrArgument, "misaligned output");
    if (K == 0) return kOk;
    if (!w || !ws || !x) return set_error(kErrArgument, "NULL operand");
    if ((uintptr_t)w % 16) return set_error(kErrUnsupported, "MXFP4 codes need 16-byte alignment");
    const size_t mxk = K / 2, mxs = K / kMxBlock;
    if (block_overlaps(w, O * mxk, y, ldy * 2, O * 2, M) || block_overlaps(ws, O * mxs, y, ldy * 2, O * 2, M))
        return set_error(kErrArgument, "the output overlaps the weights");
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
        if (ldx > kMxMaxPitch) return set_error(kErrUnsupported, "rows of pitch %zu", ldx);
        if (rows_overlap(x, ldx * 2, K * 2, y, ldy * 2, O * 2, M))
            return set_error(kErrArgument, "the output overlaps the activations");
    }
    return kOk;
}

template <bool XMX, int RT, int NT, int XR>
int few_run(const uint8_t *w, const uint8_t *ws, const void *x, const uint8_t *xs, size_t ldx,
            uint16_t *y, size_t ldy, size_t M, size_t O, size_t K) {
    const size_t nbo = cdiv(O, 16 * RT), n = nbo * cdiv(M, 16 * NT);
    if (n > 0x7fffffffu) return set_error(kErrUnsupported, "MXFP4 gemm too large");
    APUS_TIMED("k_mx_gemm_few", k_mx_gemm_few<XMX, RT, NT, XR><<<(unsigned)n, 64 * kFewWaves, 0, stream()>>>(
                                    w, ws, x, xs, ldx, y, ldy, (int)M, (int)O, (int)K, (int)nbo));
    return launch_check("k_mx_gemm_few");
}

// Estimated times in us of the product's forms. What a form takes goes by the
// workgroups of the busiest CU and, but for a fixed part, by K. Over 512 .. 12352
// outputs x 48 .. 4096 rows and K 1024 .. 4096 (105 sizes, both kinds of activations)
// the form with the least estimate was within a tenth of the best one measured.
struct FewCost {
    float fixed, one, two;                  // one, two: tiles of 16 and 32 outputs x 64 rows
    float fixed4, four;                     // and of 64 outputs (bf16 activations)
};
constexpr FewCost kFewCost[] = {{2.5f, 3.6f, 5.6f, 4.5f, 7.0f}, {2.6f, 1.3f, 2.0f}};     // bf16, MXFP4 activations
struct WideCost {
    float f1, k1, f2, k2;                   // 128 x 128 tiles: one on the busiest CU, two
    float k3;                               // the same in two halves of K (fixed part f1)
    float f4, k4, fill;                     // 256 x 256: per round; with every CU busy
    float k5, f6, k6;                       // 256 x 128: one on the busiest CU (fixed part f1), two
};
constexpr WideCost kWideCost[] = {{3.0f, 15.2f, 4.0f, 28.0f, 13.5f, 7.0f, 43.0f, 12.0f, 30.0f, 4.0f, 51.0f},
                                  {3.2f, 4.8f, 4.0f, 10.0f, 5.0f, 6.5f, 10.5f, 11.2f, 0.0f, 0.0f, 0.0f}};

size_t rounds(size_t n) { return (n + cu_count() - 1) / cu_count(); }

// Tiles of 16 outputs that a workgroup of the few-row kernel takes, and its estimate
// (more rows than 32). With few rows two from two workgroups a CU on. Four halve the
// loads of bf16 activations, which are most of a workgroup's (64 rows x 12352 outputs, K
// 2048: 15.3 us with two, 12.5 with four; 128 x 8192 16.3 and 12.0).
struct FewForm {
    int tiles;
    float cost;
};
template <bool XMX>
FewForm few_form(size_t M, size_t O, size_t K) {
    const FewCost &c = kFewCost[XMX];
    const float kk = (float)K / 2048.0f;
    const size_t t16 = cdiv(M, 16), nbm = cdiv(t16, cdiv(t16, cdiv(t16, 4)));
    auto cost = [&](float fixed, float per, size_t outputs) {
        return fixed + kk * per * rounds(cdiv(O, outputs) * nbm);
    };
    if (M <= 32) return {cdiv(O, 16) * nbm >= 2 * (size_t)cu_count() ? 2 : 1, 0.0f};
    FewForm f{1, cost(c.fixed, c.one, 16)};
    if (const float two = cost(c.fixed, c.two, 32); two < f.cost) f = {2, two};
    if (const float four = cost(c.fixed4, c.four, 64); !XMX && four < f.cost) f = {4, four};
    return f;
}

// The shape of the many-row kernel to take, or 0: the few-row one.
template <bool XMX>
int wide_shape(size_t M, size_t O, size_t K, float few) {
    const float kk = (float)K / 2048.0f;
    const WideCost &v = kWideCost[XMX];
    const size_t r2 = rounds((size_t)cdiv(O, 128) * cdiv(M, 128));
    // (one tile a CU: in halves of K, 1000 rows x 4096 x 2048 of bf16 25 -> 21 us)
    const float w2 = r2 == 1 ? v.f1 + v.k3 * kk : (r2 / 2) * (v.f2 + v.k2 * kk) + (r2 % 2) * (v.f1 + v.k1 * kk);
    const size_t n4 = (size_t)cdiv(O, 256) * cdiv(M, 256), part = mx_quarters(n4);
    const size_t r4 = rounds(n4 - std::min(n4, part));
    const float w4 = r4 * (v.f4 + v.k4 * kk) + v.fill * std::min((float)r4, (float)n4 / cu_count()) +
                     (part ? v.f1 + v.k1 * kk : 0.0f);
    const size_t r5 = rounds((size_t)cdiv(O, 256) * cdiv(M, 128));
    const float w5 = XMX ? w4 : (r5 / 2) * (v.f6 + v.k6 * kk) + (r5 % 2) * (v.f1 + v.k5 * kk);
    const float least = std::min(std::min(few, w2), std::min(w4, w5));
    return least == few ? 0 : least == w2 ? (r2 == 1 ? 3 : 2) : least == w4 ? 4 : 5;
}

template <bool XMX>
int gemm_run(const uint8_t *w, const uint8_t *ws, const void *x, const uint8_t *xs, size_t ldx,
             uint16_t *y, size_t ldy, size_t M, size_t O, size_t K) {
    if (M == 0 || O == 0) return kOk;
    if (K == 0) {
        k_mx_zero_rows<<<stream_grid(M * O), 256, 0, stream()>>>(y, ldy, O, M * O);
        return launch_check("k_mx_zero_rows");
    }
    const FewForm few = few_form<XMX>(M, O, K);
    if (M > 32) {
        const int shape = wide_shape<XMX>(M, O, K, few.cost);
        if (shape)
            return mx_gemm_wide({w, ws, x, XMX ? xs : nullptr, ldx, y, ldy, (int)M, (int)O, (int)K}, shape);
    }
    const size_t tiles = cdiv(M, 16), nt = cdiv(tiles, cdiv(tiles, 4));
#define FEW(RT, NT, XR) few_run<XMX, RT, NT, XR>(w, ws, x, xs, ldx, y, ldy, M, O, K)
#define FEW2(NT, XR) few.tiles == 2 ? FEW(2, NT, XR) : FEW(1, NT, XR)
    if constexpr (!XMX) {
        if (few.tiles == 4) return nt == 3 ? FEW(4, 3, 4) : FEW(4, 4, 4);
    }
    switch (nt) {
        case 1: return M <= 4 ? FEW2(1, 1) : FEW2(1, 4);
        case 2: return FEW2(2, 4);
        case 3: return FEW2(3, 4);
        default: return FEW2(4, 4);
    }
#undef FEW2
#undef FEW
}

}  // namespace

namespace apus {

int mx_check_dims(size_t M, size_t O, size_t K) {
    if (M > 0x7fffffffu || O > 0x7fffffffu || K > kMxMaxPitch)
        return set_error(kErrUnsupported, "MXFP4 dims past 2^31, or rows past 2^21 elements");
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
        if (ldx > kMxMaxElements / M) return set_error(kErrUnsupported, "%zu rows of pitch %zu", M, ldx);
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
        if (ldx > kMxMaxElements / M) return set_error(kErrUnsupported, "%zu rows of pitch %zu", M, ldx);
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

// mx_wide.hip -- products with MXFP4 weights for many rows: tiles of 64 TO
// outputs x 64 TMM rows, 4 wavefronts (2 x 2), one per SIMD, on the 32-wide
// MFMAs.
#include <stdint.h>

#include <type_traits>

#include "apus_dev.h"
#include "apus_host.h"
#include "mx.h"
#include "mx_dev.h"
#include "tiles.h"

using namespace apus;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pk2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, mx_bf16x2));
}

// 16 (4) bytes a lane from base + off (per lane) to LDS byte lds + 16 (4) *
// lane. live: all ones, or zero for a copy that is counted (vmcnt) but moves
// nothing; the wavefront's lanes are all active here. The two moves (the
// s_nop) are the wait state between the write of M0 and its use.
__device__ __forceinline__ void copy16(uint32_t off, const void *base, uint32_t lds, int live) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    live = __builtin_amdgcn_readfirstlane(live);
    asm volatile("s_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\t"
                 "global_load_lds_dwordx4 %0, %1\n\ts_mov_b64 exec, -1"
                 ::"v"(off), "s"(base), "{m0}"(lds), "s"(live) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t off, const void *base, uint32_t lds, int live) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    live = __builtin_amdgcn_readfirstlane(live);
    asm volatile("s_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\t"
                 "global_load_lds_dword %0, %1\n\ts_mov_b64 exec, -1"
                 ::"v"(off), "s"(base), "{m0}"(lds), "s"(live) : "memory");
}

// p, uniform over the wavefront, in scalar registers
__device__ __forceinline__ const void *uniform(const void *p) {
    const uint64_t a = (uint64_t)p;
    return (const void *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) |
                          (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) << 32);
}

// The tile's outputs, D[o][m]: lane -> m = lane % 32, o = 8 (i / 4) +
// 4 (lane / 32) + i % 4 of each 32 x 32 piece. Through LDS (this wavefront's
// quarter, rows m of 64 TO bytes, 16-byte chunk c at c ^ (m % NCH)), so that
// the stores are 16-byte pieces of whole rows; straight from the accumulators
// where y's rows are not in 16-byte pieces. No copy into sm is in flight and
// no wavefront reads it.
template <int TO, int TMM>
__device__ __forceinline__ void store_tile(char *sm, const f32x16 (&acc)[TO][TMM], uint16_t *y,
                                           size_t ldy, int ow, int mw, int O, int M, int wave,
                                           int lane) {
    if (((ldy | (size_t)O) & 7) != 0 || ((uintptr_t)y & 15) != 0) {
#pragma unroll
        for (int t = 0; t < TO; t++)
#pragma unroll
            for (int u = 0; u < TMM; u++) {
                const int m = mw + u * 32 + (lane & 31);
                if (m >= M) continue;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int o = ow + t * 32 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
                    if (o < O) y[(size_t)m * ldy + o] = f2bf(acc[t][u][i]);
                }
            }
        return;
    }
    constexpr int NCH = 4 * TO, ROW = 64 * TO;           // chunks, bytes of a row
    char *ep = sm + wave * (TMM * 32 * ROW);
#pragma unroll
    for (int t = 0; t < TO; t++)
#pragma unroll
        for (int u = 0; u < TMM; u++) {
            const int m = u * 32 + (lane & 31);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const f32x16 &v = acc[t][u];
                *reinterpret_cast<uint2 *>(ep + m * ROW + (((t * 4 + q) ^ (m & (NCH - 1))) << 4) +
                                           ((lane >> 5) << 3)) =
                    make_uint2(pk2(v[4 * q], v[4 * q + 1]), pk2(v[4 * q + 2], v[4 * q + 3]));
            }
        }
    // (own quarter only: a wavefront's LDS accesses execute in order)
    constexpr int RPI = 64 / NCH;                        // rows an instruction
    const int pc = lane & (NCH - 1), o = ow + pc * 8;
#pragma unroll 8
    for (int i = 0; i < TMM * 32 / RPI; i++) {
        const int m = i * RPI + lane / NCH;
        const uint4 v = *reinterpret_cast<const uint4 *>(ep + m * ROW + ((pc ^ (m & (NCH - 1))) << 4));
        if (o < O && mw + m < M) *reinterpret_cast<uint4 *>(y + (size_t)(mw + m) * ldy + o) = v;
    }
}

// ---- both operands MXFP4 -----------------------------------------------------
// A stage is 256 k: 128 bytes of codes and 8 of scales per row, BO weight rows,
// then BM activation rows, double-buffered in LDS. 16-byte chunk c (block c of
// the stage) of row r lies at slot c ^ (r % 8), so that the 8 rows of one LDS
// read phase hit 8 distinct slots. MFMA step s takes 64 k: lane (row l % 32,
// half g = l / 32) chunk 2 s + g, and the scale byte of the same number.
// Blocks past K (in the last stage): zero codes and scale 1 on both sides.
// AL: rows of scales are 4-byte aligned (K a multiple of 128) and are copied
// like the codes; else they pass through registers, a byte at a time.
constexpr int kMxStage = 256;

template <int TO, int TMM, bool AL>
__global__ __launch_bounds__(256, TO * TMM <= 4 ? 2 : 1) void k_mx_gemm_wide(
    const uint8_t *__restrict__ w, const uint8_t *__restrict__ ws, const uint8_t *__restrict__ x,
    const uint8_t *__restrict__ xs, uint16_t *__restrict__ y, size_t ldy, int M, int O, int K) {
    constexpr int BO = 64 * TO, BM = 64 * TMM, ROWS = BO + BM;
    constexpr int PB = BO * 128, SB = ROWS * 128, SCB = ROWS * 8;
    constexpr int PPW = ROWS / 32;                       // code copies a wavefront and stage
    constexpr int SPW = AL ? ROWS / 128 : 0;             // scale copies
    constexpr int SPT = AL ? 1 : ROWS / 32;              // else scale bytes a thread
    constexpr int NF = TO * TMM, NR = TO + TMM;
    static_assert(ROWS % 128 == 0, "copies must split evenly over the wavefronts");
    __shared__ __attribute__((aligned(16))) char sm[2 * (SB + SCB)];
    char *const scales = sm + 2 * SB;
    const int nbo = (O + BO - 1) / BO, nbm = (M + BM - 1) / BM;
    int ob, mb;
    tile_of(blockIdx.x, nbo, nbm, ob, mb);
    if (ob >= nbo) return;                               // (the grid is a multiple of 8)
    const int o0 = ob * BO, m0 = mb * BM;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wo = wave >> 1, wm = wave & 1, g = lane >> 5;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void *)sm);
    const uint32_t kc = (uint32_t)K / 2, ks = (uint32_t)K / kMxBlock;   // bytes of a row
    const int nk = (K + kMxStage - 1) / kMxStage;
    // tile-relative, so that 32-bit offsets do (rows past O or M read the last
    // row; their products are not stored)
    const uint8_t *const wt = w + (size_t)o0 * kc, *const xt = x + (size_t)m0 * kc;
    const uint8_t *const wst = ws + (size_t)o0 * ks, *const xst = xs + (size_t)m0 * ks;
    auto row_of = [&](int r) {                           // stage row -> row of its operand's tile
        return r < BO ? min(r, O - 1 - o0) : min(r - BO, M - 1 - m0);
    };
    uint32_t roff[PPW], soff[AL ? SPW : 1];
    const void *rbuf[PPW], *sbuf[AL ? SPW : 1];
#pragma unroll
    for (int i = 0; i < PPW; i++) {
        const int p = wave * PPW + i;
        roff[i] = row_of(p * 8 + (lane >> 3)) * kc;
        rbuf[i] = uniform(p < BO / 8 ? wt : xt);
    }
#pragma unroll
    for (int i = 0; i < SPW; i++) {
        const int p = wave * SPW + i;
        soff[i] = row_of(p * 32 + (lane >> 1)) * ks;
        sbuf[i] = uniform(p < BO / 32 ? wst : xst);
    }
    const uint32_t cg = ((lane & 7) ^ (lane >> 3)) * 16, sg = (lane & 1) * 4;
    auto copy_codes = [&](int i, int st, int live) {
        uint32_t at = st * 128 + cg;
        at = at < kc ? at : 0;                           // (past the row's end: masked when read)
        const int p = wave * PPW + i;
        copy16(roff[i] + at, rbuf[i], lds0 + (st & 1) * SB + p * 1024, live);
    };
    auto copy_scales = [&](int i, int st, int live) {
        uint32_t at = st * 8 + sg;
        at = at < ks ? at : 0;
        const int p = wave * SPW + i;
        copy4(soff[i] + at, sbuf[i], lds0 + 2 * SB + (st & 1) * SCB + p * 256, live);
    };
    // the unaligned form: bytes (32 rows of 8 an instruction of the workgroup)
    uint8_t sbyte[SPT];
    auto load_bytes = [&](int st) {
        if (AL) return;
        const uint32_t at = (uint32_t)st * 8 + (lane & 7);
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int r = i * 32 + wave * 8 + (lane >> 3);
            sbyte[i] = (r < BO ? wst : xst)[row_of(r) * ks + (at < ks ? at : 0)];
        }
    };
    auto put_bytes = [&](int st) {
        if (AL) return;
#pragma unroll
        for (int i = 0; i < SPT; i++)
            scales[(st & 1) * SCB + (i * 32 + wave * 8 + (lane >> 3)) * 8 + (lane & 7)] = sbyte[i];
    };
    f32x16 acc[TO][TMM];
#pragma unroll
    for (int t = 0; t < TO; t++)
#pragma unroll
        for (int u = 0; u < TMM; u++) acc[t][u] = f32x16{};
    struct Frag {
        u32x4 a[TO], b[TMM];
    };
    struct Scale {
        uint32_t a[TO][2], b[TMM][2];
    };
    const uint32_t rbase = (lane & 31) * 128 + ((g ^ (lane & 7)) << 4);
    auto rd1 = [&](int st, int s, int j, Frag &f) {      // in the MFMAs' order: a[0], b[0..], a[1..]
        const char *p = sm + (st & 1) * SB + (rbase ^ (s << 5));
        if (j == 0 || j > TMM) {
            const int t = j == 0 ? 0 : j - TMM;
            f.a[t] = *reinterpret_cast<const u32x4 *>(p + (wo * TO + t) * 4096);
        } else {
            f.b[j - 1] = *reinterpret_cast<const u32x4 *>(p + PB + (wm * TMM + j - 1) * 4096);
        }
    };
    // a row's 8 scale bytes as two words, shifted so that byte 0 (2) of word
    // s / 2 is this lane half's in an even (odd) step s
    auto rd_scales = [&](int st, Scale &c) {
        const char *p = scales + (st & 1) * SCB + (lane & 31) * 8;
#pragma unroll
        for (int t = 0; t < TO; t++) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + (wo * TO + t) * 256);
            c.a[t][0] = v.x >> (8 * g);
            c.a[t][1] = v.y >> (8 * g);
        }
#pragma unroll
        for (int u = 0; u < TMM; u++) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + BO * 8 + (wm * TMM + u) * 256);
            c.b[u][0] = v.x >> (8 * g);
            c.b[u][1] = v.y >> (8 * g);
        }
    };
    using no = std::false_type;
    using yes = std::true_type;
    // One step: its MFMAs on f, with the next step's operand reads into gn
    // (READ: step s2 of stage rst) and the copies of stage cst (COPY) fenced in
    // place between them.
    auto step = [&](auto sc, const Frag &f, const Scale &c, Frag &gn, auto read, int rst, int s2,
                    auto cpy, int cst, int live) {
        constexpr int S = decltype(sc)::value;
        constexpr bool READ = decltype(read)::value, COPY = decltype(cpy)::value;
        int r = 0, d = 0;
#pragma unroll
        for (int i = 0; i < NF; i++) {
            const int t = i / TMM, u = i % TMM;
            const u32x4 &a = f.a[t], &b = f.b[u];
            const mx_i32x8 av{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
            const mx_i32x8 bv{(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
            acc[t][u] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                av, bv, acc[t][u], 4, 4, S % 2 * 2, (int)c.a[t][S / 2], S % 2 * 2, (int)c.b[u][S / 2]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (; READ && r < NR && (i == NF - 1 || r * NF * 3 <= i * NR * 4); r++) rd1(rst, s2, r, gn);
#pragma unroll
            for (; COPY && d < PPW && d * NF < (i + 1) * PPW; d++) copy_codes(d, cst, live);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using s0 = std::integral_constant<int, 0>;
    using s1 = std::integral_constant<int, 1>;
    using s2 = std::integral_constant<int, 2>;
    using s3 = std::integral_constant<int, 3>;
    Frag f0, f1;
    Scale c0, c1;
#pragma unroll
    for (int st = 0; st < 2; st++) {
        const int live = (st - nk) >> 31;
        load_bytes(min(st, nk - 1));
        put_bytes(st);
#pragma unroll
        for (int i = 0; i < SPW; i++) copy_scales(i, st, live);
#pragma unroll
        for (int i = 0; i < PPW; i++) copy_codes(i, st, live);
    }
    if (nk >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PPW + SPW) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NR; j++) rd1(0, 0, j, f0);
    rd_scales(0, c0);
    for (int kt = 0; kt < nk - 1; kt++) {
        load_bytes(min(kt + 2, nk - 1));
        step(s0{}, f0, c0, f1, yes{}, kt, 1, no{}, 0, 0);
        step(s1{}, f1, c0, f0, yes{}, kt, 2, no{}, 0, 0);
        step(s2{}, f0, c0, f1, yes{}, kt, 3, no{}, 0, 0);
        // every operand of this stage has been read, by this wavefront (it
        // waited for f1) and after the barrier by all, and the next stage's
        // copies, the only ones in flight, have landed: stage kt + 2 goes into
        // this stage's slot
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        rd_scales(kt + 1, c1);
        put_bytes(kt + 2);
        const int live = (kt + 2 - nk) >> 31;
#pragma unroll
        for (int i = 0; i < SPW; i++) copy_scales(i, kt + 2, live);
        step(s3{}, f1, c0, f0, yes{}, kt + 1, 0, yes{}, kt + 2, live);
        c0 = c1;
    }
    // the last stage, with what lies past K masked
    const int left = K - (nk - 1) * kMxStage;
    if (left < kMxStage) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            // words of two steps: their blocks 4 h + g and 4 h + 2 + g
            const bool d0 = (4 * h + g) * 32 >= left, d1 = (4 * h + 2 + g) * 32 >= left;
            auto fix = [&](uint32_t v) {
                return (d0 ? 127u : v & 0xffu) | ((d1 ? 127u : (v >> 16) & 0xffu) << 16);
            };
#pragma unroll
            for (int t = 0; t < TO; t++) c0.a[t][h] = fix(c0.a[t][h]);
#pragma unroll
            for (int u = 0; u < TMM; u++) c0.b[u][h] = fix(c0.b[u][h]);
        }
    }
    auto mask = [&](Frag &f, int s) {
        if ((2 * s + g) * 32 < left) return;
#pragma unroll
        for (int t = 0; t < TO; t++) f.a[t] = u32x4{};
#pragma unroll
        for (int u = 0; u < TMM; u++) f.b[u] = u32x4{};
    };
    mask(f0, 0);
    step(s0{}, f0, c0, f1, yes{}, nk - 1, 1, no{}, 0, 0);
    mask(f1, 1);
    step(s1{}, f1, c0, f0, yes{}, nk - 1, 2, no{}, 0, 0);
    mask(f0, 2);
    step(s2{}, f0, c0, f1, yes{}, nk - 1, 3, no{}, 0, 0);
    mask(f1, 3);
    step(s3{}, f1, c0, f0, no{}, 0, 0, no{}, 0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    store_tile<TO, TMM>(sm, acc, y, ldy, o0 + wo * TO * 32, m0 + wm * TMM * 32, O, M, wave, lane);
}

template <int TO, int TMM>
int launch_mx_wide(const uint8_t *w, const uint8_t *ws, const uint8_t *x, const uint8_t *xs,
                   uint16_t *y, size_t ldy, int M, int O, int K) {
    const unsigned grid = tile_grid((int)cdiv(O, 64 * TO), (int)cdiv(M, 64 * TMM));
    const bool al = K % 128 == 0 && ((uintptr_t)ws | (uintptr_t)xs) % 4 == 0;
    APUS_TIMED("k_mx_gemm_wide",
               if (al) k_mx_gemm_wide<TO, TMM, true><<<grid, 256, 0, stream()>>>(w, ws, x, xs, y, ldy, M, O, K);
               else k_mx_gemm_wide<TO, TMM, false><<<grid, 256, 0, stream()>>>(w, ws, x, xs, y, ldy, M, O, K));
    return launch_check("k_mx_gemm_wide");
}

// ---- bf16 activations ----------------------------------------------------------
// A stage is 64 k of the activations, 128 bytes a row; the weights come in
// chunks of 256 k (128 bytes of codes and 8 of scales a row), both double-
// buffered in LDS. A quarter of a chunk is copied with each stage. In stage t
// of a chunk, lane (row l % 32, half g) takes the weights' block 2 t + g, one
// 16-byte read for the whole stage, and MFMA step j its codes 8 j .., widened
// to bf16 in registers, with the activations of the same k: 16-byte chunk
// 4 g + j of their row. LDS thus gives a stage's weights once, not once per 16
// k as bf16 weights would need.
constexpr int kMx16Stage = 64;

template <int TO, int TMM, bool AL>
__global__ __launch_bounds__(256, TO * TMM <= 4 ? 2 : 1) void k_mx_gemm_wide16(
    const uint8_t *__restrict__ w, const uint8_t *__restrict__ ws, const uint16_t *__restrict__ x,
    size_t ldx, uint16_t *__restrict__ y, size_t ldy, int M, int O, int K) {
    constexpr int BO = 64 * TO, BM = 64 * TMM;
    constexpr int XB = BM * 128, WB = BO * 128, SCB = BO * 8;
    constexpr int XPW = BM / 32, WPW = BO / 128;         // copies a wavefront and stage
    constexpr int SPW = AL ? BO / 128 : 0;               // and chunk
    constexpr int SPT = AL ? 1 : BO / 32;
    constexpr int NF = TO * TMM;
    __shared__ __attribute__((aligned(16))) char sm[2 * (XB + WB + SCB)];
    constexpr int W0 = 2 * XB, S0 = 2 * (XB + WB);
    const int nbo = (O + BO - 1) / BO, nbm = (M + BM - 1) / BM;
    int ob, mb;
    tile_of(blockIdx.x, nbo, nbm, ob, mb);
    if (ob >= nbo) return;                               // (the grid is a multiple of 8)
    const int o0 = ob * BO, m0 = mb * BM;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wo = wave >> 1, wm = wave & 1, g = lane >> 5;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void *)sm);
    const uint32_t kc = (uint32_t)K / 2, ks = (uint32_t)K / kMxBlock, kx = (uint32_t)K * 2;
    const int nk = (K + kMx16Stage - 1) / kMx16Stage, nch = (nk + 3) / 4;
    const uint8_t *const wst = ws + (size_t)o0 * ks;
    const void *const wt = uniform(w + (size_t)o0 * kc), *const wsb = uniform(wst),
               *const xt = uniform(x + (size_t)m0 * ldx);
    const uint32_t cg = ((lane & 7) ^ (lane >> 3)) * 16, sg = (lane & 1) * 4;
    uint32_t xoff[XPW];
#pragma unroll
    for (int i = 0; i < XPW; i++)
        xoff[i] = (uint32_t)min((wave * XPW + i) * 8 + (lane >> 3), M - 1 - m0) * (uint32_t)(ldx * 2);
    auto copy_x = [&](int i, int st, int live) {
        uint32_t at = st * 128 + cg;
        at = at < kx ? at : 0;                           // (past the row's end: masked when read)
        copy16(xoff[i] + at, xt, lds0 + (st & 1) * XB + (wave * XPW + i) * 1024, live);
    };
    // quarter q of chunk c: 64 TO / 4 rows
    auto copy_w = [&](int i, int c, int q, int live) {
        uint32_t at = c * 128 + cg;
        at = at < kc ? at : 0;
        const int p = q * (BO / 32) + wave * WPW + i;
        const uint32_t row = min(p * 8 + (lane >> 3), O - 1 - o0);
        copy16(row * kc + at, wt, lds0 + W0 + (c & 1) * WB + p * 1024, live);
    };
    auto copy_scales = [&](int i, int c, int live) {
        uint32_t at = c * 8 + sg;
        at = at < ks ? at : 0;
        const int p = wave * SPW + i;
        const uint32_t row = min(p * 32 + (lane >> 1), O - 1 - o0);
        copy4(row * ks + at, wsb, lds0 + S0 + (c & 1) * SCB + p * 256, live);
    };
    uint8_t sbyte[SPT];
    auto load_bytes = [&](int c) {
        if (AL) return;
        const uint32_t at = (uint32_t)c * 8 + (lane & 7);
#pragma unroll
        for (int i = 0; i < SPT; i++)
            sbyte[i] = wst[(uint32_t)min(i * 32 + wave * 8 + (lane >> 3), O - 1 - o0) * ks + (at < ks ? at : 0)];
    };
    auto put_bytes = [&](int c) {
        if (AL) return;
#pragma unroll
        for (int i = 0; i < SPT; i++)
            sm[S0 + (c & 1) * SCB + (i * 32 + wave * 8 + (lane >> 3)) * 8 + (lane & 7)] = sbyte[i];
    };
    // what is copied at the end of stage kt: the activations of stage kt + 2,
    // a quarter of chunk (kt + 1) / 4 + 1 (its slot's last reader was the
    // chunk before (kt + 1) / 4's)
    auto copy_scales_at = [&](int kt) {
        const int c = (kt + 1) / 4 + 1;
        if (((kt + 1) & 3) == 0 && c < nch) {
#pragma unroll
            for (int i = 0; i < SPW; i++) copy_scales(i, c, -1);
            load_bytes(c);
            put_bytes(c);
        }
    };
    auto copy_at = [&](int i, int kt) {
        if (i < XPW) {
            copy_x(i, kt + 2, (kt + 2 - nk) >> 31);
        } else {
            const int c = (kt + 1) / 4 + 1;
            copy_w(i - XPW, c, (kt + 1) & 3, (c - nch) >> 31);
        }
    };
    f32x16 acc[TO][TMM];
#pragma unroll
    for (int t = 0; t < TO; t++)
#pragma unroll
        for (int u = 0; u < TMM; u++) acc[t][u] = f32x16{};
    struct Raw {
        u32x4 v[TO];
        uint32_t s[TO];
    };
    struct Frag {
        mx_bf16x8 a[TO], b[TMM];
    };
    const uint32_t rrow = (lane & 31) * 128;
    auto rd_raw = [&](int st, int t, Raw &f) {
        const int c = st >> 2, b = 2 * (st & 3) + g;
        const char *p = sm + W0 + (c & 1) * WB + (wo * TO + t) * 4096 + rrow + ((b ^ (lane & 7)) << 4);
        f.v[t] = *reinterpret_cast<const u32x4 *>(p);
        f.s[t] = (uint8_t)sm[S0 + (c & 1) * SCB + ((wo * TO + t) * 32 + (lane & 31)) * 8 + b];
    };
    auto rd_x = [&](int st, int j, int u, Frag &f) {
        const char *p = sm + (st & 1) * XB + (wm * TMM + u) * 4096 + rrow + (((4 * g + j) ^ (lane & 7)) << 4);
        f.b[u] = *reinterpret_cast<const mx_bf16x8 *>(p);
    };
    using no = std::false_type;
    using yes = std::true_type;
    // One step: its MFMAs on f; between them, fenced in place, step j2's
    // operands into fn (from wr; READ: activations of stage rst), in the last
    // step of a stage first the next stage's weights into wn (RAW), and the
    // copies after stage kt (COPY).
    auto step = [&](const Frag &f, Frag &fn, auto read, int rst, auto j2, const Raw &wr, auto raw,
                    Raw &wn, auto cpy, int kt) {
        constexpr int J2 = decltype(j2)::value;
        constexpr bool READ = decltype(read)::value, RAW = decltype(raw)::value, COPY = decltype(cpy)::value;
        constexpr int NC = XPW + WPW;
        if (RAW) {
#pragma unroll
            for (int t = 0; t < TO; t++) rd_raw(rst, t, wn);
        }
        int r = 0, a = 0, d = 0;
#pragma unroll
        for (int i = 0; i < NF; i++) {
            acc[i / TMM][i % TMM] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                f.a[i / TMM], f.b[i % TMM], acc[i / TMM][i % TMM], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            // reads under the first half of the MFMAs, widening under the second
#pragma unroll
            for (; READ && r < TMM && r * NF < (i + 1) * TMM * 2; r++) rd_x(rst, J2, r, fn);
#pragma unroll
            for (; READ && a < TO && i >= NF / 2 - 1 && a * NF < (i + 1 - NF / 2) * TO * 2; a++) {
                const uint32_t c = (RAW ? wn : wr).v[a][J2];
                fn.a[a] = mx_widen(c, (RAW ? wn : wr).s[a]);
            }
#pragma unroll
            for (; COPY && d < NC && d * NF < (i + 1) * NC; d++) copy_at(d, kt);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (; READ && a < TO; a++) {
            const uint32_t c = (RAW ? wn : wr).v[a][J2];
            fn.a[a] = mx_widen(c, (RAW ? wn : wr).s[a]);
        }
    };
    using i0 = std::integral_constant<int, 0>;
    using i1 = std::integral_constant<int, 1>;
    using i2 = std::integral_constant<int, 2>;
    using i3 = std::integral_constant<int, 3>;
    // stages 0 and 1, chunk 0 and the first quarter of chunk 1
#pragma unroll
    for (int c = 0; c < 2; c++) {
        if (c < nch) {
            load_bytes(c);
            put_bytes(c);
#pragma unroll
            for (int i = 0; i < SPW; i++) copy_scales(i, c, -1);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int i = 0; i < WPW; i++) copy_w(i, 0, q, -1);
#pragma unroll
    for (int i = 0; i < XPW; i++) copy_x(i, 0, -1);
#pragma unroll
    for (int i = 0; i < XPW + WPW; i++) copy_at(i, -1);
    if (nk > 1 && nch > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(XPW + WPW) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    Raw r0, r1;
    Frag f0, f1;
#pragma unroll
    for (int t = 0; t < TO; t++) rd_raw(0, t, r0);
#pragma unroll
    for (int u = 0; u < TMM; u++) rd_x(0, 0, u, f0);
#pragma unroll
    for (int t = 0; t < TO; t++) {
        const uint32_t c = r0.v[t][0];
        f0.a[t] = mx_widen(c, r0.s[t]);
    }
    for (int kt = 0; kt < nk - 1; kt++) {
        step(f0, f1, yes{}, kt, i1{}, r0, no{}, r1, no{}, 0);
        step(f1, f0, yes{}, kt, i2{}, r0, no{}, r1, no{}, 0);
        step(f0, f1, yes{}, kt, i3{}, r0, no{}, r1, no{}, 0);
        // this stage's operands have been read by all after the barrier, and
        // everything in flight, the next stage's copies, has landed
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        copy_scales_at(kt);
        step(f1, f0, yes{}, kt + 1, i0{}, r0, yes{}, r1, yes{}, kt);
        r0 = r1;
    }
    // the last stage; with an odd number of blocks half of it lies past K
    const bool odd = K % kMx16Stage != 0;
    auto mask = [&](Frag &f) {
        if (!odd || g == 0) return;
#pragma unroll
        for (int t = 0; t < TO; t++) f.a[t] = mx_bf16x8{};
#pragma unroll
        for (int u = 0; u < TMM; u++) f.b[u] = mx_bf16x8{};
    };
    mask(f0);
    step(f0, f1, yes{}, nk - 1, i1{}, r0, no{}, r1, no{}, 0);
    mask(f1);
    step(f1, f0, yes{}, nk - 1, i2{}, r0, no{}, r1, no{}, 0);
    mask(f0);
    step(f0, f1, yes{}, nk - 1, i3{}, r0, no{}, r1, no{}, 0);
    mask(f1);
    step(f1, f0, no{}, 0, i0{}, r0, no{}, r1, no{}, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    store_tile<TO, TMM>(sm, acc, y, ldy, o0 + wo * TO * 32, m0 + wm * TMM * 32, O, M, wave, lane);
}

template <int TO, int TMM>
int launch_mx_wide16(const uint8_t *w, const uint8_t *ws, const uint16_t *x, size_t ldx,
                     uint16_t *y, size_t ldy, int M, int O, int K) {
    const unsigned grid = tile_grid((int)cdiv(O, 64 * TO), (int)cdiv(M, 64 * TMM));
    const bool al = K % 128 == 0 && (uintptr_t)ws % 4 == 0;
    APUS_TIMED("k_mx_gemm_wide16",
               if (al) k_mx_gemm_wide16<TO, TMM, true><<<grid, 256, 0, stream()>>>(w, ws, x, ldx, y, ldy, M, O, K);
               else k_mx_gemm_wide16<TO, TMM, false><<<grid, 256, 0, stream()>>>(w, ws, x, ldx, y, ldy, M, O, K));
    return launch_check("k_mx_gemm_wide16");
}

}  // namespace

namespace apus {

int mx_gemm_wide(const uint8_t *w, const uint8_t *ws, const uint8_t *x, const uint8_t *xs,
                 uint16_t *y, size_t ldy, int M, int O, int K, int shape) {
    return shape == 4 ? launch_mx_wide<4, 4>(w, ws, x, xs, y, ldy, M, O, K)
                      : launch_mx_wide<2, 2>(w, ws, x, xs, y, ldy, M, O, K);
}

int mx_gemm_wide16(const uint8_t *w, const uint8_t *ws, const uint16_t *x, size_t ldx, uint16_t *y,
                   size_t ldy, int M, int O, int K, int shape) {
    return shape == 4 ? launch_mx_wide16<4, 4>(w, ws, x, ldx, y, ldy, M, O, K)
                      : launch_mx_wide16<2, 2>(w, ws, x, ldx, y, ldy, M, O, K);
}

}  // namespace apus

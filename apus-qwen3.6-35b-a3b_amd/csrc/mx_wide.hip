// mx_wide.hip -- products y[m][o] = rnd(sum_k w[o][k] x[m][k]) with MXFP4 weights for
// many rows: tiles of 64 TO outputs x 64 TMM rows, 4 wavefronts (2 x 2), one per SIMD,
// on the 32-wide MFMAs; w and x are copied to LDS without registers and read there.
//
// 4096 rows x 12352 outputs, K 2048, 207 Gflop: bf16 x 175 us, 1.18 Pflop/s (a large
// bf16 library product reaches 1.32 here); MXFP4 x 78 us, 2.6 Pflop/s. With K 8192, 590
// and 223 us for 825 Gflop, 1.40 and 3.7 Pflop/s. There the chip's MFMA rate under load
// is the bound: the same loop without copies and LDS reads takes 195 of the 223 us.
// With K 2048 the 101 MB of y count beside it.
#include <stdint.h>

#include <type_traits>

#include "apus_dev.h"
#include "apus_host.h"
#include "mx.h"
#include "mx_dev.h"
#include "mx_reads.h"
#include "tiles.h"

using namespace apus;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pk2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, mx_bf16x2));
}

// 16 bytes a lane from base + off (per lane) to LDS byte lds + 16 * lane. live:
// all ones, or zero for a copy past the last stage, into a slot that nobody reads:
// it counts (vmcnt) like the others, so that what a wait leaves in flight is the
// same all along. The s_nop is the wait state between the write of M0 and its use.
__device__ __forceinline__ void copy16(uint32_t off, const void *base, uint32_t lds, int live) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off & (uint32_t)live), "s"(base), "{m0}"(lds)
                 : "memory");
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
// where y's rows are not in 16-byte pieces. Stores that keep no copy in the L2
// leave it to the operands (4096 rows x 12352 outputs, K 2048, MXFP4 activations:
// 103 us with ordinary ones, now 88; 2048 x 8192: 31, now 29). No copy into sm is in
// flight and no wavefront reads it.
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
        const u32x4 v = *reinterpret_cast<const u32x4 *>(ep + m * ROW + ((pc ^ (m & (NCH - 1))) << 4));
        if (o < O && mw + m < M)
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(y + (size_t)(mw + m) * ldy + o));
    }
}

// ---- both operands MXFP4 -----------------------------------------------------
// A stage is 256 k: 128 bytes of codes and 8 of scales per row, BO weight rows,
// then BM activation rows, double-buffered in LDS. 16-byte chunk c (block c of
// the stage) of row r lies at slot c ^ (r % 8), so that the 8 rows of one LDS
// read phase hit 8 distinct slots. MFMA step s takes 64 k: lane (row l % 32,
// half g = l / 32) chunk 2 s + g, and the scale byte of the same number.
// Blocks past the group's k (in its last stage): zero codes and scale 1 on both sides.
// Scales come for two stages at a time, through registers.
constexpr int kMxStage = 256;

template <int TO, int TMM>
constexpr int kMxLds = 2 * 64 * (TO + TMM) * (kMxStage / 2 + 16);
template <int TO, int TMM>
__device__ __forceinline__ void mx_tile(char *sm, const MxProduct &a, int o0, int m0, const KShare &share,
                                        f32x16 (&acc)[TO][TMM]) {
    constexpr int BO = 64 * TO, BM = 64 * TMM, ROWS = BO + BM;
    constexpr int PB = BO * 128, SB = ROWS * 128;
    constexpr int SCB = ROWS * 16;
    constexpr int PPW = ROWS / 32;                       // code copies a wavefront and stage
    constexpr int SPT = ROWS / 256;                      // rows of scales a thread
    constexpr int NF = TO * TMM, NR = TO + TMM;
    static_assert(ROWS % 256 == 0, "rows must split evenly over the threads");
    static_assert(2 * (SB + SCB) == kMxLds<TO, TMM>);
    char *const scales = sm + 2 * SB;
    const int M = a.M, O = a.O, k0 = share.k0, K = share.n, nk = share.nk;    // K: of this group
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int wo = wave >> 1, wm = wave & 1, g = lane >> 5;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void *)sm);
    const uint32_t kc = (uint32_t)a.K / 2, ks = (uint32_t)a.K / kMxBlock;   // bytes of a row
    const uint32_t kleft = (uint32_t)K / 2, sc0 = (uint32_t)k0 / kMxBlock;   // of the group's k; its first scale
    const int nsc = (min(nk, (K + kMxStage - 1) / kMxStage) + 1) / 2;
    // tile-relative, so that 32-bit offsets do (rows past O or M read the last
    // row; their products are not stored)
    const uint8_t *const wt = a.w + (size_t)o0 * kc + k0 / 2;
    const uint8_t *const xt = (const uint8_t *)a.x + (size_t)m0 * kc + k0 / 2;
    const uint8_t *const wst = a.ws + (size_t)o0 * ks;
    const uint8_t *const xst = a.xs + (size_t)m0 * ks;
    auto row_of = [&](int r) {                           // stage row -> row of its operand's tile
        return r < BO ? min(r, O - 1 - o0) : min(r - BO, M - 1 - m0);
    };
    uint32_t roff[PPW];
    const void *rbuf[PPW];
#pragma unroll
    for (int i = 0; i < PPW; i++) {
        const int p = wave * PPW + i;
        roff[i] = row_of(p * 8 + (lane >> 3)) * kc;
        rbuf[i] = uniform(p < BO / 8 ? wt : xt);
    }
    const uint32_t cg = ((lane & 7) ^ (lane >> 3)) * 16;
    auto copy_codes = [&](int i, int st, int live) {
        uint32_t at = st * 128 + cg;
        at = at < kleft ? at : 0;                           // (past the row's end: masked when read)
        const int p = wave * PPW + i;
        copy16(roff[i] + at, rbuf[i], lds0 + (st & 1) * SB + p * 1024, live);
    };
    // scales of this thread's rows, through registers
    const int tid = threadIdx.x & 255;
    RowScales sreg[SPT];
    auto load_scales = [&](int c) {
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int r = i * 256 + tid;
            sreg[i].load((r < BO ? wst : xst) + (size_t)row_of(r) * ks, sc0 + 16 * c, ks);
        }
    };
    auto put_scales = [&](int c) {
#pragma unroll
        for (int i = 0; i < SPT; i++)
            *reinterpret_cast<u32x4 *>(scales + (c & 1) * SCB + (i * 256 + tid) * 16) = sreg[i].v;
    };
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
        const char *p = scales + (st >> 1 & 1) * SCB + (st & 1) * 8 + (lane & 31) * 16;
#pragma unroll
        for (int t = 0; t < TO; t++) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + (wo * TO + t) * 512);
            c.a[t][0] = v.x >> (8 * g);
            c.a[t][1] = v.y >> (8 * g);
        }
#pragma unroll
        for (int u = 0; u < TMM; u++) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + BO * 16 + (wm * TMM + u) * 512);
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
    // the first scales go with the copies where they are whole 16 bytes (a wait for
    // registers here is one for all the copies)
    const bool whole = scales_whole(ks, sc0, a.ws, a.xs);
    if (whole) {
#pragma unroll
        for (int i = 0; i < SPT; i++) {
            const int p = wave * SPT + i;                // (64 rows)
            copy16(row_of(p * 64 + lane) * ks + sc0, uniform(p * 64 < BO ? wst : xst), lds0 + 2 * SB + p * 1024, -1);
        }
    } else {
        load_scales(0);
    }
#pragma unroll
    for (int st = 0; st < 2; st++) {
#pragma unroll
        for (int i = 0; i < PPW; i++) copy_codes(i, st, (st - nk) >> 31);
    }
    if (!whole) put_scales(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PPW) : "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NR; j++) rd1(0, 0, j, f0);
    rd_scales(0, c0);
    for (int kt = 0; kt < nk - 1; kt++) {
        if ((kt & 1) == 0) load_scales(min(kt / 2 + 1, nsc - 1));
        step(s0{}, f0, c0, f1, yes{}, kt, 1, no{}, 0, 0);
        step(s1{}, f1, c0, f0, yes{}, kt, 2, no{}, 0, 0);
        step(s2{}, f0, c0, f1, yes{}, kt, 3, no{}, 0, 0);
        // every operand of this stage has been read, by this wavefront (it
        // waited for f1) and after the barrier by all, and the next stage's
        // copies have landed: stage kt + 2 goes into this stage's slot
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        rd_scales(kt + 1, c1);
        if ((kt & 1) == 0) put_scales(kt / 2 + 1);
        const int live = (kt + 2 - nk) >> 31;
        step(s3{}, f1, c0, f0, yes{}, kt + 1, 0, yes{}, kt + 2, live);
        c0 = c1;
    }
    // the last stage, with what lies past the group's k masked
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
}

// ---- bf16 activations ----------------------------------------------------------
// A stage is 64 k of the activations, 128 bytes a row; the weights come in
// chunks of 2 RB k (RB bytes of codes a row), their scales of 512 k, all double-
// buffered in LDS. A part of a chunk is copied with each of its stages. In stage t
// of a chunk, lane (row l % 32, half g) takes the weights' block 2 t + g, one
// 16-byte read for the whole stage, and MFMA step j its codes 8 j .., widened
// to bf16 in registers, with the activations of the same k: 16-byte chunk
// 4 g + j of their row. LDS thus gives a stage's weights once, not once per 16
// k as bf16 weights would need.
constexpr int kMx16Stage = 64;

// The place of 16-byte chunk c of row r, rows RB bytes long, so that rows read side by
// side are in many banks.
template <int RB>
__device__ __forceinline__ int slot_of(int c, int r) { return c ^ (RB == 128 ? r & 7 : r >> 2 & 3); }

template <int TO, int TMM, int RB>
constexpr int kMx16Lds = 2 * 64 * (TMM * kMx16Stage * 2 + TO * (RB + 16));
template <int TO, int TMM, int RB>
__device__ __forceinline__ void mx16_tile(char *sm, const MxProduct &a, int o0, int m0, const KShare &share,
                                          f32x16 (&acc)[TO][TMM]) {
    constexpr int BO = 64 * TO, BM = 64 * TMM;
    constexpr int XB = BM * 128, WB = BO * RB, SCB = BO * 16;
    constexpr int CH = RB / 16, CPS = RB / 32;           // 16-byte pieces of a row, stages of a chunk
    constexpr int XPW = BM / 32, WPW = BO / 128;         // copies a wavefront and stage
    constexpr int NF = TO * TMM;
    constexpr int W0 = 2 * XB, S0 = 2 * (XB + WB);
    static_assert(S0 + 2 * SCB == (kMx16Lds<TO, TMM, RB>) && BO <= 256);
    const int M = a.M, O = a.O, k0 = share.k0, K = share.n, nk = share.nk;    // K: of this group
    const size_t ldx = a.ldx;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int tid = threadIdx.x & 255;
    const int wo = wave >> 1, wm = wave & 1, g = lane >> 5;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void *)sm);
    const uint32_t kc = (uint32_t)a.K / 2, ks = (uint32_t)a.K / kMxBlock;   // bytes of a row
    const uint32_t kleft = (uint32_t)K / 2, kx = (uint32_t)K * 2, sc0 = (uint32_t)k0 / kMxBlock;      // of the group's k; its first scale
    const int nch = (nk + CPS - 1) / CPS, nsc = (min(nk, (K + kMx16Stage - 1) / kMx16Stage) + 7) / 8;
    const uint8_t *const wrow = a.ws + (size_t)(o0 + min(tid % BO, O - 1 - o0)) * ks;
    const void *const wt = uniform(a.w + (size_t)o0 * kc + k0 / 2),
               *const xt = uniform((const uint16_t *)a.x + (size_t)m0 * ldx + k0);
    const uint32_t cg = slot_of<128>(lane & 7, lane >> 3) * 16, wg = slot_of<RB>(lane % CH, lane / CH) * 16;
    uint32_t xoff[XPW];
#pragma unroll
    for (int i = 0; i < XPW; i++)
        xoff[i] = (uint32_t)min((wave * XPW + i) * 8 + (lane >> 3), M - 1 - m0) * (uint32_t)(ldx * 2);
    auto copy_x = [&](int i, int st, int live) {
        uint32_t at = st * 128 + cg;
        at = at < kx ? at : 0;                           // (past the row's end: masked when read)
        copy16(xoff[i] + at, xt, lds0 + (st & 1) * XB + (wave * XPW + i) * 1024, live);
    };
    // part q of chunk c: its rows in CPS parts
    auto copy_w = [&](int i, int c, int q, int live) {
        uint32_t at = c * RB + wg;
        at = at < kleft ? at : 0;
        const int p = q * (BO / 32) + wave * WPW + i;
        const uint32_t row = min(p * (64 / CH) + lane / CH, O - 1 - o0);
        copy16(row * kc + at, wt, lds0 + W0 + (c & 1) * WB + p * 1024, live);
    };
    // 512 k of a row's scales, through registers
    RowScales sreg;
    auto put_scales = [&](int c) {
        if (BO == 256 || tid < BO) *reinterpret_cast<u32x4 *>(sm + S0 + (c & 1) * SCB + tid * 16) = sreg.v;
    };
    // what is copied at the end of stage kt: the activations of stage kt + 2, a
    // part of chunk (kt + 1) / CPS + 1 (its slot's last reader was the chunk
    // before (kt + 1) / CPS's)
    constexpr int GROUP = XPW + WPW;
    auto copy_at = [&](int i, int kt) {
        if (i < XPW) {
            copy_x(i, kt + 2, (kt + 2 - nk) >> 31);
        } else {
            const int c = (kt + 1) / CPS + 1;
            copy_w(i - XPW, c, (kt + 1) & (CPS - 1), (c - nch) >> 31);
        }
    };
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
        const int c = st / CPS, b = 2 * (st & (CPS - 1)) + g;
        const char *p = sm + W0 + (c & 1) * WB + ((wo * TO + t) * 32 + (lane & 31)) * RB + (slot_of<RB>(b, lane & 31) << 4);
        f.v[t] = *reinterpret_cast<const u32x4 *>(p);
        f.s[t] = (uint8_t)sm[S0 + (st >> 3 & 1) * SCB + ((wo * TO + t) * 32 + (lane & 31)) * 16 + (2 * (st & 7) + g)];
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
            for (; COPY && d < GROUP && d * NF < (i + 1) * GROUP; d++) copy_at(d, kt);
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
    // chunk 0, and what the loop finds under way: stages 0 and 1, a quarter of chunk 1
    const bool whole = scales_whole(ks, sc0, a.ws, nullptr);             // (as above)
    if (whole) {
        // (64 rows a wavefront; past the tile's, into the other slot, not in use yet)
        const int row = min(wave * 64 + lane, min(BO - 1, O - 1 - o0));
        copy16((uint32_t)row * ks + sc0, uniform(a.ws + (size_t)o0 * ks), lds0 + S0 + wave * 1024, -1);
    } else {
        sreg.load(wrow, sc0, ks);
    }
#pragma unroll
    for (int q = 0; q < CPS; q++)
#pragma unroll
        for (int i = 0; i < WPW; i++) copy_w(i, 0, q, -1);
#pragma unroll
    for (int i = 0; i < XPW; i++) copy_x(i, 0, -1);
#pragma unroll
    for (int i = 0; i < GROUP; i++) copy_at(i, -1);
    if (!whole) put_scales(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(GROUP) : "memory");
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
        const bool sc = (kt & 7) == 0;     // (the slot's last reader was stage kt - 1)
        if (sc) sreg.load(wrow, sc0 + 16 * min(kt / 8 + 1, nsc - 1), ks);
        step(f0, f1, yes{}, kt, i1{}, r0, no{}, r1, no{}, 0);
        step(f1, f0, yes{}, kt, i2{}, r0, no{}, r1, no{}, 0);
        step(f0, f1, yes{}, kt, i3{}, r0, no{}, r1, no{}, 0);
        // this stage's operands have been read by all after the barrier, and the
        // next stage's copies have landed
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (sc) put_scales(kt / 8 + 1);
        step(f1, f0, yes{}, kt + 1, i0{}, r0, yes{}, r1, yes{}, kt);
        r0 = r1;
    }
    // the last stage; half of it, or with K in halves all, may lie past the group's k
    const bool past = (nk - 1) * kMx16Stage + 32 * g >= K;
    auto mask = [&](Frag &f) {
        if (!past) return;
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
}

// ---- a product's tiles ---------------------------------------------------------
template <bool XMX, int TO, int TMM, int RB>
constexpr int kWideLds = XMX ? kMxLds<TO, TMM> : kMx16Lds<TO, TMM, RB>;
constexpr int max_of(int a, int b) { return a > b ? a : b; }
// bytes of LDS with G groups: a group's operands, then the tile on its way to y
template <bool XMX, int TO, int TMM, int RB, int G>
constexpr int kTileLds = max_of(G * kWideLds<XMX, TO, TMM, RB>, TO * TMM * 64 * 128);

// y of 64 TO outputs from o0 x 64 TMM rows from m0, by 4 wavefronts, or, with G = 2, by
// 8, each 4 of them with half of K and LDS of their own. RB: bytes of a row's weights in
// LDS at once with bf16 activations; with 64 two tiles of 256 x 128 fit a CU, and one's
// first copies and stores run under the other's products (4096 rows x 12352 outputs, K
// 1024, 2048, 4096: 92, 175, 341 us; 256 x 256 tiles 102, 179, 339). MXFP4 activations
// gain nothing by it.
template <bool XMX, int TO, int TMM, int RB, int G>
__device__ __forceinline__ void wide_tile(char *sm, const MxProduct &a, int o0, int m0) {
    constexpr int LDS = kWideLds<XMX, TO, TMM, RB>, STAGE = XMX ? kMxStage : kMx16Stage;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wave >> 2, w = wave & 3;
    const KShare share = k_share(a.K, STAGE, G, grp);
    f32x16 acc[TO][TMM];
    if constexpr (XMX) mx_tile<TO, TMM>(sm + grp * LDS, a, o0, m0, share, acc);
    else mx16_tile<TO, TMM, RB>(sm + grp * LDS, a, o0, m0, share, acc);
    if constexpr (G == 2) {                // the sum of the halves, in the first's registers
        char *p = sm + LDS + w * (TO * TMM * 4096) + lane * 16;
        static_assert(4 * TO * TMM * 4096 <= LDS, "the second half's sums fit its LDS");
#pragma unroll
        for (int i = 0; grp == 1 && i < TO * TMM * 4; i++) {
            const f32x16 &v = acc[i / 4 / TMM][i / 4 % TMM];
            const int q = i % 4 * 4;
            *reinterpret_cast<mx_f32x4 *>(p + i * 1024) = mx_f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
        }
        __syncthreads();
        if (grp == 1) return;
#pragma unroll
        for (int i = 0; i < TO * TMM * 4; i++) {
            const mx_f32x4 v = *reinterpret_cast<const mx_f32x4 *>(p + i * 1024);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i / 4 / TMM][i / 4 % TMM][i % 4 * 4 + j] += v[j];
        }
    }
    store_tile<TO, TMM>(sm, acc, a.y, a.ldy, o0 + (w >> 1) * TO * 32, m0 + (w & 1) * TMM * 32, a.O, a.M, w, lane);
}

// Workgroups [0, big) take a tile each; four of the others a quarter each of a
// tile that would be left for a last round of the chip (256 x 256 only; 4096 rows x
// 12352 outputs, K 2048, 784 tiles on 256 CUs: 101 us, 90 with the last 16 in quarters;
// bf16 x 220 and 206). G = 2 where the tiles are at most one a CU, whose 4 wavefronts
// alone leave its MFMAs waiting: 512 rows x 4096 x 4096, bf16 x, 44 us, 33 with 8; MXFP4
// x 15.1 and 13.6.
template <bool XMX, int TO, int TMM, int RB, int G>
__global__ __launch_bounds__(256 * G, TO * TMM <= 8 ? 2 : 1) void k_mx_gemm_wide(MxProduct a, int big) {
    constexpr bool QUARTERS = TO * TMM == 16;
    __shared__ __attribute__((aligned(16))) char sm[kTileLds<XMX, TO, TMM, RB, G>];
    int id = blockIdx.x, part = -1;
    if (QUARTERS && id >= big) {           // (a tile's quarters on its XCD: ids 8 apart)
        const int q = id - big;
        part = q / 8 % 4;
        id = big + q / 32 * 8 + q % 8;
    }
    const int nbo = (a.O + 64 * TO - 1) / (64 * TO), nbm = (a.M + 64 * TMM - 1) / (64 * TMM);
    int ob, mb;
    tile_of(id, nbo, nbm, ob, mb);
    if (ob >= nbo) return;                               // (the grid is a multiple of 8)
    int o0 = ob * 64 * TO, m0 = mb * 64 * TMM;
    if constexpr (QUARTERS) {
        if (part >= 0) {
            o0 += part % 2 * 128;
            m0 += part / 2 * 128;
            if (o0 < a.O && m0 < a.M) wide_tile<XMX, 2, 2, 128, 1>(sm, a, o0, m0);
            return;
        }
    }
    wide_tile<XMX, TO, TMM, RB, G>(sm, a, o0, m0);
}

template <bool XMX, int TO, int TMM, int RB, int G>
int launch_wide(const MxProduct &a) {
    const int n = tile_grid((int)cdiv(a.O, 64 * TO), (int)cdiv(a.M, 64 * TMM));
    const int big = TO * TMM == 16 ? n - (int)mx_quarters(n) : n;
    const unsigned grid = (unsigned)(big + 4 * (n - big));
    APUS_TIMED("k_mx_gemm_wide", k_mx_gemm_wide<XMX, TO, TMM, RB, G><<<grid, 256 * G, 0, stream()>>>(a, big));
    return launch_check("k_mx_gemm_wide");
}
template <int TO, int TMM, int RB, int G>
int launch_wide_of(const MxProduct &a) {
    return a.xs ? launch_wide<true, TO, TMM, RB, G>(a) : launch_wide<false, TO, TMM, RB, G>(a);
}

}  // namespace

namespace apus {

size_t mx_quarters(size_t tiles) {
    const size_t cus = (size_t)cu_count() / 8 * 8, last = (tiles + 7) / 8 * 8 % cus;
    return tiles > cus && last <= cus / 4 ? last : 0;
}

int mx_gemm_wide(const MxProduct &a, int shape) {
    // (halves need a stage each)
    if (shape == 3 && a.K <= (a.xs ? kMxStage : kMx16Stage)) shape = 2;
    switch (shape) {
        case 2: return launch_wide_of<2, 2, 128, 1>(a);
        case 3: return launch_wide_of<2, 2, 128, 2>(a);
        case 4: return launch_wide_of<4, 4, 128, 1>(a);
        default: return launch_wide<false, 4, 2, 64, 1>(a);
    }
}

}  // namespace apus

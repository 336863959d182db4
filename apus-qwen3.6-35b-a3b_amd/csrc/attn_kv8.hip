// attn_kv8.hip -- gated-GQA decode over the 8-bit KV cache (kv8.h): for each
// new token and head, q = RoPE((1+w) RMSNorm(q)) and
//   y = sigmoid(gate) * sum_j p_j v_j,  p = softmax(q . k_j / 16, j <= position),
// in one pass over K and V with a running reference point M and sum of the
// softmax (p = 2^(t - M), t the score times log2 e / 16).
//
// The 8 q heads of a kv head times up to 4 new tokens are the rows of the matrix
// products, one or two blocks of 16, so K and V come from HBM once a (sequence, kv
// head) pair. The pairs' blocks are laid end to end and cut into runs, one a
// workgroup and at most two a CU, so that every CU is as long at it however ragged
// the contexts are; a run that crosses a pair's border is two segments. The 4
// wavefronts of a workgroup take a segment's blocks in turn, each with its own M,
// sum and outputs of all rows in registers, and meet in LDS at its end. A segment
// that is a whole pair writes y; others keep (M, sum, outputs) of their rows in slot
// pair + run (no two segments share one), and k_kv8_combine joins them.
//
// A wavefront has no LDS traffic for K and V: their bytes come in operand order
// (16-byte loads, whole KiB), widen in registers (exactly: K's codes to fp16, V's
// times their scale to bf16), and the scores' registers are the operand of P V.
// Probabilities go to bf16 for that product (fp16 would cut those far below the
// largest), and their sum is that of the rounded ones: y is a mean of v with
// weights that add up to 1, and a single large weight brings no error.
//
// Bound by HBM where contexts are long: 64 sequences at 32768 with 2 kv heads, 2.15
// GB in 322 us, 6.7 TB/s (a pure read stream reaches 7.0; with loads that stay in
// the caches 361 us, against 328 then); 128 ragged ones verifying 1-4 tokens, 1.36 GB
// in 230 us, 5.9 TB/s (two row blocks: each block of K and V is worked on for twice as long
// and K's next loads wait for the scores, else the registers spill; wavefronts in
// pairs that share the keys, a row block each, 291 us). Few sequences: the chain of
// a segment, 9 us of launch, block ids, q rows and first loads, the end 4 us, and
// the second launch (one sequence, 3 tokens at 60001, 61 MB: 27 us).
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <type_traits>

#include "apus_dev.h"
#include "apus_host.h"
#include "attn_mixer.h"
#include "kv8.h"

using namespace apus;

namespace {

constexpr int D = kKv8D, ROT = 64, GRP = 8, KEYS = kKv8Keys;
constexpr int kRows = 32, kWaves = 4;
constexpr float kEps = 1e-6f;
constexpr float kL2E = 1.44269504088896341f;
constexpr int QP = D + 8, AP = D + 4;        // LDS pitches of q rows and of outputs
// t may pass M by this much before M moves: 2^10 a term (kv8_v_up: no sum overflows)
constexpr float kSlack = 10.0f;

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef kv8_bf16x8 bf16x8;
typedef kv8_f16x8 f16x8;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// over the four lanes that hold a row's scores (16 and 32 apart)
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;
// over 16 lanes
__device__ __forceinline__ float sum16(float x) {
    x += dpp<kXor1>(x);
    x += dpp<kXor2>(x);
    x += dpp<kHalfMirror>(x);
    return x + dpp<kMirror>(x);
}
__device__ __forceinline__ float max16(float x) {
    x = fmaxf(x, dpp<kXor1>(x));
    x = fmaxf(x, dpp<kXor2>(x));
    x = fmaxf(x, dpp<kHalfMirror>(x));
    return fmaxf(x, dpp<kMirror>(x));
}
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kL2E));
}

typedef const __attribute__((address_space(1))) u32x4 *gu32x4p;

// a row's 4 outputs o / l times the gate's sigmoid
__device__ __forceinline__ uint2 finish(f32x4 o, float l, uint2 gate) {
    const float inv = 1.0f / l;
    const float g[4] = {bf2f((uint16_t)gate.x), bf2f((uint16_t)(gate.x >> 16)), bf2f((uint16_t)gate.y),
                        bf2f((uint16_t)(gate.y >> 16))};
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] *= inv * sigmoid(g[e]);
    return make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
}

// How the pairs' blocks are cut into runs: of len[0] and len[1] in turn, from run
// half (even) on of len[2] and len[3].
struct Runs {
    int32_t len[4], half;
    __host__ __device__ int start(int i) const {
        const int h = i < half ? 0 : 2, j = i < half ? i : i - half;
        return (h ? half / 2 * (len[0] + len[1]) : 0) + j / 2 * (len[h] + len[h + 1]) + (j & 1) * len[h];
    }
    __host__ __device__ int of(int x) const {              // the run of block x
        const int s = half / 2 * (len[0] + len[1]), h = x < s ? 0 : 2, y = x < s ? x : x - s;
        const int both = len[h] + len[h + 1], q = y / both;
        return (h ? half : 0) + 2 * q + (y - q * both >= len[h] ? 1 : 0);
    }
};

// RB: row blocks, 2 where a sequence has more than two new tokens; their q rows
// then stay in LDS, and come from there once a block of keys.
template <int RB, int N>
__global__ __launch_bounds__(64 * kWaves, 2) void k_kv8_attn(
    Kv8SeqsN<N> sq, Kv8Ref kv, const uint16_t *__restrict__ qg, const uint16_t *__restrict__ qn_w,
    const uint16_t *__restrict__ rope, int nkv, int total, Runs runs, float c2, uint16_t *__restrict__ y,
    float *__restrict__ part, float2 *__restrict__ stat) {
    static_assert(64 * kWaves == D, "a thread a dim, a wavefront's threads 4 q rows");
    static_assert(16 * AP >= 2048 && 16 * RB * QP / 2 + kWaves * 2048 <= kWaves * 16 * AP, "room for V with a NaN");
    // (with two row blocks the q rows lie where the outputs meet later: two
    // workgroups a CU)
    __shared__ __attribute__((aligned(16))) float os[kWaves * 16 * AP];
    __shared__ __attribute__((aligned(16))) _Float16 qown[RB == 1 ? 16 * QP : 1];
    _Float16 *const qs = RB == 1 ? qown : reinterpret_cast<_Float16 *>(os);
    __shared__ float qsc[16 * RB];
    // the wavefronts' M, and the sum of each of a row's four lanes
    __shared__ __attribute__((aligned(16))) float ms[16 * RB][kWaves], ls[16 * RB][kWaves][4];
    __shared__ int first_nan[D];           // the first key whose v is NaN there, in the blocks not all rows see
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x1 = min(runs.start((int)blockIdx.x + 1), total), nh = nkv * GRP;
    int nx = 0;
    for (int x = runs.start((int)blockIdx.x); x < x1; x = nx) {
        // (opaque: or every address of a lane is formed ahead of this loop, and spilled)
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, n = lane & 15, g = lane >> 4;
        const Kv8At a = kv8_find<false>(sq, x / nkv);
        const int t0 = a.t0, tq = a.tokens, p0 = a.p0, row = a.row;
        const int nbp = a.blocks, nb = (p0 + tq + KEYS - 1) / KEYS, local = x - nkv * a.off;
        const int kvh = local / nbp, b0 = local % nbp, b1 = min(b0 + x1 - x, nb), pair = a.s * nkv + kvh;
        nx = min(x1, x + nbp - b0);
        if (b0 >= nb) continue;                            // (nothing but padding)
        const int rows = tq * GRP, last = b1 - 1;

        // q rows (token, head): 16 threads a row, thread e the dims 8 c .. and 128 + 8 c ..,
        // c such that the dims +-32 of a rotary pair are the neighbour's
        const int qr = tid >> 4, e = tid & 15, c8 = ((e & 8) | (e & 6) >> 1 | (e & 1) << 2) * 8;
        u16x8 qa[RB], qc[RB], wa, wc, co[RB], si[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            const int t = min(rb * 2 + (qr >> 3), tq - 1);
            const uint16_t *p = qg + ((size_t)(t0 + t) * nh + kvh * GRP + (qr & 7)) * 2 * D + c8;
            qa[rb] = *reinterpret_cast<const u16x8 *>(p);
            qc[rb] = *reinterpret_cast<const u16x8 *>(p + 128);
            const uint16_t *cs = rope + (size_t)(p0 + t) * ROT + (c8 & 31);
            co[rb] = *reinterpret_cast<const u16x8 *>(cs);
            si[rb] = *reinterpret_cast<const u16x8 *>(cs + ROT / 2);
        }
        wa = *reinterpret_cast<const u16x8 *>(qn_w + c8);
        wc = *reinterpret_cast<const u16x8 *>(qn_w + 128 + c8);
        __builtin_amdgcn_sched_barrier(0);
        // the first block's loads, under the q rows' work
        u32x4 kr[8], vr[8];
        float ks = 0.0f, vs = 0.0f, kn = 0.0f, vn = 0.0f;
        // (scalar bases 4 KiB apart, so that one register holds the lane's offset; behind
        // the last block the loads, which the wait counts want, take a line each)
        uint32_t lane16 = (uint32_t)lane * 16;
        auto load = [&](u32x4 (&r)[8], const uint8_t *base, uint32_t id) {
            const uint8_t *const p = base + ((size_t)id * nkv + kvh) * kKv8Bytes;
#pragma unroll
            for (int i = 0; i < 8; i++)
                r[i] = __builtin_nontemporal_load((gu32x4p)(p + i / 4 * 4096 + (lane16 + i % 4 * 1024)));
        };
        auto scales = [&](uint32_t id, float &k_, float &v_) {
            const int32_t *p = (const int32_t *)(kv.scale + ((size_t)id * nkv + kvh) * 2);
            k_ = __int_as_float(sload_i32(p, 8, 0));
            v_ = __int_as_float(sload_i32(p, 8, 1));
        };
        uint32_t id = kv8_id_u(kv, row, min(b0 + wave, last));
        uint32_t idn = kv8_id_u(kv, row, min(b0 + wave + kWaves, last));
        load(kr, kv.k, id);
        load(vr, kv.v, id);
        scales(id, ks, vs);
        __builtin_amdgcn_sched_barrier(0);
        first_nan[tid] = 0x7fffffff;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss += bf2f(qa[rb][i]) * bf2f(qa[rb][i]) + bf2f(qc[rb][i]) * bf2f(qc[rb][i]);
            const float rs = 1.0f / sqrtf(sum16(ss) / (float)D + kEps);
            float va[8], vc[8], mx = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = bf2f(qa[rb][i]) * rs * (1.0f + bf2f(wa[i])), w = dpp<kXor1>(v);
                const float r = v * bf2f(co[rb][i]) + (e & 1 ? w : -w) * bf2f(si[rb][i]);
                va[i] = e < 8 ? r : v;
                vc[i] = bf2f(qc[rb][i]) * rs * (1.0f + bf2f(wc[i]));
                mx = fmaxf(mx, fmaxf(fabsf(va[i]), fabsf(vc[i])));
            }
            // (rows past the tokens repeat the last one)
            const float sc = kv8_row_scale(max16(mx)), inv = 1.0f / sc;
            f16x8 oa, oc;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                oa[i] = (_Float16)(va[i] * inv);
                oc[i] = (_Float16)(vc[i] * inv);
            }
            *reinterpret_cast<f16x8 *>(qs + (rb * 16 + qr) * QP + c8) = oa;
            *reinterpret_cast<f16x8 *>(qs + (rb * 16 + qr) * QP + 128 + c8) = oc;
            if (e == 0) qsc[rb * 16 + qr] = sc * c2;
        }
        __syncthreads();
        // k-step (i, u): dims (4 i + g) 16 + 8 u ..
        auto q_of = [&](int rb, int i) {
            return *reinterpret_cast<const f16x8 *>(qs + (rb * 16 + n) * QP + (i / 2 * 4 + g) * 16 + i % 2 * 8);
        };
        f16x8 q[8];
        float qf[RB];                                      // scores' factor, with log2 e / 16
#pragma unroll
        for (int rb = 0; rb < RB; rb++) qf[rb] = qsc[rb * 16 + n];
        if (RB == 1) {
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = q_of(0, i);
        }
        f32x4 acc[RB][16];
        float M[RB], l[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            M[rb] = -INFINITY;
            l[rb] = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) acc[rb][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int j = b0 + wave; j < b1; j += kWaves) {
            f32x4 S[RB][2];
#pragma unroll
            for (int rb = 0; rb < RB; rb++) S[rb][0] = S[rb][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 8; i++) {                  // dims' chunks 4 (i / 2) .., their first or second 8
                const u32x4 w0 = kr[i / 2], w1 = kr[4 + i / 2];    // both halves of the keys
                const f16x8 k0 = kv8_f16(w0[i % 2 * 2], w0[i % 2 * 2 + 1]), k1 = kv8_f16(w1[i % 2 * 2], w1[i % 2 * 2 + 1]);
#pragma unroll
                for (int rb = 0; rb < RB; rb++) {
                    const f16x8 qi = RB == 1 ? q[i] : q_of(rb, i);
                    S[rb][0] = mfma16(k0, qi, S[rb][0]);
                    S[rb][1] = mfma16(k1, qi, S[rb][1]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (j + kWaves >= b1) lane16 = 0;
            id = idn;
            if (RB == 1) load(kr, kv.k, id);
            scales(id, kn, vn);
            idn = kv8_id_u(kv, row, min(j + 2 * kWaves, last));
            __builtin_amdgcn_sched_barrier(0);
            const bool tail = (j + 1) * KEYS > p0 + 1;     // some row does not see some key
            const float up = (float)kv8_v_up(vs);
            bf16x8 pb[RB];                                 // the lane's 8 keys
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                float t[8];
                const float f = qf[rb] * ks;
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = S[rb][i / 4][i % 4] * f;
                if (tail) {
                    const int lim = p0 + min(rb * 2 + (n >> 3), tq - 1) - j * KEYS - g * 4;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (i / 4 * 16 + i % 4 > lim) t[i] = -INFINITY;
                }
                const float mx = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])),
                                       fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7]))) + up;
                if (__any(mx > M[rb] + kSlack)) {          // (always at a row's first keys)
                    const float m = fmaxf(M[rb], row_max(mx));
                    const float d = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M[rb] - m);
                    M[rb] = m;
                    l[rb] *= d;
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[rb][i] *= d;
                }
                const float ref = M[rb] == -INFINITY ? 0.0f : M[rb];
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = __builtin_amdgcn_exp2f(t[i] - ref);
                u32x4 pk;
#pragma unroll
                for (int i = 0; i < 4; i++) pk[i] = pack2(t[2 * i], t[2 * i + 1]);
                pb[rb] = __builtin_bit_cast(bf16x8, pk);
                // (the rounded ones: what the product with V is made of)
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = __uint_as_float(i % 2 ? pk[i / 2] & 0xffff0000u : pk[i / 2] << 16);
                l[rb] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
            }
            if (tail) {
                // keys past the last token: whatever lies there counts as zero
                const int lim = p0 + tq - j * KEYS - g * 4;
                uint32_t mk[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i / 4 * 16 + i % 4 < lim) mk[i / 4] |= 0xffu << (i % 4 * 8);
                uint32_t wild = 0;
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        vr[i][w] &= mk[w % 2];
                        wild |= kv8_nan_codes(vr[i][w]);
                    }
                if (__any(wild != 0)) {
                    // a NaN reaches the rows that see its key and no other: taken
                    // out of the product, the first key of each dim kept (in a loop
                    // over 8 KiB of os, unrolled it took 60 registers: with one row block
                    // where this wavefront's outputs go, since others may have ended and
                    // written theirs; with two behind the q rows, all wait before they write)
                    u32x4 *const mine_ = reinterpret_cast<u32x4 *>(
                        RB == 1 ? os + wave * 16 * AP : os + 16 * RB * QP / 2 + wave * 2048) + lane;
#pragma unroll
                    for (int i = 0; i < 8; i++) mine_[i * 64] = vr[i];
#pragma unroll 1
                    for (int i = 0; i < 32; i++) {
                        uint32_t *const c = reinterpret_cast<uint32_t *>(mine_ + i / 4 * 64) + i % 4;
                        const uint32_t bad = kv8_nan_codes(*c);
                        if (bad) {
                            *c &= ~bad;
                            atomicMin(&first_nan[i / 2 * 16 + n],
                                      j * KEYS + i % 2 * 16 + g * 4 + (__ffs((int)bad) - 1) / 8);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) vr[i] = mine_[i * 64];
                }
            }
            if (RB > 1) {                                  // (here: the scores' registers are free)
                __builtin_amdgcn_sched_barrier(0);
                load(kr, kv.k, id);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bf16x8 va = kv8_bf16(vr[i][0], vr[i][1], vs), vb = kv8_bf16(vr[i][2], vr[i][3], vs);
#pragma unroll
                for (int rb = 0; rb < RB; rb++) {
                    acc[rb][2 * i] = mfma16(va, pb[rb], acc[rb][2 * i]);
                    acc[rb][2 * i + 1] = mfma16(vb, pb[rb], acc[rb][2 * i + 1]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load(vr, kv.v, id);
            __builtin_amdgcn_sched_barrier(0);
            ks = kn;
            vs = vn;
        }

        // the wavefronts meet, a row block at a time
        const bool whole = b0 == 0 && b1 == nb;
        const size_t slot = (size_t)(pair + (int)blockIdx.x) * kRows;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            if (rb * 16 >= rows) break;
            if (RB > 1) __syncthreads();                   // (q rows, or the block before, are done with)
            if (rb * 16 + n < rows) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    *reinterpret_cast<f32x4 *>(os + (wave * 16 + n) * AP + i * 16 + g * 4) = acc[rb][i];
                ls[rb * 16 + n][wave][g] = l[rb];
                if (g == 0) ms[rb * 16 + n][wave] = M[rb];
            }
            __syncthreads();
            // every fourth row, four dims a lane
            const int d = lane * 4;
#pragma unroll
            for (int i = 0; i < 16 / kWaves; i++) {
                const int r16 = i * kWaves + wave, r = rb * 16 + r16;
                if (r >= rows) break;
                const f32x4 mw = *reinterpret_cast<const f32x4 *>(ms[r]);
                const float m = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
                float lt = 0.0f;
                f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; w++) {         // (one without a block has zeros)
                    const float f = mw[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw[w] - m);
                    const f32x4 lw = *reinterpret_cast<const f32x4 *>(ls[r][w]);
                    lt += ((lw[0] + lw[1]) + (lw[2] + lw[3])) * f;
                    o += *reinterpret_cast<const f32x4 *>(os + (w * 16 + r16) * AP + d) * f;
                }
#pragma unroll
                for (int e_ = 0; e_ < 4; e_++)
                    if (first_nan[d + e_] <= p0 + (r >> 3)) o[e_] = NAN;
                if (whole) {
                    const size_t at = (size_t)(t0 + (r >> 3)) * nh + kvh * GRP + (r & 7);
                    const uint2 gate = *reinterpret_cast<const uint2 *>(qg + at * 2 * D + D + d);
                    *reinterpret_cast<uint2 *>(y + at * D + d) = finish(o, lt, gate);
                } else {
                    *reinterpret_cast<f32x4 *>(part + (slot + r) * D + d) = o;
                    if (lane == 0) stat[slot + r] = make_float2(m, lt);
                }
            }
        }
        if (nx < x1) __syncthreads();                      // (qs and os are the next segment's)
    }
}

// SP wavefronts a (token, head) of a pair that lies in several runs, each with
// its share of the segments, 8 loads at a time: up to 8 segments one wavefront, up
// to 32 four, else 16, so that a call of few tokens takes one or two rounds of loads
// (one sequence of 3 tokens at 60001, 126 segments: 28.6 us in all with 4 wavefronts,
// 26.8 with 16). Bound by the latency of its rounds: 3 to 6 us.
template <int SP, int N>
__global__ __launch_bounds__(64 * (SP > 4 ? SP : 4)) void k_kv8_combine(Kv8SeqsN<N> sq, const float *__restrict__ part,
                                                     const float2 *__restrict__ stat,
                                                     const uint16_t *__restrict__ qg, int nkv, Runs runs, int items,
                                                     uint16_t *__restrict__ y) {
    const int lane = threadIdx.x & 63, d = lane * 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = wave % SP;
    constexpr int W = SP > 4 ? SP : 4;
    const int item = min((int)blockIdx.x * (W / SP) + wave / SP, items - 1);   // (the last again: the same y)
    const int nh = nkv * GRP, h = item % nh, tt = sq.e[0].cu + item / nh;
    const Kv8At a = kv8_find<true>(sq, tt);
    const int kvh = h / GRP, r = (tt - a.t0) * GRP + h % GRP;
    const int nb = (a.p0 + a.tokens + KEYS - 1) / KEYS, x = nkv * a.off + kvh * a.blocks;
    const int w0 = runs.of(x), w1 = runs.of(x + nb - 1), pair = a.s * nkv + kvh;
    if (w0 == w1) return;                                  // (the whole pair: written already)
    const size_t at = (size_t)tt * nh + h;
    const uint2 gate = *reinterpret_cast<const uint2 *>(qg + at * 2 * D + D + d);
    const size_t slot0 = (size_t)(pair + w0) * kRows + r;
    const int segs = w1 - w0 + 1;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = share; w < segs; w += 8 * SP) {
        f32x4 v[8];
        float2 u[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t sl = slot0 + (size_t)min(w + i * SP, segs - 1) * kRows;
            v[i] = *reinterpret_cast<const f32x4 *>(part + sl * D + d);
            u[i] = stat[sl];
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < 8; i++) mn = fmaxf(mn, u[i].x);
        const float k = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= k;
        o *= k;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (w + i * SP >= segs) continue;
            const float f = u[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(u[i].x - m);   // (0 keeps a NaN)
            l += u[i].y * f;
            o += v[i] * f;
        }
    }
    if (SP > 1) {
        __shared__ f32x4 os[W][64];
        __shared__ float2 st[W];
        os[wave][lane] = o;
        if (lane == 0) st[wave] = make_float2(m, l);
        __syncthreads();
        if (share) return;
        float mt = -INFINITY;
#pragma unroll
        for (int i = 0; i < SP; i++) mt = fmaxf(mt, st[wave + i].x);
        l = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < SP; i++) {
            const float2 u = st[wave + i];
            const float f = u.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(u.x - mt);
            l += u.y * f;
            o += os[wave + i][lane] * f;
        }
    }
    *reinterpret_cast<uint2 *>(y + at * D + d) = finish(o, l, gate);
}

int32_t ctx_blocks(int32_t pos0, int32_t n) { return n > 0 ? (pos0 + n + KEYS - 1) / KEYS : 0; }

// How a call is cut. Two workgroups a CU at most (more runs only add segments: 64
// sequences at 32768, two a CU 328 us, four 340, eight 355).
//
// Short contexts: a pair is a run (the same slot for each, as long as the longest
// context), with no partial results and no second launch: up to 24 blocks (one
// sequence at 500: 8.9 us, cut 9.3; at 1500, 47 blocks, 20 and 9.5), or to 96
// where the pairs alone nearly fill the chip (100 sequences at 1500: 28 and 34).
// Else a segment counts for kPad blocks more than it has, what its start and end
// take (128 ragged sequences: 250 us with none, 244 with 8, 241 with 16, 244 with
// 32; 64 equal ones 330, 330, 332, 335), which also keeps two segments out of one
// short run. Runs have a block for each wavefront at least, and grow with the
// total as its root, up to 16, since every run costs the second launch a partial
// result (one sequence at 60001: 19 us with runs of 15, 22 with 11 and 21 with 8).
constexpr int32_t kPad = 8, kShort = 24, kShortMany = 96;
// Runs of more than kLong blocks, two a CU, are not equal: of the two workgroups of a
// CU the first is served first, and of two neighbouring XCDs (workgroups go to the
// XCDs in turn) the odd one reads less while all of them read (64 equal contexts of
// 32768 in equal runs: 230 and 277 us on even XCDs, 280 and 313 on odd ones). A
// run's share of the mean, even and odd ones of the first 256 and of the others:
// 1.18, 0.97, 0.98 and 0.87 (64 at 32768 328 us equal, 322 so; 128 ragged ones
// verifying 1-4 tokens 239 and 230; 128 at 8000 171 and 167). Shorter runs differ by
// few blocks and stay equal. The shares are those of a card with nothing else on it:
// where other work shifts them the runs end less evenly, with the same results.
constexpr int32_t kLong = 32;
constexpr double kShare[3] = {1.18, 0.97, 0.98};
size_t max_runs() { return 2 * (size_t)cu_count(); }
int32_t whole_pairs(size_t B, const int32_t *cu, const int32_t *pos0, size_t nkv) {
    int32_t longest = 0;
    size_t pairs = 0;
    for (size_t s = 0; s < B; s++) {
        longest = std::max(longest, ctx_blocks(pos0[s], cu[s + 1] - cu[s]));
        pairs += cu[s + 1] > cu[s] ? nkv : 0;
    }
    return longest <= kShort || (longest <= kShortMany && 4 * pairs >= 3 * (size_t)cu_count()) ? longest : 0;
}
int32_t counted_blocks(int32_t pos0, int32_t n, int32_t whole) {
    return n <= 0 ? 0 : whole ? whole : ctx_blocks(pos0, n) + kPad;
}
Runs cut_runs(size_t total, int32_t whole) {
    const size_t root = std::min<size_t>(16, (size_t)(sqrt((double)total / 16.0) + 0.5)), n = max_runs();
    const int32_t len = (int32_t)std::max({(total + n - 1) / n, root, (size_t)kWaves});
    if (whole) return Runs{{whole, whole, whole, whole}, 0};
    if (len <= kLong || n % 4) return Runs{{len, len, len, len}, 0};
    const double q = (double)total / (double)n;
    Runs r = {{(int32_t)(q * kShare[0]), (int32_t)(q * kShare[1]), (int32_t)(q * kShare[2]), 0}, (int32_t)(n / 2)};
    r.len[3] = (int32_t)((4 * total + n - 1) / n) - r.len[0] - r.len[1] - r.len[2];
    return r;
}

}  // namespace

namespace apus {

int attn_kv8_check(const ApusHipAttnLayer *L, const ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                   const int32_t *cu, const int32_t *pos0, bool writes, const ApusHipKv8Cache *kv, Kv8Ref *r, size_t *T) {
    if (int e = attn_check_layer(L)) return e;
    if (!w) return set_error(kErrArgument, "NULL workspace");
    if (w->device != current_device())
        return set_error(kErrArgument, "the workspace is on device %d, the library on %d", w->device, current_device());
    if (w->nkv != L->nkv || w->rot != L->rot || w->theta != L->theta)
        return set_error(kErrArgument, "the workspace was made for a layer of other dims");
    if (int e = kv8_check(kv, L->nkv, B, rows, cu, pos0, writes, r, T)) return e;
    if (!*T) return kOk;
    for (size_t s = 0; s < B; s++)
        if (cu[s + 1] > cu[s] && (size_t)pos0[s] + (size_t)(cu[s + 1] - cu[s]) > w->max_pos)
            return set_error(kErrArgument, "sequence %zu reaches position %lld, the workspace's tables %zu", s,
                             (long long)pos0[s] + (cu[s + 1] - cu[s]), w->max_pos);
    if (!L->qn_w || !L->kn_w) return set_error(kErrArgument, "NULL operand");
    if ((uintptr_t)L->qn_w % 16 || (uintptr_t)L->kn_w % 16)
        return set_error(kErrUnsupported, "the attention operands need 16-byte alignment");
    if (writes && (kv8_overlap_cache(kv, L->nkv, L->qn_w, D * 2) || kv8_overlap_cache(kv, L->nkv, L->kn_w, D * 2)))
        return set_error(kErrArgument, "an input overlaps the cache");
    return kOk;
}

int attn_kv8_check_operands(const ApusHipAttnLayer *L, size_t T, const uint16_t *qg, const uint16_t *k,
                            const uint16_t *v, const ApusHipKv8Cache *kv, const uint16_t *y) {
    if (!k != !v) return set_error(kErrArgument, "k and v are both given or both NULL");
    if (!T) return kOk;
    if (!qg || !y) return set_error(kErrArgument, "NULL operand");
    if ((uintptr_t)qg % 16 || (uintptr_t)y % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16)
        return set_error(kErrUnsupported, "the attention operands need 16-byte alignment");
    const size_t ny = T * L->nh * D * 2, nk = T * L->nkv * D * 2;
    if (kv8_overlap(y, ny, qg, 2 * ny) || (k && (kv8_overlap(y, ny, k, nk) || kv8_overlap(y, ny, v, nk))) ||
        kv8_overlap_cache(kv, L->nkv, y, ny) || kv8_overlap(y, ny, L->qn_w, D * 2) || kv8_overlap(y, ny, L->kn_w, D * 2))
        return set_error(kErrArgument, "y overlaps an input");
    if (kv->block_table && kv8_overlap(y, ny, kv->block_table, kv->max_rows * kv->max_blocks * 4))
        return set_error(kErrArgument, "y overlaps the block table");
    if (k && (kv8_overlap_cache(kv, L->nkv, qg, 2 * ny) || kv8_overlap_cache(kv, L->nkv, k, nk) ||
              kv8_overlap_cache(kv, L->nkv, v, nk)))       // (the cache is written)
        return set_error(kErrArgument, "an input overlaps the cache");
    return kOk;
}

int attn_decode_kv8_run(const ApusHipAttnLayer *L, ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                        const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                        const uint16_t *v, const Kv8Ref &kv, uint16_t *y) {
    const size_t nkv = L->nkv;
    if (k)
        if (int e = kv8_append_run(kv, nkv, B, rows, cu, pos0, k, nkv * D, v, nkv * D, L->kn_w, w->rope)) return e;
    const int32_t whole = whole_pairs(B, cu, pos0, nkv);
    return kv8_launches(B, rows, cu, pos0, [&](size_t s) { return counted_blocks(pos0[s], cu[s + 1] - cu[s], whole); },
                        [&](const auto &q) {
        constexpr int N = sizeof(q.e) / sizeof(q.e[0]) - 1;
        const size_t total = (size_t)q.e[q.n].off * nkv;
        if (!total) return (int)kOk;
        int most = 0;
        for (int s = 0; s < q.n; s++) most = std::max(most, q.e[s + 1].cu - q.e[s].cu);
        const Runs runs = cut_runs(total, whole);
        size_t segs = 1;                                   // the most of a pair
        for (int s = 0; s < q.n; s++) {
            const size_t nb = (size_t)ctx_blocks(q.e[s].pos0, q.e[s + 1].cu - q.e[s].cu);
            size_t x = nkv * (size_t)q.e[s].off;
            for (size_t h = 0; nb && h < nkv; h++, x += (size_t)(q.e[s + 1].off - q.e[s].off))
                segs = std::max(segs, (size_t)(runs.of((int)(x + nb - 1)) - runs.of((int)x) + 1));
        }
        const float c2 = (float)(1.44269504088896341 / sqrt((double)D));
        auto launch = [&](auto rb) {
            APUS_TIMED("k_kv8_attn",
                       k_kv8_attn<decltype(rb)::value, N><<<(unsigned)runs.of((int)total - 1) + 1, 64 * kWaves, 0, stream()>>>(
                           q, kv, qg, L->qn_w, w->rope, (int)nkv, (int)total, runs, c2, y, w->part, w->stat));
        };
        if (most <= 2) launch(std::integral_constant<int, 1>{});
        else launch(std::integral_constant<int, 2>{});
        if (int e = launch_check("k_kv8_attn")) return e;
        if (segs == 1) return (int)kOk;
        const size_t items = (size_t)(q.e[q.n].cu - q.e[0].cu) * L->nh;
        auto combine = [&](auto sp) {
            constexpr int SP = decltype(sp)::value;
            constexpr int W = SP > 4 ? SP : 4;
            APUS_TIMED("k_kv8_combine",
                       k_kv8_combine<SP, N><<<cdiv(items, W / SP), 64 * W, 0, stream()>>>(
                           q, w->part, w->stat, qg, (int)nkv, runs, (int)items, y));
        };
        if (segs <= 8) combine(std::integral_constant<int, 1>{});
        else if (segs <= 32) combine(std::integral_constant<int, 4>{});
        else combine(std::integral_constant<int, 16>{});
        return launch_check("k_kv8_combine");
    });
}

bool attn_decode_kv8_fits(const ApusHipAttnKv8Work *w, size_t B, const int32_t *cu, const int32_t *pos0) {
    size_t total = 0;
    for (size_t s = 0; s < B; s++) {
        if (cu[s + 1] - cu[s] > kRows / GRP) return false;
        if (s % kKv8Seqs == 0) total = 0;
        total += (size_t)counted_blocks(pos0[s], cu[s + 1] - cu[s], 0) * w->nkv;
        if (total > 0x7f000000) return false;
    }
    return B <= w->max_seqs;
}

int attn_decode_kv8_check(const ApusHipAttnLayer *L, const ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                          const int32_t *cu, const int32_t *pos0, bool writes, const ApusHipKv8Cache *kv, Kv8Ref *r,
                          size_t *T) {
    if (int e = attn_kv8_check(L, w, B, rows, cu, pos0, writes, kv, r, T)) return e;
    if (B > w->max_seqs)
        return set_error(kErrArgument, "%zu sequences, the workspace holds %zu", B, w->max_seqs);
    for (size_t s = 0; s < B; s++)
        if (cu[s + 1] - cu[s] > kRows / GRP)
            return set_error(kErrUnsupported, "decode takes 0..%d new tokens per sequence (got %d)", kRows / GRP,
                             cu[s + 1] - cu[s]);
    return attn_decode_kv8_fits(w, B, cu, pos0) ? (int)kOk
                                                : set_error(kErrUnsupported, "too many cached keys in one call");
}

}  // namespace apus

extern "C" {

int apus_hip_attn_kv8_work_create(const ApusHipAttnLayer *L, size_t max_seqs, size_t max_pos,
                                  ApusHipAttnKv8Work **out) {
    APUS_ENABLED();
    if (!out) return set_error(kErrArgument, "NULL output");
    *out = nullptr;
    if (int r = attn_check_layer(L)) return r;
    if (!max_seqs || max_seqs > ((size_t)1 << 24) || L->nkv > kKv8MaxHeads || !max_pos || max_pos > ((size_t)1 << 24))
        return set_error(kErrUnsupported, "an attention workspace for %zu sequences, %zu kv heads, %zu positions",
                         max_seqs, L->nkv, max_pos);
    if (int r = mx_ready()) return r;
    auto *w = new (std::nothrow) ApusHipAttnKv8Work{L->nkv, max_seqs, max_pos, L->rot, L->theta, current_device(),
                                                    nullptr, 0, nullptr, nullptr, nullptr};
    if (!w) return set_error(kErrHip, "out of host memory");
    // decode: a slot of 32 rows a segment, pair + run, both below their counts in one
    // launch; prefill: 128 rows a part of a tile, two a CU
    w->rows = std::max((std::min<size_t>(max_seqs, kKv8Seqs) * L->nkv + max_runs()) * kRows, max_runs() * 128);
    const size_t pb = w->rows * D * 4, sb = w->rows * 8, rb = max_pos * ROT * 2;
    if (hipMalloc((void **)&w->base, pb + sb + rb) != hipSuccess) {
        delete w;
        (void)hipGetLastError();           // (not for the next launch to report)
        return set_error(kErrHip, "hipMalloc of %zu bytes failed", pb + sb + rb);
    }
    w->part = (float *)w->base;
    w->stat = (float2 *)(w->base + pb);
    w->rope = (uint16_t *)(w->base + pb + sb);
    // a table of its own: the library's moves when it grows, a graph keeps this one
    const uint16_t *rope = rope_table(L->rot, L->theta, max_pos);
    if (!rope || hipMemcpyAsync(w->rope, rope, rb, hipMemcpyDeviceToDevice, stream()) != hipSuccess ||
        hipStreamSynchronize(stream()) != hipSuccess) {
        (void)hipFree(w->base);
        delete w;
        return rope ? set_error(kErrHip, "filling the workspace failed") : (int)kErrHip;
    }
    *out = w;
    return kOk;
}

int apus_hip_attn_kv8_work_destroy(ApusHipAttnKv8Work *w) {
    APUS_ENABLED();
    if (!w) return kOk;
    if (int r = mx_ready()) return r;
    APUS_HIP_TRY(hipStreamSynchronize(stream()));
    (void)hipFree(w->base);
    delete w;
    return kOk;
}

int apus_hip_attn_decode_kv8(const ApusHipAttnLayer *L, ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                             const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                             const uint16_t *v, const ApusHipKv8Cache *kv, uint16_t *y) {
    APUS_ENABLED();
    Kv8Ref r;
    size_t T = 0;
    if (int e = attn_decode_kv8_check(L, w, B, rows, cu, pos0, k || v, kv, &r, &T)) return e;
    if (int e = attn_kv8_check_operands(L, T, qg, k, v, kv, y)) return e;
    if (int e = mx_ready()) return e;
    if (!T) return kOk;
    return attn_decode_kv8_run(L, w, B, rows, cu, pos0, qg, k, v, r, y);
}

}  // extern "C"

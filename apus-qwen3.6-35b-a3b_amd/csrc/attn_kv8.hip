// attn_kv8.hip -- gated-GQA decode over the 8-bit KV cache (kv8.h): for each
// new token and head, q = RoPE((1+w) RMSNorm(q)) and
//   y = sigmoid(gate) * sum_j p_j v_j,  p = softmax(q . k_j / 16, j <= position),
// in one pass over K and V with a running reference point M and sum of the
// softmax (p = 2^(t - M), t the score times log2 e / 16).
//
// The 8 q heads of a kv head times up to 4 new tokens are the rows of the matrix
// products (one or two blocks of 16), so K and V are read once a (sequence, kv
// head) pair. The pairs' blocks are laid end to end and cut into equal runs, one
// a workgroup and as many as CUs, so that every CU reads as much however ragged
// the contexts are; a run that crosses a pair's border is two segments. The 8
// wavefronts of a workgroup take every eighth block of a segment, each with its
// own M, sum and outputs in registers, and meet in LDS at its end. A segment
// that is a whole pair writes y; others keep 32 rows of (M, sum, outputs) in
// slot pair + run (no two segments share one), and k_kv8_combine joins them.
//
// A wavefront has no LDS traffic in its loop: K's and V's bytes come in operand
// order (16-byte loads, whole KiB), widen in registers (exactly: K's codes to fp16,
// V's times their scale to bf16), and the scores' registers are the operand of
// P V. Probabilities go to bf16 for that product (fp16 would cut those far below
// the largest).
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "apus_dev.h"
#include "apus_host.h"
#include "attn_mixer.h"
#include "kv8.h"

using namespace apus;

namespace {

constexpr int D = kKv8D, ROT = 64, GRP = 8, KEYS = kKv8Keys;
constexpr int kRows = 32;
// wavefronts of a workgroup: with two row blocks one a SIMD, for their registers
template <int NRB> constexpr int kv8_waves() { return NRB == 1 ? 8 : 4; }
constexpr float kEps = 1e-6f;
constexpr float kL2E = 1.44269504088896341f;
constexpr int QP = D + 8, AP = D + 4;        // LDS pitches of q rows and of outputs
// t may pass M by this much before M moves: 2^10 a term, far from overflow
constexpr float kSlack = 10.0f;

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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
__device__ __forceinline__ float row_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float sigmoid(float x) {
    return 1.0f / (1.0f + __builtin_amdgcn_exp2f(-x * kL2E));
}

typedef const __attribute__((address_space(1))) u32x4 *gu32x4p;

template <int NRB, int N>
__global__ __launch_bounds__(64 * kv8_waves<NRB>()) void k_kv8_attn(
    Kv8SeqsN<N> sq, Kv8Ref kv, const uint16_t *__restrict__ qg, const uint16_t *__restrict__ qn_w,
    const uint16_t *__restrict__ rope, int nkv, int total, int run, float c2, uint16_t *__restrict__ y,
    float *__restrict__ part, float2 *__restrict__ stat) {
    constexpr int kWaves = kv8_waves<NRB>();
    __shared__ __attribute__((aligned(16))) uint16_t qs[16 * NRB * QP];
    __shared__ float qsc[16 * NRB];
    __shared__ __attribute__((aligned(16))) float os[kWaves * 16 * AP];
    __shared__ float2 ml[kWaves][16 * NRB];
    __shared__ int first_nan[D];           // the first key whose v is NaN there, in the blocks not all rows see
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x1 = min(((int)blockIdx.x + 1) * run, total);
    int nx = 0;
    for (int x = (int)blockIdx.x * run; x < x1; x = nx) {
        const int s = kv8_seq_of(sq.off, sq.n, x / nkv);
        const int nb = sq.off[s + 1] - sq.off[s], local = x - nkv * sq.off[s];
        const int kvh = local / nb, b0 = local % nb, b1 = min(b0 + x1 - x, nb), pair = s * nkv + kvh;
        nx = x + b1 - b0;
        const int t0 = sq.cu[s], tq = sq.cu[s + 1] - t0, p0 = sq.pos0[s], row = sq.row[s];
        const int nh = nkv * GRP;

        // the first block's loads, under the q rows' work
        const int last = b1 - 1;
        u32x4 kr[8], vr[8];
        float ks = 0.0f, vs = 0.0f, kn = 0.0f, vn = 0.0f;
        auto at = [&](const uint8_t *base, int b) {
            return base + ((size_t)kv8_id_u(kv, row, b) * nkv + kvh) * kKv8Bytes;
        };
        auto load = [&](u32x4 (&r)[8], const uint8_t *p) {
            const gu32x4p q = (gu32x4p)(p + lane * 16);
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] = __builtin_nontemporal_load(q + i * 64);
        };
        auto scales = [&](int b, float &k_, float &v_) {
            const float *p = kv.scale + ((size_t)kv8_id_u(kv, row, b) * nkv + kvh) * 2;
            k_ = __int_as_float(sload_i32((const int32_t *)p, 8, 0));
            v_ = __int_as_float(sload_i32((const int32_t *)p, 8, 1));
        };
        int b = min(b0 + wave, last);
        load(kr, at(kv.k, b));
        load(vr, at(kv.v, b));
        scales(b, ks, vs);

        for (int i = tid; i < D; i += 64 * kWaves) first_nan[i] = 0x7fffffff;
        // q rows n = (token, head) into LDS: 16 threads a row, dims 8 e .. and 128 + 8 e ..
        for (int r = tid >> 4; r < 16 * NRB; r += 4 * kWaves) {
            const int e = tid & 15, t = r >> 3, h = kvh * GRP + (r & 7);
            u16x8 a = {}, c = {};
            if (t < tq) {
                const uint16_t *p = qg + ((size_t)(t0 + t) * nh + h) * 2 * D + e * 8;
                a = *reinterpret_cast<const u16x8 *>(p);
                c = *reinterpret_cast<const u16x8 *>(p + 128);
            }
            const u16x8 wa = *reinterpret_cast<const u16x8 *>(qn_w + e * 8);
            const u16x8 wc = *reinterpret_cast<const u16x8 *>(qn_w + 128 + e * 8);
            const uint16_t *cs = rope + (size_t)(p0 + min(t, tq - 1)) * ROT + (e & 3) * 8;
            const u16x8 co = *reinterpret_cast<const u16x8 *>(cs);
            const u16x8 si = *reinterpret_cast<const u16x8 *>(cs + ROT / 2);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss += bf2f(a[i]) * bf2f(a[i]) + bf2f(c[i]) * bf2f(c[i]);
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) ss += __shfl_xor(ss, d);
            const float rs = 1.0f / sqrtf(ss / (float)D + kEps);
            float va[8], vc[8], mx = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = bf2f(a[i]) * rs * (1.0f + bf2f(wa[i]));
                const float w = __shfl_xor(v, 4);          // the dims +-32
                const float r_ = v * bf2f(co[i]) + (e < 4 ? -w : w) * bf2f(si[i]);
                va[i] = e < 8 ? r_ : v;
                vc[i] = bf2f(c[i]) * rs * (1.0f + bf2f(wc[i]));
                mx = fmaxf(mx, fmaxf(fabsf(va[i]), fabsf(vc[i])));
            }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
            const float sc = kv8_row_scale(mx), inv = 1.0f / sc;
            f16x8 oa, oc;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                oa[i] = (_Float16)(va[i] * inv);
                oc[i] = (_Float16)(vc[i] * inv);
            }
            *reinterpret_cast<f16x8 *>(qs + r * QP + e * 8) = oa;
            *reinterpret_cast<f16x8 *>(qs + r * QP + 128 + e * 8) = oc;
            if (e == 0) qsc[r] = sc * c2;
        }
        __syncthreads();
        // k-step (i, u): dims (4 i + g) 16 + 8 u ..
        f16x8 q[NRB][8];
        float qf[NRB];                                     // scores' factor, with log2 e / 16
#pragma unroll
        for (int rb = 0; rb < NRB; rb++) qf[rb] = qsc[rb * 16 + n];
#pragma unroll
        for (int rb = 0; rb < NRB; rb++)
#pragma unroll
            for (int i = 0; i < 8; i++)
                q[rb][i] = *reinterpret_cast<const f16x8 *>(qs + (rb * 16 + n) * QP + (i / 2 * 4 + g) * 16 + i % 2 * 8);

        f32x4 acc[NRB][16];
        float M[NRB], l[NRB];
#pragma unroll
        for (int rb = 0; rb < NRB; rb++) {
            M[rb] = -INFINITY;
            l[rb] = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) acc[rb][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int j = b0 + wave; j < b1; j += kWaves) {
            const int next = min(j + kWaves, last);
            f32x4 S[NRB][2];
#pragma unroll
            for (int rb = 0; rb < NRB; rb++) S[rb][0] = S[rb][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 8; i++) {                  // key half i / 4, dims' chunks 4 (i % 4) ..
                const f16x8 ka = kv8_f16(kr[i][0], kr[i][1]), kb = kv8_f16(kr[i][2], kr[i][3]);
#pragma unroll
                for (int rb = 0; rb < NRB; rb++) {
                    S[rb][i / 4] = mfma16(ka, q[rb][i % 4 * 2], S[rb][i / 4]);
                    S[rb][i / 4] = mfma16(kb, q[rb][i % 4 * 2 + 1], S[rb][i / 4]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load(kr, at(kv.k, next));
            scales(next, kn, vn);
            __builtin_amdgcn_sched_barrier(0);
            const bool tail = (j + 1) * KEYS > p0 + 1;     // some row does not see some key
            uint32_t p[NRB][4];                            // the lane's 8 keys, bf16
#pragma unroll
            for (int rb = 0; rb < NRB; rb++) {
                float t[8];
                const float f_ = qf[rb] * ks;
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = S[rb][i / 4][i % 4] * f_;
                if (tail) {
                    const int lim = p0 + min(rb * 2 + (n >> 3), tq - 1) - j * KEYS - g * 4;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (i / 4 * 16 + i % 4 > lim) t[i] = -INFINITY;
                }
                const float mx = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])),
                                       fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
                if (__any(mx > M[rb] + kSlack)) {          // (always at a row's first keys)
                    const float m = fmaxf(M[rb], row_max(mx));
                    const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M[rb] - m);
                    M[rb] = m;
                    l[rb] *= f;
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[rb][i] *= f;
                }
                const float ref = M[rb] == -INFINITY ? 0.0f : M[rb];
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = __builtin_amdgcn_exp2f(t[i] - ref);
                l[rb] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
#pragma unroll
                for (int i = 0; i < 4; i++) p[rb][i] = pack2(t[2 * i], t[2 * i + 1]);
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
                    // out of the product, the first key of each dim kept
#pragma unroll
                    for (int i = 0; i < 8; i++)
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const uint32_t bad = kv8_nan_codes(vr[i][w]);
                            vr[i][w] &= ~bad;
                            if (bad)
                                atomicMin(&first_nan[(2 * i + w / 2) * 16 + n],
                                          j * KEYS + w % 2 * 16 + g * 4 + (__ffs((int)bad) - 1) / 8);
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bf16x8 va = kv8_bf16(vr[i][0], vr[i][1], vs), vb = kv8_bf16(vr[i][2], vr[i][3], vs);
#pragma unroll
                for (int rb = 0; rb < NRB; rb++) {
                    const bf16x8 pb = __builtin_bit_cast(bf16x8, u32x4{p[rb][0], p[rb][1], p[rb][2], p[rb][3]});
                    acc[rb][2 * i] = mfma16(va, pb, acc[rb][2 * i]);
                    acc[rb][2 * i + 1] = mfma16(vb, pb, acc[rb][2 * i + 1]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load(vr, at(kv.v, next));
            __builtin_amdgcn_sched_barrier(0);
            ks = kn;
            vs = vn;
        }

        // the wavefronts' outputs at a common reference point
#pragma unroll
        for (int rb = 0; rb < NRB; rb++) {
            l[rb] = row_sum(l[rb]);
            if (g == 0) ml[wave][rb * 16 + n] = make_float2(M[rb], l[rb]);
        }
        const bool whole = b0 == 0 && b1 == nb;
        const size_t slot = (size_t)(pair + (int)blockIdx.x) * kRows;
        const int rows = tq * GRP;
#pragma unroll
        for (int rb = 0; rb < NRB; rb++) {
            __syncthreads();
            if (rb * 16 >= rows) break;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; w++) m = fmaxf(m, ml[w][rb * 16 + n].x);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M[rb] - m);
            if (rb * 16 + n < rows) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    *reinterpret_cast<f32x4 *>(os + (wave * 16 + n) * AP + i * 16 + g * 4) = acc[rb][i] * f;
            }
            __syncthreads();
            // 64 threads a row, four dims each
#pragma unroll
            for (int r = tid >> 6; r < 16; r += kWaves) {
                const int rr = rb * 16 + r, d = lane * 4;
                if (rr >= rows) break;
                float mt = -INFINITY, lt = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; w++) mt = fmaxf(mt, ml[w][rr].x);
                f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float2 u = ml[w][rr];
                    lt += u.x == -INFINITY ? 0.0f : u.y * __builtin_amdgcn_exp2f(u.x - mt);
                    o += *reinterpret_cast<const f32x4 *>(os + (w * 16 + r) * AP + d);
                }
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (first_nan[d + e] <= p0 + (rr >> 3)) o[e] = NAN;
                if (whole) {
                    const size_t at_ = ((size_t)(t0 + (rr >> 3)) * nh + kvh * GRP + (rr & 7));
                    const uint2 gc = *reinterpret_cast<const uint2 *>(qg + at_ * 2 * D + D + d);
                    const float inv = 1.0f / lt;
                    const float o0 = o[0] * inv * sigmoid(bf2f((uint16_t)gc.x)), o1 = o[1] * inv * sigmoid(bf2f((uint16_t)(gc.x >> 16)));
                    const float o2 = o[2] * inv * sigmoid(bf2f((uint16_t)gc.y)), o3 = o[3] * inv * sigmoid(bf2f((uint16_t)(gc.y >> 16)));
                    *reinterpret_cast<uint2 *>(y + at_ * D + d) =
                        make_uint2(f2bf(o0) | (uint32_t)f2bf(o1) << 16, f2bf(o2) | (uint32_t)f2bf(o3) << 16);
                } else {
                    *reinterpret_cast<f32x4 *>(part + (slot + rr) * D + d) = o;
                    if (lane == 0) stat[slot + rr] = make_float2(mt, lt);
                }
            }
        }
        __syncthreads();                                   // (qs, ml and os are the next segment's)
    }
}

// One workgroup a (token, head) of a pair that lies in several runs: its
// segments' outputs at a common reference point, every fourth by a wavefront.
template <int N>
__global__ __launch_bounds__(256) void k_kv8_combine(Kv8SeqsN<N> sq, const float *__restrict__ part,
                                                     const float2 *__restrict__ stat,
                                                     const uint16_t *__restrict__ qg, int nkv, int run,
                                                     uint16_t *__restrict__ y) {
    __shared__ f32x4 os[4][64];
    const int nh = nkv * GRP, h = blockIdx.x % nh, tt = sq.cu[0] + blockIdx.x / nh;
    const int s = kv8_seq_of(sq.cu, sq.n, tt), kvh = h / GRP, r = (tt - sq.cu[s]) * GRP + h % GRP;
    const int nb = sq.off[s + 1] - sq.off[s], x = nkv * sq.off[s] + kvh * nb;
    const int w0 = x / run, w1 = (x + nb - 1) / run, pair = s * nkv + kvh;
    if (w0 == w1) return;                                  // (the whole pair: written already)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = lane * 4;
    const size_t at = (size_t)tt * nh + h;
    const uint2 gc = *reinterpret_cast<const uint2 *>(qg + at * 2 * D + D + d);
    const size_t slot0 = (size_t)(pair + w0) * kRows + r;
    float m = -INFINITY;
    for (int w = lane; w <= w1 - w0; w += 64) m = fmaxf(m, stat[slot0 + (size_t)w * kRows].x);
#pragma unroll
    for (int e = 32; e; e >>= 1) m = fmaxf(m, __shfl_xor(m, e));
    float l = 0.0f;
    for (int w = lane; w <= w1 - w0; w += 64) {
        const float2 u = stat[slot0 + (size_t)w * kRows];
        l += u.x == -INFINITY ? 0.0f : u.y * __builtin_amdgcn_exp2f(u.x - m);
    }
#pragma unroll
    for (int e = 32; e; e >>= 1) l += __shfl_xor(l, e);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = wave; w <= w1 - w0; w += 32) {
        f32x4 v[8];
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t a = slot0 + (size_t)min(w + 4 * i, w1 - w0) * kRows;
            v[i] = *reinterpret_cast<const f32x4 *>(part + a * D + d);
            f[i] = stat[a].x;
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (w + 4 * i <= w1 - w0 && f[i] != -INFINITY) o += v[i] * __builtin_amdgcn_exp2f(f[i] - m);
    }
    os[wave][lane] = o;
    __syncthreads();
    if (wave) return;
    o = (os[0][lane] + os[1][lane]) + (os[2][lane] + os[3][lane]);
    const float inv = 1.0f / l;
    const float o0 = o[0] * inv * sigmoid(bf2f((uint16_t)gc.x)), o1 = o[1] * inv * sigmoid(bf2f((uint16_t)(gc.x >> 16)));
    const float o2 = o[2] * inv * sigmoid(bf2f((uint16_t)gc.y)), o3 = o[3] * inv * sigmoid(bf2f((uint16_t)(gc.y >> 16)));
    *reinterpret_cast<uint2 *>(y + at * D + d) =
        make_uint2(f2bf(o0) | (uint32_t)f2bf(o1) << 16, f2bf(o2) | (uint32_t)f2bf(o3) << 16);
}

// Blocks of a sequence's context.
int32_t ctx_blocks(int32_t pos0, int32_t n) { return n > 0 ? (pos0 + n + KEYS - 1) / KEYS : 0; }

// the most runs of a launch
size_t max_runs() { return (size_t)cu_count(); }

}  // namespace

namespace apus {

int attn_kv8_check(const ApusHipAttnLayer *L, const ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                   const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                   const uint16_t *v, const ApusHipKv8Cache *kv, const uint16_t *y, Kv8Ref *r, size_t *T) {
    if (int e = attn_check_layer(L)) return e;
    if (!w) return set_error(kErrArgument, "NULL workspace");
    if (w->nkv != L->nkv || w->rot != L->rot || w->theta != L->theta)
        return set_error(kErrArgument, "the workspace was made for a layer of other dims");
    if (!k != !v) return set_error(kErrArgument, "k and v are both given or both NULL");
    if (int e = kv8_check(kv, L->nkv, B, rows, cu, pos0, k != nullptr, r, T)) return e;
    if (!*T) return kOk;
    for (size_t s = 0; s < B; s++)
        if (cu[s + 1] > cu[s] && (size_t)pos0[s] + (size_t)(cu[s + 1] - cu[s]) > w->max_pos)
            return set_error(kErrArgument, "sequence %zu reaches position %lld, the workspace's tables %zu", s,
                             (long long)pos0[s] + (cu[s + 1] - cu[s]), w->max_pos);
    if (!L->qn_w || !L->kn_w || !qg || !y) return set_error(kErrArgument, "NULL operand");
    if ((uintptr_t)qg % 16 || (uintptr_t)y % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 ||
        (uintptr_t)L->qn_w % 16 || (uintptr_t)L->kn_w % 16)
        return set_error(kErrUnsupported, "the attention operands need 16-byte alignment");
    const size_t ny = *T * L->nh * D * 2, nk = *T * L->nkv * D * 2, nb = kv->blocks * L->nkv * kKv8Bytes;
    if (kv8_overlap(y, ny, qg, 2 * ny) || (k && (kv8_overlap(y, ny, k, nk) || kv8_overlap(y, ny, v, nk))) ||
        kv8_overlap(y, ny, kv->k, nb) || kv8_overlap(y, ny, kv->v, nb) ||
        kv8_overlap(y, ny, kv->scale, kv->blocks * L->nkv * 8) ||
        kv8_overlap(y, ny, L->qn_w, D * 2) || kv8_overlap(y, ny, L->kn_w, D * 2))
        return set_error(kErrArgument, "y overlaps an input");
    return kOk;
}

int attn_decode_kv8_run(const ApusHipAttnLayer *L, ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                        const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                        const uint16_t *v, const Kv8Ref &kv, uint16_t *y) {
    const size_t nkv = L->nkv;
    if (k)
        if (int e = kv8_append_run(kv, nkv, B, rows, cu, pos0, k, nkv * D, v, nkv * D, L->kn_w, w->rope)) return e;
    return kv8_launches(B, rows, cu, pos0, [&](size_t s) { return ctx_blocks(pos0[s], cu[s + 1] - cu[s]); },
                        [&](const auto &q) {
        constexpr int N = sizeof(q.pos0) / 4;
        const size_t total = (size_t)q.off[q.n] * nkv;
        if (!total) return (int)kOk;
        int most = 0;
        for (int s = 0; s < q.n; s++) most = std::max(most, q.cu[s + 1] - q.cu[s]);
        // a block for each wavefront at least
        const size_t waves = most <= 2 ? kv8_waves<1>() : kv8_waves<2>();
        const size_t run = std::max((total + max_runs() - 1) / max_runs(), waves);
        bool split = false;
        for (int s = 0; s < q.n; s++) {
            const size_t nb = (size_t)(q.off[s + 1] - q.off[s]), x = nkv * (size_t)q.off[s];
            for (size_t h = 0; nb && !split && h < nkv; h++) split = (x + h * nb) / run != (x + (h + 1) * nb - 1) / run;
        }
        const float c2 = (float)(1.44269504088896341 / sqrt((double)D));
        auto launch = [&](auto nrb) {
            constexpr int NRB = decltype(nrb)::value;
            APUS_TIMED("k_kv8_attn",
                       k_kv8_attn<NRB, N><<<(unsigned)((total + run - 1) / run), 64 * kv8_waves<NRB>(), 0, stream()>>>(
                           q, kv, qg, L->qn_w, w->rope, (int)nkv, (int)total, (int)run, c2, y, w->part, w->stat));
        };
        if (most <= 2) launch(std::integral_constant<int, 1>{});
        else launch(std::integral_constant<int, 2>{});
        if (int e = launch_check("k_kv8_attn")) return e;
        if (!split) return (int)kOk;
        APUS_TIMED("k_kv8_combine",
                   k_kv8_combine<N><<<(unsigned)((size_t)(q.cu[q.n] - q.cu[0]) * L->nh), 256, 0, stream()>>>(
                       q, w->part, w->stat, qg, (int)nkv, (int)run, y));
        return launch_check("k_kv8_combine");
    });
}

int attn_decode_kv8_check(const ApusHipAttnLayer *L, const ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                          const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                          const uint16_t *v, const ApusHipKv8Cache *kv, const uint16_t *y, Kv8Ref *r, size_t *T) {
    if (int e = attn_kv8_check(L, w, B, rows, cu, pos0, qg, k, v, kv, y, r, T)) return e;
    if (B > w->max_seqs)
        return set_error(kErrArgument, "%zu sequences, the workspace holds %zu", B, w->max_seqs);
    size_t total = 0;
    for (size_t s = 0; s < B; s++) {
        if (cu[s + 1] - cu[s] > kRows / GRP)
            return set_error(kErrUnsupported, "decode takes 0..%d new tokens per sequence (got %d)", kRows / GRP,
                             cu[s + 1] - cu[s]);
        if (s % kKv8Seqs == 0) total = 0;
        total += (size_t)ctx_blocks(pos0[s], cu[s + 1] - cu[s]) * L->nkv;
        if (total > 0x7ff00000) return set_error(kErrUnsupported, "too many cached keys in one call");
    }
    return kOk;
}

}  // namespace apus

extern "C" {

int apus_hip_attn_kv8_work_create(const ApusHipAttnLayer *L, size_t max_seqs, size_t max_pos,
                                  ApusHipAttnKv8Work **out) {
    APUS_ENABLED();
    if (!out) return set_error(kErrArgument, "NULL output");
    *out = nullptr;
    if (int r = attn_check_layer(L)) return r;
    if (!max_seqs || max_seqs > ((size_t)1 << 24) || L->nkv > 1024 || !max_pos || max_pos > ((size_t)1 << 24))
        return set_error(kErrUnsupported, "an attention workspace for %zu sequences, %zu kv heads, %zu positions",
                         max_seqs, L->nkv, max_pos);
    if (int r = mx_ready()) return r;
    auto *w = new (std::nothrow) ApusHipAttnKv8Work{L->nkv, max_seqs, max_pos, L->rot, L->theta, current_device(),
                                                    nullptr, nullptr, nullptr, nullptr};
    if (!w) return set_error(kErrHip, "out of host memory");
    // slots: a segment's is pair + run, both below their counts in one launch
    const size_t slots = std::min<size_t>(max_seqs, kKv8Seqs) * L->nkv + max_runs();
    const size_t pb = slots * kRows * D * 4, sb = slots * kRows * 8, rb = max_pos * ROT * 2;
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
    if (int e = attn_decode_kv8_check(L, w, B, rows, cu, pos0, qg, k, v, kv, y, &r, &T)) return e;
    if (int e = mx_ready()) return e;
    if (!T) return kOk;
    return attn_decode_kv8_run(L, w, B, rows, cu, pos0, qg, k, v, r, y);
}

}  // extern "C"

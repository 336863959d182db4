// attn_kv8_fa.hip -- gated-GQA attention of any number of new tokens a sequence
// over the 8-bit KV cache (kv8.h), the formula of attn_kv8.hip.
//
// One workgroup a (tile of 32 or 16 tokens, kv head), the longest first: the 8 q
// heads times 32 tokens are 256 rows, 32 a wavefront, whose q and outputs stay in
// registers. The keys are walked once, a block at a time, with a running reference
// point M and sum of the softmax. A block's codes go from memory to registers while
// the block before is worked on, widen there (exactly: K's codes to fp16, V's times
// their scale to bf16) and come into LDS in operand order. The products run on the
// 32x32x16 MFMA with keys (or dims) on the M side: S^T = K Q^T leaves each lane 16
// scores of one row, which are the operand of O^T += V^T P^T with no exchange, if
// V's keys are laid out in the same order: lane half h takes the keys 8 q + 4 h +
// 0..3, q = 0..3, 8 a step. Roundings (q to fp16, probabilities to bf16, their
// sum) as in attn_kv8.hip.
//
// Bound by the matrix cores under load: a prompt of 8192 tokens, 550 GFLOP in 483 to
// 505 us from card to card, 1.09 to 1.14 PFLOP/s of the 1.24 to 1.36 that a large bf16
// product reaches here, at 1.85 to 2.0 GHz (power). A step of 32 keys is 2048 cycles of MFMA and some 3200 in
// all: the softmax's exponents and packing stand between the two products of a
// wavefront, and the other wavefront of its SIMD fills only part of that. Slower:
// products of one step interleaved with the softmax of the next, q partly in LDS
// for it (538 us against 497 then), wavefronts half a step apart (540), one operand
// read ahead instead of two (527; three and four 495 and 499), 64 rows a wavefront
// (spills). Short calls are bound by a tile's start and end, some 13 us together.
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "apus_dev.h"
#include "apus_host.h"
#include "attn_mixer.h"
#include "kv8.h"

using namespace apus;

namespace {

constexpr int D = kKv8D, ROT = 64, GRP = 8, KEYS = kKv8Keys;
constexpr int kWaves = 8;
constexpr int kAhead = 2;                    // operands read ahead of their products
constexpr int KP = D * 2 + 16;               // LDS pitches (bytes): a key's K row, a dim's V row
constexpr int VP = KEYS * 2 + 16;
constexpr int kYP = D + 16;                  // of half a row of y
constexpr float kEps = 1e-6f, kL2E = 1.44269504088896341f;
constexpr float kSlack = 10.0f;              // as in attn_kv8.hip

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef kv8_bf16x8 bf16x8;
typedef kv8_f16x8 f16x8;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// 4 e4m3 codes times a power of two as bf16
__device__ __forceinline__ u32x2 widen4(uint32_t a, float s) {
    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false);
    const bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true);
    return u32x2{__builtin_bit_cast(uint32_t, p), __builtin_bit_cast(uint32_t, q)};
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
// over the two lanes of a row, 32 apart
template <class F> __device__ __forceinline__ float pair32(float x, F f) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max32(float x) {
    return pair32(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum32(float x) {
    return pair32(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

typedef const __attribute__((address_space(1))) u32x4 *gu32x4p;

constexpr int kPartRows = 128;               // rows of a part: of a tile of 16 tokens and a kv head

struct Step {
    u32x4 k, v;                              // a thread's pieces of a block
    f32x2 sc;                                // its scales, K's and V's
};
__device__ __forceinline__ float uni(float x) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

// KS 1: the 8 wavefronts have 32 rows each, of 32 tokens. KS 2: 16 tokens, and
// wavefronts w and w + 4 have the same rows, the even and the odd blocks of the
// keys, and join what they have at the end: half the chain of steps, for calls
// whose longest tile would take longer than their work spread over the chip. If
// that is not enough a tile's keys go to several workgroups (KS 2 only), which leave
// outputs, M and sum in slot item - split0 for k_kv8_fa_combine.
template <int KS, int N>
__global__ __launch_bounds__(64 * kWaves, 2) void k_kv8_fa(Kv8SeqsN<N> sq, Kv8Cut<N> cut, Kv8Ref kv, const uint16_t *__restrict__ qg,
                                                           const uint16_t *__restrict__ qn_w,
                                                           const uint16_t *__restrict__ rope, int nkv,
                                                           uint16_t *__restrict__ y, int split0,
                                                           float *__restrict__ part, float2 *__restrict__ stat) {
    constexpr int kKl = KEYS * KP, kVl = D * VP, kRowBlocks = kWaves / KS, kTok = 4 * kRowBlocks;
    // two buffers of KS blocks' K and V; then outputs that meet: 64 registers of 8 wavefronts
    __shared__ __attribute__((aligned(16))) char lds[2 * KS * (kKl + kVl)];
    static_assert(2 * KS * (kKl + kVl) >= (KS == 1 ? kWaves * 32 * kYP : kWaves * 64 * (64 * 4 + 8)), "room for outputs");
    static_assert(32 * kYP <= 16384, "half a wavefront's rows where 64 registers of it were");
    auto kl = [&](int buf, int u) { return lds + (buf * KS + u) * kKl; };
    auto vl = [&](int buf, int u) { return lds + 2 * KS * kKl + (buf * KS + u) * kVl; };
    __shared__ int first_nan[D], any_nan;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rblk = wave % kRowBlocks, kg = wave / kRowBlocks;
    const int kvh = blockIdx.x % nkv, item = ((int)gridDim.x - 1 - (int)blockIdx.x) / nkv;
    const Kv8At a = kv8_find<false>(sq, item);
    const int parts = KS == 1 ? 1 : cut.parts[a.s], tile = (item - a.off) / parts, pt = (item - a.off) % parts;
    const int t0 = a.t0, ns = a.blocks / parts * kTok - cut.lack[a.s], p0 = a.p0, row = a.row, nh = nkv * GRP;
    const int f0 = tile * kTok;                            // the tile's first token in its sequence
    const int end = p0 + min(f0 + kTok, ns);               // keys that some row sees
    const int ctx = p0 + ns, nbt = (end + KEYS - 1) / KEYS;
    // this workgroup's blocks (none, where a tile has fewer than parts)
    const int b0 = nbt * pt / parts, nb = nbt * (pt + 1) / parts, steps = (nb - b0 + KS - 1) / KS, last = KS == 1 ? nb - 1 : max(nb - 1, 0);
    if (tid < D) first_nan[tid] = 0x7fffffff;
    if (tid == 0) any_nan = 0;

    Step next;                                             // (one block at a time: KS 2 brings its second after the scores)
    // Block ids and scales by vector loads (of a zero offset that the compiler does
    // not know): scalar loads count where LDS reads do, and out of order, so that
    // every wait for an LDS operand would be one for them too.
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));
    const uint32_t tid16 = (uint32_t)tid * 16;
    auto id_of = [&](int b) {
        const size_t at = (size_t)row * kv.bstride + b;
        return kv.btab ? *(const __attribute__((address_space(1))) uint32_t *)((const char *)(kv.btab + at) + zero) : (uint32_t)at;
    };
    uint32_t id[KS];
#pragma unroll
    for (int u = 0; u < KS; u++) id[u] = id_of(min(b0 + u, last));
    auto fetch = [&](int st, int u) {
        const size_t hb = (size_t)min((uint32_t)__builtin_amdgcn_readfirstlane(id[u]), kv.blocks - 1) * nkv + kvh;
        next.k = *(gu32x4p)(kv.k + hb * kKv8Bytes + tid16);
        next.v = *(gu32x4p)(kv.v + hb * kKv8Bytes + tid16);
        next.sc = *(const __attribute__((address_space(1))) f32x2 *)((const char *)(kv.scale + hb * 2) + zero);
        id[u] = id_of(min(b0 + (st + 1) * KS + u, last));
    };
    // a thread's pieces (kv8.h) to their places in LDS
    float cs = 0.0f;                                       // of this wavefront's block: K's scale,
    int up = 0;                                            // and kv8_v_up
    auto put = [&](int st, int u, int buf) {
        const float vs = uni(next.sc[1]);
        char *const kd = kl(buf, u) + (tid / 256 * 16 + tid % 16) * KP + tid / 16 % 16 * 32;
        *reinterpret_cast<f16x8 *>(kd) = kv8_f16(next.k[0], next.k[1]);
        *reinterpret_cast<f16x8 *>(kd + 16) = kv8_f16(next.k[2], next.k[3]);
        const int g = tid / 16 % 4, d = tid / 64 * 32 + tid % 16, b = b0 + st * KS + u;
        u32x4 c4 = next.v;
        const int k0 = b * KEYS + g * 4;               // the piece's keys: k0 .. + 3 and 16 on
        if ((b + 1) * KEYS > p0 + f0) {                // some row does not see some key
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const int left = ctx - (k0 + w % 2 * 16);      // past the last token: zero
                c4[w] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
                const uint32_t bad = kv8_nan_codes(c4[w]);
                if (bad) {                             // out of the product, its first key kept
                    c4[w] &= ~bad;
                    any_nan = 1;
                    atomicMin(&first_nan[d + w / 2 * 16], k0 + w % 2 * 16 + (__ffs((int)bad) - 1) / 8);
                }
            }
        }
        // four keys from 4 G: half G % 2, step G / 4, its first or second four
        char *const vd = vl(buf, u) + d * VP + g % 2 * 16 + g / 2 * 8;
#pragma unroll
        for (int w = 0; w < 4; w++)
            *reinterpret_cast<u32x2 *>(vd + (w / 2 * 16 * VP + w % 2 * 32)) = widen4(c4[w], vs);
        if (KS == 1 || u == kg) {
            cs = uni(next.sc[0]);
            up = kv8_v_up(vs);
        }
    };
    fetch(0, 0);

    // the wavefront's q rows n = (token 4 rblk + n / 8, head n % 8): k-step i, dims 16 i + 8 hf ..
    const int tok = f0 + rblk * 4 + (n >> 3), h = kvh * GRP + (n & 7);
    const int pos = p0 + min(tok, ns - 1);
    // (KS 2: wavefronts of the same rows form half of the dims each and exchange them;
    // both forming all took 22.3 us for 16 tokens after 240, so 19.6)
    constexpr int QI = 16 / KS;
    const int c0 = KS == 1 ? 0 : kg * QI;                  // the first of its k-steps
    f16x8 q[16];
    float qf;                                              // scores' factor, a power of two (log2 e is in q)
    {
        const uint16_t *qr = qg + ((size_t)(t0 + min(tok, ns - 1)) * nh + h) * 2 * D + c0 * 16 + hf * 8;
        // (every load at once: the outputs' registers are free yet)
        u16x8 x[QI], w[QI], co[2], si[2];
#pragma unroll
        for (int i = 0; i < QI; i++) x[i] = *reinterpret_cast<const u16x8 *>(qr + i * 16);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            co[i] = *reinterpret_cast<const u16x8 *>(rope + (size_t)pos * ROT + i * 16 + hf * 8);
            si[i] = *reinterpret_cast<const u16x8 *>(rope + (size_t)pos * ROT + ROT / 2 + i * 16 + hf * 8);
        }
#pragma unroll
        for (int i = 0; i < QI; i++) w[i] = *reinterpret_cast<const u16x8 *>(qn_w + (c0 + i) * 16 + hf * 8);
        __builtin_amdgcn_sched_barrier(0);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < QI; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) ss += bf2f(x[i][e]) * bf2f(x[i][e]);
        ss = sum32(ss);
        float o[QI][8], mq = 0.0f;                         // (1 + w) x and its RoPE; the norm's factor comes later
#pragma unroll
        for (int i = 0; i < QI; i++) {                     // (or their fp32 values are kept from the sum)
            u32x4 t = __builtin_bit_cast(u32x4, x[i]);
            asm volatile("" : "+v"(t));
            x[i] = __builtin_bit_cast(u16x8, t);
        }
#pragma unroll
        for (int i = 0; i < QI; i++) {
#pragma unroll
            for (int e = 0; e < 8; e++) o[i][e] = bf2f(x[i][e]) * (1.0f + bf2f(w[i][e]));
            __builtin_amdgcn_sched_barrier(0);
        }
        if (KS == 1 || kg == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++)                    // RoPE: with the chunk 32 dims on
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float u = o[i][e], v = o[i + 2][e], c = bf2f(co[i][e]), s_ = bf2f(si[i][e]);
                    o[i][e] = u * c - v * s_;
                    o[i + 2][e] = v * c + u * s_;
                }
        }
#pragma unroll
        for (int i = 0; i < QI; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) mq = fmaxf(mq, fabsf(o[i][e]));
        mq = max32(mq);
        f16x8 *const ex = reinterpret_cast<f16x8 *>(lds) + lane;       // [wavefront][k-step][lane]
        if (KS == 2) {
            float2 *const sm = reinterpret_cast<float2 *>(lds + kWaves * QI * 1024) + n;
            if (hf == 0) sm[wave * 32] = make_float2(ss, mq);
            __syncthreads();
            const float2 u = sm[(wave ^ kRowBlocks) * 32];
            ss += u.x;
            mq = fmaxf(mq, u.y);
        }
        const float rs = 1.0f / sqrtf(ss / (float)D + kEps);
        // (so the scores' factors are exact, and a score less M, by fma, is what M was
        // formed from: a rounded product's residual of a score past 2^31 gave infinities)
        const float sc = kv8_row_scale(mq * rs), inv = kL2E / sc;
        qf = sc / 16.0f;
        f16x8 mine[QI];
#pragma unroll
        for (int i = 0; i < QI; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) mine[i][e] = (_Float16)(o[i][e] * rs * inv);
        if (KS == 1) {
#pragma unroll
            for (int i = 0; i < QI; i++) q[i] = mine[i];
        } else {
#pragma unroll
            for (int i = 0; i < QI; i++) ex[(wave * QI + i) * 64] = mine[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; i++) q[i] = ex[((rblk + i / QI * kRowBlocks) * QI + i % QI) * 64];
        }
    }
    __syncthreads();                                       // (first_nan is clear)
    put(0, 0, 0);
    if (KS == 2) {
        fetch(0, 1);
        put(0, 1, 0);
    }

    f32x16 acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][e] = 0.0f;
    float M = -INFINITY, l = 0.0f;
    const int wfirst = p0 + min(f0 + rblk * 4, ns - 1), wlast = p0 + min(f0 + rblk * 4 + 3, ns - 1);
    for (int st = 0; st < steps; st++) {
        const int buf = st & 1, k0 = (b0 + st * KS + kg) * KEYS;
        const float csn = cs;
        const int upn = up;
        fetch(min(st + 1, steps - 1), 0);
        __syncthreads();
        bf16x8 pb[2];
        const char *vp = vl(buf, kg) + n * VP + hf * 16;
        auto v_of = [&](int i) { return *reinterpret_cast<const bf16x8 *>(vp + i % 8 * 32 * VP + i / 8 * 32); };
        const bool work = k0 <= wlast && (KS == 1 || k0 < nb * KEYS);
        if (work) {                                        // (wave-uniform)
            f32x16 S;
#pragma unroll
            for (int e = 0; e < 16; e++) S[e] = 0.0f;
            const char *kp = kl(buf, kg) + n * KP + hf * 16;
            auto k_of = [&](int i) { return *reinterpret_cast<const f16x8 *>(kp + i * 32); };
            f16x8 kf[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) kf[i] = k_of(i);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                S = mfma32(kf[i % kAhead], q[i], S);
                if (i + kAhead < 16) kf[i % kAhead] = k_of(i + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
            // (at least the smallest normal: 0 would make a NaN of a masked -inf)
            const float sf = fmaxf(qf * csn, 0x1p-126f);
            if (k0 + KEYS > wfirst + 1) {
                int tl = threadIdx.x;
                asm volatile("" : "+v"(tl));
                const int lim = p0 + min(f0 + rblk * 4 + ((tl & 31) >> 3), ns - 1) - k0 - 4 * ((tl >> 5) & 1);
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (8 * (e / 4) + e % 4 > lim) S[e] = -INFINITY;
            }
            float mx = S[0];
#pragma unroll
            for (int e = 1; e < 16; e++) mx = fmaxf(mx, S[e]);
            mx = mx * sf + (float)upn;
            if (__any(mx > M + kSlack)) {
                const float m = fmaxf(M, max32(mx));
                const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - m);
                M = m;
                l *= f;
#pragma unroll
                for (int i = 0; i < 8; i++) acc[i] *= f;
            }
            const float ref = M == -INFINITY ? 0.0f : M;
            uint32_t p[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float x0 = __builtin_amdgcn_exp2f(fmaf(S[e], sf, -ref)), x1 = __builtin_amdgcn_exp2f(fmaf(S[e + 1], sf, -ref));
                p[e / 2] = pack2(x0, x1);
                l += __uint_as_float(p[e / 2] << 16) + __uint_as_float(p[e / 2] & 0xffff0000u);   // (the rounded ones)
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
                pb[i] = __builtin_bit_cast(bf16x8, u32x4{p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]});
        }
        if (KS == 2 && st + 1 < steps) {
            put(st + 1, 0, buf ^ 1);
            fetch(st + 1, 1);
        }
        if (work) {
            bf16x8 vf[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) vf[i] = v_of(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                acc[i % 8] = mfma32(vf[i % kAhead], pb[i / 8], acc[i % 8]);
                if (i + kAhead < 16) vf[i % kAhead] = v_of(i + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (st + 1 < steps) put(st + 1, KS - 1, buf ^ 1);
    }
    __syncthreads();                                       // (first_nan is whole)
    l = sum32(l);
    // (formed again: kept, they took registers from the loop)
    int tl = threadIdx.x;
    asm volatile("" : "+v"(tl));
    const int ln = tl & 63, hf_ = ln >> 5, row_ = ln & 31, pos_ = p0 + f0 + rblk * 4 + (row_ >> 3);
    const bool nans = any_nan != 0;
    auto with_nans = [&](f32x16 &t, int d) __attribute__((always_inline)) {
        if (nans) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (first_nan[d + e / 4 * 8 + 4 * hf_ + e % 4] <= pos_) t[e] = NAN;
        }
    };
    // Half of the dims of the wavefront's rows, from dim d0: f t sigmoid(gate). A lane
    // holds four dims here and there of one row, so the gates come and y goes as whole
    // lines through LDS (8.5 KiB of this wavefront's own; straight from the lanes, 16
    // bytes of 32 rows an instruction, the end of a tile of 32 tokens took 31000 cycles).
    auto finish = [&](f32x16 (&t)[4], int d0, float f, char *buf) __attribute__((always_inline)) {
        // chunk j: the row 4 j + ln / 16, so token j / 2
        auto at = [&](int j) {
            return (size_t)(t0 + min(f0 + rblk * 4 + j / 2, ns - 1)) * nh + kvh * GRP + j % 2 * 4 + ln / 16;
        };
        char *const mine = buf + row_ * kYP + hf_ * 8, *const line = buf + ln / 16 * kYP + ln % 16 * 16;
        u32x4 gl[8];
#pragma unroll
        for (int j = 0; j < 8; j++) gl[j] = *reinterpret_cast<const u32x4 *>(qg + at(j) * 2 * D + D + d0 + ln % 16 * 8);
#pragma unroll
        for (int j = 0; j < 8; j++) *reinterpret_cast<u32x4 *>(line + j * 4 * kYP) = gl[j];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            with_nans(t[i], d0 + 32 * i);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                u32x2 *const p = reinterpret_cast<u32x2 *>(mine + i * 64 + c * 16);
                const u32x2 g = *p;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float gv = __uint_as_float(e % 2 ? g[e / 2] & 0xffff0000u : g[e / 2] << 16);
                    v[e] = t[i][4 * c + e] * f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-gv * kL2E));
                }
                *p = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (f0 + rblk * 4 + j / 2 < ns)
                *reinterpret_cast<u32x4 *>(y + at(j) * D + d0 + ln % 16 * 8) = *reinterpret_cast<u32x4 *>(line + j * 4 * kYP);
    };
    if (KS == 1) {
        const float inv = 1.0f / l;
        char *const buf = lds + wave * 32 * kYP;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            f32x16 t[4] = {acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
            finish(t, 128 * i, inv, buf);
        }
        return;
    }
    // KS 2: two wavefronts have the same rows; each finishes half of the dims
    float *const os = reinterpret_cast<float *>(lds) + ln;
    float2 *const ml = reinterpret_cast<float2 *>(lds + kWaves * 64 * 64 * 4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f32x16 t = kg ? acc[i] : acc[4 + i];
#pragma unroll
        for (int e = 0; e < 16; e++) os[wave * 4096 + (i * 16 + e) * 64] = t[e];
    }
    ml[tl] = make_float2(M, l);
    __syncthreads();
    const int other = wave ^ kRowBlocks;
    const float2 o = ml[other * 64 + ln];
    const float m = fmaxf(M, o.x);
    const float fa = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - m);
    const float fb = o.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(o.x - m);
    f32x16 t[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        t[i] = kg ? acc[4 + i] : acc[i];
#pragma unroll
        for (int e = 0; e < 16; e++) t[i][e] = t[i][e] * fa + os[other * 4096 + (i * 16 + e) * 64] * fb;
    }
    if (parts > 1) {                                       // as they lie in the lanes: whole KiB
        const size_t slot = (size_t)(item - split0) * nkv + kvh;
        float *const p = part + (slot * kWaves + wave) * 4096 + ln * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            with_nans(t[i], 128 * kg + 32 * i);
#pragma unroll
            for (int c = 0; c < 4; c++)
                *reinterpret_cast<f32x4 *>(p + (i * 4 + c) * 256) =
                    f32x4{t[i][4 * c], t[i][4 * c + 1], t[i][4 * c + 2], t[i][4 * c + 3]};
        }
        if (wave < kRowBlocks && hf_ == 0) stat[slot * kPartRows + rblk * 32 + row_] = make_float2(m, l * fa + o.y * fb);
        return;
    }
    finish(t, 128 * kg, 1.0f / (l * fa + o.y * fb), lds + other * 16384);      // (where only this wavefront reads)
}

// Joins the parts of the split tiles. A wavefront, or SP of them with parts apart,
// has 1 KiB of each part: four dims of 32 rows and two lane halves. sq: off counts
// tiles, pos0 is the number of parts and row the first slot.
template <int SP, int N>
__global__ __launch_bounds__(256) void k_kv8_fa_combine(Kv8SeqsN<N> sq, Kv8Cut<N> cut, const float *__restrict__ part,
                                                        const float2 *__restrict__ stat,
                                                        const uint16_t *__restrict__ qg, int nkv,
                                                        uint16_t *__restrict__ y) {
    constexpr int kTok = 16, kTasks = 128 * SP / 4;        // workgroups a tile and kv head
    const int ln = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = wv % SP;
    const int kvh = blockIdx.x / kTasks % nkv, g = blockIdx.x / kTasks / nkv;
    const int task = (int)(blockIdx.x % kTasks) * (4 / SP) + wv / SP, w = task / 16, ch = task % 16;
    const Kv8At a = kv8_find<false>(sq, g);
    const int parts = a.p0, tile = g - a.off, ns = a.blocks * kTok - cut.lack[a.s];
    const int r = w % 4 * 32 + (ln & 31), tok = tile * kTok + r / 8;
    const int d = w / 4 * 128 + ch / 4 * 32 + ch % 4 * 8 + ln / 32 * 4;
    const size_t at = (size_t)(a.t0 + min(tok, ns - 1)) * nkv * GRP + kvh * GRP + r % 8;
    const uint2 gate = *reinterpret_cast<const uint2 *>(qg + at * 2 * D + D + d);
    const size_t slot0 = (size_t)(a.row + tile * parts) * nkv + kvh;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = share; j < parts; j += 8 * SP) {
        f32x4 v[8];
        float2 u[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t s = slot0 + (size_t)min(j + i * SP, parts - 1) * nkv;
            v[i] = *reinterpret_cast<const f32x4 *>(part + (s * kWaves + w) * 4096 + ch * 256 + ln * 4);
            u[i] = stat[s * kPartRows + r];
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
            if (j + i * SP >= parts) continue;
            const float f = u[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(u[i].x - m);   // (0 keeps a NaN)
            l += u[i].y * f;
            o += v[i] * f;
        }
    }
    if (SP > 1) {
        __shared__ f32x4 os[4][64];
        __shared__ float2 st[4][64];
        os[wv][ln] = o;
        st[wv][ln] = make_float2(m, l);
        __syncthreads();
        if (share) return;
        float mt = -INFINITY;
#pragma unroll
        for (int i = 0; i < SP; i++) mt = fmaxf(mt, st[wv + i][ln].x);
        l = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < SP; i++) {
            const float2 u = st[wv + i][ln];
            const float f = u.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(u.x - mt);
            l += u.y * f;
            o += os[wv + i][ln] * f;
        }
    }
    if (tok >= ns) return;
    const float inv = 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float gv = bf2f((uint16_t)((e < 2 ? gate.x : gate.y) >> (16 * (e % 2))));
        o[e] *= inv * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-gv * kL2E));
    }
    *reinterpret_cast<uint2 *>(y + at * D + d) = make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
}

}  // namespace

extern "C" {

int apus_hip_attn_prefill_kv8(const ApusHipAttnLayer *L, ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                              const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                              const uint16_t *v, const ApusHipKv8Cache *kv, uint16_t *y) {
    APUS_ENABLED();
    Kv8Ref r;
    size_t T = 0;
    if (int e = attn_kv8_check(L, w, B, rows, cu, pos0, k || v, kv, &r, &T)) return e;
    if (int e = attn_kv8_check_operands(L, T, qg, k, v, kv, y)) return e;
    if (int e = mx_ready()) return e;
    if (!T) return kOk;
    // up to 4 new tokens a sequence: decode's kernels, whose tiles are 16 or 32 rows
    // and not 128 (us, decode's and these: one sequence, 3 tokens after 100 10 and 19;
    // 2 after 60000 20 and 47; 64, 4 after 8000 106 and 194)
    if (attn_decode_kv8_fits(w, B, cu, pos0)) return attn_decode_kv8_run(L, w, B, rows, cu, pos0, qg, k, v, r, y);
    const size_t nkv = L->nkv;
    if (k)
        if (int e = kv8_append_run(r, nkv, B, rows, cu, pos0, k, nkv * D, v, nkv * D, L->kn_w, w->rope)) return e;
    const Kv8Plan plan = kv8_fa_plan(B, cu, pos0, nkv, w->rows / kPartRows, (size_t)cu_count());
    return kv8_launches(B, rows, cu, pos0, [&](size_t s) { return (cu[s + 1] - cu[s] + plan.tok - 1) / plan.tok; },
                        [&](auto &q) {
        constexpr int N = sizeof(q.e) / sizeof(q.e[0]) - 1;
        if (!q.e[q.n].off) return (int)kOk;
        const Kv8Cut<N> cut = kv8_by_length(q, plan);
        const size_t grid = (size_t)q.e[q.n].off * nkv;
        const int split0 = q.e[kv8_first_split(q, cut)].off;
        auto launch = [&](auto ks) {
            APUS_TIMED("k_kv8_fa", k_kv8_fa<decltype(ks)::value, N><<<(unsigned)grid, 64 * kWaves, 0, stream()>>>(
                                       q, cut, r, qg, L->qn_w, w->rope, (int)nkv, y, split0, w->part, w->stat));
            return launch_check("k_kv8_fa");
        };
        if (plan.tok == 32) return launch(std::integral_constant<int, 1>{});
        if (int e = launch(std::integral_constant<int, 2>{})) return e;
        if (split0 == q.e[q.n].off) return (int)kOk;
        const Kv8Joins<N> j = kv8_joins(q, cut);
        auto combine = [&](auto sp) {
            constexpr int SP = decltype(sp)::value;
            APUS_TIMED("k_kv8_fa_combine",
                       k_kv8_fa_combine<SP, N><<<(unsigned)((size_t)j.tiles * nkv * 32 * SP), 256, 0, stream()>>>(
                           j.sq, j.cut, w->part, w->stat, qg, (int)nkv, y));
            return launch_check("k_kv8_fa_combine");
        };
        return j.most <= 8 ? combine(std::integral_constant<int, 1>{}) : combine(std::integral_constant<int, 4>{});
    });
}

}  // extern "C"

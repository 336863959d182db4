// kv8.hip -- the 8-bit KV cache (kv8.h): rows written into it as e4m3 codes
// with a power-of-two scale a block of 32 positions and kv head, and read back.
//
// The scale of a block is 2^e, e the smallest integer with amax <= 448 2^e (448
// is e4m3's largest value) over the positions written, at least -117. A code is
// x / 2^e rounded to nearest even: half a step, 2^-4 of a normal value. A block
// that gets more tokens keeps those before them: where the new ones need a
// larger scale its codes are rounded again at that scale, which moves their
// exponents and is exact but for values that become subnormal (below 2^-6 of the
// scale). The scale of a block that is being filled never falls: tokens taken
// back (positions written again) keep their mark on it. An infinity or NaN
// becomes the NaN code and does not count in the scale. At the largest scale, 2^120,
// codes end at 240: 256 2^120 is past bf16 (and fp32), so finite values from 248 2^120
// on, which would round there, take 240 (at most 15 of their 255 steps off: within
// half a step, 2^-4).
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>

#include "apus_dev.h"
#include "apus_host.h"
#include "kv8.h"

using namespace apus;

namespace {

constexpr int D = kKv8D, ROT = 64, KEYS = kKv8Keys;
constexpr float kEps = 1e-6f;

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// 4 bf16 codes (two dwords) / scale as e4m3 codes
__device__ __forceinline__ uint32_t to_fp8(uint32_t a, uint32_t b, float scale) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, a), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), scale, true);
    return __builtin_bit_cast(uint32_t, r);
}
// 4 e4m3 codes times scale as bf16 codes
__device__ __forceinline__ u32x2 from_fp8(uint32_t c, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
// codes at a scale 2^up times as large (from the values themselves: one rounding)
__device__ __forceinline__ uint32_t rescale(uint32_t c, float up) {
    const u32x2 v = from_fp8(c, 1.0f);
    return to_fp8(v[0], v[1], up);
}

// codes past 240 as 240 (0x77), NaN too
__device__ __forceinline__ uint32_t up_to_240(uint32_t c) {
    const uint32_t over = ((((c & 0x7f7f7f7fu) + 0x08080808u) & 0x80808080u) >> 7) * 0x7fu;
    return (c & ~over) | (0x77777777u & over);
}

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent of the scale for a largest magnitude of bf16 code m:
// (1 + f / 128) 2^(x - 127) <= 1.75 2^(8 + e).
__device__ __forceinline__ int scale_exp(uint32_t m) {
    const int x = (int)(m >> 7), f = (int)(m & 127);
    return max(x - 135 + (f > 96 ? 1 : 0), kKv8MinExp);
}

// One workgroup a (block, kv head, K or V): its new rows, 32 at most, in
// registers (a thread has 8 dims of four rows), normed and roped for K where the
// layer's weights are given, their largest magnitude, the codes. K's bytes go
// straight to their places, 8 a time; V's go through LDS, where a thread
// gathers the 16 of a piece, and a block that is not written as a whole brings
// its old pieces with the rows (one round of loads in all). Bound by HBM for large
// fills (2.1 million tokens of 2 heads, 4.3 GB in and 2.15 out: 1.30 ms, 5.0 TB/s);
// a prompt of 8192 tokens, 25 MB, takes 7.1 us, of which 3.6 are launch, loads and
// stores of a single block, one after the other. With K's norm and RoPE a single block
// takes 7.0 (the ordered sum of a row's 256 squares, by a thread a row while the others
// wait, weights and RoPE rows after it), 128 sequences of 1 to 4 tokens 13, 8192 tokens
// 17.
template <bool NORM, int N>
__global__ __launch_bounds__(256) void k_kv8_append(Kv8SeqsN<N> sq, Kv8Ref kv, const uint16_t *__restrict__ k,
                                                    size_t ldk, const uint16_t *__restrict__ v, size_t ldv,
                                                    int nkv, const uint16_t *__restrict__ kn_w,
                                                    const uint16_t *__restrict__ rope) {
    constexpr int RP = D + 8, CP = D + 4;          // pitches: rows on distinct banks
    __shared__ __attribute__((aligned(16))) char lds[NORM ? KEYS * RP * 2 : KEYS * CP];
    __shared__ float rs[KEYS];
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x, which = blockIdx.x & 1, kvh = (blockIdx.x >> 1) % nkv;
    const int item = (blockIdx.x >> 1) / nkv;
    const Kv8At a = kv8_find<false>(sq, item);
    const int p0 = a.p0, ns = a.tokens, b = p0 / KEYS + item - a.off;
    const int lo = max(p0 - b * KEYS, 0), hi = min(p0 + ns - b * KEYS, KEYS);
    const int t0 = a.t0 + b * KEYS - p0;       // the token of the block's first position
    const uint32_t id = kv8_id(kv, a.row, b);
    if (kv.btab && (uint32_t)kv.btab[(size_t)a.row * kv.bstride + b] != id) return;   // a stale entry
    const size_t hb = (size_t)id * nkv + kvh;
    uint8_t *const blk = (which ? kv.v : kv.k) + hb * kKv8Bytes;
    float *const sc = kv.scale + hb * 2 + which;
    const int r0 = tid >> 5, pc = tid & 31;        // rows r0 + 8 i, dims 8 pc ..
    u16x8 x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = min(max(r0 + 8 * i, lo), hi - 1);
        const size_t t = (size_t)(t0 + r);
        x[i] = *reinterpret_cast<const u16x8 *>((which ? v + t * ldv : k + t * ldk) + kvh * D + pc * 8);
    }
    float old_s = lo > 0 ? *sc : 0.0f;
    u32x4 old[2];
    if (which && (lo > 0 || hi < KEYS)) {
#pragma unroll
        for (int j = 0; j < 2; j++) old[j] = *reinterpret_cast<const u32x4 *>(blk + (tid + 256 * j) * 16);
    }
    if (NORM && !which) {
        // (1+w) RMSNorm with the sum in the reference's order (c/attn.h:175-186)
        // and the partial RoPE (c/attn.h:244-266), rounded where they round:
        // the row that the bf16 cache would hold
        uint16_t *const xs = reinterpret_cast<uint16_t *>(lds);
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<u16x8 *>(xs + (r0 + 8 * i) * RP + pc * 8) = x[i];
        __syncthreads();
        if (tid < KEYS) {
            const u16x8 *xr = reinterpret_cast<const u16x8 *>(xs + tid * RP);
            float ss = 0.0f;
#pragma unroll 4
            for (int j = 0; j < D / 8; j++) {
                const u16x8 e = xr[j];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float f = bf2f(e[i]);
                    ss = fmaf(f, f, ss);           // (f * f is exact)
                }
            }
            rs[tid] = 1.0f / sqrtf(ss / (float)D + kEps);
        }
        __syncthreads();
        constexpr int R = ROT / 2;
        const int pp = pc ^ (R / 8), i0 = (pc & (R / 8 - 1)) * 8;
        const u16x8 w = *reinterpret_cast<const u16x8 *>(kn_w + pc * 8);
        const u16x8 wp = *reinterpret_cast<const u16x8 *>(kn_w + pp * 8);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + 8 * i;
            const float rr = rs[r];
            float n[8];
#pragma unroll
            for (int e = 0; e < 8; e++) n[e] = rndf((bf2f(x[i][e]) * rr) * (1.0f + bf2f(w[e])));
            if (pc < ROT / 8) {
                const int pos = b * KEYS + min(max(r, lo), hi - 1);
                const u16x8 xp = *reinterpret_cast<const u16x8 *>(xs + r * RP + pp * 8);
                const u16x8 cv = *reinterpret_cast<const u16x8 *>(rope + (size_t)pos * ROT + i0);
                const u16x8 sv = *reinterpret_cast<const u16x8 *>(rope + (size_t)pos * ROT + R + i0);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float np = rndf((bf2f(xp[e]) * rr) * (1.0f + bf2f(wp[e])));
                    const float c = bf2f(cv[e]), sn = bf2f(sv[e]);
                    x[i][e] = f2bf(rndf(n[e] * c) + rndf((pc < R / 8 ? -np : np) * sn));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[i][e] = f2bf(n[e]);
            }
        }
    }
    // the largest finite magnitude (rows outside [lo, hi) repeat one inside it)
    uint32_t m = 0, wild = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t u = x[i][e] & 0x7fffu;
            wild |= u >= 0x7f80u;
            m = max(m, u >= 0x7f80u ? 0u : u);
        }
#pragma unroll
    for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    int e = scale_exp(m), up = 0;
    if (lo > 0) {
        const int eo = min(max((int)(__float_as_uint(old_s) >> 23 & 255) - 127, kKv8MinExp), kKv8MaxExp);
        e = max(e, eo);
        up = min(e - eo, 60);                      // (past 2^18 nothing is left of a code)
    }
    const float scale = exp2i(e), ups = exp2i(up);
    if (tid == 0) *sc = scale;
    u32x2 c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const u32x4 xi = __builtin_bit_cast(u32x4, x[i]);
        const uint32_t x0 = xi[0], x1 = xi[1], x2 = xi[2], x3 = xi[3];
        uint32_t c0 = to_fp8(x0, x1, scale), c1 = to_fp8(x2, x3, scale);
        if (e == kKv8MaxExp) c0 = up_to_240(c0), c1 = up_to_240(c1);
        if (__any((int)wild)) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if ((x[i][j] & 0x7fffu) >= 0x7f80u) c0 |= 0x7fu << (8 * j);
                if ((x[i][4 + j] & 0x7fffu) >= 0x7f80u) c1 |= 0x7fu << (8 * j);
            }
        }
        c[i] = u32x2{c0, c1};
    }
    if (!which) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + 8 * i;
            u32x2 *const at = reinterpret_cast<u32x2 *>(blk + kv8_k_at(r, pc * 8));
            if (r >= lo && r < hi) {
                *at = c[i];
            } else if (r < lo && up) {
                const u32x2 o = *at;
                const uint32_t o0 = o[0], o1 = o[1];
                *at = u32x2{rescale(o0, ups), rescale(o1, ups)};
            }
        }
        return;
    }
    uint8_t *const cs = reinterpret_cast<uint8_t *>(lds);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t *const at = reinterpret_cast<uint32_t *>(cs + (r0 + 8 * i) * CP + pc * 8);
        at[0] = c[i][0];
        at[1] = c[i][1];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int q = tid + 256 * j, g = q / 16 % 4;
        u32x4 out;
#pragma unroll
        for (int w = 0; w < 4; w++) {              // dims (w / 2) * 16 apart, keys of half w % 2
            const int d = q / 64 * 32 + w / 2 * 16 + q % 16, k0 = w % 2 * 16 + g * 4;
            uint32_t got = 0, mask = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                got |= (uint32_t)cs[(k0 + i) * CP + d] << (8 * i);
                if (k0 + i >= lo && k0 + i < hi) mask |= 0xffu << (8 * i);
            }
            uint32_t o = 0;
            if (lo > 0 || hi < KEYS) {
                o = old[j][w];
                if (up) o = rescale(o, ups);
            }
            out[w] = (got & mask) | (o & ~mask);
        }
        *reinterpret_cast<u32x4 *>(blk + q * 16) = out;
    }
}

// One workgroup a (block, kv head, K or V): the block's pieces into LDS as
// [key][d], then rows of it out, 16 bytes a thread. 8192 tokens of 2 heads, 25 MB,
// in 4.8 to 6.4 us; one block 2.2.
template <int N>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8SeqsN<N> sq, Kv8Ref kv, uint16_t *__restrict__ k, size_t ldk,
                                                  uint16_t *__restrict__ v, size_t ldv, int nkv) {
    constexpr int CP = D + 16;
    __shared__ __attribute__((aligned(16))) uint8_t cs[KEYS * CP];
    const int tid = threadIdx.x, which = blockIdx.x & 1, kvh = (blockIdx.x >> 1) % nkv;
    const int item = (blockIdx.x >> 1) / nkv;
    const Kv8At a = kv8_find<false>(sq, item);
    const int p0 = a.p0, ns = a.tokens, b = p0 / KEYS + item - a.off;
    const int lo = max(p0 - b * KEYS, 0), hi = min(p0 + ns - b * KEYS, KEYS);
    const int t0 = a.t0 + b * KEYS - p0;
    const size_t hb = (size_t)kv8_id(kv, a.row, b) * nkv + kvh;
    const uint8_t *const blk = (which ? kv.v : kv.k) + hb * kKv8Bytes;
    const float scale = kv.scale[hb * 2 + which];
    u32x4 piece[2];
#pragma unroll
    for (int j = 0; j < 2; j++) piece[j] = *reinterpret_cast<const u32x4 *>(blk + (tid + 256 * j) * 16);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int q = tid + 256 * j;
        if (!which) {
            *reinterpret_cast<u32x4 *>(cs + (q / 256 * 16 + q % 16) * CP + q / 16 % 16 * 16) = piece[j];
        } else {
            const int g = q / 16 % 4;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const int d = q / 64 * 32 + w / 2 * 16 + q % 16, k0 = w % 2 * 16 + g * 4;
#pragma unroll
                for (int i = 0; i < 4; i++) cs[(k0 + i) * CP + d] = (uint8_t)(piece[j][w] >> (8 * i));
            }
        }
    }
    __syncthreads();
    const int r0 = tid >> 5, pc = tid & 31;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = r0 + 8 * i;
        if (r < lo || r >= hi) continue;
        const u32x2 c = *reinterpret_cast<const u32x2 *>(cs + r * CP + pc * 8);
        const uint32_t c0 = c[0], c1 = c[1];
        const u32x2 x = from_fp8(c0, scale), z = from_fp8(c1, scale);
        const size_t t = (size_t)(t0 + r);
        *reinterpret_cast<u32x4 *>((which ? v + t * ldv : k + t * ldk) + kvh * D + pc * 8) = u32x4{x[0], x[1], z[0], z[1]};
    }
}

// blocks that positions pos0 .. pos0 + n - 1 touch
int32_t touched(int32_t pos0, int32_t n) { return n > 0 ? (pos0 + n - 1) / KEYS - pos0 / KEYS + 1 : 0; }

constexpr size_t kMaxPitch = (size_t)1 << 30, kMaxElements = (size_t)1 << 40;
// (block, kv head) pairs of a launch's new tokens: with two workgroups of 256 threads
// each (cache), or two of 512 (prefill: a tile of 16 tokens and a head) it stays under
// HIP's 2^32 threads. k and v of so many take 137 GB.
constexpr size_t kMaxHeadBlocks = (size_t)1 << 22;

// rows of k or v: T of them, n elements each, apart from the cache (and its table,
// where they are written)
int check_rows(const ApusHipKv8Cache *c, const void *p, size_t ld, size_t nkv, size_t T, const char *what, bool written) {
    const size_t n = nkv * D;
    if (!p) return set_error(kErrArgument, "NULL %s", what);
    if (ld < n) return set_error(kErrArgument, "%s rows of %zu elements with pitch %zu", what, n, ld);
    if (ld > kMaxPitch || ld > kMaxElements / T) return set_error(kErrUnsupported, "%zu %s rows of pitch %zu", T, what, ld);
    if ((uintptr_t)p % 16 || ld % 8)
        return set_error(kErrUnsupported, "%s rows need 16-byte alignment (pitch %zu)", what, ld);
    const size_t nb = c->blocks * nkv * kKv8Bytes;
    if (block_overlaps(c->k, nb, p, ld * 2, n * 2, T) || block_overlaps(c->v, nb, p, ld * 2, n * 2, T) ||
        block_overlaps(c->scale, c->blocks * nkv * 8, p, ld * 2, n * 2, T))
        return set_error(kErrArgument, "the %s rows overlap the cache", what);
    if (written && c->block_table && block_overlaps(c->block_table, c->max_rows * c->max_blocks * 4, p, ld * 2, n * 2, T))
        return set_error(kErrArgument, "the %s rows overlap the block table", what);
    return kOk;
}

}  // namespace

namespace apus {

bool kv8_overlap(const void *a, size_t na, const void *b, size_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

bool kv8_overlap_cache(const ApusHipKv8Cache *c, size_t nkv, const void *p, size_t n) {
    const size_t nb = c->blocks * nkv * kKv8Bytes;
    return kv8_overlap(p, n, c->k, nb) || kv8_overlap(p, n, c->v, nb) || kv8_overlap(p, n, c->scale, c->blocks * nkv * 8);
}

int kv8_check(const ApusHipKv8Cache *c, size_t nkv, size_t B, const int32_t *rows, const int32_t *cu,
              const int32_t *pos0, bool writes, Kv8Ref *r, size_t *tokens) {
    if (!c || !c->k || !c->v || !c->scale) return set_error(kErrArgument, "bad 8-bit KV cache descriptor");
    if (!nkv || nkv > kKv8MaxHeads) return set_error(kErrUnsupported, "%zu kv heads", nkv);
    if (!c->blocks || c->blocks > 0x7fffffff || !c->max_blocks || c->max_blocks > kKv8MaxBlocks ||
        !c->max_rows || c->max_rows > 0x7fffffff)
        return set_error(kErrArgument, "8-bit KV cache: %zu blocks, %zu rows of %zu", c->blocks, c->max_rows,
                         c->max_blocks);
    if (!c->block_table && c->max_rows > c->blocks / c->max_blocks)
        return set_error(kErrArgument, "%zu rows of %zu blocks in a flat cache of %zu", c->max_rows,
                         c->max_blocks, c->blocks);
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || (uintptr_t)c->scale % 8 || (uintptr_t)c->block_table % 4)
        return set_error(kErrUnsupported, "misaligned 8-bit KV cache arrays");
    const size_t nb = c->blocks * nkv * kKv8Bytes, sb = c->blocks * nkv * 8;
    if (kv8_overlap(c->k, nb, c->v, nb) || kv8_overlap(c->k, nb, c->scale, sb) || kv8_overlap(c->v, nb, c->scale, sb))
        return set_error(kErrArgument, "overlapping 8-bit KV cache arrays");
    if (c->block_table && kv8_overlap_cache(c, nkv, c->block_table, c->max_rows * c->max_blocks * 4))
        return set_error(kErrArgument, "the block table overlaps the 8-bit KV cache arrays");
    *r = Kv8Ref{c->k, c->v, c->scale, c->block_table, (int32_t)c->max_blocks, (uint32_t)c->blocks};
    *tokens = 0;
    if (!B) return kOk;
    if (B > ((size_t)1 << 24)) return set_error(kErrUnsupported, "%zu sequences", B);
    if (!cu || !pos0 || cu[0] != 0) return set_error(kErrArgument, "bad offsets");
    // the rows written to (no exception may leave an entry point)
    std::unique_ptr<int32_t[]> used(writes && rows ? new (std::nothrow) int32_t[B] : nullptr);
    if (writes && rows && !used) return set_error(kErrHip, "out of host memory");
    size_t nused = 0, heads = 0;
    for (size_t s = 0; s < B; s++) {
        const int64_t n = (int64_t)cu[s + 1] - cu[s], end = (int64_t)pos0[s] + n;
        if (n < 0) return set_error(kErrArgument, "token offsets must ascend");
        if (pos0[s] < 0 || end > (int64_t)c->max_blocks * KEYS)
            return set_error(kErrArgument, "sequence %zu overflows the cache (%d+%lld > %zu)", s, pos0[s],
                             (long long)n, c->max_blocks * KEYS);
        const int64_t row = rows ? rows[s] : (int64_t)s;
        if (row < 0 || row >= (int64_t)c->max_rows)
            return set_error(kErrArgument, "row %lld of sequence %zu is outside the cache's %zu rows",
                             (long long)row, s, c->max_rows);
        if (c->row_blocks && n) {
            const int32_t held = c->row_blocks[row];
            if (held < 0) return set_error(kErrArgument, "row %lld of sequence %zu is not open", (long long)row, s);
            if (end > (int64_t)held * KEYS)
                return set_error(kErrArgument, "sequence %zu reaches position %lld but row %lld has reserved %lld "
                                 "positions", s, (long long)end, (long long)row, (long long)held * KEYS);
        }
        if (writes && n && rows) used[nused++] = (int32_t)row;
        if (s % kKv8Seqs == 0) heads = 0;
        heads += (size_t)touched(pos0[s], (int32_t)n) * nkv;
        if (heads >= kMaxHeadBlocks)
            return set_error(kErrUnsupported, "the new tokens of %d sequences touch %zu blocks and kv heads, of up to %zu",
                             kKv8Seqs, heads, kMaxHeadBlocks - 1);
    }
    std::sort(used.get(), used.get() + nused);
    if (std::adjacent_find(used.get(), used.get() + nused) != used.get() + nused)
        return set_error(kErrArgument, "two sequences of a call write to one row");
    *tokens = (size_t)cu[B];
    return kOk;
}

int kv8_append_run(const Kv8Ref &kv, size_t nkv, size_t B, const int32_t *rows, const int32_t *cu,
                   const int32_t *pos0, const uint16_t *k, size_t ldk, const uint16_t *v, size_t ldv,
                   const uint16_t *kn_w, const uint16_t *rope) {
    return kv8_launches(B, rows, cu, pos0, [&](size_t s) { return touched(pos0[s], cu[s + 1] - cu[s]); },
                        [&](const auto &q) {
        constexpr int N = sizeof(q.e) / sizeof(q.e[0]) - 1;
        const size_t grid = (size_t)q.e[q.n].off * nkv * 2;
        if (!grid) return (int)kOk;
        if (kn_w)
            APUS_TIMED("k_kv8_append", k_kv8_append<true, N><<<(unsigned)grid, 256, 0, stream()>>>(
                                           q, kv, k, ldk, v, ldv, (int)nkv, kn_w, rope));
        else
            APUS_TIMED("k_kv8_append", k_kv8_append<false, N><<<(unsigned)grid, 256, 0, stream()>>>(
                                           q, kv, k, ldk, v, ldv, (int)nkv, nullptr, nullptr));
        return launch_check("k_kv8_append");
    });
}

}  // namespace apus

extern "C" {

int apus_hip_kv8_append(const ApusHipKv8Cache *kv, size_t nkv, size_t B, const int32_t *rows, const int32_t *cu,
                        const int32_t *pos0, const uint16_t *k, size_t ldk, const uint16_t *v, size_t ldv) {
    APUS_ENABLED();
    Kv8Ref r;
    size_t T = 0;
    if (int e = kv8_check(kv, nkv, B, rows, cu, pos0, true, &r, &T)) return e;
    if (T) {
        if (int e = check_rows(kv, k, ldk, nkv, T, "k", false)) return e;
        if (int e = check_rows(kv, v, ldv, nkv, T, "v", false)) return e;
    }
    if (int e = mx_ready()) return e;
    if (!T) return kOk;
    return kv8_append_run(r, nkv, B, rows, cu, pos0, k, ldk, v, ldv, nullptr, nullptr);
}

int apus_hip_kv8_read(const ApusHipKv8Cache *kv, size_t nkv, size_t B, const int32_t *rows, const int32_t *cu,
                      const int32_t *pos0, uint16_t *k, size_t ldk, uint16_t *v, size_t ldv) {
    APUS_ENABLED();
    Kv8Ref r;
    size_t T = 0;
    if (int e = kv8_check(kv, nkv, B, rows, cu, pos0, false, &r, &T)) return e;
    if (T) {
        if (int e = check_rows(kv, k, ldk, nkv, T, "k", true)) return e;
        if (int e = check_rows(kv, v, ldv, nkv, T, "v", true)) return e;
        if (rows_overlap(k, ldk * 2, nkv * D * 2, v, ldv * 2, nkv * D * 2, T))
            return set_error(kErrArgument, "the k rows overlap the v rows");
    }
    if (int e = mx_ready()) return e;
    if (!T) return kOk;
    return kv8_launches(B, rows, cu, pos0, [&](size_t s) { return touched(pos0[s], cu[s + 1] - cu[s]); },
                        [&](const auto &q) {
        constexpr int N = sizeof(q.e) / sizeof(q.e[0]) - 1;
        const size_t grid = (size_t)q.e[q.n].off * nkv * 2;
        if (!grid) return (int)kOk;
        APUS_TIMED("k_kv8_read", k_kv8_read<N><<<(unsigned)grid, 256, 0, stream()>>>(q, r, k, ldk, v, ldv, (int)nkv));
        return launch_check("k_kv8_read");
    });
}

}  // extern "C"

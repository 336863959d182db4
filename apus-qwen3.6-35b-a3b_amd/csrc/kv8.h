// kv8.h -- the 8-bit KV cache: its blocks, its scales, and the per-call
// metadata of the kernels that write, read and attend over it.
//
// A block holds 32 positions of one kv head as e4m3 codes, K and V 8 KiB each,
// with one power-of-two scale for K and one for V: value = code * scale. The
// bytes lie in the order in which the matrix instructions of the decode kernel
// take them (16x16x32: lane l holds row l % 16 and the 8 k of group g = l / 16),
// so that a wavefront's 16-byte loads are whole KiB and go to the matrix cores
// as they come, without a pass through LDS:
//   K, key x d: [key / 16][d / 16][key % 16][d % 16]. A 1 KiB load is 16 keys'
//     d-chunks 4 i .. 4 i + 3, lane group g the chunk 4 i + g: two k-steps of 8.
//   V, d x key: [d / 32][g][d % 16][(d / 16) % 2][8], the 8 bytes the keys
//     4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3: those that lane group g has
//     scores of after K Q^T, so the probabilities go on to P V from the
//     registers that they are formed in.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/apus_hip.h"
#include "apus_dev.h"
#include "apus_rt.h"
#include "kv8_plan.h"
#include "mx.h"

namespace apus {

constexpr int kKv8D = 256;                   // head dim
constexpr int kKv8Bytes = kKv8Keys * kKv8D;  // bytes of a head's K or V block
constexpr int kKv8MinExp = -117;             // smallest exponent of a scale: its codes' steps stay normal in bf16
constexpr int kKv8MaxExp = 120;              // the largest, that of bf16's largest values; its codes end at 240

constexpr size_t kKv8MaxHeads = 1024;        // kv heads, and blocks of a row (positions count in 32 bits)
constexpr size_t kKv8MaxBlocks = (size_t)1 << 25;

struct Kv8Ref {
    uint8_t *k, *v;
    float *scale;                            // [block][nkv][2]: K's, V's
    const int32_t *btab;                     // nullptr: flat
    int32_t bstride;                         // blocks per table row
    uint32_t blocks;                         // blocks of the arrays
};

// byte of (key, d) in a K block, of (d, key) in a V block
__host__ __device__ constexpr int kv8_k_at(int key, int d) {
    return ((key / 16) * 16 + d / 16) * 256 + (key % 16) * 16 + d % 16;
}
__host__ __device__ constexpr int kv8_v_at(int d, int key) {
    return (d / 32) * 1024 + ((key % 16) / 4 * 16 + d % 16) * 16 + (d / 16 % 2) * 8 +
           key / 16 * 4 + key % 4;
}

// The id of block b of the table row h; what the table holds past the arrays'
// blocks reads as their last block (a stale entry must not reach past them).
__device__ __forceinline__ uint32_t kv8_id(const Kv8Ref &r, int h, int b) {
    const size_t at = (size_t)h * r.bstride + b;
    return min(r.btab ? (uint32_t)r.btab[at] : (uint32_t)at, r.blocks - 1);
}
// the same for a wave-uniform (h, b), through the scalar cache
__device__ __forceinline__ uint32_t kv8_id_u(const Kv8Ref &r, int h, int b) {
    const size_t at = (size_t)__builtin_amdgcn_readfirstlane(h) * r.bstride;
    const int bu = __builtin_amdgcn_readfirstlane(b);
    const uint32_t id = r.btab ? (uint32_t)sload_i32(r.btab + at, (uint32_t)r.bstride * 4, bu)
                               : (uint32_t)at + (uint32_t)bu;
    return min(id, r.blocks - 1);
}

// A sequence of a launch: its number, entry, and what it has of blocks and tokens.
struct Kv8At {
    int s, off, blocks, t0, tokens, p0, row;
};
// The last sequence whose off (TOKEN: cu) is at most the wave-uniform x. The lanes
// look at all entries at once, so everything about it is known after one round
// of loads (with a binary search and scalar loads it was a chain of four, some
// 2 us at the start of every workgroup). Called by whole wavefronts.
template <bool TOKEN, int N> __device__ __forceinline__ Kv8At kv8_find(const Kv8SeqsN<N> &sq, int x) {
    constexpr int C = (N + 64) / 64;
    const int lane = threadIdx.x & 63;
    Kv8Seq v[C];
    int k = 0;
#pragma unroll
    for (int c = 0; c < C; c++) v[c] = sq.e[min(c * 64 + lane, N)];
#pragma unroll
    for (int c = 0; c < C; c++)
        k += __builtin_popcountll(__ballot((TOKEN ? v[c].cu : v[c].off) <= x && c * 64 + lane <= N));
    const int s = __builtin_amdgcn_readfirstlane(k) - 1;
    auto get = [&](auto f, int i) {
        int r = 0;
#pragma unroll
        for (int c = 0; c < C; c++)
            if (i / 64 == c) r = __builtin_amdgcn_readlane(f(v[c]), i % 64);
        return r;
    };
    auto off = [](const Kv8Seq &q) { return q.off; };
    auto cu = [](const Kv8Seq &q) { return q.cu; };
    Kv8At a;
    a.s = s;
    a.off = get(off, s);
    a.blocks = get(off, s + 1) - a.off;
    a.t0 = get(cu, s);
    a.tokens = get(cu, s + 1) - a.t0;
    a.p0 = get([](const Kv8Seq &q) { return q.pos0; }, s);
    a.row = get([](const Kv8Seq &q) { return q.row; }, s);
    return a;
}

// ---- for the attention kernels -------------------------------------------
// The scores' product runs in fp16: a code is an fp16 value (up to 448, steps
// down to 2^-9), and q keeps 11 bits there where bf16 has 8 (its rounding was
// the largest error of y: 0.004 of y's norm, now 0.002 with y's own rounding).
// A row of q is divided by a power of two that brings its largest magnitude to
// [2^6, 2^7), which keeps 256 products with codes in fp32's range with room and
// the small elements out of fp16's subnormals; the power and the block's scale
// are factors of the scores (log2 e too, or it is in q). (A row of zeros: 1. One that holds an infinity or
// NaN: NaN.)
typedef _Float16 kv8_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv8_f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 kv8_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 kv8_bf16x2 __attribute__((ext_vector_type(2)));

// the power of two for a largest magnitude amax (finite)
__device__ __forceinline__ float kv8_row_scale(float amax) {
    const int e = min(max((int)(__float_as_uint(amax) >> 23), 1), 247);
    return amax == 0.0f ? 1.0f : __uint_as_float((uint32_t)max(e - 6, 1) << 23);
}
// 8 codes as fp16, and times a power of two as bf16
__device__ __forceinline__ kv8_f16x8 kv8_f16(uint32_t a, uint32_t b) {
    const kv8_f16x2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
    const kv8_f16x2 q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const kv8_f16x2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
    const kv8_f16x2 u = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return kv8_f16x8{p[0], p[1], q[0], q[1], r[0], r[1], u[0], u[1]};
}
__device__ __forceinline__ kv8_bf16x8 kv8_bf16(uint32_t a, uint32_t b, float s) {
    const kv8_bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false);
    const kv8_bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true);
    const kv8_bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false);
    const kv8_bf16x2 u = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true);
    return kv8_bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], u[0], u[1]};
}
// the codes among c's four that are NaN, 0xff each
__device__ __forceinline__ uint32_t kv8_nan_codes(uint32_t c) {
    return ((((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
}

// Weights p = 2^(t - M) go into the sums of p v as they are, up to 2^10 each (M
// moves when t passes it by 10), for up to 2^24 keys: fp32 holds the sums while a
// block's scale of V is at most 2^84 (values below 2^93). For a block past that M is
// formed as if its scores were higher by so many powers of two, which makes its
// weights, and all others, as much smaller: no sum passes 2^(24 + 10 + 93) = 2^127.
// (A weight below 2^-126 is 0, so at the largest scale one below 2^-90 of the largest.)
__device__ __forceinline__ int kv8_v_up(float vs) {
    return max((int)(__float_as_uint(vs) >> 23 & 255) - (127 + 84), 0);
}

// Host checks, the same with and without a device.
// The batch against the cache: offsets, positions, rows (distinct where tokens
// are written). Fills r and the number of tokens.
int kv8_check(const ApusHipKv8Cache *c, size_t nkv, size_t B, const int32_t *rows, const int32_t *cu,
              const int32_t *pos0, bool writes, Kv8Ref *r, size_t *tokens);
// k, v: dense rows [token][nkv][256], or of a pitch. kn_w: the K rows are normed
// and roped first (rope: the table's rows).
int kv8_append_run(const Kv8Ref &kv, size_t nkv, size_t B, const int32_t *rows, const int32_t *cu,
                   const int32_t *pos0, const uint16_t *k, size_t ldk, const uint16_t *v, size_t ldv,
                   const uint16_t *kn_w, const uint16_t *rope);
bool kv8_overlap(const void *a, size_t na, const void *b, size_t nb);
bool kv8_overlap_cache(const ApusHipKv8Cache *c, size_t nkv, const void *p, size_t n);    // with its arrays

// Checks of the attention calls: of everything but their operands (the weights, the
// batch against workspace and cache; writes: new rows go into it), decode's with its
// limits; and of the operands, of T tokens.
int attn_kv8_check(const ApusHipAttnLayer *L, const ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                   const int32_t *cu, const int32_t *pos0, bool writes, const ApusHipKv8Cache *kv, Kv8Ref *r, size_t *T);
int attn_decode_kv8_check(const ApusHipAttnLayer *L, const ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                          const int32_t *cu, const int32_t *pos0, bool writes, const ApusHipKv8Cache *kv, Kv8Ref *r,
                          size_t *T);
int attn_kv8_check_operands(const ApusHipAttnLayer *L, size_t T, const uint16_t *qg, const uint16_t *k,
                            const uint16_t *v, const ApusHipKv8Cache *kv, const uint16_t *y);
bool attn_decode_kv8_fits(const ApusHipAttnKv8Work *w, size_t B, const int32_t *cu, const int32_t *pos0);
int attn_decode_kv8_run(const ApusHipAttnLayer *L, ApusHipAttnKv8Work *w, size_t B, const int32_t *rows,
                        const int32_t *cu, const int32_t *pos0, const uint16_t *qg, const uint16_t *k,
                        const uint16_t *v, const Kv8Ref &kv, uint16_t *y);

}  // namespace apus

struct ApusHipAttnKv8Work {
    size_t nkv, max_seqs, max_pos;
    size_t rot;
    double theta;
    int device;
    char *base;
    size_t rows;                             // of partial results
    float *part;                             // [row][256]
    float2 *stat;                            // [row]: reference point, sum
    uint16_t *rope;                          // [max_pos][64] cos, sin
};

// mx_dev.h -- device building blocks of the products with MXFP4 or bf16
// weights at few rows: one wavefront forms 16 outputs x 16 rows at a time on
// the 16-wide MFMAs, its operands straight from memory.
//
// MXFP4 (the OCP microscaling format): 32 consecutive elements of a row share
// a scale 2^(s - 127), s one byte (255: the block is NaN); an element is e2m1
// (sign, two exponent bits, one mantissa bit: 0 .5 1 1.5 2 3 4 6), two to a
// byte, the even element in the low half. An e2m1 value times a power of two
// is a bf16 value (up to its range), so a weight widens to bf16 exactly and
// its product with a bf16 activation is exact in fp32.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "apus_dev.h"

namespace apus {

constexpr int kMxBlock = 32;                 // elements per scale

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

// 8 codes (one dword) widened to bf16 times the scale whose byte is s
__device__ __forceinline__ mx_bf16x8 mx_widen(uint32_t c, uint32_t s) {
    const float sc = __uint_as_float(s << 23);           // (the exponent alone is used)
    const mx_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0);
    const mx_bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1);
    const mx_bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2);
    const mx_bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3);
    return mx_bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// A wavefront's operands of one step of 128 k. Lane l serves row l % 16 (of
// the weights, or of the activations), k group g = l / 16. Both operands of a
// product assign k to (lane group, MFMA) in the same way, and any way will do:
// MXFP4 weights give lane group g the whole 32-element block g (16 bytes and
// its scale), MFMA j its codes 8 j ..; bf16 weights give MFMA j the 32 k from
// 32 j, group g 8 of them, so that the 4 lanes of a row read 64 bytes in one
// piece. live: this lane's k of the step lie inside K (K is a multiple of 32);
// outside, both operands are zero.
struct WBf16 {
    static constexpr bool mx = false;
    struct Row {
        const char *p;
    };
    struct Frag {
        u32x4 v[4];
    };
    static __device__ __forceinline__ Row row(const void *w, const uint8_t *, size_t r, int K, int g) {
        return {(const char *)w + r * (size_t)K * 2 + g * 16};
    }
    static __device__ __forceinline__ void load(Frag &f, const Row &r, int k, int K) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool live = k + 32 * j < K;
            f.v[j] = *reinterpret_cast<const u32x4 *>(r.p + (size_t)(live ? k + 32 * j : 0) * 2);
            if (!live) f.v[j] = u32x4{};
        }
    }
    static __device__ __forceinline__ mx_bf16x8 operand(const Frag &f, int j) {
        return __builtin_bit_cast(mx_bf16x8, f.v[j]);
    }
};
struct WMx {
    static constexpr bool mx = true;
    struct Row {
        const uint8_t *p, *s;
    };
    struct Frag {
        u32x4 v;
        uint32_t s;
    };
    static __device__ __forceinline__ Row row(const void *w, const uint8_t *ws, size_t r, int K, int g) {
        return {(const uint8_t *)w + r * (size_t)(K / 2) + g * 16, ws + r * (size_t)(K / kMxBlock)};
    }
    static __device__ __forceinline__ void load(Frag &f, const Row &r, int k, int K) {
        const int g = (threadIdx.x >> 4) & 3;
        const bool live = k + 32 * g < K;
        f.v = *reinterpret_cast<const u32x4 *>(r.p + (live ? k / 2 : -16 * g));
        f.s = r.s[live ? k / kMxBlock + g : 0];
        if (!live) {
            f.v = u32x4{};
            f.s = 127;
        }
    }
    static __device__ __forceinline__ mx_bf16x8 operand(const Frag &f, int j) {
        return mx_widen(f.v[j], f.s);
    }
};

// bf16 activations for weights of kind W
template <class W>
struct XBf16 {
    struct Row {
        const char *p;
    };
    struct Frag {
        u32x4 v[4];
    };
    static __device__ __forceinline__ Row row(const uint16_t *x, size_t ld, size_t r, int g) {
        return {(const char *)(x + r * ld + (W::mx ? 32 * g : 8 * g))};
    }
    static __device__ __forceinline__ void load(Frag &f, const Row &r, int k, int K) {
        const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool live = W::mx ? k + 32 * g < K : k + 32 * j < K;
            const int off = W::mx ? (live ? k : -32 * g) + 8 * j : (live ? k + 32 * j : 0);
            f.v[j] = *reinterpret_cast<const u32x4 *>(r.p + (ptrdiff_t)off * 2);
            if (!live) f.v[j] = u32x4{};
        }
    }
};

__device__ __forceinline__ mx_f32x4 mfma16(const mx_bf16x8 &a, const mx_bf16x8 &b, const mx_f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// 128 k of two MXFP4 operands (format 4 = e2m1)
__device__ __forceinline__ mx_f32x4 mfma16_mx(const WMx::Frag &a, const WMx::Frag &b, const mx_f32x4 &c) {
    const mx_i32x8 av{(int)a.v[0], (int)a.v[1], (int)a.v[2], (int)a.v[3], 0, 0, 0, 0};
    const mx_i32x8 bv{(int)b.v[0], (int)b.v[1], (int)b.v[2], (int)b.v[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)a.s, 0, (int)b.s);
}

}  // namespace apus

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

// Loads through a buffer resource: the address is a base and size in scalar
// registers, a lane's offset and a uniform one, so that a tile's 16 rows take
// one address register (as 64-bit pointers the loops' addresses did not fit the
// registers), and an offset past the size reads zero (the uniform offset stays
// under the size, which no tile has zero of: the check subtracts it).
__device__ f32x4_t llvm_raw_buffer_load_v4f32(i32x4 r, int voff, int soff, int aux)
    __asm("llvm.amdgcn.raw.buffer.load.v4f32");
__device__ float llvm_raw_buffer_load_f32(i32x4 r, int voff, int soff, int aux)
    __asm("llvm.amdgcn.raw.buffer.load.f32");
__device__ uint8_t llvm_raw_buffer_load_u8(i32x4 r, int voff, int soff, int aux)
    __asm("llvm.amdgcn.raw.buffer.load.i8");
constexpr uint32_t kPast = 0x7fffffff;       // an offset past every tile
__device__ __forceinline__ u32x4 ld16(i32x4 r, uint32_t off, int at) {
    return __builtin_bit_cast(u32x4, llvm_raw_buffer_load_v4f32(r, (int)off, at, 0));
}

// A wavefront's operands of one step of 128 k for the 16-wide MFMAs. Lane l
// serves row l % 16 (of the weights, or of the activations), k group g = l / 16.
// Both operands of a product assign k to (lane group, MFMA) in the same way, and
// any way will do: MXFP4 weights give lane group g the whole 32-element block g
// (16 bytes and its scale), MFMA j its codes 8 j ..; bf16 weights give MFMA j the
// 32 k from 32 j, group g 8 of them. What lies past K (a multiple of 32) reads as
// zero, in both operands.
//
// From memory to these operands: lanes load along the rows (load_raw), write what
// they got to LDS of the wavefront's own (put) and read the operands from there
// (get). Each lane loading its own has neighbouring lanes read different rows, and
// the address unit takes such a load a lane at a time, about 60 clocks instead of 16
// (XBf16::load does, for activations of few rows, most lanes' the same). The LDS
// places are permuted so that neither side's lanes share banks.

// 16 rows of a step of 128 bf16 values: load i has rows 4 i .., 16 lanes a row
struct RowsBf16 {
    static constexpr int kTile = 4096;       // LDS bytes
    struct Raw {
        u32x4 v[4];
    };
    static __device__ __forceinline__ void put(char *m, const Raw &f, int l) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = 4 * i + (l >> 4);
            *reinterpret_cast<u32x4 *>(m + row * 256 + (((l & 15) ^ row) << 4)) = f.v[i];
        }
    }
    // 16-byte piece c of this lane's row
    static __device__ __forceinline__ u32x4 piece(const char *m, int c, int l) {
        return *reinterpret_cast<const u32x4 *>(m + (l & 15) * 256 + ((c ^ (l & 15)) << 4));
    }
};

struct WBf16 {
    static constexpr bool mx = false;
    static constexpr int kTile = RowsBf16::kTile;
    struct Tile {
        i32x4 w;
    };
    struct Lane {
        uint32_t off;
    };
    struct Frag {
        u32x4 v[4];
    };
    typedef RowsBf16::Raw Raw;
    // up to 16 rows from r0 (uniform) of w [][K]; rows past them read as zero
    static __device__ __forceinline__ Tile tile(const void *w, const uint8_t *, size_t r0, int rows, int K) {
        return {dma_rsrc((const char *)w + r0 * (size_t)K * 2, (uint32_t)rows * (uint32_t)K * 2)};
    }
    static __device__ __forceinline__ mx_bf16x8 operand(const Frag &f, int j) {
        return __builtin_bit_cast(mx_bf16x8, f.v[j]);
    }
    static __device__ __forceinline__ Lane raw_lane(int l, int K) {
        return {(uint32_t)(l >> 4) * (uint32_t)K * 2 + (l & 15) * 16};
    }
    template <bool S = true>
    static __device__ __forceinline__ void load_raw(Raw &f, const Tile &t, const Lane &l, int step, int K) {
        const int k = step * 128;
        const bool live = k + 8 * (int)(threadIdx.x & 15) < K;
#pragma unroll
        for (int i = 0; i < 4; i++)
            f.v[i] = ld16(t.w, live ? l.off + 8 * i * (uint32_t)K : kPast, k < K ? k * 2 : 0);
    }
    static __device__ __forceinline__ void put(char *m, const Raw &f, int l) { RowsBf16::put(m, f, l); }
    template <bool S = true>
    static __device__ __forceinline__ void get(Frag &f, const char *m, const Raw &, int l) {
#pragma unroll
        for (int j = 0; j < 4; j++) f.v[j] = RowsBf16::piece(m, 4 * j + (l >> 4), l);
    }
};
struct WMx {
    static constexpr bool mx = true;
    static constexpr int kTile = 1024;
    struct Tile {
        i32x4 w, s;
    };
    struct Lane {
        uint32_t off, soff;
    };
    struct Frag {
        u32x4 v;
        uint32_t s;
    };
    typedef Frag Raw;
    static __device__ __forceinline__ Tile tile(const void *w, const uint8_t *ws, size_t r0, int rows, int K) {
        return {dma_rsrc((const uint8_t *)w + r0 * (size_t)(K / 2), (uint32_t)rows * (uint32_t)(K / 2)),
                dma_rsrc(ws + r0 * (size_t)(K / kMxBlock), (uint32_t)rows * (uint32_t)(K / kMxBlock))};
    }
    static __device__ __forceinline__ mx_bf16x8 operand(const Frag &f, int j) {
        return mx_widen(f.v[j], f.s);
    }
    // 4 lanes a row, each a block of the step (past K: zero codes, at the scale
    // 2^-127); the scales go between lanes without LDS memory, or (S false) are
    // brought in strips (Strip)
    static __device__ __forceinline__ Lane raw_lane(int l, int K) {
        const uint32_t row = l >> 2, block = l & 3;
        return {row * (uint32_t)(K / 2) + block * 16, row * (uint32_t)(K / kMxBlock) + block};
    }
    template <bool S = true>
    static __device__ __forceinline__ void load_raw(Raw &f, const Tile &t, const Lane &l, int step, int K) {
        const int k = step * 128;
        const bool live = k + 32 * (int)(threadIdx.x & 3) < K;
        f.v = ld16(t.w, live ? l.off : kPast, k < K ? k / 2 : 0);
        if (S) f.s = llvm_raw_buffer_load_u8(t.s, (int)(live ? l.soff : kPast), k < K ? k / kMxBlock : 0, 0);
    }
    static __device__ __forceinline__ void put(char *m, const Raw &f, int l) {
        const int row = l >> 2;
        *reinterpret_cast<u32x4 *>(m + row * 64 + (((l & 3) ^ (row >> 2)) << 4)) = f.v;
    }
    template <bool S = true>
    static __device__ __forceinline__ void get(Frag &f, const char *m, const Raw &raw, int l) {
        const int r = l & 15, g = l >> 4;
        f.v = *reinterpret_cast<const u32x4 *>(m + r * 64 + ((g ^ (r >> 2)) << 4));
        if (S) f.s = (uint32_t)__builtin_amdgcn_ds_bpermute((r * 4 + g) * 4, (int)raw.s);
    }
};

// The scales of 16 steps (64 bytes a row) of a tile's 16 rows, through LDS of the
// wavefront's own: a byte a lane and step took the streaming kernels a seventh of
// their time. Rows in whole words (K a multiple of 128); past K zero.
struct Strip {
    static constexpr int kTile = 1024, kSteps = 16;
    uint32_t v[4];
    __device__ __forceinline__ void load(const WMx::Tile &t, int step, int K) {
        const uint32_t l = threadIdx.x & 63, w = l & 15, ks = (uint32_t)K / kMxBlock, at = 4 * step;   // step: a multiple of kSteps
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            v[i] = __builtin_bit_cast(uint32_t, llvm_raw_buffer_load_f32(
                t.s, (int)(at + 4 * w < ks ? (4 * i + l / 16) * ks + 4 * w : kPast), at < ks ? (int)at : 0, 0));
    }
    // word w of row r at w ^ r
    __device__ __forceinline__ void put(char *m) const {
        const uint32_t l = threadIdx.x & 63;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t row = 4 * i + l / 16;
            *reinterpret_cast<uint32_t *>(m + row * 64 + (((l & 15) ^ row) << 2)) = v[i];
        }
    }
    // the scale of lane group g's block in a step, for row l % 16
    static __device__ __forceinline__ uint32_t get(const char *m, int step, int l) {
        return (uint8_t)m[(l & 15) * 64 + (((step & (kSteps - 1)) ^ (l & 15)) << 2) + (l >> 4)];
    }
};

// bf16 activations for weights of kind W: the row at byte `off` of a buffer
template <class W>
struct XBf16 {
    struct Frag {
        u32x4 v[4];
    };
    static __device__ __forceinline__ uint32_t lane(uint32_t off, int g) { return off + (W::mx ? 64 * g : 16 * g); }
    static __device__ __forceinline__ void load(Frag &f, i32x4 x, uint32_t l, int step, int K) {
        const int g = (threadIdx.x >> 4) & 3, k = step * 128;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool in = W::mx ? k < K : k + 32 * j < K;                  // (uniform)
            const bool live = W::mx ? k + 32 * g < K : in;
            f.v[j] = ld16(x, live ? l : kPast, in ? 2 * k + (W::mx ? 16 : 64) * j : 0);
        }
    }
    // rows[i]: byte offsets of the rows 4 i + lane / 16; loads past the first XR are
    // of rows that are not there
    template <int XR = 4>
    static __device__ __forceinline__ void load_raw(RowsBf16::Raw &f, i32x4 x, const uint32_t (&rows)[4], int step, int K) {
        const int c = threadIdx.x & 15, k = step * 128;
        const bool live = k + 8 * c < K;
#pragma unroll
        for (int i = 0; i < 4; i++)
            f.v[i] = i < XR ? ld16(x, live ? rows[i] + 16 * c : kPast, k < K ? 2 * k : 0) : u32x4{};
    }
    // the 16-byte piece of a step that lane group g takes to MFMA j
    static __device__ __forceinline__ int piece_of(int j, int g) { return W::mx ? 4 * g + j : 4 * j + g; }
    static __device__ __forceinline__ mx_bf16x8 piece(const char *m, int j, int l) {
        return __builtin_bit_cast(mx_bf16x8, RowsBf16::piece(m, piece_of(j, l >> 4), l));
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

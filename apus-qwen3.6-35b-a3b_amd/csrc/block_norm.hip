// block_norm.hip -- the residual and the norms between one block of a model
// and the next: h' = h + scale * gate * post(y), x = pre(h'), post and pre the
// (1+w) RMSNorm of the hidden size. One pass: a row's y, h and gate are read
// once, h' stays in registers for the second norm. fp32 throughout; h' and x
// are each rounded once.
//
// A row belongs to a wavefront up to 2048 elements (no barrier between a
// row's loads and its stores), to a workgroup of four past them. Aligned rows
// go 8 elements a load, others one.
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "apus_dev.h"
#include "apus_host.h"
#include "mx.h"

using namespace apus;

namespace {

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr size_t kMaxHidden = 16384, kMaxRows = (size_t)1 << 24;

struct NormArgs {
    const uint16_t *y, *w_post, *w_pre, *gate;
    const void *h;
    void *h_out;
    uint16_t *x;
    size_t ldy, ldh, ldo, ldx, ldg;
    int hidden, rows;
    float scale, eps;
};

// 8 elements of a row from element i on (VEC), or the elements i, i + step, ...
template <bool VEC> __device__ __forceinline__ void ld8(float (&v)[8], const uint16_t *p, int i, int step, int n) {
    if (VEC) {
        const u16x8 u = *reinterpret_cast<const u16x8 *>(p + i);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = bf2f(u[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = bf2f(p[min(i + e * step, n - 1)]);
    }
}
template <bool VEC> __device__ __forceinline__ void ld8(float (&v)[8], const float *p, int i, int step, int n) {
    if (VEC) {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(p + i), b = *reinterpret_cast<const f32x4 *>(p + i + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = p[min(i + e * step, n - 1)];
    }
}
template <bool VEC> __device__ __forceinline__ void st8(uint16_t *p, const float (&v)[8], int i, int step, int n) {
    if (VEC) {
        u16x8 u;
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = f2bf(v[e]);
        *reinterpret_cast<u16x8 *>(p + i) = u;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (i + e * step < n) p[i + e * step] = f2bf(v[e]);
    }
}
template <bool VEC> __device__ __forceinline__ void st8(float *p, const float (&v)[8], int i, int step, int n) {
    if (VEC) {
        *reinterpret_cast<f32x4 *>(p + i) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4 *>(p + i + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (i + e * step < n) p[i + e * step] = v[e];
    }
}

// TPR threads a row, NV eights a thread; H: the residual's type. VEC: hidden
// and every row's start in whole vectors.
template <class H, bool VEC, int TPR, int NV>
__global__ __launch_bounds__(256) void k_block_norm(NormArgs a) {
    const int tid = threadIdx.x, lane = tid % TPR;
    const int row = min((int)blockIdx.x * (256 / TPR) + tid / TPR, a.rows - 1);   // (the last row again: same values)
    const bool live = (int)blockIdx.x * (256 / TPR) + tid / TPR < a.rows;
    __shared__ float red[2][4];
    // the sum over the row's threads
    auto total = [&](float s, int k) {
#pragma unroll
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
        if (TPR == 64) return s;
        if ((tid & 63) == 0) red[k][tid >> 6] = s;
        __syncthreads();
        return (red[k][0] + red[k][1]) + (red[k][2] + red[k][3]);
    };
    const int n = a.hidden, step = VEC ? 1 : TPR;
    int at[NV];
    bool in[NV][VEC ? 1 : 8];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = VEC ? (j * TPR + lane) * 8 : j * 8 * TPR + lane;
        if (VEC) {
            in[j][0] = i < n;
            at[j] = min(i, n - 8);
        } else {
            at[j] = i;
#pragma unroll
            for (int e = 0; e < (VEC ? 1 : 8); e++) in[j][e] = i + e * step < n;
        }
    }
    float h[NV][8], y[NV][8], g[NV][8], wa[NV][8], wb[NV][8];
    const H *hr = reinterpret_cast<const H *>(a.h) + (size_t)row * a.ldh;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        ld8<VEC>(h[j], hr, at[j], step, n);
        if (a.y) ld8<VEC>(y[j], a.y + (size_t)row * a.ldy, at[j], step, n);
        if (a.y && a.gate) ld8<VEC>(g[j], a.gate + (size_t)row * a.ldg, at[j], step, n);
        if (a.y && a.w_post) ld8<VEC>(wa[j], a.w_post, at[j], step, n);
        if (a.x) ld8<VEC>(wb[j], a.w_pre, at[j], step, n);
    }
    if (a.y) {
        float rs = 1.0f;
        if (a.w_post) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (in[j][VEC ? 0 : e]) s += y[j][e] * y[j][e];
            rs = 1.0f / sqrtf(total(s, 0) / (float)n + a.eps);
        }
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float v = y[j][e];
                if (a.w_post) v = v * rs * (1.0f + wa[j][e]);
                if (a.gate) v *= g[j][e];
                h[j][e] += a.scale * v;
            }
        }
    if (a.h_out && live) {
        H *o = reinterpret_cast<H *>(a.h_out) + (size_t)row * a.ldo;
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (in[j][0]) st8<VEC>(o, h[j], at[j], step, n);
    }
    if (!a.x) return;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (in[j][VEC ? 0 : e]) s += h[j][e] * h[j][e];
    const float rs = 1.0f / sqrtf(total(s, 1) / (float)n + a.eps);
    if (!live) return;
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
        for (int e = 0; e < 8; e++) h[j][e] = h[j][e] * rs * (1.0f + wb[j][e]);
        if (in[j][0]) st8<VEC>(a.x + (size_t)row * a.ldx, h[j], at[j], step, n);
    }
}

template <class H> int launch(const NormArgs &a, bool vec) {
    auto go = [&](auto v, auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value;
        APUS_TIMED("k_block_norm",
                   k_block_norm<H, decltype(v)::value, TPR, decltype(nv)::value>
                       <<<cdiv((size_t)a.rows, 256 / TPR), 256, 0, stream()>>>(a));
        return launch_check("k_block_norm");
    };
    auto size = [&](auto v) {
        const std::integral_constant<int, 64> one;
        const std::integral_constant<int, 256> four;
        if (a.hidden <= 512) return go(v, one, std::integral_constant<int, 1>{});
        if (a.hidden <= 1024) return go(v, one, std::integral_constant<int, 2>{});
        if (a.hidden <= 2048) return go(v, one, std::integral_constant<int, 4>{});
        if (a.hidden <= 4096) return go(v, four, std::integral_constant<int, 2>{});
        if (a.hidden <= 8192) return go(v, four, std::integral_constant<int, 4>{});
        return go(v, four, std::integral_constant<int, 8>{});
    };
    return vec ? size(std::true_type{}) : size(std::false_type{});
}

}  // namespace

extern "C" {

int apus_hip_block_norm(const ApusHipBlockNorm *N, size_t T, const uint16_t *y, size_t ldy, const void *h,
                        size_t ldh, void *h_out, size_t ldo, uint16_t *x, size_t ldx) {
    APUS_ENABLED();
    if (!N) return set_error(kErrArgument, "NULL norm");
    const size_t n = N->hidden;
    if (!n || n > kMaxHidden) return set_error(kErrUnsupported, "hidden size %zu (1 .. %zu)", n, kMaxHidden);
    if (T > kMaxRows) return set_error(kErrUnsupported, "%zu rows", T);
    if (!(N->eps >= 0.0f)) return set_error(kErrArgument, "eps is negative or NaN");
    const size_t hb = N->h_f32 ? 4 : 2;
    const bool gated = y && N->gate;
    if (T) {
        if (!h) return set_error(kErrArgument, "NULL residual");
        if (y ? !h_out : !x) return set_error(kErrArgument, "NULL output");
        if (x && !N->w_pre) return set_error(kErrArgument, "x needs the pre-norm's weights");
        struct Rows { const void *p; size_t ld, b; const char *what; };
        const Rows rows[] = {{y, ldy, 2, "y"}, {h, ldh, hb, "h"}, {h_out, ldo, hb, "h_out"}, {x, ldx, 2, "x"},
                             {gated && N->ld_gate ? N->gate : nullptr, N->ld_gate, 2, "gate"}};
        for (const Rows &r : rows) {
            if (!r.p) continue;
            if (r.ld < n) return set_error(kErrArgument, "%s rows of %zu elements with pitch %zu", r.what, n, r.ld);
            if (r.ld > ((size_t)1 << 40) / T) return set_error(kErrUnsupported, "%zu %s rows of pitch %zu", T, r.what, r.ld);
            if ((uintptr_t)r.p % r.b) return set_error(kErrArgument, "misaligned %s", r.what);
        }
        for (const uint16_t *w : {N->w_post, N->w_pre, N->gate})
            if ((uintptr_t)w % 2) return set_error(kErrArgument, "misaligned weights");
        auto apart = [&](const Rows &o, const Rows &i, bool same_ok) {
            if (!o.p || !i.p || (same_ok && o.p == i.p && o.ld == i.ld && o.b == i.b)) return true;
            return !rows_overlap(o.p, o.ld * o.b, n * o.b, i.p, i.ld * i.b, n * i.b, T);
        };
        auto clear = [&](const Rows &o, const uint16_t *w) {
            return !o.p || !w || !block_overlaps(w, n * 2, o.p, o.ld * o.b, n * o.b, T);
        };
        const Rows &ry = rows[0], &rh = rows[1], &ro = rows[2], &rx = rows[3], &rg = rows[4];
        if (!apart(ro, ry, false) || !apart(ro, rh, true) || !apart(ro, rx, false) || !apart(ro, rg, false) ||
            !apart(rx, ry, true) || !apart(rx, rh, false) || !apart(rx, rg, false) ||
            !clear(ro, N->w_post) || !clear(ro, N->w_pre) || !clear(rx, N->w_post) || !clear(rx, N->w_pre) ||
            (gated && !N->ld_gate && (!clear(ro, N->gate) || !clear(rx, N->gate))))
            return set_error(kErrArgument, "an output overlaps another operand");
    }
    if (int r = mx_ready()) return r;
    if (!T) return kOk;
    const NormArgs a{y, N->w_post, N->w_pre, gated ? N->gate : nullptr, h, h_out, x, ldy, ldh, ldo, ldx,
                     N->ld_gate, (int)n, (int)T, N->scale, N->eps};
    // whole vectors: 8 elements of 2 bytes, or twice 4 of 4
    auto whole = [&](const void *p, size_t ld) { return !p || ((uintptr_t)p % 16 == 0 && ld % 8 == 0); };
    const bool vec = n % 8 == 0 && whole(y, ldy) && whole(h, ldh) && whole(h_out, ldo) && whole(x, ldx) &&
                     whole(a.gate, N->ld_gate) && whole(a.w_post, 0) && whole(a.w_pre, 0);
    return N->h_f32 ? launch<float>(a, vec) : launch<uint16_t>(a, vec);
}

}  // extern "C"

// block_norm.hip -- the residual and the norms between one block of a model
// and the next: h' = h + scale * gate * post(y), x = pre(h'), post and pre the
// (1+w) RMSNorm of the hidden size. One pass: a row's y, h and gate are read
// once, h' stays in registers for the second norm. fp32 throughout; h' and x
// are each rounded once.
//
// A row belongs to a wavefront up to 1024 elements (no barrier between its
// loads and its stores), to a workgroup of four past them (2048, 8192 rows: 46.5
// us with a workgroup a row, 48.8 with a wavefront; 1529, element by element: 11.9
// and 16.3), to one of eight past 8192 (16384, 2000 rows: 67 us, with four 74, with
// sixteen 83; 16001, element by element: 111, 153, 142). Aligned rows go 8 elements a
// load, others one, at about twice what memory would take: 2000 rows of 16001 97 us, of
// 16384 56 (bf16, no gate; 49 and 50 at a copy's rate), of 5001 36, of 5008 22. An
// element is a load and a register of its own: with two eights a thread or more that is
// 128 to 256 registers, which leave two to four wavefronts a SIMD to hide the loads (the
// bf16 kernel of eight wavefronts a row spills 4). Bound by memory: 8192 rows of 2048,
// fp32 residuals and a gate, 235 MB in 44.5 us, 5.3 TB/s, what a copy of 1 GiB reaches; a
// single row (2 us) by its launch.
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

// 8 elements of a row as they lie in memory: from element i on (VEC), or i, i +
// step, ... one by one. Widened when they are used: as fp32 from the start a
// row's took twice the registers, and half as many rows were on their way (8192
// rows of 2048 with fp32 residuals: 64 us).
template <class T, bool VEC> struct Eight;
template <> struct Eight<uint16_t, true> {
    u16x8 u;
    __device__ void load(const uint16_t *p, int i, int, int) { u = *reinterpret_cast<const u16x8 *>(p + i); }
    __device__ float operator[](int e) const { return bf2f(u[e]); }
};
template <> struct Eight<float, true> {
    f32x4 a, b;
    __device__ void load(const float *p, int i, int, int) {
        a = *reinterpret_cast<const f32x4 *>(p + i);
        b = *reinterpret_cast<const f32x4 *>(p + i + 4);
    }
    __device__ float operator[](int e) const { return e < 4 ? a[e & 3] : b[e & 3]; }
};
template <class T> struct Eight<T, false> {
    T u[8];
    __device__ void load(const T *p, int i, int step, int n) {
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = p[min(i + e * step, n - 1)];
    }
    __device__ float operator[](int e) const { return widen(u[e]); }
    static __device__ float widen(uint16_t x) { return bf2f(x); }
    static __device__ float widen(float x) { return x; }
};
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
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_block_norm(NormArgs a) {
    constexpr int R = TPR < 256 ? 256 / TPR : 1;           // rows of a workgroup
    const int tid = threadIdx.x, lane = tid % TPR;
    const int row = min((int)blockIdx.x * R + tid / TPR, a.rows - 1);     // (the last row again: same values)
    const bool live = (int)blockIdx.x * R + tid / TPR < a.rows;
    __shared__ __attribute__((aligned(16))) float red[2][TPR > 64 ? TPR / 64 : 1];
    // the sum over the row's threads
    auto total = [&](float s, int k) {
#pragma unroll
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
        if (TPR == 64) return s;
        if ((tid & 63) == 0) red[k][tid >> 6] = s;
        __syncthreads();
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; i += 4) s += (red[k][i] + red[k][i + 1]) + (red[k][i + 2] + red[k][i + 3]);
        return s;
    };
    const int n = a.hidden, step = VEC ? 1 : TPR;
    // of the eight j: its first element, and whether its element e is in the row
    auto at = [&](int j) { return VEC ? min((j * TPR + lane) * 8, n - 8) : j * 8 * TPR + lane; };
    auto in = [&](int j, int e) { return VEC ? (j * TPR + lane) * 8 < n : j * 8 * TPR + lane + e * step < n; };
    Eight<H, VEC> hr[NV];
    Eight<uint16_t, VEC> y[NV], g[NV], w[NV];
    const H *hp = reinterpret_cast<const H *>(a.h) + (size_t)row * a.ldh;
    if (a.y) {
#pragma unroll
        for (int j = 0; j < NV; j++) y[j].load(a.y + (size_t)row * a.ldy, at(j), step, n);
    }
#pragma unroll
    for (int j = 0; j < NV; j++) hr[j].load(hp, at(j), step, n);
    if (a.y && a.gate) {
#pragma unroll
        for (int j = 0; j < NV; j++) g[j].load(a.gate + (size_t)row * a.ldg, at(j), step, n);
    }
    if (a.y && a.w_post) {
#pragma unroll
        for (int j = 0; j < NV; j++) w[j].load(a.w_post, at(j), step, n);
    }
    float h[NV][8], s = 0.0f;
    if (a.y) {
        float rs = 1.0f;
        if (a.w_post) {
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (in(j, e)) s += y[j][e] * y[j][e];
            rs = 1.0f / sqrtf(total(s, 0) / (float)n + a.eps);
        }
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float v = y[j][e];
                if (a.w_post) v = v * rs * (1.0f + w[j][e]);
                if (a.gate) v *= g[j][e];
                h[j][e] = hr[j][e] + a.scale * v;
            }
    } else {
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) h[j][e] = hr[j][e];
    }
    if (a.x) {
#pragma unroll
        for (int j = 0; j < NV; j++) w[j].load(a.w_pre, at(j), step, n);
    }
    if (a.h_out && live) {
        H *o = reinterpret_cast<H *>(a.h_out) + (size_t)row * a.ldo;
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (in(j, 0)) st8<VEC>(o, h[j], at(j), step, n);
    }
    if (!a.x) return;
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (in(j, e)) s += h[j][e] * h[j][e];
    const float rs = 1.0f / sqrtf(total(s, 1) / (float)n + a.eps);
    if (!live) return;
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
        for (int e = 0; e < 8; e++) h[j][e] = h[j][e] * rs * (1.0f + w[j][e]);
        if (in(j, 0)) st8<VEC>(a.x + (size_t)row * a.ldx, h[j], at(j), step, n);
    }
}

// (rows of a launch: with 512 threads a row 2^31 threads, of the 2^32 - 1 that a
// launch can have; more rows take several)
constexpr size_t kLaunchRows = (size_t)1 << 22;

template <class H> int launch(const NormArgs &all, bool vec) {
    NormArgs a = all;
    auto go = [&](auto v, auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value;
        for (size_t r = 0; r < (size_t)all.rows; r += kLaunchRows) {
            auto from = [&](auto *p, size_t ld) { return p ? p + r * ld : p; };
            a.y = from(all.y, a.ldy);
            a.gate = from(all.gate, a.ldg);
            a.h = (const H *)all.h + r * a.ldh;
            a.h_out = from((H *)all.h_out, a.ldo);
            a.x = from(all.x, a.ldx);
            a.rows = (int)std::min(kLaunchRows, (size_t)all.rows - r);
            APUS_TIMED("k_block_norm",
                       k_block_norm<H, decltype(v)::value, TPR, decltype(nv)::value>
                           <<<cdiv((size_t)a.rows, TPR < 256 ? 256 / TPR : 1), TPR > 256 ? TPR : 256, 0, stream()>>>(a));
            if (int e = launch_check("k_block_norm")) return e;
        }
        return (int)kOk;
    };
    auto size = [&](auto v) {
        const std::integral_constant<int, 64> one;
        const std::integral_constant<int, 256> four;
        if (a.hidden <= 512) return go(v, one, std::integral_constant<int, 1>{});
        if (a.hidden <= 1024) return go(v, one, std::integral_constant<int, 2>{});
        if (a.hidden <= 2048) return go(v, four, std::integral_constant<int, 1>{});
        if (a.hidden <= 4096) return go(v, four, std::integral_constant<int, 2>{});
        if (a.hidden <= 8192) return go(v, four, std::integral_constant<int, 4>{});
        return go(v, std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
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

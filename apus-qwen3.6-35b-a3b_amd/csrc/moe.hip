// moe.hip -- the mixture-of-experts layer of a decode step (up to
// kMoeMaxTokens tokens): per token x
//   l_e = w_router[e] . x,  the topk largest l_e (ties to the lowest index),
//   p_e = exp(l_e - max) / sum of the same over the chosen (norm_topk) or all,
//   y = sum_e p_e down_e(silu(gate_e x) * (up_e x))
//       + sigmoid(w_shared_gate . x) shared(x),
// everything in fp32, rounded once, at y. The weights are bf16 or MXFP4.
//
// For few tokens the layer is the reading of the chosen experts' weights.
// Launches: router logits; the choice; gate, up and silu of every (expert,
// 16 outputs) with that expert's tokens as the columns of an MFMA; down of
// every (expert, 64 outputs) into fp32 partial rows; the weighted sum.
// The intermediate h = silu(g) u goes to the down product as two bf16 numbers
// (its leading 8 bits and the rest rounded to 8), which keeps 16 bits of it: the
// product reads weights, not h, so the second MFMA costs no time, and a single
// bf16 h would put an error of a bf16 rounding into y beside y's own.
#include <stdint.h>

#include <algorithm>

#include "../../include/apus_hip.h"
#include "apus_dev.h"
#include "apus_host.h"
#include "mx.h"
#include "mx_dev.h"

using namespace apus;

// The device buffers of calls on one layer shape, and the shape they fit.
struct ApusHipMoeWork {
    size_t max_tokens, hidden, inter, experts, topk, shared;
    char *base = nullptr;
    float *logits;       // [T][E + 1]: the experts', then the shared gate's
    int32_t *ids;        // [T][topk]
    float *wts;          // [T][topk + 1]: p, then the shared expert's weight
    uint16_t *h;         // [T topk][2][inter], then [T][2][shared]
    float *part;         // [T topk + T][hidden]
};

namespace {

constexpr size_t kMoeMaxTokens = 1024, kMoeMaxExperts = 1024, kMoeMaxTopk = 32;

struct MoeArgs {
    const uint16_t *x, *w_router, *w_sgate;
    const void *w_gu, *w_dn, *w_sgu, *w_sdn;
    const uint8_t *s_gu, *s_dn, *s_sgu, *s_sdn;
    float *logits, *wts, *part;
    int32_t *ids;
    uint16_t *h;
    uint16_t *y;
    int T, H, I, E, k, Is, norm;
};

// ---- router ---------------------------------------------------------------
// 16 experts (the shared gate as one more) x 16 tokens a workgroup, K over
// its 4 wavefronts.
__global__ __launch_bounds__(256) void k_moe_router(MoeArgs a) {
    __shared__ mx_f32x4 red[4][64];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int E1 = a.E + 1, e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
    const int er = min(e0 + r, a.w_sgate ? a.E : a.E - 1);
    const auto wr = er < a.E ? WBf16::row(a.w_router, nullptr, er, a.H, g)
                             : WBf16::row(a.w_sgate, nullptr, 0, a.H, g);
    const auto xr = XBf16<WBf16>::row(a.x, a.H, min(t0 + r, a.T - 1), g);
    mx_f32x4 acc{};
    for (int k = wave * 128; k < a.H; k += 512) {
        WBf16::Frag wf;
        XBf16<WBf16>::Frag xf;
        WBf16::load(wf, wr, k, a.H);
        XBf16<WBf16>::load(xf, xr, k, a.H);
#pragma unroll
        for (int j = 0; j < 4; j++)
            acc = mfma16(WBf16::operand(wf, j), __builtin_bit_cast(mx_bf16x8, xf.v[j]), acc);
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    acc = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    if (t0 + r >= a.T) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (e0 + 4 * g + i < E1) a.logits[(size_t)(t0 + r) * E1 + e0 + 4 * g + i] = acc[i];
}

// Order of logits as unsigned numbers: NaN above all, -0 and +0 alike.
__device__ __forceinline__ uint32_t order_key(float f) {
    uint32_t u = __float_as_uint(f + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if (u == 0x80000000u) u = 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// A wavefront's choice for token t: lane l holds logits l, l + 64, ...
template <int NJ>
__device__ __forceinline__ void choose(const MoeArgs &a, int t, int lane) {
    const float *lg = a.logits + (size_t)t * (a.E + 1);
    float l[NJ];
    uint32_t key[NJ];                      // 0: past E, or taken (no number's key is 0)
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int e = lane + 64 * j;
        l[j] = e < a.E ? lg[e] : 0.0f;
        key[j] = e < a.E ? order_key(l[j]) : 0;
    }
    float top = 0.0f, mine = 0.0f, sum = 0.0f;
    int my_e = 0;
    for (int n = 0; n < a.k; n++) {
        uint32_t bk = 0;
        int be = 0;
        float bl = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; j++)
            if (key[j] > bk) {             // (ties: the lane's lowest index first)
                bk = key[j];
                be = lane + 64 * j;
                bl = l[j];
            }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t ok = __shfl_xor(bk, d);
            const int oe = __shfl_xor(be, d);
            const float ol = __shfl_xor(bl, d);
            if (ok > bk || (ok == bk && oe < be)) {
                bk = ok;
                be = oe;
                bl = ol;
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; j++)
            if (be == lane + 64 * j) key[j] = 0;
        if (n == 0) top = bl;
        const float p = expf(bl - top);
        sum += p;
        if (lane == n) {
            mine = p;
            my_e = be;
        }
    }
    if (!a.norm) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; j++)
            if (lane + 64 * j < a.E) s += expf(l[j] - top);
        sum = wave_sum(s);
    }
    if (lane < a.k) {
        a.ids[t * a.k + lane] = my_e;
        a.wts[t * (a.k + 1) + lane] = mine / sum;
    }
    if (lane == 0)
        a.wts[t * (a.k + 1) + a.k] = a.w_sgate ? 1.0f / (1.0f + expf(-lg[a.E])) : 1.0f;
}

__global__ __launch_bounds__(256) void k_moe_topk(MoeArgs a) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= a.T) return;
    if (a.E <= 256) choose<4>(a, t, lane);
    else choose<16>(a, t, lane);
}

// ---- experts ----------------------------------------------------------------
// Blocks of a launch: first nsh for the shared expert, then per slot nper. A
// slot is an expert, or, where the tokens make fewer choices than there are
// experts, a choice; of the choices of one expert the first does the work.
// Returns the expert (E: shared), or -1: nothing to do. list: the choices
// t * k + n that fell on it (shared: T k + t), cnt of them, in any order (a
// choice's values do not depend on its place).
__device__ __forceinline__ int gather(const MoeArgs &a, int b, int nsh, int nper, int &part,
                                      uint16_t *list, int *cnt) {
    const int n = a.T * a.k;
    if (b < nsh) {
        part = b;
        for (int t = threadIdx.x; t < a.T; t += blockDim.x) list[t] = (uint16_t)(n + t);
        if (threadIdx.x == 0) *cnt = a.T;
        __syncthreads();
        return a.E;
    }
    const int slot = (b - nsh) / nper;
    part = (b - nsh) % nper;
    const bool by_choice = n < a.E;
    const int e = by_choice ? a.ids[slot] : slot;
    if (threadIdx.x == 0) *cnt = 0;
    __syncthreads();
    int dup = 0;
    for (int q = threadIdx.x; q < n; q += blockDim.x)
        if (a.ids[q] == e) {
            dup |= by_choice && q < slot;
            // (a token chooses an expert once: at most T; the test holds for
            // any contents of ids)
            const int p = atomicAdd(cnt, 1);
            if (p < (int)kMoeMaxTokens) list[p] = (uint16_t)q;
        }
    dup = __syncthreads_or(dup);
    if (threadIdx.x == 0 && *cnt > a.T) *cnt = a.T;
    __syncthreads();
    return dup || *cnt == 0 ? -1 : e;
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

// h = silu(gate x) * (up x): 16 outputs of one expert for its tokens, 16 at a
// time, K over the 4 wavefronts.
template <class W>
__global__ __launch_bounds__(256) void k_moe_up(MoeArgs a, int nsh, int nper) {
    __shared__ uint16_t list[kMoeMaxTokens];
    __shared__ int cnt;
    __shared__ mx_f32x4 red[4][2][64];
    int part;
    const int e = gather(a, blockIdx.x, nsh, nper, part, list, &cnt);
    if (e < 0) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool sh = e == a.E;
    const int I = sh ? a.Is : a.I, n = cnt, o0 = part * 16;
    const size_t row0 = sh ? 0 : (size_t)e * 2 * I;
    const void *w = sh ? a.w_sgu : a.w_gu;
    const uint8_t *ws = sh ? a.s_sgu : a.s_gu;
    const auto wg = W::row(w, ws, row0 + o0 + r, a.H, g);
    const auto wu = W::row(w, ws, row0 + I + o0 + r, a.H, g);
    for (int c0 = 0; c0 < n; c0 += 16) {
        const int q = list[min(c0 + r, n - 1)];
        const int t = sh ? q - a.T * a.k : q / a.k;
        const auto xr = XBf16<W>::row(a.x, a.H, t, g);
        mx_f32x4 ag{}, au{};
        for (int k = wave * 128; k < a.H; k += 512) {
            typename W::Frag fg, fu;
            typename XBf16<W>::Frag fx;
            W::load(fg, wg, k, a.H);
            W::load(fu, wu, k, a.H);
            XBf16<W>::load(fx, xr, k, a.H);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const mx_bf16x8 xv = __builtin_bit_cast(mx_bf16x8, fx.v[j]);
                ag = mfma16(W::operand(fg, j), xv, ag);
                au = mfma16(W::operand(fu, j), xv, au);
            }
        }
        red[wave][0][lane] = ag;
        red[wave][1][lane] = au;
        __syncthreads();
        if (wave == 0 && c0 + r < n) {
            ag = (red[0][0][lane] + red[1][0][lane]) + (red[2][0][lane] + red[3][0][lane]);
            au = (red[0][1][lane] + red[1][1][lane]) + (red[2][1][lane] + red[3][1][lane]);
            uint16_t *h = a.h + (sh ? (size_t)a.T * a.k * 2 * a.I + (size_t)t * 2 * I : (size_t)q * 2 * I);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = silu(ag[i]) * au[i];
                // the leading bits, cut, and the rest, rounded (none of an
                // infinity or NaN)
                const uint32_t u = __float_as_uint(v);
                const bool fin = (u & 0x7f800000u) != 0x7f800000u;
                const uint16_t hi = fin ? (uint16_t)(u >> 16) : f2bf(v);
                const int o = o0 + 4 * g + i;
                h[o] = hi;
                h[I + o] = fin ? f2bf(v - bf2f(hi)) : 0;
            }
        }
        __syncthreads();
    }
}

// part[choice] = down h: 64 outputs of one expert, 16 a wavefront
template <class W>
__global__ __launch_bounds__(256) void k_moe_down(MoeArgs a, int nsh, int nper) {
    __shared__ uint16_t list[kMoeMaxTokens];
    __shared__ int cnt;
    int part;
    const int e = gather(a, blockIdx.x, nsh, nper, part, list, &cnt);
    if (e < 0) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool sh = e == a.E;
    const int I = sh ? a.Is : a.I, n = cnt, o0 = part * 64 + wave * 16;
    if (o0 >= a.H) return;                 // (H is a multiple of 32; no barrier follows)
    const size_t row0 = sh ? 0 : (size_t)e * a.H;
    const auto wr = W::row(sh ? a.w_sdn : a.w_dn, sh ? a.s_sdn : a.s_dn, row0 + o0 + r, I, g);
    for (int c0 = 0; c0 < n; c0 += 16) {
        const int q = list[min(c0 + r, n - 1)];
        const uint16_t *h = a.h + (sh ? (size_t)a.T * a.k * 2 * a.I + (size_t)(q - a.T * a.k) * 2 * I
                                      : (size_t)q * 2 * I);
        const auto xh = XBf16<W>::row(h, 0, 0, g), xl = XBf16<W>::row(h + I, 0, 0, g);
        mx_f32x4 acc{};
        for (int k = 0; k < I; k += 128) {
            typename W::Frag fw;
            typename XBf16<W>::Frag fh, fl;
            W::load(fw, wr, k, I);
            XBf16<W>::load(fh, xh, k, I);
            XBf16<W>::load(fl, xl, k, I);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const mx_bf16x8 wv = W::operand(fw, j);
                acc = mfma16(wv, __builtin_bit_cast(mx_bf16x8, fh.v[j]), acc);
                acc = mfma16(wv, __builtin_bit_cast(mx_bf16x8, fl.v[j]), acc);
            }
        }
        if (c0 + r < n)
            *reinterpret_cast<mx_f32x4 *>(a.part + (size_t)q * a.H + o0 + 4 * g) = acc;
    }
}

// y = rnd(sum over the choices, in order, then the shared expert)
__global__ __launch_bounds__(256) void k_moe_combine(MoeArgs a) {
    const int H4 = a.H / 4;
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.T * H4) return;
    const int t = i / H4, c = (i % H4) * 4;
    mx_f32x4 s{};
    for (int n = 0; n < a.k; n++)
        s += *reinterpret_cast<const mx_f32x4 *>(a.part + (size_t)(t * a.k + n) * a.H + c) *
             a.wts[t * (a.k + 1) + n];
    if (a.Is)
        s += *reinterpret_cast<const mx_f32x4 *>(a.part + ((size_t)a.T * a.k + t) * a.H + c) *
             a.wts[t * (a.k + 1) + a.k];
    ushort4 o = make_ushort4(f2bf(s[0]), f2bf(s[1]), f2bf(s[2]), f2bf(s[3]));
    *reinterpret_cast<ushort4 *>(a.y + (size_t)t * a.H + c) = o;
}

template <class W>
int experts_run(const MoeArgs &a) {
    const size_t slots = (size_t)std::min(a.T * a.k, a.E);
    {
        const int nsh = a.Is / 16, nper = a.I / 16;
        APUS_TIMED("k_moe_up", k_moe_up<W><<<(unsigned)(nsh + slots * nper), 256, 0, stream()>>>(a, nsh, nper));
        APUS_LAUNCHED("k_moe_up");
    }
    const int nper = (int)cdiv(a.H, 64), nsh = a.Is ? nper : 0;
    APUS_TIMED("k_moe_down", k_moe_down<W><<<(unsigned)(nsh + slots * nper), 256, 0, stream()>>>(a, nsh, nper));
    return launch_check("k_moe_down");
}

int check_layer(const ApusHipMoeLayer *L) {
    if (!L) return set_error(kErrArgument, "NULL layer");
    if (!L->experts || !L->topk || L->topk > L->experts)
        return set_error(kErrArgument, "topk of %zu experts must be 1 .. %zu (is %zu)", L->experts,
                         L->experts, L->topk);
    if (L->experts > kMoeMaxExperts || L->topk > kMoeMaxTopk)
        return set_error(kErrUnsupported, "mixture of up to %zu experts, %zu a token", kMoeMaxExperts,
                         kMoeMaxTopk);
    if (!L->hidden || L->hidden % 32 || !L->inter || L->inter % 32 || L->shared_inter % 32)
        return set_error(kErrUnsupported, "mixture of experts needs hidden, inter and shared_inter "
                         "multiples of 32 (%zu, %zu, %zu)", L->hidden, L->inter, L->shared_inter);
    if (L->hidden > (1u << 20) || L->inter > (1u << 20) || L->shared_inter > (1u << 20))
        return set_error(kErrUnsupported, "mixture of experts takes sizes up to 2^20");
    return kOk;
}

int check_weights(const ApusHipMoeLayer *L) {
    const bool sh = L->shared_inter != 0;
    for (const void *p : {(const void *)L->w_router, L->w_gate_up, L->w_down,
                          sh ? L->w_shared_gate_up : L->w_down, sh ? L->w_shared_down : L->w_down,
                          sh && L->w_shared_gate ? (const void *)L->w_shared_gate : L->w_down}) {
        if (!p) return set_error(kErrArgument, "NULL weight");
        if ((uintptr_t)p % 16) return set_error(kErrUnsupported, "weights need 16-byte alignment");
    }
    if (L->mxfp4 && (!L->s_gate_up || !L->s_down || (sh && (!L->s_shared_gate_up || !L->s_shared_down))))
        return set_error(kErrArgument, "NULL scales");
    return kOk;
}

}  // namespace

extern "C" {

int apus_hip_moe_work_create(const ApusHipMoeLayer *L, size_t max_tokens, ApusHipMoeWork **out) {
    APUS_ENABLED();
    if (!out) return set_error(kErrArgument, "NULL output");
    *out = nullptr;
    if (int r = check_layer(L)) return r;
    if (!max_tokens || max_tokens > kMoeMaxTokens)
        return set_error(kErrUnsupported, "a mixture-of-experts call takes 1 .. %zu tokens (%zu)",
                         kMoeMaxTokens, max_tokens);
    if (int r = mx_ready()) return r;
    auto *w = new ApusHipMoeWork{max_tokens, L->hidden, L->inter, L->experts, L->topk, L->shared_inter};
    const size_t T = max_tokens, k = L->topk;
    size_t n = 0;
    auto take = [&](size_t bytes) {
        const size_t at = n;
        n += (bytes + 255) / 256 * 256;
        return at;
    };
    const size_t logits = take(T * (L->experts + 1) * 4), ids = take(T * k * 4),
                 wts = take(T * (k + 1) * 4), h = take(T * (k * L->inter + L->shared_inter) * 4),
                 part = take(T * (k + 1) * L->hidden * 4);
    if (hipMalloc((void **)&w->base, n) != hipSuccess) {
        delete w;
        return set_error(kErrHip, "hipMalloc of %zu bytes failed", n);
    }
    w->logits = (float *)(w->base + logits);
    w->ids = (int32_t *)(w->base + ids);
    w->wts = (float *)(w->base + wts);
    w->h = (uint16_t *)(w->base + h);
    w->part = (float *)(w->base + part);
    *out = w;
    return kOk;
}

int apus_hip_moe_work_destroy(ApusHipMoeWork *w) {
    APUS_ENABLED();
    if (!w) return kOk;
    if (int r = mx_ready()) return r;
    APUS_HIP_TRY(hipStreamSynchronize(stream()));
    (void)hipFree(w->base);
    delete w;
    return kOk;
}

int apus_hip_moe_layer_decode(const ApusHipMoeLayer *L, ApusHipMoeWork *w, size_t T,
                              const uint16_t *x, uint16_t *y) {
    APUS_ENABLED();
    if (int r = check_layer(L)) return r;
    if (!w) return set_error(kErrArgument, "NULL workspace");
    if (w->hidden != L->hidden || w->inter != L->inter || w->experts != L->experts ||
        w->topk != L->topk || w->shared != L->shared_inter)
        return set_error(kErrArgument, "the workspace was made for a layer of another shape");
    if (T > w->max_tokens)
        return set_error(kErrArgument, "%zu tokens, the workspace holds %zu", T, w->max_tokens);
    if (T) {
        if (int r = check_weights(L)) return r;
        if (!x || !y) return set_error(kErrArgument, "NULL operand");
        if ((uintptr_t)x % 16 || (uintptr_t)y % 16)
            return set_error(kErrUnsupported, "x and y need 16-byte alignment");
    }
    if (int r = mx_ready()) return r;
    if (!T) return kOk;
    MoeArgs a{};
    a.x = x;
    a.y = y;
    a.w_router = L->w_router;
    a.w_sgate = L->shared_inter ? L->w_shared_gate : nullptr;
    a.w_gu = L->w_gate_up;
    a.w_dn = L->w_down;
    a.w_sgu = L->w_shared_gate_up;
    a.w_sdn = L->w_shared_down;
    a.s_gu = L->s_gate_up;
    a.s_dn = L->s_down;
    a.s_sgu = L->s_shared_gate_up;
    a.s_sdn = L->s_shared_down;
    a.logits = w->logits;
    a.wts = w->wts;
    a.part = w->part;
    a.ids = w->ids;
    a.h = w->h;
    a.T = (int)T;
    a.H = (int)L->hidden;
    a.I = (int)L->inter;
    a.E = (int)L->experts;
    a.k = (int)L->topk;
    a.Is = (int)L->shared_inter;
    a.norm = L->norm_topk;
    const dim3 rg(cdiv(L->experts + (a.w_sgate ? 1 : 0), 16), cdiv(T, 16));
    APUS_TIMED("k_moe_router", k_moe_router<<<rg, 256, 0, stream()>>>(a));
    APUS_LAUNCHED("k_moe_router");
    APUS_TIMED("k_moe_topk", k_moe_topk<<<cdiv(T, 4), 256, 0, stream()>>>(a));
    APUS_LAUNCHED("k_moe_topk");
    if (int r = L->mxfp4 ? experts_run<WMx>(a) : experts_run<WBf16>(a)) return r;
    APUS_TIMED("k_moe_combine", k_moe_combine<<<cdiv(T * (L->hidden / 4), 256), 256, 0, stream()>>>(a));
    return launch_check("k_moe_combine");
}

}  // extern "C"

// moe.hip -- the mixture-of-experts layer of a decode step (up to
// kMoeMaxTokens tokens): per token x
//   l_e = w_router[e] . x,  the topk largest l_e (ties to the lowest index),
//   p_e = exp(l_e - max) / sum of the same over the chosen (norm_topk) or all,
//   y = sum_e p_e down_e(silu(gate_e x) * (up_e x))
//       + sigmoid(w_shared_gate . x) shared(x),
// everything in fp32, rounded once, at y. The weights are bf16 or MXFP4.
//
// For few tokens the layer is the reading of the chosen experts' weights, so
// every kernel streams weights through the MFMA with tokens as its 16 columns.
// Launches:
//   k_moe_router     logits; by the last workgroup of each 16 tokens to finish the
//                    choice, by the last of those the choices sorted by expert
//   k_moe_up[_stream]   h = silu(gate) up of every (expert, 16 outputs)
//   k_moe_down[_stream] fp32 rows of every (expert, 32 outputs), and
//   k_moe_combine       their weighted sum; or for little work
//   k_moe_down_few      both in one.
// The intermediate h = silu(g) u goes to the down product as three bf16 numbers that sum
// to its 24 bits: three MFMAs, of exact products, where fp32 operands would take sixteen.
// The product reads weights, not h, so they cost little. (As two numbers, 16 bits, 56 to
// 72 of 13728 outputs rounded another way than those of 64 bits, now 0 to 5, as plain fp32
// sums do; us: 64 tokens, MXFP4, 88, now 89; 325 tokens, bf16, 341, now 338.)
//
// Times below: hidden 2048, 256 experts of 512 inner elements, 8 a token, a shared
// expert of 512, inputs other than the call before's. The whole layer, us at
// 1 / 5 / 16 / 64 / 325 tokens: MXFP4 19 / 40 / 63 / 110 / 154 (bytes alone, at a
// large copy's 5.2 TB/s: 3 / 14 / 35 / 74 / 86), bf16 27 / 71 / 152 / 291 / 359
// (11 / 51 / 127 / 272 / 314): with many choices it is bound by the weights' bytes,
// with few by three launches' latency. Where a rule gives two sides, the tokens share a
// direction, so that some experts are preferred.
#include <stdint.h>

#include <algorithm>
#include <new>

#include "../../include/apus_hip.h"
#include "apus_dev.h"
#include "apus_host.h"
#include "mx.h"
#include "mx_dev.h"

using namespace apus;

// The device buffers of calls on one layer shape, and the shape they fit.
struct ApusHipMoeWork {
    size_t max_tokens, hidden, inter, experts, topk, shared;
    int device;
    char *base = nullptr;
    float *logits;       // [T][E + 1]: the experts', then the shared gate's
    int32_t *ids;        // [T][topk]
    float *wts;          // [T][topk + 1]: p, then the shared expert's weight
    uint16_t *h;         // [T topk][inter / 4][2][4], then [T][shared / 4][2][4]: h's upper 16 bits
    uint16_t *hl;        // [T topk][inter], then [T][shared]: the rest
    float *part;         // [T topk + T][hidden]
    uint32_t *done;      // workgroups of k_moe_router done, per 16 tokens, then of
                         // those the ones that have chosen (0 between calls)
    int4 *slots;         // expert, first of its choices in list, how many (up to group)
    uint16_t *list;      // [T topk]: choices by expert
};

namespace {

constexpr size_t kMoeMaxTokens = 1024, kMoeMaxExperts = 1024, kMoeMaxTopk = 32;
// Most rows of a slot. 32 from 8 choices an expert on, MXFP4 weights from 30, where that
// leaves 2048 blocks of 16 inner elements; else 16: the kernels for 16 have fewer registers
// and less LDS and more wavefronts, but read the weights of an expert with more rows again
// (us with 16 | 32: bf16, 192 tokens 300 | 302, 256 tokens 321 | 320, 768 tokens 471 | 428;
// 128 experts of 768, 8 a token, 128 tokens 252 | 249, 1024 tokens 602 | 480; 8 experts of
// 14336, 2 a token, 64 tokens 682 | 631. MXFP4, 96 tokens 104 | 111, 768 tokens 240 | 251,
// 1024 tokens 294 | 292; 128 experts of 768, 256 tokens 136 | 148, 512 tokens 203 | 205; 60 of
// 1408, 4 a token, 300 tokens 134 | 137, 900 tokens 264 | 255; 8 of 14336, 100 tokens 370 |
// 372, 128 tokens 462 | 398. 20 experts of 224, 3 a token, 512 tokens 38 | 44, bf16 49 | 55).
int slot_rows(size_t n, size_t E, size_t I, bool mx) {
    return n <= (mx ? 30 : 8) * E || (E + n / 32) * (I / 16) < 2048 ? 16 : 32;
}
// Choices are slots of their own, and nothing is sorted, while about two of them at
// most are expected to share an expert, whose weights are then read twice: n choices
// of E experts, n^2 / (2 E) of them. (Sorted | not, us: 3 tokens, MXFP4 32 | 29, bf16 51 |
// 49; 6 tokens 40 | 39, 74 | 75; 60 experts of 1408, 4 a token, MXFP4, 3 tokens 34 | 33, 6
// tokens 40 | 41; 8 experts of 4096, 2 a token, 3 tokens 41 | 48.)
bool choices_apart(size_t T, size_t n, size_t E) { return T == 1 || n * n <= 4 * E; }

struct MoeArgs {
    const uint16_t *x, *w_router, *w_sgate;
    const void *w_gu, *w_dn, *w_sgu, *w_sdn;
    const uint8_t *s_gu, *s_dn, *s_sgu, *s_sdn;
    float *logits, *wts, *part;
    int32_t *ids;
    uint32_t *done;
    int4 *slots;
    uint16_t *list;
    uint16_t *h, *hl;
    uint16_t *y;
    int T, H, I, E, k, Is, norm, nslots;
    int group;             // most rows of a slot: 16 or 32
    int apart;             // choices are slots of their own
};

// ---- router ---------------------------------------------------------------
// slots that T tokens can fill
size_t moe_slots(size_t T, size_t k, size_t E, size_t group) { return std::min(T * k, E) + T * k / group; }

// Order of logits as unsigned numbers: NaN above all, -0 and +0 alike. No
// number's key is 0.
__device__ __forceinline__ uint32_t order_key(float f) {
    uint32_t u = __float_as_uint(f + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if (u == 0x80000000u) u = 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return k == 0xffffffffu ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
// over the wavefront: within rows of 16 by lane permutations, the four rows
// from scalars
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp<0xb1>(v));                            // lane ^ 1
    v = max(v, dpp<0x4e>(v));                            // lane ^ 2
    v = max(v, dpp<0x141>(v));                           // mirrored halves of a row
    v = max(v, dpp<0x140>(v));                           // mirrored row
    auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    return max(max(at(0), at(16)), max(at(32), at(48)));
}
__device__ __forceinline__ float wave_sum(float f) {
    auto add = [](float a, uint32_t b) { return a + __uint_as_float(b); };
    f = add(f, dpp<0xb1>(__float_as_uint(f)));
    f = add(f, dpp<0x4e>(__float_as_uint(f)));
    f = add(f, dpp<0x141>(__float_as_uint(f)));
    f = add(f, dpp<0x140>(__float_as_uint(f)));
    return (lane_bcast(f, 0) + lane_bcast(f, 16)) + (lane_bcast(f, 32) + lane_bcast(f, 48));
}

// A wavefront's choice for token t, in index order: lane l holds logits l,
// l + 64, ... The k-th largest key is found two bits at a time from the top,
// counting by ballots (of 8 of 256, k rounds of a maximum over the wavefront took
// 8 us, this takes about one); of the keys equal to it the lowest indices are taken.
template <int NJ, class Logit>
__device__ __forceinline__ void choose(const MoeArgs &a, int t, int lane, int *sids, Logit logit) {
    float l[NJ];
    uint32_t key[NJ], best = 0;            // key 0: past E
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const int e = lane + 64 * j;
        l[j] = logit(min(e, a.E - 1));
        key[j] = e < a.E ? order_key(l[j]) : 0;
    }
    const float sgate = logit(a.w_sgate ? a.E : 0);
#pragma unroll
    for (int j = 0; j < NJ; j++) best = max(best, key[j]);
    const float top = key_value(wave_max(best));
    auto count = [&](uint32_t v) {         // keys >= v
        int n = 0;
#pragma unroll
        for (int j = 0; j < NJ; j++) n += __popcll(__ballot(key[j] >= v));
        return n;
    };
    uint32_t v = 0;
    for (int b = 30; b >= 0; b -= 2) {
        const uint32_t c1 = v | 1u << b, c2 = v | 2u << b, c3 = v | 3u << b;
        const int n1 = count(c1), n2 = count(c2), n3 = count(c3);
        if (n1 < a.k) continue;
        v = n3 >= a.k ? c3 : n2 >= a.k ? c2 : c1;
        if ((n3 >= a.k ? n3 : n2 >= a.k ? n2 : n1) == a.k) break;
    }
    const int above = v == 0xffffffffu ? 0 : count(v + 1);           // keys > v
    int ties = a.k - above, at = 0;        // of the keys equal to v, the first `ties`
    const uint64_t below = (1ull << lane) - 1;
    int pos[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const uint64_t eq = __ballot(key[j] == v);
        const bool in = key[j] > v || (key[j] == v && __popcll(eq & below) < ties);
        const uint64_t m = __ballot(in);
        pos[j] = in ? at + __popcll(m & below) : -1;
        at += __popcll(m);
        ties -= min(ties, (int)__popcll(eq));
    }
    float p[NJ], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        p[j] = expf(l[j] - top);
        if (lane + 64 * j < a.E && (pos[j] >= 0 || !a.norm)) sum += p[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < NJ; j++)
        if (pos[j] >= 0) {
            __hip_atomic_store(a.ids + t * a.k + pos[j], lane + 64 * j, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
            sids[pos[j]] = lane + 64 * j;
            a.wts[t * (a.k + 1) + pos[j]] = p[j] / sum;
        }
    if (lane == 0)
        a.wts[t * (a.k + 1) + a.k] = a.w_sgate ? 1.0f / (1.0f + expf(-sgate)) : 1.0f;
}

constexpr int kRouterWaves = 16;

// The choices of all tokens by expert, by one workgroup: count, sum, place (2.5 us).
// In which order an expert's choices come does not matter: a choice's values do not
// depend on its place.
__device__ __forceinline__ void make_slots(const MoeArgs &a, const int *sids, int lane, int wave) {
    __shared__ int cursor[kMoeMaxExperts], wsum[2][kRouterWaves];
    constexpr int THREADS = 64 * kRouterWaves, KEEP = 4;
    const int tid = threadIdx.x, n = a.T * a.k;
    auto id = [&](int q) {                 // from LDS, or as chosen by other workgroups of this launch
        const int e = sids ? sids[q] : __hip_atomic_load(a.ids + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return min(max(e, 0), a.E - 1);    // (in range whatever ids holds)
    };
    int mine[KEEP];                        // the first ids, read once
#pragma unroll
    for (int i = 0; i < KEEP; i++) mine[i] = tid + i * THREADS < n ? id(tid + i * THREADS) : 0;
    cursor[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (tid + i * THREADS < n) atomicAdd(&cursor[mine[i]], 1);
    for (int q = tid + KEEP * THREADS; q < n; q += THREADS) atomicAdd(&cursor[id(q)], 1);
    __syncthreads();
    // thread e: running sums over the experts, of the choices and of the slots
    const int c = cursor[tid], k = (c + a.group - 1) / a.group;
    int at = c, slot = k;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(at, d), u = __shfl_up(slot, d);
        if (lane >= d) {
            at += o;
            slot += u;
        }
    }
    if (lane == 63) {
        wsum[0][wave] = at;
        wsum[1][wave] = slot;
    }
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kRouterWaves; w++) {
        if (w < wave) {
            at += wsum[0][w];
            slot += wsum[1][w];
        }
        total += wsum[1][w];
    }
    for (int i = 0; i < k; i++)
        a.slots[slot - k + i] = make_int4(tid, at - c + i * a.group, min(a.group, c - i * a.group), 0);
    for (int i = total + tid; i < a.nslots; i += THREADS) a.slots[i] = make_int4(0, 0, 0, 0);
    cursor[tid] = at - c;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (tid + i * THREADS < n) a.list[atomicAdd(&cursor[mine[i]], 1)] = (uint16_t)(tid + i * THREADS);
    for (int q = tid + KEEP * THREADS; q < n; q += THREADS) a.list[atomicAdd(&cursor[id(q)], 1)] = (uint16_t)q;
}

// ET tiles of 16 experts (the shared gate's one row is a tile of its own) x 16
// tokens a workgroup, K over its 16 / ET wavefronts of a tile. The last workgroup
// of the 16 tokens to finish chooses for them, a wavefront each, and unless choices
// stay apart the last of those sorts them: what a workgroup hands on it
// stores where all XCDs see it, waits for the stores, and counts itself; nobody
// waits for anybody. Bound by latency: 7 us for one token, 12 for 16, 14 for 64, 21
// for 325. (Choosing in every workgroup of the next launch instead costs that launch
// as much as is saved here.) Of up to kSmallTiles tiles of few elements one workgroup
// takes all, and hands nothing on: 13 tokens of 1056, 20 experts, 7 us, 9 with the
// hand-over (small layers, us with one workgroup | several: one token, 8 experts, hidden
// 4096 17.0 | 18.1, 8192 27.3 | 26.7; 40 experts, 1024 13.2 | 13.8, 2048 15.4 | 14.8, 4096
// 20.8 | 18.2).
constexpr int kSmallTiles = 4, kSmallElements = 4096;    // tiles, tiles times hidden
static_assert(64 * kRouterWaves >= kMoeMaxExperts, "a thread per expert");
int router_tiles(const MoeArgs &a) { return (a.E + 15) / 16 + (a.w_sgate ? 1 : 0); }
template <int NJ, int ET>
__global__ __launch_bounds__(64 * kRouterWaves) void k_moe_router(MoeArgs a) {
    constexpr int KW = kRouterWaves / ET;
    __shared__ __attribute__((aligned(16))) char sm[kRouterWaves * WBf16::kTile];
    __shared__ int last, sids[16 * kMoeMaxTopk];
    __shared__ float slog[ET == 1 ? 1 : 16 * (16 * ET + 1)];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int E1 = a.E + 1, t0 = blockIdx.y * 16;
    const int ntiles = (a.E + 15) / 16 + (a.w_sgate ? 1 : 0), tile = ET == 1 ? blockIdx.x : wave / KW;
    const bool gate = a.w_sgate && tile == ntiles - 1;
    const int e0 = gate ? a.E : tile * 16, ne = tile >= ntiles ? 0 : gate ? 1 : min(16, a.E - e0);
    const auto wt = gate ? WBf16::tile(a.w_sgate, nullptr, 0, 1, a.H)
                         : WBf16::tile(a.w_router, nullptr, min(e0, a.E - 1), ne, a.H);
    const auto wl = WBf16::raw_lane(lane, a.H);
    using X = XBf16<WBf16>;
    const i32x4 xb = dma_rsrc(a.x, (uint32_t)a.T * (uint32_t)a.H * 2);
    uint32_t xl[4];
#pragma unroll
    for (int i = 0; i < 4; i++) xl[i] = (uint32_t)(t0 + 4 * i + g) * (uint32_t)a.H * 2;
    char *const m = sm + wave * WBf16::kTile;
    mx_f32x4 acc{};
    for (int st = wave % KW; st * 128 < a.H && ne; st += KW) {
        WBf16::Raw wf;
        RowsBf16::Raw xf;
        WBf16::load_raw(wf, wt, wl, st, a.H);
        X::load_raw(xf, xb, xl, st, a.H);
        WBf16::Frag f;
        WBf16::put(m, wf, lane);
        WBf16::get(f, m, wf, lane);
        RowsBf16::put(m, xf, lane);
#pragma unroll
        for (int j = 0; j < 4; j++) acc = mfma16(WBf16::operand(f, j), X::piece(m, j, lane), acc);
    }
    *reinterpret_cast<mx_f32x4 *>(m + lane * 16) = acc;
    __syncthreads();
    if (wave % KW == 0) {                  // the logits of a tile: expert 4 g + i of it, token r
        mx_f32x4 s[4] = {};
#pragma unroll
        for (int i = 0; i < KW; i++) s[i & 3] += *reinterpret_cast<const mx_f32x4 *>(m + i * WBf16::kTile + lane * 16);
        acc = (s[0] + s[1]) + (s[2] + s[3]);
    }
    auto count = [&](uint32_t *done, uint32_t of) {      // thread 0: the last of `of`?
        const uint32_t n = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = n == of - 1;
        if (last) *done = 0;                             // for the next call
    };
    if constexpr (ET == 1) {
        if (wave == 0) {
            if (t0 + r < a.T) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (4 * g + i < ne)
                        __hip_atomic_store(a.logits + (size_t)(t0 + r) * E1 + e0 + 4 * g + i, acc[i],
                                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (lane == 0) count(a.done + blockIdx.y, gridDim.x);
        }
        __syncthreads();
        if (!last) return;
        const float *lg = a.logits + (size_t)(t0 + wave) * E1;
        if (t0 + wave < a.T)
            choose<NJ>(a, t0 + wave, lane, sids + wave * a.k, [&](int e) {
                return __hip_atomic_load(lg + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            });
    } else {
        constexpr int P = 16 * ET + 1;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (wave % KW == 0 && 4 * g + i < ne) slog[r * P + e0 + 4 * g + i] = acc[i];
        __syncthreads();
        if (t0 + wave < a.T)
            choose<NJ>(a, t0 + wave, lane, sids + wave * a.k, [&](int e) { return slog[wave * P + e]; });
    }
    if (a.apart) return;
    if (gridDim.y == 1) {                  // (one workgroup has chosen for all)
        __syncthreads();
        return make_slots(a, sids, lane, wave);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) count(a.done + gridDim.y, gridDim.y);
    __syncthreads();
    if (last) make_slots(a, nullptr, lane, wave);
}

// ---- experts ----------------------------------------------------------------
// What a workgroup works on: n rows of the activations, for the expert's row
// blocks. Blocks of a launch: first the shared expert's, nsh row blocks for
// every `group` tokens; then nper row blocks per slot. A slot is up to `group` of
// an expert's choices (a popular expert has several, side by side on the chip
// instead of one after the other), or, where they stay apart, a choice.
struct Task {
    int e, part, first, n;                 // e == E: shared; n = 0: nothing
    const uint16_t *list;                  // or null: choices first, first + 1, ..
};
__device__ __forceinline__ Task task_of(const MoeArgs &a, int b, int nsh, int nper) {
    const int groups = nsh ? (a.T + a.group - 1) / a.group : 0;
    if (b < nsh * groups) {
        const int t = b / nsh * a.group;
        return {a.E, b % nsh, a.T * a.k + t, min(a.group, a.T - t), nullptr};
    }
    b -= nsh * groups;
    const int slot = b / nper, part = b % nper;
    if (a.apart) return {__builtin_amdgcn_readfirstlane(a.ids[slot]), part, slot, 1, nullptr};
    const int4 s = a.slots[slot];
    return {__builtin_amdgcn_readfirstlane(s.x), part, 0, __builtin_amdgcn_readfirstlane(s.z),
            a.list + __builtin_amdgcn_readfirstlane(s.y)};
}
__device__ __forceinline__ int choice(const Task &k, int i) {
    i = min(i, k.n - 1);
    return k.list ? k.list[i] : k.first + i;
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

// h goes to the down product as three numbers of bf16 (Split): the first and the second in
// a.h, 4 of either in turn, the third in a.hl. Choice q has a row of I: the elements before
// it, and all.
__device__ __forceinline__ uint32_t h_at(const MoeArgs &a, int q, bool sh) {
    const uint32_t n = a.T * a.k;
    return sh ? n * a.I + (q - n) * a.Is : q * a.I;
}
__device__ __forceinline__ uint32_t h_all(const MoeArgs &a) { return a.T * (a.k * a.I + a.Is); }

// The 24 bits of an fp32 number as three numbers of bf16 that sum to it (as far as bf16
// reaches down, 2^-133): its leading 8 bits, the next 8, both cut, and the rest. All have
// its sign, and none is zero where the first is not: times an infinite weight that would
// make NaN of an infinite y. What would be zero is bf16's least number. Two at a time.
struct Split {
    uint32_t v[3];
};
__device__ __forceinline__ Split split2(uint32_t a, uint32_t b) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    auto top = [](uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302); };
    auto rest = [](float f) { return f - __uint_as_float(__float_as_uint(f) & 0xffff0000u); };
    const uint32_t hi = top(a, b);
    // (of infinite and NaN no rest: fmaxf drops a NaN)
    const float ra = fmaxf(rest(__uint_as_float(a & 0x7fffffffu)), 0.0f);
    const float rb = fmaxf(rest(__uint_as_float(b & 0x7fffffffu)), 0.0f);
    const mx_bf16x2 lo{(__bf16)rest(ra), (__bf16)rest(rb)};
    const u16x2 least = __builtin_elementwise_min(__builtin_bit_cast(u16x2, hi & 0x7fff7fffu), u16x2{1, 1});
    auto full = [&](uint32_t x) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, x), least)) | (hi & 0x80008000u);
    };
    return {hi, full(top(__float_as_uint(ra), __float_as_uint(rb))), full(__builtin_bit_cast(uint32_t, lo))};
}

// Two forms of each expert kernel. k_moe_up and k_moe_down share a row block's K
// out over the 8 wavefronts of a workgroup, whose partial sums meet in LDS: most
// bytes on their way at once for a task, for calls with few of them. Where the
// row blocks are enough wavefronts to fill the chip, in k_moe_up_stream and
// k_moe_down_stream each walks all of K for its rows by itself.
// In all of them weights come along their rows (load_raw) and become operands in the
// wavefront's own LDS; loaded by each lane for itself they took the address unit four
// times as long (one token: 31 us for the layer, now 26; MXFP4 23, now 19).
constexpr int kMoeWaves = 8;

// h = silu(gate x) * (up x): 16 outputs a workgroup, 16 rows at a time. One token: 9.2
// us for bf16's 38 MB, 4.2 for MXFP4's 10 MB: latency of one round of loads.
template <class W>
__global__ __launch_bounds__(64 * kMoeWaves) void k_moe_up(MoeArgs a, int nsh, int nper) {
    constexpr int S = 2;                   // steps in flight at once
    constexpr int LDS = W::kTile < 2048 ? 2048 : W::kTile;
    __shared__ __attribute__((aligned(16))) char sm[kMoeWaves * LDS];
    __shared__ int rows[16];
    using X = XBf16<W>;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Task task = task_of(a, blockIdx.x, nsh, nper);
    if (task.n == 0) return;
    const bool sh = task.e == a.E;
    const int I = sh ? a.Is : a.I, o0 = task.part * 16;
    typename W::Tile wt[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        wt[i] = W::tile(sh ? a.w_sgu : a.w_gu, sh ? a.s_sgu : a.s_gu,
                        (sh ? 0 : (size_t)task.e * 2 * I) + i * I + o0, 16, a.H);
    const auto wl = W::raw_lane(lane, a.H);
    const i32x4 xb = dma_rsrc(a.x, (uint32_t)a.T * (uint32_t)a.H * 2);
    char *const m = sm + wave * LDS;
    for (int c = 0; c < task.n; c += 16) {
        const int q = choice(task, c + r);
        // (each lane its own row: of few rows most lanes read the same one)
        const uint32_t xl = X::lane((uint32_t)(sh ? q - a.T * a.k : q / a.k) * (uint32_t)a.H * 2, g);
        if (c) __syncthreads();                          // the sums have been read
        mx_f32x4 acc[2] = {};
        for (int st = wave * S; st * 128 < a.H; st += kMoeWaves * S) {
            typename W::Raw fw[S][2];
            typename X::Frag fx[S];
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int i = 0; i < 2; i++) W::load_raw(fw[s][i], wt[i], wl, st + s, a.H);
#pragma unroll
            for (int s = 0; s < S; s++) X::load(fx[s], xb, xl, st + s, a.H);
            // (all loads issued before the first use)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    typename W::Frag f;
                    W::put(m, fw[s][i], lane);
                    W::get(f, m, fw[s][i], lane);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[i] = mfma16(W::operand(f, j), __builtin_bit_cast(mx_bf16x8, fx[s].v[j]), acc[i]);
                }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) *reinterpret_cast<mx_f32x4 *>(m + i * 1024 + lane * 16) = acc[i];
        if (wave == 0 && g == 0) rows[r] = q;
        __syncthreads();
        // a thread finishes one output of a row, 16 outputs of a row side by side
        const int o = threadIdx.x & 15, row = threadIdx.x >> 4;
        if (row < 16 && c + row < task.n) {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kMoeWaves; w++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    s[i] += *reinterpret_cast<const float *>(sm + w * LDS + i * 1024 + ((o >> 2) * 16 + row) * 16 +
                                                             (o & 3) * 4);
            const uint32_t at = h_at(a, rows[row], sh) + o0 + o;
            const Split v = split2(__float_as_uint(silu(s[0]) * s[1]), 0);
            uint16_t *const h = a.h + (at & ~3u) * 2 + at % 4;
            h[0] = (uint16_t)v.v[0];
            h[4] = (uint16_t)v.v[1];
            a.hl[at] = (uint16_t)v.v[2];
        }
    }
}

// wavefronts that share a row block's K in k_moe_down, a step each (longer rows:
// more rounds), for I inner elements, and the rows of a workgroup
__host__ __device__ constexpr int down_split(int I) { return I > 512 ? 8 : I > 256 ? 4 : I > 128 ? 2 : 1; }
__host__ __device__ constexpr int down_tiles(int I) { return I > 512 ? 4 : 2; }          // of a wavefront
__host__ __device__ constexpr int down_rows(int I) { return kMoeWaves / down_split(I) * 16 * down_tiles(I); }

// The three numbers of h are three products with the same weights. Where a task has up to
// kSideRows rows, they go side by side through one MFMA, as its columns kSideRows p + i.
// Their sums meet at the end, in the same order in both cases: an expert's choices fall into
// its slots in any order, and what a choice gets does not depend on its slot.
constexpr int kSideRows = 4;
__device__ __forceinline__ mx_f32x4 sum3(const mx_f32x4 (&v)[3]) { return v[0] + (v[1] + v[2]); }
__device__ __forceinline__ mx_f32x4 sum3(const mx_f32x4 (&v)[1]) {
    mx_f32x4 s = v[0];
#pragma unroll
    for (int i = 0; i < 4; i++) {          // of column i (lane i of 16) and the ones kSideRows and twice as many past it
        const float f = v[0][i];
        const uint32_t u = __float_as_uint(f);
        s[i] += __uint_as_float(dpp<0x100 + kSideRows>(u)) + __uint_as_float(dpp<0x100 + 2 * kSideRows>(u));
    }
    return s;
}

// part[choice] = down h: 32 outputs a group of wavefronts, 16 rows at a time (13 tokens
// of 1056, 20 experts of 224, MXFP4: 4.6 us). HL: loads of two rows of h (2 HL rows and no more
// with fewer than 8).
template <class W, int RT, int HL>
__device__ __forceinline__ void down_part(const MoeArgs &a, const Task &task, char *sm, int *rows) {
    constexpr bool SIDE = 2 * HL == kSideRows;
    constexpr int LDS = RowsBf16::kTile, N3 = SIDE ? 1 : 3;
    using X = XBf16<W>;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool sh = task.e == a.E;
    const int I = sh ? a.Is : a.I, ks = down_split(I), kw = wave % ks, rg = wave / ks;
    const int o0 = task.part * down_rows(I);
    typename W::Tile wt[RT];               // (a tile past H, not stored, repeats the last)
#pragma unroll
    for (int t = 0; t < RT; t++)
        wt[t] = W::tile(sh ? a.w_sdn : a.w_dn, sh ? a.s_sdn : a.s_dn,
                        (sh ? 0 : (size_t)task.e * a.H) + min(o0 + (rg * RT + t) * 16, a.H - 16), 16, I);
    const auto wl = W::raw_lane(lane, I);
    const i32x4 hb = dma_rsrc(a.h, h_all(a) * 4), lb = dma_rsrc(a.hl, h_all(a) * 2);
    char *const m = sm + wave * LDS;
    const int half = lane >> 5, e4 = lane & 31;
    for (int c = 0; c < task.n; c += 16) {
        const int q = choice(task, c + r);
        uint32_t at[HL], lat[HL / 2];
#pragma unroll
        for (int i = 0; i < HL; i++) at[i] = (h_at(a, choice(task, c + 2 * i + half), sh) + 4 * e4) * 4;
#pragma unroll
        for (int i = 0; i < HL / 2; i++) lat[i] = (h_at(a, choice(task, c + 4 * i + g), sh) + 8 * r) * 2;
        if (c) __syncthreads();                          // the sums have been read
        mx_f32x4 acc[RT][N3] = {};
        for (int st = kw; st * 128 < I; st += ks) {
            typename W::Raw fw[RT];
            u32x4 fh[HL], fl[HL / 2];
#pragma unroll
            for (int t = 0; t < RT; t++) W::load_raw(fw[t], wt[t], wl, st, I);
            const bool live = st * 128 + 4 * e4 < I, llive = st * 128 + 8 * r < I;
#pragma unroll
            for (int i = 0; i < HL; i++) fh[i] = ld16(hb, live ? at[i] : kPast, 512 * st);
#pragma unroll
            for (int i = 0; i < HL / 2; i++) fl[i] = ld16(lb, llive ? lat[i] : kPast, 256 * st);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            typename W::Frag f[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                W::put(m, fw[t], lane);
                W::get(f[t], m, fw[t], lane);
            }
            // (they share their LDS: what is written is read before the next)
            mx_bf16x8 h[N3][4];
#pragma unroll
            for (int p = 0; p < 3; p++) {
#pragma unroll
                for (int i = 0; i < HL; i++) {
                    const int row = (SIDE ? kSideRows * p : 0) + 2 * i + half;
                    char *const to = m + row * 256 + ((e4 / 2 ^ row) << 4) + e4 % 2 * 8;
                    if (p == 0) *reinterpret_cast<uint2 *>(to) = make_uint2(fh[i][0], fh[i][1]);
                    if (p == 1) *reinterpret_cast<uint2 *>(to) = make_uint2(fh[i][2], fh[i][3]);
                }
#pragma unroll
                for (int i = 0; i < HL / 2; i++) {
                    const int row = (SIDE ? kSideRows * p : 0) + 4 * i + g;
                    if (p == 2) *reinterpret_cast<u32x4 *>(m + row * 256 + ((r ^ row) << 4)) = fl[i];
                }
                if (SIDE && p < 2) continue;
#pragma unroll
                for (int j = 0; j < 4; j++) h[SIDE ? 0 : p][j] = X::piece(m, j, lane);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const mx_bf16x8 wv = W::operand(f[t], j);
#pragma unroll
                    for (int p = 0; p < N3; p++) acc[t][p] = mfma16(wv, h[p][j], acc[t][p]);
                }
        }
#pragma unroll
        for (int t = 0; t < RT; t++) *reinterpret_cast<mx_f32x4 *>(m + t * 1024 + lane * 16) = sum3(acc[t]);
        if (wave == 0 && g == 0) rows[r] = q;
        __syncthreads();
        // a thread finishes 4 outputs of a row
        for (int e = threadIdx.x; e < kMoeWaves / ks * RT * 64; e += 64 * kMoeWaves) {
            const int l = e & 63, t = (e >> 6) % RT, x = (e >> 6) / RT;
            const int o = o0 + (x * RT + t) * 16;
            if (c + (l & 15) >= task.n || o >= a.H) continue;
            const char *p = sm + x * ks * LDS + t * 1024 + l * 16;
            mx_f32x4 s = *reinterpret_cast<const mx_f32x4 *>(p);
            for (int y = 1; y < ks; y++) s += *reinterpret_cast<const mx_f32x4 *>(p + y * LDS);
            *reinterpret_cast<mx_f32x4 *>(a.part + (size_t)rows[l & 15] * a.H + o + 4 * (l >> 4)) = s;
        }
    }
}
template <class W, int RT>
__device__ __forceinline__ void down_part_of(const MoeArgs &a, const Task &task, char *sm, int *rows) {
    if (task.n <= kSideRows) down_part<W, RT, kSideRows / 2>(a, task, sm, rows);
    else if (task.n <= 8) down_part<W, RT, 4>(a, task, sm, rows);
    else down_part<W, RT, 8>(a, task, sm, rows);
}
template <class W>
__global__ __launch_bounds__(64 * kMoeWaves) void k_moe_down(MoeArgs a, int nsh, int nper) {
    __shared__ __attribute__((aligned(16))) char sm[kMoeWaves * RowsBf16::kTile];
    __shared__ int rows[16];
    const Task task = task_of(a, blockIdx.x, nsh, nper);
    if (task.n == 0) return;
    if (down_tiles(task.e == a.E ? a.Is : a.I) == 4) down_part_of<W, 4>(a, task, sm, rows);
    else down_part_of<W, 2>(a, task, sm, rows);
}

// ---- the same, a wavefront alone: no partial sums, and D steps of weights (up: and
// activations) on their way all along its walk. Up: bf16, 325 tokens, 191
// us for 1.09 GB fetched, 5.7 TB/s; MXFP4, 64 tokens, 45 us for 194 MB, 4.3 TB/s. Down:
// 103 us for 0.57 GB, 5.5 TB/s; 27 us for 103 MB, 3.8 TB/s. More steps on their way (3, 4)
// changed nothing, nor did whole 128-byte lines of MXFP4 codes a load.
constexpr int kStreamWaves = 4;

// (what comes before stays before)
__device__ __forceinline__ void fence() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// steps [0, n) of a walk: load(slot, step), and mul(slot, step), which takes the
// slot's operands before it requests the step D after. The last round may go up
// to D - 1 steps past n: zeros.
template <int D, class Mul>
__device__ __forceinline__ void walk_on(int n, Mul mul) {
    for (int b = 0; b < n; b += D) {
#pragma unroll
        for (int d = 0; d < D; d++) mul(d, b + d);
    }
}
template <int D, class Load, class Mul>
__device__ __forceinline__ void walk(int n, Load load, Mul mul) {
#pragma unroll
    for (int d = 0; d < D; d++) load(d, d);
    fence();
    walk_on<D>(n, mul);
}

// XR: loads of four rows that a tile of activations takes (1 for up to 4 rows). SC:
// MXFP4 weights' scales in strips.
template <class W, int NT, int D, int XR, bool SC>
__device__ __forceinline__ void up_stream(const MoeArgs &a, const Task &task, int o0, char *m, int lane) {
    using X = XBf16<W>;
    const int r = lane & 15, g = lane >> 4;
    const bool sh = task.e == a.E;
    const int I = sh ? a.Is : a.I;
    typename W::Tile wt[2];                // gate, up
#pragma unroll
    for (int i = 0; i < 2; i++)
        wt[i] = W::tile(sh ? a.w_sgu : a.w_gu, sh ? a.s_sgu : a.s_gu,
                        (sh ? 0 : (size_t)task.e * 2 * I) + i * I + o0, 16, a.H);
    const auto wl = W::raw_lane(lane, a.H);
    const i32x4 xb = dma_rsrc(a.x, (uint32_t)a.T * (uint32_t)a.H * 2);
    int q[NT];
    uint32_t xl[NT][4];
#pragma unroll
    for (int u = 0; u < NT; u++) {
        q[u] = choice(task, 16 * u + r);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int x = choice(task, 16 * u + 4 * i + g);
            xl[u][i] = (uint32_t)(sh ? x - a.T * a.k : x / a.k) * (uint32_t)a.H * 2;
        }
    }
    typename W::Raw fw[D][2];
    RowsBf16::Raw fx[D][NT];
    char *const mx = m + 2 * W::kTile, *const ms = mx + NT * RowsBf16::kTile;
    Strip strip[SC ? 2 : 1];
    auto load = [&](int d, int st) {
        if constexpr (SC) {
            if ((st & (Strip::kSteps - 1)) == 0) {
#pragma unroll
                for (int t = 0; t < 2; t++) strip[t].load(wt[t], st, a.H);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) W::template load_raw<!SC>(fw[d][i], wt[i], wl, st, a.H);
#pragma unroll
        for (int u = 0; u < NT; u++) X::template load_raw<XR>(fx[d][u], xb, xl[u], st, a.H);
    };
    mx_f32x4 acc[2][NT] = {};
    walk<D>((a.H + 127) / 128, load, [&](int d, int st) {
#pragma unroll
        for (int t = 0; t < 2; t++) W::put(m + t * W::kTile, fw[d][t], lane);
#pragma unroll
        for (int u = 0; u < NT; u++) RowsBf16::put(mx + u * RowsBf16::kTile, fx[d][u], lane);
        typename W::Frag f[2];
#pragma unroll
        for (int t = 0; t < 2; t++) W::template get<!SC>(f[t], m + t * W::kTile, fw[d][t], lane);
        if constexpr (SC) {
            if ((st & (Strip::kSteps - 1)) == 0) {
#pragma unroll
                for (int t = 0; t < 2; t++) strip[t].put(ms + t * Strip::kTile);
            }
#pragma unroll
            for (int t = 0; t < 2; t++) f[t].s = Strip::get(ms + t * Strip::kTile, st, lane);
        }
        fence();
        load(d, st + D);
        fence();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mx_bf16x8 x[NT];
#pragma unroll
            for (int u = 0; u < NT; u++) x[u] = X::piece(mx + u * RowsBf16::kTile, j, lane);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const mx_bf16x8 w = W::operand(f[i], j);
#pragma unroll
                for (int u = 0; u < NT; u++) acc[i][u] = mfma16(w, x[u], acc[i][u]);
            }
        }
        fence();
    });
#pragma unroll
    for (int u = 0; u < NT; u++) {
        if (16 * u + r >= task.n) continue;
        const uint32_t at = h_at(a, q[u], sh) + o0 + 4 * g;
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __float_as_uint(silu(acc[0][u][i]) * acc[1][u][i]);
        const Split s0 = split2(v[0], v[1]), s1 = split2(v[2], v[3]);
        *reinterpret_cast<u32x4 *>(a.h + at * 2) = u32x4{s0.v[0], s1.v[0], s0.v[1], s1.v[1]};
        *reinterpret_cast<uint2 *>(a.hl + at) = make_uint2(s0.v[2], s1.v[2]);
    }
}

template <class W, int NT, bool SC>
__global__ __launch_bounds__(64 * kStreamWaves, W::mx ? 3 : 2) void k_moe_up_stream(MoeArgs a, int nsh, int nper) {
    constexpr int LDS = 2 * (W::kTile + (SC ? Strip::kTile : 0)) + NT * RowsBf16::kTile;
    __shared__ __attribute__((aligned(16))) char sm[kStreamWaves * LDS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Task task = task_of(a, blockIdx.x, nsh, nper);
    const int o0 = (task.part * kStreamWaves + wave) * 16;
    if (task.n == 0 || o0 >= (task.e == a.E ? a.Is : a.I)) return;       // (no barrier in this kernel)
    if (NT > 1 && task.n > 16) up_stream<W, NT, 2, 4, SC>(a, task, o0, sm + wave * LDS, lane);
    else if (task.n > 4) up_stream<W, 1, 2, 4, SC>(a, task, o0, sm + wave * LDS, lane);
    else up_stream<W, 1, 2, 1, SC>(a, task, o0, sm + wave * LDS, lane);
}

// part[choice] = down h: 32 outputs a block, P blocks a wavefront in one walk (one
// block where I takes several chunks). h of the task's rows is brought to LDS once for all
// the workgroup's blocks, a chunk of 512 elements (with SIDE, of up to kSideRows rows, 2048)
// at a time; the next chunk's is on its way, in registers, while one is walked.
constexpr int kDownTiles = 2;                            // of 16 outputs, in a block
// wavefronts of a workgroup: two of 8 a CU, with bf16 weights, whose registers leave room for
// 8 wavefronts, two of 4, or one of 8 where h takes more LDS (128 experts of 768, 8 a token,
// bf16, 64 tokens 222 us with one of 8, now 218; 1024 tokens, 32 rows, 661 with 4, 524 with 8)
template <class W, int NT>
constexpr int kDownWaves = W::mx || NT > 1 ? 8 : 4;
constexpr int kDownChunk = 4;                            // steps of 128 elements
constexpr int kDownH = 16 * 3 * kDownChunk * 256;        // LDS bytes of 16 rows of a chunk
static_assert(3 * kSideRows * (kDownChunk * 16 / kSideRows) * 256 <= kDownH, "a chunk side by side fits");
template <class W, int NT, int D, int WAVES, bool MANY, bool SIDE>
__device__ __forceinline__ void down_stream(const MoeArgs &a, const Task &task, int b0, int nb, char *h, char *m,
                                            int lane) {
    static_assert(NT == 1 || !SIDE);
    constexpr int RT = kDownTiles;
    using X = XBf16<W>;
    constexpr int N3 = SIDE ? 1 : 3;       // MFMAs for the three numbers
    constexpr int CHUNK = SIDE ? kDownChunk * 16 / kSideRows : kDownChunk;
    const int r = lane & 15, g = lane >> 4;
    const bool sh = task.e == a.E;
    const int I = sh ? a.Is : a.I, steps = (I + 127) / 128, chunks = (steps + CHUNK - 1) / CHUNK;
    const auto wl = W::raw_lane(lane, I);
    typename W::Raw fw[D][RT];
    int lb = b0, ls = 0, mb = b0, ms = 0;  // row block and step to load, to multiply
    auto load = [&](int d, int) {
        const bool in = lb < b0 + nb;                    // (past the last: zeros)
#pragma unroll
        for (int t = 0; t < RT; t++)       // (a tile past H, not stored, repeats the last)
            W::load_raw(fw[d][t],
                        W::tile(sh ? a.w_sdn : a.w_dn, sh ? a.s_sdn : a.s_dn,
                                (sh ? 0 : (size_t)task.e * a.H) + min((in ? lb * RT + t : 0) * 16, a.H - 16), 16, I),
                        wl, in ? ls : steps, I);
        if (++ls == steps) {
            ls = 0;
            lb++;
        }
    };
#pragma unroll
    for (int d = 0; d < D; d++) load(d, d);
    fence();
    // Pieces of 8 elements of a row of h, and bytes of a row of one of its three numbers in
    // LDS: where there may be chunks of 512, whole ones, so that a wavefront brings a row.
    constexpr bool ROWS = MANY && !SIDE;
    const int pc = ROWS ? CHUNK * 16 : min(steps, CHUNK) * 16, pitch = pc * 16;
    // Piece c of number p of the task's row i lies at c ^ k within its 256 bytes, in LDS row
    // 3 i + p, k = i, or with SIDE in row k = kSideRows p + i. A thread's pieces past the last
    // row are the last row's again.
    constexpr int PIECES = ((SIDE ? kSideRows : 16 * NT) * (MANY ? CHUNK : kDownChunk) * 16 + 64 * WAVES - 1) / (64 * WAVES);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto row_of = [&](int n) {
        return min(ROWS ? wave + n * WAVES : (int)(threadIdx.x + n * 64 * WAVES) / pc, task.n - 1);
    };
    auto piece_of = [&](int n) { return ROWS ? lane : (int)(threadIdx.x + n * 64 * WAVES) % pc; };
    uint32_t at[PIECES];                   // elements before the rows
#pragma unroll
    for (int n = 0; n < PIECES; n++) at[n] = h_at(a, choice(task, row_of(n)), sh);
    u32x4 hr[PIECES][3];
    auto fetch = [&](int chunk) {          // (zeros past I)
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            const int k = chunk * CHUNK * 128 + piece_of(n) * 8;
            const uint32_t from = at[n] + (k < I ? k : 0);
            hr[n][0] = *reinterpret_cast<const u32x4 *>(a.h + (size_t)from * 2);
            hr[n][1] = *reinterpret_cast<const u32x4 *>(a.h + (size_t)from * 2 + 8);
            hr[n][2] = *reinterpret_cast<const u32x4 *>(a.hl + from);
#pragma unroll
            for (int p = 0; p < 3; p++)
                if (k >= I) hr[n][p] = u32x4{};
        }
    };
    auto put_h = [&]() {
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            if ((n * WAVES + wave) * 64 >= task.n * pc) continue;       // (all past the last row)
            const int i = row_of(n);
            const u32x4 a0 = hr[n][0], a1 = hr[n][1];
            const u32x4 v[3] = {u32x4{a0[0], a0[1], a1[0], a1[1]}, u32x4{a0[2], a0[3], a1[2], a1[3]}, hr[n][2]};
#pragma unroll
            for (int p = 0; p < 3; p++) {
                const int to = SIDE ? kSideRows * p + i : 3 * i + p, key = SIDE ? to : i & 15;
                *reinterpret_cast<u32x4 *>(h + to * pitch + ((piece_of(n) ^ key) << 4)) = v[p];
            }
        }
    };
    mx_f32x4 acc[RT][NT][N3] = {};
    auto mul = [&](int d, int st) {
#pragma unroll
        for (int t = 0; t < RT; t++) W::put(m + t * W::kTile, fw[d][t], lane);
        typename W::Frag f[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) W::get(f[t], m + t * W::kTile, fw[d][t], lane);
        fence();
        load(d, st + D);
        fence();
        // (a step past the last, of zero weights, reads the last step's h)
        const char *hs = h + (SIDE ? min(r, 3 * kSideRows - 1) : 3 * r) * pitch + min(ms, steps - 1) % CHUNK * 256;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mx_bf16x8 v[NT][N3];
#pragma unroll
            for (int u = 0; u < NT; u++)
#pragma unroll
                for (int p = 0; p < N3; p++)
                    v[u][p] = *reinterpret_cast<const mx_bf16x8 *>(hs + (u * 48 + p) * pitch + ((X::piece_of(j, g) ^ r) << 4));
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const mx_bf16x8 w = W::operand(f[t], j);
#pragma unroll
                for (int u = 0; u < NT; u++)
#pragma unroll
                    for (int p = 0; p < N3; p++) acc[t][u][p] = mfma16(w, v[u][p], acc[t][u][p]);
            }
        }
        fence();
        if (++ms < steps) return;
        ms = 0;
#pragma unroll
        for (int u = 0; u < NT; u++)
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int o = (mb * RT + t) * 16;
                const mx_f32x4 s = sum3(acc[t][u]);
                if (16 * u + r < task.n && o < a.H && mb < b0 + nb)
                    *reinterpret_cast<mx_f32x4 *>(a.part + (size_t)choice(task, 16 * u + r) * a.H + o + 4 * g) = s;
#pragma unroll
                for (int p = 0; p < N3; p++) acc[t][u][p] = mx_f32x4{};
            }
        mb++;
    };
    fetch(0);
    put_h();
    __syncthreads();
    if (!MANY) return walk_on<D>(nb * steps, mul);
    for (int c = 0;; c++) {                // (every wavefront comes to every barrier)
        const bool more = c + 1 < chunks;
        if (more) fetch(c + 1);
        fence();
        if (nb > 0) walk_on<D>(min(CHUNK, steps - c * CHUNK), mul);
        if (!more) break;
        __syncthreads();                   // the chunk has been read
        put_h();
        __syncthreads();
    }
}

template <class W, int NT, bool MANY>
__global__ __launch_bounds__((64 * kDownWaves<W, NT>), W::mx && NT == 1 ? 4 : 2) void k_moe_down_stream(MoeArgs a, int nsh, int nper, int P) {
    constexpr int LDS = kDownTiles * W::kTile, WAVES = kDownWaves<W, NT>;
    __shared__ __attribute__((aligned(16))) char sm[WAVES * LDS + NT * kDownH];
    char *const h = sm + WAVES * LDS;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Task task = task_of(a, blockIdx.x, nsh, nper);
    if (task.n == 0) return;
    char *const m = sm + wave * LDS;
    const int blocks = (a.H + 16 * kDownTiles - 1) / (16 * kDownTiles), b0 = (task.part * WAVES + wave) * P;
    const int nb = min(P, blocks - b0);
    if (NT > 1 && task.n > 16) down_stream<W, NT, 2, WAVES, MANY, false>(a, task, b0, nb, h, m, lane);
    else if (task.n > kSideRows) down_stream<W, 1, 2, WAVES, MANY, false>(a, task, b0, nb, h, m, lane);
    else down_stream<W, 1, 2, WAVES, MANY, true>(a, task, b0, nb, h, m, lane);
}

// y of up to 16 tokens: 16 outputs a workgroup, the steps of 128 k of every (token,
// expert) dealt to its 12 wavefronts (9 experts of 4 steps, one token: 3 each, all on
// their way at once). A step's product lands in the token's column with the
// expert's weight; the columns of other tokens (all multiplied with this token's h)
// are left out. One token: 6.0 us for bf16's 19 MB, 5.5 for MXFP4's 5 MB.
constexpr int kFewWaves = 12, kFewUnits = 3;
template <class W>
__global__ __launch_bounds__(64 * kFewWaves) void k_moe_down_few(MoeArgs a) {
    constexpr int HB = 3 * 256, LDS = W::kTile + kFewUnits * HB;     // bytes of a unit's h, of a wavefront
    __shared__ __attribute__((aligned(16))) char sm[kFewWaves * LDS];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = blockIdx.x * 16, n = a.T * a.k;
    const int si = (a.I + 127) / 128, ss = (a.Is + 127) / 128;
    const int units = n * si + a.T * ss;
    constexpr int U = kFewUnits;
    using X = XBf16<W>;
    char *const m = sm + wave * LDS, *const mh = m + W::kTile;
    const i32x4 hb = dma_rsrc(a.h, h_all(a) * 4), lb = dma_rsrc(a.hl, h_all(a) * 2);
    mx_f32x4 acc{};
    for (int b = wave; b < units; b += kFewWaves * U) {
        // choice, its expert, step and weight of each
        int q[U], e[U], st[U];
        float p[U];
        bool on[U], sh[U];
#pragma unroll
        for (int i = 0; i < U; i++) {
            const bool live = b + kFewWaves * i < units;
            const int u = live ? b + kFewWaves * i : b;
            sh[i] = u >= n * si;
            q[i] = sh[i] ? n + (u - n * si) / ss : u / si;
            st[i] = sh[i] ? (u - n * si) % ss : u % si;
            const int t = sh[i] ? q[i] - n : q[i] / a.k;
            e[i] = a.ids[sh[i] ? 0 : q[i]];
            p[i] = a.wts[t * (a.k + 1) + (sh[i] ? a.k : q[i] % a.k)];
            on[i] = live && t == r;
        }
        typename W::Raw fw[U];
        u32x4 fh[U], fl[U];                // h of a step, 4 elements in each of 32 lanes, 8 in each of 16
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int k = st[i] * 128, I = sh[i] ? a.Is : a.I;
            const uint32_t at = h_at(a, q[i], sh[i]);
            fh[i] = ld16(hb, lane < 32 && k + 4 * lane < I ? (at + 4 * lane) * 4 : kPast, 4 * k);
            fl[i] = ld16(lb, lane < 16 && k + 8 * lane < I ? (at + 8 * lane) * 2 : kPast, 2 * k);
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int I = sh[i] ? a.Is : a.I, x = __builtin_amdgcn_readfirstlane(e[i]);
            const auto wt = W::tile(sh[i] ? a.w_sdn : a.w_dn, sh[i] ? a.s_sdn : a.s_dn,
                                    (sh[i] ? 0 : (size_t)x * a.H) + o0, 16, I);
            W::load_raw(fw[i], wt, W::raw_lane(lane, I), st[i], I);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (lane < 32) {
                *reinterpret_cast<uint2 *>(mh + i * HB + lane * 8) = make_uint2(fh[i][0], fh[i][1]);
                *reinterpret_cast<uint2 *>(mh + i * HB + 256 + lane * 8) = make_uint2(fh[i][2], fh[i][3]);
            }
            if (lane < 16) *reinterpret_cast<u32x4 *>(mh + i * HB + 512 + lane * 16) = fl[i];
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            mx_f32x4 d{};
            typename W::Frag f;
            W::put(m, fw[i], lane);
            W::get(f, m, fw[i], lane);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const mx_bf16x8 wv = W::operand(f, j);
#pragma unroll
                for (int p = 0; p < 3; p++)
                    d = mfma16(wv, *reinterpret_cast<const mx_bf16x8 *>(mh + i * HB + p * 256 + X::piece_of(j, g) * 16), d);
            }
            if (on[i]) acc += d * p[i];
        }
    }
    *reinterpret_cast<mx_f32x4 *>(m + lane * 16) = acc;
    __syncthreads();
    if (wave || r >= a.T) return;
    mx_f32x4 s[4] = {};
#pragma unroll
    for (int i = 0; i < kFewWaves; i++) s[i & 3] += *reinterpret_cast<const mx_f32x4 *>(sm + i * LDS + lane * 16);
    acc = (s[0] + s[1]) + (s[2] + s[3]);
    *reinterpret_cast<ushort4 *>(a.y + (size_t)r * a.H + o0 + 4 * g) =
        make_ushort4(f2bf(acc[0]), f2bf(acc[1]), f2bf(acc[2]), f2bf(acc[3]));
}

// y = rnd(sum over the choices, in order, then the shared expert): bytes, 4.6 us for 64
// tokens, 7 for 325 (27 MB)
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

// the launch of an expert kernel: nsh row parts of the shared expert per `group`
// tokens, nper of every slot
struct Grid {
    int nsh, nper;
    unsigned n;
};
Grid grid_of(const MoeArgs &a, size_t slots, size_t nper, size_t nsh) {
    if (!a.Is) nsh = 0;
    return {(int)nsh, (int)nper, (unsigned)(nsh * cdiv(a.T, a.group) + slots * nper)};
}

template <class W>
int up_run(const MoeArgs &a, size_t slots) {
    const Grid g = grid_of(a, slots, a.I / 16, a.Is / 16);
    APUS_TIMED("k_moe_up", k_moe_up<W><<<g.n, 64 * kMoeWaves, 0, stream()>>>(a, g.nsh, g.nper));
    return launch_check("k_moe_up");
}
template <class W>
int down_run(const MoeArgs &a, size_t slots) {
    const Grid g = grid_of(a, slots, cdiv(a.H, down_rows(a.I)), cdiv(a.H, down_rows(a.Is)));
    APUS_TIMED("k_moe_down", k_moe_down<W><<<g.n, 64 * kMoeWaves, 0, stream()>>>(a, g.nsh, g.nper));
    return launch_check("k_moe_down");
}
template <class W, int NT>
int up_stream_run(const MoeArgs &a, size_t slots) {
    const int rows = 16 * kStreamWaves;
    const Grid g = grid_of(a, slots, cdiv(a.I, rows), cdiv(a.Is, rows));
    const unsigned threads = 64 * kStreamWaves;
    // (strips: rows of scales in whole, aligned words)
    const bool strips = W::mx && a.H % 128 == 0 && ((uintptr_t)a.s_gu | (uintptr_t)a.s_sgu) % 4 == 0;
    APUS_TIMED("k_moe_up_stream",
               if (strips) k_moe_up_stream<W, NT, W::mx><<<g.n, threads, 0, stream()>>>(a, g.nsh, g.nper);
               else k_moe_up_stream<W, NT, false><<<g.n, threads, 0, stream()>>>(a, g.nsh, g.nper));
    return launch_check("k_moe_up_stream");
}
template <class W, int NT>
int down_stream_run(const MoeArgs &a, size_t slots) {
    // blocks of a wavefront, so that the launch keeps about 8192 wavefronts:
    // more share a workgroup's copy of h
    constexpr int WAVES = kDownWaves<W, NT>;
    const size_t blocks = cdiv(a.H, 16 * kDownTiles);
    const bool many = std::max(a.I, a.Is) > kDownChunk * 128;
    const int P = many ? 1 : (int)std::max<size_t>(1, std::min<size_t>(4, slots * blocks / 8192));
    const size_t nper = cdiv(blocks, WAVES * P);
    const Grid g = grid_of(a, slots, nper, nper);
    APUS_TIMED("k_moe_down_stream",
               if (many) k_moe_down_stream<W, NT, true><<<g.n, 64 * WAVES, 0, stream()>>>(a, g.nsh, g.nper, P);
               else k_moe_down_stream<W, NT, false><<<g.n, 64 * WAVES, 0, stream()>>>(a, g.nsh, g.nper, P));
    return launch_check("k_moe_down_stream");
}

// The streaming forms from 1024 wavefronts on, 4 a CU (the layer, us split | streamed;
// up, MXFP4: 5 tokens 38 | 40, 16 tokens 58 | 54, 64 tokens 100 | 90, 325 tokens 181 | 153;
// down: 5 tokens 48 | 39, 64 tokens 149 | 90; bf16 72 | 67, 266 | 231). bf16 weights' up
// product is 4 times the bytes a step, which the split form keeps on their way as well with
// few rows a slot (16 tokens 130 | 130, 64 tokens 239 | 231, 325 tokens 393 | 345).
// Inner sizes of several chunks too (down, 128 experts of 768, 8 a token, MXFP4: 16 tokens
// 76 | 59, 64 tokens 116 | 85; bf16 163 | 153, 234 | 218), but the split form where a
// wavefront's walk is long and the choices are few (MXFP4: 60 experts of 1408, a shared one
// of 5632, 4 tokens 40 | 59; 8 experts of 14336, 2 a token, 64 tokens 302 | 342, 128 tokens
// 417 | 397; bf16, 16 tokens 507 | 557, 64 tokens 664 | 631).
// k_moe_down_few for one token (us without | with it: MXFP4 24 | 19, bf16 33 | 27; 128 experts
// of 768, 8 a token, 23 | 23, 34 | 34; 60 of 1408, 4 a token, and a shared one of 5632, 27 | 27,
// 47 | 43; 8 of 14336, 69 | 64, 154 | 140), for two whose work a few rounds of its loads cover
// (MXFP4 26 | 25, the other layers 28 | 29, 31 | 37, 91 | 107; bf16 42 | 38, 50 | 47, 58 | 60,
// 240 | 248), and for up to 16 whose work one round does (12 tokens, 16 experts of 128, 2 a
// token 18 | 16).
template <class W>
int experts_run(const MoeArgs &a) {
    const size_t slots = a.nslots;
    const bool one = a.group == 16;
    const bool ups = slots * a.I / 16 >= 1024 && (W::mx || a.T * a.k >= a.E);
    if (int r = !ups ? up_run<W>(a, slots) : one ? up_stream_run<W, 1>(a, slots) : up_stream_run<W, 2>(a, slots))
        return r;
    const int units = a.T * (a.k * cdiv(a.I, 128) + cdiv(a.Is, 128));
    if (a.T == 1 || (a.T <= 16 && units <= kFewWaves * kFewUnits * (a.T > 2 ? 1 : W::mx ? 2 : 3))) {
        APUS_TIMED("k_moe_down_few", k_moe_down_few<W><<<(unsigned)a.H / 16, 64 * kFewWaves, 0, stream()>>>(a));
        return launch_check("k_moe_down_few");
    }
    const int inner = std::max(a.I, a.Is);
    const bool downs = slots * a.H / 32 >= 1024 && (inner <= 2048 || a.T * a.k >= (W::mx ? 32 : 16) * a.E);
    if (int r = !downs ? down_run<W>(a, slots) : one ? down_stream_run<W, 1>(a, slots) : down_stream_run<W, 2>(a, slots))
        return r;
    APUS_TIMED("k_moe_combine",
               k_moe_combine<<<cdiv((size_t)a.T * (a.H / 4), 256), 256, 0, stream()>>>(a));
    return launch_check("k_moe_combine");
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

// y of T tokens shares bytes with a weight
bool over_weights(const ApusHipMoeLayer *L, size_t T, const uint16_t *y) {
    const size_t H = L->hidden, down = L->experts * H * L->inter, sdown = H * L->shared_inter;    // elements
    auto over = [&](const void *p, size_t bytes) { return bytes && block_overlaps(p, bytes, y, T * H * 2, T * H * 2, 1); };
    auto weight = [&](const void *p, const uint8_t *s, size_t n) {
        return over(p, L->mxfp4 ? n / 2 : n * 2) || (L->mxfp4 && over(s, n / kMxBlock));
    };
    return over(L->w_router, L->experts * H * 2) || weight(L->w_gate_up, L->s_gate_up, 2 * down) ||
           weight(L->w_down, L->s_down, down) || weight(L->w_shared_gate_up, L->s_shared_gate_up, 2 * sdown) ||
           weight(L->w_shared_down, L->s_shared_down, sdown) ||
           (sdown && L->w_shared_gate && over(L->w_shared_gate, H * 2));
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
    const size_t hs = max_tokens * (L->topk * L->inter + L->shared_inter) * 4;   // (offsets are 32 bits)
    if (hs > 0x7fff0000u || max_tokens * L->hidden * 2 > 0x7fff0000u)
        return set_error(kErrUnsupported, "mixture-of-experts intermediates of up to 2 GiB");
    if (int r = mx_ready()) return r;
    auto *w = new (std::nothrow) ApusHipMoeWork{max_tokens, L->hidden, L->inter, L->experts, L->topk,
                                                L->shared_inter, current_device()};
    if (!w) return set_error(kErrHip, "out of host memory");
    const size_t T = max_tokens, k = L->topk;
    size_t n = 0;
    auto take = [&](size_t bytes) {
        const size_t at = n;
        n += (bytes + 255) / 256 * 256;
        return at;
    };
    const size_t logits = take(T * (L->experts + 1) * 4), ids = take(T * k * 4),
                 wts = take(T * (k + 1) * 4), h = take(hs), hl = take(hs / 2),
                 part = take(T * (k + 1) * L->hidden * 4), done = take(((T + 15) / 16 + 1) * 4),
                 slots = take(moe_slots(T, k, L->experts, 16) * 16), list = take(T * k * 2);
    if (hipMalloc((void **)&w->base, n) != hipSuccess) {
        delete w;
        (void)hipGetLastError();           // (not for the next launch to report)
        return set_error(kErrHip, "hipMalloc of %zu bytes failed", n);
    }
    // (the counters are clear before any stream's first call)
    if (hipMemset(w->base + done, 0, ((T + 15) / 16 + 1) * 4) != hipSuccess ||
        hipStreamSynchronize(nullptr) != hipSuccess) {
        (void)hipFree(w->base);
        delete w;
        return set_error(kErrHip, "clearing the workspace failed");
    }
    w->done = (uint32_t *)(w->base + done);
    w->slots = (int4 *)(w->base + slots);
    w->list = (uint16_t *)(w->base + list);
    w->logits = (float *)(w->base + logits);
    w->ids = (int32_t *)(w->base + ids);
    w->wts = (float *)(w->base + wts);
    w->h = (uint16_t *)(w->base + h);
    w->hl = (uint16_t *)(w->base + hl);
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
        if (over_weights(L, T, y)) return set_error(kErrArgument, "the output overlaps the weights");
    }
    if (int r = mx_ready()) return r;
    if (w->device != current_device())
        return set_error(kErrArgument, "the workspace is on device %d, the library on %d", w->device, current_device());
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
    a.done = w->done;
    a.slots = w->slots;
    a.list = w->list;
    a.h = w->h;
    a.hl = w->hl;
    a.T = (int)T;
    a.H = (int)L->hidden;
    a.I = (int)L->inter;
    a.E = (int)L->experts;
    a.k = (int)L->topk;
    a.Is = (int)L->shared_inter;
    a.norm = L->norm_topk;
    a.group = slot_rows(T * L->topk, L->experts, L->inter, L->mxfp4 != 0);
    a.apart = choices_apart(T, T * L->topk, L->experts);
    a.nslots = (int)(a.apart ? T * L->topk : moe_slots(T, L->topk, L->experts, a.group));
    const int tiles = router_tiles(a);
    const bool small = tiles <= kSmallTiles && tiles * a.H <= kSmallElements;
    const dim3 rg(small ? 1 : tiles, cdiv(T, 16));
    APUS_TIMED("k_moe_router",
               if (small) k_moe_router<1, kSmallTiles><<<rg, 64 * kRouterWaves, 0, stream()>>>(a);
               else if (a.E <= 256) k_moe_router<4, 1><<<rg, 64 * kRouterWaves, 0, stream()>>>(a);
               else k_moe_router<16, 1><<<rg, 64 * kRouterWaves, 0, stream()>>>(a));
    APUS_LAUNCHED("k_moe_router");
    return L->mxfp4 ? experts_run<WMx>(a) : experts_run<WBf16>(a);
}

}  // extern "C"

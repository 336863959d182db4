// kv8_plan.h -- how a call on the 8-bit KV cache is dealt to launches and, for
// prefill, cut into tiles and parts. Host code, with the structures that go to the
// kernels: it is checked against what the kernels index on the CPU.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <functional>

#include "apus_rt.h"

namespace apus {

constexpr int kKv8Keys = 32;                 // positions of a block

// The sequences of one launch, by value (a captured call keeps them; longer
// batches take several launches). Few sequences: the short form, whose copy at
// launch is shorter. Entry i: the blocks (in the kernel's count) and tokens
// before sequence i, its cached positions and its row; entry n has the totals,
// entries past it none that is ever found.
constexpr int kKv8Seqs = 208, kKv8FewSeqs = 8;     // (a kernel's arguments within 4 KiB)
struct Kv8Seq {
    int32_t off, cu, pos0, row;
};
template <int N> struct alignas(16) Kv8SeqsN {
    Kv8Seq e[N + 1];
    int32_t n;
};

// Calls f(seqs) for each launch's share of a batch; count(s) is the number of
// blocks of sequence s. f may reorder its copy of the entries, and returns a status.
template <class Count, class F>
int kv8_launches(size_t B, const int32_t *rows, const int32_t *cu, const int32_t *pos0, Count count, F f) {
    for (size_t s0 = 0; s0 < B; s0 += kKv8Seqs) {
        const size_t n = B - s0 < (size_t)kKv8Seqs ? B - s0 : (size_t)kKv8Seqs;
        auto fill = [&](auto &q) {
            constexpr size_t N = sizeof(q.e) / sizeof(q.e[0]) - 1;
            q.n = (int32_t)n;
            int32_t off = 0;
            for (size_t i = 0; i < n; i++) {
                const size_t s = s0 + i;
                q.e[i] = Kv8Seq{off, cu[s], pos0[s], rows ? rows[s] : (int32_t)s};
                off += count(s);
            }
            q.e[n] = Kv8Seq{off, cu[s0 + n], 0, 0};
            for (size_t i = n + 1; i <= N; i++) q.e[i] = Kv8Seq{0x7fffffff, 0x7fffffff, 0, 0};
            return f(q);
        };
        int r;
        if (n <= (size_t)kKv8FewSeqs) {
            Kv8SeqsN<kKv8FewSeqs> q;
            r = fill(q);
        } else {
            Kv8SeqsN<kKv8Seqs> q;
            r = fill(q);
        }
        if (r) return r;
    }
    return kOk;
}

// ---- prefill
// Of each sequence of a launch: the tokens that its last tile lacks of being full
// (the sequences are not in the batch's order, so the entries' cu do not tell),
// and the parts that each tile's keys are cut into.
template <int N> struct Kv8Cut {
    uint8_t lack[N], parts[N];
};
// How a call is cut: tokens of a tile, and blocks of a part (0: tiles are whole).
struct Kv8Plan {
    int tok;
    int32_t len;
};
constexpr int kKv8MostParts = 64;
// (one at least: a sequence without tokens may end at 0, and has no tile to cut)
inline int kv8_parts(const Kv8Plan &p, int32_t end) {
    const int32_t blocks = (end + kKv8Keys - 1) / kKv8Keys;
    return p.len ? std::clamp((blocks + p.len - 1) / p.len, (int32_t)1, (int32_t)kKv8MostParts) : 1;
}

// Puts a launch's sequences in the order of their ends: its tiles start with the
// last, so the longest go first (6 ragged prompts: 105 us in the batch's order,
// 93 so), and those with several parts are the last entries.
template <int N> Kv8Cut<N> kv8_by_length(Kv8SeqsN<N> &q, const Kv8Plan &p) {
    struct {
        Kv8Seq e;
        int32_t n;
    } s[N];
    Kv8Cut<N> cut = {};
    for (int i = 0; i < q.n; i++) s[i] = {q.e[i], q.e[i + 1].cu - q.e[i].cu};
    std::sort(s, s + q.n, [](const auto &a, const auto &b) { return a.e.pos0 + a.n < b.e.pos0 + b.n; });
    int32_t off = 0;
    for (int i = 0; i < q.n; i++) {
        const int32_t tiles = (s[i].n + p.tok - 1) / p.tok, parts = kv8_parts(p, s[i].e.pos0 + s[i].n);
        q.e[i] = s[i].e;
        q.e[i].off = off;
        cut.lack[i] = (uint8_t)(tiles * p.tok - s[i].n);
        cut.parts[i] = (uint8_t)parts;
        off += tiles * parts;
    }
    q.e[q.n].off = off;
    return cut;
}

// The split sequences of such a launch, in tiles, for the kernel that joins their
// parts: off counts tiles, pos0 is the number of parts and row the first slot. A
// workgroup's slot is its item less split0.
template <int N> struct Kv8Joins {
    Kv8SeqsN<N> sq;
    Kv8Cut<N> cut;
    int32_t tiles, most;                     // most: parts of a tile
};
// the first sequence of several parts
template <int N> int kv8_first_split(const Kv8SeqsN<N> &q, const Kv8Cut<N> &cut) {
    int first = 0;
    while (first < q.n && cut.parts[first] == 1) first++;
    return first;
}
template <int N> Kv8Joins<N> kv8_joins(const Kv8SeqsN<N> &q, const Kv8Cut<N> &cut) {
    const int first = kv8_first_split(q, cut);
    const int32_t split0 = q.e[first].off;
    Kv8Joins<N> j = {};
    j.sq.n = q.n - first;
    j.most = 1;
    for (int i = 0; i < j.sq.n; i++) {
        const Kv8Seq &e = q.e[first + i];
        const int32_t parts = cut.parts[first + i];
        j.sq.e[i] = Kv8Seq{j.tiles, e.cu, parts, e.off - split0};
        j.cut.lack[i] = cut.lack[first + i];
        j.tiles += (q.e[first + i + 1].off - e.off) / parts;
        j.most = std::max(j.most, parts);
    }
    for (int i = j.sq.n; i <= N; i++) j.sq.e[i] = Kv8Seq{i == j.sq.n ? j.tiles : 0x7fffffff, 0x7fffffff, 0, 0};
    return j;
}

// The plan of least time, by the time of the busiest CU from a tile's alone on the
// chip (us; 16 + 1.38 a block of keys with 32 tokens, 13.2 + 0.83 with 16), tiles
// dealt longest first: the longest, all of them over the CUs (a full chip's clock:
// 1.26 and 1.18 times), and where some more than CUs remain, two that share a CU.
// Parts cost a start and an end each, their outputs' way through memory and the
// launch that joins them. Measured (us; 32 tokens, 16, 16 in parts): one prompt of 256
// 28, 20; 1024 62, 41, 47; 4096 201, 159; 6000 313, 330; 8192 490; 512 tokens after 8000
// 389, 235, 88; 16 after 4080 193, 120, 20; 8 times 500 after 4000 256, 294, 263; 16
// times 128 after 2000 112, 84; 6 ragged prompts of up to 900 143, 92. It takes the host
// 0.6 us for up to 6 sequences, 2.7 for 64, 4.4 for 128 and 7.0 for 208, before the
// call's first launch.
inline Kv8Plan kv8_fa_plan(size_t B, const int32_t *cu, const int32_t *pos0, size_t nkv, size_t slots,
                           size_t cus) {
    int32_t end = 0;
    auto busiest = [&](const Kv8Plan &p, double base, double per, double full) {
        size_t items = 0, split = 0;
        double sum = 0.0, longest = 0.0;
        for (size_t s = 0; s < B; s++) {
            const int64_t n = cu[s + 1] - cu[s];
            if (!n) continue;
            const int parts = kv8_parts(p, pos0[s] + (int32_t)n);
            const size_t t = (size_t)((n + p.tok - 1) / p.tok) * nkv;
            items += t * (size_t)parts;
            if (parts > 1) split += t * (size_t)parts;
            longest = std::max(longest, base + per * (double)(pos0[s] + n) / kKv8Keys / parts);
            sum += (double)t * (base * parts + per * ((double)pos0[s] + (double)(n + p.tok) / 2) / kKv8Keys);
        }
        if (split > slots) return 1e30;
        sum /= (double)cus;
        const double load = 1.0 + 0.15 * std::min(1.0, sum / longest);
        double us = std::max(longest * load, sum * full);
        double t[1024];
        if (items > cus && items <= std::min<size_t>(2 * cus, 1024)) {
            double *e = t;
            for (size_t s = 0; s < B; s++) {
                const int64_t n = cu[s + 1] - cu[s];
                const int parts = n ? kv8_parts(p, pos0[s] + (int32_t)n) : 1;
                for (int64_t x = 0; x < n; x += p.tok, e += nkv * (size_t)parts)
                    std::fill_n(e, nkv * (size_t)parts,
                                base + per * (double)(pos0[s] + std::min<int64_t>(x + p.tok, n)) / kKv8Keys / parts);
            }
            std::nth_element(t, t + cus, e, std::greater<double>());
            us = std::max(us, 2.0 * t[cus] * load);
        }
        return us + (split ? 6.0 + 0.05 * (double)split : 0.0);
    };
    for (size_t s = 0; s < B; s++)
        if (cu[s + 1] > cu[s]) end = std::max(end, pos0[s] + cu[s + 1] - cu[s]);
    Kv8Plan best = {32, 0};
    double us = busiest(best, 16.0, 1.38, 1.26);
    for (const int k : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
        const int32_t len = k == 1 ? 0 : (end + kKv8Keys - 1) / kKv8Keys / k;
        if (k > 1 && (len < 2 || B > (size_t)kKv8Seqs)) break;
        const Kv8Plan p = {16, len};
        const double t = busiest(p, 13.2, 0.83, 1.18);
        if (t < us) {
            us = t;
            best = p;
        }
    }
    return best;
}

}  // namespace apus

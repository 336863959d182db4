// Host driver: how a prefill call on the 8-bit KV cache is cut (csrc/kv8_plan.h),
// against what its kernels index: every token's tile once, every block of keys of a
// tile in one part, a slot of its own for each part, inside the workspace, and the
// join's entries the parts' slots. Arguments: the seed and the number of batches.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <set>
#include <vector>

#include "kv8_plan.h"

using namespace apus;

static int bad = 0, split_plans = 0;
static std::vector<int32_t> g_n, g_p;
static void report(const char *what) {
    if (bad++ >= 10) return;
    printf("%s: new", what);
    for (int32_t x : g_n) printf(" %d", x);
    printf(" cached");
    for (int32_t x : g_p) printf(" %d", x);
    printf("\n");
    fflush(stdout);
}
#define CHECK(c)            \
    do {                    \
        if (!(c)) report(#c); \
    } while (0)

// the kernels' search: the last entry whose off is at most x
template <int N> static int find(const Kv8SeqsN<N> &q, int x) {
    int s = -1;
    for (int i = 0; i <= N; i++)
        if (q.e[i].off <= x) s = i;
    return s;
}

// one launch; cu, pos0: the batch's
template <int N>
static void launch(Kv8SeqsN<N> &q, const Kv8Plan &plan, size_t nkv, size_t slots) {
    const Kv8SeqsN<N> was = q;
    const Kv8Cut<N> cut = kv8_by_length(q, plan);
    const int items = q.e[q.n].off;
    for (int i = 0; i < q.n; i++) CHECK(cut.parts[i] >= 1 && cut.parts[i] <= kKv8MostParts);
    if (bad) return;
    const int split0 = q.e[kv8_first_split(q, cut)].off;
    std::set<std::pair<int, int>> done;                    // (first token of a tile, part)
    std::set<size_t> used;
    std::vector<std::pair<int, int>> slot_of(items, {-1, -1});
    for (int item = 0; item < items; item++) {
        const int s = find(q, item);
        CHECK(s >= 0 && s < q.n);
        const Kv8Seq &e = q.e[s];
        const int parts = cut.parts[s], tile = (item - e.off) / parts, pt = (item - e.off) % parts;
        const int n = (q.e[s + 1].off - e.off) / parts * plan.tok - cut.lack[s], f0 = tile * plan.tok;
        int at = 0;                                        // the sequence in the batch
        while (at < q.n && !(was.e[at].cu == e.cu && was.e[at + 1].cu > e.cu)) at++;
        CHECK(at < q.n && n == was.e[at + 1].cu - e.cu && e.pos0 == was.e[at].pos0 && e.row == was.e[at].row);
        CHECK(f0 < n && done.insert({e.cu + f0, pt}).second);
        const int end = e.pos0 + std::min(f0 + plan.tok, n), nbt = (end + kKv8Keys - 1) / kKv8Keys;
        const int b0 = nbt * pt / parts, b1 = nbt * (pt + 1) / parts;
        CHECK(b0 <= b1 && (pt || !b0) && (pt < parts - 1 || b1 == nbt));
        if (parts > 1) {
            CHECK(plan.tok == 16 && item >= split0 && (size_t)(item - split0 + 1) * nkv <= slots);
            slot_of[item] = {e.cu + f0, pt};
        }
    }
    int tiles = 0;
    for (int i = 0; i < q.n; i++) tiles += (was.e[i + 1].cu - was.e[i].cu + plan.tok - 1) / plan.tok;
    std::set<int> firsts;
    for (auto &d : done) firsts.insert(d.first);
    CHECK((int)firsts.size() == tiles);
    if (split0 == items) return;
    split_plans++;
    const Kv8Joins<N> j = kv8_joins(q, cut);
    int joined = 0;
    for (int g = 0; g < j.tiles; g++) {
        const int s = find(j.sq, g);
        CHECK(s >= 0 && s < j.sq.n);
        const Kv8Seq &e = j.sq.e[s];
        const int tile = g - e.off, n = (j.sq.e[s + 1].off - e.off) * 16 - j.cut.lack[s];
        CHECK(e.pos0 > 1 && e.pos0 <= j.most && tile * 16 < n);
        for (int pt = 0; pt < e.pos0; pt++, joined++) {
            const int item = split0 + e.row + tile * e.pos0 + pt;
            CHECK(item < items && slot_of[item] == std::make_pair(e.cu + tile * 16, pt));
        }
    }
    int parts = 0;
    for (auto &x : slot_of) parts += x.first >= 0;
    CHECK(joined == parts);
}

static void batch(const std::vector<int32_t> &n, const std::vector<int32_t> &p, size_t nkv, const Kv8Plan *forced = nullptr) {
    const size_t cus = 256, slots = 2 * cus;
    g_n = n;
    g_p = p;
    std::vector<int32_t> cu = {0};
    for (int32_t x : n) cu.push_back(cu.back() + x);
    if (!cu.back()) return;
    const Kv8Plan plan = forced ? *forced : kv8_fa_plan(n.size(), cu.data(), p.data(), nkv, slots, cus);
    CHECK((plan.tok == 16 || plan.tok == 32) && (plan.tok == 16 || !plan.len));
    kv8_launches(n.size(), nullptr, cu.data(), p.data(), [&](size_t s) { return (cu[s + 1] - cu[s] + plan.tok - 1) / plan.tok; },
                 [&](auto &q) {
        if (q.e[q.n].off) launch(q, plan, nkv, forced ? (size_t)1 << 40 : slots);
        return 0;
    });
}

int main(int, char **argv) {
    std::mt19937 rng(atoi(argv[1]));
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    // sequences without tokens, at 0 and behind a context, beside split and whole ones
    batch({0, 16}, {0, 4080}, 2);
    batch({0, 500}, {0, 700}, 2);
    batch({0, 20, 20}, {0, 5000, 40}, 2);
    batch({20, 0, 20, 0}, {5000, 0, 40, 30000}, 2);
    batch({0, 0, 7}, {0, 0, 9000}, 1);
    for (int i = atoi(argv[2]); i > 0 && !bad; i--) {
        const int B = pick(0, 9) ? pick(1, 12) : pick(1, 300), kind = pick(0, 3);
        std::vector<int32_t> n, p;
        for (int s = 0; s < B; s++) {
            n.push_back(pick(0, 2) ? pick(1, kind == 0 ? 2000 / B + 1 : 60) : 0);
            p.push_back(pick(0, 2) ? pick(0, kind == 1 ? 60000 : 3000) : 0);
        }
        batch(n, p, (size_t)pick(1, 4));
        const Kv8Plan cut = {16, pick(2, 40)};
        batch(n, p, (size_t)pick(1, 4), &cut);
    }
    if (!split_plans) report("no plan with parts");
    printf("%s\n", bad ? "failed" : "ok");
    return bad != 0;
}

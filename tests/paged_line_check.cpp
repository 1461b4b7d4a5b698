// Host check of the division of work of the attention over a paged cache
// (csrc/paged_line.cuh): for random geometries, every key block of every unit
// belongs to exactly one piece, segments stay inside the tensors, partial rows
// stay inside the workspace and never overlap, and the second kernel finds the
// partials where the first one leaves them.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "paged_line.cuh"

using namespace cuflash::detail;

#define CHECK(x)                                                              \
    do {                                                                      \
        if (!(x)) {                                                           \
            std::printf("%s fails (line %d, geometry %d)\n", #x, __LINE__, it); \
            std::exit(1);                                                     \
        }                                                                     \
    } while (0)

int main(int argc, char** argv) {
    const int rounds = argc > 1 ? std::atoi(argv[1]) : 1000;
    std::mt19937 gen(1);
    auto R = [&](int a, int b) { return static_cast<int>(a + gen() % static_cast<unsigned>(b - a + 1)); };
    int it = -1;
    for (int n = 0; n <= 40; ++n)  // the closed form against the sum itself
        for (int k = 0; k < 200; ++k) {
            const int m = R(1, 200), a = R(0, 300), b = R(0, 5000);
            int s = 0;
            for (int i = 0; i < n; ++i) s += (a * i + b) / m;
            CHECK(floor_sum(n, m, a, b) == s);
        }
    long long pieces = 0;
    for (it = 0; it < rounds; ++it) {
        PagedLine p{};
        p.prefix_mode = it & 1;
        p.hkv = R(1, 8);
        const int kind = R(0, 9);
        const int group = kind < 7 ? R(1, 9) : (kind == 8 ? R(100, 140) : R(120, 300));
        p.hq = p.hkv * group;
        p.B = R(0, 4) == 0 ? R(1, 700) : R(1, 20);
        p.page_shift = R(3, 8);
        p.causal = p.prefix_mode ? 0 : R(0, 1);
        const int cap = R(0, 3) == 0 ? 20000 : 700;
        p.max_pages = (cap >> p.page_shift) + 1;
        p.max_prefix_pages = p.max_pages;
        std::vector<int> lens(p.B), cu(p.B + 1, 0);
        const int most = p.B > 50 ? 5 : (R(0, 4) == 0 ? 1500 : 40);
        for (int b = 0; b < p.B; ++b) {
            lens[b] = R(0, 3) == 0 ? R(-2, 3) : R(0, cap);
            cu[b + 1] = cu[b] + (R(0, 3) == 0 ? 0 : R(0, most));
        }
        int plen = R(0, 3) == 0 ? R(0, 2) : R(0, cap);
        p.num_tokens = p.prefix_mode ? p.B : std::max(1, cu[p.B] + R(0, 3));
        p.seq_lens = lens.data();
        p.cu_seqlens = cu.data();
        p.prefix_len = &plen;
        set_tiles(p, R(0, 2) ? 16 : 0);
        CHECK(p.tpt >= 1 && p.tpt * p.gt <= kTileRows && p.gt * p.chunks >= group &&
              p.gt * (p.chunks - 1) < group);
        const int grid = R(0, 2) ? 148 : R(1, 200);
        long long rows, records;
        CHECK(set_parts(p, grid, rows, records));
        int per;
        std::vector<int> starts(static_cast<size_t>(p.B) * p.hkv * p.chunks, -1);
        std::vector<Split> split(grid);
        for (auto& s : split) s.last = -1;
        p.per = &per;
        if (p.prefix_mode)
            p.unit_start = starts.data();
        else
            p.split = split.data();
        const int c_lo = p.prefix_mode ? -1 : 0;
        const int heads = p.hkv * p.chunks;
        std::vector<int> base;
        int total = 0;
        for (int c = c_lo; c < p.B; ++c) {
            const Ctx x = load_ctx(p, c);
            int sum = 0;
            if (x.head_cost)
                for (int q = 0; q < x.pairs; ++q) {
                    CHECK(pairs_cost(p, x, q) == sum);
                    sum += unit_blocks(p, x, q) * mode_weight(p, unit_mode(x, q));
                }
            CHECK(x.head_cost == sum);
            base.push_back(total);
            total += x.head_cost * heads;
        }
        per = std::max((total + grid - 1) / grid, p.min_per);
        using Key = std::tuple<int, int, int>;  // context, first head, first token
        std::map<Key, std::vector<std::pair<int, Seg>>> units;
        std::set<int> taken;
        for (int i = 0; i < grid; ++i) {
            const int x0 = i * per, x1 = std::min(x0 + per, total);
            if (x0 >= x1) continue;
            int c = c_lo;
            while (c + 1 < p.B && base[c + 1 - c_lo] <= x0) ++c;
            while (load_ctx(p, c).head_cost == 0) --c;
            Walk w;
            walk_start(p, w, load_ctx(p, c), c, base[c - c_lo], x0, x1, per, i);
            Seg s = {};
            int n = 0;
            while (walk_next(p, w, s)) {
                ++n;
                ++pieces;
                CHECK(s.n_blk > 0 && s.blk0 >= 0);
                CHECK(s.tok0 >= 0 && s.tok0 < s.tok_end && s.tok_end <= p.num_tokens);
                CHECK(s.nh > 0 && s.head0 + s.nh <= p.hq && s.hk == s.head0 / group &&
                      (s.head0 + s.nh - 1) / group == s.hk);
                if (s.mode == kTwoTiles) CHECK(s.tok0 + p.tpt < s.tok_end);
                if (s.mode == kOneTile) CHECK(s.tok0 + p.tpt >= s.tok_end);
                if (s.mode == kFew) CHECK((s.tok_end - s.tok0) * p.gt <= p.few_rows);
                if (s.part_row >= 0) {
                    const bool own = p.prefix_mode && s.ctx >= 0;
                    const int span = own ? p.gt : 2 * kTileRows;
                    CHECK(s.part_rows == (own ? p.gt : kTileRows));
                    CHECK(s.part_row + span <= rows);
                    for (int q = 0; q < span; q += own ? 1 : kTileRows) CHECK(taken.insert(s.part_row + q).second);
                }
                units[Key(s.ctx, s.head0, s.tok0)].push_back({i, s});
            }
            CHECK(n > 0 || x1 - x0 < p.min_per);
        }
        size_t count = 0;
        for (int c = c_lo; c < p.B; ++c) {
            const Ctx x = load_ctx(p, c);
            if (!x.head_cost) continue;
            for (int hk = 0; hk < p.hkv; ++hk)
                for (int ch = 0; ch < p.chunks; ++ch)
                    for (int q = 0; q < x.pairs; ++q) {
                        ++count;
                        const auto u = units.find(Key(c, hk * group + ch * p.gt, x.tok + q * 2 * p.tpt));
                        CHECK(u != units.end());
                        const auto& v = u->second;
                        int at = 0;
                        for (size_t k = 0; k < v.size(); ++k) {
                            CHECK(v[k].second.blk0 == at && (k == 0 || v[k].first == v[k - 1].first + 1));
                            at += v[k].second.n_blk;
                        }
                        CHECK(at == unit_blocks(p, x, q));
                        const int last = std::min((q + 1) * 2 * p.tpt, x.ntok) - 1;  // token of the context
                        CHECK(at * kBlockKeys >= (p.causal ? std::min(x.len, x.len - x.ntok + last + 1) : x.len));
                        if (p.prefix_mode) continue;
                        if (v.size() == 1) {
                            CHECK(v[0].second.part_row == -1);
                            continue;
                        }
                        const Split& s = split[v[0].first];
                        CHECK(s.last == v.back().first && s.tok0 == v[0].second.tok0 &&
                              s.head0 == v[0].second.head0 && s.mode == v[0].second.mode);
                        for (size_t k = 0; k < v.size(); ++k)
                            CHECK(v[k].second.part_row ==
                                  (2 * (v[0].first + static_cast<int>(k)) + (k == 0 ? 1 : 0)) * 2 * kTileRows);
                    }
        }
        CHECK(count == units.size());
        if (p.prefix_mode) {
            const Ctx pre = load_ctx(p, -1);
            for (int t = 0; t < 40; ++t) {
                const int b = R(0, p.B - 1), h = R(0, p.hq - 1);
                const Ctx own = load_ctx(p, b);
                const int hk = h / group, ch = (h % group) / p.gt, hr = (h % group) % p.gt;
                const PrefixParts q = prefix_parts(p, per, pre, own, b, hk * p.chunks + ch, hr);
                const int tile = b / p.tpt;
                if (pre.len > 0) {
                    const auto& v = units[Key(-1, hk * group + ch * p.gt, (tile / 2) * 2 * p.tpt)];
                    CHECK(static_cast<int>(v.size()) == q.n1 && q.r1 == (b % p.tpt) * p.gt + hr);
                    for (int k = 0; k < q.n1; ++k) {
                        CHECK(v[k].second.mode == kTwoTiles || tile % 2 == 0);
                        CHECK(q.row1 + k * 2 * kTileRows == v[k].second.part_row + (tile % 2) * kTileRows);
                    }
                } else {
                    CHECK(q.n1 == 0);
                }
                if (own.len > 0) {
                    const auto& v = units[Key(b, hk * group + ch * p.gt, b)];
                    CHECK(static_cast<int>(v.size()) == q.n2 && q.r2 == hr);
                    for (int k = 0; k < q.n2; ++k) CHECK(q.row2 + k * p.gt == v[k].second.part_row);
                } else {
                    CHECK(q.n2 == 0);
                }
            }
        } else {
            for (int i = 0; i < grid; ++i) {
                if (split[i].last < 0) continue;
                bool found = false;
                for (const auto& u : units) found = found || (u.second.size() > 1 && u.second[0].first == i);
                CHECK(found);
            }
        }
    }
    std::printf("ok: %d geometries, %lld pieces\n", rounds, pieces);
}

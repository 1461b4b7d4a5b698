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
        const int few[4] = {0, 4, 8, 16};
        set_tiles(p, few[R(0, 3)]);
        CHECK(p.tpt >= 1 && p.tpt * p.gt <= kTileRows && p.gt * p.chunks >= group &&
              p.gt * (p.chunks - 1) < group);
        const int grid = R(0, 2) ? 148 : R(1, 200);
        long long rows, records;
        CHECK(set_parts(p, grid, rows, records));
        long long per[2];
        std::vector<Span> span(static_cast<size_t>(p.B + p.prefix_pairs) * p.heads, Span{-1, -1});
        std::vector<Split> split(2 * grid);
        for (auto& s : split) s.last = -1;
        if (p.prefix_mode)
            p.span = span.data();
        else
            p.split = split.data();
        const int c_lo = p.prefix_mode ? -1 : 0;
        const int heads = p.heads;
        std::vector<long long> base;  // position of each context on its line
        long long total[2] = {0, 0};
        for (int c = c_lo; c < p.B; ++c) {
            const Ctx x = load_ctx(p, c);
            long long sum = 0;
            if (x.head_cost)
                for (int q = 0; q < x.pairs; ++q) {
                    CHECK(pairs_cost(p, x, q) == sum);
                    sum += unit_length(p, x, q);
                }
            CHECK(x.head_cost == sum);
            base.push_back(total[line_of(x)]);
            total[line_of(x)] += x.head_cost * heads;
        }
        auto next_ctx = [&](int c, int line, Ctx& out) {
            while (++c < p.B) {
                out = load_ctx(p, c);
                if (out.head_cost != 0 && line_of(out) == line) return c;
            }
            CHECK(!"a context behind the last");
            return c;
        };
        using Key = std::tuple<int, int, int>;  // context, first head, first token
        std::map<Key, std::vector<std::pair<int, Seg>>> units;
        std::set<int> taken;
        for (int li = 0; li < 2 * grid; ++li) {
            const int line = li / grid, i = li % grid;
            per[line] = piece_length(total[line], grid);
            CHECK(per[line] * grid >= total[line]);
            const long long x0 = i * per[line], x1 = std::min(x0 + per[line], total[line]);
            if (x0 >= x1) continue;
            int c = c_lo;
            while (true) {  // the context that holds x0
                const Ctx x = load_ctx(p, c);
                if (line_of(x) == line && x0 >= base[c - c_lo] && x0 < base[c - c_lo] + x.head_cost * heads) break;
                ++c;
                CHECK(c < p.B);
            }
            Walk w;
            walk_start(p, w, load_ctx(p, c), c, base[c - c_lo], x0, x1, per[line], line, i, true);
            Seg s = {};
            int n = 0;
            while (walk_next(p, w, s, next_ctx)) {
                ++n;
                CHECK((s.mode == kFew) == (line == kFewLine));
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
                    const bool few = !p.prefix_mode && s.mode == kFew;
                    const int span = own ? p.gt : (few ? kFewTile : 2 * kTileRows);
                    CHECK(s.part_rows == (own ? p.gt : (few ? kFewTile : kTileRows)));
                    CHECK(s.mode != kFew || (s.tok_end - s.tok0) * p.gt <= s.part_rows);
                    CHECK(s.part_row >= 0 && s.part_row + span <= rows);
                    for (int q = 0; q < span; ++q) CHECK(taken.insert(s.part_row + q).second);
                }
                units[Key(s.ctx, s.head0, s.tok0)].push_back({i, s});
            }
            CHECK(n > 0 || x1 - x0 < per[line] || x1 - x0 < 2 * (kBlockKeys + kUnitCost));
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
                        CHECK(at == (unit_keys(p, x, q) + kBlockKeys - 1) / kBlockKeys);
                        const int last = std::min((q + 1) * 2 * p.tpt, x.ntok) - 1;  // token of the context
                        CHECK(at * kBlockKeys >= (p.causal ? std::min(x.len, x.len - x.ntok + last + 1) : x.len));
                        if (p.prefix_mode) continue;
                        if (v.size() == 1) {
                            CHECK(v[0].second.part_row == -1);
                            continue;
                        }
                        const bool few = v[0].second.mode == kFew;
                        const Split& s = split[(few ? grid : 0) + v[0].first];
                        CHECK(s.last == v.back().first && s.tok0 == v[0].second.tok0 &&
                              s.head0 == v[0].second.head0 && s.mode == v[0].second.mode);
                        for (size_t k = 0; k < v.size(); ++k)
                            CHECK(v[k].second.part_row ==
                                  (few ? p.few_part_row : 0) +
                                      (2 * (v[0].first + static_cast<int>(k)) + (k == 0 ? 1 : 0)) *
                                          (few ? kFewTile : 2 * kTileRows));
                    }
        }
        CHECK(count == units.size());
        if (p.prefix_mode) {
            for (const auto& u : units) {
                const Seg& s0 = u.second[0].second;
                const int hc = s0.hk * p.chunks + (s0.head0 - s0.hk * group) / p.gt;
                const int pair = s0.ctx < 0 ? s0.tok0 / (2 * p.tpt) : 0;
                const int n = s0.ctx < 0 ? hc * p.prefix_pairs + pair : heads * p.prefix_pairs + s0.ctx * heads + hc;
                const Span sp = span[n];
                CHECK(sp.first == u.second[0].first && sp.last == u.second.back().first);
                // the second kernel's addresses
                for (size_t k = 0; k < u.second.size(); ++k) {
                    const int piece = sp.first + static_cast<int>(k);
                    CHECK(u.second[k].second.part_row ==
                          (s0.ctx < 0 ? (n + piece) * 2 * kTileRows
                                      : p.own_part_row + (n - heads * p.prefix_pairs + piece) * p.gt));
                }
            }
        } else {
            for (int i = 0; i < 2 * grid; ++i) {
                if (split[i].last < 0) continue;
                bool found = false;
                for (const auto& u : units)
                    found = found || (u.second.size() > 1 && u.second[0].first == i % grid &&
                                      (u.second[0].second.mode == kFew) == (i >= grid));
                CHECK(found);
            }
        }
    }
    std::printf("ok: %d geometries, %lld pieces\n", rounds, pieces);
}

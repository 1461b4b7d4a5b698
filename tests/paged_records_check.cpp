// Host check of who writes the records of the ragged attention's split units
// (csrc/paged_line.cuh).  CTAs are ordered by nothing: one may reset its records
// after another has walked its pieces.  So each CTA here resets and walks on its
// own, in shuffled orders, and the records have to be the same as with all of them
// reset before any walk; and a CTA's reset has to touch exactly the records of the
// pieces it takes.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <numeric>
#include <random>
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
    const int rounds = argc > 1 ? std::atoi(argv[1]) : 300;
    std::mt19937 gen(5);
    auto R = [&](int a, int b) { return static_cast<int>(a + gen() % static_cast<unsigned>(b - a + 1)); };
    int it = 0;
    long long seen[2] = {0, 0};  // records of each line
    for (; it < rounds; ++it) {
        PagedLine p{};
        p.hkv = R(1, 8);
        p.hq = p.hkv * R(1, 9);
        p.B = R(1, 40);
        p.page_shift = R(3, 8);
        p.causal = R(0, 1);
        const int cap = R(0, 2) == 0 ? 60000 : 3000;
        p.max_pages = (cap >> p.page_shift) + 1;
        std::vector<int> lens(p.B), cu(p.B + 1, 0);
        for (int b = 0; b < p.B; ++b) {
            lens[b] = R(0, 4) == 0 ? R(0, 3) : R(0, cap);
            cu[b + 1] = cu[b] + (R(0, 1) ? 1 : R(0, 300));  // single tokens between chunks
        }
        p.num_tokens = std::max(1, cu[p.B]);
        p.seq_lens = lens.data();
        p.cu_seqlens = cu.data();
        const int few[4] = {0, 4, 8, 16};
        set_tiles(p, few[R(0, 3)]);
        const int grid = R(0, 2) ? 148 : R(1, 200);
        long long rows, bytes;
        CHECK(set_parts(p, grid, rows, bytes));
        CHECK(bytes == static_cast<long long>(2 * grid * sizeof(Split)));

        long long total[2] = {0, 0};
        std::vector<long long> base;
        for (int c = 0; c < p.B; ++c) {
            const Ctx x = load_ctx(p, c);
            base.push_back(total[line_of(x)]);
            total[line_of(x)] += x.head_cost * p.heads;
        }
        auto next_ctx = [&](int c, int line, Ctx& out) {
            while (++c < p.B) {
                out = load_ctx(p, c);
                if (out.head_cost != 0 && line_of(out) == line) return c;
            }
            return p.B - 1;
        };
        auto walk = [&](int cta) {
            for (int line = 0; line < 2; ++line) {
                const int piece = piece_index(p, line, cta);
                const long long per = piece_length(total[line], grid);
                const long long x0 = std::min(piece * per, total[line]), x1 = std::min(x0 + per, total[line]);
                if (x0 >= x1) continue;
                int c = 0;
                for (;; ++c) {
                    CHECK(c < p.B);
                    const Ctx x = load_ctx(p, c);
                    if (line_of(x) == line && x0 >= base[c] && x0 < base[c] + x.head_cost * p.heads) break;
                }
                Walk w;
                walk_start(p, w, load_ctx(p, c), c, base[c], x0, x1, per, line, piece, true);
                Seg s = {};
                while (walk_next(p, w, s, next_ctx)) {
                }
            }
        };

        Split fill;
        std::memset(&fill, 0x5a, sizeof(fill));  // what an earlier call left
        std::vector<Split> want(2 * grid, fill), got;
        p.split = want.data();
        for (int cta = 0; cta < grid; ++cta) reset_records(p, cta);
        for (const Split& s : want) CHECK(s.last == -1);  // every record is reset
        for (int cta = 0; cta < grid; ++cta) walk(cta);
        for (int i = 0; i < 2 * grid; ++i) seen[i / grid] += want[i].last >= 0;

        std::vector<int> order(grid);
        std::iota(order.begin(), order.end(), 0);
        for (int turn = 0; turn < 4; ++turn) {
            if (turn == 1) std::reverse(order.begin(), order.end());
            if (turn > 1) std::shuffle(order.begin(), order.end(), gen);
            got.assign(2 * grid, fill);
            p.split = got.data();
            for (int cta : order) {
                reset_records(p, cta);
                walk(cta);
            }
            CHECK(std::memcmp(got.data(), want.data(), got.size() * sizeof(Split)) == 0);
        }
        for (int cta = 0; cta < grid; ++cta) {
            got.assign(2 * grid, fill);
            p.split = got.data();
            reset_records(p, cta);
            for (int i = 0; i < 2 * grid; ++i)
                CHECK((got[i].last == -1) == (i == piece_index(p, i / grid, cta) + (i / grid) * grid));
        }
    }
    CHECK(seen[kTiles] > rounds && seen[kFewLine] > rounds);  // both kinds were split
    std::printf("ok: %d geometries, %lld and %lld records\n", rounds, seen[0], seen[1]);
}

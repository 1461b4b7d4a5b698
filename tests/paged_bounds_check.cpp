// Host check of the paged-cache kernels' bounds (csrc/paged.cuh, paged_line.cuh):
// no lengths or offsets that device memory may hold lead behind a table, and no
// length of a segment makes its waits run out.
#include <climits>
#include <cstdio>
#include <cstdlib>

#include "paged.cuh"
#include "paged_line.cuh"

using namespace cuflash::detail;

#define CHECK(x)                                        \
    do {                                                \
        if (!(x)) {                                     \
            std::printf("%s fails (%d)\n", #x, __LINE__); \
            std::exit(1);                               \
        }                                               \
    } while (0)

int main() {
    const int lens[] = {0, 1, 2, 127, 4096, INT_MAX};
    // offsets that do not ascend put a token behind its sequence's end
    const int ends[] = {INT_MIN, -70000, -1, 0, 1, 2, 127, 70000, INT_MAX};
    for (int len : lens)
        for (int end : ends)
            for (int causal = 0; causal < 2; ++causal) {
                const int n = visible_keys(len, end, causal);
                CHECK(n <= len);
                if (!causal) CHECK(n == len);
                if (causal && end >= 1) CHECK(n == len - (end - 1));
            }
    for (int most : lens)
        for (int n : ends) {
            const int c = clamp_len(n, most);
            CHECK(c >= 0 && c <= most && (n < 0 || n > most || c == n));
        }
    // Up to the blocks of the longest table (2^31 - 1 rows): a block takes up to 4 us
    // (two row tiles, 32 boxes of 8 rows), and a wait for a segment is bounded by an
    // hour all the same.
    for (int n_blk : {1, 2, 1000, 100000, 1 << 20, 1 << 24})
        for (unsigned base : {50u, 3906250u}) {
            const double us = 1.024 * wait_ticks(base, n_blk);
            CHECK(us >= 4.0 * n_blk && us <= 3600e6);
            CHECK(us >= base && (n_blk > 1000 || us <= 1.2 * base + 100e3));  // usual ones stay near the base
        }
    std::printf("ok\n");
}

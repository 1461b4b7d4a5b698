// Host check of the paged-cache kernels' bounds (csrc/paged.cuh): no lengths or
// offsets that device memory may hold lead behind a table.
#include <climits>
#include <cstdio>
#include <cstdlib>

#include "paged.cuh"

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
    std::printf("ok\n");
}

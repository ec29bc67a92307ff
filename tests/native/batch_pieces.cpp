// CPU walk of the pieces of keys that the groups of four waves of a tile of 128 queries take in turns
// (prompt_tile_impl), for test_batch_pieces.py, built so that an overflow of int ends it.  Prints "ok" or the first
// mistake.
//   pieces seed [mistake]  ranges of four waves, some or all of them without a key; a mistake: without g2b_span_*
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "g2_batch_plan.h"

int main(int argc, char **argv)
{
    if (argc < 2) return 2;
    std::mt19937 r(std::atoi(argv[1]));
    const bool mistake = argc > 2;
    for (int n = 0; n < 2000; ++n) {
        int low = INT_MAX, high = -INT_MAX;
        for (int w = 0; w < 4; ++w) {
            const int kind = n % 8 == 0 ? 0 : (int)(r() % 3), base = n % 5 ? 0 : (1 << 24) - 1000;
            const int a = base + (int)(r() % 500), b = a + 1 + (int)(r() % 500);
            low = std::min(low, kind ? a : INT_MAX);
            high = std::max(high, kind ? b : -INT_MAX);
        }
        const int k0 = mistake ? low : g2b_span_begin(low, high), k1 = mistake ? high : g2b_span_end(low, high);
        for (int KT = 1; KT <= 2; ++KT)
            for (int KW = 1; KW <= 2; ++KW) {
                std::vector<int> seen(std::max(0, low < high ? high - low : 0), 0);
                const int STEP = 32 * KT * KW;
                int turns[2] = {};
                for (int kw = 0; kw < KW; ++kw) {
                    int j0 = k0 + 32 * KT * kw;
                    for (int left = k1 - k0; KW == 1 ? j0 < k1 : left > 0; left -= STEP, j0 += STEP, ++turns[kw])
                        for (int j = j0; j < std::min(j0 + 32 * KT, k1); ++j) {
                            if (j < low || j >= high || seen[j - low]++) return std::printf("a key outside or twice: %d of %d .. %d\n", j, low, high), 0;
                        }
                }
                for (int c : seen)
                    if (c != 1) return std::printf("a key is in no piece: %d .. %d\n", low, high), 0;
                if (KW == 2 && turns[0] != turns[1]) return std::printf("barriers: %d and %d\n", turns[0], turns[1]), 0;
                if (low >= high && (turns[0] || turns[1])) return std::printf("%d turns over no keys\n", turns[0]), 0;
            }
    }
    std::puts("ok");
    return 0;
}

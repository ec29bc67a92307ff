// CPU walk of the index arithmetic of the operators for several texts at once
// (g2_batch_plan.h), for test_batch_addresses.py.  Prints "ok" or the first mistake.
//   cache S NKV max_seq [mistake]  the parts of a cache buffer
//   items NKV tiles                every piece of work is one work-group's
//   search n seed                  counts in ordered lists, an end in others
//   rows seed                      the keys of a row, whatever its starts hold
//   beams groups rows slices n_out the parts of the selection's workspace
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "g2_batch_plan.h"

static int bad(const char *what, long a, long b, long c)
{
    std::printf("%s: %ld %ld %ld\n", what, a, b, c);
    return 0;
}

static int cache(long S, int NKV, long max_seq, int mistake)
{
    const long tiles = g2b_tiles(max_seq);
    std::vector<unsigned char> seen(g2b_bytes(S, NKV, tiles), 0);
    for (long s = 0; s < S; ++s)
        for (int h = 0; h < NKV; ++h)
            for (long p = 0; p < tiles * G2B_TILE; ++p)
                for (int kv = 0; kv < 2; ++kv) {
                    const size_t t = g2b_tile_at(NKV, tiles, s, h, p / G2B_TILE);
                    const int i = (int)(mistake ? (p + 1) % G2B_TILE / 2 : p % G2B_TILE);
                    if (t % 16) return bad("a tile is not aligned", s, h, p);
                    for (unsigned b = 0; b < G2B_ROW; ++b) {
                        const size_t at = t + g2b_code_at(kv, i) + b;
                        if (at >= seen.size() || seen[at]++) return bad("codes outside or twice", s, h, p);
                    }
                    for (unsigned b = 0; b < 4; ++b) {
                        const size_t at = t + g2b_scale_at(kv, i) + b;
                        if (at >= seen.size() || seen[at]++) return bad("scales outside or twice", s, h, p);
                    }
                }
    for (unsigned char c : seen)
        if (c != 1) return bad("a byte is nobody's", 0, 0, 0);
    return 1;
}

static int items(int NKV, long tiles)
{
    std::vector<unsigned char> seen(NKV * tiles, 0);
    for (long b = 0; b < NKV * tiles; ++b) {
        int h;
        long t;
        g2b_prompt_item(b, NKV, tiles, &h, &t);
        if (h < 0 || h >= NKV || t < 0 || t >= tiles || seen[h * tiles + t]++) return bad("a piece outside or twice", b, h, t);
        if (h < NKV / 8 * 8 && h % 8 != b % 8) return bad("a head on another XCD", b, h, t);
        if (labs(tiles - 1 - t - b / NKV) * NKV > 256 + NKV) return bad("tiles in another order", b, h, t);
    }
    return 1;
}

// what the wave does: 64 probes, the number of those at or below the value
static int count(const std::vector<int> &list, int value, int *steps)
{
    int lo = 0, left = (int)list.size();
    for (*steps = 0;; ++*steps) {
        int c = 0;
        if (left < 0 || lo < 0 || lo + left > (int)list.size() || *steps > 10) return -1;
        for (int lane = 0; lane < 64; ++lane) {
            const int at = g2b_probe(left, lane);
            const size_t entry = (size_t)lo + (at < left ? at : 0);
            if (at < left) {
                if (entry >= list.size()) return -1;
                c += list[entry] <= value;
            }
        }
        if (g2b_narrow(&lo, &left, c)) return lo;
    }
}

static int search(int n, int seed)
{
    std::mt19937 r(seed);
    int steps;
    std::vector<int> list(n);
    for (int round = 0; round < 20; ++round) {
        int at = (int)(r() % 5) - 2;
        for (int i = 0; i < n; ++i) list[i] = at += (int)(r() % 4) * (int)(r() % 3);
        for (int v = -3; v < at + 3; v += 1 + at / 500) {
            long want = 0;
            for (int x : list) want += x <= v;
            if (count(list, v, &steps) != want) return bad("count", v, want, count(list, v, &steps));
        }
        for (int i = 0; i < n; ++i) list[i] = (int)(r() % 2 ? r() : r() % 100);
        for (int i = 0; i < 50; ++i) {
            const int c = count(list, (int)(r() % 2 ? r() : r() % 100), &steps);
            if (c < 0 || c > n) return bad("a list in no order", n, c, steps);
        }
    }
    return 1;
}

static int rows(int seed)
{
    std::mt19937 r(seed);
    auto any = [&]() {
        switch (r() % 6) {
        case 0: return (int)r();
        case 1: return INT_MAX;
        case 2: return INT_MIN;
        case 3: return -(int)(r() % 50);
        default: return (int)(r() % 60);
        }
    };
    for (int i = 0; i < 2000000; ++i) {
        const int q_rows = 1 + (int)(r() % 50), k_rows = (int)(r() % 50), row = (int)(r() % q_rows);
        const int q0 = any(), q1 = any(), k0 = any(), k1 = any();
        const g2b_row x = g2b_row_keys(row, 1, q0, q1, k0, k1, q_rows, k_rows);
        if (x.lo < 0 || x.lo > x.end || x.end > k_rows) return bad("keys outside", x.lo, x.end, k_rows);
        if (x.there != (row >= q0 && row < q1)) return bad("a row's sequence", row, q0, q1);
        if (q0 >= 0 && q0 <= row && q1 > row && q1 <= q_rows && k0 >= 0 && k1 >= k0 && k1 <= k_rows) {
            const int n = q1 - q0, m = k1 - k0, sees = row - q0 + m - n + 1;
            if (x.lo != k0 || x.end - x.lo != (sees > 0 ? sees : 0)) return bad("keys of a row", row, x.lo, x.end);
        }
        const g2b_row none = g2b_row_keys(row, 0, q0, q1, k0, k1, q_rows, k_rows);
        if (none.there || none.end != none.lo) return bad("a row of no sequence", row, 0, 0);
    }
    return 1;
}

static int beams(long groups, long n, int slices, int n_out)
{
    const size_t st = g2b_stats_at(groups), at = g2b_cands_at(groups, n, slices), all = g2b_beam_bytes(groups, n, slices, n_out);
    if (st % 8 || at % 8 || st < (size_t)groups * 4 || at < st + (size_t)n * slices * 8 || all != at + (size_t)n * slices * n_out * 8)
        return bad("parts", n, slices, n_out);
    return 1;
}

int main(int n, char **v)
{
    auto arg = [&](int i) { return i < n ? std::atol(v[i]) : 0; };
    int ok = 0;
    if (n > 1 && !std::strcmp(v[1], "cache")) ok = cache(arg(2), (int)arg(3), arg(4), (int)arg(5));
    else if (n > 1 && !std::strcmp(v[1], "items")) ok = items((int)arg(2), arg(3));
    else if (n > 1 && !std::strcmp(v[1], "search")) ok = search((int)arg(2), (int)arg(3));
    else if (n > 1 && !std::strcmp(v[1], "rows")) ok = rows((int)arg(2));
    else if (n > 1 && !std::strcmp(v[1], "beams")) ok = beams(arg(2), arg(3), (int)arg(4), (int)arg(5));
    if (ok) std::printf("ok\n");
    return ok ? 0 : 1;
}

// CPU walk of the low-bit operators' index arithmetic (g2_lowbit_plan.h), for
// test_lowbit_addresses.py.  Prints "ok" or the first mistake.
//   weights N K [mistake]        every lane's reads of every chunk
//   cache S NH max_seq           the parts of a cache buffer
//   append S NH T                the waves' work
//   attend blocks span splits waves len [mistake]   the blocks a head's waves take
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "g2_lowbit_plan.h"

static int bad(const char *what, long a, long b, long c)
{
    std::printf("%s: %ld %ld %ld\n", what, a, b, c);
    return 0;
}

static int weights(long N, long K, int mistake)
{
    const size_t bytes = g2l_code_bytes(N, K);
    const long steps = g2l_steps(K);
    std::vector<unsigned char> words(bytes / 4, 0);
    for (long t = 0; t < g2l_tiles(N); ++t)
        for (long c = 0; c < g2l_chunks(K); ++c) {
            const int r = g2l_chunk_steps(K, c);
            if (r < 1 || r > 4) return bad("steps of a chunk", t, c, r);
            for (int lane = 0; lane < 64; ++lane) {
                const size_t own = g2l_code_at(K, t, c, lane);
                // (the kernel: a chunk's base is 1024 bytes times c into its tile)
                const size_t at = g2l_code_at(K, t, 0, 0) + 1024 * (size_t)c + (mistake == 1 ? (size_t)lane * 4 * r : g2l_lane_at(K, c, lane));
                const int shift = mistake == 2 ? 0 : g2l_lane_shift(K, c, lane);
                if (at + 16 > bytes || at % 4) return bad("a lane reads outside the codes", t, c, lane);
                for (int j = 0; j < r; ++j) {
                    if (j + shift > 3 || at + 4 * (j + shift) != own + 4 * (size_t)j) return bad("a step's word is not where the lane has it", c, lane, j);
                    if (words[own / 4 + j]++) return bad("a word is two lanes'", c, lane, j);
                }
            }
        }
    for (size_t i = 0; i < words.size(); ++i)
        if (words[i] != 1) return bad("a word is nobody's", (long)i, steps, 0);
    for (int group = 32; group <= 128; group *= 2) {
        std::vector<unsigned char> s(g2l_scale_count(N, K, group), 0);
        for (long t = 0; t < g2l_tiles(N); ++t)
            for (long c = 0; c < g2l_chunks(K); ++c)
                for (int row = 0; row < 16; ++row)
                    for (int g = 0; g < 128 / group; ++g) {
                        const size_t i = g2l_scale_at(K, group, t, c, row, g);
                        if (i >= s.size() || s[i]++) return bad("a scale outside or twice", t, c, row);
                        // (the kernel: base of the tile, chunk and row strides of 32 * 128 / group and 2 * 128 / group bytes)
                        if (2 * i != 2 * g2l_scale_at(K, group, t, 0, 0, 0) + c * 32 * (128 / group) + row * 2 * (128 / group) + 2 * g)
                            return bad("a scale's address", t, c, row);
                    }
        for (unsigned char v : s)
            if (v != 1) return bad("a scale is nobody's", group, 0, 0);
    }
    return 1;
}

static int cache(long S, int NH, long max_seq)
{
    const long nb = g2l_blocks(max_seq);
    const size_t sc = g2l_kv_scales(S, NH, nb), la = g2l_kv_last(S, NH, nb), all = g2l_kv_bytes(S, NH, nb);
    if (nb * 16 < max_seq || (nb - 1) * 16 >= max_seq) return bad("blocks", nb, max_seq, 0);
    if (sc % 16 || la % 16 || la < sc + (size_t)S * NH * nb * 8) return bad("parts overlap or are not aligned", 0, 0, 0);
    std::vector<unsigned char> seen(S * NH * nb * 2, 0), ends(S * NH * 2, 0);
    for (long s = 0; s < S; ++s)
        for (int h = 0; h < NH; ++h)
            for (int kv = 0; kv < 2; ++kv) {
                for (long b = 0; b < nb; ++b) {
                    const size_t c = g2l_kv_code_at(NH, nb, s, h, b, kv), i = g2l_kv_scale_at(NH, nb, s, h, b, kv);
                    if (c + 1024 > sc || c != 1024 * i || i >= seen.size() || seen[i]++) return bad("a block's codes or scale", s, h, b);
                }
                const size_t l = g2l_kv_last_at(NH, s, h, kv);
                if (la + 4 * (l + 1024) > all || l % 1024 || ends[l / 1024]++) return bad("a last block", s, h, kv);
            }
    return 1;
}

static int append(int S, int NH, int T)
{
    const long n = g2l_append_waves(S, NH, T);
    const int per = (int)g2l_append_blocks(T);
    for (int p0 = 0; p0 < 16; ++p0) // blocks that fill, from any position in one, are all somebody's
        if ((p0 + T) / 16 > per) return bad("too few waves", T, p0, per);
    std::vector<unsigned char> seen((size_t)n, 0);
    for (long item = 0; item < (n + 3) / 4 * 4; ++item) {
        int h, kv, i;
        long s;
        g2l_append_item((unsigned)item, NH, T, &h, &kv, &i, &s);
        if (item >= n) {
            if (s < S) return bad("a wave behind the last has work", item, s, 0);
            continue;
        }
        if (h < 0 || h >= NH || kv < 0 || kv > 1 || i < 0 || i >= per || s < 0 || s >= S) return bad("a wave's work", item, s, h);
        const size_t at = (((size_t)s * NH + h) * 2 + kv) * per + i;
        if (seen[at]++) return bad("work of two waves", item, s, h);
    }
    return 1;
}

static int attend(int blocks, int span, int splits, int nw, int len, int mistake)
{
    const int full = len / 16, left = len % 16;
    if ((long)span * splits < blocks) return bad("the parts do not cover the blocks", span, splits, blocks);
    std::vector<int> seen(blocks + 1, 0);
    int tails = 0;
    for (int p = 0; p < splits; ++p)
        for (int w = 0; w < nw; ++w) {
            const int end = g2l_attn_end(p, span, full);
            for (int b = g2l_attn_first(p, span, w); b < end; b += g2l_attn_step(nw) - (mistake == 1))
                for (int u = 0; u < 4; ++u)
                    if (b + u < end) {
                        if (b + u < 0 || b + u >= full || seen[b + u]++) return bad("a block outside or twice", p, w, b + u);
                    }
            if (left && (mistake == 2 ? full / span == p && w == (full % span + 3) / 4 : g2l_attn_left(p, span, full, w, nw))) ++tails;
        }
    for (int b = 0; b < full; ++b)
        if (!seen[b]) return bad("a block is nobody's", b, full, 0);
    if (tails != (left ? 1 : 0)) return bad("takers of the last block", tails, len, 0);
    return 1;
}

int main(int n, char **v)
{
    auto arg = [&](int i) { return i < n ? std::atol(v[i]) : 0; };
    int ok = 0;
    if (n > 1 && !std::strcmp(v[1], "weights")) ok = weights(arg(2), arg(3), (int)arg(4));
    else if (n > 1 && !std::strcmp(v[1], "cache")) ok = cache(arg(2), (int)arg(3), arg(4));
    else if (n > 1 && !std::strcmp(v[1], "append")) ok = append((int)arg(2), (int)arg(3), (int)arg(4));
    else if (n > 1 && !std::strcmp(v[1], "attend")) ok = attend((int)arg(2), (int)arg(3), (int)arg(4), (int)arg(5), (int)arg(6), (int)arg(7));
    if (ok) std::printf("ok\n");
    return ok ? 0 : 1;
}

/*
 * g2_batch_plan.h -- layout of the 4-bit K/V cache and index arithmetic of
 * the operators for several texts at once (packed prompt attention, 4-bit
 * cache, beam search), shared by the C99 host (g2_batch.c), the gfx950 device
 * code (g2_batch.hip) and the CPU address checks.
 *
 * 4-bit cache of S sequences, NKV key heads of 64 dims: tiles of 32 positions
 *  [S][NKV][tiles] of G2B_TILE_BYTES:
 *   codes  [K, V][32][32 bytes], a byte holding two dims, the even one in its
 *   low half; scales [K, V][32][2] bf16, one for 32 dims.
 */
#ifndef G2_BATCH_PLAN_H
#define G2_BATCH_PLAN_H

#include <stddef.h>
#include <stdint.h>

#if defined(__HIPCC__) || defined(__HIP__)
#define G2B_FN __host__ __device__ __forceinline__
#else
#define G2B_FN static inline
#endif

#define G2B_DH 64
#define G2B_TILE 32                                   /* positions of a tile */
#define G2B_ROW (G2B_DH / 2)                          /* bytes of a position's codes */
#define G2B_SCALES (2 * G2B_TILE * G2B_ROW)           /* byte of a tile where its scales begin */
#define G2B_TILE_BYTES (G2B_SCALES + 2 * G2B_TILE * 4) /* 2304 */

G2B_FN long g2b_tiles(long max_seq) { return (max_seq + G2B_TILE - 1) / G2B_TILE; }
G2B_FN size_t g2b_bytes(long S, int NKV, long tiles) { return (size_t)S * NKV * tiles * G2B_TILE_BYTES; }
/* first byte of tile t of key head h of sequence s */
G2B_FN size_t g2b_tile_at(int NKV, long tiles, long s, int h, long t)
{
    return (((size_t)s * NKV + h) * tiles + t) * G2B_TILE_BYTES;
}
/* in a tile: byte of position p % 32's codes, and of its two scales (kv: 0 keys, 1 values) */
G2B_FN unsigned g2b_code_at(int kv, int p) { return (unsigned)(kv * G2B_TILE + p) * G2B_ROW; }
G2B_FN unsigned g2b_scale_at(int kv, int p) { return G2B_SCALES + (unsigned)(kv * G2B_TILE + p) * 4; }

/* the cache attention's workspace: parts of a head's positions at most, floats
 * for each (maximum, sum, 64 dims) */
#define G2B_SPLITS 32
#define G2B_PART_FLOATS (2 + G2B_DH)

/* ---- packed prompts */

/* Search of a list of `left` ascending values from its entry lo on, 64 probes at a
 * time: probe `lane`'s entry, counted from lo, and what c probes at or below
 * the value leave; 1 when lo is the count of entries at or below it.  It ends
 * for any c in 0 .. 64 that a list in no order gives. */
G2B_FN int g2b_probe(int left, int lane) { return lane * ((left + 63) / 64); }
G2B_FN int g2b_narrow(int *lo, int *left, int c)
{
    const int step = (*left + 63) / 64, rest = *left - (c - 1) * step;
    if (step <= 1 || c == 0) {
        *lo += c;
        return 1;
    }
    *lo += (c - 1) * step;
    *left = rest < step ? rest : step;
    return 0;
}

/* The keys lo .. end - 1 that query row `row` sees, and whether it is one of its
 * sequence's (in: one was found; q0, q1, k0, k1: its starts and the next one's,
 * whatever they hold): lo and end are in 0 .. k_rows. */
typedef struct {
    int lo, end, there;
} g2b_row;
G2B_FN int g2b_clamp(int v, int hi) { return v < 0 ? 0 : v < hi ? v : hi; }
G2B_FN g2b_row g2b_row_keys(int row, int in, int q0, int q1, int k0, int k1, int q_rows, int k_rows)
{
    g2b_row r;
    if (q1 > q_rows) q1 = q_rows;
    r.there = in && row >= q0 && row < q1;
    r.lo = g2b_clamp(k0, k_rows);
    r.end = r.lo;
    if (r.there) {
        const int end = g2b_clamp(k1, k_rows) - (q1 - 1 - row);
        if (end > r.lo) r.end = end;
    }
    return r;
}

/* The keys that a tile's rows see together, from the least and the greatest of its
 * waves' own: those begin at INT_MAX and end at -INT_MAX where no row sees any, which
 * is no range to count pieces in.  Such a tile has the keys 0 .. -1. */
G2B_FN int g2b_span_begin(int low, int high) { return low < high ? low : 0; }
G2B_FN int g2b_span_end(int low, int high) { return low < high ? high : 0; }

/* Work-group b of tiles * NKV: its key head and tile of queries.  Work-group b
 * runs on XCD b % 8.  The last tiles, whose rows see most keys, come first, all
 * heads of a tile side by side; of the heads, 8 n of them keep to XCD head % 8,
 * whose L2 then has their keys, and the rest go where there is room.  Of each 32
 * work-groups of an XCD (one for each of its CUs) every other 32 are turned
 * round, so that a CU gets a shorter one behind a longer one. */
G2B_FN void g2b_prompt_item(long b, int NKV, long tiles, int *head, long *tile)
{
    const long x = b % 8, k = b / 8, turn = k / 32, n = NKV * tiles;
    const long i = turn % 2 && (turn + 1) * 256 <= n ? 8 * (turn * 32 + 31 - k % 32) + x : b;
    const long rank = i / NKV;
    const int j = (int)(i % NKV), fixed = NKV / 8 * 8;
    *tile = tiles - 1 - rank;
    *head = j < fixed ? j / 8 * 8 + (int)x : fixed + j % 8;
}

/* ---- beam search: ids of a work-group's slice of a row,
 * most beams and continuations of a group; ints from count to count (a cache
 * line: the work-groups of a group meet there) */
#define G2B_SLICE 4096 /* times 1, 4 or 7 */
#define G2B_MAX_BEAMS 32
#define G2B_MAX_OUT 64
#define G2B_COUNT_INTS 16
/* The workspace: a count of work-groups for each group (0 between calls), for
 * each row and slice its largest logit and sum of exponentials (8 bytes), then
 * n_out candidates (8 bytes each: a logit's order and its id). */
G2B_FN size_t g2b_stats_at(long groups) { return (size_t)groups * G2B_COUNT_INTS * 4; }
G2B_FN size_t g2b_cands_at(long groups, long rows, int slices) { return g2b_stats_at(groups) + (size_t)rows * slices * 8; }
G2B_FN size_t g2b_beam_bytes(long groups, long rows, int slices, int n_out)
{
    return g2b_cands_at(groups, rows, slices) + (size_t)rows * slices * n_out * 8;
}

#endif

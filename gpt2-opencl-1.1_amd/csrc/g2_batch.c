/*
 * g2_batch.c -- entry points for several texts at once: packed prompt
 * attention, the 4-bit K/V cache, beam search (kernels: g2_batch.hip,
 * layouts: g2_batch_plan.h).
 *
 * Every call checks its arguments before it asks for the runtime, so a wrong
 * call is G2_E_ARG or G2_E_LIMIT without a device too.
 */
#include <math.h>
#include <string.h>

#include "g2_internal.h"
#include "g2_batch_plan.h"

#define MAX_ROWS (1 << 24)   /* rows of a packed buffer, positions of a cache */
#define MAX_STRIDE (1 << 24) /* elements from row to row: 31 rows apart is below 2^32 bytes */
#define MAX_HEADS 1024
#define MAX_SCALE 0x1p127f    /* times log2 e it is finite, so that a score of 0 stays 0 */
#define MAX_SEQS (1 << 20)
#define MAX_VOCAB (1 << 18)

static int aligned(const void *p, size_t a) { return (uintptr_t)p % a == 0; }
/* whether the arrays of ints (NULL: not there) are at ints' addresses: a kernel may read
 * an entry that all lanes want by a scalar load, which drops an address's last two bits */
static int ints_ok(const char *fn, const int *const *p, int n)
{
    for (int i = 0; i < n; ++i)
        if (!aligned(p[i], sizeof(int))) return g2i_err(G2_E_ARG, "%s: an array of ints is not at an int's address", fn);
    return G2_OK;
}
#define INTS_OK(fn, ...) ints_ok(fn, (const int *const[]){ __VA_ARGS__ }, (int)(sizeof((const int *const[]){ __VA_ARGS__ }) / sizeof(int *)))
static unsigned cdiv(long a, long b) { return (unsigned)((a + b - 1) / b); }
static int fits(long groups) { return groups <= (long)UINT32_MAX / 256; }
static int ready(void) { return g2i_ready() ? G2_OK : g2i_err(G2_E_STATE, "g2_init has not been called"); }
static size_t dsize(int dtype) { return dtype == G2_F16 ? 2 : 4; }

/* bytes from the first element to the last of `rows` rows of n elements */
static size_t span_of(long rows, long stride, long n, size_t size)
{
    return rows < 1 ? 0 : ((size_t)(rows - 1) * (size_t)stride + (size_t)n) * size;
}

static int heads_check(const char *fn, int n_head, int n_kv)
{
    if (n_head < 1 || n_kv < 1 || n_head % n_kv) return g2i_err(G2_E_ARG, "%s: %d heads on %d key heads", fn, n_head, n_kv);
    if (n_head > MAX_HEADS) return g2i_err(G2_E_LIMIT, "%s: %d heads above %d", fn, n_head, MAX_HEADS);
    return G2_OK;
}

/* ---------------------------------------------------------- packed prompts */

/* Work-groups of 128 queries convert each key once for four times as many of them,
 * those of 32 are four times as many.  Measured, in us (tiles, parts):
 *                                 groups of 128    128     32    two groups of waves
 *   fp32  1001 rows,   12 heads              96     75     23
 *         2 x 1000,    16                   256     77     48
 *         4001,        12                   384    300    179
 *         8 x 500,     20                   640     49     71
 *         4 x 1000,    25                   800    105    131
 *         16 x 100 to 1023, 25             1700    153    224
 *   fp16  1001,        12                    96     30     12      22
 *         1000,        25                   200     31     16      23
 *         40 x 20 to 60 behind 700, 16/4    200     28     22      26
 *         16 x 200,    12                   300     12     15      12
 *         2 x 1000,    25                   400     34     32      27
 *         8001,        16/4                1000    235    287     193
 *         16 x 100 to 1023, 25             1700     55     98      68
 *         2 x 2900,    16/4                 728     89    129      74
 * fp32: 128 from two work-groups a CU on.  fp16: from 300 on, with two groups of
 * waves where keys are long or tiles too few for four to a CU.  Long by their mean, all
 * that the host knows: one text of 4000 before 60 of 70 (16/4) counts as short and takes
 * 91, with two groups 75; one of 8000 before ten of 10 212, and 218. */
int g2i_prompt_form(int f16, int q_rows, int k_rows, int n_seq, int n_head, int n_kv, long *tiles)
{
    const long queries = (long)q_rows * (n_head / n_kv);
    const int many = (queries + 127) / 128 * n_kv >= (f16 ? 300 : 512), size = many ? 128 : 32;
    /* (tiles of up to 63 sequences are their own, the last of each may not be full; of more
     * sequences they are of all rows: prompt_find has both sides) */
    *tiles = n_seq > 1 && n_seq < 64 ? queries / size + n_seq : (queries + size - 1) / size;
    return !many ? PF_SPLIT : f16 && (k_rows / n_seq >= 1500 || *tiles * n_kv < 1024) ? PF_DUO : PF_TILE;
}

int g2_attn_prompt(const void *q, int q_stride, const void *k, const void *v, int kv_stride, void *out, int out_stride,
                   int dtype, const int *q_start, const int *k_start, int n_seq, int q_rows, int k_rows, int n_head,
                   int n_kv, float scale)
{
    static const char fn[] = "g2_attn_prompt";
    if (!q || !k || !v || !out) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (dtype != G2_F32 && dtype != G2_F16) return g2i_err(G2_E_ARG, "%s: bad dtype %d", fn, dtype);
    int rc = heads_check(fn, n_head, n_kv);
    if (rc) return rc;
    if (n_seq < 1 || q_rows < 1 || k_rows < 0) return g2i_err(G2_E_ARG, "%s: %d sequences, %d rows, %d keys", fn, n_seq, q_rows, k_rows);
    if (n_seq > 1 && (!q_start || !k_start)) return g2i_err(G2_E_ARG, "%s: %d sequences need their starts", fn, n_seq);
    const int nq = n_head * G2B_DH, nk = n_kv * G2B_DH;
    if ((q_rows > 1 && (q_stride < nq || out_stride < nq)) || (k_rows > 1 && kv_stride < nk))
        return g2i_err(G2_E_ARG, "%s: strides %d, %d and %d of rows of %d and %d", fn, q_stride, out_stride, kv_stride, nq, nk);
    if (q_rows > MAX_ROWS || k_rows > MAX_ROWS || n_seq > MAX_SEQS ||
        (q_rows > 1 && (q_stride > MAX_STRIDE || out_stride > MAX_STRIDE)) || (k_rows > 1 && kv_stride > MAX_STRIDE))
        return g2i_err(G2_E_LIMIT, "%s: at most %d rows, %d elements apart, and %d sequences", fn, MAX_ROWS, MAX_STRIDE, MAX_SEQS);
    if (!(fabsf(scale) <= MAX_SCALE)) return g2i_err(G2_E_ARG, "%s: the scale is not finite or above 2^127", fn);
    const size_t size = dsize(dtype), no = span_of(q_rows, out_stride, nq, size), ns = ((size_t)n_seq + 1) * sizeof(int);
    if (!aligned(q, size) || !aligned(k, size) || !aligned(v, size) || !aligned(out, size))
        return g2i_err(G2_E_ARG, "%s: a buffer is not at an element's address", fn);
    if ((rc = INTS_OK(fn, q_start, k_start))) return rc;
    const size_t nkv = span_of(k_rows, kv_stride, nk, size);
    if (g2i_overlap(out, no, q, span_of(q_rows, q_stride, nq, size)) || g2i_overlap(out, no, k, nkv) || g2i_overlap(out, no, v, nkv) ||
        (q_start && g2i_overlap(out, no, q_start, ns)) || (k_start && g2i_overlap(out, no, k_start, ns)))
        return g2i_err(G2_E_ARG, "%s: the output overlaps an input", fn);
    long tiles;
    const int f16 = dtype == G2_F16, form = g2i_prompt_form(f16, q_rows, k_rows, n_seq, n_head, n_kv, &tiles);
    if (!fits(2 * tiles * n_kv) || (long)q_rows * (n_head / n_kv) > INT32_MAX - 128) return g2i_err(G2_E_LIMIT, "%s: too many rows and heads for one call", fn);
    if ((rc = ready())) return rc;
    g2_attn_prompt_args a = { q, k, v, out, q_start, k_start, q_rows > 1 ? q_stride : nq, k_rows > 1 ? kv_stride : nk,
                              q_rows > 1 ? out_stride : nq, n_seq, q_rows, k_rows, n_head, n_kv, (int)tiles,
                              aligned(k, 4) && aligned(v, 4) && (k_rows <= 1 || kv_stride % 2 == 0), scale };
    const int fid = form == PF_SPLIT ? (!f16 ? G2F_PROMPT_SPLIT_F32 : a.even ? G2F_PROMPT_SPLIT_F16 : G2F_PROMPT_SPLIT_F16_ODD)
                  : form == PF_DUO ? G2F_PROMPT_DUO_F16 : f16 ? G2F_PROMPT_TILE_F16 : G2F_PROMPT_TILE_F32;
    return g2i_launch(fid, (unsigned)(tiles * n_kv), 1, form == PF_DUO ? 512 : 256, &a);
}

/* -------------------------------------------------------------- 4-bit cache */

static int kv4_sizes(int n_seq, int n_kv, int max_seq)
{
    return n_seq >= 1 && n_kv >= 1 && n_kv <= MAX_HEADS && max_seq >= 1 && max_seq <= MAX_ROWS && n_seq <= (1 << 22) / n_kv;
}

size_t g2_kv4_bytes(int n_seq, int n_kv, int max_seq)
{
    return kv4_sizes(n_seq, n_kv, max_seq) ? g2b_bytes(n_seq, n_kv, g2b_tiles(max_seq)) : 0;
}

size_t g2_kv4_work_bytes(int n_seq, int n_head)
{
    return kv4_sizes(n_seq, n_head, 1) ? (size_t)n_seq * n_head * G2B_SPLITS * G2B_PART_FLOATS * sizeof(float) : 0;
}

static int kv4_check(const char *fn, const void *cache, int n_seq, int n_kv, int max_seq)
{
    if (!cache) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (n_seq < 1 || n_kv < 1 || max_seq < 1) return g2i_err(G2_E_ARG, "%s: sizes must be positive", fn);
    if (!kv4_sizes(n_seq, n_kv, max_seq))
        return g2i_err(G2_E_LIMIT, "%s: %d sequences x %d heads x %d positions: at most %d heads, %d positions, 4M sequences x heads",
                       fn, n_seq, n_kv, max_seq, MAX_HEADS, MAX_ROWS);
    if (!aligned(cache, 16)) return g2i_err(G2_E_ARG, "%s: the cache must be 16-byte aligned", fn);
    return G2_OK;
}

int g2_kv4_append(const void *k, const void *v, int stride, int dtype, void *cache, const int *row_start, const int *pos,
                  int start, int n_seq, int rows, int n_kv, int max_seq)
{
    static const char fn[] = "g2_kv4_append";
    int rc = kv4_check(fn, cache, n_seq, n_kv, max_seq);
    if (rc) return rc;
    if (!k || !v) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (dtype != G2_F32 && dtype != G2_F16) return g2i_err(G2_E_ARG, "%s: bad dtype %d", fn, dtype);
    if (rows < 1 || (rows > 1 && stride < n_kv * G2B_DH))
        return g2i_err(G2_E_ARG, "%s: %d rows of %d, %d apart", fn, rows, n_kv * G2B_DH, stride);
    if (rows > MAX_ROWS || (rows > 1 && stride > MAX_STRIDE))
        return g2i_err(G2_E_LIMIT, "%s: at most %d rows, %d elements apart", fn, MAX_ROWS, MAX_STRIDE);
    if (!row_start && rows % n_seq) return g2i_err(G2_E_ARG, "%s: %d rows of %d sequences need their starts", fn, rows, n_seq);
    if (!pos && (start < 0 || start >= max_seq)) return g2i_err(G2_E_ARG, "%s: position %d outside the cache of %d", fn, start, max_seq);
    const size_t size = dsize(dtype), n = span_of(rows, stride, n_kv * G2B_DH, size), nc = g2_kv4_bytes(n_seq, n_kv, max_seq);
    if (!aligned(k, size) || !aligned(v, size)) return g2i_err(G2_E_ARG, "%s: a buffer is not at an element's address", fn);
    if ((rc = INTS_OK(fn, row_start, pos))) return rc;
    if (g2i_overlap(cache, nc, k, n) || g2i_overlap(cache, nc, v, n) || (row_start && g2i_overlap(cache, nc, row_start, ((size_t)n_seq + 1) * 4)) ||
        (pos && g2i_overlap(cache, nc, pos, (size_t)n_seq * 4)))
        return g2i_err(G2_E_ARG, "%s: overlapping buffers", fn);
    const long waves = ((long)rows + 7) / 8 * 2 * n_kv;
    if (!fits((waves + 3) / 4)) return g2i_err(G2_E_LIMIT, "%s: too many rows for one call", fn);
    if ((rc = ready())) return rc;
    g2_kv4_append_args a = { k, v, cache, row_start, pos, rows > 1 ? stride : 0, start, n_seq, rows, row_start ? 0 : rows / n_seq,
                             n_kv, max_seq, (int)g2b_tiles(max_seq) };
    return g2i_launch(dtype == G2_F16 ? G2F_KV4_APPEND_F16 : G2F_KV4_APPEND_F32, cdiv(waves, 4), 1, 256, &a);
}

int g2_kv4_read(const void *cache, float *k, float *v, const int *origin, const int *len, int T_kv, int start, int T,
                int n_seq, int n_kv, int max_seq)
{
    static const char fn[] = "g2_kv4_read";
    int rc = kv4_check(fn, cache, n_seq, n_kv, max_seq);
    if (rc) return rc;
    if (!k || !v) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (T_kv < 0 || T_kv > max_seq || start < 0 || T < 1 || start > max_seq - T)
        return g2i_err(G2_E_ARG, "%s: positions %d..%ld, length %d, cache of %d", fn, start, (long)start + T - 1, T_kv, max_seq);
    if (!aligned(k, 4) || !aligned(v, 4)) return g2i_err(G2_E_ARG, "%s: a buffer is not at an element's address", fn);
    if ((rc = INTS_OK(fn, origin, len))) return rc;
    const size_t n = (size_t)n_seq * T * n_kv * 256, nc = g2_kv4_bytes(n_seq, n_kv, max_seq), nl = (size_t)n_seq * 4;
    const size_t nt = (size_t)n_seq * max_seq * 4;
    if (g2i_overlap(k, n, v, n) || g2i_overlap(k, n, cache, nc) || g2i_overlap(v, n, cache, nc) ||
        (len && (g2i_overlap(k, n, len, nl) || g2i_overlap(v, n, len, nl))) ||
        (origin && (g2i_overlap(k, n, origin, nt) || g2i_overlap(v, n, origin, nt))))
        return g2i_err(G2_E_ARG, "%s: overlapping buffers", fn);
    if ((rc = ready())) return rc;
    g2_kv4_read_args a = { cache, k, v, origin, len, T_kv, start, T, n_seq, n_kv, max_seq, (int)g2b_tiles(max_seq) };
    const long threads = (long)(n / 16);
    return g2i_launch(G2F_KV4_READ, threads > (1l << 20) * 256 ? 1u << 20 : cdiv(threads, 256), 1, 256, &a);
}

/* Query heads to a pass over their key head's positions, passes to a key head,
 * parts of the positions and tiles to a part, waves to a work-group.  us, one call
 * after the other, caches that no cache holds where they are large:
 *  - up to four heads share a pass, fewer where that leaves less than 200
 *    work-groups: the sums of four heads take four times as long as one's, and
 *    a CU for each pays more than the codes read again (64 sequences of 2 x 8
 *    heads x 1000 12.0 with 4, 12.9 with 2, 15.7 with 1; 30 of 4 x 4 x 128 5.3,
 *    4.2, 5.0; one of 4 x 4 x 1000 11.4, 7.7, 5.6);
 *  - parts above 1024 positions, of 256 and more, as many as 256 work-groups
 *    (12 heads x 4000 7.1 in 16 parts, 8.0 in 32, 8.6 in 4; 16 x 50000 on 4 key
 *    heads 13.0 in 16, 14.0 in 32);
 *  - waves of 64 positions a step, each of which costs the same at the end: one up
 *    to 128 positions, for many heads up to 256 (3600 heads x 200 15.6, four 20.1;
 *    360 x 128 4.2, 4.9), eight from 800 for few heads (96 x 901 6.3, four 6.5; 256
 *    passes of two heads x 2000 12.1, 14.6), four else (12 x 700 5.0, eight 5.3;
 *    1200 x 640 14.4, eight 17.5, one 15.3).
 * Positions are T_kv, all that the host knows: where it is a bound far above the lengths, as
 * in a recorded step, a call takes the bound's form (1024 for lengths of 60, 250 and 700:
 * 48 x 25 heads 6.9 for 4.7, 8.3 for 7.6, 13.3 for 13.2; 8 x 12 heads 4.5 for 3.6, 4.3 for
 * 3.9, 5.3 for 5.1; 50000 for 5000, 16 heads on 4: 12.9 for 7.2, the parts beyond being
 * empty). */
int g2i_kv4_form(int n_seq, int n_head, int n_kv, int T_kv, int *heads, int *chunks, int *span, int *waves)
{
    const int group = n_head / n_kv;
    const long tiles = g2b_tiles(T_kv) > 0 ? g2b_tiles(T_kv) : 1;
    long wgs, splits = 1;
    for (int most = 4;; most /= 2) {
        *chunks = (group + most - 1) / most;
        *heads = (group + *chunks - 1) / *chunks;
        wgs = (long)n_seq * n_kv * *chunks;
        if (wgs >= 200 || most == 1) break;
    }
    if (tiles > 32 && wgs < 256) {
        splits = tiles / 8 < 256 / wgs ? tiles / 8 : 256 / wgs;
        if (splits > G2B_SPLITS) splits = G2B_SPLITS;
    }
    *span = (int)((tiles + splits - 1) / splits);
    splits = (tiles + *span - 1) / *span;
    *waves = *heads == 1 && *span <= (wgs * splits >= 1024 ? 8 : 4) ? 1 : *span > 24 && wgs * splits < 512 ? 8 : 4;
    return (int)splits;
}

int g2_attn_kv4(const float *q, int q_stride, const void *cache, float *out, int out_stride, const int *origin,
                const int *len, int T_kv, int n_seq, int n_head, int n_kv, int max_seq, float scale, float *work)
{
    static const char fn[] = "g2_attn_kv4";
    int rc = heads_check(fn, n_head, n_kv);
    if (!rc) rc = kv4_check(fn, cache, n_seq, n_kv, max_seq);
    if (rc) return rc;
    if (!kv4_sizes(n_seq, n_head, 1)) return g2i_err(G2_E_LIMIT, "%s: %d sequences x %d heads above 4M", fn, n_seq, n_head);
    if (!q || !out || !work) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    const int D = n_head * G2B_DH;
    if (T_kv < 0 || T_kv > max_seq || (n_seq > 1 && (q_stride < D || out_stride < D)))
        return g2i_err(G2_E_ARG, "%s: length %d of %d, strides %d and %d of rows of %d", fn, T_kv, max_seq, q_stride, out_stride, D);
    if (!(fabsf(scale) <= MAX_SCALE)) return g2i_err(G2_E_ARG, "%s: the scale is not finite or above 2^127", fn);
    if (!aligned(q, 4) || !aligned(out, 4) || !aligned(work, 4)) return g2i_err(G2_E_ARG, "%s: a buffer is not at an element's address", fn);
    if ((rc = INTS_OK(fn, origin, len))) return rc;
    const size_t nq = span_of(n_seq, q_stride, D, 4), no = span_of(n_seq, out_stride, D, 4), nl = (size_t)n_seq * 4;
    const size_t nc = g2_kv4_bytes(n_seq, n_kv, max_seq), nw = g2_kv4_work_bytes(n_seq, n_head), nt = nl * max_seq;
    if (g2i_overlap(out, no, q, nq) || g2i_overlap(out, no, cache, nc) || g2i_overlap(out, no, work, nw) ||
        g2i_overlap(work, nw, q, nq) || g2i_overlap(work, nw, cache, nc) ||
        (len && (g2i_overlap(out, no, len, nl) || g2i_overlap(work, nw, len, nl))) ||
        (origin && (g2i_overlap(out, no, origin, nt) || g2i_overlap(work, nw, origin, nt))))
        return g2i_err(G2_E_ARG, "%s: overlapping buffers", fn);
    if ((rc = ready())) return rc;
    g2_kv4_attn_args a;
    memset(&a, 0, sizeof a);
    a.q = q; a.cache = cache; a.out = out; a.part = work; a.origin = origin; a.len = len;
    a.q_stride = n_seq > 1 ? q_stride : 0; a.out_stride = n_seq > 1 ? out_stride : 0;
    a.T_kv = T_kv; a.S = n_seq; a.NH = n_head; a.NKV = n_kv; a.max_seq = max_seq; a.tiles = (int)g2b_tiles(max_seq);
    a.scale = scale;
    int waves;
    a.splits = g2i_kv4_form(n_seq, n_head, n_kv, T_kv, &a.heads, &a.chunks, &a.span, &waves);
    const int fid = a.heads == 1 ? (waves == 1 ? G2F_KV4_ATTN1_1 : waves == 4 ? G2F_KV4_ATTN1_4 : G2F_KV4_ATTN1_8)
                  : a.heads == 2 ? (waves == 4 ? G2F_KV4_ATTN2_4 : G2F_KV4_ATTN2_8)
                                 : (waves == 4 ? G2F_KV4_ATTN4_4 : G2F_KV4_ATTN4_8);
    rc = g2i_launch(fid + (origin ? 1 : 0), (unsigned)((long)n_seq * n_kv * a.chunks * a.splits), 1, 64u * (unsigned)waves, &a);
    if (!rc && a.splits > 1) rc = g2i_launch(G2F_KV4_JOIN, (unsigned)(n_seq * n_head), 1, 256, &a);
    return rc;
}

/* -------------------------------------------------------------- beam search */

static int beam_sizes(int groups, int beams, int V, int n_out)
{
    return groups >= 1 && beams >= 1 && V >= 1 && n_out >= 1 && beams <= G2B_MAX_BEAMS && n_out <= G2B_MAX_OUT && V <= MAX_VOCAB &&
           groups <= (1 << 16) / beams;
}

/* Slices of 4096 ids while that makes at most 256 work-groups (one for each CU, which
 * it has to itself), else of 16384, else of 28672.  us, rows of 50257, eight chosen in
 * groups of one beam (of eight):
 *                 4096         16384        28672
 *    16 rows   9.3 (10.8)   10.1 (12.1)  10.6 (11.8)
 *    32       13.6 (15.0)   10.1 (12.7)  10.8 (12.1)
 *    64       22.9 (22.2)   10.6 (12.4)  11.2 (11.9)
 *   128       42.5 (36.3)   20.4 (22.2)  11.7 (12.8)
 *   512        172  (129)    74  (68)    43.9 (41.9) */
int g2i_beam_form(int rows, int V, int *slices)
{
    const int times = (long)rows * cdiv(V, G2B_SLICE) <= 256 ? 1 : (long)rows * cdiv(V, 4 * G2B_SLICE) <= 256 ? 4 : 7;
    *slices = (int)cdiv(V, times * G2B_SLICE);
    return times;
}

size_t g2_beam_work_bytes(int groups, int beams, int V, int n_out)
{
    int slices;
    if (!beam_sizes(groups, beams, V, n_out)) return 0;
    g2i_beam_form(groups * beams, V, &slices);
    return g2b_beam_bytes(groups, (long)groups * beams, slices, n_out);
}

int g2_beam_select(const float *logits, const float *score, const int *done, int eos, float *out_score, int *out_parent,
                   int *out_id, int *out_done, int groups, int beams, int V, int n_out, void *work)
{
    static const char fn[] = "g2_beam_select";
    if (!logits || !score || !out_score || !out_parent || !out_id || !work) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (groups < 1 || beams < 1 || V < 1 || n_out < 1) return g2i_err(G2_E_ARG, "%s: sizes must be positive", fn);
    if (!beam_sizes(groups, beams, V, n_out))
        return g2i_err(G2_E_LIMIT, "%s: %d groups of %d beams, %d ids, %d continuations: at most %d beams, %d rows, %d ids, %d continuations",
                       fn, groups, beams, V, n_out, G2B_MAX_BEAMS, 1 << 16, MAX_VOCAB, G2B_MAX_OUT);
    if (eos < -1 || eos >= V || (done && eos < 0)) return g2i_err(G2_E_ARG, "%s: end id %d of %d", fn, eos, V);
    if (!aligned(work, 8)) return g2i_err(G2_E_ARG, "%s: the workspace must be 8-byte aligned", fn);
    if (!aligned(logits, 4) || !aligned(score, 4) || !aligned(out_score, 4)) return g2i_err(G2_E_ARG, "%s: a buffer is not at an element's address", fn);
    int rc = INTS_OK(fn, done, out_parent, out_id, out_done);
    if (rc) return rc;
    const long rows = (long)groups * beams;
    const size_t n = (size_t)groups * n_out * 4, nr = (size_t)rows * 4, nw = g2_beam_work_bytes(groups, beams, V, n_out);
    const struct { const void *p; size_t n; } in[] = { { logits, nr * V }, { score, nr }, { done, done ? nr : 0 } };
    const struct { const void *p; size_t n; } outs[] = { { out_score, n }, { out_parent, n }, { out_id, n }, { out_done, out_done ? n : 0 }, { work, nw } };
    for (int i = 0; i < 5; ++i) {
        int bad = 0;
        for (int j = 0; j < 3; ++j) bad |= outs[i].n && in[j].n && g2i_overlap(outs[i].p, outs[i].n, in[j].p, in[j].n);
        for (int j = 0; j < i; ++j) bad |= outs[i].n && outs[j].n && g2i_overlap(outs[i].p, outs[i].n, outs[j].p, outs[j].n);
        if (bad) return g2i_err(G2_E_ARG, "%s: overlapping buffers", fn);
    }
    if ((rc = ready())) return rc;
    char *p = work;
    g2_beam_args a;
    memset(&a, 0, sizeof a);
    a.logits = logits; a.score = score; a.done = done;
    a.out_score = out_score; a.out_parent = out_parent; a.out_id = out_id; a.out_done = out_done;
    a.eos = eos; a.groups = groups; a.beams = beams; a.V = V; a.n_out = n_out;
    const int times = g2i_beam_form((int)rows, V, &a.slices);
    a.counts = work;
    a.stats = (unsigned long long *)(p + g2b_stats_at(groups));
    a.cands = (unsigned long long *)(p + g2b_cands_at(groups, rows, a.slices));
    return g2i_launch(times == 1 ? G2F_BEAM_SELECT1 : times == 4 ? G2F_BEAM_SELECT4 : G2F_BEAM_SELECT7, (unsigned)(rows * a.slices), 1, 1024, &a);
}

int g2_beam_reorder(const int *ids, int *ids_out, int ids_stride, const int *next, const int *origin, int *origin_out,
                    int origin_stride, const int *parent, const int *len, int T, int groups, int beams)
{
    static const char fn[] = "g2_beam_reorder";
    const int has_ids = ids || ids_out, has_origin = origin || origin_out;
    if (!parent || (!has_ids && !has_origin) || (has_ids && (!ids || !ids_out || !next)) || (has_origin && (!origin || !origin_out)))
        return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (groups < 1 || beams < 1) return g2i_err(G2_E_ARG, "%s: sizes must be positive", fn);
    if (beams > G2B_MAX_BEAMS || groups > (1 << 16) / beams)
        return g2i_err(G2_E_LIMIT, "%s: %d groups of %d beams: at most %d beams, %d rows", fn, groups, beams, G2B_MAX_BEAMS, 1 << 16);
    if (T < 0 || (has_ids && T >= ids_stride) || (has_origin && T >= origin_stride))
        return g2i_err(G2_E_ARG, "%s: %d ints and one more in rows of %d and %d", fn, T, ids_stride, origin_stride);
    if (T >= MAX_ROWS) return g2i_err(G2_E_LIMIT, "%s: rows of %d: at most %d", fn, T, MAX_ROWS);
    int rc = INTS_OK(fn, ids, ids_out, next, origin, origin_out, parent, len);
    if (rc) return rc;
    const long rows = (long)groups * beams;
    const size_t ni = has_ids ? span_of(rows, ids_stride, T + 1, 4) : 0, no = has_origin ? span_of(rows, origin_stride, T + 1, 4) : 0;
    const size_t nr = (size_t)rows * 4;
    const struct { const void *p; size_t n; } in[] = { { parent, nr }, { len, len ? (size_t)groups * 4 : 0 }, { next, has_ids ? nr : 0 } };
    int bad = (has_ids && ids != ids_out && g2i_overlap(ids, ni, ids_out, ni)) ||
              (has_origin && origin != origin_out && g2i_overlap(origin, no, origin_out, no)) ||
              (has_ids && has_origin && (g2i_overlap(ids_out, ni, origin_out, no) || g2i_overlap(ids_out, ni, origin, no) || g2i_overlap(ids, ni, origin_out, no)));
    for (int i = 0; i < 3; ++i)
        bad |= in[i].n && ((has_ids && g2i_overlap(ids_out, ni, in[i].p, in[i].n)) || (has_origin && g2i_overlap(origin_out, no, in[i].p, in[i].n)));
    if (bad) return g2i_err(G2_E_ARG, "%s: overlapping buffers", fn);
    const long chunks = ((long)T + 1 + 255) / 256;
    if (!fits(chunks * rows)) return g2i_err(G2_E_LIMIT, "%s: too many ints for one call", fn);
    if ((rc = ready())) return rc;
    g2_beam_move_args a = { ids, ids_out, next, origin, origin_out, parent, len, ids_stride, origin_stride, T, groups, beams };
    if ((has_ids && ids == ids_out) || (has_origin && origin == origin_out))
        return g2i_launch(G2F_BEAM_MOVE, (unsigned)(chunks * groups), 1, 256, &a);
    return g2i_launch(G2F_BEAM_COPY, (unsigned)(chunks * rows), 1, 256, &a);
}

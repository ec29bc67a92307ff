/*
 * g2_lowbit.c -- entry points of the 4-bit weights, the 8-bit K/V cache and
 * the rules on logits (kernels: g2_lowbit.hip, layouts: g2_lowbit_plan.h).
 *
 * Every call checks its arguments before it asks for the runtime, so a wrong
 * call is G2_E_ARG or G2_E_LIMIT without a device too.
 */
#include <math.h>
#include <string.h>

#include "g2_internal.h"
#include "g2_lowbit_plan.h"

#define MAX_DIM (1 << 24)      /* N, K: products of two stay far inside 64 bits */
#define MAX_SEQ (1 << 24)      /* positions of a cache */
#define MAX_HEADS 1024
#define MAX_VOCAB (1 << 18)
#define MAX_LIST 65535         /* ids of a context, entries of a bias list: counted in 16 bits */

static int aligned(const void *p, size_t a) { return (uintptr_t)p % a == 0; }
static unsigned cdiv(long a, long b) { return (unsigned)((a + b - 1) / b); }
/* work-groups of 256 threads for n items, the kernel strides over the rest */
static unsigned strided(long n) { return n > (1l << 20) * 256 ? 1u << 20 : cdiv(n, 256); }
/* Whether a launch of this many threads is one that HIP takes. */
static int fits(long threads) { return threads <= (long)UINT32_MAX; }

static int ready(void) { return g2i_ready() ? G2_OK : g2i_err(G2_E_STATE, "g2_init has not been called"); }

/* ------------------------------------------------------------ 4-bit weights */

static int q4_sizes(int N, int K, int group)
{
    return N >= 1 && K >= 1 && N <= MAX_DIM && K <= MAX_DIM && (group == 32 || group == 64 || group == 128);
}

size_t g2_q4_code_bytes(int N, int K) { return q4_sizes(N, K, 32) ? g2l_code_bytes(N, K) : 0; }

size_t g2_q4_scale_bytes(int N, int K, int group)
{
    return q4_sizes(N, K, group) ? g2l_scale_count(N, K, group) * sizeof(uint16_t) : 0;
}

static int q4_check(const char *fn, const void *codes, const void *scales, int N, int K, int group)
{
    if (!codes || !scales) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (N < 1 || K < 1) return g2i_err(G2_E_ARG, "%s: N and K must be positive", fn);
    if (N > MAX_DIM || K > MAX_DIM) return g2i_err(G2_E_LIMIT, "%s: N=%d K=%d above %d", fn, N, K, MAX_DIM);
    if (!q4_sizes(N, K, group)) return g2i_err(G2_E_ARG, "%s: group %d is not 32, 64 or 128", fn, group);
    if (!aligned(codes, 16) || !aligned(scales, 16))
        return g2i_err(G2_E_ARG, "%s: codes and scales must be 16-byte aligned", fn);
    return G2_OK;
}

/* Work-groups that lay out or read back: 32 rows of 128 columns of [K,N], two
 * times 16 of [N,K]; the kernels stride over what is more. */
static unsigned q4_groups(int N, int K, int in_out)
{
    const long chunks = g2l_chunks(K), tiles = g2l_tiles(N);
    const long n = in_out ? (tiles + 1) / 2 * chunks : (tiles * chunks + 1) / 2;
    return n < 1 << 20 ? (unsigned)n : 1u << 20; /* (threads of a launch: below 2^32) */
}

int g2_quantize_q4(const void *W, int w_dtype, int in_out, uint8_t *codes, uint16_t *scales, int N, int K, int group)
{
    int rc = q4_check("g2_quantize_q4", codes, scales, N, K, group);
    if (rc) return rc;
    if (!W) return g2i_err(G2_E_ARG, "g2_quantize_q4: NULL buffer");
    if (w_dtype != G2_F32 && w_dtype != G2_F16) return g2i_err(G2_E_ARG, "g2_quantize_q4: bad dtype %d", w_dtype);
    const size_t nc = g2_q4_code_bytes(N, K), ns = g2_q4_scale_bytes(N, K, group);
    const size_t nw = (size_t)N * K * (w_dtype == G2_F16 ? 2 : 4);
    if (g2i_overlap(codes, nc, scales, ns) || g2i_overlap(W, nw, codes, nc) || g2i_overlap(W, nw, scales, ns))
        return g2i_err(G2_E_ARG, "g2_quantize_q4: overlapping buffers");
    if ((rc = ready())) return rc;
    g2_q4_args a = { W, codes, scales, NULL, N, K, group, in_out ? 1 : 0 };
    if (in_out) return g2i_launch(w_dtype == G2_F16 ? G2F_Q4_PACK_T_F16 : G2F_Q4_PACK_T_F32, q4_groups(N, K, 1), 1, 512, &a);
    return g2i_launch(w_dtype == G2_F16 ? G2F_Q4_PACK_F16 : G2F_Q4_PACK_F32, q4_groups(N, K, 0), 1, 256, &a);
}

int g2_dequantize_q4(const uint8_t *codes, const uint16_t *scales, float *W, int in_out, int N, int K, int group)
{
    int rc = q4_check("g2_dequantize_q4", codes, scales, N, K, group);
    if (rc) return rc;
    if (!W) return g2i_err(G2_E_ARG, "g2_dequantize_q4: NULL buffer");
    const size_t nw = (size_t)N * K * 4;
    if (g2i_overlap(W, nw, codes, g2_q4_code_bytes(N, K)) || g2i_overlap(W, nw, scales, g2_q4_scale_bytes(N, K, group)))
        return g2i_err(G2_E_ARG, "g2_dequantize_q4: overlapping buffers");
    if ((rc = ready())) return rc;
    g2_q4_args a = { NULL, (uint8_t *)codes, (uint16_t *)scales, W, N, K, group, in_out ? 1 : 0 };
    return g2i_launch(in_out ? G2F_Q4_READ_T : G2F_Q4_READ, q4_groups(N, K, in_out), 1, in_out ? 512 : 256, &a);
}

/* The kernel of a product.  Two forms: the loop (a work-group of 8 or 16 waves
 * takes TR tiles of 16 rows, each wave every 8th or 16th chunk of 128 columns)
 * and the held form (fewer work-groups, which keep their chunks' activations
 * and take tiles in turn).  us in a replayed graph, matrices that no cache
 * holds, groups of 32 (of 128 where two figures stand):
 *  - one row: the loop over single tiles; 16 waves for the few tiles of long
 *    columns (1600 x 6400 4.8, with 8 waves 5.1; 1600 x 1600 3.1 both); the
 *    held form from 2048 tiles on, where splitting the activations anew for
 *    each tile costs most (50257 x 1600 11.4 and 9.7, loop 14.1 and 12.7; 50257
 *    x 768 7.2, 8.4; but 16000 x 1600 5.9, 5.1);
 *  - up to 8 rows, whose activations take longer to split: 16 waves up to 128
 *    tiles (1600 x 1600 4.1, 4.4; 1600 x 6400 8.1, 9.1); 2 tiles from 256, 4
 *    from 512 on (6400 x 1600 5.8, 5.7, 6.7 for 1, 2, 4; 10000 x 6400 21, 18,
 *    16); held from 2048 tiles (50257 x 1600 15.0, loop 24), with 16 waves and K
 *    to 4096 from 512 (12000 x 4000 9.9, loop 12.0).
 * Work-groups of the held form: as many as the registers leave resident (80 of
 * them a lane for 768). */
int g2i_q4_form(int M, int N, int K, int *waves, unsigned *wgs)
{
    const long tiles = g2l_tiles(N), chunks = g2l_chunks(K);
    long most = 0;
    int fid, tr = 1;
    *waves = 8;
    if (tiles >= 2048 && chunks <= 16) {
        most = M == 1 || chunks <= 8 ? 768 : 512;
        fid = M == 1 ? (chunks <= 8 ? G2F_Q4_MVH1_8_1_32 : G2F_Q4_MVH1_8_2_32)
                     : (chunks <= 8 ? G2F_Q4_MVH8_8_1_32 : G2F_Q4_MVH8_8_2_32);
    } else if (M > 1 && tiles >= 512 && chunks > 16 && chunks <= 32) {
        most = 256;
        *waves = 16;
        fid = G2F_Q4_MVH8_16_2_32;
    } else if (tiles <= 128 && chunks > (M == 1 ? 16 : 8)) {
        *waves = 16;
        fid = M == 1 ? G2F_Q4_MV1_16_1_32 : G2F_Q4_MV8_16_1_32;
    } else if (M == 1) fid = G2F_Q4_MV1_8_1_32;
    else {
        tr = tiles < 256 ? 1 : tiles < 512 ? 2 : 4;
        fid = tr == 1 ? G2F_Q4_MV8_8_1_32 : tr == 2 ? G2F_Q4_MV8_8_2_32 : G2F_Q4_MV8_8_4_32;
    }
    *wgs = (unsigned)(most ? (tiles < most ? tiles : most) : (tiles + tr - 1) / tr);
    return fid;
}

int g2_matvec_q4(const float *x, const uint8_t *codes, const uint16_t *scales, const float *bias, const float *residual,
                 float *y, int M, int N, int K, int group, int apply_gelu)
{
    int rc = q4_check("g2_matvec_q4", codes, scales, N, K, group);
    if (rc) return rc;
    if (!x || !y) return g2i_err(G2_E_ARG, "g2_matvec_q4: NULL buffer");
    if (M < 1) return g2i_err(G2_E_ARG, "g2_matvec_q4: M must be positive");
    if (M > 65535) return g2i_err(G2_E_LIMIT, "g2_matvec_q4: M=%d above 65535", M);
    const size_t ny = (size_t)M * N * 4;
    if (g2i_overlap(y, ny, x, (size_t)M * K * 4) || g2i_overlap(y, ny, codes, g2_q4_code_bytes(N, K)) ||
        g2i_overlap(y, ny, scales, g2_q4_scale_bytes(N, K, group)) || (bias && g2i_overlap(y, ny, bias, (size_t)N * 4)) ||
        (residual && residual != y && g2i_overlap(y, ny, residual, ny)))
        return g2i_err(G2_E_ARG, "g2_matvec_q4: the output overlaps an input");
    if ((rc = ready())) return rc;
    g2_q4mv_args a = { x, codes, scales, bias, residual, y, M, N, K, group, apply_gelu ? 1 : 0 };
    int waves;
    unsigned wgs;
    const int fid = g2i_q4_form(M, N, K, &waves, &wgs);
    return g2i_launch(fid + (group == 32 ? 0 : group == 64 ? 1 : 2), wgs, cdiv(M, 8), 64u * (unsigned)waves, &a);
}

/* ------------------------------------------------------------- 8-bit cache */

static int kv8_sizes(int n_seq, int n_head, int max_seq)
{
    return n_seq >= 1 && n_head >= 1 && n_head <= MAX_HEADS && max_seq >= 1 && max_seq <= MAX_SEQ &&
           n_seq <= (1 << 22) / n_head;
}

size_t g2_kv8_bytes(int n_seq, int n_head, int max_seq)
{
    return kv8_sizes(n_seq, n_head, max_seq) ? g2l_kv_bytes(n_seq, n_head, g2l_blocks(max_seq)) : 0;
}

size_t g2_kv8_work_bytes(int n_seq, int n_head)
{
    return kv8_sizes(n_seq, n_head, 1) ? (size_t)n_seq * n_head * G2L_SPLITS * G2L_PART_FLOATS * sizeof(float) : 0;
}

static int kv8_check(const char *fn, const void *cache, int n_seq, int n_head, int max_seq)
{
    if (!cache) return g2i_err(G2_E_ARG, "%s: NULL buffer", fn);
    if (n_seq < 1 || n_head < 1 || max_seq < 1) return g2i_err(G2_E_ARG, "%s: sizes must be positive", fn);
    if (!kv8_sizes(n_seq, n_head, max_seq))
        return g2i_err(G2_E_LIMIT, "%s: %d sequences x %d heads x %d positions: at most %d heads, %d positions, 4M sequences x heads",
                       fn, n_seq, n_head, max_seq, MAX_HEADS, MAX_SEQ);
    if (!aligned(cache, 16)) return g2i_err(G2_E_ARG, "%s: the cache must be 16-byte aligned", fn);
    return G2_OK;
}

int g2_kv8_append(const float *qkv, void *cache, const int *pos, const int *count, int start, int n_seq, int T,
                  int n_head, int max_seq)
{
    int rc = kv8_check("g2_kv8_append", cache, n_seq, n_head, max_seq);
    if (rc) return rc;
    if (!qkv) return g2i_err(G2_E_ARG, "g2_kv8_append: NULL buffer");
    if (T < 1 || T > max_seq || (!pos && (start < 0 || start > max_seq - T)))
        return g2i_err(G2_E_ARG, "g2_kv8_append: %d positions from %d outside the cache of %d", T, pos ? 0 : start, max_seq);
    const size_t size = g2_kv8_bytes(n_seq, n_head, max_seq), ints = (size_t)n_seq * sizeof(int);
    if (g2i_overlap(qkv, (size_t)n_seq * T * 3 * n_head * 256, cache, size) || (pos && g2i_overlap(pos, ints, cache, size)) ||
        (count && g2i_overlap(count, ints, cache, size)))
        return g2i_err(G2_E_ARG, "g2_kv8_append: overlapping buffers");
    const long waves = g2l_append_waves(n_seq, n_head, T);
    if (!fits((waves + 3) * 64)) return g2i_err(G2_E_LIMIT, "g2_kv8_append: too many rows for one call");
    if ((rc = ready())) return rc;
    const long nb = g2l_blocks(max_seq);
    char *c = cache;
    g2_kv8_append_args a = { qkv, (int8_t *)c, (float *)(c + g2l_kv_scales(n_seq, n_head, nb)),
                             (float *)(c + g2l_kv_last(n_seq, n_head, nb)), pos, count, start, T, n_seq, n_head, max_seq, (int)nb };
    return g2i_launch(G2F_KV8_APPEND, cdiv(waves, 4), 1, 256, &a);
}

int g2_kv8_read(const void *cache, float *k, float *v, const int *len, int T_kv, int start, int T, int n_seq,
                int n_head, int max_seq)
{
    int rc = kv8_check("g2_kv8_read", cache, n_seq, n_head, max_seq);
    if (rc) return rc;
    if (!k || !v) return g2i_err(G2_E_ARG, "g2_kv8_read: NULL buffer");
    if (T_kv < 0 || T_kv > max_seq || start < 0 || T < 1 || start > max_seq - T)
        return g2i_err(G2_E_ARG, "g2_kv8_read: positions %d..%ld, length %d, cache of %d", start, (long)start + T - 1, T_kv, max_seq);
    const size_t n = (size_t)n_seq * T * n_head * 256, nc = g2_kv8_bytes(n_seq, n_head, max_seq);
    if (g2i_overlap(k, n, v, n) || g2i_overlap(k, n, cache, nc) || g2i_overlap(v, n, cache, nc) ||
        (len && (g2i_overlap(k, n, len, (size_t)n_seq * 4) || g2i_overlap(v, n, len, (size_t)n_seq * 4))))
        return g2i_err(G2_E_ARG, "g2_kv8_read: overlapping buffers");
    if ((rc = ready())) return rc;
    const long nb = g2l_blocks(max_seq);
    const char *c = cache;
    g2_kv8_read_args a = { (const int8_t *)c, (const float *)(c + g2l_kv_scales(n_seq, n_head, nb)),
                           (const float *)(c + g2l_kv_last(n_seq, n_head, nb)), k, v, len, T_kv, start, T, n_seq, n_head, (int)nb };
    return g2i_launch(G2F_KV8_READ, strided((long)(n / 16)), 1, 256, &a);
}

/* Parts of a head's positions, blocks to a part and waves to a work-group.  us
 * in a replayed graph, caches that no cache holds:
 *  - one launch up to 1024 positions, and for 256 heads and more of any length;
 *    beyond, parts of 256 positions and more, as many as 512 work-groups (16
 *    heads x 2000 9.0 whole, 7.4 in parts; 16 x 4000 10.4 in 3 parts, 7.9 in
 *    15; 25 x 1024 6.4 and 7.1; 256 x 4000 27.0 and 28.3; numbers of heads that
 *    do not fill the 256 CUs evenly, 257 to 511, were not measured in parts);
 *  - a wave takes 64 positions at a time: one wave up to 64 (12 heads 3.3, four
 *    waves 3.7), for many heads up to 128 (1600 heads 8.7, 9.9), four up to 512
 *    (200 heads x 512 5.7, eight 6.0), eight beyond (25 x 1024 6.4, four 6.7,
 *    sixteen 6.7), but four for many heads, which fill the chip either way
 *    (1200 heads x 1024 within 1%) and may be much shorter than the bound. */
int g2i_kv8_form(long heads, int T_kv, int *span, int *waves)
{
    const long blocks = g2l_blocks(T_kv) > 0 ? g2l_blocks(T_kv) : 1;
    long splits = 1;
    if (blocks > 64 && heads < 256) {
        splits = blocks / 16 < 512 / heads ? blocks / 16 : 512 / heads;
        if (splits > G2L_SPLITS) splits = G2L_SPLITS;
    }
    *span = (int)((blocks + splits - 1) / splits);
    splits = (blocks + *span - 1) / *span;
    const int many = heads >= 512;
    *waves = *span <= 4 || (*span <= 8 && many) ? 1 : *span <= 32 || many ? 4 : 8;
    return (int)splits;
}

int g2_attn_kv8(const float *q, int q_stride, const void *cache, float *out, int out_stride, const int *len, int T_kv,
                int n_seq, int n_head, int max_seq, float scale, float *work)
{
    int rc = kv8_check("g2_attn_kv8", cache, n_seq, n_head, max_seq);
    if (rc) return rc;
    if (!q || !out || !work) return g2i_err(G2_E_ARG, "g2_attn_kv8: NULL buffer");
    const int D = n_head * G2L_DH;
    if (T_kv < 0 || T_kv > max_seq || (n_seq > 1 && (q_stride < D || out_stride < D)))
        return g2i_err(G2_E_ARG, "g2_attn_kv8: length %d of %d, strides %d and %d of rows of %d", T_kv, max_seq, q_stride, out_stride, D);
    const size_t nq = ((size_t)(n_seq - 1) * (size_t)(n_seq > 1 ? q_stride : 0) + D) * 4;
    const size_t no = ((size_t)(n_seq - 1) * (size_t)(n_seq > 1 ? out_stride : 0) + D) * 4;
    const size_t nc = g2_kv8_bytes(n_seq, n_head, max_seq), nw = g2_kv8_work_bytes(n_seq, n_head);
    if (g2i_overlap(out, no, q, nq) || g2i_overlap(out, no, cache, nc) || g2i_overlap(out, no, work, nw) ||
        g2i_overlap(work, nw, q, nq) || g2i_overlap(work, nw, cache, nc) || (len && g2i_overlap(out, no, len, (size_t)n_seq * 4)) ||
        (len && g2i_overlap(work, nw, len, (size_t)n_seq * 4)))
        return g2i_err(G2_E_ARG, "g2_attn_kv8: overlapping buffers");
    if ((rc = ready())) return rc;
    const long nb = g2l_blocks(max_seq);
    const char *c = cache;
    g2_kv8_attn_args a;
    memset(&a, 0, sizeof a);
    a.q = q; a.codes = (const int8_t *)c;
    a.scales = (const float *)(c + g2l_kv_scales(n_seq, n_head, nb));
    a.last = (const float *)(c + g2l_kv_last(n_seq, n_head, nb));
    a.out = out; a.part = work; a.len = len;
    a.q_stride = n_seq > 1 ? q_stride : 0; a.out_stride = n_seq > 1 ? out_stride : 0;
    a.T_kv = T_kv; a.S = n_seq; a.NH = n_head; a.blocks = (int)nb;
    a.scale = scale;
    const long heads = (long)n_seq * n_head;
    int waves;
    a.splits = g2i_kv8_form(heads, T_kv, &a.span, &waves);
    rc = g2i_launch(waves == 1 ? G2F_KV8_ATTN1 : waves == 4 ? G2F_KV8_ATTN4 : G2F_KV8_ATTN8, (unsigned)(heads * a.splits), 1,
                   64u * (unsigned)waves, &a);
    if (!rc && a.splits > 1) rc = g2i_launch(G2F_KV8_JOIN, (unsigned)heads, 1, 256, &a);
    return rc;
}

/* --------------------------------------------------------- rules on logits */

static int logits_rows(int rows) { return rows >= 1 && rows <= 1 << 16; }

size_t g2_logits_work_bytes(int rows) { return logits_rows(rows) ? (size_t)rows * G2L_CELL * sizeof(uint64_t) : 0; }

/* Whether the rules take the wide slices, and the slices of a row: 1024 ids each,
 * 8192 where that makes more than 1024 work-groups (us: 16 rows of 50257 7.2,
 * wide 7.4; 32 rows 8.7, 7.9; 64 rows 14.0, 12.1). */
int g2i_logits_form(int rows, int V, int *parts)
{
    const int wide = (long)rows * cdiv(V, G2L_SLICE) > 1024;
    *parts = (int)cdiv(V, wide ? G2L_SLICE_WIDE : G2L_SLICE);
    return wide;
}

int g2_apply_logit_rules(const float *logits, float *out, int *pick, int rows, int V, const g2_logit_rules *rules,
                         void *work)
{
    if (!logits || !rules || (!out && !pick)) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: NULL buffer");
    if (rows < 1 || V < 1) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: rows and V must be positive");
    if (!logits_rows(rows) || V > MAX_VOCAB)
        return g2i_err(G2_E_LIMIT, "g2_apply_logit_rules: %d rows of %d: at most %d of %d", rows, V, 1 << 16, MAX_VOCAB);
    const g2_logit_rules *r = rules;
    if (r->max_ctx > MAX_LIST || r->n_bias > MAX_LIST)
        return g2i_err(G2_E_LIMIT, "g2_apply_logit_rules: context of %d, %d biases: at most %d", r->max_ctx, r->n_bias, MAX_LIST);
    if (r->max_ctx < 0 || r->n_bias < 0 || (r->max_ctx && !r->ctx) || (r->n_bias && (!r->bias_id || !r->bias)))
        return g2i_err(G2_E_ARG, "g2_apply_logit_rules: bad context or bias list");
    if (!(r->repetition >= 0.f) || !isfinite(r->repetition) || !isfinite(r->frequency) || !isfinite(r->presence))
        return g2i_err(G2_E_ARG, "g2_apply_logit_rules: penalties must be finite, the repetition penalty not below 0");
    if (r->mask && r->mask_stride != 0 && r->mask_stride < (V + 31) / 32)
        return g2i_err(G2_E_ARG, "g2_apply_logit_rules: mask rows of %d words for %d ids", r->mask_stride, V);
    if (r->forbid < -1 || r->forbid >= V) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: forbidden id %d of %d", r->forbid, V);
    if (pick && (!work || !aligned(work, 8))) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: a pick needs the workspace");
    const size_t n = (size_t)rows * V * 4, nw = pick ? g2_logits_work_bytes(rows) : 0, np = pick ? (size_t)rows * 4 : 0;
    const struct { const void *p; size_t n; } in[] = {
        { r->ctx, r->max_ctx ? (size_t)rows * r->max_ctx * 4 : 0 }, { r->ctx_len, r->ctx_len ? (size_t)rows * 4 : 0 },
        { r->bias_id, (size_t)r->n_bias * 4 }, { r->bias, (size_t)r->n_bias * 4 },
        { r->mask, r->mask ? ((size_t)(rows - 1) * r->mask_stride + (V + 31) / 32) * 4 : 0 } };
    int bad = (out && out != logits && g2i_overlap(out, n, logits, n)) ||
              (pick && (g2i_overlap(pick, np, logits, n) || g2i_overlap(work, nw, logits, n) || g2i_overlap(work, nw, pick, np) ||
                        (out && (g2i_overlap(out, n, pick, np) || g2i_overlap(out, n, work, nw)))));
    for (size_t i = 0; i < sizeof in / sizeof *in; ++i)
        bad |= in[i].n && ((out && g2i_overlap(out, n, in[i].p, in[i].n)) ||
                           (pick && (g2i_overlap(pick, np, in[i].p, in[i].n) || g2i_overlap(work, nw, in[i].p, in[i].n))));
    if (bad) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: overlapping buffers");
    const int rc = ready();
    if (rc) return rc;
    g2_logits_args a;
    memset(&a, 0, sizeof a);
    a.logits = logits; a.out = out; a.pick = pick; a.cells = work;
    a.ctx = r->max_ctx ? r->ctx : NULL; a.ctx_len = r->ctx_len; a.max_ctx = r->max_ctx;
    a.bias_id = r->bias_id; a.bias = r->bias; a.n_bias = r->n_bias;
    a.mask = r->mask; a.mask_stride = r->mask_stride; a.forbid = r->forbid;
    a.rows = rows; a.V = V;
    a.repetition = r->repetition > 0.f ? r->repetition : 1.f; a.frequency = r->frequency; a.presence = r->presence;
    const int wide = g2i_logits_form(rows, V, &a.parts);
    return g2i_launch(wide ? G2F_LOGITS_WIDE : G2F_LOGITS, (unsigned)(rows * a.parts), 1, wide ? 1024 : 256, &a);
}

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
    const long items = g2l_tiles(N) * 16 * g2l_chunks(K) * (128 / group);
    return g2i_launch(w_dtype == G2_F16 ? G2F_Q4_PACK_F16 : G2F_Q4_PACK_F32, strided(items), 1, 256, &a);
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
    return g2i_launch(G2F_Q4_READ, strided((long)N * K), 1, 256, &a);
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
    if (!fits((long)N * 256)) return g2i_err(G2_E_LIMIT, "g2_matvec_q4: N=%d too large", N);
    return g2i_launch(G2F_Q4_MATVEC, (unsigned)N, (unsigned)M, 256, &a);
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
    if (g2i_overlap(qkv, (size_t)n_seq * T * 3 * n_head * 256, cache, g2_kv8_bytes(n_seq, n_head, max_seq)))
        return g2i_err(G2_E_ARG, "g2_kv8_append: overlapping buffers");
    const long waves = (long)n_seq * n_head * 2 * (T / G2L_BLOCK + 2);
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
    if (g2i_overlap(k, n, v, n) || g2i_overlap(k, n, cache, nc) || g2i_overlap(v, n, cache, nc))
        return g2i_err(G2_E_ARG, "g2_kv8_read: overlapping buffers");
    if ((rc = ready())) return rc;
    const long nb = g2l_blocks(max_seq);
    const char *c = cache;
    g2_kv8_read_args a = { (const int8_t *)c, (const float *)(c + g2l_kv_scales(n_seq, n_head, nb)),
                           (const float *)(c + g2l_kv_last(n_seq, n_head, nb)), k, v, len, T_kv, start, T, n_seq, n_head, (int)nb };
    return g2i_launch(G2F_KV8_READ, strided((long)(n / 2)), 1, 256, &a);
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
    return g2i_launch(G2F_KV8_ATTN, (unsigned)(n_seq * n_head), 1, 64, &a);
}

/* --------------------------------------------------------- rules on logits */

static int logits_rows(int rows) { return rows >= 1 && rows <= 1 << 16; }

size_t g2_logits_work_bytes(int rows) { return logits_rows(rows) ? (size_t)rows * G2L_PARTS * 2 * sizeof(float) : 0; }

int g2_apply_logit_rules(const float *logits, float *out, int *pick, int rows, int V, const g2_logit_rules *rules,
                         void *work)
{
    if (!logits || !rules || (!out && !pick)) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: NULL buffer");
    if (rows < 1 || V < 1) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: rows and V must be positive");
    if (!logits_rows(rows) || V > G2L_PARTS * G2L_SLICE)
        return g2i_err(G2_E_LIMIT, "g2_apply_logit_rules: %d rows of %d: at most %d of %d", rows, V, 1 << 16, G2L_PARTS * G2L_SLICE);
    const g2_logit_rules *r = rules;
    if (r->max_ctx < 0 || r->n_bias < 0 || (r->max_ctx && !r->ctx) || (r->n_bias && (!r->bias_id || !r->bias)))
        return g2i_err(G2_E_ARG, "g2_apply_logit_rules: bad context or bias list");
    if (!(r->repetition >= 0.f) || !isfinite(r->repetition) || !isfinite(r->frequency) || !isfinite(r->presence))
        return g2i_err(G2_E_ARG, "g2_apply_logit_rules: penalties must be finite, the repetition penalty not below 0");
    if (r->mask && r->mask_stride != 0 && r->mask_stride < (V + 31) / 32)
        return g2i_err(G2_E_ARG, "g2_apply_logit_rules: mask rows of %d words for %d ids", r->mask_stride, V);
    if (r->forbid < -1 || r->forbid >= V) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: forbidden id %d of %d", r->forbid, V);
    if (pick && (!work || !aligned(work, 4))) return g2i_err(G2_E_ARG, "g2_apply_logit_rules: a pick needs the workspace");
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
    int rc = ready();
    if (rc) return rc;
    g2_logits_args a;
    memset(&a, 0, sizeof a);
    a.logits = logits; a.out = out; a.pick = pick; a.part = pick ? work : NULL;
    a.ctx = r->max_ctx ? r->ctx : NULL; a.ctx_len = r->ctx_len; a.max_ctx = r->max_ctx;
    a.bias_id = r->bias_id; a.bias = r->bias; a.n_bias = r->n_bias;
    a.mask = r->mask; a.mask_stride = r->mask_stride; a.forbid = r->forbid;
    a.rows = rows; a.V = V;
    a.repetition = r->repetition > 0.f ? r->repetition : 1.f; a.frequency = r->frequency; a.presence = r->presence;
    a.slice = V > 1024 * G2L_PARTS ? (int)cdiv(V, G2L_PARTS) : 1024;
    a.parts = (int)cdiv(V, a.slice);
    rc = g2i_launch(G2F_LOGITS, (unsigned)(rows * a.parts), 1, 256, &a);
    if (!rc && pick) rc = g2i_launch(G2F_LOGITS_PICK, (unsigned)rows, 1, 64, &a);
    return rc;
}

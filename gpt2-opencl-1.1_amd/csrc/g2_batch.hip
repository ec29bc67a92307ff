/*
 * g2_batch.hip -- several texts at once (included by g2_kernels.hip behind
 * g2_lowbit.hip, whose helpers it uses): causal attention of packed prompts,
 * the 4-bit K/V cache with its single-query attention, beam search.  Layouts
 * and index functions are in g2_batch_plan.h.
 */
namespace gb {
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x4u __attribute__((ext_vector_type(4), aligned(2)));

/* ---------------------------------------------------------- packed rows */

/* How many of the n + 1 ascending starts are at or below row (the same row in
 * every lane): 64 of them probed at a time.  Whatever the list holds, it ends
 * with a count between 0 and n + 1. */
__device__ __forceinline__ int starts_below(const int *start, int n, int row, int lane)
{
    int lo = 0, left = n + 1; /* the count lies in lo .. lo + left */
    for (;;) {
        const int at = g2b_probe(left, lane);
        const bool in = at < left && start[lo + (at < left ? at : 0)] <= row;
        const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
        if (g2b_narrow(&lo, &left, c)) return lo;
    }
}

/* The sequence of a lane's row, `row` being one of row0 .. row1 (the same in
 * every lane); -1 before the first start. */
__device__ __forceinline__ int seq_of_row(const int *start, int n, int row0, int row1, int row, int lane)
{
    int s = starts_below(start, n, row0, lane) - 1;
    for (int at = s + 1; at <= n; at += 64) {
        const int b = at + lane <= n ? start[at + lane] : INT_MAX;
        for (int t = 0; t < 64; ++t) {
            const int v = __builtin_amdgcn_readlane(b, t);
            if (v > row1) return s;
            if (v <= row) s = at + t;
        }
    }
    return s;
}

/* ======================================================================
 * Causal attention of packed prompts
 * ==================================================================== */

/* Eight values as three bf16 parts each, packed in twos: v = p1 + p2 + p3, 8
 * significant bits each, exactly above 2^-102.  The first is cut off (rounded, it
 * would leave the range of finite values at its end), the others are rounded to
 * nearest, so that the products left out, below 2^-21, have either sign. */
__device__ __forceinline__ void parts3(const float (&v)[8], u32x4 (&o)[3])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned a = __float_as_uint(v[2 * e]), b = __float_as_uint(v[2 * e + 1]);
        o[0][e] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        f32x2 r = { v[2 * e] - __uint_as_float(a & 0xffff0000u), v[2 * e + 1] - __uint_as_float(b & 0xffff0000u) };
        const unsigned w = __builtin_bit_cast(unsigned, __builtin_convertvector(r, bf16x2));
        o[1][e] = w;
        r[0] -= __uint_as_float(w << 16);
        r[1] -= __uint_as_float(w & 0xffff0000u);
        o[2][e] = __builtin_bit_cast(unsigned, __builtin_convertvector(r, bf16x2));
    }
}

__device__ __forceinline__ f32x16 mma32(const u32x4 &a, const u32x4 &b, const f32x16 &c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32h(const f16x8 &a, const f16x8 &b, const f32x16 &c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
/* c + a . b, the six products of parts that are above 2^-21 of it, small ones first */
__device__ __forceinline__ f32x16 mma32_parts(const u32x4 (&a)[3], const u32x4 (&b)[3], f32x16 c)
{
    constexpr int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
    for (int p = 0; p < 6; ++p) c = mma32(a[pa[p]], b[pb[p]], c);
    return c;
}

__device__ __forceinline__ float swap_max(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float swap_sum(float v)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

__device__ __forceinline__ int lanes_min_int(int v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o));
    return v;
}

/* Where a work-group's tile of queries is.  With up to 63 sequences the tiles are the
 * sequences' own, deepest first: a tile's depth, its place in its sequence, is what
 * its rows see, so long work begins first, and the starts are read once, an entry
 * to a lane.  With more sequences tiles are cut from all rows in their order, and each
 * row's sequence is searched: full tiles of short texts (64 of 20 rows, 12 heads: 9.3
 * us, 63 in tiles of their own 11.8), but a wave goes through the keys of all its rows'
 * sequences, which is slow where each has many of them (one row behind 700 keys: 63
 * sequences 47 us, 64 of them 332). */
struct prompt_place {
    int first;          /* the tile's first query: in its sequence, or of all */
    int q0, q1, k0, k1; /* the sequence's rows and keys */
    bool own;
};
__device__ __forceinline__ prompt_place prompt_find(const g2_attn_prompt_args &a, int size, int rank, int lane)
{
    prompt_place r = { (a.tiles - 1 - rank) * size, 0, 0, 0, 0, a.S < 64 };
    if (!r.own) return r;
    const int group = a.NH / a.NKV, at = min(lane, a.S);
    const int qs = a.q_start ? a.q_start[at] : at ? a.q_rows : 0, ks = a.k_start ? a.k_start[at] : at ? a.k_rows : 0;
    const int q0 = g2b_clamp(qs, a.q_rows), q1 = __shfl_down(q0, 1), n = lane < a.S ? max(0, q1 - q0) : 0;
    const int tiles = (int)(((unsigned)n * (unsigned)group + (unsigned)size - 1) / (unsigned)size);
    unsigned long long mask = 1;
    int depth;
    if (a.S == 1) depth = __builtin_amdgcn_readfirstlane(tiles) - 1 - rank;
    else {
        depth = -lanes_min_int(-tiles);
        for (;;) {
            --depth;
            mask = __builtin_amdgcn_ballot_w64(tiles > depth);
            const int c = __builtin_popcountll(mask);
            if (depth < 0 || rank < c) break;
            rank -= c;
        }
        mask = __builtin_amdgcn_ballot_w64(mask >> lane & 1 && __builtin_popcountll(mask & ((1ull << lane) - 1)) == rank);
    }
    const int s = depth < 0 ? 0 : __builtin_ctzll(mask);
    r.first = depth * size; /* (below 0: no work is left) */
    r.q0 = __builtin_amdgcn_readlane(qs, s);
    r.q1 = __builtin_amdgcn_readlane(qs, s + 1);
    r.k0 = __builtin_amdgcn_readlane(ks, s);
    r.k1 = __builtin_amdgcn_readlane(ks, s + 1);
    return r;
}

/* One wave takes 32 queries (column l % 32 of a lane) against 32 keys at a time,
 * products transposed: S^T = K Q^T and O^T = V^T P^T with 32x32x16 matrix
 * instructions (lane l supplies A[l % 32][8 (l / 32) ..+7] and B[8 (l / 32)
 * ..+7][l % 32] and gets D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32], r = 0..15).
 * So a lane has its query's scores of 16 of the 32 keys; those of r = 8u .. 8u +
 * 7 are its operand of the second product's step u if V's operand takes the
 * keys in the same order, 16 u + 8 (e / 4) + 4 (l / 32) + e % 4.
 *
 * Queries are the rows' heads that share a key head, row by row: 32
 * of them are fewer rows where heads are grouped, so less is masked.
 *
 * What bounds it: instructions, not memory.  Vector and matrix instructions are under
 * way on 48 % and 41 % of the SIMDs' cycles in the fp32 tiles, 68 % and 28 % in the fp16
 * ones: their times nearly add.  32 x 32 scores are 8 matrix instructions in fp16,
 * 48 in fp32 (six products of parts), beside some 135 and 430 others for
 * exponentials, sums, maxima and parts.  Timed at the forms below. */
template <typename T> struct prompt_op; /* an operand of one instruction, 8 values a lane */
template <> struct prompt_op<float> { u32x4 p[3]; };
template <> struct prompt_op<_Float16> { f16x8 p; };

__device__ __forceinline__ f32x16 prompt_mma(const prompt_op<float> &a, const prompt_op<float> &b, const f32x16 &c) { return mma32_parts(a.p, b.p, c); }
__device__ __forceinline__ f32x16 prompt_mma(const prompt_op<_Float16> &a, const prompt_op<_Float16> &b, const f32x16 &c) { return mma32h(a.p, b.p, c); }
__device__ __forceinline__ void prompt_pack(const float (&v)[8], prompt_op<float> &o) { parts3(v, o.p); }
__device__ __forceinline__ void prompt_pack(const _Float16 (&v)[8], prompt_op<_Float16> &o)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) o.p[e] = v[e];
}

/* Eight values of a row's dims, at any element's address. */
template <typename T> __device__ __forceinline__ void prompt_load_k(T (&x)[8], const T *p)
{
    if constexpr (sizeof(T) == 4) {
        const f32x4 a = *(const f32x4u *)p, b = *(const f32x4u *)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
    } else {
        const f16x8 a = *(const f16x8u *)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = a[e];
    }
}

/* The rows of keys or values from j0 on, up to 32 and below k1, as a buffer:
 * what is read behind the last of them is 0 (everything, unless any). */
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t prompt_rows(const T *p, int j0, int k1, long stride, bool any = true)
{
    const int n = min(32, k1 - j0);
    const unsigned bytes = any ? ((unsigned)(n - 1) * (unsigned)stride + G2B_DH) * (unsigned)sizeof(T) : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void *)(p + (size_t)j0 * stride), (short)0, bytes, 0x00020000);
}
template <typename T> __device__ __forceinline__ void prompt_load_k(T (&x)[8], __amdgpu_buffer_rsrc_t rows, unsigned at)
{
    constexpr int W = 4 * (int)sizeof(T) / 2; /* dwords */
    unsigned w[W];
#pragma unroll
    for (int i = 0; i < W; i += 4) {
        const u32x4 z = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, (int)(at + 4u * (unsigned)i), 0, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i + e] = z[e];
    }
    __builtin_memcpy(x, w, sizeof x);
}
/* Two dims' values of the eight keys that a lane of half g takes in step u (in the
 * second product's order): where the first of them is, from the buffer's begin.
 * (Where the others are is added up for each load: eight registers held for it
 * cost the fp32 tiles a wave.) */
template <typename T> __device__ __forceinline__ unsigned prompt_value_at(int u, int g, int pair, long stride)
{
    return ((unsigned)(16 * u + 4 * g) * (unsigned)stride + 2u * (unsigned)pair) * (unsigned)sizeof(T);
}
/* They stay the pairs that they are in memory. */
template <typename T> struct prompt_pairs;
template <> struct prompt_pairs<float> { unsigned x[16]; };
template <> struct prompt_pairs<_Float16> { unsigned x[8]; };
/* Eight loads of two elements each from a buffer: the first at byte `at`, the others
 * step0 bytes on from one to the next and step1 more from the fourth to the fifth
 * (the same in every lane).  Each address comes from the one before: the multiples of
 * step0 would be held in more scalar registers than there are. */
__device__ __forceinline__ void prompt_next(unsigned &at, int e, unsigned step0, unsigned step1)
{
    at += e == 3 ? step0 + step1 : step0;
    asm volatile("" : "+v"(at));
}
__device__ __forceinline__ void prompt_load8(unsigned (&x)[16], __amdgpu_buffer_rsrc_t rows, unsigned at, unsigned step0, unsigned step1, int)
{
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rows, (int)at, 0, 0));
        x[2 * e] = w[0];
        x[2 * e + 1] = w[1];
        prompt_next(at, e, step0, step1);
    }
}
/* (`even` where pairs of fp16 are at multiples of four bytes, which a load of both asks for) */
__device__ __forceinline__ void prompt_load8(unsigned (&x)[8], __amdgpu_buffer_rsrc_t rows, unsigned at, unsigned step0, unsigned step1, int even)
{
    asm volatile("" : "+v"(at));
    if (even)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = (unsigned)__builtin_amdgcn_raw_buffer_load_b32(rows, (int)at, 0, 0);
            prompt_next(at, e, step0, step1);
        }
    else
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = (unsigned)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rows, (int)at, 0, 0) | (unsigned)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rows, (int)at + 2, 0, 0) << 16;
            prompt_next(at, e, step0, step1);
        }
}
template <typename T> __device__ __forceinline__ void prompt_load_v(prompt_pairs<T> &v, __amdgpu_buffer_rsrc_t rows, unsigned at, long stride, int even)
{
    const unsigned sb = (unsigned)stride * (unsigned)sizeof(T);
    prompt_load8(v.x, rows, at, sb, 4 * sb, even);
}
/* The operand of dim t of the pairs. */
__device__ __forceinline__ void prompt_pack(const prompt_pairs<float> &v, int t, prompt_op<float> &o)
{
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(v.x[2 * e + t]);
    parts3(x, o.p);
}
__device__ __forceinline__ void prompt_pack(const prompt_pairs<_Float16> &v, int t, prompt_op<_Float16> &o)
{
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_perm(v.x[2 * e + 1], v.x[2 * e], t ? 0x07060302u : 0x05040100u);
    o.p = __builtin_bit_cast(f16x8, w);
}

/* The operand of the first or second eight dims of a key. */
__device__ __forceinline__ void prompt_key(const prompt_pairs<float> &k, int h, prompt_op<float> &o)
{
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(k.x[8 * h + e]);
    parts3(x, o.p);
}
__device__ __forceinline__ void prompt_key(const prompt_pairs<_Float16> &k, int h, prompt_op<_Float16> &o)
{
    const u32x4 w = { k.x[4 * h], k.x[4 * h + 1], k.x[4 * h + 2], k.x[4 * h + 3] };
    o.p = __builtin_bit_cast(f16x8, w);
}

/* Scores in units of log 2; not 0, which would make NaN of the masked ones, but so small
 * that no score makes a difference (those below 2^128 then are below 2^-21). */
__device__ __forceinline__ float prompt_unit(float scale)
{
    const float c = fmaxf(fabsf(scale) * 1.44269504f, 0x1p-149f);
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(c)));
}
/* The weight of a state of maximum m beside one of maximum top (an empty one's is
 * -infinity).  (Halves: their difference does not overflow.) */
__device__ __forceinline__ float prompt_factor(float m, float top, float c) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(2.f * ((0.5f * m - 0.5f * top) * c)); }

/* A lane's query: its row's keys, its operands of the four steps of 16 dims, its
 * state, where its output goes. */
template <typename T> struct prompt_query {
    g2b_row keys;
    int row, head; /* (row -1: none) */
    int k0, k1;    /* k0 .. k1 - 1: what the wave's queries see together */
    prompt_op<T> q[4];
    f32x16 o[2];
    float m, l, base; /* base: added to a score in units of log 2, this time */
};

template <typename T>
__device__ __forceinline__ void prompt_start(prompt_query<T> &y, const g2_attn_prompt_args &a, int hk, const prompt_place &place, int off, int lane)
{
    const int group = a.NH / a.NKV, g = lane >> 5, first = place.first + off;
    const unsigned at = (unsigned)(first + (lane & 31));
    y.row = (int)(at / (unsigned)group);
    y.head = hk * group + (int)(at % (unsigned)group);
    if (place.own) {
        y.row += max(place.q0, 0);
        y.keys = g2b_row_keys(y.row, 1, place.q0, place.q1, place.k0, place.k1, a.q_rows, a.k_rows);
    } else {
        const int s = seq_of_row(a.q_start, a.S, (int)((unsigned)first / (unsigned)group), (int)((unsigned)(first + 31) / (unsigned)group), y.row, lane);
        const bool in = s >= 0 && s < a.S;
        const int i = in ? s : 0;
        y.keys = g2b_row_keys(y.row, in, a.q_start[i], a.q_start[i + 1], a.k_start[i], a.k_start[i + 1], a.q_rows, a.k_rows);
    }
    const bool sees = y.keys.end > y.keys.lo; /* (a row that is none of a sequence's has no keys) */
    y.k0 = __builtin_amdgcn_readfirstlane(lanes_min_int(sees ? y.keys.lo : INT_MAX));
    y.k1 = __builtin_amdgcn_readfirstlane(-lanes_min_int(sees ? -y.keys.end : INT_MAX));
    const T *qp = (const T *)a.q + (size_t)min(y.row, a.q_rows - 1) * a.q_stride + y.head * G2B_DH + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        T x[8];
        prompt_load_k(x, qp + 16 * s);
        if (a.scale < 0.f)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = -x[e]; /* (the unit is positive: prompt_unit) */
        prompt_pack(x, y.q[s]);
    }
    if (!y.keys.there) y.row = -1;
    /* (loaded now: a wait for them inside the loop would wait for the keys, too) */
    if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int s = 0; s < 4; ++s) asm volatile("" : "+v"(y.q[s].p));
    y.o[0] = y.o[1] = f32x16{};
    y.m = -INFINITY;
    y.l = 0.f;
}

/* Scores of the keys j0 .. j0 + 31 to weights, with the state's maximum and sum.
 * The state follows the maximum only where a query's grew by more than 2^8: then
 * the sums are scaled down to it, else weights up to 2^8 are as good (fp16
 * weights are 2^6 times that, so that small ones keep their bits: up to 2^14 and
 * a rounding, exact down to 2^-20 of the largest).  Whether it grew is a matter of the
 * difference: products with c have steps of their own, 8 and more from 2^26 on. */
template <typename T>
__device__ __forceinline__ void prompt_follow(prompt_query<T> &y, f32x16 &s, int j0, float c, int g)
{
    if (wave_any(y.keys.lo > j0 || y.keys.end < j0 + 32)) { /* some query does not see all of them */
        const int at = j0 + 4 * g - y.keys.lo, n = y.keys.end - y.keys.lo;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if ((unsigned)(at + 8 * (r / 4) + r % 4) >= (unsigned)n) s[r] = -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = swap_max(top);
    const bool grew = (top - y.m) * c > 8.f; /* (an empty state's maximum is -infinity, and two of them are no growth) */
    if (wave_any(grew)) {
        if (!grew) top = y.m; /* (each query by itself: its result does not depend on its neighbours') */
        const float down = prompt_factor(y.m, top, c);
        y.l *= down;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) y.o[t][r] *= down;
        y.m = top;
    }
    /* The exponent will be one operation on the score: what the rounding of m c adds is
     * one factor for all weights beside the same maximum, 2^(2^-15) at most below 2^10,
     * about what scores of that size have lost in their own sums; weights beside another
     * maximum (earlier ones, other waves') have another.  From 2^10 on the scores
     * become differences now. */
    const bool far = !(fabsf(y.m * c) < 0x1p10f) && y.m != -INFINITY;
    if (wave_any(far)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = far ? s[r] - y.m : s[r];
        y.base = far ? 0.f : y.m;
    } else y.base = y.m;
    y.base = (sizeof(T) == 2 ? 6.f : 0.f) - (y.base == -INFINITY ? 0.f : y.base * c);
}
/* Scores to weights, and their sum. */
template <typename T>
__device__ __forceinline__ void prompt_weights(prompt_query<T> &y, f32x16 &s, float c)
{
    float sum[2] = {};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, y.base));
        sum[r & 1] += s[r];
    }
    y.l += sum[0] + sum[1];
}

/* The operand of the weights of step u.  fp16: rounded to fp16, which adds 1.6e-4 to the
 * 2.0e-4 of the outputs' own rounding (2-norms; 2.6e-4 together).  Two parts of a weight,
 * four more matrix instructions and 24 others to a piece, leave the outputs' alone, and
 * take 262 us for 8001 rows instead of 201, 61 for 51 (16 texts of 25 heads), 22.3 for
 * 21.1 (40 turns). */
__device__ __forceinline__ void prompt_weight_op(const f32x16 &s, int u, prompt_op<float> &p)
{
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s[8 * u + e];
    parts3(x, p.p);
}
__device__ __forceinline__ void prompt_weight_op(const f32x16 &s, int u, prompt_op<_Float16> &p)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) p.p[e] = (_Float16)s[8 * u + e];
}

/* Whether one of eight values is not finite; such values are then 0: they must not
 * meet the weights 0 of queries that do not see them, nor those that are 0 in 32 bits
 * alone.  prompt_odd adds them to the outputs of the queries that see them. */
__device__ __forceinline__ bool prompt_look(const prompt_pairs<float> &v)
{
    float z[2] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        z[0] = fmaf(__uint_as_float(v.x[2 * e]), 0.f, z[0]);
        z[1] = fmaf(__uint_as_float(v.x[2 * e + 1]), 0.f, z[1]);
    }
    return wave_any(z[0] + z[1] != 0.f);
}
__device__ __forceinline__ bool prompt_look(const prompt_pairs<_Float16> &v)
{
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 zero = { (_Float16)0.f, (_Float16)0.f };
    f16x2 z = zero;
#pragma unroll
    for (int e = 0; e < 8; ++e) z = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, v.x[e]), zero, z);
    return wave_any((__builtin_bit_cast(unsigned, z) & 0x7FFF7FFFu) != 0);
}
__device__ __forceinline__ void prompt_clean(prompt_pairs<float> &v)
{
#pragma unroll
    for (int e = 0; e < 16; ++e) v.x[e] = __builtin_isfinite(__uint_as_float(v.x[e])) ? v.x[e] : 0u;
}
__device__ __forceinline__ void prompt_clean(prompt_pairs<_Float16> &v)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if ((v.x[e] & 0x7C00u) == 0x7C00u) v.x[e] &= 0xFFFF0000u;
        if ((v.x[e] & 0x7C000000u) == 0x7C000000u) v.x[e] &= 0xFFFFu;
    }
}
/* Pieces of 32 keys j0 .. with such values: the first, and what follows the last. */
struct prompt_span {
    int lo, end;
};
__device__ __forceinline__ void prompt_note(prompt_span &s, bool odd, int j0)
{
    s.lo = odd ? min(s.lo, j0) : s.lo;
    s.end = odd ? max(s.end, j0 + 32) : s.end;
}
/* What is not finite among the eight dims of a query's output from d on, for the keys of
 * the span that it sees; at the end, because sums that held it would be scaled by 0 where later
 * scores are far larger. */
template <typename T>
__device__ __forceinline__ void prompt_odd(f32x4 (&x)[2], const g2b_row &keys, const T *v, long stride, prompt_span s, int d)
{
    const int end = min(s.end, keys.end);
#pragma unroll 4
    for (int j = max(s.lo, keys.lo); j < end; ++j) {
        T z[8];
        prompt_load_k(z, v + (size_t)j * stride + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e & 1][e >> 1] += __builtin_isfinite((float)z[e]) ? 0.f : (float)z[e];
    }
}

/* Eight dims of a row: quads of registers, of tile 0 and 1, side by side. */
template <typename T> __device__ __forceinline__ void prompt_store(T *p, const f32x4 &a, const f32x4 &b)
{
    if constexpr (sizeof(T) == 2)
        *(f16x8u *)p = f16x8u{ (_Float16)a[0], (_Float16)b[0], (_Float16)a[1], (_Float16)b[1], (_Float16)a[2], (_Float16)b[2], (_Float16)a[3], (_Float16)b[3] };
    else {
        *(f32x4u *)p = f32x4{ a[0], b[0], a[1], b[1] };
        *(f32x4u *)(p + 4) = f32x4{ a[2], b[2], a[3], b[3] };
    }
}

template <typename T>
__device__ __forceinline__ void prompt_out(const prompt_query<T> &y, const g2_attn_prompt_args &a, float l, int g, const T *vp, prompt_span odd)
{
    const float one = 1.f / l;
    T *out = (T *)a.out + (size_t)y.row * a.out_stride + y.head * G2B_DH + 8 * g;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        f32x4 v[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[t][e] = y.keys.end > y.keys.lo ? y.o[t][4 * q + e] * one : 0.f;
        if (odd.lo < odd.end) prompt_odd(v, y.keys, vp, a.kv_stride, odd, 16 * q + 8 * g);
        prompt_store(out + 16 * q, v[0], v[1]);
    }
}

/* ---- few queries: a work-group takes 32 of them, its four waves every fourth 32
 * keys each, whose rows they read as the operands that they are (a key's dims
 * 16 bytes at a time, a value's dims side by side, so that eight loads are
 * eight keys of a dim); the waves' states meet at the end.  Each wave converts its
 * own keys, for 32 queries only: the price of having four times the waves.
 * 1001 rows of 12 heads 23 us in fp32 (68 TFLOP/s of useful products; a tile of
 * 128 queries: 75) and 12 in fp16; 40 turns of 20 to 60 rows behind 700 keys, 16
 * heads on 4, fp16: 22.2 us; one text of 17 rows 5.5, a launch's own time.
 * Eight waves to a work-group instead of four: 50 us where this takes 40 (1001
 * rows, 25 heads). */
template <typename T, int KW, int EVEN>
__device__ void prompt_split_impl(const g2_attn_prompt_args &a)
{
    __shared__ float red[KW][34][64];
    __shared__ prompt_span odds[KW];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    int hk;
    long tile;
    g2b_prompt_item(blockIdx.x, a.NKV, a.tiles, &hk, &tile);
    prompt_query<T> y;
    const prompt_place place = prompt_find(a, 32, a.tiles - 1 - (int)tile, lane);
    if (place.first < 0) return;
    prompt_start(y, a, hk, place, 0, lane);
    const float c = prompt_unit(a.scale);
    const long stride = a.kv_stride;
    const T *kp = (const T *)a.k + hk * G2B_DH, *vp = (const T *)a.v + hk * G2B_DH;
    T k[4][8];
    prompt_pairs<T> v[2]; /* of the two steps */
    const unsigned at[2] = { prompt_value_at<T>(0, g, lane & 31, stride), prompt_value_at<T>(1, g, lane & 31, stride) };
    const unsigned at_key = ((unsigned)(lane & 31) * (unsigned)stride + 8u * (unsigned)g) * (unsigned)sizeof(T);
    auto load_k = [&](int j0) {
        if constexpr (EVEN) {
            const __amdgpu_buffer_rsrc_t rows = prompt_rows(kp, min(j0, y.k1 - 1), y.k1, stride, j0 < y.k1);
#pragma unroll
            for (int s = 0; s < 4; ++s) prompt_load_k(k[s], rows, at_key + 16u * (unsigned)s * (unsigned)sizeof(T));
        } else {
            const T *p = kp + (size_t)min(j0 + (lane & 31), y.k1 - 1) * stride + 8 * g;
#pragma unroll
            for (int s = 0; s < 4; ++s) prompt_load_k(k[s], p + 16 * s);
        }
    };
    auto load_v = [&](int j0) {
        const __amdgpu_buffer_rsrc_t rows = prompt_rows(vp, min(j0, y.k1 - 1), y.k1, stride, j0 < y.k1);
#pragma unroll
        for (int u = 0; u < 2; ++u) prompt_load_v(v[u], rows, at[u], stride, EVEN);
    };
    int j0 = y.k0 < y.k1 ? y.k0 + 32 * w : y.k1;
    prompt_span odd = { INT_MAX, 0 };
    if (j0 < y.k1) { load_k(j0); load_v(j0); }
    for (; j0 < y.k1; j0 += 32 * KW) {
        const int j1 = j0 + 32 * KW;
        f32x16 s = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            prompt_op<T> x;
            prompt_pack(k[i], x);
            s = prompt_mma(x, y.q[i], s);
        }
        /* (always, behind the last ones of no bytes: with a branch around keys or values
         * what waits for the ones waits for the others, too) */
        load_k(j1);
        prompt_follow(y, s, j0, c, g);
        prompt_weights(y, s, c);
        const bool odd0 = prompt_look(v[0]), odd1 = prompt_look(v[1]);
        if (odd0 || odd1) {
            prompt_clean(v[0]);
            prompt_clean(v[1]);
            prompt_note(odd, true, j0);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            prompt_op<T> p, x;
            prompt_weight_op(s, u, p);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                prompt_pack(v[u], t, x);
                y.o[t] = prompt_mma(x, p, y.o[t]);
            }
        }
        load_v(j1);
    }
    y.l = swap_sum(y.l);
    /* the waves' parts meet; the first four waves write a quarter of the dims each */
    if (lane == 0) odds[w] = odd;
    red[w][0][lane] = y.m;
    red[w][1][lane] = y.l;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) red[w][2 + 16 * t + r][lane] = y.o[t][r];
    __syncthreads();
    if (y.row < 0 || w >= 4) return;
    float top = -INFINITY, part[KW], l = 0.f;
#pragma unroll
    for (int i = 0; i < KW; ++i) top = fmaxf(top, red[i][0][lane]);
#pragma unroll
    for (int i = 0; i < KW; ++i) {
        part[i] = prompt_factor(red[i][0][lane], top, c);
        l = fmaf(red[i][1][lane], part[i], l);
        odd.lo = min(odd.lo, odds[i].lo);
        odd.end = max(odd.end, odds[i].end);
    }
    const float one = 1.f / l;
    T *out = (T *)a.out + (size_t)y.row * a.out_stride + y.head * G2B_DH + 8 * g;
    f32x4 x[2] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int j = 0; j < KW; ++j) x[t][e] = fmaf(red[j][2 + 16 * t + 4 * w + e][lane], part[j], x[t][e]);
            x[t][e] = y.keys.end > y.keys.lo ? x[t][e] * one : 0.f;
        }
    if (odd.lo < odd.end) prompt_odd(x, y.keys, vp, stride, odd, 16 * w + 8 * g);
    prompt_store(out + 16 * w, x[0], x[1]);
}
/* (f16_odd: pairs of values at odd multiples of two bytes.  A kernel of its own: beside
 * a branch between the two kinds of loads the wait for the keys was one for the values,
 * too.) */
#define PROMPT_SPLIT(NAME, T, KW, EVEN)                                                                                \
    extern "C" __global__ __launch_bounds__(64 * KW) __attribute__((amdgpu_waves_per_eu(2)))                           \
    void NAME(const g2_attn_prompt_args a) { prompt_split_impl<T, KW, EVEN>(a); }
PROMPT_SPLIT(g2k_prompt_split_f32, float, 4, 1)
PROMPT_SPLIT(g2k_prompt_split_f16, _Float16, 4, 1)
PROMPT_SPLIT(g2k_prompt_split_f16_odd, _Float16, 4, 0)

/* ---- many queries: a work-group takes 128 of them, 32 a wave, and its waves
 * read KT times 32 keys and values together, once, as operands in LDS: unit
 * (part, step, lane) of 16 bytes is what the lane reads of it, so that reads and
 * writes are both rows of units.  Two stages: the next keys are on their way from
 * memory while the products of these run, and one barrier stands between.  Of 32
 * keys two waves bring the keys, two the values (a step each), in turns.
 * With KW = 2 two such groups take every other piece of the same queries' keys,
 * and their states meet at the end.
 * fp32, 16 texts of 100 to 1023 rows, 25 heads: 153 us, 132 TFLOP/s of useful
 * products (790 of bf16 ones; a large library product reaches 1223), three
 * work-groups to a CU by registers and LDS; four waves a group, one piece.
 * fp16, one text of 8001 rows, 16 heads on 4: 193 us, 680 TFLOP/s, with vector
 * instructions on 68 % and matrix instructions on 28 % of the cycles; one group of
 * waves takes 235.  Two groups of fp32 waves: 212 us for 153.
 * Tried beside it: the next keys' scores among this piece's exponentials (fp32 171,
 * fp16 up to 1.5 times as long: registers), no LDS, each wave by itself (187),
 * two waves a SIMD with all operands in registers (175). */
template <typename T, int KT, int KW>
__device__ void prompt_tile_impl(const g2_attn_prompt_args &a)
{
    constexpr int P = sizeof(T) == 4 ? 3 : 1, UNITS = P * 256; /* of 32 keys, and of their values */
    __shared__ u32x4 all[KW][2][KT][2 * UNITS];
    __shared__ int range[4][2], odds[KW][2][KT][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3, kw = wave >> 2;
    const int g = lane >> 5, m = lane & 31;
    auto &lds = all[kw];
    auto &odd = odds[kw];
    int hk;
    long tile;
    g2b_prompt_item(blockIdx.x, a.NKV, a.tiles, &hk, &tile);
    prompt_query<T> y;
    const prompt_place place = prompt_find(a, 128, a.tiles - 1 - (int)tile, lane);
    if (place.first < 0) return;
    prompt_start(y, a, hk, place, 32 * w, lane);
    if (lane == 0 && kw == 0) { range[w][0] = y.k0; range[w][1] = y.k1; }
    __syncthreads();
    const int low = __builtin_amdgcn_readfirstlane(min(min(range[0][0], range[1][0]), min(range[2][0], range[3][0])));
    const int high = __builtin_amdgcn_readfirstlane(max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1])));
    const int k0 = g2b_span_begin(low, high), k1 = g2b_span_end(low, high);
    const float c = prompt_unit(a.scale);
    const long stride = a.kv_stride;
    const T *kp = (const T *)a.k + hk * G2B_DH, *vp = (const T *)a.v + hk * G2B_DH;
    /* This lane's share of 32 keys: 16 dims of a key, or two dims of eight keys. */
    prompt_pairs<T> x[KT];
    auto brings_keys = [&](int i) { return ((w >> 1) ^ i) & 1; };
    const int chunk = 4 * (w & 1) + 2 * g;
    const unsigned sb = (unsigned)stride * (unsigned)sizeof(T);
    const unsigned at_key = (unsigned)m * sb + 8 * (unsigned)chunk * (unsigned)sizeof(T), at_value = prompt_value_at<T>(w & 1, g, m, stride);
    auto load = [&](int j0) {
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const int j = min(j0 + 32 * i, k1 - 1); /* (keys behind the last are masked) */
            const bool keys = brings_keys(i);
            /* fp32: either way eight loads of a pair into the same registers.  Where a
             * wave's keys were four wide loads and its values eight others, both
             * meeting in them, 16 texts of 100 to 1023 rows took 163 us, now 153;
             * fp16 keys in pairs take 274 us for 8001 rows, which take 193. */
            if constexpr (P == 3) prompt_load8(x[i].x, prompt_rows(keys ? kp : vp, j, k1, stride), keys ? at_key : at_value, keys ? 8u : sb, keys ? 0u : 4 * sb, 0);
            else if (keys) {
                const T *p = kp + (size_t)j * stride + (size_t)min(m, k1 - j - 1) * stride + 8 * chunk;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4 z = __builtin_bit_cast(u32x4, *(const f16x8u *)(p + 8 * h));
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i].x[4 * h + e] = z[e];
                }
            } else prompt_load_v(x[i], prompt_rows(vp, j, k1, stride), at_value, stride, a.even);
        }
    };
    auto put = [&](u32x4 *p, const prompt_op<T> &z) {
        if constexpr (P == 3) {
#pragma unroll
            for (int i = 0; i < 3; ++i) p[256 * i] = z.p[i];
        } else *p = __builtin_bit_cast(u32x4, z.p);
    };
    auto stage = [&](int b) {
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            prompt_op<T> z;
            if (brings_keys(i)) {
                prompt_key(x[i], 0, z);
                put(lds[b][i] + chunk * 32 + m, z);
                prompt_key(x[i], 1, z);
                put(lds[b][i] + chunk * 32 + 32 + m, z);
            } else {
                const bool any = prompt_look(x[i]);
                if (any) prompt_clean(x[i]);
                if (lane == 0) odd[b][i][w & 1] = any;
                prompt_pack(x[i], 0, z);
                put(lds[b][i] + UNITS + (w & 1) * 64 + lane, z);
                prompt_pack(x[i], 1, z);
                put(lds[b][i] + UNITS + 128 + (w & 1) * 64 + lane, z);
            }
        }
    };
    auto fetch = [&](const u32x4 *p, prompt_op<T> &z) {
        if constexpr (P == 3) {
#pragma unroll
            for (int i = 0; i < 3; ++i) z.p[i] = p[256 * i];
        } else z.p = __builtin_bit_cast(f16x8, *p);
    };
    /* (the groups of four waves take every KW-th piece; all go through as many barriers) */
    constexpr int STEP = 32 * KT * KW;
    int j0 = k0 + 32 * KT * kw, b = 0;
    prompt_span any = { INT_MAX, 0 };
    if (j0 < k1) {
        load(j0);
        stage(0);
    }
    __syncthreads();
    for (int left = k1 - k0; KW == 1 ? j0 < k1 : left > 0; left -= STEP, j0 += STEP, b ^= 1) {
        const bool more = j0 + STEP < k1;
        if (more) load(j0 + STEP);
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const int j = j0 + 32 * i;
            if (j >= y.k1 || j + 32 <= y.k0) continue; /* (none of the wave's queries sees any of them) */
            const u32x4 *kd = lds[b][i] + lane, *vd = kd + UNITS;
            f32x16 s = {};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                prompt_op<T> z;
                fetch(kd + 64 * t, z);
                s = prompt_mma(z, y.q[t], s);
            }
            prompt_follow(y, s, j, c, g);
            prompt_weights(y, s, c);
            prompt_note(any, __builtin_amdgcn_readfirstlane(odd[b][i][0] | odd[b][i][1]), j);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                prompt_op<T> p, z;
                prompt_weight_op(s, u, p);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    fetch(vd + 128 * t + 64 * u, z);
                    y.o[t] = prompt_mma(z, p, y.o[t]);
                }
            }
        }
        if (more) stage(b ^ 1);
        __syncthreads();
    }
    y.l = swap_sum(y.l);
    if constexpr (KW > 1) { /* the groups' states meet where the keys were */
        static_assert(KW == 2 && sizeof(all) >= 34 * 256 * sizeof(float), "one state a query in LDS");
        float *red = (float *)all + w * 64 + lane;
        if (kw) {
            if (lane == 0) { range[w][0] = any.lo; range[w][1] = any.end; }
            red[0] = y.m;
            red[256] = y.l;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) red[256 * (2 + 16 * t + r)] = y.o[t][r];
        }
        __syncthreads();
        if (kw) return;
        any.lo = min(any.lo, __builtin_amdgcn_readfirstlane(range[w][0]));
        any.end = max(any.end, __builtin_amdgcn_readfirstlane(range[w][1]));
        const float top = fmaxf(y.m, red[0]), mine = prompt_factor(y.m, top, c), other = prompt_factor(red[0], top, c);
        y.l = y.l * mine + red[256] * other;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) y.o[t][r] = y.o[t][r] * mine + red[256 * (2 + 16 * t + r)] * other;
    }
    if (y.row >= 0) prompt_out(y, a, y.l, g, vp, any);
}
#define PROMPT_TILE(NAME, T, KT, KW, WAVES)                                                                            \
    extern "C" __global__ __launch_bounds__(256 * KW) __attribute__((amdgpu_waves_per_eu(WAVES)))                      \
    void NAME(const g2_attn_prompt_args a) { prompt_tile_impl<T, KT, KW>(a); }
PROMPT_TILE(g2k_prompt_tile_f32, float, 1, 1, 3)
PROMPT_TILE(g2k_prompt_tile_f16, _Float16, 2, 1, 4)
PROMPT_TILE(g2k_prompt_duo_f16, _Float16, 2, 2, 4)

/* ======================================================================
 * 4-bit K/V cache: each position, head and 32 dims on their own, codes and
 * scale as those of the 4-bit weights.
 * ==================================================================== */

/* A wave takes 8 rows of keys or values of a head, eight lanes of 8 dims to a
 * row, neighbouring waves neighbouring heads.  Bound by memory: 7 bytes read for
 * one written; 16 texts of 100 to 1023 rows, 25 heads, in 30 us, 4.3 TB/s (a large
 * copy: 4.8), one token of 8 texts in 3.6. */
template <typename T>
__device__ void kv4_append_impl(const g2_kv4_append_args &a)
{
    const int lane = threadIdx.x & 63, part = lane & 7;
    const long wave = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)(wave % a.NKV), kv = (int)(wave / a.NKV % 2);
    const long r0 = wave / a.NKV / 2 * 8;
    if (r0 >= a.rows) return;
    const int row = (int)r0 + (lane >> 3);
    typedef T t8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const t8 raw = *(const t8 *)((const T *)(kv ? a.v : a.k) + (size_t)min(row, a.rows - 1) * a.stride + h * G2B_DH + 8 * part);
    int s, q0, q1;
    if (a.row_start) {
        s = seq_of_row(a.row_start, a.S, (int)r0, (int)r0 + 7, row, lane);
        const int i = clampi(s, 0, a.S - 1);
        q0 = a.row_start[i];
        q1 = min(a.row_start[i + 1], a.rows);
    } else {
        s = row / a.per;
        q0 = s * a.per;
        q1 = q0 + a.per;
    }
    const bool there = s >= 0 && s < a.S && row >= q0 && row < q1 && row < a.rows;
    const long p = there ? (long)(a.pos ? a.pos[s] : a.start) + ((long)row - q0) : -1;
    float x[8];
    unsigned amax = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = (float)raw[e];
        const unsigned u = __float_as_uint(x[e]) & 0x7FFFFFFF;
        amax = u > amax ? u : amax;
    }
    amax = q4_group_max(amax, 32);
    const uint16_t sc = q4_scale(amax);
    const unsigned codes = q4_codes(x, bf16_f(sc));
    if (p < 0 || p >= a.max_seq) return;
    unsigned char *t = a.cache + g2b_tile_at(a.NKV, a.tiles, s, h, p / G2B_TILE);
    const int i = (int)(p % G2B_TILE);
    *(unsigned *)(t + g2b_code_at(kv, i) + 4 * part) = codes;
    if (!(part & 3)) *(uint16_t *)(t + g2b_scale_at(kv, i) + 2 * (part >> 2)) = sc;
}
G2K void g2k_kv4_append_f32(const g2_kv4_append_args a) { kv4_append_impl<float>(a); }
G2K void g2k_kv4_append_f16(const g2_kv4_append_args a) { kv4_append_impl<_Float16>(a); }

/* One thread per four dims of a position, keys and values, in the order of the
 * output, which does not stay in the L2.  30 us for what the above puts down. */
G2K void g2k_kv4_read(const g2_kv4_read_args a)
{
    const unsigned quads = (unsigned)a.NKV * (G2B_DH / 4);
    const long n = (long)a.S * a.T * quads;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += gridDim.x * 256l) {
        const long row = n <= UINT32_MAX ? (unsigned)i / quads : i / quads;
        const unsigned e = (unsigned)(i - row * quads), d = e % (G2B_DH / 4) * 4;
        const int h = (int)(e / (G2B_DH / 4)), s = a.S == 1 ? 0 : (int)((unsigned)row / (unsigned)a.T);
        const int p = a.start + (int)(row - (long)s * a.T);
        if (p >= kv8_length(a.len, a.T_kv, s)) continue;
        const int from = a.origin ? a.origin[(size_t)(unsigned)s * (unsigned)a.max_seq + (unsigned)p] : s;
        if ((unsigned)from >= (unsigned)a.S) continue;
        const unsigned char *t = a.cache + g2b_tile_at(a.NKV, a.tiles, from, h, p / G2B_TILE);
        f32x4 v[2];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const unsigned c = *(const uint16_t *)(t + g2b_code_at(kv, p % G2B_TILE) + d / 2);
            const float sc = bf16_f(*(const uint16_t *)(t + g2b_scale_at(kv, p % G2B_TILE) + d / 32 * 2));
            const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
            v[kv] = f32x4{ lo[0] * sc, lo[1] * sc, hi[0] * sc, hi[1] * sc };
        }
        __builtin_nontemporal_store(v[0], (f32x4u *)(a.k + 4 * i));
        __builtin_nontemporal_store(v[1], (f32x4u *)(a.v + 4 * i));
    }
}

/* ---- single-query attention.  A wave takes U times 64 / LP positions at a time,
 * LP lanes of DL = 64 / LP dims to a position, for G query heads that share a key
 * head: codes are used where they were loaded, a score is the sum over LP lanes,
 * and each position slot keeps a running maximum and sum of its own, which
 * follows the maximum only where it grew by more than 2^8.  The slots meet once,
 * at the end: over the lanes, over the waves in LDS, and over the parts of a long
 * sequence in a second launch.  The next positions' loads go out before the last
 * ones' sums.
 * 72 bytes a position and head hold 128 numbers: reading them at the speed of
 * memory leaves few instructions for each, so codes become values by one conversion
 * a pair, scales enter once a position, and the work is spread for its latency
 * where it is small.  48 texts of 256 to 1024 positions, 25 heads: 15.2 us, 3.7 TB/s;
 * 8 beams of 901 through their table 6.3; 50001 positions of 4 heads, 16 queries:
 * 13.4 with the second launch, which is 3.9 of it. */
template <int W, int U> struct kv4_in {
    unsigned k[U][W], v[U][W];
    unsigned ks[U], vs[U]; /* bf16 */
    bool there[U];
};

template <int G, int LP, int NW, int U, bool ORIGIN>
__device__ void kv4_attn_impl(const g2_kv4_attn_args &a)
{
    constexpr int DL = 64 / LP, SLOTS = 64 / LP, W = DL / 8, STEP = SLOTS * U;
    typedef unsigned words __attribute__((ext_vector_type(W)));
    __shared__ float part[NW][G][G2B_PART_FLOATS];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slot = lane / LP, d0 = DL * (lane % LP);
    const unsigned split = blockIdx.x % (unsigned)a.splits, rest = blockIdx.x / (unsigned)a.splits;
    const int ch = (int)(rest % (unsigned)a.chunks), hk = (int)(rest / (unsigned)a.chunks % (unsigned)a.NKV);
    const int s = (int)(rest / (unsigned)a.chunks / (unsigned)a.NKV);
    const int group = a.NH / a.NKV, h0 = hk * group + ch * a.heads, nh = min(a.heads, group - ch * a.heads);
    const int len = __builtin_amdgcn_readfirstlane(kv8_length(a.len, a.T_kv, s));
    const int p0 = (int)split * a.span * G2B_TILE, p1 = min(len, p0 + a.span * G2B_TILE);
    const unsigned char *cache = a.cache + g2b_tile_at(a.NKV, a.tiles, s, hk, 0);
    const size_t seq = (size_t)a.NKV * (unsigned)a.tiles * G2B_TILE_BYTES;
    const unsigned code0 = (unsigned)d0 / 2, scale0 = (unsigned)d0 / 32 * 2;
    int from[U]; /* of the step that is loaded next */
    auto origins = [&](int b) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = b + u * SLOTS + slot;
            from[u] = p < p1 ? a.origin[(size_t)(unsigned)s * (unsigned)a.max_seq + (unsigned)p] : -1;
        }
    };
    typedef kv4_in<W, U> in_t;
    auto load = [&](in_t &x, int b) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int bu = min(b + u * SLOTS, p1 - 1) / SLOTS * SLOTS, p = b + u * SLOTS + slot, i = (bu + slot) % G2B_TILE;
            const unsigned char *t;
            if constexpr (ORIGIN) {
                x.there[u] = (unsigned)from[u] < (unsigned)a.S;
                t = a.cache + g2b_tile_at(a.NKV, a.tiles, 0, hk, bu / G2B_TILE) + (size_t)(x.there[u] ? (unsigned)from[u] : 0u) * seq;
            } else {
                x.there[u] = p < p1;
                t = cache + (size_t)(unsigned)(bu / G2B_TILE) * G2B_TILE_BYTES;
            }
            const words *kp = (const words *)(t + (g2b_code_at(0, i) + code0)), *vp = (const words *)(t + (g2b_code_at(1, i) + code0));
            words k, v;
            if constexpr (ORIGIN) { k = *kp; v = *vp; }
            else { k = __builtin_nontemporal_load(kp); v = __builtin_nontemporal_load(vp); }
#pragma unroll
            for (int j = 0; j < W; ++j) { x.k[u][j] = k[j]; x.v[u][j] = v[j]; }
            x.ks[u] = *(const uint16_t *)(t + (g2b_scale_at(0, i) + scale0));
            x.vs[u] = *(const uint16_t *)(t + (g2b_scale_at(1, i) + scale0));
        }
    };
    float q[G][DL], o[G][DL], m[G], l[G];
    const float qf = a.scale * 1.44269504f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const float *p = a.q + (size_t)(unsigned)s * (unsigned)a.q_stride + (h0 + min(i, nh - 1)) * G2B_DH + d0;
#pragma unroll
        for (int e = 0; e < DL; e += 4) {
            const f32x4 v = *(const f32x4u *)(p + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) q[i][e + j] = v[j];
        }
    }
    in_t next;
    int b = p0 + STEP * w;
    if (b < p1) {
        if constexpr (ORIGIN) origins(b);
        load(next, b);
        if constexpr (ORIGIN) origins(b + STEP * NW);
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
        for (int e = 0; e < DL; ++e) { q[i][e] *= qf; o[i][e] = 0.f; }
        m[i] = -INFINITY;
        l[i] = 0.f;
    }
    for (; b < p1; b += STEP * NW) {
        const in_t x = next;
        if (b + STEP * NW < p1) {
            load(next, b + STEP * NW);
            if constexpr (ORIGIN) origins(b + 2 * STEP * NW);
        }
        float sc[U][G];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < G; ++j) sc[u][j] = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                float v[8];
                q4_values(x.k[u][i], 1.f, v);
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sc[u][j] = fmaf(q[j][8 * i + e], v[e], sc[u][j]);
            }
        }
        bool grew = false;
        float top[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            top[j] = m[j];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float d = sc[u][j] * __uint_as_float(x.ks[u] << 16);
                d += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(d), 0xB1, 0xF, 0xF, false)); /* lanes 1 0 3 2 */
                if (LP == 4) d += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(d), 0x4E, 0xF, 0xF, false));
                sc[u][j] = x.there[u] ? d : -INFINITY;
                top[j] = fmaxf(top[j], sc[u][j]);
            }
            grew |= top[j] > m[j] + 8.f; /* (an empty state's maximum is -infinity) */
        }
        if (wave_any(grew)) {
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const float f = kv8_factor(m[j], top[j]);
                m[j] = top[j];
                l[j] *= f;
#pragma unroll
                for (int e = 0; e < DL; ++e) o[j][e] *= f;
            }
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const float base = m[j] == -INFINITY ? 0.f : m[j];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = __builtin_amdgcn_exp2f(sc[u][j] - base);
                l[j] += p;
                sc[u][j] = p * __uint_as_float(x.there[u] ? x.vs[u] << 16 : 0u);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                float v[8];
                q4_values(x.v[u][i], 1.f, v);
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[j][8 * i + e] = fmaf(sc[u][j], v[e], o[j][8 * i + e]);
            }
    }
    /* the wave's position slots: each step halves the dims that a lane keeps */
#pragma unroll
    for (int i = 0; i < G; ++i) {
        float top = slots_max(m[i]);
        if (LP == 2) top = fmaxf(top, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(top), 0x4E, 0xF, 0xF, false)));
        const float f = kv8_factor(m[i], top);
        float sum = l[i] * f;
        if (LP == 2) sum += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(sum), 0x4E, 0xF, 0xF, false));
        sum += lane_xor4(sum);
        sum += lane_xor8(sum);
        sum = lane_fold16(sum, sum);
        sum = lane_fold32(sum, sum);
        float *v = o[i];
#pragma unroll
        for (int e = 0; e < DL; ++e) v[e] *= f;
#pragma unroll
        for (int e = 0; e < DL / 2; ++e) v[e] = lane_fold32(v[e], v[e + DL / 2]);
#pragma unroll
        for (int e = 0; e < DL / 4; ++e) v[e] = lane_fold16(v[e], v[e + DL / 4]);
#pragma unroll
        for (int e = 0; e < DL / 8; ++e) {
            const float lo = v[e] + lane_xor8(v[e]), hi = v[e + DL / 8] + lane_xor8(v[e + DL / 8]);
            v[e] = lane & 8 ? hi : lo;
        }
#pragma unroll
        for (int e = 0; e < DL / 16; ++e) {
            const float lo = v[e] + lane_xor4(v[e]), hi = v[e + DL / 16] + lane_xor4(v[e + DL / 16]);
            v[e] = lane & 4 ? hi : lo;
        }
        if (LP == 2) {
            const float lo = v[0] + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v[0]), 0x4E, 0xF, 0xF, false));
            const float hi = v[1] + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v[1]), 0x4E, 0xF, 0xF, false));
            v[0] = lane & 2 ? hi : lo;
        }
        if (lane == 0) { part[w][i][0] = top; part[w][i][1] = sum; }
        part[w][i][2 + d0 + slot] = v[0];
    }
    __syncthreads();
    for (int i = w; i < nh; i += NW) {
        float top = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
        for (int j = 0; j < NW; ++j) top = fmaxf(top, part[j][i][0]);
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const float f = kv8_factor(part[j][i][0], top);
            sum = fmaf(part[j][i][1], f, sum);
            y = fmaf(part[j][i][2 + lane], f, y);
        }
        if (a.splits > 1) {
            float *r = a.part + (((size_t)(unsigned)s * (unsigned)a.NH + (unsigned)(h0 + i)) * (unsigned)a.splits + split) * G2B_PART_FLOATS;
            if (lane == 0) { r[0] = top; r[1] = sum; }
            r[2 + lane] = y;
        } else
            a.out[(size_t)(unsigned)s * (unsigned)a.out_stride + (h0 + i) * G2B_DH + lane] = sum == 0.f ? 0.f : y / sum;
    }
}
#define KV4_ATTN(G, LP, NW, U)                                                                                         \
    extern "C" __global__ __launch_bounds__(64 * NW) void g2k_kv4_attn##G##_##NW(const g2_kv4_attn_args a)            \
    { kv4_attn_impl<G, LP, NW, U, false>(a); }                                                                         \
    extern "C" __global__ __launch_bounds__(64 * NW) void g2k_kv4_attn##G##_##NW##_o(const g2_kv4_attn_args a)        \
    { kv4_attn_impl<G, LP, NW, U, true>(a); }
KV4_ATTN(1, 2, 1, 2)
KV4_ATTN(1, 2, 4, 2)
KV4_ATTN(1, 2, 8, 2)
KV4_ATTN(2, 4, 4, 2)
KV4_ATTN(2, 4, 8, 2)
KV4_ATTN(4, 4, 4, 2)
KV4_ATTN(4, 4, 8, 2)

/* Joins the parts of a head: four waves of eight parts each, all their loads at
 * once, then the waves. */
G2K void g2k_kv4_join(const g2_kv4_attn_args a)
{
    __shared__ float part[4][G2B_PART_FLOATS];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float *r = a.part + (size_t)blockIdx.x * (unsigned)a.splits * G2B_PART_FLOATS;
    float m[G2B_SPLITS / 4], l[G2B_SPLITS / 4], v[G2B_SPLITS / 4], top = -INFINITY, o = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < G2B_SPLITS / 4; ++i) {
        const int n = w * (G2B_SPLITS / 4) + i;
        const float *p = r + min(n, a.splits - 1) * G2B_PART_FLOATS;
        m[i] = p[0];
        l[i] = p[1];
        v[i] = p[2 + lane];
        if (n >= a.splits) m[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < G2B_SPLITS / 4; ++i) top = fmaxf(top, m[i]);
#pragma unroll
    for (int i = 0; i < G2B_SPLITS / 4; ++i) {
        if (w * (G2B_SPLITS / 4) + i >= a.splits) continue;
        const float f = kv8_factor(m[i], top);
        sum = fmaf(l[i], f, sum);
        o = fmaf(v[i], f, o);
    }
    if (lane == 0) { part[w][0] = top; part[w][1] = sum; }
    part[w][2 + lane] = o;
    __syncthreads();
    if (w) return;
    top = fmaxf(fmaxf(part[0][0], part[1][0]), fmaxf(part[2][0], part[3][0]));
    sum = o = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = kv8_factor(part[i][0], top);
        sum = fmaf(part[i][1], f, sum);
        o = fmaf(part[i][2 + lane], f, o);
    }
    const unsigned s = blockIdx.x / (unsigned)a.NH, h = blockIdx.x - s * (unsigned)a.NH;
    a.out[(size_t)s * (unsigned)a.out_stride + h * G2B_DH + lane] = sum == 0.f ? 0.f : o / sum;
}

/* ======================================================================
 * Beam search
 * ==================================================================== */

/* Candidates are few once a bound is known that n of them reach.  One is the
 * least of the greatest of G >= n groups: of values that are spread over the
 * groups, about G (1 + 1/2 + ... + 1/G) reach it (54 for 16).  What reaches it is
 * put down in LDS, in any order, and each candidate counts those above it.
 * A row is read once, its ids in registers meanwhile.  128 rows of 50257 ids: 12.8 us
 * (25.7 MB, 2.0 TB/s: a work-group's sixteen waves of 101 registers have a CU to
 * themselves, so nothing is loaded while it ranks and picks); 4 rows 9.1, of which the
 * last work-group's pick, one wait for memory behind another, is about half.  One
 * launch instead of two: the last of a group's work-groups, by a count that it leaves
 * at 0, picks. */

#define BEAM_THREADS 1024
#define BEAM_WAVES (BEAM_THREADS / 64)
#define BEAM_LIST 1024 /* candidates that LDS holds; a slice or group with more (many equal ones) takes them one by one */

/* A number that orders as a double does (no NaN), 0 below all. */
__device__ __forceinline__ unsigned long long double_key(double v)
{
    const unsigned long long u = __double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double key_double(unsigned long long k)
{
    return __longlong_as_double(k >> 63 ? k & ~(1ull << 63) : ~k);
}
__device__ __forceinline__ float key_logit(unsigned long long k)
{
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ unsigned long long ld_agent64(const unsigned long long *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void st_agent64(unsigned long long *p, unsigned long long v)
{
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

/* A candidate: its total as a key (0: none), and its beam and id, which order as beam
 * V + id does; lower first of equal ones. */
struct beam_cand {
    unsigned long long k;
    unsigned f;
};
#define BEAM_ID_BITS 18 /* (V is 2^18 at most) */
__device__ __forceinline__ bool beam_above(const beam_cand &a, const beam_cand &b) { return a.k > b.k || (a.k == b.k && a.f < b.f); }

__device__ __forceinline__ float lanes_sum(float v)
{
    v = dpp_quad_sum(v);
    v += lane_xor4(v);
    v += lane_xor8(v);
    v = lane_fold16(v, v);
    return lane_fold32(v, v);
}
/* The least of the greatest of the wave's 2^log groups, those that have something
 * above -infinity, and how many those are; lanes that differ in their high bits
 * are of different groups. */
struct beam_groups {
    float least;
    int count;
};
__device__ __forceinline__ beam_groups beam_bound(float v, int log)
{
    const int most = 6 - log;
    auto step = [&](int i, float o) { v = i < most ? fmaxf(v, o) : fminf(v, o); };
    beam_groups r = { 0.f, 0 };
    auto meet = [&](int i) { /* the groups are whole */
        if (i != most) return;
        r.count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(v > -INFINITY)) >> most;
        v = v > -INFINITY ? v : INFINITY;
    };
    step(0, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, false))); /* lanes 1 0 3 2 */
    step(1, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, false))); /* 2 3 0 1 */
    meet(2);
    step(2, lane_xor4(v));
    meet(3);
    step(3, lane_xor8(v));
    meet(4);
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]);
    step(4, __uint_as_float(s[1]));
    meet(5);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(t[0]);
    step(5, __uint_as_float(t[1]));
    meet(6);
    r.least = v;
    return r;
}
/* The groups of a wave that make n of `full` waves (16 at most, then there are fewer than n). */
__device__ __forceinline__ int beam_groups_log(int n, int full) { return n <= full ? 0 : n <= 2 * full ? 1 : n <= 4 * full ? 2 : n <= 8 * full ? 3 : 4; }
/* The work-group's bound from those of its waves: -infinity where they have fewer than n groups. */
__device__ __forceinline__ float beam_bound_of(const float *least, const int *count, int n)
{
    float v = INFINITY;
    int all = 0;
#pragma unroll
    for (int i = 0; i < BEAM_WAVES; ++i) {
        v = fminf(v, least[i]);
        all += count[i];
    }
    return all >= n ? v : -INFINITY;
}
/* How many of LDS's first n keys are above hi, and how many are lo or above; the list is a multiple of 8 long, 0 behind the n-th. */
__device__ __forceinline__ int beam_rank(const unsigned long long *list, int n, unsigned long long hi, unsigned long long lo, int &reach)
{
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    int at = 0;
    reach = 0;
    for (int j = 0; j < n; j += 8) {
        u64x2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *(const u64x2 *)(list + j + 2 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at += (v[i][0] > hi) + (v[i][1] > hi);
            reach += (v[i][0] >= lo) + (v[i][1] >= lo);
        }
    }
    return at;
}

union beam_lds {
    struct {
        alignas(16) float top[BEAM_WAVES], sum[BEAM_WAVES], bound[BEAM_WAVES];
        alignas(16) int groups[BEAM_WAVES];
        alignas(16) unsigned long long list[BEAM_LIST + 8];
    } slice;
    struct {
        double lse[G2B_MAX_BEAMS]; /* score - log sum exp; NaN: no continuations */
        float most[G2B_MAX_BEAMS]; /* a row's largest logit */
        unsigned close;            /* beams whose sums 32 bits do not tell apart */
        double sum[BEAM_WAVES];
        alignas(16) unsigned long long list[BEAM_LIST + 8];
        unsigned flat[BEAM_LIST];
        alignas(16) float bound[BEAM_WAVES];
        alignas(16) int groups[BEAM_WAVES];
        /* (below: what is taken one by one) */
        unsigned long long best[BEAM_WAVES];
        unsigned best_flat[BEAM_WAVES];
    } pick;
};

/* Beams' sums of exponentials come from the slices in 32 bits. What their logarithm is
 * off by: three maxima (a wave's, a slice's, the row's) below each other scale a term by
 * three exponentials, each within 2^-23, of exponents off by 2.25 * 2^-24 of the
 * distance to the row's largest logit, of which the terms' mean is log V at most (28 *
 * 2^-24 at 2^18 ids); two products and 51 additions: 87 * 2^-24 together, below 2^-17.
 * So totals of two beams that are further apart than 2^-16 are in order. Beams with
 * closer ones among the n_out best (with gaps of 0.1 between them, one group in a
 * thousand) are summed again, in 64 bits, by the group's last work-group: some 20 us a row of
 * 50257, bound by the exponentials. */
#define BEAM_CLOSE 0x1p-16
/* score - log sum exp of the beams whose bit is set, in 64 bits. */
__device__ void beam_exact(const g2_beam_args &a, unsigned row0, unsigned beams, beam_lds &lds)
{
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    while (beams) {
        const unsigned b = (unsigned)__builtin_ctz(beams);
        beams &= beams - 1;
        if (!__builtin_isfinite(lds.pick.lse[b])) continue; /* (the same in every thread) */
        const float *in = a.logits + (size_t)(row0 + b) * (unsigned)a.V;
        const double most = (double)lds.pick.most[b];
        double sum = 0;
#pragma unroll 1
        for (int i0 = tid; i0 < a.V; i0 += 8 * BEAM_THREADS) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = in[min(i0 + BEAM_THREADS * e, a.V - 1)];
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += i0 + BEAM_THREADS * e < a.V ? exp((double)x[e] - most) : 0.;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) lds.pick.sum[w] = sum;
        __syncthreads();
        if (tid == 0) {
            sum = 0;
            for (int i = 0; i < BEAM_WAVES; ++i) sum += lds.pick.sum[i];
            lds.pick.lse[b] = (double)a.score[row0 + b] - (most + log(sum));
        }
        __syncthreads();
    }
}

/* The last of a group's work-groups: the n_out best of all its slices' candidates.
 * One work-group, once: what it costs are its waits for memory (one, for sums and
 * candidates together) and instructions that no one has run before. */
__device__ void beam_pick(const g2_beam_args &a, unsigned g, beam_lds &lds, int *count)
{
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = a.n_out;
    const unsigned row0 = g * (unsigned)a.beams, beams = (unsigned)a.beams, slices = (unsigned)a.slices;
    /* candidate c: entry c % n of a list; the beams' first slices first, so that a group
     * of the bound has candidates of several beams; behind them the ended beams as they are */
    const unsigned listed = beams * slices * (unsigned)n, all = a.done ? listed + beams : listed;
    auto load = [&](unsigned c, unsigned &beam) {
        const unsigned l = c / (unsigned)n, s = l / beams;
        beam = l - s * beams;
        return ld_agent64(a.cands + ((size_t)(row0 + beam) * slices + s) * (unsigned)n + (c - l * (unsigned)n));
    };
    unsigned beam0 = 0;
    const unsigned long long key0 = (unsigned)tid < listed ? load((unsigned)tid, beam0) : 0;
#pragma unroll 1
    for (int b = w; b < a.beams; b += BEAM_WAVES) { /* (a row has 64 slices at most) */
        const unsigned long long v = lane < a.slices ? ld_agent64(a.stats + (size_t)(row0 + (unsigned)b) * slices + (unsigned)lane) : 0xFF800000ull;
        const float top = __uint_as_float((unsigned)v), most = lanes_max(top);
        double sum = (double)(__uint_as_float((unsigned)(v >> 32)) * (top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((top - most) * 1.44269504f)));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) {
            lds.pick.most[b] = most;
            lds.pick.lse[b] = a.done && a.done[row0 + (unsigned)b] ? __longlong_as_double(0x7ff8000000000000ll) : (double)a.score[row0 + (unsigned)b] - ((double)most + log(sum));
        }
    }
    if (tid == 0) { *count = 0; lds.pick.close = 0; }
    __syncthreads();
    auto cand = [&](unsigned beam, unsigned long long k) { /* from its logit's key */
        const double t = (double)key_logit(k) + lds.pick.lse[beam];
        beam_cand c = { 0, beam << BEAM_ID_BITS | ((1u << BEAM_ID_BITS) - 1 & ~(unsigned)k) };
        if (k && t > -INFINITY) c.k = double_key(t);
        return c;
    };
    auto get = [&](unsigned c) {
        unsigned beam;
        if (c < listed) {
            const unsigned long long k = load(c, beam);
            return cand(beam, k);
        }
        beam = c - listed;
        beam_cand e = { 0, beam << BEAM_ID_BITS | (unsigned)a.eos };
        const float score = a.score[row0 + beam];
        if (a.done[row0 + beam] && score > -INFINITY) e.k = double_key((double)score);
        return e;
    };
    const int full = min((int)(listed / 64), BEAM_WAVES);
    const beam_cand none = { 0, ~0u };
    auto put = [&](int i, const beam_cand &c) {
        const size_t at = (size_t)g * (unsigned)n + (unsigned)i;
        const int parent = c.k ? (int)(c.f >> BEAM_ID_BITS) : -1, id = c.k ? (int)(c.f & ((1u << BEAM_ID_BITS) - 1)) : -1;
        a.out_score[at] = c.k ? (float)key_double(c.k) : -INFINITY;
        a.out_parent[at] = parent;
        a.out_id[at] = id;
        if (a.out_done) a.out_done[at] = c.k && (id == a.eos || (a.done && a.done[row0 + (unsigned)parent]));
    };
    /* Once, or twice where beams come too close for sums in 32 bits. */
#pragma unroll 1
    for (bool exact = false;; exact = true) {
        beam_cand c0 = { 0, 0 };
        if ((unsigned)tid < listed) c0 = cand(beam0, key0);
        else if ((unsigned)tid < all) c0 = get((unsigned)tid);
        float best = c0.k ? (float)key_double(c0.k) : -INFINITY;
#pragma unroll 1
        for (unsigned c = (unsigned)tid + BEAM_THREADS; c < all; c += BEAM_THREADS) {
            const beam_cand x = get(c);
            if (x.k) best = fmaxf(best, (float)key_double(x.k));
        }
        beam_groups own = { INFINITY, 0 };
        if (w < full) own = beam_bound(best, beam_groups_log(n, full));
        if (lane == 0) { lds.pick.bound[w] = own.least; lds.pick.groups[w] = own.count; }
        __syncthreads();
        /* (rounded to 32 bits a total keeps its place among the others, but for equal ones;
         * those close to the n-th are wanted, too, 2^-22 for the bound's own rounding) */
        float bound = beam_bound_of(lds.pick.bound, lds.pick.groups, n);
        if (__builtin_isfinite(bound)) bound -= (float)BEAM_CLOSE + fabsf(bound) * 0x1p-22f;
        auto reaches = [&](const beam_cand &c) { return c.k && (float)key_double(c.k) >= bound; };
        auto add = [&](const beam_cand &c) {
            if (!reaches(c)) return;
            const int at = atomicAdd(count, 1);
            if (at < BEAM_LIST) { lds.pick.list[at] = c.k; lds.pick.flat[at] = c.f; }
        };
        add(c0);
#pragma unroll 1
        for (unsigned c = (unsigned)tid + BEAM_THREADS; c < all; c += BEAM_THREADS) add(get(c));
        __syncthreads();
        const int total = *count;
        int at = tid; /* (whose place is below n is put down) */
        beam_cand mine = none;
        if (total <= BEAM_LIST) {
            if (tid < 8) lds.pick.list[total + tid] = 0;
            __syncthreads();
            if (tid < total) {
                mine = { lds.pick.list[tid], lds.pick.flat[tid] };
                const double t = key_double(mine.k), near = exact ? 0. : BEAM_CLOSE;
                const unsigned long long hi = double_key(t + near), lo = double_key(t - near);
                int reach;
                at = beam_rank(lds.pick.list, total, hi, lo, reach);
                if (reach - at > 1 && at < n) {
                    at = 0;
                    unsigned close = 0;
#pragma unroll 1
                    for (int j = 0; j < total; ++j) {
                        const beam_cand x = { lds.pick.list[j], lds.pick.flat[j] };
                        at += beam_above(x, mine);
                        if (x.k <= hi && x.k >= lo && x.f >> BEAM_ID_BITS != mine.f >> BEAM_ID_BITS) close |= 1u << (x.f >> BEAM_ID_BITS) | 1u << (mine.f >> BEAM_ID_BITS);
                    }
                    if (close && !exact) atomicOr(&lds.pick.close, close);
                }
            }
        } else {
            beam_cand last = { ~0ull, 0 }; /* (the list is free: it takes what is chosen) */
            unsigned close = 0;
#pragma unroll 1
            for (int i = 0; i < n + !exact; ++i) { /* one by one: the best that is below the last one */
                beam_cand c = none;
#pragma unroll 1
                for (unsigned l = (unsigned)tid; l < all; l += BEAM_THREADS) {
                    const beam_cand x = get(l);
                    if (reaches(x) && (i == 0 || beam_above(last, x)) && beam_above(x, c)) c = x;
                }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    const beam_cand x = { __shfl_xor(c.k, o), __shfl_xor(c.f, o) };
                    if (beam_above(x, c)) c = x;
                }
                __syncthreads();
                if (lane == 0) { lds.pick.best[w] = c.k; lds.pick.best_flat[w] = c.f; }
                __syncthreads();
                for (int t = 0; t < BEAM_WAVES; ++t) {
                    const beam_cand x = { lds.pick.best[t], lds.pick.best_flat[t] };
                    if (beam_above(x, c)) c = x;
                }
                if (i && c.k && c.f >> BEAM_ID_BITS != last.f >> BEAM_ID_BITS && key_double(last.k) - key_double(c.k) <= BEAM_CLOSE)
                    close |= 1u << (c.f >> BEAM_ID_BITS) | 1u << (last.f >> BEAM_ID_BITS);
                if (tid == 0 && i < n) { lds.pick.list[i] = c.k; lds.pick.flat[i] = c.f; }
                last = c.k ? c : beam_cand{ 1, 0 }; /* (no key is 1: nothing is left) */
            }
            if (tid == 0 && !exact) lds.pick.close = close;
            __syncthreads();
            if (tid < n) mine = { lds.pick.list[tid], lds.pick.flat[tid] };
        }
        if (at < n) put(at, mine);
        if (exact) return;
        __syncthreads();
        const unsigned close = lds.pick.close;
        if (__builtin_expect(!close, 1)) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); /* (what was put down is there before another thread's) */
        if (tid == 0) *count = 0;
        beam_exact(a, row0, close, lds);
        __syncthreads();
    }
}

/* A slice of a row: its largest logit, the sum of exponentials below it, and its
 * n_out greatest logits (of equal ones the lower ids) as keys, 0 for none; then
 * the group's last work-group picks.  What one work-group leaves for another goes
 * to the coherence point and is there before the count goes up. */
template <int QUADS>
__device__ void beam_select_impl(const g2_beam_args &a)
{
    constexpr int SLICE = 4 * BEAM_THREADS * QUADS, Q = 4 * QUADS;
    __shared__ beam_lds lds;
    __shared__ int count, last;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = a.n_out;
    const unsigned row = blockIdx.x / (unsigned)a.slices, slice = blockIdx.x - row * (unsigned)a.slices;
    const int v0 = (int)slice * SLICE, nv = min(a.V - v0, SLICE);
    const float *in = a.logits + (size_t)row * (unsigned)a.V + v0;
    float x[Q];
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
        const int i = 4 * (tid + BEAM_THREADS * q);
        if (i + 4 <= nv) {
            const f32x4 v = *(const f32x4u *)(in + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * q + e] = v[e];
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * q + e] = i + e < nv ? in[i + e] : -INFINITY;
    }
    if (tid == 0) count = 0;
    float mine = -INFINITY;
#pragma unroll
    for (int q = 0; q < Q; ++q) mine = fmaxf(mine, x[q]);
    const float top = lanes_max(mine), base = top == -INFINITY ? 0.f : top;
    float sum = 0.f; /* (NaN where a logit is; ids behind the row add nothing) */
#pragma unroll
    for (int q = 0; q < Q; ++q) sum += __builtin_amdgcn_exp2f((x[q] - base) * 1.44269504f);
    sum = lanes_sum(sum);
    /* (groups of the waves that have ids for every lane; without one the slice is short) */
    const int full = min(nv / 256, BEAM_WAVES);
    beam_groups own = { INFINITY, 0 };
    if (w < full) own = beam_bound(mine, beam_groups_log(n, full));
    if (lane == 0) { lds.slice.top[w] = top; lds.slice.sum[w] = sum; lds.slice.bound[w] = own.least; lds.slice.groups[w] = own.count; }
    __syncthreads();
    const float bound = beam_bound_of(lds.slice.bound, lds.slice.groups, n);
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (x[q] >= bound && x[q] > -INFINITY) {
            const int at = atomicAdd(&count, 1);
            if (at < BEAM_LIST) lds.slice.list[at] = logit_key(x[q], v0 + 4 * (tid + BEAM_THREADS * (q / 4)) + q % 4);
        }
    __syncthreads();
    const int total = count;
    const size_t cell = blockIdx.x;
    unsigned long long *cands = a.cands + cell * (unsigned)n;
    if (total <= BEAM_LIST) {
        if (tid < 8) lds.slice.list[total + tid] = 0;
        __syncthreads();
        if (tid < total) {
            const unsigned long long k = lds.slice.list[tid];
            int reach; /* (keys differ: at + 1) */
            const int at = beam_rank(lds.slice.list, total, k, k, reach);
            if (at < n) st_agent64(cands + at, k);
        } else if (tid < n) st_agent64(cands + tid, 0);
    } else {
        unsigned long long below = ~0ull;
        for (int i = 0; i < n; ++i) { /* one by one: the greatest key below the last one */
            unsigned long long k = 0;
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (x[q] > -INFINITY) {
                    const unsigned long long y = logit_key(x[q], v0 + 4 * (tid + BEAM_THREADS * (q / 4)) + q % 4);
                    k = y < below && y > k ? y : k;
                }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const unsigned long long y = __shfl_xor(k, o);
                k = y > k ? y : k;
            }
            __syncthreads();
            if (lane == 0) lds.slice.list[w] = k;
            __syncthreads();
            for (int t = 0; t < BEAM_WAVES; ++t) k = lds.slice.list[t] > k ? lds.slice.list[t] : k;
            if (tid == 0) st_agent64(cands + i, k);
            below = k;
        }
    }
    if (tid == 0) {
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < BEAM_WAVES; ++i) m = fmaxf(m, lds.slice.top[i]);
#pragma unroll
        for (int i = 0; i < BEAM_WAVES; ++i) l += lds.slice.sum[i] * (lds.slice.top[i] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((lds.slice.top[i] - m) * 1.44269504f));
        st_agent64(a.stats + cell, (unsigned long long)__float_as_uint(l) << 32 | __float_as_uint(m));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const unsigned g = row / (unsigned)a.beams;
    if (tid == 0) {
        unsigned *cell = a.counts + (size_t)g * G2B_COUNT_INTS;
        last = __hip_atomic_fetch_add(cell, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(a.beams * a.slices) - 1;
        if (last) __hip_atomic_store(cell, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (last) beam_pick(a, g, lds, &count);
}
#define BEAM_SELECT(NAME, QUADS) \
    extern "C" __global__ __launch_bounds__(BEAM_THREADS) void NAME(const g2_beam_args a) { beam_select_impl<QUADS>(a); }
BEAM_SELECT(g2k_beam_select1, 1)
BEAM_SELECT(g2k_beam_select4, 4)
BEAM_SELECT(g2k_beam_select7, 7)

/* Rows of the tables in their parents' order, 256 ints of a row to a work-group.
 * Beams move by their tables alone (8 bytes a position): 128 rows of 1001 in 4 us. */
G2K void g2k_beam_copy(const g2_beam_move_args a)
{
    const int chunks = (a.T + 1 + 255) / 256;
    const long row = blockIdx.x / chunks;
    const int g = (int)(row / a.beams), p = (int)(blockIdx.x % chunks) * 256 + threadIdx.x;
    const int n = a.len ? clampi(a.len[g], 0, a.T) : a.T;
    const int from = a.parent[row];
    if (p > n || from < 0 || from >= a.beams) return;
    const long src = (long)g * a.beams + from;
    int id = 0, at = 0;
    if (a.ids_out) id = p < n ? a.ids[src * a.ids_stride + p] : a.next[row];
    if (a.origin_out) at = p < n ? a.origin[src * a.origin_stride + p] : (int)row;
    if (a.ids_out) a.ids_out[row * a.ids_stride + p] = id;
    if (a.origin_out) a.origin_out[row * a.origin_stride + p] = at;
}

/* The same where a table is moved in place: a thread reads its column of all
 * beams before it writes it. */
G2K void g2k_beam_move(const g2_beam_move_args a)
{
    __shared__ int col[2][G2B_MAX_BEAMS][256];
    const int tid = threadIdx.x, chunks = (a.T + 1 + 255) / 256;
    const long g = blockIdx.x / chunks, row0 = g * a.beams;
    const int p = (int)(blockIdx.x % chunks) * 256 + tid;
    const int n = a.len ? clampi(a.len[g], 0, a.T) : a.T;
    if (p > n) return;
    if (p < n)
#pragma unroll 4
        for (int b = 0; b < a.beams; ++b) {
            if (a.ids_out) col[0][b][tid] = a.ids[(row0 + b) * a.ids_stride + p];
            if (a.origin_out) col[1][b][tid] = a.origin[(row0 + b) * a.origin_stride + p];
        }
#pragma unroll 4
    for (int b = 0; b < a.beams; ++b) {
        const int from = a.parent[row0 + b];
        if (from < 0 || from >= a.beams) continue;
        if (a.ids_out) a.ids_out[(row0 + b) * a.ids_stride + p] = p < n ? col[0][from][tid] : a.next[row0 + b];
        if (a.origin_out) a.origin_out[(row0 + b) * a.origin_stride + p] = p < n ? col[1][from][tid] : (int)(row0 + b);
    }
}
} // namespace gb

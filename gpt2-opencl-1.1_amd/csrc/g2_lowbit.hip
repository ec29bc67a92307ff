/*
 * g2_lowbit.hip -- what a decode step reads in fewer bits, and the choice of
 * its token (included by g2_kernels.hip, which provides the shared helpers
 * and types): products with 4-bit weights, the 8-bit K/V cache and the
 * single-query attention over it, rules on logits.  The layouts and their
 * index functions are in g2_lowbit_plan.h.
 */

__device__ __forceinline__ float bf16_f(uint16_t b) { return __uint_as_float((unsigned)b << 16); }

/* bf16 of a finite positive value, to nearest even */
__device__ __forceinline__ uint16_t f_bf16(float v)
{
    const unsigned u = __float_as_uint(v);
    return (uint16_t)((u + 0x7FFF + ((u >> 16) & 1)) >> 16);
}

/* ======================================================================
 * 4-bit weights: E2M1 values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives
 * (code: sign, 2 exponent bits, 1 mantissa bit) times a bf16 scale for each
 * row and group of 32, 64 or 128 columns.
 *
 * The scale of a group is bf16(max |w| / 6), each step rounded to nearest, a
 * weight's code the value nearest to fp32(w / scale), a tie to the even code.
 * (bf16 has fp32's range, and the scale's own 2^-9 only moves the grid that
 * the codes are then chosen on.)  A group that holds an infinity, a NaN or a
 * magnitude above 2^96 (whose products could pass fp32's range while their
 * sum does not) gets a NaN scale: it reads back as NaN.
 * ==================================================================== */

/* scale of a group from the largest bit pattern of its magnitudes */
__device__ __forceinline__ uint16_t q4_scale(unsigned amax)
{
    if (amax > 0x6F800000u) return 0x7FC0;
    return f_bf16(__uint_as_float(amax) / 6.0f);
}

/* a / b correctly rounded, for b of 8 significant bits (a bf16 scale) between
 * 2^-100 and 2^100, from r, the correctly rounded 1 / b: a step on the remainder,
 * which the fused multiply-add has exactly.  The step's result is within 2^-22
 * of a last place of a / b before it is rounded; a / b is no nearer than 2^-9 of
 * one to where the rounding changes, since 25 bits times 8 have 33 and a has
 * 24.  Where the remainder falls below the normal range, so does a, and the
 * quotient lies far below the first border between codes. */
__device__ __forceinline__ float quotient(float a, float b, float r)
{
    const float q = a * r;
    return fmaf(fmaf(-q, b, a), r, q);
}

/* The codes of eight weights over a scale.  The conversion rounds a value to
 * the nearest code, ties to even and at most 6, as the definition does; it is
 * given the quotient correctly rounded (the division itself for scales at the
 * ends of the range).  A code of -0 becomes 0; a group's scale of 0 or NaN has
 * codes 0. */
__device__ __forceinline__ unsigned q4_codes(const float w[8], float s)
{
    unsigned c = 0;
    if (s > 0x1p-100f && s < 0x1p+100f) {
        const float r = 1.0f / s;
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = quotient(w[i], s, r);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[0], q[1], 1.0f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[2], q[3], 1.0f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[4], q[5], 1.0f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[6], q[7], 1.0f, 3);
    } else if (s > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const unsigned b = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, w[i] / s, w[i + 1] / s, 1.0f, 0);
            c |= (b & 255) << 4 * i;
        }
    }
    const unsigned mag = c & 0x77777777u;
    return c & (0x77777777u | ((mag + 0x77777777u) & 0x88888888u));
}

/* The largest magnitude (as bits) among the lanes of a group: four lanes have
 * the 32 columns of a step, 16 a chunk. */
template <int CTRL> __device__ __forceinline__ unsigned dpp_umax(unsigned v)
{
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return o > v ? o : v;
}
__device__ __forceinline__ unsigned q4_group_max(unsigned amax, int group)
{
    amax = dpp_umax<0xB1>(amax);                   /* quad: lanes 1 0 3 2 */
    amax = dpp_umax<0x4E>(amax);                   /* 2 3 0 1 */
    if (group > 32) amax = dpp_umax<0x141>(amax);  /* half rows of 8, mirrored */
    if (group > 64) amax = dpp_umax<0x140>(amax);  /* rows of 16, mirrored */
    return amax;
}

/* Eight weights of a row from column k on, 0 behind the matrix. */
template <typename WT> struct q4_raw { WT v[8]; };
template <typename WT>
__device__ __forceinline__ q4_raw<WT> q4_load8(const WT *W, long n, long k, long N, long K)
{
    typedef WT w8 __attribute__((ext_vector_type(8), aligned(sizeof(WT))));
    q4_raw<WT> r;
    if (n < N && k + 8 <= K) {
        const w8 v = *(const w8 *)(W + n * K + k);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = n < N && k + i < K ? W[n * K + k + i] : (WT)0.f;
    }
    return r;
}

/* Scale and codes of a lane's eight weights to their places: row r of tile t,
 * step j and place p of chunk c. */
template <typename WT>
__device__ __forceinline__ void q4_pack8(const g2_q4_args &a, const q4_raw<WT> &raw, long t, long c, int r, int j, int p)
{
    float w[8];
    unsigned amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        w[i] = (float)raw.v[i];
        const unsigned u = __float_as_uint(w[i]) & 0x7FFFFFFF;
        amax = u > amax ? u : amax;
    }
    const uint16_t sb = q4_scale(q4_group_max(amax, a.group));
    const int steps = g2l_chunk_steps(a.K, c), per = a.group / 32;
    if (j < steps) *(unsigned *)(a.codes + g2l_code_at(a.K, t, c, 16 * p + r) + 4 * j) = q4_codes(w, bf16_f(sb));
    if (p == 0 && j % per == 0) a.scales[g2l_scale_at(a.K, a.group, t, c, r, j / per)] = sb;
}

/* W [N,K]: a work-group takes chunks of 16 rows x 128 columns, two at a time:
 * thread = row, step, place, eight consecutive columns.  50257 x 768 fp16 27.6
 * us, 3.6 TB/s (a thread per row and group, which walked its 32 columns one by
 * one: 204); loads that do not stay in the L2 were slower (a lane's 32 bytes are
 * two loads), as were 32-bit quotients in place of the divisions here. */
template <typename WT>
__device__ void q4_pack_impl(const g2_q4_args &a)
{
    const WT *W = (const WT *)a.W;
    const int tid = threadIdx.x, r = tid >> 4, j = tid >> 2 & 3, p = tid & 3;
    const long chunks = g2l_chunks(a.K), items = g2l_tiles(a.N) * chunks;
    for (long i = blockIdx.x * 2l; i < items; i += gridDim.x * 2l) {
        q4_raw<WT> w[2];
        long t[2], c[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            t[u] = (i + u) / chunks;
            c[u] = (i + u) % chunks;
            w[u] = q4_load8<WT>(W, t[u] * 16 + r, c[u] * 128 + 32 * j + 8 * p, a.N, a.K);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (i + u < items) q4_pack8<WT>(a, w[u], t[u], c[u], r, j, p);
    }
}
G2K void g2k_q4_pack_f32(const g2_q4_args a) { q4_pack_impl<float>(a); }
G2K void g2k_q4_pack_f16(const g2_q4_args a) { q4_pack_impl<_Float16>(a); }

/* W [K,N]: 32 rows x 128 columns at a time through LDS (32 neighbouring
 * values of a column are one run in memory), all of a thread's eight loads in
 * flight: 768 x 768 3.7 us, 6400 x 1600 14.9 (4.6 and 22.4 with 64 rows, whose
 * two work-groups to a CU wait more than these four). */
#define Q4_TROW 33
template <typename WT>
__device__ void q4_pack_t_impl(const g2_q4_args &a)
{
    __shared__ WT ws[128 * Q4_TROW];
    const WT *W = (const WT *)a.W;
    const int tid = threadIdx.x, u = tid >> 8, r = tid >> 4 & 15, j = tid >> 2 & 3, p = tid & 3;
    const long chunks = g2l_chunks(a.K), tiles = g2l_tiles(a.N), items = (tiles + 1) / 2 * chunks;
    for (long i = blockIdx.x; i < items; i += gridDim.x) {
        const long t0 = i / chunks * 2, c = i % chunks, n = t0 * 16 + (tid & 31);
        const WT *col = W + (n < a.N ? n : a.N - 1);
        WT v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const long k = c * 128 + (tid >> 5) + 16 * e;
            v[e] = col[(k < a.K ? k : a.K - 1) * a.N];
            if (n >= a.N || k >= a.K) v[e] = (WT)0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ws[((tid >> 5) + 16 * e) * Q4_TROW + (tid & 31)] = v[e];
        __syncthreads();
        q4_raw<WT> w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w.v[e] = ws[(32 * j + 8 * p + e) * Q4_TROW + 16 * u + r];
        if (t0 + u < tiles) q4_pack8<WT>(a, w, t0 + u, c, r, j, p);
        __syncthreads();
    }
}
extern "C" __global__ __launch_bounds__(512) void g2k_q4_pack_t_f32(const g2_q4_args a) { q4_pack_t_impl<float>(a); }
extern "C" __global__ __launch_bounds__(512) void g2k_q4_pack_t_f16(const g2_q4_args a) { q4_pack_t_impl<_Float16>(a); }

/* The eight values of a lane's word of codes. */
__device__ __forceinline__ void q4_values(unsigned w, float s, float v[8])
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
    v[4] = c[0] * s; v[5] = c[1] * s; v[6] = d[0] * s; v[7] = d[1] * s;
}
__device__ __forceinline__ unsigned q4_word(const g2_q4_args &a, long t, long c, int r, int j, int p, float *s)
{
    *s = bf16_f(a.scales[g2l_scale_at(a.K, a.group, t, c, r, 32 * j / a.group)]);
    return j < g2l_chunk_steps(a.K, c) ? *(const unsigned *)(a.codes + g2l_code_at(a.K, t, c, 16 * p + r) + 4 * j) : 0u;
}

/* To [N,K]: threads as in the laying out; the 16 lanes of a row then take its
 * 128 columns four at a time, so that a store is 256 bytes of each of four
 * rows.  Where rows are whole 64-byte pieces the stores do not stay in the L2.
 * 50257 x 768, values that no cache holds, 26.4 us; with ordinary stores 39.0
 * (10388 x 3715, whose rows are not, 53.7 and 59.3 the other way round); with a
 * lane's own 32 bytes in two stores 46.9. */
G2K void g2k_q4_read(const g2_q4_args a)
{
    const int tid = threadIdx.x, r = tid >> 4, j = tid >> 2 & 3, p = tid & 3, lane = tid & 63, l = tid & 15;
    const bool whole = a.K % 16 == 0 && (uintptr_t)a.out % 64 == 0;
    const long chunks = g2l_chunks(a.K), items = g2l_tiles(a.N) * chunks;
    for (long i = blockIdx.x * 2l; i < items; i += gridDim.x * 2l) {
        unsigned w[2];
        float s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const long iu = i + u < items ? i + u : items - 1;
            w[u] = q4_word(a, iu / chunks, iu % chunks, r, j, p, &s[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const long n = (i + u) / chunks * 16 + r, k0 = (i + u) % chunks * 128 + 4 * l;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int from = (lane & 48) + 8 * h + (l >> 1); /* the lane that has columns 64 h + 4 l .. + 3 */
                const unsigned wh = (unsigned)__shfl((int)w[u], from) >> 16 * (l & 1);
                const float sh = __shfl(s[u], from);
                const long k = k0 + 64 * h;
                if (i + u >= items || n >= a.N || k >= a.K) continue;
                typedef float f32x2 __attribute__((ext_vector_type(2)));
                const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(wh, 1.0f, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(wh, 1.0f, 1);
                const f32x4 v = { lo[0] * sh, lo[1] * sh, hi[0] * sh, hi[1] * sh };
                float *o = a.out + n * a.K + k;
                if (whole) __builtin_nontemporal_store(v, (f32x4 *)o);
                else if (k + 4 <= a.K) *(f32x4u *)o = v;
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k + e < a.K) o[e] = v[e];
            }
        }
    }
}

/* To [K,N], through LDS. */
extern "C" __global__ __launch_bounds__(512) void g2k_q4_read_t(const g2_q4_args a)
{
    __shared__ float ws[128 * Q4_TROW];
    const int tid = threadIdx.x, u = tid >> 8, r = tid >> 4 & 15, j = tid >> 2 & 3, p = tid & 3;
    const long chunks = g2l_chunks(a.K), tiles = g2l_tiles(a.N), items = (tiles + 1) / 2 * chunks;
    for (long i = blockIdx.x; i < items; i += gridDim.x) {
        const long t0 = i / chunks * 2, c = i % chunks, n = t0 * 16 + (tid & 31);
        float s, v[8];
        const unsigned w = q4_word(a, t0 + u < tiles ? t0 + u : tiles - 1, c, r, j, p, &s);
        q4_values(w, s, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) ws[(32 * j + 8 * p + e) * Q4_TROW + 16 * u + r] = v[e];
        __syncthreads();
#pragma unroll
        for (int k = tid >> 5; k < 128; k += 16)
            if (n < a.N && c * 128 + k < a.K) a.out[(c * 128 + k) * a.N + n] = ws[k * Q4_TROW + (tid & 31)];
        __syncthreads();
    }
}

/* ---- products: y = x W^T on the matrix cores.  A chunk of 128 columns of a
 * tile of 16 rows is one 16-byte load a lane; the hardware's conversion makes
 * fp16 of it (exact; two values an operation) and four 16x16x32 products of
 * it, one operand the 16 weight rows, the other up to 8 activation rows, each
 * as two fp16 parts: hi = fp16(x'), lo = fp16(2^11 (x' - hi)), x' the activation
 * times a power of two that brings the largest of its 128 to 2^14..2^15.  hi +
 * 2^-11 lo is within 2^-22 of x' where |x'| is 2^-14 or more.  A chunk with an
 * activation below that (2^-28 of its largest, but not 0) or an infinity is left
 * to the vector units, which multiply and add in fp32 (q4_add_plain; one in 10^6
 * rows of normally distributed values): so every activation enters with 2^-22
 * of its own value.  Such a chunk costs a product 2 to 8 us (6400 x 1600, one and
 * 8 rows), in the held form, which then takes all chunks so, more (50257 x 1600
 * 45 and 152 us in all).  A group's scale multiplies its sum, the power of two a
 * chunk's; all sums are fp32.
 *
 * Bounded by HBM for large matrices and by the launch and two load latencies
 * for small ones: 50257 x 1600, groups of 128, 9.7 us in a replayed graph with
 * matrices that no cache holds, 4.3 TB/s, 8.5 from the cache behind it; 768 x
 * 768 2.5 us.  Which form a product takes: g2i_q4_form. */
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int I> __device__ __forceinline__ void q4_half(f16x8 &r, unsigned w)
{
    const f16x2 h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, I);
    r[2 * I] = h[0];
    r[2 * I + 1] = h[1];
}
__device__ __forceinline__ f16x8 q4_operand(unsigned w)
{
    f16x8 r;
    q4_half<0>(r, w);
    q4_half<1>(r, w);
    q4_half<2>(r, w);
    q4_half<3>(r, w);
    return r;
}

/* The power of two (and its inverse) that brings a value of these bits, the
 * largest of its chunk, to 2^14..2^15; 2^126 at most. */
struct q4_power { float down, up; };
__device__ __forceinline__ q4_power q4_power_of(unsigned amax)
{
    const unsigned e = amax >> 23 > 15 ? amax >> 23 : 15;
    return { __uint_as_float((268 - e) << 23), __uint_as_float((e - 14) << 23) };
}

/* hi and lo parts of two activations (every step but the two conversions is exact) */
#define Q4_LO 2048.0f
__device__ __forceinline__ void q4_split(float a, float b, float down, f16x2 &hi, f16x2 &lo)
{
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(a * down, b * down));
    lo[0] = (_Float16)(__builtin_fmaf(a, down, -(float)hi[0]) * Q4_LO);
    lo[1] = (_Float16)(__builtin_fmaf(b, down, -(float)hi[1]) * Q4_LO);
}

/* Whether any lane says so, as one value of the wave (the compiler takes __any's
 * for a lane's: both sides of its branch then hold their registers at once). */
__device__ __forceinline__ bool wave_any(bool b) { return __builtin_amdgcn_ballot_w64(b) != 0; }

template <int CTRL> __device__ __forceinline__ float dpp_max(float v)
{
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true)));
}

#define Q4_XROW 136 /* halves from row to row of a wave's split activations: 128 and 16 bytes against bank conflicts */

template <int MT> struct q4_x {
    float v[MT == 1 ? 2 : 16];
    bool behind; /* no column of the lane's lies in the matrix */
};

/* The chunk's activations: MT == 1: two columns a lane; else lane 8 m + i has
 * columns 16 i .. 16 i + 15 of row m. */
template <int MT>
__device__ __forceinline__ q4_x<MT> q4_load_x(const g2_q4mv_args &a, int m0, int c, int lane)
{
    q4_x<MT> x;
    const int n = MT == 1 ? 2 : 16, m = m0 + (MT == 1 ? 0 : lane >> 3), k = 128 * c + n * (MT == 1 ? lane : lane & 7);
    const float *p = a.x + (size_t)(m < a.M ? m : a.M - 1) * a.K; /* (a row behind the last: the last, not written) */
    x.behind = k >= a.K;
    if (MT == 1 && 128 * c + 128 <= a.K) { /* (uniform) */
        x.v[0] = p[k];
        x.v[1] = p[k + 1];
    } else if (MT > 1 && (128 * c + 128 <= a.K || a.K % 16 == 0)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 q = *(const f32x4u *)(p + (k < a.K ? k : 0) + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[(4 * i + e) % n] = k < a.K ? q[e] : 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < n; ++i) x.v[i] = p[k + i < a.K ? k + i : a.K - 1];
#pragma unroll
        for (int i = 0; i < n; ++i) x.v[i] = k + i < a.K ? x.v[i] : 0.f;
    }
    return x;
}

/* The largest of the lane's row of the chunk, of magnitudes as bits. */
template <int MT>
__device__ __forceinline__ unsigned q4_largest(unsigned amax)
{
    amax = q4_group_max(amax, 64); /* 8 lanes */
    if constexpr (MT == 1) {
        amax = dpp_umax<0x140>(amax); /* rows of 16, mirrored */
        const unsigned r0 = __builtin_amdgcn_readlane(amax, 0), r1 = __builtin_amdgcn_readlane(amax, 16);
        const unsigned r2 = __builtin_amdgcn_readlane(amax, 32), r3 = __builtin_amdgcn_readlane(amax, 48);
        const unsigned m0 = r0 > r1 ? r0 : r1, m1 = r2 > r3 ? r2 : r3;
        amax = m0 > m1 ? m0 : m1;
    }
    return amax;
}

/* The powers of two of the lane's row; plain: whether any row's parts would not
 * hold a value of it: an infinity, or one below 2^-14 up that is not 0 (at the
 * least power both parts hold the smallest numbers too).  A NaN counts for
 * neither: it is a NaN in both parts.  Zeros are told from small values behind
 * the branch (1600 x 6400, 8 rows, 8.1 us; for every chunk 8.5). */
struct q4_seen {
    q4_power own;
    bool plain;
};
template <int MT> __device__ __forceinline__ q4_seen q4_look(const q4_x<MT> &x)
{
    constexpr int N = MT == 1 ? 2 : 16;
    float amax = 0.f, least = INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        amax = fmaxf(amax, fabsf(x.v[i]));
        least = fminf(least, fabsf(x.v[i]));
    }
    const unsigned top = q4_largest<MT>(__float_as_uint(amax));
    q4_seen s = { q4_power_of(top), false };
    const float low = s.own.up > 0x1p-126f ? s.own.up * 0x1p-14f : 0.f;
    if (wave_any((top == 0x7F800000u) | ((least < low) & !x.behind))) {
        bool plain = top == 0x7F800000u;
#pragma unroll
        for (int i = 0; i < N; ++i) plain |= (x.v[i] != 0.f) & (fabsf(x.v[i]) < low);
        s.plain = wave_any(plain);
    }
    return s;
}

/* Splits them into xs ([part of row][Q4_XROW]) and gives the inverse powers of
 * two of the lane's own rows of the product: MT == 1: row 0; else rows
 * 2 (lane / 16) and + 1. */
template <int MT>
__device__ __forceinline__ void q4_split_x(const q4_x<MT> &x, const q4_power &own, _Float16 *xs, float *xe, int lane, float e[2])
{
    constexpr int N = MT == 1 ? 2 : 16;
    f16x2 hi[N / 2], lo[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) q4_split(x.v[2 * i], x.v[2 * i + 1], own.down, hi[i], lo[i]);
    _Float16 *row = xs + (MT == 1 ? 0 : 2 * (lane >> 3)) * Q4_XROW + N * (MT == 1 ? lane : lane & 7);
    if constexpr (MT == 1) {
        *(f16x2 *)row = hi[0];
        *(f16x2 *)(row + Q4_XROW) = lo[0];
        e[0] = e[1] = own.up;
    } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            f16x8 h, l;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[i] = hi[4 * g + i / 2][i % 2];
                l[i] = lo[4 * g + i / 2][i % 2];
            }
            *(f16x8 *)(row + 8 * g) = h;
            *(f16x8 *)(row + Q4_XROW + 8 * g) = l;
        }
        if ((lane & 7) == 0) xe[lane >> 3] = own.up;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if constexpr (MT > 1) {
        e[0] = xe[2 * (lane >> 4)];
        e[1] = xe[2 * (lane >> 4) + 1];
    }
}

/* Where a lane finds its weights in a chunk. */
struct q4_lane {
    unsigned whole, part; /* bytes into a chunk of four steps, of fewer */
    int shift, last;      /* words to move there; the chunk of fewer steps, -1 */
};
__device__ __forceinline__ q4_lane q4_lane_of(const g2_q4mv_args &a, int lane)
{
    const int c = (int)g2l_chunks(a.K) - 1;
    return { 16u * lane, g2l_lane_at(a.K, c, lane), g2l_lane_shift(a.K, c, lane), g2l_chunk_steps(a.K, c) < 4 ? c : -1 };
}

/* One load each of codes and scales, at a uniform base and the lane's offset
 * and without a branch (behind a branch the compiler waits for every load in
 * flight; 64-bit addresses per lane had cost as many operations as the
 * products). */
template <int G> struct q4_w {
    u32x4 w;
    uint16_t s[128 / G];
};
template <int G>
__device__ __forceinline__ q4_w<G> q4_load_w(const uint8_t *codes, const uint16_t *scales, unsigned at, unsigned sat)
{
    constexpr int P = 128 / G;
    typedef uint16_t sv __attribute__((ext_vector_type(P == 1 ? 2 : P)));
    typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(4)));
    q4_w<G> r;
    r.w = *(const u32x4u *)(codes + at);
    if constexpr (P == 1) r.s[0] = *(const uint16_t *)((const char *)scales + sat);
    else {
        const sv v = *(const sv *)((const char *)scales + sat);
#pragma unroll
        for (int g = 0; g < P; ++g) r.s[g] = v[g];
    }
    return r;
}
__device__ __forceinline__ void q4_shift(u32x4 &w, int n)
{
    if (n & 1) w = u32x4{ w[1], w[2], w[3], 0u };
    if (n & 2) w = u32x4{ w[2], w[3], 0u, 0u };
}

/* Adds a chunk's products to the lane's sums: MT == 1: of row 0; else of rows
 * 2 (lane / 16) and + 1; column lane % 16 of the tile.  The empty statement
 * keeps the sums of the products' results in the block of the products: moved
 * behind a branch, the first of them was left without the wait that it needs
 * after a matrix instruction (test_matrix_waits.py looks for such places). */
template <int MT, int G>
__device__ __forceinline__ void q4_products(const f16x8 x[4], const u32x4 &w, const uint16_t *scale, const float e[2], float *y)
{
    constexpr int P = 128 / G;
    float s[2] = {};
#pragma unroll
    for (int g = 0; g < P; ++g) {
        f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 4 / P * g; j < 4 / P * (g + 1); ++j)
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[j], q4_operand(w[j]), d, 0, 0, 0);
        const float sc = bf16_f(scale[g]);
        s[0] = fmaf(sc, fmaf(d[1], 1.f / Q4_LO, d[0]), s[0]);
        if constexpr (MT > 1) s[1] = fmaf(sc, fmaf(d[3], 1.f / Q4_LO, d[2]), s[1]);
    }
    y[0] = fmaf(s[0], e[0], y[0]);
    if constexpr (MT > 1) y[1] = fmaf(s[1], e[1], y[1]);
    if constexpr (MT > 1) asm volatile("" : "+v"(y[0]), "+v"(y[1]));
    else asm volatile("" : "+v"(y[0]));
}

/* Adds chunk c's products to the sums of the TR tiles in fp32: a lane takes the
 * columns of its own codes, four at a time, for all activation rows, and the four
 * lanes of a weight row meet. */
template <int MT, int TR, int G>
__device__ __forceinline__ void q4_add_plain(const g2_q4mv_args &a, int m0, int c, int lane, const uint8_t *const *codes,
                                             const uint16_t *const *scales, const q4_lane &ql, float (*y)[2])
{
    constexpr int P = 128 / G;
    const unsigned at = c == ql.last ? ql.part : ql.whole;
    const int shift = c == ql.last ? ql.shift : 0;
    float sum[TR][MT] = {};
#pragma unroll 1
    for (int j = 0; j < 8; ++j) { /* half a word of codes */
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const int k = 128 * c + 32 * (j >> 1) + 8 * (lane >> 4) + 4 * (j & 1);
        const int word = (j >> 1) + shift < 3 ? (j >> 1) + shift : 3; /* (behind K: x is 0) */
        f32x4 x[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const float *p = a.x + (size_t)(m0 + m < a.M ? m0 + m : a.M - 1) * a.K;
            if (128 * c + 128 <= a.K || a.K % 4 == 0) { /* (uniform) */
                x[m] = *(const f32x4u *)(p + (k < a.K ? k : 0));
                if (k >= a.K) x[m] = f32x4{ 0.f, 0.f, 0.f, 0.f };
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[m][i] = k + i < a.K ? p[k + i < a.K ? k + i : 0] : 0.f;
            }
        }
#pragma unroll
        for (int t = 0; t < TR; ++t) {
            const unsigned q = *(const unsigned *)(codes[t] + c * 1024l + at + 4 * word) >> 16 * (j & 1);
            const float s = bf16_f(scales[t][(c * 16l + (lane & 15)) * P + (j >> 1) * P / 4]);
            const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
            const float v[4] = { lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s };
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[t][m] = fmaf(v[i], x[m][i], sum[t][m]);
        }
    }
#pragma unroll
    for (int t = 0; t < TR; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float v = sum[t][m];
            v += __shfl_xor(v, 16);
            v += __shfl_xor(v, 32);
            y[t][m & 1] += MT == 1 || lane >> 4 == m >> 1 ? v : 0.f;
        }
}

template <int MT>
__device__ __forceinline__ void q4_put(float (*red)[16], int lane, const float *y)
{
    if constexpr (MT == 1) {
        if (lane < 16) red[0][lane] = y[0];
    } else {
        red[2 * (lane >> 4)][lane & 15] = y[0];
        red[2 * (lane >> 4) + 1][lane & 15] = y[1];
    }
}

/* Outputs of the TR tiles from t0 on: the waves' sums, in order, and the epilogue. */
template <int MT, int KW, int TR>
__device__ __forceinline__ void q4_outputs(const g2_q4mv_args &a, int t0, int m0, const float (*red)[TR][MT][16])
{
    for (int o = threadIdx.x; o < TR * MT * 16; o += KW * 64) {
        const int r = o & 15, m = o / 16 % MT, i = o / 16 / MT;
        const long n = (t0 + i) * 16l + r;
        if (n >= a.N || m0 + m >= a.M) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) v += red[k][i][m][r];
        const size_t at = (size_t)(m0 + m) * a.N + n;
        if (a.bias) v += a.bias[n];
        if (a.res) v += a.res[at];
        a.y[at] = a.gelu ? gelu_f(v) : v;
    }
}

/* The loop: the waves of a work-group take the chunks of the same TR tiles in
 * turn, each splits its own chunk of the activations; the sums of the waves
 * meet in LDS, in order.  The next chunk's loads go out before a chunk's
 * products.  Chunks left to fp32 come behind the loop, where their registers
 * are not beside the loop's. */
template <int MT, int KW, int TR, int G>
__device__ void q4_matvec_impl(const g2_q4mv_args &a)
{
    constexpr int ROWS = MT == 1 ? 2 : 16, SB = 32 * (128 / G); /* bytes of a chunk's scales */
    __shared__ __align__(16) _Float16 xs[KW][ROWS * Q4_XROW];
    __shared__ float xe[KW][8];
    __shared__ float red[KW][TR][MT][16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (int)g2l_tiles(a.N), t0 = blockIdx.x * TR, m0 = blockIdx.y * 8, chunks = (int)g2l_chunks(a.K);
    const q4_lane ql = q4_lane_of(a, lane);
    const unsigned sat = (lane & 15) * (SB / 16);
    const _Float16 *frag = xs[w] + (lane & (ROWS - 1)) * Q4_XROW + 8 * (lane >> 4);
    const uint8_t *codes[TR];
    const uint16_t *scales[TR];
    float y[TR][2] = {};
    q4_w<G> wn[TR];
    q4_x<MT> xn;
    auto load = [&](int c) {
        xn = q4_load_x<MT>(a, m0, c, lane);
#pragma unroll
        for (int i = 0; i < TR; ++i)
            wn[i] = q4_load_w<G>(codes[i] + c * 1024l, scales[i] + c * (SB / 2), c == ql.last ? ql.part : ql.whole, sat);
    };
#pragma unroll
    for (int i = 0; i < TR; ++i) {
        const int t = t0 + i < tiles ? t0 + i : tiles - 1; /* (a tile behind the last: the last again, not written) */
        codes[i] = a.codes + g2l_code_at(a.K, t, 0, 0);
        scales[i] = a.scales + g2l_scale_at(a.K, G, t, 0, 0, 0);
    }
    bool plain = false;
    if (w < chunks) load(w);
    for (int c = w; c < chunks; c += KW) {
        q4_w<G> wc[TR];
        const q4_x<MT> xc = xn;
#pragma unroll
        for (int i = 0; i < TR; ++i) wc[i] = wn[i];
        if (c + KW < chunks) load(c + KW);
        const q4_seen seen = q4_look<MT>(xc);
        if (seen.plain) {
            plain = true;
            continue;
        }
        float e[2];
        q4_split_x<MT>(xc, seen.own, xs[w], xe[w], lane, e);
        f16x8 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *(const f16x8 *)(frag + 32 * j);
        __builtin_amdgcn_wave_barrier();
        if (c == ql.last)
#pragma unroll
            for (int i = 0; i < TR; ++i) q4_shift(wc[i].w, ql.shift);
#pragma unroll
        for (int i = 0; i < TR; ++i) q4_products<MT, G>(x, wc[i].w, wc[i].s, e, y[i]);
    }
    if (plain)
#pragma unroll 1
        for (int c = w; c < chunks; c += KW)
            if (q4_look<MT>(q4_load_x<MT>(a, m0, c, lane)).plain) q4_add_plain<MT, TR, G>(a, m0, c, lane, codes, scales, ql, y);
#pragma unroll
    for (int i = 0; i < TR; ++i) q4_put<MT>(red[w][i], lane, y[i]);
    __syncthreads();
    q4_outputs<MT, KW, TR>(a, t0, m0, red);
}
#define Q4_MATVEC(MT, KW, TR)                                                                                          \
    extern "C" __global__ __launch_bounds__(64 * KW) void g2k_q4_mv##MT##_##KW##_##TR##_32(const g2_q4mv_args a)      \
    { q4_matvec_impl<MT, KW, TR, 32>(a); }                                                                             \
    extern "C" __global__ __launch_bounds__(64 * KW) void g2k_q4_mv##MT##_##KW##_##TR##_64(const g2_q4mv_args a)      \
    { q4_matvec_impl<MT, KW, TR, 64>(a); }                                                                             \
    extern "C" __global__ __launch_bounds__(64 * KW) void g2k_q4_mv##MT##_##KW##_##TR##_128(const g2_q4mv_args a)     \
    { q4_matvec_impl<MT, KW, TR, 128>(a); }
Q4_MATVEC(1, 8, 1)
Q4_MATVEC(1, 16, 1)
Q4_MATVEC(8, 8, 1)
Q4_MATVEC(8, 16, 1)
Q4_MATVEC(8, 8, 2)
Q4_MATVEC(8, 8, 4)

/* The held form: a wave's NC chunks of the activations stay in its registers
 * for all tiles that the work-group takes in turn; a tile's loads (its bias and
 * residual with them, since loads return in order) go out a tile ahead; more
 * tiles ahead are no faster (50257 x 1600 on 512 work-groups 12.4 us with two
 * and 14.3 with four, 11.9 with one).  A work-group with a chunk that is left to
 * fp32 takes all of its tiles' products there. */
template <int NC, int G> struct q4_stage {
    q4_w<G> w[NC];
    float bias, res;
};

template <int MT, int KW, int NC, int G>
__device__ void q4_held_impl(const g2_q4mv_args &a)
{
    constexpr int ROWS = MT == 1 ? 2 : 16, SB = 32 * (128 / G);
    __shared__ __align__(16) _Float16 xs[KW][ROWS * Q4_XROW];
    __shared__ float xe[KW][8];
    __shared__ float red[2][KW][MT][16];
    __shared__ int left[KW]; /* the wave has a chunk that is left to fp32 */
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = (int)g2l_tiles(a.N), m0 = blockIdx.y * 8, chunks = (int)g2l_chunks(a.K), step = gridDim.x;
    const q4_lane ql = q4_lane_of(a, lane);
    unsigned at[NC], sat[NC];
    q4_x<MT> xr[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = w + KW * i < chunks ? w + KW * i : chunks - 1;
        xr[i] = q4_load_x<MT>(a, m0, c, lane);
        at[i] = c * 1024 + (c == ql.last ? ql.part : ql.whole);
        sat[i] = c * SB + (lane & 15) * (SB / 16);
    }
    const size_t tile_codes = g2l_code_at(a.K, 1, 0, 0), tile_scales = g2l_scale_at(a.K, G, 1, 0, 0, 0);
    /* this thread's output of a tile: row r of the tile, activation row m */
    const int r = tid & 15, m = tid >> 4, mr = m0 + m < a.M ? m : a.M - 1 - m0;
    const float *bias = a.bias ? a.bias : a.x, *res = a.res ? a.res + (size_t)m0 * a.N : a.x; /* (readable, not used) */
    auto load = [&](int t) {
        q4_stage<NC, G> s;
        t = t < tiles ? t : tiles - 1;
        const unsigned left = a.N - 16 * t - 1, n = (unsigned)r < left ? r : left;
        s.bias = bias[a.bias ? 16l * t + n : 0];
        s.res = res[a.res ? (size_t)mr * a.N + 16l * t + n : 0];
#pragma unroll
        for (int i = 0; i < NC; ++i)
            s.w[i] = q4_load_w<G>(a.codes + t * tile_codes, a.scales + t * tile_scales, at[i], sat[i]);
        return s;
    };
    q4_stage<NC, G> st = load(blockIdx.x);
    q4_power own[NC];
    bool plain = false;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const q4_seen seen = q4_look<MT>(xr[i]);
        own[i] = seen.own;
        plain |= seen.plain;
    }
    if (lane == 0) left[w] = plain;
    f16x8 x[NC][4];
    float e[NC][2];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        q4_split_x<MT>(xr[i], own[i], xs[w], xe[w], lane, e[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = *(const f16x8 *)(xs[w] + (lane & (ROWS - 1)) * Q4_XROW + 8 * (lane >> 4) + 32 * j);
        __builtin_amdgcn_wave_barrier();
    }
    int b = 0;
    for (int t = blockIdx.x; t < tiles; t += step) {
        b ^= 1;
        float y[2] = {};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (w + KW * i < chunks) {
                if (w + KW * i == ql.last) q4_shift(st.w[i].w, ql.shift);
                q4_products<MT, G>(x[i], st.w[i].w, st.w[i].s, e[i], y);
            }
        }
        const float add = (a.bias ? st.bias : 0.f) + (a.res ? st.res : 0.f);
        st = load(t + step);
        q4_put<MT>(red[b][w], lane, y);
        __syncthreads();
        if (t == (int)blockIdx.x) /* (before the first output) */
            if (__builtin_expect(__builtin_amdgcn_readfirstlane(wave_any(left[lane % KW])), 0)) {
                float(*one)[1][MT][16] = (float(*)[1][MT][16])red[0];
#pragma unroll 1
                for (; t < tiles; t += step) {
                    const uint8_t *codes = a.codes + t * tile_codes;
                    const uint16_t *scales = a.scales + t * tile_scales;
                    float y[1][2] = {};
#pragma unroll 1
                    for (int c = w; c < chunks; c += KW) q4_add_plain<MT, 1, G>(a, m0, c, lane, &codes, &scales, ql, y);
                    q4_put<MT>(one[w][0], lane, y[0]);
                    __syncthreads();
                    q4_outputs<MT, KW, 1>(a, t, m0, one);
                    __syncthreads();
                }
                return;
            }
        if (m < MT && 16l * t + r < a.N && m0 + m < a.M) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < KW; ++k) v += red[b][k][m][r];
            v += add;
            a.y[(size_t)(m0 + m) * a.N + 16l * t + r] = a.gelu ? gelu_f(v) : v;
        }
    }
}
/* (WAVES: of a SIMD, which the registers leave resident: see g2i_q4_form) */
#define Q4_HELD_G(MT, KW, NC, WAVES, G)                                                                                \
    extern "C" __global__ __launch_bounds__(64 * KW) __attribute__((amdgpu_waves_per_eu(WAVES)))                       \
    void g2k_q4_mvh##MT##_##KW##_##NC##_##G(const g2_q4mv_args a) { q4_held_impl<MT, KW, NC, G>(a); }
#define Q4_HELD(MT, KW, NC, WAVES)                                                                                     \
    Q4_HELD_G(MT, KW, NC, WAVES, 32) Q4_HELD_G(MT, KW, NC, WAVES, 64) Q4_HELD_G(MT, KW, NC, WAVES, 128)
Q4_HELD(1, 8, 1, 6)
Q4_HELD(1, 8, 2, 6)
Q4_HELD(8, 8, 1, 6)
Q4_HELD(8, 8, 2, 4)
Q4_HELD(8, 16, 2, 4)

/* ======================================================================
 * 8-bit K/V cache: a block of 16 positions of one head holds the codes
 * rint(fp32(x / scale)), scale = fp32(max |x| / 127), and stands for code *
 * scale; the positions of a sequence's last block stand in fp32 until the
 * block is full, so that what a cache holds does not depend on how many
 * positions came at a time; they are kept there when it is, until the next
 * block begins, so that a sequence can be cut back to any length in it.  A
 * block that holds an infinity or NaN gets a NaN scale.
 * ==================================================================== */

/* One wave per sequence, head, keys or values and block of the call; load i of
 * a lane is four dims of position 4 i + lane / 16, so that a load is 256 bytes
 * of each of four rows, and neighbouring waves have neighbouring heads.  The
 * first block's wave reads the positions that came before from `last` and then
 * writes there what the call has of its last block, full or not: in one wave,
 * since both may be the same rows.  Four prompts of 1001 rows x 25 heads: 13.0 us, 5.0
 * TB/s of the keys and values read and the codes written (17.3 when a reading
 * back just before had left its values in the L2, and 19.0 then with the blocks
 * of one head side by side, whose loads are 16 rows 19 KB apart); one token:
 * 3.3, the latency of a load, the maximum over the wave and a store. */
G2K void g2k_kv8_append(const g2_kv8_append_args a)
{
    const int lane = threadIdx.x & 63, t0 = lane >> 4, d0 = 4 * (lane & 15);
    const int D = a.NH * G2L_DH;
    int h, kv, i;
    long s;
    g2l_append_item(__builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), a.NH, a.T, &h, &kv, &i, &s);
    if (s >= a.S) return;
    const int p0 = a.pos ? a.pos[s] : a.start;
    int n = a.count ? (a.count[s] < a.T ? a.count[s] : a.T) : a.T;
    if (p0 < 0 || p0 >= a.max_seq || n <= 0) return;
    if (n > a.max_seq - p0) n = a.max_seq - p0;
    const int end = p0 + n, b = p0 / G2L_BLOCK + i;
    const float *rows = a.qkv + (size_t)s * a.T * 3 * D + (1 + kv) * D + h * G2L_DH + d0;
    float *last = a.last + g2l_kv_last_at(a.NH, s, h, kv) + d0;
    if ((b + 1) * G2L_BLOCK <= end) {
        f32x4 x[4];
        unsigned amax = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = 4 * u + t0, p = b * G2L_BLOCK + t;
            x[u] = *(const f32x4u *)(p < p0 ? last + t * G2L_DH : rows + (size_t)(p - p0) * 3 * D);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned m = __float_as_uint(x[u][e]) & 0x7FFFFFFF;
                amax = m > amax ? m : amax;
            }
        amax = q4_group_max(amax, 128); /* 16 lanes */
        const unsigned r0 = __builtin_amdgcn_readlane(amax, 0), r1 = __builtin_amdgcn_readlane(amax, 16);
        const unsigned r2 = __builtin_amdgcn_readlane(amax, 32), r3 = __builtin_amdgcn_readlane(amax, 48);
        const unsigned m0 = r0 > r1 ? r0 : r1, m1 = r2 > r3 ? r2 : r3;
        amax = m0 > m1 ? m0 : m1;
        const float sc = amax < 0x7F800000u ? __uint_as_float(amax) / 127.0f : __uint_as_float(0x7FC00000u);
        int8_t *codes = a.codes + g2l_kv_code_at(a.NH, a.blocks, s, h, b, kv) + d0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            unsigned w = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float r = fminf(fmaxf(rintf(x[u][e] / sc), -127.f), 127.f);
                w |= (sc > 0.f ? (unsigned)(int)r & 255u : 0u) << 8 * e;
            }
            *(unsigned *)(codes + (4 * u + t0) * G2L_DH) = w;
        }
        if (lane == 0) a.scales[g2l_kv_scale_at(a.NH, a.blocks, s, h, b, kv)] = sc;
    }
    if (i) return;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int t = 4 * u + t0, p = (end - 1) / G2L_BLOCK * G2L_BLOCK + t;
        if (p >= p0 && p < end) *(f32x4 *)(last + t * G2L_DH) = *(const f32x4u *)(rows + (size_t)(p - p0) * 3 * D);
    }
}

__device__ __forceinline__ int kv8_length(const int *len, int T_kv, long s)
{
    if (!len) return T_kv;
    const int n = len[s];
    return n < 0 ? 0 : n < T_kv ? n : T_kv;
}

/* One thread per four dims of a position, keys and values; positions in the
 * order of the output.  Four times 1001 positions x 25 heads 12.4 us, 5.2 TB/s,
 * four fifths of it written (41 with a thread per value). */
G2K void g2k_kv8_read(const g2_kv8_read_args a)
{
    const int quads = a.NH * (G2L_DH / 4);
    const long n = (long)a.S * a.T * quads;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += gridDim.x * 256l) {
        const long row = n <= UINT32_MAX ? (unsigned)i / (unsigned)quads : i / quads;
        const int q = (int)(i - row * quads), h = q / (G2L_DH / 4), d = q % (G2L_DH / 4) * 4;
        const long s = a.S == 1 ? 0 : (unsigned)row / (unsigned)a.T;
        const int p = a.start + (int)(row - s * a.T), len = kv8_length(a.len, a.T_kv, s);
        if (p >= len) continue;
        const int at = p % G2L_BLOCK * G2L_DH + d, b = p / G2L_BLOCK;
        f32x4 kv[2];
        if (b < len / G2L_BLOCK) {
            const size_t c = g2l_kv_code_at(a.NH, a.blocks, s, h, b, 0) + at;
            const float *sc = a.scales + g2l_kv_scale_at(a.NH, a.blocks, s, h, b, 0);
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
                const unsigned w = *(const unsigned *)(a.codes + c + i2 * (G2L_BLOCK * G2L_DH));
                const float f = sc[i2];
#pragma unroll
                for (int e = 0; e < 4; ++e) kv[i2][e] = (float)(int8_t)(w >> 8 * e) * f;
            }
        } else {
            const float *l = a.last + g2l_kv_last_at(a.NH, s, h, 0) + at;
            kv[0] = *(const f32x4 *)l;
            kv[1] = *(const f32x4 *)(l + G2L_BLOCK * G2L_DH);
        }
        __builtin_nontemporal_store(kv[0], (f32x4u *)(a.k + 4 * i));
        __builtin_nontemporal_store(kv[1], (f32x4u *)(a.v + 4 * i));
    }
}

/* ---- single-query attention.  A wave takes four blocks (64 positions) at a
 * time: 1 KB of keys and 1 KB of values each, every lane 16 bytes of one
 * position, so that the codes are used where they were loaded: the four lanes
 * of a position add up its score, and each weighs its own 16 dims of the
 * value.  Each position slot (16 a wave) keeps a running maximum and sum of
 * its own; they meet once, at the end: over the lanes, over the waves in LDS,
 * and over the parts of a long sequence in a second launch.  Scores are held
 * in units of log 2, the queries carrying the factor.
 *
 * Bounded by HBM for many or long sequences (48 x 25 heads x 1024 28 us, 5.7
 * TB/s; 16 heads x 50001 18 us and 4 to join, 4.7 TB/s; a wave for each head, a
 * position at a time, took 35 ms there), by latency for one short
 * sequence (12 heads x 701 5.2 us: the launch, the length, two rounds of
 * loads, the sums over lanes and waves).  The next four blocks' loads go out
 * before the last ones' sums, and the sums over the lanes need no LDS (25 heads
 * x 1024 6.4 us, 7.2 without either). */

/* The 16 dims of a wave's lane: lane l has position l / 4 of a block, dims 16
 * (l % 4) .. + 15. */
struct kv16 { f32x4 v[4]; };
__device__ __forceinline__ kv16 kv_load(const float *p)
{
    kv16 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = *(const f32x4u *)(p + 4 * i);
    return r;
}
struct kv8_sum {
    float m, l, o[16];
};

__device__ __forceinline__ float kv8_byte(unsigned w, int i) { return (float)(int8_t)(w >> 8 * i); }

__device__ __forceinline__ float dpp_quad_sum(float v)
{
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, false)); /* lanes 1 0 3 2 */
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, false)); /* 2 3 0 1 */
}

/* The weight that a state of maximum m has beside one of maximum top (an empty
 * state's maximum is -infinity; all empty: 0). */
__device__ __forceinline__ float kv8_factor(float m, float top) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top); }

/* Adds N positions' scores and values (codes times vs, or fp32) to a state. */
template <int N, typename V>
__device__ __forceinline__ void kv8_add(kv8_sum &a, const float *s, const float *vs, V value)
{
    float top = a.m;
#pragma unroll
    for (int u = 0; u < N; ++u) top = fmaxf(top, s[u]);
    const float base = top == -INFINITY ? 0.f : top, f = __builtin_amdgcn_exp2f(a.m - base);
    float p[N], l = 0.f;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        p[u] = __builtin_amdgcn_exp2f(s[u] - base);
        l += p[u];
        p[u] *= vs[u];
    }
    a.l = fmaf(a.l, f, l);
    a.m = top;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float o = a.o[e] * f;
#pragma unroll
        for (int u = 0; u < N; ++u) o = fmaf(p[u], value(u, e), o);
        a.o[e] = o;
    }
}

/* Four blocks' codes and scales; a block behind the last one of the part is the
 * last again.  (Asking for the first four by the bound of the lengths, before
 * the length is there, saved 0.1 us where they were needed and cost up to half
 * the time of many short sequences under a high bound.)  Codes are read once:
 * loads that do not stay in the L2 (48 x 25 heads x 1024 28.0 us, ordinary ones
 * 32.8; 16 heads x 50001 21.8, 23.1; a few heads the same). */
struct kv8_four {
    u32x4 k[4], v[4];
    float sk[4], sv[4];
};
__device__ __forceinline__ kv8_four kv8_load(const int8_t *codes, const float *scales, int b, int last, int lane)
{
    kv8_four r;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int bu = b + u < last ? b + u : last;
        const int8_t *p = codes + (size_t)bu * (2 * G2L_BLOCK * G2L_DH) + 16 * lane;
        r.k[u] = __builtin_nontemporal_load((const u32x4 *)p);
        r.v[u] = __builtin_nontemporal_load((const u32x4 *)(p + G2L_BLOCK * G2L_DH));
        r.sk[u] = scales[2 * bu];
        r.sv[u] = scales[2 * bu + 1];
    }
    return r;
}

/* Exchange with the lane whose number differs in one bit (4, 8; 16 and 32 below). */
__device__ __forceinline__ float lane_xor4(float v)
{
    const int m = __builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, false); /* i ^ 7 */
    return __int_as_float(__builtin_amdgcn_mov_dpp(m, 0x1B, 0xF, 0xF, false));         /* i ^ 3 */
}
__device__ __forceinline__ float lane_xor8(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, false)); /* rows of 16 turned by 8 */
}
/* lo of this lane and its partner's where the lane's bit is 0, hi of both where it is 1 */
__device__ __forceinline__ float lane_fold32(float lo, float hi)
{
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float lane_fold16(float lo, float hi)
{
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float slots_max(float v)
{
    v = fmaxf(v, lane_xor4(v));
    v = fmaxf(v, lane_xor8(v));
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int NW>
__device__ void kv8_attn_impl(const g2_kv8_attn_args &a)
{
    __shared__ float part[NW][G2L_PART_FLOATS];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t = lane >> 2, d0 = 16 * (lane & 3);
    const int split = blockIdx.x % a.splits, h = blockIdx.x / a.splits % a.NH;
    const long s = blockIdx.x / a.splits / a.NH;
    const int8_t *codes = a.codes + g2l_kv_code_at(a.NH, a.blocks, s, h, 0, 0);
    const float *scales = a.scales + g2l_kv_scale_at(a.NH, a.blocks, s, h, 0, 0);
    const int first = g2l_attn_first(split, a.span, w);
    kv16 q = kv_load(a.q + s * a.q_stride + h * G2L_DH + d0);
    const int len = kv8_length(a.len, a.T_kv, s), full = len / G2L_BLOCK;
    const int b1 = g2l_attn_end(split, a.span, full);
    /* (without a branch, which the compiler makes a wait of; a wave without blocks reads one that it does not use) */
    kv8_four next = kv8_load(codes, scales, first, b1 > 0 ? b1 - 1 : 0, lane);
    const float qf = a.scale * 1.44269504f;
#pragma unroll
    for (int e = 0; e < 16; ++e) q.v[e / 4][e % 4] *= qf;
    kv8_sum st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) st.o[e] = 0.f;
    for (int b = first; b < b1; b += g2l_attn_step(NW)) {
        const kv8_four f = next;
        if (b + g2l_attn_step(NW) < b1) next = kv8_load(codes, scales, b + g2l_attn_step(NW), b1 - 1, lane);
        float x[4], sv[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) d = fmaf(q.v[e / 4][e % 4], kv8_byte(f.k[u][e / 4], e % 4), d);
            x[u] = b + u < b1 ? dpp_quad_sum(d) * f.sk[u] : -INFINITY;
            sv[u] = b + u < b1 ? f.sv[u] : 0.f;
        }
        kv8_add<4>(st, x, sv, [&](int u, int e) { return kv8_byte(f.v[u][e / 4], e % 4); });
    }
    /* the block that is not full, in the part that holds its place: the next wave in turn */
    const int left = len % G2L_BLOCK;
    if (left && g2l_attn_left(split, a.span, full, w, NW)) {
        const float *p = a.last + g2l_kv_last_at(a.NH, s, h, 0) + t * G2L_DH + d0;
        kv16 k = {}, v = {};
        if (t < left) {
            k = kv_load(p);
            v = kv_load(p + G2L_BLOCK * G2L_DH);
        }
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) d = fmaf(q.v[e / 4][e % 4], k.v[e / 4][e % 4], d);
        d = dpp_quad_sum(d);
        const float x = t < left ? d : -INFINITY, one = 1.f;
        kv8_add<1>(st, &x, &one, [&](int, int e) { return v.v[e / 4][e % 4]; });
    }
    /* the wave's 16 position slots: each step halves the dims that a lane keeps */
    float top = slots_max(st.m);
    const float f = kv8_factor(st.m, top);
    float l = st.l * f;
    l += lane_xor4(l);
    l += lane_xor8(l);
    l = lane_fold16(l, l);
    l = lane_fold32(l, l);
#pragma unroll
    for (int e = 0; e < 16; ++e) st.o[e] *= f;
#pragma unroll
    for (int e = 0; e < 8; ++e) st.o[e] = lane_fold32(st.o[e], st.o[e + 8]);
#pragma unroll
    for (int e = 0; e < 4; ++e) st.o[e] = lane_fold16(st.o[e], st.o[e + 4]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float lo = st.o[e] + lane_xor8(st.o[e]), hi = st.o[e + 2] + lane_xor8(st.o[e + 2]);
        st.o[e] = lane & 8 ? hi : lo;
    }
    {
        const float lo = st.o[0] + lane_xor4(st.o[0]), hi = st.o[1] + lane_xor4(st.o[1]);
        st.o[0] = lane & 4 ? hi : lo;
    }
    if (NW > 1 || a.splits > 1) {
        if (lane == 0) { part[w][0] = top; part[w][1] = l; }
        part[w][2 + d0 + t] = st.o[0];
        __syncthreads();
        if (tid >= 64) return;
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NW; ++i) top = fmaxf(top, part[i][0]);
        float o = 0.f;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float g = kv8_factor(part[i][0], top);
            l = fmaf(part[i][1], g, l);
            o = fmaf(part[i][2 + lane], g, o);
        }
        if (a.splits > 1) {
            float *r = a.part + ((s * a.NH + h) * a.splits + split) * G2L_PART_FLOATS;
            if (lane == 0) { r[0] = top; r[1] = l; }
            r[2 + lane] = o;
            return;
        }
        a.out[s * a.out_stride + h * G2L_DH + lane] = len ? o / l : 0.f;
    } else
        a.out[s * a.out_stride + h * G2L_DH + d0 + t] = len ? st.o[0] / l : 0.f;
}
extern "C" __global__ __launch_bounds__(64) void g2k_kv8_attn1(const g2_kv8_attn_args a) { kv8_attn_impl<1>(a); }
extern "C" __global__ __launch_bounds__(256) void g2k_kv8_attn4(const g2_kv8_attn_args a) { kv8_attn_impl<4>(a); }
extern "C" __global__ __launch_bounds__(512) void g2k_kv8_attn8(const g2_kv8_attn_args a) { kv8_attn_impl<8>(a); }

/* Joins the parts of a head: four waves of eight parts each (all their loads
 * at once: one after the other they took 11 us for 32), then the waves. */
G2K void g2k_kv8_join(const g2_kv8_attn_args a)
{
    __shared__ float part[4][G2L_PART_FLOATS];
    const int h = blockIdx.x % a.NH, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const long s = blockIdx.x / a.NH;
    const float *r = a.part + (s * a.NH + h) * a.splits * G2L_PART_FLOATS;
    float m[G2L_SPLITS / 4], l[G2L_SPLITS / 4], v[G2L_SPLITS / 4], top = -INFINITY, o = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < G2L_SPLITS / 4; ++i) {
        const int n = w * (G2L_SPLITS / 4) + i;
        const float *p = r + (n < a.splits ? n : a.splits - 1) * G2L_PART_FLOATS;
        m[i] = p[0];
        l[i] = p[1];
        v[i] = p[2 + lane];
        if (n >= a.splits) m[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < G2L_SPLITS / 4; ++i) top = fmaxf(top, m[i]);
#pragma unroll
    for (int i = 0; i < G2L_SPLITS / 4; ++i) {
        const float f = kv8_factor(m[i], top);
        if (w * (G2L_SPLITS / 4) + i >= a.splits) continue;
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
    a.out[s * a.out_stride + h * G2L_DH + lane] = kv8_length(a.len, a.T_kv, s) ? o / sum : 0.f;
}

/* ======================================================================
 * Rules on logits (see g2_logit_rules): ids of the context are counted per
 * slice of the vocabulary in LDS (integers, so no order of the atomics
 * changes anything), the bias list likewise keeps an id's last entry; then
 * one pass over the slice's logits.  Every step is its own fp32 rounding (no
 * fused multiply-add), so equal logits stay equal.
 * ==================================================================== */
/* Maximum, minimum over the wave. */
__device__ __forceinline__ float lanes_max(float v)
{
    v = dpp_max<0xB1>(v);  /* quad: lanes 1 0 3 2 */
    v = dpp_max<0x4E>(v);  /* 2 3 0 1 */
    return slots_max(v);
}
__device__ __forceinline__ unsigned lanes_min(unsigned v)
{
#define LANES_MIN(CTRL) { const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false); v = o < v ? o : v; }
    LANES_MIN(0xB1) LANES_MIN(0x4E) LANES_MIN(0x141) LANES_MIN(0x140)
#undef LANES_MIN
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = s[0] < s[1] ? s[0] : s[1];
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] < r[1] ? r[0] : r[1];
}

/* A logit and its id as one number: greater for a greater logit, of equal ones
 * for the lower id; 0 is below all (-infinity and NaN have none). */
__device__ __forceinline__ unsigned long long logit_key(float v, int id)
{
    const unsigned u = __float_as_uint(v + 0.f); /* (-0 counts as 0) */
    return (unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (unsigned)~id;
}

template <int THREADS, int QUADS>
__device__ void logits_impl(const g2_logits_args &a)
{
#pragma clang fp contract(off)
    constexpr int SLICE = THREADS * QUADS * 4;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    __shared__ i32x4 seen[SLICE / 4]; /* an id's times in the context; 65536 times its entry of the bias list + 1 */
    __shared__ unsigned long long keys[THREADS / 64];
    const int tid = threadIdx.x, row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int v0 = part * SLICE, nv = a.V - v0 < SLICE ? a.V - v0 : SLICE;
    const float *in = a.logits + (size_t)row * a.V + v0;
    float *out = a.out + (size_t)row * a.V + v0;
    f32x4 x[QUADS];
    unsigned allowed[QUADS];
#pragma unroll
    for (int q = 0; q < QUADS; ++q) { /* in flight while the ids are counted */
        const int i = 4 * (tid + THREADS * q);
        if (i + 4 <= nv) x[q] = *(const f32x4u *)(in + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) x[q][e] = i + e < nv ? in[i + e] : -INFINITY;
        const int v = v0 + (i < nv ? i : 0);
        allowed[q] = a.mask ? a.mask[(size_t)row * a.mask_stride + (v >> 5)] >> (v & 31) : 15u;
    }
    /* so are the first entries of the lists, to ids that are none where there are fewer */
    const int *ctx = a.ctx + (size_t)row * a.max_ctx;
    int id = -1, bid = -1;
    if (a.ctx) id = ctx[tid < a.max_ctx ? tid : 0];
    if (a.n_bias) bid = a.bias_id[tid < a.n_bias ? tid : 0];
    const int n = !a.ctx ? 0 : a.ctx_len ? clampi(a.ctx_len[row], 0, a.max_ctx) : a.max_ctx;
#pragma unroll
    for (int q = 0; q < QUADS; ++q) seen[tid + THREADS * q] = i32x4{ 0, 0, 0, 0 };
    __syncthreads();
    for (int i = tid; i < a.n_bias; i += THREADS) {
        const unsigned k = (unsigned)(i == tid ? bid : a.bias_id[i]) - (unsigned)v0;
        if (k < (unsigned)nv) atomicMax((unsigned *)seen + k, (unsigned)(i + 1) << 16);
    }
    if (a.n_bias) __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
        const unsigned k = (unsigned)(i == tid ? id : ctx[i]) - (unsigned)v0;
        if (k < (unsigned)nv) atomicAdd((unsigned *)seen + k, 1u);
    }
    __syncthreads();
    float best = -INFINITY;
    int at = 0; /* 4 q + e of the best */
#pragma unroll
    for (int q = 0; q < QUADS; ++q) {
        const int i = 4 * (tid + THREADS * q);
        const i32x4 s = seen[tid + THREADS * q];
        if (s[0] | s[1] | s[2] | s[3]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y = x[q][e];
                const unsigned n = s[e] & 65535, l = (unsigned)s[e] >> 16;
                if (n) {
                    y = y > 0.f ? y / a.repetition : y * a.repetition;
                    y = y - a.frequency * (float)n - a.presence;
                }
                if (l) y = y + a.bias[l - 1];
                x[q][e] = y;
            }
        }
        if (a.mask || a.forbid >= 0) { /* (uniform) */
            const unsigned f = (unsigned)(a.forbid - v0 - i);
            const unsigned ok = f < 4u ? allowed[q] & ~(1u << f) : allowed[q];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[q][e] = ok >> e & 1 ? x[q][e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) /* (ids behind the slice are -infinity) */
            if (x[q][e] > best) { best = x[q][e]; at = 4 * q + e; }
        if (a.out) {
            if (i + 4 <= nv) *(f32x4u *)(out + i) = x[q];
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < nv) out[i + e] = x[q][e];
        }
    }
    if (!a.pick) return;
    /* the wave's best value, the lowest id that has it, the slice's best key */
    const float top = lanes_max(best);
    const int mine = v0 + 4 * (tid + THREADS * (at >> 2)) + (at & 3);
    const unsigned low = lanes_min(best == top && best > -INFINITY ? (unsigned)mine : ~0u);
    unsigned long long key = low == ~0u ? 0 : logit_key(top, (int)low);
    if ((tid & 63) == 0) keys[tid >> 6] = key;
    __syncthreads();
    if (tid) return;
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) key = keys[w] > key ? keys[w] : key;
    if (a.parts > 1) {
        unsigned long long *cell = a.cells + G2L_CELL * (size_t)row;
        /* the maximum has its old value back, so it is done, before the count goes up */
        const unsigned long long was = __hip_atomic_fetch_max(cell, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const unsigned long long one = was == ~0ull ? 2 : 1; /* (1: no key is all ones) */
        if (__hip_atomic_fetch_add(cell + 1, one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (unsigned)a.parts - 1) return;
        key = __hip_atomic_exchange(cell, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(cell + 1, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    a.pick[row] = key ? (int)~(unsigned)key : -1;
}
G2K void g2k_logits(const g2_logits_args a) { logits_impl<256, 1>(a); }
extern "C" __global__ __launch_bounds__(1024) void g2k_logits_wide(const g2_logits_args a) { logits_impl<1024, 2>(a); }


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

__device__ __forceinline__ unsigned q4_code(float w, float s)
{
    const float q = w / s, a = fabsf(q);
    const unsigned c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
    return s > 0.f && c ? c | (q < 0.f ? 8u : 0u) : 0u;
}

__device__ __forceinline__ float q4_value(unsigned code)
{
    const unsigned e = (code >> 1) & 3, m = code & 1;
    const float v = e ? (float)((2 + m) << e) * 0.25f : 0.5f * (float)m;
    return code & 8 ? -v : v;
}

/* One thread per row and group. */
template <typename WT>
__device__ void q4_pack_impl(const g2_q4_args &a)
{
    const WT *W = (const WT *)a.W;
    const int gpc = 128 / a.group;
    const long groups = g2l_chunks(a.K) * gpc, rows = g2l_tiles(a.N) * 16;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < rows * groups; i += gridDim.x * 256l) {
        const long n = i / groups, g = i % groups, t = n / 16;
        const int r = (int)(n % 16);
        const long k0 = g * a.group, k1 = k0 + a.group < 32 * g2l_steps(a.K) ? k0 + a.group : 32 * g2l_steps(a.K);
        const size_t sn = a.in_out ? 1 : (size_t)a.K, sk = a.in_out ? (size_t)a.N : 1;
        unsigned amax = 0;
        for (long k = k0; k < k1; ++k)
            if (n < a.N && k < a.K) {
                const unsigned u = __float_as_uint(ldw<WT>(W, n * sn + k * sk)) & 0x7FFFFFFF;
                amax = u > amax ? u : amax;
            }
        const uint16_t sb = q4_scale(amax);
        const float s = bf16_f(sb);
        a.scales[g2l_scale_at(a.K, a.group, t, g / gpc, r, (int)(g % gpc))] = sb;
        for (long k = k0; k < k1; k += 2) {
            unsigned b = 0;
            for (int h = 0; h < 2; ++h)
                if (n < a.N && k + h < a.K) b |= q4_code(ldw<WT>(W, n * sn + (k + h) * sk), s) << 4 * h;
            const long c = k / 128;
            const int j = (int)(k % 128 / 32), place = (int)(k % 32 / 8);
            a.codes[g2l_code_at(a.K, t, c, 16 * place + r) + 4 * j + k % 8 / 2] = (uint8_t)b;
        }
    }
}
G2K void g2k_q4_pack_f32(const g2_q4_args a) { q4_pack_impl<float>(a); }
G2K void g2k_q4_pack_f16(const g2_q4_args a) { q4_pack_impl<_Float16>(a); }

__device__ __forceinline__ float q4_at(const uint8_t *codes, const uint16_t *scales, long K, int group, long n, long k)
{
    const long t = n / 16, c = k / 128;
    const int r = (int)(n % 16), j = (int)(k % 128 / 32), place = (int)(k % 32 / 8);
    const unsigned b = codes[g2l_code_at(K, t, c, 16 * place + r) + 4 * j + k % 8 / 2];
    return q4_value(b >> 4 * (k & 1) & 15) * bf16_f(scales[g2l_scale_at(K, group, t, c, r, (int)(k % 128) / group)]);
}

/* One thread per weight. */
G2K void g2k_q4_read(const g2_q4_args a)
{
    for (long i = blockIdx.x * 256l + threadIdx.x; i < (long)a.N * a.K; i += gridDim.x * 256l) {
        const long n = a.in_out ? i % a.N : i / a.K, k = a.in_out ? i / a.N : i % a.K;
        a.out[i] = q4_at(a.codes, a.scales, a.K, a.group, n, k);
    }
}

/* One work-group per output. */
G2K void g2k_q4_matvec(const g2_q4mv_args a)
{
    __shared__ float red[4];
    const long n = blockIdx.x, m = blockIdx.y;
    float s = 0.f;
    for (long k = threadIdx.x; k < a.K; k += 256)
        s = fmaf(q4_at(a.codes, a.scales, a.K, a.group, n, k), a.x[m * a.K + k], s);
    s = block_sum(s, red);
    if (threadIdx.x == 0) {
        if (a.bias) s += a.bias[n];
        if (a.res) s += a.res[m * a.N + n];
        a.y[m * a.N + n] = a.gelu ? gelu_f(s) : s;
    }
}

/* ======================================================================
 * 8-bit K/V cache: a block of 16 positions of one head holds the codes
 * rint(fp32(x / scale)), scale = fp32(max |x| / 127), and stands for code *
 * scale; the positions of a sequence's last block stand in fp32 until the
 * block is full, so that what a cache holds does not depend on how many
 * positions came at a time.  A block that holds an infinity or NaN gets a
 * NaN scale.
 * ==================================================================== */

/* The 16 dims of a wave's lane: lane l has position l / 4 of the block, dims
 * 16 (l % 4) .. + 15. */
struct kv16 { f32x4 v[4]; };
__device__ __forceinline__ kv16 kv_load(const float *p)
{
    kv16 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = *(const f32x4u *)(p + 4 * i);
    return r;
}

/* One wave per sequence, head, keys or values and block of the call; the
 * first block's wave reads the positions that came before from `last` and
 * then writes there what the call leaves of its last block: in one wave,
 * since both may be the same rows. */
G2K void g2k_kv8_append(const g2_kv8_append_args a)
{
    const int lane = threadIdx.x & 63, t = lane >> 2, d0 = 16 * (lane & 3);
    const int per = a.T / G2L_BLOCK + 2, D = a.NH * G2L_DH;
    const long item = blockIdx.x * 4l + (threadIdx.x >> 6);
    const int i = (int)(item % per), kv = (int)(item / per % 2), h = (int)(item / per / 2 % a.NH);
    const long s = item / per / 2 / a.NH;
    if (s >= a.S) return;
    const int p0 = a.pos ? a.pos[s] : a.start;
    int n = a.count ? (a.count[s] < a.T ? a.count[s] : a.T) : a.T;
    if (p0 < 0 || p0 >= a.max_seq || n <= 0) return;
    if (n > a.max_seq - p0) n = a.max_seq - p0;
    const int end = p0 + n, first = p0 / G2L_BLOCK, b = first + i;
    const float *rows = a.qkv + (size_t)s * a.T * 3 * D + (1 + kv) * D + h * G2L_DH + d0;
    float *last = a.last + g2l_kv_last_at(a.NH, s, h, kv) + t * G2L_DH + d0;
    if ((b + 1) * G2L_BLOCK <= end) {
        const int p = b * G2L_BLOCK + t;
        const kv16 x = kv_load(p < p0 ? last : rows + (size_t)(p - p0) * 3 * D);
        unsigned amax = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const unsigned u = __float_as_uint(x.v[e / 4][e % 4]) & 0x7FFFFFFF;
            amax = u > amax ? u : amax;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned u = __shfl_xor(amax, o);
            amax = u > amax ? u : amax;
        }
        const float sc = amax < 0x7F800000u ? __uint_as_float(amax) / 127.0f : __uint_as_float(0x7FC00000u);
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            unsigned u = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float r = fminf(fmaxf(rintf(x.v[q][e] / sc), -127.f), 127.f);
                u |= (sc > 0.f ? (unsigned)(int)r & 255u : 0u) << 8 * e;
            }
            w[q] = u;
        }
        *(u32x4 *)(a.codes + g2l_kv_code_at(a.NH, a.blocks, s, h, b, kv) + 16 * lane) = w;
        if (lane == 0) a.scales[g2l_kv_scale_at(a.NH, a.blocks, s, h, b, kv)] = sc;
    }
    const int p = end / G2L_BLOCK * G2L_BLOCK + t;
    if (i == 0 && p >= p0 && p < end) {
        const kv16 x = kv_load(rows + (size_t)(p - p0) * 3 * D);
#pragma unroll
        for (int q = 0; q < 4; ++q) *(f32x4 *)(last + 4 * q) = x.v[q];
    }
}

__device__ __forceinline__ int kv8_length(const int *len, int T_kv, long s)
{
    if (!len) return T_kv;
    const int n = len[s];
    return n < 0 ? 0 : n < T_kv ? n : T_kv;
}

/* One thread per value. */
G2K void g2k_kv8_read(const g2_kv8_read_args a)
{
    const int D = a.NH * G2L_DH;
    const long n = (long)a.S * a.T * D;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < 2 * n; i += gridDim.x * 256l) {
        const int kv = i >= n;
        const long j = kv ? i - n : i, s = j / D / a.T;
        const int c = (int)(j % D), p = a.start + (int)(j / D % a.T), len = kv8_length(a.len, a.T_kv, s);
        if (p >= len) continue;
        const int h = c / G2L_DH, at = p % G2L_BLOCK * G2L_DH + c % G2L_DH, b = p / G2L_BLOCK;
        const float v = b < len / G2L_BLOCK
                            ? (float)a.codes[g2l_kv_code_at(a.NH, a.blocks, s, h, b, kv) + at] *
                                  a.scales[g2l_kv_scale_at(a.NH, a.blocks, s, h, b, kv)]
                            : a.last[g2l_kv_last_at(a.NH, s, h, kv) + at];
        (kv ? a.v : a.k)[j] = v;
    }
}

/* One wave per sequence and head, a lane per dim, one position at a time
 * with the running maximum and sum of the softmax. */
extern "C" __global__ __launch_bounds__(64) void g2k_kv8_attn(const g2_kv8_attn_args a)
{
    const int h = blockIdx.x % a.NH, d = threadIdx.x;
    const long s = blockIdx.x / a.NH;
    const int len = kv8_length(a.len, a.T_kv, s);
    const float q = a.q[s * a.q_stride + h * G2L_DH + d];
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int p = 0; p < len; ++p) {
        const int b = p / G2L_BLOCK, at = p % G2L_BLOCK * G2L_DH + d;
        float kv[2];
        for (int i = 0; i < 2; ++i)
            kv[i] = b < len / G2L_BLOCK ? (float)a.codes[g2l_kv_code_at(a.NH, a.blocks, s, h, b, i) + at] *
                                              a.scales[g2l_kv_scale_at(a.NH, a.blocks, s, h, b, i)]
                                        : a.last[g2l_kv_last_at(a.NH, s, h, i) + at];
        const float x = wave_sum(q * kv[0]) * a.scale, top = fmaxf(m, x), f = expf(m - top), e = expf(x - top);
        l = l * f + e;
        o = o * f + e * kv[1];
        m = top;
    }
    a.out[s * a.out_stride + h * G2L_DH + d] = len ? o / l : 0.f;
}

/* ======================================================================
 * Rules on logits (see g2_logit_rules): ids of the context are counted per
 * slice of the vocabulary in LDS (integers, so no order of the atomics
 * changes anything), the bias list likewise keeps an id's last entry; then
 * one pass over the slice's logits.  Every step is its own fp32 rounding (no
 * fused multiply-add), so equal logits stay equal.
 * ==================================================================== */
G2K void g2k_logits(const g2_logits_args a)
{
#pragma clang fp contract(off)
    __shared__ int hits[2 * G2L_SLICE]; /* [slice] counts, [slice] entry of the bias list + 1 */
    __shared__ float bv[4];
    __shared__ int bi[4];
    const int tid = threadIdx.x, row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const int v0 = part * a.slice, nv = a.V - v0 < a.slice ? a.V - v0 : a.slice;
    for (int i = tid; i < 2 * a.slice; i += 256) hits[i] = 0;
    __syncthreads();
    if (a.ctx) {
        const int n = a.ctx_len ? clampi(a.ctx_len[row], 0, a.max_ctx) : a.max_ctx;
        for (int i = tid; i < n; i += 256) {
            const unsigned id = (unsigned)a.ctx[(size_t)row * a.max_ctx + i] - (unsigned)v0;
            if (id < (unsigned)nv) atomicAdd(&hits[id], 1);
        }
    }
    for (int i = tid; i < a.n_bias; i += 256) {
        const unsigned id = (unsigned)a.bias_id[i] - (unsigned)v0;
        if (id < (unsigned)nv) atomicMax(&hits[a.slice + id], i + 1);
    }
    __syncthreads();
    float best = -INFINITY;
    int at = -1;
    for (int i = tid; i < nv; i += 256) {
        const int v = v0 + i, n = hits[i], e = hits[a.slice + i];
        float x = a.logits[(size_t)row * a.V + v];
        if (n) {
            x = x > 0.f ? x / a.repetition : x * a.repetition;
            x = x - a.frequency * (float)n - a.presence;
        }
        if (e) x = x + a.bias[e - 1];
        if (v == a.forbid || (a.mask && !(a.mask[(size_t)row * a.mask_stride + (v >> 5)] >> (v & 31) & 1))) x = -INFINITY;
        if (a.out) a.out[(size_t)row * a.V + v] = x;
        if (x > best) { best = x; at = v; }
    }
    if (!a.part) return;
    for (int o = 32; o > 0; o >>= 1) {
        const float ov = __shfl_xor(best, o);
        const int oi = __shfl_xor(at, o);
        if (ov > best || (ov == best && (unsigned)oi < (unsigned)at)) { best = ov; at = oi; }
    }
    if ((tid & 63) == 0) { bv[tid >> 6] = best; bi[tid >> 6] = at; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 4; ++w)
            if (bv[w] > best || (bv[w] == best && (unsigned)bi[w] < (unsigned)at)) { best = bv[w]; at = bi[w]; }
        float *p = a.part + ((size_t)row * a.parts + part) * 2;
        p[0] = best;
        p[1] = __int_as_float(at);
    }
}

/* One wave per row: the best of its slices (at most 64). */
extern "C" __global__ __launch_bounds__(64) void g2k_logits_pick(const g2_logits_args a)
{
    const int i = threadIdx.x, row = blockIdx.x;
    const float *p = a.part + ((size_t)row * a.parts + i) * 2;
    float best = i < a.parts ? p[0] : -INFINITY;
    int at = i < a.parts ? __float_as_int(p[1]) : -1;
    for (int o = 32; o > 0; o >>= 1) {
        const float ov = __shfl_xor(best, o);
        const int oi = __shfl_xor(at, o);
        if (ov > best || (ov == best && (unsigned)oi < (unsigned)at)) { best = ov; at = oi; }
    }
    if (i == 0) a.pick[row] = at;
}

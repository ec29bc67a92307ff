/*
 * g2_lowbit_plan.h -- layouts of the 4-bit weights and of the 8-bit K/V
 * cache, shared by the C99 host (g2_lowbit.c), the gfx950 device code
 * (g2_lowbit.hip) and the CPU address checks.
 *
 * 4-bit weights W[N,K], group = 32, 64 or 128 columns to a scale.
 *  Codes: tiles of 16 rows; a tile holds its columns 32 at a time ("steps",
 *  ceil(K / 32) of them, 256 bytes each), four steps to a chunk.  In a chunk
 *  of r steps (4, or what is left in the last one) lane = 16 * place + row
 *  (place 0..3) has 4 * r bytes side by side: for each step 4 bytes with the
 *  columns 32 * step + 8 * place + 0..7, an even column in the low half of
 *  its byte.  That is the operand of one 16x16x32 matrix instruction a step,
 *  and a wave reads a chunk as one contiguous run.
 *  Scales (bf16): [tile][chunk][row][128 / group].
 *  Rows behind N and columns behind K have code 0, groups behind K scale 0.
 *
 * 8-bit cache of S sequences, NH heads of 64 dims, blocks of 16 positions:
 *  codes  [S][NH][blocks][K, V][16][64] int8,
 *  scales [S][NH][blocks][K, V] fp32 (padded to 256 bytes),
 *  last   [S][NH][K, V][16][64] fp32: the positions of the block that was
 *  appended to last, as they came.
 */
#ifndef G2_LOWBIT_PLAN_H
#define G2_LOWBIT_PLAN_H

#include <stddef.h>
#include <stdint.h>

#if defined(__HIPCC__) || defined(__HIP__)
#define G2L_FN __host__ __device__ __forceinline__
#else
#define G2L_FN static inline
#endif

/* ---- 4-bit weights */
G2L_FN long g2l_tiles(long N) { return (N + 15) / 16; }
G2L_FN long g2l_steps(long K) { return (K + 31) / 32; }
G2L_FN long g2l_chunks(long K) { return (K + 127) / 128; }
/* steps of chunk c */
G2L_FN int g2l_chunk_steps(long K, long c)
{
    const long left = g2l_steps(K) - 4 * c;
    return left < 4 ? (int)left : 4;
}
/* byte of the codes where lane `lane` of chunk c of tile t begins */
G2L_FN size_t g2l_code_at(long K, long t, long c, int lane)
{
    return ((size_t)t * g2l_steps(K) + 4 * c) * 256 + (size_t)lane * 4 * g2l_chunk_steps(K, c);
}
/* Where lane `lane` reads 16 bytes of chunk c, as bytes into the chunk.  A chunk
 * of fewer than four steps is read as if it had four: what lies behind a lane's
 * own bytes meets activations that are 0, and lanes that would read past the
 * chunk's end read up to it and move g2l_lane_shift words to their places. */
G2L_FN unsigned g2l_lane_at(long K, long c, int lane)
{
    const unsigned steps = (unsigned)g2l_chunk_steps(K, c), at = (unsigned)lane * 4 * steps, most = 256 * steps - 16;
    return at < most ? at : most;
}
G2L_FN int g2l_lane_shift(long K, long c, int lane)
{
    return (int)((unsigned)lane * 4 * (unsigned)g2l_chunk_steps(K, c) - g2l_lane_at(K, c, lane)) / 4;
}
/* element of the scales: row r (0..15) of tile t, group g of chunk c */
G2L_FN size_t g2l_scale_at(long K, int group, long t, long c, int r, int g)
{
    return (((size_t)t * g2l_chunks(K) + c) * 16 + r) * (128 / group) + g;
}
G2L_FN size_t g2l_code_bytes(long N, long K) { return (size_t)g2l_tiles(N) * g2l_steps(K) * 256; }
G2L_FN size_t g2l_scale_count(long N, long K, int group) { return (size_t)g2l_tiles(N) * g2l_chunks(K) * 16 * (128 / group); }

/* ---- 8-bit cache */
#define G2L_BLOCK 16
#define G2L_DH 64
G2L_FN long g2l_blocks(long max_seq) { return (max_seq + G2L_BLOCK - 1) / G2L_BLOCK; }
/* first code of block b of head h of sequence s (kv: 0 keys, 1 values) */
G2L_FN size_t g2l_kv_code_at(int NH, long nb, long s, int h, long b, int kv)
{
    return ((((size_t)s * NH + h) * nb + b) * 2 + kv) * (G2L_BLOCK * G2L_DH);
}
G2L_FN size_t g2l_kv_scale_at(int NH, long nb, long s, int h, long b, int kv)
{
    return (((size_t)s * NH + h) * nb + b) * 2 + kv;
}
G2L_FN size_t g2l_kv_last_at(int NH, long s, int h, int kv)
{
    return (((size_t)s * NH + h) * 2 + kv) * (G2L_BLOCK * G2L_DH);
}
/* byte offsets of the scales and of the last blocks, and the whole size */
G2L_FN size_t g2l_kv_scales(long S, int NH, long nb) { return (size_t)S * NH * nb * (2 * G2L_BLOCK * G2L_DH); }
G2L_FN size_t g2l_kv_last(long S, int NH, long nb)
{
    return g2l_kv_scales(S, NH, nb) + ((size_t)S * NH * nb * 8 + 255) / 256 * 256;
}
G2L_FN size_t g2l_kv_bytes(long S, int NH, long nb)
{
    return g2l_kv_last(S, NH, nb) + (size_t)S * NH * (2 * G2L_BLOCK * G2L_DH) * 4;
}

/* the attention's workspace: parts of a head's positions at most, floats for
 * each (maximum, sum, 64 dims) */
#define G2L_SPLITS 32
#define G2L_PART_FLOATS (2 + G2L_DH)

/* Work of g2k_kv8_append: wave `item` of a call of T rows has head, keys or
 * values, the i-th block from the one that holds the first position, sequence
 * (heads first: neighbouring waves read neighbouring parts of the same rows). */
G2L_FN unsigned g2l_append_blocks(int T) { return (unsigned)T / G2L_BLOCK + 2; }
G2L_FN long g2l_append_waves(int S, int NH, int T) { return (long)S * NH * 2 * g2l_append_blocks(T); }
G2L_FN void g2l_append_item(unsigned item, int NH, int T, int *h, int *kv, int *i, long *s)
{
    const unsigned row = item / (unsigned)NH, per = g2l_append_blocks(T);
    *h = (int)(item % (unsigned)NH);
    *kv = (int)(row % 2);
    *i = (int)(row / 2 % per);
    *s = row / 2 / per;
}
/* Work of g2k_kv8_attn*: wave w of nw takes four whole blocks at a time, from
 * g2l_attn_first on and g2l_attn_step apart, below the end of its part; the
 * block that is not full is g2l_attn_left's. */
G2L_FN int g2l_attn_first(int split, int span, int w) { return split * span + 4 * w; }
G2L_FN int g2l_attn_step(int nw) { return 4 * nw; }
G2L_FN int g2l_attn_end(int split, int span, int full) { return (split + 1) * span < full ? (split + 1) * span : full; }
G2L_FN int g2l_attn_left(int split, int span, int full, int w, int nw)
{
    const int at = full - split * span;
    return at >= 0 && at < span && w == (at + 3) / 4 % nw;
}

/* ---- rules on logits: ids of a work-group's slice (narrow and wide form);
 * 64-bit words from row to row of the workspace (a cache line: the slices of
 * all rows meet there) */
#define G2L_SLICE 1024
#define G2L_SLICE_WIDE 8192
#define G2L_CELL 16

#endif

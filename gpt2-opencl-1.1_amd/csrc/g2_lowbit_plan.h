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
 *  last   [S][NH][K, V][16][64] fp32: the positions of the block that is not
 *  full yet.
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

/* ---- rules on logits: ids of a work-group's slice (narrow and wide form),
 * slices of a row at most */
#define G2L_SLICE 1024
#define G2L_SLICE_WIDE 8192
#define G2L_PARTS 64

#endif

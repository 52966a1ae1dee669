/* gpt2_int4.h -- weights of 4 bits with a scale for each group along k: the quantiser, its inverse, and the product
 * of one row, a few rows or many with them.  No counterpart in the reference, whose weights are fp16 or INT8 with a
 * scale for each output (gpt2_kernels.h).
 *
 * Scheme.  w[N][K] is cut into groups of `group` (32, 64 or 128) consecutive k of one output n; the last group of a row may be
 * shorter.  s = fp16(absmax / 7), 1 where that is 0; q = clamp(rint(w / s), -7, 7), in fp32.  NaN counts as 0, infinities as
 * +-65504.  The products take any code in [-8, 7] and any finite scale, so that weights quantised elsewhere can be laid out for them.
 *
 *     C[m][n] = epi( sum over groups g of s[n][g] * (sum over k in g of A[m][k] q[n][k]) + bias[n] )
 *
 * in fp32 (a code is exact in fp16, its products are exact in fp32), rounded to fp16 once, after the epilogue: nothing, gelu_new, or
 * resid[m][n] + ...  Every M sums a group in the same products, but in an order that depends on M and on the sizes.
 *
 * Layout, in which the matrix instructions take it: tiles of 16 n by 128 k, tile (n / 16, k / 128) at n / 16 * ceil(K / 128) + k / 128.
 *   codes, 1 KB a tile: the 32-bit word [k % 32 / 8][n % 16][k % 128 / 32] has eight consecutive k as q + 8 in four bits each, k % 8 = e at bit
 *   4 (e / 2) + 16 (e % 2);
 *   scales, 16 * 128 / group a tile: [n % 16 / 4][k % 128 / group][n % 4].
 * Codes past K are 0 (held as 8) and their groups' scales finite; rows past N mean nothing, but are read.
 *
 * Every call but alloc and free only enqueues kernels on the stream of gpt2_set_stream, so it can be captured; there is no workspace, and calls may overlap.  Errors
 * as in gpt2_kernels.h.
 */
#ifndef GPT2_INT4_H
#define GPT2_INT4_H

#include "gpt2_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct GPT2Int4W {
    uint8_t *codes;    /* device, 16-byte aligned, gpt2_int4_code_bytes */
    gpt2_half *scales; /* device, 16-byte aligned, gpt2_int4_scale_count of them */
    int N, K, group;
    void *arena;       /* owns the buffers when gpt2_int4_alloc made them */
} GPT2Int4W;

/* Sizes of the two buffers; 0 where N, K or group is none. */
size_t gpt2_int4_code_bytes(int N, int K);
size_t gpt2_int4_scale_count(int N, int K, int group);
/* Buffers for an N x K matrix, their contents undefined.  0 on success.  A caller with buffers of its own fills the struct. */
int gpt2_int4_alloc(GPT2Int4W *w, int N, int K, int group);
void gpt2_int4_free(GPT2Int4W *w);

/* w := src[N][K] (fp16, row-major). */
void gpt2_quantize_int4(const GPT2Int4W *w, const gpt2_half *src);
/* dst[N][K] := fp16(s q). */
void gpt2_dequantize_int4(gpt2_half *dst, const GPT2Int4W *w);

#define GPT2_EPI_NONE 0
#define GPT2_EPI_GELU 1
#define GPT2_EPI_ADD 2
/* C[M][N] as above, M at most 2^21, M * N below some 2^37 (what the work-groups of one launch can have; more is refused); bias [N] or NULL; resid [M][N], with GPT2_EPI_ADD only, may be C.  C overlaps neither A nor the weights.  A, C, bias and
 * resid need the alignment of their type only; from 17 rows on, A with rows at 16 bytes (K % 8 == 0) is faster. */
void gpt2_matmul_int4(gpt2_half *C, const gpt2_half *A, const GPT2Int4W *w, const gpt2_half *bias, int M, int epi,
                      const gpt2_half *resid);

#ifdef __cplusplus
}
#endif
#endif

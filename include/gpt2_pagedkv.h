/* gpt2_pagedkv.h -- a paged K/V cache for several sequences, its pages held in INT8; the attention that
 * reads it; forking, reordering, freeing and compacting; and beam search's selection.  No counterpart in
 * the reference, whose cache (gpt2_kvcache.h) holds one sequence in fp16 and whose decode is greedy.
 *
 * Pages.  A page is GPT2_PAGE_TOKENS consecutive tokens of one sequence, in every layer.  Complete pages
 * live in a pool of nPages, in INT8, with one fp32 scale for each layer, page, K|V and head; they never
 * change again, so sequences that share a beginning share its pages (refs counts the sequences).  The tokens
 * after a sequence's last complete page stay in fp16 in an open page of its own (there is one for each
 * sequence) until it is full: every value is rounded to 8 bits once.  Scheme per page, head and K|V, as
 * the weights': s = absmax / 127 (1 if absmax is 0), q = clamp(rint(x / s), -127, 127), in fp32.  A cache
 * holds finite values only: NaN is stored as 0, infinities as +-65504.
 *
 * What a row attends to is what the cache holds after its call's append.  A page that the call completes is INT8 for all of the call's
 * rows, its scale the largest of all 32 tokens, later ones than the row among them; while a page is open its tokens are fp16.  So a
 * row's output depends, by the rounding of pages, on how a prompt was cut into calls.  Normal keys and values, 300 to 1000 tokens, against
 * 64 bits over unrounded ones: 1.1e-2 of the result's norm with the prompt in one call, 0.7e-2 to 0.8e-2 token by token, as much between the two;
 * with one channel of 64 four times as wide 2.5e-2, 2.0e-2 to 2.3e-2, 1.0e-2 to 1.4e-2.
 *
 * A ragged batch.  `rows` is a device array of nSeq + 1 offsets: rows[s] .. rows[s+1] - 1 are sequence s's
 * new rows in the activations (qkv [nRows][3 E], x and att [nRows][E], E = nHead * headDim), none is fine.
 * nRows, at most 2^23, is how many rows the call may look at, all of rows[nSeq] at least; those past rows[nSeq] are left as they are.
 * How a call runs goes by nRows, since the host does not know the offsets: up to nSeq, as for one row a sequence (a decode step passes
 * nSeq, even if its buffers hold more); past it, as for prompts.  Results differ in the order of sums and the bits of weights.  One step
 * of a model over a batch:
 *     gpt2_pkv_grow(c, rows, nRows);              once: pages for the new rows, positions, lengths
 *     gpt2_pkv_embed(x, wte, wpe, ids, c, rows, nRows);
 *     per layer L: ... qkv ...; gpt2_pkv_append(c, L, qkv, rows, nRows);
 *                  gpt2_pkv_attn(att, qkv, c, L, rows, nRows, group, ws, wsBytes); ...
 * and between steps of a beam search gpt2_beam_select, then gpt2_pkv_fork with the parents it gives.
 *
 * Every call but alloc, free and status only enqueues kernels on the stream of gpt2_set_stream: no
 * allocation, copy or wait, so a step can be captured into a graph and replayed (its state is in device
 * memory).  Calls that change a cache (grow, append, fork, compact, reset) use its `plan` buffer and run one at
 * a time, ordered with the calls that read it, as on one stream.  Calls run on the current device, which has
 * to be the one that holds the cache.
 *
 * Errors: host-side arguments as in gpt2_kernels.h (recorded, nothing launched).  What only the device sees
 * (no free page, a sequence longer than maxPages, offsets or parents out of range) refuses that whole grow or
 * fork, which then leaves the cache as it was with no new rows (start = len, so the step's appends and
 * attention do nothing), and is kept until gpt2_pkv_status asks.  Every kernel checks the pages, slots and lengths
 * that it reads from device memory before it uses them: a page number outside the pool stands for a page that is not
 * there (its keys weigh nothing; it reads back as 0).
 */
#ifndef GPT2_PAGEDKV_H
#define GPT2_PAGEDKV_H

#include "gpt2_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GPT2_PAGE_TOKENS 32
#define GPT2_PAGE_TILE (GPT2_PAGE_TOKENS * GPT2_HEAD_DIM) /* values of one page, head and K|V */
#define GPT2_PKV_MAX_SEQ 4096
#define GPT2_BEAM_MAX 16
#define GPT2_BEAM_MAX_VOCAB 65536

/* Device buffers, codes and open 16-byte aligned.  A tile (GPT2_PAGE_TILE values) is K as [token][dim] and V as
 * [token / 8][dim][token % 8], the order in which the attention's matrix instructions take them.  Element (L, page,
 * kv, h) of codes is ((L * nPages + page) * 2 + kv) * nHead + h tiles in; open pages alike, by slot. */
typedef struct GPT2PagedKV {
    int8_t *codes;   /* [nLayer][nPages][K|V][nHead] tiles */
    float *scales;   /* [nLayer][nPages][K|V][nHead] */
    gpt2_half *open; /* [nLayer][nSeq][K|V][nHead] tiles */
    int *table;      /* [nSeq][maxPages] page numbers; entries past a sequence's complete pages mean nothing */
    int *len;        /* [nSeq] tokens */
    int *start;      /* [nSeq] position of the first row of the last grow (len where it gave none) */
    int *slot;       /* [nSeq] which open page is the sequence's: a permutation */
    int *refs;       /* [nPages] sequences that hold the page; 0: free */
    int *status;     /* [4]: the first device-side error, the live pages as the last compact counted them, 0, 0 */
    int *plan;       /* [GPT2_PKV_PLAN_INTS] scratch of the calls that change the cache */
    int nLayer, nHead, headDim, nPages, nSeq, maxPages;
    void *arena;     /* owns the buffers when gpt2_pkv_alloc made them */
} GPT2PagedKV;
#define GPT2_PKV_PLAN_INTS(nSeq, maxPages, nPages) ((size_t)(nSeq) * (maxPages) + 4 * (size_t)(nSeq) + 3 * (size_t)(nPages) + 16)

/* A cache of nPages pages for nSeq sequences (at most GPT2_PKV_MAX_SEQ) of up to maxLen tokens, empty.  headDim is
 * GPT2_HEAD_DIM.  0 on success.  A caller with buffers of its own fills the struct and calls gpt2_pkv_reset. */
int gpt2_pkv_alloc(GPT2PagedKV *c, int nLayer, int nHead, int nPages, int nSeq, int maxLen);
void gpt2_pkv_free(GPT2PagedKV *c);
/* Empties every sequence and frees every page. */
void gpt2_pkv_reset(GPT2PagedKV *c);
/* Waits for the stream; the first device-side error since the last call (E_ARG, E_CAPACITY; 0: none), which it
 * also records for gpt2_last_error and clears. */
int gpt2_pkv_status(GPT2PagedKV *c);

/* start = len, len += the new rows, and the lowest free pages, in order of the sequences, for the pages that
 * they complete (all layers). */
void gpt2_pkv_grow(GPT2PagedKV *c, const int *rows, int nRows);
/* x[row] = fp16(wte[ids[row]] + wpe[position of the row]) (GPT2_N_EMBD wide); a token outside the vocabulary or a
 * position past GPT2_N_CTX adds nothing, as gpt2_embed_one's kernel has it.  x, wte and wpe are
 * 16-byte aligned. */
void gpt2_pkv_embed(gpt2_half *x, const gpt2_half *wte, const gpt2_half *wpe, const int *ids, const GPT2PagedKV *c,
                    const int *rows, int nRows);
/* The keys and values of the new rows into layer L: open pages, and the pages that they complete:
 * once for each layer after a grow. */
void gpt2_pkv_append(GPT2PagedKV *c, int L, const gpt2_half *qkv, const int *rows, int nRows);
/* att[row] = softmax(q . k / 8) v over the tokens up to the row's own, from the cache.  `group`: 1, or how many
 * consecutive sequences (at most 16) are beams of one prompt: in a call with nRows <= nSeq the leading pages that all of a group share are
 * then read once, if its sequences have one row each at most (a batch with a prompt in it is faster with 1; past nSeq, group means
 * nothing); results are the same but for the order of sums and the bits of the weights.  Scores and sums are fp32.  The softmax's weights have
 * 22 bits where the call has no more rows than sequences (nRows <= nSeq) and a sequence has at most 8 of them, a group of beams
 * with one row each at most 8 beams; elsewhere they are rounded to fp16, which takes an output's error against 64 bits from 2.1e-4 of the
 * result's norm, its own rounding, to 2.4e-4.  ws: at least gpt2_pkv_attn_ws bytes of device memory, 16-byte aligned, with no meaning between calls; calls that may overlap need one each.  More rows may need
 * less (they are split less): a workspace for calls of several sizes has the largest of theirs. */
size_t gpt2_pkv_attn_ws(const GPT2PagedKV *c, int nRows);
void gpt2_pkv_attn(gpt2_half *att, const gpt2_half *qkv, const GPT2PagedKV *c, int L, const int *rows, int nRows,
                   int group, void *ws, size_t wsBytes);
/* Rows out of the cache: kv[row] = k | v (2 E wide, fp16) of sequence s's positions pos[s], pos[s] + 1, ... for rows
 * rows[s] .. rows[s+1] - 1 (rows, pos: device).  Positions past the sequence read as 0. */
void gpt2_pkv_read(gpt2_half *kv, const GPT2PagedKV *c, int L, const int *rows, const int *pos, int nRows);

/* Sequence i goes on as what sequence parent[i] was (device array of nSeq; -1: empty), for all i at once: reorders,
 * forks and frees.  Complete pages are shared; the first child of a parent keeps its open page, further ones get a copy of
 * the tokens in it. */
void gpt2_pkv_fork(GPT2PagedKV *c, const int *parent);
/* Moves the pages that any sequence holds to the lowest numbers: the k-th of those past the place of the last goes to the
 * k-th free page below it.  status[1] is how many there are. */
void gpt2_pkv_compact(GPT2PagedKV *c);

/* Beam search's selection.  Of groups x beams rows of logits (row r at logits + r * ld, V of them), the best `beams`
 * of each group's beams x V continuations by score[r] + log_softmax(logits[r])[token], best first: token, parent (its
 * row), score_out, done_out, [groups * beams] each.  Equal scores: the lower row first, within a row the larger logit,
 * then the lower token.  A logit that is NaN counts as -inf, +inf as 65504, a score that is NaN as -inf.  A row with
 * done[r] != 0 has one continuation, `eos` at its own score; done_out marks rows that end with eos.  eos < 0: there is no
 * end token, and done is not read (may be NULL; done_out is 0).  score_out and done_out may be score and done.  Exponentials
 * are fp32, and up to 33 of them are summed in fp32, what those make in fp64, where scores are formed and compared: a score is within 95
 * 2^-24 of the exact one before it is rounded to fp32.  A row's sum depends on its logits alone, not on where it lies, so
 * equal rows with equal scores tie.  ws as for gpt2_pkv_attn. */
size_t gpt2_beam_select_ws(int groups, int beams, int V);
void gpt2_beam_select(int *token, int *parent, float *score_out, int *done_out, const gpt2_half *logits, long ld,
                      const float *score, const int *done, int groups, int beams, int V, int eos, void *ws, size_t wsBytes);

#ifdef __cplusplus
}
#endif
#endif

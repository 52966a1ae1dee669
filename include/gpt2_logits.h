/* gpt2_logits.h -- what shapes logits before a token is chosen (gpt2_beam_select): penalties for tokens that a sequence
 * has already, n-gram bans, biases and grammar masks; and the sequences' token histories that they go by.  No counterpart in
 * the reference, whose decode is greedy.
 *
 * In a step of several sequences (gpt2_pagedkv.h):
 *     logits of each sequence's last row
 *     gpt2_logits_adjust(logits, logits, V, nSeq, V, &rules);
 *     gpt2_beam_select(ids, parent, ...);
 *     gpt2_pkv_fork(c, parent);
 *     gpt2_history_step(h, parent, rows, ids, nSeq, 0);          rows: 0, 1, 2, ..
 * and after a prompt gpt2_history_step(h, NULL, rows, ids, nRows, 1) with the prompt's own offsets.
 *
 * Both only enqueue kernels on the stream of gpt2_set_stream, and go by device memory, so a step can be captured and
 * replayed.  Errors of host-side arguments as in gpt2_kernels.h.  What only the device sees is checked before it is used and
 * counts as said below.
 */
#ifndef GPT2_LOGITS_H
#define GPT2_LOGITS_H

#include "gpt2_pagedkv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GPT2_HISTORY_MAX_ROOM (1 << 24)

/* The tokens of nSeq sequences (at most GPT2_PKV_MAX_SEQ), at most `room` each; device buffers.  Lengths outside [0, room] count
 * as the nearer end. */
typedef struct GPT2History {
    int *tokens;  /* [nSeq][room]; those past a sequence's length mean nothing and are left as they are */
    int *len;     /* [nSeq] */
    int *start;   /* [nSeq] where the tokens begin that presence and frequency count: the prompt's end */
    int *arrived; /* [1] 0 between calls: work-groups of a step that are done */
    int nSeq, room;
    void *arena;  /* owns the buffers when gpt2_history_alloc made them */
} GPT2History;

/* Empty histories.  0 on success.  A caller with buffers of its own fills the struct and calls gpt2_history_reset. */
int gpt2_history_alloc(GPT2History *h, int nSeq, int room);
void gpt2_history_free(GPT2History *h);
void gpt2_history_reset(GPT2History *h);
/* For all sequences at once: s becomes what parent[s] was (device; NULL: all stay; a number that is no sequence: empty), and the tokens
 * ids[rows[s]] .. ids[rows[s+1] - 1] are appended (device; rows NULL: none; offsets out of order or past nRows: none for that
 * sequence); what exceeds `room` is dropped.  prompt != 0: where tokens were appended, `start` becomes the new length.  Calls
 * that change a history run one at a time, ordered with those that read it. */
void gpt2_history_step(GPT2History *h, const int *parent, const int *rows, const int *ids, int nRows, int prompt);

/* All pointers but `history` are to device memory; NULL: the rule is off. */
typedef struct GPT2LogitsRules {
    const GPT2History *history;                         /* row r goes by sequence r */
    const float *repetition, *presence, *frequency;     /* [rows] */
    int ngram;                                          /* 0: off; else the length of n-grams that may not come again */
    int n_bias;                                         /* entries in bias_token and bias_value */
    const int *bias_start;                              /* [rows + 1]: row r's entries, clamped to [0, n_bias] */
    const int *bias_token;                              /* tokens outside the vocabulary are passed over; of a row's entries for one token the last counts */
    const float *bias_value;
    const uint32_t *mask;                               /* [n_masks][ceil(V / 32)]: token t is allowed if bit t % 32 of word t / 32 is set */
    const int *mask_row;                                /* [rows] which mask; outside [0, n_masks): none.  NULL: row r has mask r */
    int n_masks;
} GPT2LogitsRules;

/* out[r][t], rows ld apart, from logits[r][t] (out may be logits, or have nothing in common with it):
 *     x = logit + bias
 *     t in the history:  x = x > 0 ? x / repetition : x * repetition
 *     c > 0 times from `start` on:  x = x - (frequency * c + presence)
 *     -inf where the mask has no bit, or t would complete an n-gram (`ngram` tokens) that the history has
 * in fp32, rounded to fp16 once.  A NaN stays one unless it is masked or banned; a mask of nothing leaves a row of -inf.  repetition > 0.
 * An n-gram of the history that begins as its last n - 1 tokens do is compared with them token by token, so a long history of one token, over and over, costs its
 * length times n comparisons.
 * Without a history (NULL) there are no penalties and no n-grams.  With out == logits, rows without a mask are touched
 * only where a token is penalised, banned or biased. */
void gpt2_logits_adjust(gpt2_half *out, const gpt2_half *logits, long ld, int rows, int V, const GPT2LogitsRules *rules);

#ifdef __cplusplus
}
#endif
#endif

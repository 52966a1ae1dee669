// logits.hip -- penalties, n-gram bans, biases and grammar masks on logits, and the token histories that they go by
// (gpt2_logits.h).
#include <cmath>
#include <cstring>

#include "common.h"
#include "gpt2_logits.h"

namespace g2 {

// ------------------------------------------------------------------ histories
// All sequences change at once, in place: a work-group has a few columns of every sequence's row in its registers before it writes
// any.  The lengths, which every work-group reads, are written by the one that arrives last.
constexpr int HIST_THREADS = 1024, HIST_ITEMS = 16;   // tokens a thread holds

struct HistSeq {
    int from, past, after, row0;   // from: the sequence that it goes on as, or -1
};
__device__ __forceinline__ HistSeq hist_seq(const GPT2History &h, const int *__restrict__ parent, const int *__restrict__ rows, int nRows, int s) {
    HistSeq q;
    q.from = parent ? parent[s] : s;
    if ((unsigned)q.from >= (unsigned)h.nSeq) q.from = -1;
    q.past = q.from < 0 ? 0 : min(max(h.len[q.from], 0), h.room);
    int a = 0, b = 0;
    if (rows) {
        a = rows[s];
        b = rows[s + 1];
        if (a < 0 || b < a || b > nRows) a = b = 0;
    }
    q.row0 = a;
    q.after = q.past + min(b - a, h.room - q.past);
    return q;
}

__global__ __launch_bounds__(HIST_THREADS) void k_history_step(GPT2History h, const int *__restrict__ parent, const int *__restrict__ rows,
                                                               const int *__restrict__ ids, int nRows, int prompt, int width_log2) {
    const int tid = threadIdx.x, threads = blockDim.x, width = 1 << width_log2, c = (blockIdx.x << width_log2) + (tid & (width - 1));
    const int per = threads >> width_log2, s0 = tid >> width_log2;   // sequences at once; this thread's first
    int value[HIST_ITEMS];
    uint32_t write = 0;
#pragma unroll
    for (int i = 0; i < HIST_ITEMS; ++i) {
        const int s = s0 + i * per;
        value[i] = 0;
        if (s < h.nSeq && c < h.room) {
            const HistSeq q = hist_seq(h, parent, rows, nRows, s);
            if (c < q.past) {
                if (q.from != s) {
                    value[i] = h.tokens[(size_t)q.from * h.room + c];
                    write |= 1u << i;
                }
            } else if (c < q.after) {
                value[i] = ids[q.row0 + (c - q.past)];
                write |= 1u << i;
            }
        }
    }
    // every token and length has been read: passing through here waits for the loads
#pragma unroll
    for (int i = 0; i < HIST_ITEMS; ++i) asm volatile("" : "+v"(value[i]) : : "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HIST_ITEMS; ++i)
        if (write >> i & 1) h.tokens[(size_t)(s0 + i * per) * h.room + c] = value[i];
    __shared__ int last;
    if (tid == 0) {
        __threadfence();
        last = atomicAdd(h.arrived, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    int len[HIST_ITEMS], start[HIST_ITEMS];   // at most 4096 sequences: 4 a thread of 1024, 16 of 256
#pragma unroll
    for (int i = 0; i < HIST_ITEMS; ++i) {
        const int s = tid + i * threads;
        len[i] = start[i] = 0;
        if (s < h.nSeq) {
            const HistSeq q = hist_seq(h, parent, rows, nRows, s);
            len[i] = q.after;
            start[i] = prompt && q.after > q.past ? q.after : q.from < 0 ? 0 : h.start[q.from];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HIST_ITEMS; ++i) {
        const int s = tid + i * threads;
        if (s < h.nSeq) {
            h.len[s] = len[i];
            h.start[s] = start[i];
        }
    }
    if (tid == 0) *h.arrived = 0;
}

__global__ void k_history_reset(GPT2History h) {
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s < h.nSeq) h.len[s] = h.start[s] = 0;
    if (s == 0) *h.arrived = 0;
}

static bool history_refused(const GPT2History *h, const char *what) {
    if (!h || !h->tokens || !h->len || !h->start || !h->arrived || h->nSeq < 1 || h->nSeq > GPT2_PKV_MAX_SEQ || h->room < 1 || h->room > GPT2_HISTORY_MAX_ROOM ||
        (((uintptr_t)h->tokens | (uintptr_t)h->len | (uintptr_t)h->start | (uintptr_t)h->arrived) & 3))
        return arg_fail(what);
    return false;
}

// ------------------------------------------------------------------ logits
// A work-group has SLICE tokens of a row.  What the row's history says of each is counted in LDS: how often it was said since
// `start`, whether it was said at all, whether it would end a known n-gram.  A bias list's entry of a token is its last, by the largest index.
constexpr int SLICE = 4096;
constexpr uint32_t SEEN = 1u << 31, BANNED = 1u << 30, COUNT = BANNED - 1;

struct RowRules {
    float rep, freq, pres;
};
__device__ __forceinline__ float adjusted(float x, uint32_t said, float bias, const RowRules &r) {
    x += bias;
    if (said) {
        x = x > 0.f ? x / r.rep : x * r.rep;
        const uint32_t n = said & COUNT;
        if (n) x -= __builtin_fmaf(r.freq, (float)n, r.pres);
        if (said & BANNED) x = -INFINITY;
    }
    return x;
}

__global__ __launch_bounds__(256) void k_logits_adjust(uint16_t *out, const uint16_t *logits, long ld, int V, GPT2LogitsRules r, GPT2History h) {
    __shared__ uint32_t said[SLICE], bias_at[SLICE];
    const int tid = threadIdx.x, row = blockIdx.y, t0 = blockIdx.x * SLICE, nt = min(SLICE, V - t0);
    const uint16_t *x = logits + (size_t)row * ld + t0;
    uint16_t *y = out + (size_t)row * ld + t0;
    for (int i = tid; i < SLICE; i += 256) {
        said[i] = 0;
        bias_at[i] = 0;
    }
    __syncthreads();
    if (h.tokens) {
        const int n = min(max(h.len[row], 0), h.room), start = h.start[row];
        const int *tok = h.tokens + (size_t)row * h.room;
        for (int i = tid; i < n; i += 256) {
            const unsigned t = (unsigned)(tok[i] - t0);
            if (t < (unsigned)nt) {
                if (i >= start) atomicAdd(&said[t], 1u);
                else atomicOr(&said[t], SEEN);
            }
        }
        if (r.ngram > 0 && n >= r.ngram) {
            const int *tail = tok + n - (r.ngram - 1);
            for (int i = tid; i + r.ngram <= n; i += 256) {
                const unsigned t = (unsigned)(tok[i + r.ngram - 1] - t0);
                if (t >= (unsigned)nt) continue;
                bool same = true;
                for (int j = 0; j < r.ngram - 1 && same; ++j) same = tok[i + j] == tail[j];
                if (same) atomicOr(&said[t], BANNED);
            }
        }
    }
    if (r.n_bias) {
        const int a = min(max(r.bias_start[row], 0), r.n_bias), b = min(r.bias_start[row + 1], r.n_bias);
        for (int i = a + tid; i < b; i += 256) {
            const unsigned t = (unsigned)(r.bias_token[i] - t0);
            if (t < (unsigned)nt) atomicMax(&bias_at[t], (unsigned)i + 1);
        }
    }
    __syncthreads();
    const RowRules rules = {r.repetition ? r.repetition[row] : 1.f, r.frequency ? r.frequency[row] : 0.f, r.presence ? r.presence[row] : 0.f};
    const uint32_t *mask = nullptr;
    if (r.n_masks) {
        const int m = r.mask_row ? r.mask_row[row] : row;
        if ((unsigned)m < (unsigned)r.n_masks) mask = r.mask + (size_t)m * ((V + 31) >> 5);
    }
    for (int i = tid; i < nt; i += 256) {
        float v = adjusted(h2f(x[i]), said[i], bias_at[i] ? r.bias_value[bias_at[i] - 1] : 0.f, rules);
        const int t = t0 + i;
        if (mask && !(mask[t >> 5] >> (t & 31) & 1)) v = -INFINITY;
        y[i] = f2h(v);
    }
}

static size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace g2

using namespace g2;

extern "C" int gpt2_history_alloc(GPT2History *h, int nSeq, int room) {
    if (!h) return arg_fail("gpt2_history_alloc: null"), 1;
    memset(h, 0, sizeof(*h));
    if (nSeq < 1 || nSeq > GPT2_PKV_MAX_SEQ || room < 1 || room > GPT2_HISTORY_MAX_ROOM) return arg_fail("gpt2_history_alloc: sizes out of range"), 1;
    const size_t tokens = align16((size_t)nSeq * room * 4), book = align16((size_t)nSeq * 4);
    char *p = (char *)gpt2_dmalloc(tokens + 2 * book + 16);
    if (!p) return 1;
    *h = GPT2History{(int *)p, (int *)(p + tokens), (int *)(p + tokens + book), (int *)(p + tokens + 2 * book), nSeq, room, p};
    gpt2_history_reset(h);
    return 0;
}

extern "C" void gpt2_history_free(GPT2History *h) {
    if (h && h->arena) {
        gpt2_dfree(h->arena);
        memset(h, 0, sizeof(*h));
    }
}

extern "C" void gpt2_history_reset(GPT2History *h) {
    if (history_refused(h, "gpt2_history_reset: bad history")) return;
    hipLaunchKernelGGL(k_history_reset, dim3(cdiv(h->nSeq, 256)), dim3(256), 0, stream(), *h);
    check_launch("k_history_reset");
}

extern "C" void gpt2_history_step(GPT2History *h, const int *parent, const int *rows, const int *ids, int nRows, int prompt) {
    if (history_refused(h, "gpt2_history_step: bad history")) return;
    if (nRows < 0 || (rows && nRows && !ids) || (((uintptr_t)parent | (uintptr_t)rows | (uintptr_t)ids) & 3)) {
        arg_fail("gpt2_history_step: bad rows");
        return;
    }
    int width = 6;   // log2 of the columns that a work-group takes
    while ((h->nSeq << width) > HIST_THREADS * HIST_ITEMS) --width;
    int threads = 256;
    while (threads < HIST_THREADS && (h->nSeq << width) > threads) threads *= 2;
    hipLaunchKernelGGL(k_history_step, dim3(cdiv(h->room, 1 << width)), dim3(threads), 0, stream(), *h, parent, rows, ids, nRows, prompt, width);
    check_launch("k_history_step");
}

extern "C" void gpt2_logits_adjust(gpt2_half *out, const gpt2_half *logits, long ld, int rows, int V, const GPT2LogitsRules *rules) {
    if (rows == 0) return;
    if (rows < 0 || rows > 65535 || V < 1 || V > 1 << 24 || ld < V) { arg_fail("gpt2_logits_adjust: sizes out of range"); return; }
    if (!out || !logits || (((uintptr_t)out | (uintptr_t)logits) & 1) || !rules) { arg_fail("gpt2_logits_adjust: null/unaligned"); return; }
    GPT2LogitsRules r = *rules;
    GPT2History h = {};
    if (r.history) {
        if (history_refused(r.history, "gpt2_logits_adjust: bad history")) return;
        h = *r.history;
    }
    r.history = nullptr;
    if (!r.bias_start) r.n_bias = 0;
    if (!r.mask) r.n_masks = 0;
    if ((h.tokens && h.nSeq < rows) || r.ngram < 0 || r.n_bias < 0 || r.n_masks < 0 || (r.n_bias && (!r.bias_token || !r.bias_value)) ||
        (((uintptr_t)r.repetition | (uintptr_t)r.presence | (uintptr_t)r.frequency | (uintptr_t)r.bias_start | (uintptr_t)r.bias_token | (uintptr_t)r.bias_value |
          (uintptr_t)r.mask | (uintptr_t)r.mask_row) & 3)) {
        arg_fail("gpt2_logits_adjust: bad rules");
        return;
    }
    hipLaunchKernelGGL(k_logits_adjust, dim3(cdiv(V, SLICE), rows), dim3(256), 0, stream(), out, logits, ld, V, r, h);
    check_launch("k_logits_adjust");
}

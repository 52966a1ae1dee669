// logits.hip -- penalties, n-gram bans, biases and grammar masks on logits, and the token histories that they go by
// (gpt2_logits.h).
#include <cmath>
#include <cstring>
#include <type_traits>

#include "common.h"
#include "gpt2_logits.h"

namespace g2 {

// ------------------------------------------------------------------ histories
// All sequences change at once, in place: a work-group has what it moves in its registers before it writes any.  Where parents lie in their
// children's block of R sequences (9 to 16: one is a multiple of any number of beams up to 16), it moves such a block's rows by long pieces; else a few
// columns of every sequence.  1024 sequences of up to 4000 tokens, with a copy of the lengths ahead: 12.7 us by blocks, in
// groups of 8; 14.9 by columns, any sequence from any, whose rows are 64 bytes each, 16 KB apart.  The lengths, which every work-group reads, are written by the one that arrives last.
constexpr int HIST_THREADS = 1024, HIST_ITEMS = 4;   // pieces a thread holds: 16 sequences of 256, or 4096 of one

struct HistSeq {
    int from, past, after;   // from: the sequence that it goes on as, or -1
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
    q.after = q.past + min(b - a, h.room - q.past);
    return q;
}

// Waits for the wave's loads.  A barrier alone waits for nothing but LDS, and a load whose value is used behind it may still be under way.
__device__ __forceinline__ void all_loaded() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A thread's pieces are W consecutive tokens (4 where rows lie at 16 bytes, else 1).
template <int W>
__global__ __launch_bounds__(HIST_THREADS) void k_history_step(GPT2History h, const int *__restrict__ parent, const int *__restrict__ rows,
                                                               const int *__restrict__ ids, int nRows, int prompt, int width_log2) {
    typedef std::conditional_t<W == 4, i32x4, int> piece;
    const int tid = threadIdx.x;
    // sequence s0 + i * per for i < HIST_ITEMS, where below `end`; pieces at column c
    auto move = [&](int s0, int per, int end, int c) {
        piece value[HIST_ITEMS];
        uint32_t moved = 0, grown = 0;
        int past[HIST_ITEMS], after[HIST_ITEMS];
#pragma unroll
        for (int i = 0; i < HIST_ITEMS; ++i) {
            const int s = s0 + i * per;
            past[i] = after[i] = 0;
            if (s < end) {
                const HistSeq q = hist_seq(h, parent, rows, nRows, s);
                past[i] = q.past;
                after[i] = q.after;
                if (q.from != s && c < q.past) {
                    value[i] = *reinterpret_cast<const piece *>(h.tokens + (size_t)q.from * h.room + c);
                    moved |= 1u << i;
                }
                if (q.after > q.past && c < q.after && c + W > q.past) grown |= 1u << i;   // so there are rows and ids
            }
        }
        all_loaded();   // every token that is moved over, and every length that the last work-group writes over
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HIST_ITEMS; ++i) {
            int *to = h.tokens + (size_t)(s0 + i * per) * h.room + c;
            if (moved >> i & 1) {
                if (c + W <= past[i]) *reinterpret_cast<piece *>(to) = value[i];
                else if constexpr (W == 4)
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        if (c + e < past[i]) to[e] = value[i][e];
            }
            if (grown >> i & 1) {   // few: tokens that are appended
                const int row0 = rows[s0 + i * per];
                for (int e = max(0, past[i] - c); e < W && c + e < after[i]; ++e) to[e] = ids[row0 + (c + e - past[i])];
            }
        }
    };
    int block = 16;
    if (h.nSeq > 16) {
        __shared__ uint32_t fit;   // bit k: blocks of 9 + k
        if (tid == 0) fit = 0xff;
        __syncthreads();
        uint32_t mine = 0xff;
        if (parent)
            for (int s = tid; s < h.nSeq; s += HIST_THREADS) {
                const unsigned p = (unsigned)parent[s];
                if (p < (unsigned)h.nSeq && p != (unsigned)s)
#pragma unroll
                    for (unsigned k = 0; k < 8; ++k)
                        if ((unsigned)s / (9 + k) != p / (9 + k)) mine &= ~(1u << k);
            }
        uint32_t wave = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) wave |= __ballot(!(mine >> k & 1)) ? 0u : 1u << k;
        if ((tid & 63) == 0) atomicAnd(&fit, wave);
        __syncthreads();
        block = fit ? 9 + 31 - __builtin_clz(fit) : 0;
    }
    const int width = 1 << width_log2, blocks = block ? (h.nSeq + block - 1) / block : 0;
    auto units = [&](int columns) { return block ? blocks * ((columns + 256 * W - 1) / (256 * W)) : (columns + (W << width_log2) - 1) / (W << width_log2); };
    int longest = h.room;
    if (units(h.room) > (int)gridDim.x) {   // room for far more than there may be: as far as the longest goes
        __shared__ int most;
        if (tid == 0) most = 0;
        __syncthreads();
        int mine = 0;
        for (int s = tid; s < h.nSeq; s += HIST_THREADS) mine = max(mine, hist_seq(h, parent, rows, nRows, s).after);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) mine = max(mine, __shfl_xor(mine, o, 64));
        if ((tid & 63) == 0) atomicMax(&most, mine);
        __syncthreads();
        longest = most;
    }
    const int n = units(longest), chunks = block ? max(1, n / blocks) : 1;
    for (int u = blockIdx.x; u < n; u += gridDim.x) {
        if (block) {
            const int first = u / chunks * block;
            move(first + (tid >> 8), 4, min(first + block, h.nSeq), W * ((u % chunks << 8) + (tid & 255)));
        } else move(tid >> width_log2, HIST_THREADS >> width_log2, h.nSeq, W * ((u << width_log2) + (tid & (width - 1))));
    }
    __shared__ int last;
    // No fence: every length has been read ahead of a barrier (move, or the exchange of the longest), and what was written is for later kernels (a fence writes the L2 back: 19 us for 1024 sequences).
    if (tid == 0) {
        last = atomicAdd(h.arrived, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    constexpr int LENS = GPT2_PKV_MAX_SEQ / HIST_THREADS, threads = HIST_THREADS;
    int len[LENS], start[LENS];
#pragma unroll
    for (int i = 0; i < LENS; ++i) {
        const int s = tid + i * threads;
        len[i] = start[i] = 0;
        if (s < h.nSeq) {
            const HistSeq q = hist_seq(h, parent, rows, nRows, s);
            len[i] = q.after;
            start[i] = prompt && q.after > q.past ? q.after : q.from < 0 ? 0 : h.start[q.from];
        }
    }
    all_loaded();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LENS; ++i) {
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
// A work-group has SLICE tokens of a row.  What the row's history says of each is counted in LDS: how often it was said since `start`, whether it was said at
// all, whether it would end a known n-gram.  The tokens that were said are listed as their first mention is counted; for those, and those with a bias, a thread each
// works out the logit, in LDS, through which the slice goes by octets: 16 bytes of logits, wherever the row begins, a byte of the mask.  An entry of the bias list marks
// its token; only where a list is longer than the work-group, or a token has two, are entries compared for the last.
// 256 rows of 50257 with masks, 300 biases and histories of up to 4096 take 20.1 us (2.8 TB/s), without any of them 14: every slice goes through the row's whole
// history, and a work-group is a chain of lengths, tokens, counts and barriers.  Slices of 4096 with counts of 32 bits and a table for the biases' indexes took 24.4;
// rules worked out where the row is copied, or claimed by a second pass over the history, 25 to 31 with either.
// Counts have 16 bits where a history's room allows it.
template <bool HALF>
struct Said {
    static constexpr uint32_t SEEN = HALF ? 0x8000u : 1u << 31, BANNED = SEEN >> 1, BIASED = SEEN >> 2, COUNT = BIASED - 1;
    static constexpr int BYTES = HALF ? 2 : 4;
    uint32_t *words;
    __device__ __forceinline__ uint32_t add(unsigned t, uint32_t v) const {   // what it was before
        if constexpr (HALF) return atomicAdd(&words[t >> 1], v << (16 * (t & 1))) >> (16 * (t & 1)) & 0xffffu;
        else return atomicAdd(&words[t], v);
    }
    __device__ __forceinline__ uint32_t mark(unsigned t, uint32_t v) const {
        if constexpr (HALF) return atomicOr(&words[t >> 1], v << (16 * (t & 1))) >> (16 * (t & 1)) & 0xffffu;
        else return atomicOr(&words[t], v);
    }
    __device__ __forceinline__ void clear(unsigned t, uint32_t v) const {
        if constexpr (HALF) atomicAnd(&words[t >> 1], ~(v << (16 * (t & 1))));
        else atomicAnd(&words[t], ~v);
    }
    __device__ __forceinline__ uint32_t at(unsigned t) const {
        if constexpr (HALF) return reinterpret_cast<const uint16_t *>(words)[t];
        else return words[t];
    }
};
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(4)));

struct RowRules {
    float rep, freq, pres;
};
template <bool HALF>
__device__ __forceinline__ float adjusted(float x, uint32_t said, float bias, const RowRules &r) {
    x += bias;
    if (said) {
        x = x > 0.f ? x / r.rep : x * r.rep;
        const uint32_t n = said & Said<HALF>::COUNT;
        if (n) x -= __builtin_fmaf(r.freq, (float)n, r.pres);
        if (said & Said<HALF>::BANNED) x = -INFINITY;
    }
    return x;
}
// Bytes of LDS: what was said, counters, the list, the slice's logits, a piece of the bias list.
template <int SLICE, int THREADS, bool HALF>
constexpr int tables_bytes() { return SLICE * (Said<HALF>::BYTES + 2 + 2) + 16 + THREADS * 4; }

template <int SLICE, int THREADS, bool HALF>
__global__ __launch_bounds__(THREADS) void k_logits_adjust(uint16_t *out, const uint16_t *logits, long ld, int V, GPT2LogitsRules r, GPT2History h) {
    __shared__ __attribute__((aligned(16))) uint32_t tables[tables_bytes<SLICE, THREADS, HALF>() / 4];
    constexpr int OCTETS = SLICE / 8 / THREADS, WORDS = SLICE * Said<HALF>::BYTES / 4;
    constexpr uint32_t SEEN = Said<HALF>::SEEN, COUNT = Said<HALF>::COUNT;
    const Said<HALF> said = {tables};
    uint32_t *const listed = tables + WORDS, *const biases = listed + 1, *const twice = listed + 2;   // how many are in the list, and in the piece; whether a token has two biases
    uint16_t *const list = reinterpret_cast<uint16_t *>(tables + WORDS + 4), *const value = list + SLICE;   // tokens that were said; the slice's logits
    uint32_t *const piece = tables + WORDS + 4 + SLICE;
    const int tid = threadIdx.x, row = blockIdx.y, t0 = blockIdx.x * SLICE, nt = min(SLICE, V - t0);
    const uint16_t *x = logits + (size_t)row * ld + t0;
    uint16_t *y = out + (size_t)row * ld + t0;
    // the octets, the thread's first tokens and its first bias are asked for together
    u16x8_any v[OCTETS];
    if (out != logits || r.n_masks)
#pragma unroll
        for (int o = 0; o < OCTETS; ++o) {
            const int i = 8 * (tid + THREADS * o);
            if (i + 8 <= nt) v[o] = *reinterpret_cast<const u16x8_any *>(x + i);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[o][e] = i + e < nt ? x[i + e] : 0;
        }
    const int *tok = h.tokens ? h.tokens + (size_t)row * h.room : nullptr;
    const int len = tok ? min(max(h.len[row], 0), h.room) : 0, start = tok ? h.start[row] : 0;
    const int bias0 = r.n_bias ? min(max(r.bias_start[row], 0), r.n_bias) : 0, bias1 = r.n_bias ? min(max(r.bias_start[row + 1], 0), r.n_bias) : 0;
    const uint8_t *mask = nullptr;
    if (r.n_masks) {
        const int m = r.mask_row ? r.mask_row[row] : row;
        if ((unsigned)m < (unsigned)r.n_masks) mask = reinterpret_cast<const uint8_t *>(r.mask + (size_t)m * ((V + 31) >> 5)) + (t0 >> 3);
    }
    const bool sparse = out == logits && !mask;   // only what a rule names is touched
    const RowRules rules = {r.repetition ? r.repetition[row] : 1.f, r.frequency ? r.frequency[row] : 0.f, r.presence ? r.presence[row] : 0.f};
    i32x4_any w0 = {};
    int bias_t0 = -1;
    float bias_v0 = 0.f;
    if (4 * tid + 4 <= len) w0 = *reinterpret_cast<const i32x4_any *>(tok + 4 * tid);
    if (bias1 - 1 - tid >= bias0) {
        bias_t0 = r.bias_token[bias1 - 1 - tid];
        bias_v0 = r.bias_value[bias1 - 1 - tid];
    }
    uint32_t allowed[OCTETS];
#pragma unroll
    for (int o = 0; o < OCTETS; ++o) allowed[o] = mask && 8 * (tid + THREADS * o) < nt ? mask[tid + THREADS * o] : 0xffu;
    for (int i = 4 * tid; i < WORDS + 4; i += 4 * THREADS) *reinterpret_cast<i32x4 *>(tables + i) = i32x4{0, 0, 0, 0};
    __syncthreads();
    if (len) {
        const int last = r.ngram > 0 ? len - r.ngram : -1;   // n-grams begin at 0 .. last
        const int *tail = tok + len - (r.ngram - 1);
        const int first = r.ngram > 1 && last >= 0 ? tail[0] : 0;
        auto ends = [&](int i, int w) {   // n-grams from i on that begin as the last n - 1 tokens
            if (i > last || (r.ngram > 1 && w != first)) return;
            bool same = true;
            for (int j = 1; j < r.ngram - 1 && same; ++j) same = tok[i + j] == tail[j];
            const unsigned end = (unsigned)(tok[i + r.ngram - 1] - t0);
            if (same && end < (unsigned)nt) said.mark(end, Said<HALF>::BANNED);
        };
        // counts first, then the list of those that were new: one place of it for each of a wave's, by one addition
        auto take = [&](int i, const i32x4_any &w, int n) {
            uint32_t before[4];
            uint64_t fresh[4];
            int total = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned t = (unsigned)(w[e] - t0);
                before[e] = SEEN;
                if (e < n && t < (unsigned)nt) before[e] = i + e >= start ? said.add(t, 1u) : said.mark(t, SEEN);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                fresh[e] = __ballot(!(before[e] & (SEEN | COUNT)));
                total += __popcll(fresh[e]);
            }
            if (total) {
                int at = 0;
                const uint64_t here = __ballot(true);
                if ((tid & 63) == __builtin_ctzll(here)) at = (int)atomicAdd(listed, (uint32_t)total);
                at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!(before[e] & (SEEN | COUNT)))
                        list[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(fresh[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)fresh[e], 0u))] = (uint16_t)(w[e] - t0);
                    at += __popcll(fresh[e]);
                }
            }
            if (r.ngram > 0)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < n) ends(i + e, w[e]);
        };
        for (int i = 4 * tid; i < len; i += 4 * THREADS) {
            i32x4_any w = w0;
            if (i + 4 <= len) {
                if (i != 4 * tid) w = *reinterpret_cast<const i32x4_any *>(tok + i);
            } else
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = i + e < len ? tok[i + e] : 0;
            take(i, w, min(4, len - i));
        }
    }
    // the thread's first bias takes the token with all its rules, and the list of what was said leaves it out; a second bias of a token is told
    const unsigned bias_t = (unsigned)(bias_t0 - t0);
    const bool biased = bias1 - 1 - tid >= bias0 && bias_t < (unsigned)nt;
    if (biased && said.mark(bias_t, Said<HALF>::BIASED) & Said<HALF>::BIASED) *twice = 1;
    if (!sparse)
#pragma unroll
        for (int o = 0; o < OCTETS; ++o) *reinterpret_cast<i32x4 *>(value + 8 * (tid + THREADS * o)) = __builtin_bit_cast(i32x4, v[o]);
    __syncthreads();
    auto put = [&](unsigned t, float bias) {
        const uint16_t to = f2h(adjusted<HALF>(h2f(sparse ? x[t] : value[t]), said.at(t) & ~Said<HALF>::BIASED, bias, rules));
        if (sparse) y[t] = to;
        else value[t] = to;
    };
    if (bias1 - bias0 <= THREADS && !*twice) {
        if (biased) put(bias_t, bias_v0);
    } else {
        // A long list, or a token with two biases: the list from its end, a piece of THREADS entries at a time; an entry counts if no later one of its piece, and none of a
        // later piece, has its token.
        if (biased) said.clear(bias_t, Said<HALF>::BIASED);
        __syncthreads();
        for (int end = bias1; end > bias0; end -= THREADS) {
            const bool is_first = end == bias1;
            const int i = end - 1 - tid;   // thread 0 has the last
            unsigned t = ~0u;
            float bias = 0.f;
            if (i >= bias0) {
                t = (unsigned)((is_first ? bias_t0 : r.bias_token[i]) - t0);
                bias = is_first ? bias_v0 : r.bias_value[i];
            }
            const bool mine = t < (unsigned)nt && !(said.at(t) & Said<HALF>::BIASED);
            if (mine) piece[atomicAdd(biases, 1u)] = t << 16 | (uint32_t)tid;
            __syncthreads();
            if (mine) {
                bool counts = true;
                for (int k = 0, n = (int)*biases; k < n; k += 8) {
                    const i32x4 a = *reinterpret_cast<const i32x4 *>(piece + k), b = *reinterpret_cast<const i32x4 *>(piece + k + 4);   // what is past n is not looked at
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t other = (uint32_t)(e < 4 ? a[e & 3] : b[e & 3]);
                        counts &= k + e >= n || (other >> 16) != t || (int)(other & 0xffffu) >= tid;
                    }
                }
                if (counts) {
                    put(t, bias);
                    said.mark(t, Said<HALF>::BIASED);
                }
            }
            __syncthreads();
            if (tid == 0) *biases = 0;
            if (end - THREADS > bias0) __syncthreads();
        }
    }
    for (int i = tid, n = (int)*listed; i < n; i += THREADS)
        if (!(said.at(list[i]) & Said<HALF>::BIASED)) put(list[i], 0.f);
    if (sparse) return;
    __syncthreads();
#pragma unroll
    for (int o = 0; o < OCTETS; ++o) {
        const int i = 8 * (tid + THREADS * o);
        if (i >= nt) break;
        u16x8_any to = __builtin_bit_cast(u16x8_any, *reinterpret_cast<const i32x4 *>(value + i));
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (!(allowed[o] >> e & 1)) to[e] = 0xfc00;
        if (i + 8 <= nt) *reinterpret_cast<u16x8_any *>(y + i) = to;
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < nt) y[i + e] = to[e];
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
    const bool wide = h->room % 4 == 0 && aligned16(h->tokens);
    const int w = wide ? 4 : 1;
    int width = wide ? 4 : 6;   // log2 of the pieces of a row that a work-group takes: 256 bytes
    while ((h->nSeq << width) > HIST_THREADS * HIST_ITEMS) --width;
    const long blocks = (long)cdiv(h->nSeq, 16) * cdiv(h->room, 256 * w), slabs = h->nSeq > 16 ? cdiv(h->room, w << width) : 1;
    const long most = blocks > slabs ? blocks : slabs;
    hipLaunchKernelGGL(wide ? k_history_step<4> : k_history_step<1>, dim3((unsigned)(most < 512 ? most : 512)), dim3(HIST_THREADS), 0, stream(), *h, parent, rows, ids,
                       nRows, prompt, width);
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
    // 16-bit counts where a count cannot pass them, and slices of twice the length where there is a work-group of them for every CU (256 rows, histories of up to 600, trigrams:
    // 16.8 us for 17.3, in place 11.3 for 14.0; of up to 4096 with masks and biases 20.1 for 20.7; 8 rows 4.9 for 4.7)
    const bool half = !h.tokens || h.room <= (int)Said<true>::COUNT;
    if (half && (long)rows * cdiv(V, 8192) >= 256)
        hipLaunchKernelGGL((k_logits_adjust<8192, 512, true>), dim3(cdiv(V, 8192), rows), dim3(512), 0, stream(), out, logits, ld, V, r, h);
    else hipLaunchKernelGGL((k_logits_adjust<4096, 512, false>), dim3(cdiv(V, 4096), rows), dim3(512), 0, stream(), out, logits, ld, V, r, h);
    check_launch("k_logits_adjust");
}

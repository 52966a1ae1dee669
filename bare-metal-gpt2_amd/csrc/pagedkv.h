// pagedkv.h -- what the kernels over the paged K/V cache (gpt2_pagedkv.h) share: the sequences of a ragged
// batch, checked before use, and where tiles lie.
#pragma once

#include "common.h"
#include "gpt2_pagedkv.h"

namespace g2 {

constexpr int PKV_P = GPT2_PAGE_TOKENS, PKV_D = GPT2_HEAD_DIM, PKV_TILE = GPT2_PAGE_TILE;
static_assert(PKV_P == 32 && PKV_D == 64 && GPT2_N_EMBD % PKV_D == 0, "the tiles' layouts are written for these");

// A sequence's new rows [row0, row0 + n), positions [start, start + n), start + n = len.  n is 0 where the book says
// nothing usable: lengths out of range, rows that do not match them, a slot that is none.
struct PkvSeq {
    int start, len, row0, n, slot;
};
__device__ __forceinline__ PkvSeq pkv_seq(const GPT2PagedKV &c, const int *__restrict__ rows, int nRows, int s) {
    PkvSeq q;
    q.start = c.start[s];
    q.len = c.len[s];
    q.row0 = rows[s];
    q.n = rows[s + 1] - q.row0;
    q.slot = c.slot[s];
    const bool ok = q.start >= 0 && q.n > 0 && q.row0 >= 0 && q.n <= nRows && q.row0 <= nRows - q.n && q.len - q.start == q.n &&
                    q.len / PKV_P <= c.maxPages && (long)q.len <= (long)c.maxPages * PKV_P && (unsigned)q.slot < (unsigned)c.nSeq;
    if (!ok) q.n = 0;
    return q;
}

// The sequence whose rows include `row` by the offsets, or -1 (offsets in any order are read within bounds).
__device__ __forceinline__ int pkv_seq_of_row(const int *__restrict__ rows, int nSeq, int row) {
    int lo = 0, hi = nSeq;   // the last s with rows[s] <= row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (rows[mid] <= row) lo = mid;
        else hi = mid;
    }
    return rows[lo] <= row && row < rows[lo + 1] ? lo : -1;
}

// Work units are handed to work-groups in the sequences' order; `units(s)` says how many s has.  The sequence of unit u
// (`u` becomes the unit's number in it), or -1 past the last.  All 64 lanes of the wave call it.
template <typename F>
__device__ __forceinline__ int pkv_seq_of_unit(int &u, int nSeq, F units) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < nSeq; base += 64) {
        const int mine = base + lane < nSeq ? units(base + lane) : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o, 64);
            if (lane >= o) sum += v;
        }
        const int total = __builtin_amdgcn_readlane(sum, 63);
        if (u < total) {
            const int l = __builtin_ctzll(__ballot(sum > u));
            u -= __builtin_amdgcn_readlane(sum - mine, l);
            return base + l;
        }
        u -= total;
    }
    return -1;
}

__device__ __forceinline__ bool pkv_page_ok(const GPT2PagedKV &c, int page) { return (unsigned)page < (unsigned)c.nPages; }
// Tile (layer L, page or slot, K|V, head) in units of tiles; `per`: pages, or open pages, in a layer.
__device__ __forceinline__ size_t pkv_tile(const GPT2PagedKV &c, int per, int L, int page, int kv, int h) {
    return (((size_t)L * per + page) * 2 + kv) * c.nHead + h;
}
// Value (token, dim) in a K tile and in a V tile.
__device__ __forceinline__ int pkv_k_at(int tok, int d) { return tok * PKV_D + d; }
__device__ __forceinline__ int pkv_v_at(int tok, int d) { return ((tok >> 3) * PKV_D + d) * 8 + (tok & 7); }

// Host: a cache that the kernels can run on (`what`: the caller, for the error).
bool pkv_refused(const GPT2PagedKV *c, const char *what);
bool pkv_refused_batch(const GPT2PagedKV *c, int L, const int *rows, int nRows, const char *what);

}  // namespace g2

// pagedkv.hip -- the paged K/V cache (gpt2_pagedkv.h): bookkeeping of its pages (growing, forking, compacting), the
// append that quantises complete pages, and reading rows back.  Its attention is attn_paged.hip.
//
// All of it is bound by memory or, at the sizes of a decode step, by launch latency: the kernels are few, take what
// depends on the sequences' lengths from device memory, and never come back to the host.  Times in this file: a launch under
// the tracer, the median over two sets of inputs in turn, 12 heads, one layer unless said.
#include <cmath>
#include <cstring>

#include "attn_prefill.h"   // tr_read
#include "pagedkv.h"

namespace g2 {

// The plan buffer: staged page tables | per-sequence words | per-page words | a few words.
struct PkvPlan {
    int *tables;                   // [nSeq][maxPages]
    int *len, *slot, *from;        // [nSeq] after a fork; from: the open page copied, or -1
    int *map, *hole, *mover;       // [nPages] of a compaction; a grow's free pages are in map
    int *word;                     // [0] moves of a compaction, [1] a fork's parents are in range
};
__host__ __device__ __forceinline__ PkvPlan pkv_plan(const GPT2PagedKV &c) {
    PkvPlan p;
    p.tables = c.plan;
    p.len = p.tables + (size_t)c.nSeq * c.maxPages;
    p.slot = p.len + c.nSeq;
    p.from = p.slot + c.nSeq;
    p.map = p.len + 4 * (size_t)c.nSeq;
    p.hole = p.map + c.nPages;
    p.mover = p.hole + c.nPages;
    p.word = p.mover + c.nPages;
    return p;
}

// A wave's own LDS accesses happen in order; this keeps the compiler from reordering them.
__device__ __forceinline__ void pkv_lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// Exclusive sum over a work-group of 64 NW threads; `total` for all.  Ends with a barrier, so `lds` can be used again.
template <int NW>
__device__ __forceinline__ int block_scan(int v, int *lds, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(sum, o, 64);
        if (lane >= o) sum += u;
    }
    if (lane == 63) lds[w] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int x = lds[i];
        if (i < w) before += x;
        total += x;
    }
    __syncthreads();
    return before + sum - v;
}

__global__ void k_pkv_reset(GPT2PagedKV c) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < c.nSeq) {
        c.len[i] = 0;
        c.start[i] = 0;
        c.slot[i] = i;
    }
    if (i < c.nPages) c.refs[i] = 0;
    if (i < 4) c.status[i] = 0;
}

// ------------------------------------------------------------------ grow
// One work-group: needs and their sums over the sequences, then a walk over refs that hands the lowest free pages out in
// order, which stops when enough are found (its first step is under way meanwhile); tables, refs and lengths are written once they
// are.  Bound by the latency of its few dependent loads and barriers: 4.3 us for 48 sequences with T = 256 threads, 5.2 with 1024; where
// hundreds of pages are handed out (48 prompts of up to 1000 rows) 8.0 and 6.4.
template <int T>
__global__ __launch_bounds__(T) void k_pkv_grow(GPT2PagedKV c, const int *__restrict__ rows, int nRows) {
    constexpr int NW = T / 64, PER = GPT2_PKV_MAX_SEQ / 1024, FREE = 8;
    __shared__ int off[PER * T], place[PER * T], lds[2][NW + 2], flags[NW];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const PkvPlan plan = pkv_plan(c);
    int ref[FREE];
    auto load_refs = [&](int base) {
#pragma unroll
        for (int j = 0; j < FREE; ++j) ref[j] = base + FREE * tid + j < c.nPages ? c.refs[base + FREE * tid + j] : 1;
    };
    load_refs(0);
    int len[PER], add[PER], need[PER], sum = 0;
    bool bad_arg = false, bad_len = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int s = tid * PER + j;
        len[j] = add[j] = need[j] = 0;
        if (s < c.nSeq) {
            const int a = rows[s], b = rows[s + 1];
            len[j] = c.len[s];
            add[j] = b - a;
            bad_arg |= a < 0 || b < a || b > nRows || len[j] < 0;
            const long after = (long)len[j] + add[j];
            bad_len |= after > (long)c.maxPages * PKV_P;
            if (!bad_arg && !bad_len) need[j] = (int)(after / PKV_P) - len[j] / PKV_P;
        }
        sum += need[j];
    }
    const int flag = (__ballot(bad_arg) ? 1 : 0) | (__ballot(bad_len) ? 2 : 0);
    if (lane == 0) flags[w] = flag;
    int total, all = 0;
    int at = block_scan<NW>(sum, lds[0], total);
#pragma unroll
    for (int i = 0; i < NW; ++i) all |= flags[i];
    bool full = all & 2;
    if (!all && total > 0) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            off[tid * PER + j] = at;
            place[tid * PER + j] = (tid * PER + j) * c.maxPages + len[j] / PKV_P - at;   // of the k-th page handed out, less k
            at += need[j];
        }
        int found = 0;
        for (int base = 0; base < c.nPages && found < total; base += FREE * T) {
            if (base) load_refs(base);
            int n = 0;
#pragma unroll
            for (int j = 0; j < FREE; ++j) n += ref[j] == 0;
            int here, k = found + block_scan<NW>(n, lds[1], here);
            found += here;
#pragma unroll
            for (int j = 0; j < FREE; ++j)
                if (ref[j] == 0) {
                    if (k < total) plan.map[k] = base + FREE * tid + j;
                    ++k;
                }
        }
        full = found < total;   // the same in every thread
        __syncthreads();
        if (!full)
            for (int k = tid; k < total; k += T) {
                // the last sequence whose pages begin at or before the k-th; it needs one
                int lo = 0, hi = c.nSeq;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (off[mid] <= k) lo = mid;
                    else hi = mid;
                }
                const int page = plan.map[k];
                c.table[place[lo] + k] = page;
                c.refs[page] = 1;
            }
    }
    const bool refuse = (all & 1) || full;
    if (refuse && tid == 0) atomicCAS(c.status, 0, all & 1 ? E_ARG : E_CAPACITY);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int s = tid * PER + j;
        if (s < c.nSeq) {
            c.start[s] = len[j];
            if (!refuse) c.len[s] = len[j] + add[j];
        }
    }
}

// ------------------------------------------------------------------ embed
// A work-group a row, four values a thread: 8-byte loads and stores.  48 rows of 48 sequences 2.6 us, the chain from the offsets, looked up by
// halving, to the books, the token and its row; 30666 rows 28 us, 94 MB in and 47 out (some of the table's rows are in a cache).
constexpr int EMBED_THREADS = GPT2_N_EMBD / 4;
__global__ __launch_bounds__(EMBED_THREADS) void k_pkv_embed(uint16_t *__restrict__ x, const uint16_t *__restrict__ wte,
                                                             const uint16_t *__restrict__ wpe, const int *__restrict__ ids, GPT2PagedKV c,
                                                             const int *__restrict__ rows, int nRows) {
    constexpr int E = GPT2_N_EMBD;
    static_assert(E % 4 == 0, "four values a thread");
    const int row = blockIdx.x, e = 4 * threadIdx.x;
    const int s = pkv_seq_of_row(rows, c.nSeq, row);
    if (s < 0) return;
    const PkvSeq q = pkv_seq(c, rows, nRows, s);
    if (q.n == 0) return;
    const int pos = q.start + row - q.row0, id = ids[row];
    f16x4 te = {}, pe = {}, y;
    if ((unsigned)id < (unsigned)GPT2_VOCAB) te = *reinterpret_cast<const f16x4 *>(wte + (size_t)id * E + e);
    if ((unsigned)pos < (unsigned)GPT2_N_CTX) pe = *reinterpret_cast<const f16x4 *>(wpe + (size_t)pos * E + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (f16)((float)te[i] + (float)pe[i]);
    *reinterpret_cast<f16x4 *>(x + (size_t)row * E + e) = y;
}

// ------------------------------------------------------------------ append
// A tile on its way: 16 pairs of a lane.  By rows, pair 4 i + j is dims 8 (lane & 7) + 2 j, + 1 of token 8 i + lane / 8; by
// dims, tokens 8 i + 2 j, + 1 of dim `lane` (both in the order of the tile that they go to).
constexpr int PKV_ROW = 160;   // bytes of a token's row in LDS: neither its writes nor the transposing reads meet a bank conflict

// What the cache can hold of a value: codes stand for finite numbers only.
__device__ __forceinline__ uint16_t pkv_finite(uint16_t v) {
    const float f = h2f(v);
    return f != f ? (uint16_t)0 : f2h(fminf(fmaxf(f, -65504.f), 65504.f));
}
__device__ __forceinline__ bool pkv_is_finite(const uint32_t (&d)[16]) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, d[i] & 0x7fff7fffu));
    return max((int)m[0], (int)m[1]) < 0x7c00;
}
__device__ __forceinline__ void pkv_make_finite(uint32_t (&d)[16]) {
    if (__ballot(!pkv_is_finite(d)))   // hardly ever
#pragma unroll
        for (int i = 0; i < 16; ++i) d[i] = pkv_finite((uint16_t)d[i]) | (uint32_t)pkv_finite((uint16_t)(d[i] >> 16)) << 16;
}

// By rows: the page's tokens that are new rows (`src`: the row of position `start`), zeros elsewhere.
__device__ __forceinline__ void pkv_load_rows(const uint16_t *__restrict__ src, size_t ld, int pos0, const PkvSeq &q, uint32_t (&d)[16]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = pos0 + 8 * i + (lane >> 3);
        i32x4 v = {0, 0, 0, 0};
        if (pos >= q.start && pos < q.len) v = *reinterpret_cast<const i32x4 *>(src + (size_t)(pos - q.start) * ld + 8 * (lane & 7));
#pragma unroll
        for (int j = 0; j < 4; ++j) d[4 * i + j] = (uint32_t)v[j];
    }
}

// Rows to dims, through the wave's own LDS and the transposing reads (lane 16 G + j: dim 16 G + j of four tokens each).
__device__ __forceinline__ void pkv_by_dims(uint32_t (&d)[16], char *lds) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<i32x4 *>(lds + (8 * i + (lane >> 3)) * PKV_ROW + 16 * (lane & 7)) = i32x4{(int)d[4 * i], (int)d[4 * i + 1], (int)d[4 * i + 2], (int)d[4 * i + 3]};
    pkv_lds_order();
    const char *col = lds + ((lane & 15) >> 2) * PKV_ROW + 2 * (16 * (lane >> 4) + 4 * (lane & 3));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint2 v = __builtin_bit_cast(uint2, tr_read(col + 4 * i * PKV_ROW));
        d[2 * i] = v.x;
        d[2 * i + 1] = v.y;
    }
    pkv_lds_order();
}

// Codes of a whole tile and its scale: q = rint(fl(x / s)), |x / s| <= 127 (1 + 2^-24).  x / s is y = x (1 / s) to within
// 2^-16; only where y lies within twice that of the middle between two whole numbers are the quotients formed (three tiles in ten of
// normal values have such a one, nearly always a middle itself: fp16 values have few bits).  y + 1.5 2^23 is the nearest whole number in its low byte.
__device__ __forceinline__ float pkv_quantize(const uint32_t (&d)[16], uint32_t (&out)[8]) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, d[i] & 0x7fff7fffu));
    const float peak = wave_max_u(fmaxf(h2f(m[0]), h2f(m[1])));
    const float s = peak == 0.f ? 1.0f : peak / 127.0f, inv = 1.0f / s;
    constexpr float magic = 12582912.f;
    float far = 0.f;
    uint32_t w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float x = h2f((uint16_t)(d[i / 2] >> (16 * (i & 1))));
        const float y = fmaf(x, inv, magic);
        w[i] = __float_as_uint(y);
        far = fmaxf(far, fabsf(fmaf(x, inv, magic - y)));
    }
    if (__ballot(far > 0.5f - 1.f / 32768)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float x = h2f((uint16_t)(d[i / 2] >> (16 * (i & 1))));
            w[i] = (uint32_t)(int)fminf(fmaxf(rintf(x / s), -127.f), 127.f);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        out[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[4 * i + 3], w[4 * i + 2], 0x0c0c0400u),
                                       __builtin_amdgcn_perm(w[4 * i + 1], w[4 * i], 0x0c0c0400u), 0x05040100u);
    return s;
}

// A sequence's units: the pages that its new rows complete, one at least.  Unit 0 also writes the open page, whose rows
// before the call it reads, so no other work-group touches it.
__device__ __forceinline__ int pkv_append_units(const PkvSeq &q) {
    return q.n ? max(1, q.len / PKV_P - q.start / PKV_P) : 0;
}

// One wave per unit, K|V and head: whole row pieces in, 16 bytes a lane, the tile's maximum over the wave, 8 bytes of codes a
// lane and store, 512 contiguous.  48 prompts of 250 to 1000 rows: 40 us, 3.4 TB/s of rows in and codes out (a row's
// piece of a head is 128 bytes, every 4.5 KB); a decode step's 48 rows 6.8 us, its chain of loads and the code's own way from memory.
__device__ __forceinline__ void pkv_append_unit(const GPT2PagedKV &c, int L, const uint16_t *__restrict__ qkv, const PkvSeq &q,
                                                int seq, int u, int kv, int h, char *lds) {
    const int lane = threadIdx.x & 63;
    const int E = c.nHead * PKV_D;
    const int had = q.start / PKV_P, full = q.len / PKV_P;
    const uint16_t *src = qkv + (size_t)q.row0 * 3 * E + (1 + kv) * E + h * PKV_D;   // row of position start
    uint16_t *open = c.open + pkv_tile(c, c.nSeq, L, q.slot, kv, h) * PKV_TILE;
    uint32_t d[16];
    if (had + u < full) {
        const int page = c.table[(size_t)seq * c.maxPages + had + u], kept = u ? 0 : q.start % PKV_P;
        i32x4 old[4] = {};   // the open page's tokens from before the call, under way with the rows
        if (kept)
#pragma unroll
            for (int i = 0; i < 4; ++i) old[i] = *reinterpret_cast<const i32x4 *>(open + 8 * (64 * i + lane));
        pkv_load_rows(src, 3 * (size_t)E, (had + u) * PKV_P, q, d);
        if (kv) pkv_by_dims(d, lds);
        if (kept) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = kv ? kept - (8 * i + 2 * j) : kept > 8 * i + (lane >> 3) ? 2 : 0;   // of the pair, how many
                    const uint32_t keep = n >= 2 ? ~0u : n == 1 ? 0xffffu : 0u;
                    d[4 * i + j] = ((uint32_t)old[i][j] & keep) | (d[4 * i + j] & ~keep);
                }
            }
        }
        pkv_make_finite(d);
        uint32_t w[8];
        const float scale = pkv_quantize(d, w);
        if (pkv_page_ok(c, page)) {
            const size_t at = pkv_tile(c, c.nPages, L, page, kv, h);
            if (lane == 0) c.scales[at] = scale;
            uint2 *tile = reinterpret_cast<uint2 *>(c.codes + at * PKV_TILE);
#pragma unroll
            for (int i = 0; i < 4; ++i) tile[64 * i + lane] = uint2{w[2 * i], w[2 * i + 1]};
        }
    }
    const int first = max(q.start, full * PKV_P);
    if (u || first >= q.len) return;
    if (q.len - first <= 2) {
        for (int pos = first; pos < q.len; ++pos) {
            const int tok = pos % PKV_P;
            open[kv ? pkv_v_at(tok, lane) : pkv_k_at(tok, lane)] = pkv_finite(src[(size_t)(pos - q.start) * 3 * E + lane]);
        }
        return;
    }
    pkv_load_rows(src, 3 * (size_t)E, full * PKV_P, q, d);
    pkv_make_finite(d);
    const int t0 = first % PKV_P, t1 = q.len % PKV_P;   // tokens [t0, t1) are written, no others
    if (kv) pkv_by_dims(d, lds);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int tok = 8 * i + (lane >> 3);
        if (kv ? t0 <= 8 * i && 8 * i + 8 <= t1 : t0 <= tok && tok < t1)
            *reinterpret_cast<i32x4 *>(open + 8 * (64 * i + lane)) = i32x4{(int)d[4 * i], (int)d[4 * i + 1], (int)d[4 * i + 2], (int)d[4 * i + 3]};
        else if (kv)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (t0 <= 8 * i + e && 8 * i + e < t1) open[8 * (64 * i + lane) + e] = (uint16_t)(d[4 * i + e / 2] >> (16 * (e & 1)));
    }
}

// BY_SEQ: work-groups per sequence that do all of its units, gridDim.z of them in turn (no more rows than sequences: nearly always
// one unit each); else one per unit.
template <bool BY_SEQ>
__global__ __launch_bounds__(256) void k_pkv_append(GPT2PagedKV c, int L, const uint16_t *__restrict__ qkv,
                                                    const int *__restrict__ rows, int nRows) {
    __shared__ __attribute__((aligned(16))) char lds[4][PKV_P * PKV_ROW];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int u = BY_SEQ ? blockIdx.z : blockIdx.x;
    const int seq = BY_SEQ ? (int)blockIdx.x : pkv_seq_of_unit(u, c.nSeq, [&](int s) { return pkv_append_units(pkv_seq(c, rows, nRows, s)); });
    if (seq < 0) return;
    const PkvSeq q = pkv_seq(c, rows, nRows, seq);
    const int n = BY_SEQ ? pkv_append_units(q) : u + 1;
    for (; u < n; u += gridDim.z)   // 1 but by sequences
        for (int kh = blockIdx.y * 4 + w; kh < 2 * c.nHead; kh += 4 * gridDim.y)   // wave-uniform; there is no barrier
            pkv_append_unit(c, L, qkv, q, seq, u, kh >= c.nHead, kh % c.nHead, lds[w]);
}

// ------------------------------------------------------------------ read
// A unit is a page that the rows of a sequence touch; a wave takes one K|V and head of it: the tile in its own order,
// 8 values a lane and piece, V through LDS to rows, 16-byte stores.  Bound by memory: 46 MB of codes to 92 MB of rows in 26.6 us, 5.2 TB/s.
struct PkvRead {
    long pos;        // of the sequence's first row
    int row0, n;
};
__device__ __forceinline__ PkvRead pkv_read_rows(const int *__restrict__ rows, const int *__restrict__ pos, int nRows, int s) {
    PkvRead r;
    r.pos = pos[s];
    r.row0 = rows[s];
    r.n = rows[s + 1] - r.row0;
    if (r.row0 < 0 || r.n < 0 || r.n > nRows || r.row0 > nRows - r.n) r.n = 0;
    return r;
}
__global__ __launch_bounds__(256) void k_pkv_read(uint16_t *__restrict__ out, GPT2PagedKV c, int L, const int *__restrict__ rows,
                                                  const int *__restrict__ pos, int nRows) {
    __shared__ __attribute__((aligned(16))) uint16_t lds[4][PKV_P][PKV_D];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane >> 3, d0 = (lane & 7) * 8;
    const int kh = blockIdx.y * 4 + w;
    if (kh >= 2 * c.nHead) return;   // wave-uniform; no barrier follows
    int u = blockIdx.x;
    const int s = pkv_seq_of_unit(u, c.nSeq, [&](int s) {
        const PkvRead r = pkv_read_rows(rows, pos, nRows, s);
        return r.n ? (int)(((r.pos + r.n - 1) >> 5) - (r.pos >> 5)) + 1 : 0;
    });
    if (s < 0) return;
    const PkvRead r = pkv_read_rows(rows, pos, nRows, s);
    const long p = (r.pos >> 5) + u;   // the page's number; its first row is that of position 32 p
    const int kv = kh >= c.nHead, h = kh - kv * c.nHead, len = (int)min((long)c.len[s], (long)c.maxPages * PKV_P), slot = c.slot[s];
    f16x8 v[4] = {};
    if (p >= 0 && p < len / PKV_P) {
        const int page = c.table[(size_t)s * c.maxPages + p];
        if (pkv_page_ok(c, page)) {
            const size_t at = pkv_tile(c, c.nPages, L, page, kv, h);
            const float scale = c.scales[at];
            const uint2 *tile = reinterpret_cast<const uint2 *>(c.codes + at * PKV_TILE);
            uint2 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = tile[64 * i + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f16x8 x = i8x8_to_f16x8(q[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = (f16)((float)x[e] * scale);
            }
        }
    } else if (p >= 0 && p * PKV_P < len && (unsigned)slot < (unsigned)c.nSeq) {
        const uint16_t *tile = c.open + pkv_tile(c, c.nSeq, L, slot, kv, h) * PKV_TILE;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f16x8 *>(tile + 8 * (64 * i + lane));
    }
    if (kv) {   // lane: 8 tokens of its dim; rows from the wave's own LDS
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const f16 x = v[i][e];   // a copy: a bit cast of the element itself takes the vector's first
                lds[w][8 * i + e][lane] = __builtin_bit_cast(uint16_t, x);
            }
        pkv_lds_order();
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f16x8 *>(&lds[w][8 * i + t][d0]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long at = p * PKV_P + 8 * i + t, j = at - r.pos;
        if (j >= 0 && j < r.n)
            *reinterpret_cast<f16x8 *>(out + (size_t)(r.row0 + j) * 2 * c.nHead * PKV_D + (size_t)kh * PKV_D + d0) = at < len ? v[i] : f16x8{};
    }
}

// ------------------------------------------------------------------ fork
// First launch: work-group 1 + s stages sequence s's page table and settles its pages' counts by its children; the first, which
// takes longest, settles the open pages: a parent's first child keeps its slot, the others (and empty ones) take, in order, the slots of the
// sequences without a child, of which there are as many.
__global__ __launch_bounds__(256) void k_pkv_fork_plan(GPT2PagedKV c, const int *__restrict__ parent) {
    // the books are read once, all of them under way together; what follows is in LDS (sequences and slots in 16 bits: every
    // work-group of the launch takes this much of it)
    __shared__ int lds[4], len[GPT2_PKV_MAX_SEQ], first[GPT2_PKV_MAX_SEQ];
    __shared__ short par[GPT2_PKV_MAX_SEQ], slot[GPT2_PKV_MAX_SEQ], spare[GPT2_PKV_MAX_SEQ];
    static_assert(GPT2_PKV_MAX_SEQ < 32768, "16 bits");
    const int tid = threadIdx.x, me = (int)blockIdx.x - 1;
    const PkvPlan plan = pkv_plan(c);
    bool bad = false;
    if (me >= 0) {
        const int full = min(c.len[me] / PKV_P, c.maxPages);
        int mine = 0;
        for (int i = tid; i < c.nSeq; i += 256) {
            const int p = parent[i];
            bad |= p < -1 || p >= c.nSeq;
            mine += p == me;
        }
        if (__syncthreads_or(bad)) return;
        int n;
        block_scan<4>(mine, lds, n);
        for (int t = tid; t < full; t += 256) {
            const int page = c.table[(size_t)me * c.maxPages + t];
            plan.tables[(size_t)me * c.maxPages + t] = page;
            if (n != 1 && pkv_page_ok(c, page)) atomicAdd(c.refs + page, n - 1);
        }
        return;
    }
#pragma nounroll
    for (int i = tid; i < c.nSeq; i += 256) {
        const int p = parent[i], at = c.slot[i];
        bad |= p < -1 || p >= c.nSeq;
        par[i] = (short)p;
        len[i] = c.len[i];
        slot[i] = (short)((unsigned)at < (unsigned)c.nSeq ? at : -1);   // one that is none stays so
        first[i] = c.nSeq;   // no child
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        plan.word[1] = !bad;
        if (bad) atomicCAS(c.status, 0, E_ARG);
    }
    if (bad) return;
    for (int i = tid; i < c.nSeq; i += 256)
        if (par[i] >= 0) atomicMin(first + par[i], i);
    __syncthreads();
    const int per = (c.nSeq + 255) / 256, i0 = min(tid * per, c.nSeq), i1 = min(i0 + per, c.nSeq);
    int n = 0, total;
    for (int i = i0; i < i1; ++i) n += first[i] == c.nSeq;
    int k = block_scan<4>(n, lds, total);
    for (int i = i0; i < i1; ++i)
        if (first[i] == c.nSeq) spare[k++] = slot[i];
    n = 0;
    for (int i = i0; i < i1; ++i) n += par[i] < 0 || first[par[i]] != i;
    k = block_scan<4>(n, lds, total);   // its barriers order spare's writes before the reads below
    for (int i = i0; i < i1; ++i) {
        const int p = par[i];
        const bool heir = p >= 0 && first[p] == i;
        plan.len[i] = p >= 0 ? len[p] : 0;
        plan.slot[i] = heir ? slot[p] : spare[k++];
        plan.from[i] = heir || p < 0 ? -1 : slot[p];
    }
}

// Second launch: blockIdx.y 0 the books, then the open page of sequence blockIdx.x, a layer's K or V and four heads each, only the
// tokens in it.  A thread copies piece `tid` (16 bytes) of the four tiles, all under way together; of a V tile's octet that the tokens
// end in, it puts those that are there among what was.  32 prompts of 8 beams, all layers: 151 MB that have to move in
// 44 us (3.4 TB/s, 4.1 with the rest of those octets; 35 us over one set of inputs, which is then in a cache); there a work-group for all the
// heads took 36.6, and for one prompt's four beams 4.0, 3.3 here.
__global__ __launch_bounds__(256) void k_pkv_fork(GPT2PagedKV c, const int *__restrict__ parent) {
    const int me = blockIdx.x, tid = threadIdx.x;
    const PkvPlan plan = pkv_plan(c);
    if (!plan.word[1]) {
        if (blockIdx.y == 0 && blockIdx.z == 0 && tid == 0) c.start[me] = c.len[me];
        return;
    }
    const int p = parent[me], len = plan.len[me];
    if (blockIdx.y == 0) {
        if (blockIdx.z) return;
        if (tid == 0) {
            c.len[me] = c.start[me] = len;
            c.slot[me] = plan.slot[me];
        }
        if (p < 0 || p == me) return;
        for (int t = tid; t < min(len / PKV_P, c.maxPages); t += 256)
            c.table[(size_t)me * c.maxPages + t] = plan.tables[(size_t)p * c.maxPages + t];
        return;
    }
    const int from = plan.from[me], to = plan.slot[me], used = len % PKV_P;
    if (used <= 0 || (unsigned)from >= (unsigned)c.nSeq || (unsigned)to >= (unsigned)c.nSeq) return;
    const int L = (blockIdx.y - 1) >> 1, kv = (blockIdx.y - 1) & 1;
    const int n = kv ? used - 8 * (tid >> 6) : 8 * (used > tid >> 3);   // the piece's values that are there
    if (n <= 0) return;
    i32x4 keep = {-1, -1, -1, -1};
#pragma unroll
    for (int e = 0; e < 4; ++e) keep[e] = n >= 2 * e + 2 ? -1 : n == 2 * e + 1 ? 0xffff : 0;
    const i32x4 *src = reinterpret_cast<const i32x4 *>(c.open + pkv_tile(c, c.nSeq, L, from, kv, 0) * PKV_TILE) + tid;
    i32x4 *dst = reinterpret_cast<i32x4 *>(c.open + pkv_tile(c, c.nSeq, L, to, kv, 0) * PKV_TILE) + tid;
    const int h = 4 * blockIdx.z;
    i32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = src[(size_t)min(h + i, c.nHead - 1) * (PKV_TILE / 8)];
    if (n < 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (v[i] & keep) | (dst[(size_t)min(h + i, c.nHead - 1) * (PKV_TILE / 8)] & ~keep);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (h + i < c.nHead) dst[(size_t)(h + i) * (PKV_TILE / 8)] = v[i];
}

// ------------------------------------------------------------------ compact
// First launch, one work-group: live pages counted, then ranked: holes below the count, movers at or past it (as many).
__global__ __launch_bounds__(1024) void k_pkv_compact_plan(GPT2PagedKV c) {
    __shared__ int lds[16];
    const int tid = threadIdx.x;
    const PkvPlan plan = pkv_plan(c);
    int n = 0, live;
    for (int p = tid; p < c.nPages; p += 1024) n += c.refs[p] != 0;
    block_scan<16>(n, lds, live);
    int holes = 0, movers = 0;
    for (int base = 0; base < c.nPages; base += 4 * 1024) {
        const int p0 = base + 4 * tid;
        bool hole[4], mover[4];
        int mine = 0;   // holes in the upper half, movers in the lower: at most 4096 of a step
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + j;
            const bool in = p < c.nPages, used = in && c.refs[p] != 0;
            hole[j] = in && !used && p < live;
            mover[j] = used && p >= live;
            mine += (hole[j] << 16) + mover[j];
            if (in) plan.map[p] = p;
        }
        int total;
        const int before = block_scan<16>(mine, lds, total);
        int kh = holes + (before >> 16), km = movers + (before & 0xffff);
        holes += total >> 16;
        movers += total & 0xffff;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (hole[j]) plan.hole[kh++] = p0 + j;
            if (mover[j]) plan.mover[km++] = p0 + j;
        }
    }
    __syncthreads();
    for (int k = tid; k < movers; k += 1024) {
        const int to = plan.hole[k], from = plan.mover[k];
        plan.map[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (tid == 0) {
        plan.word[0] = movers;
        c.status[1] = live;
    }
}

// Second launch: the first `copiers` work-groups move pages (a unit is eight tiles of one layer, and their scales), the
// others renumber the page tables.  Bound by memory: 373 pages of 12 layers, 441 MB in and out, in 93 us, 4.7 TB/s.
__global__ __launch_bounds__(256) void k_pkv_compact(GPT2PagedKV c, int copiers) {
    const int tid = threadIdx.x;
    const PkvPlan plan = pkv_plan(c);
    if ((int)blockIdx.x >= copiers) {
        const size_t i = (size_t)(blockIdx.x - copiers) * 256 + tid;
        if (i >= (size_t)c.nSeq * c.maxPages) return;
        const int s = (int)(i / c.maxPages), t = (int)(i % c.maxPages);
        if (t >= c.len[s] / PKV_P) return;
        const int page = c.table[i];
        if (pkv_page_ok(c, page)) c.table[i] = plan.map[page];
        return;
    }
    const int parts = (2 * c.nHead + 7) / 8, per = parts * c.nLayer;
    const long units = (long)plan.word[0] * per;
    for (long u = blockIdx.x; u < units; u += copiers) {
        const int k = (int)(u / per), r = (int)(u % per), L = r / parts, t0 = 8 * (r % parts);   // tiles t0 .. + 7, two at a time
        const size_t from = pkv_tile(c, c.nPages, L, plan.mover[k], 0, 0) + t0, to = pkv_tile(c, c.nPages, L, plan.hole[k], 0, 0) + t0;
        const i32x4 *src = reinterpret_cast<const i32x4 *>(c.codes + from * PKV_TILE) + tid;
        i32x4 *dst = reinterpret_cast<i32x4 *>(c.codes + to * PKV_TILE) + tid;
        const int n = min(8, 2 * c.nHead - t0), half = tid >> 7;
        i32x4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = src[2 * i + half < n ? 256 * i : 0];   // past the last: what is there anyhow
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (2 * i + half < n) dst[256 * i] = v[i];
        if (tid < n) c.scales[to + tid] = c.scales[from + tid];
    }
}

// ------------------------------------------------------------------ host
constexpr int PKV_MAX_ROWS = 1 << 23;   // a launch of a work-group a row has fewer than 2^32 threads
bool pkv_refused(const GPT2PagedKV *c, const char *what) {
    if (!c) return arg_fail(what);
    const void *p[] = {c->scales, c->table, c->len, c->start, c->slot, c->refs, c->status, c->plan};
    for (const void *q : p)
        if (!q || ((uintptr_t)q & 3)) return arg_fail(what);
    if (!c->codes || !c->open || !aligned16(c->codes) || !aligned16(c->open)) return arg_fail(what);
    if (c->headDim != PKV_D || c->nLayer < 1 || c->nLayer > 32000 || c->nHead < 1 || c->nHead > 4096 || c->nPages < 1 || c->nPages > (1 << 26) ||
        c->nSeq < 1 || c->nSeq > GPT2_PKV_MAX_SEQ || c->maxPages < 1 || c->maxPages > (1 << 25) ||
        (long)c->nSeq * c->maxPages > (1L << 30))
        return arg_fail(what);
    return false;
}

bool pkv_refused_batch(const GPT2PagedKV *c, int L, const int *rows, int nRows, const char *what) {
    if (pkv_refused(c, what)) return true;
    if (L < 0 || L >= c->nLayer || !rows || ((uintptr_t)rows & 3) || nRows < 0 || nRows > PKV_MAX_ROWS) return arg_fail(what);
    return false;
}

}  // namespace g2

using namespace g2;

static size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

extern "C" int gpt2_pkv_alloc(GPT2PagedKV *c, int nLayer, int nHead, int nPages, int nSeq, int maxLen) {
    if (!c) return arg_fail("gpt2_pkv_alloc: null cache"), 1;
    memset(c, 0, sizeof(*c));
    if (nLayer < 1 || nLayer > 32000 || nHead < 1 || nHead > 4096 || nPages < 1 || nPages > (1 << 26) || nSeq < 1 || nSeq > GPT2_PKV_MAX_SEQ || maxLen < 1 ||
        maxLen > (1 << 30) || (long)nSeq * cdiv(maxLen, PKV_P) > (1L << 30))
        return arg_fail("gpt2_pkv_alloc: sizes out of range"), 1;
    if ((double)nLayer * nHead * ((double)nPages + nSeq) > 0x1p40)   // the sizes below would not fit 64 bits
        return arg_fail("gpt2_pkv_alloc: sizes out of range"), 1;
    const size_t maxPages = cdiv(maxLen, PKV_P), tiles = (size_t)nLayer * nPages * 2 * nHead, opens = (size_t)nLayer * nSeq * 2 * nHead;
    const size_t sizes[] = {tiles * PKV_TILE, tiles * 4, opens * PKV_TILE * 2, (size_t)nSeq * maxPages * 4, (size_t)nSeq * 4, (size_t)nSeq * 4,
                            (size_t)nSeq * 4, (size_t)nPages * 4, 16, GPT2_PKV_PLAN_INTS(nSeq, maxPages, nPages) * 4};
    size_t total = 0;
    for (size_t n : sizes) total += align16(n);
    size_t freeB = 0, totB = 0;
    if (hipMemGetInfo(&freeB, &totB) != hipSuccess || total + ((size_t)64 << 20) > freeB) return set_error(E_CAPACITY, "gpt2_pkv_alloc: not enough memory"), 1;
    char *p = (char *)gpt2_dmalloc(total);
    if (!p) return 1;
    void **field[] = {(void **)&c->codes, (void **)&c->scales, (void **)&c->open, (void **)&c->table, (void **)&c->len,
                      (void **)&c->start, (void **)&c->slot, (void **)&c->refs, (void **)&c->status, (void **)&c->plan};
    c->arena = p;
    for (size_t i = 0; i < sizeof sizes / sizeof *sizes; ++i) {
        *field[i] = p;
        p += align16(sizes[i]);
    }
    c->nLayer = nLayer;
    c->nHead = nHead;
    c->headDim = PKV_D;
    c->nPages = nPages;
    c->nSeq = nSeq;
    c->maxPages = (int)maxPages;
    gpt2_pkv_reset(c);
    return 0;
}

extern "C" void gpt2_pkv_free(GPT2PagedKV *c) {
    if (c && c->arena) {
        gpt2_dfree(c->arena);
        memset(c, 0, sizeof(*c));
    }
}

extern "C" void gpt2_pkv_reset(GPT2PagedKV *c) {
    if (pkv_refused(c, "gpt2_pkv_reset: bad cache")) return;
    const int n = c->nPages > c->nSeq ? c->nPages : c->nSeq;
    hipLaunchKernelGGL(k_pkv_reset, dim3(cdiv(n, 256)), dim3(256), 0, stream(), *c);
    check_launch("k_pkv_reset");
}

extern "C" int gpt2_pkv_status(GPT2PagedKV *c) {
    if (pkv_refused(c, "gpt2_pkv_status: bad cache")) return E_ARG;
    int code = 0;
    const int none = 0;
    if (int e = gpt2_d2h(&code, c->status, sizeof code)) return e;
    if (code) {
        gpt2_h2d(c->status, &none, sizeof none);
        set_error(code, code == E_CAPACITY ? "paged K/V cache: no free page, or a sequence longer than its table" : "paged K/V cache: offsets or parents out of range");
    }
    return code;
}

extern "C" void gpt2_pkv_grow(GPT2PagedKV *c, const int *rows, int nRows) {
    if (pkv_refused_batch(c, 0, rows, nRows, "gpt2_pkv_grow: bad cache or rows")) return;
    if (c->nSeq <= 1024 && c->nPages <= 1 << 14 && nRows <= 256 * PKV_P) hipLaunchKernelGGL(k_pkv_grow<256>, dim3(1), dim3(256), 0, stream(), *c, rows, nRows);
    else hipLaunchKernelGGL(k_pkv_grow<1024>, dim3(1), dim3(1024), 0, stream(), *c, rows, nRows);
    check_launch("k_pkv_grow");
}

extern "C" void gpt2_pkv_embed(gpt2_half *x, const gpt2_half *wte, const gpt2_half *wpe, const int *ids, const GPT2PagedKV *c,
                               const int *rows, int nRows) {
    if (pkv_refused_batch(c, 0, rows, nRows, "gpt2_pkv_embed: bad cache or rows")) return;
    if (nRows == 0) return;
    if (!x || !wte || !wpe || !ids || !aligned16(x) || !aligned16(wte) || !aligned16(wpe) || ((uintptr_t)ids & 3)) {
        arg_fail("gpt2_pkv_embed: null/unaligned");
        return;
    }
    hipLaunchKernelGGL(k_pkv_embed, dim3(nRows), dim3(EMBED_THREADS), 0, stream(), x, wte, wpe, ids, *c, rows, nRows);
    check_launch("k_pkv_embed");
}

extern "C" void gpt2_pkv_append(GPT2PagedKV *c, int L, const gpt2_half *qkv, const int *rows, int nRows) {
    if (pkv_refused_batch(c, L, rows, nRows, "gpt2_pkv_append: bad cache, layer or rows")) return;
    if (nRows == 0) return;
    if (!qkv || !aligned16(qkv)) { arg_fail("gpt2_pkv_append: null/unaligned"); return; }
    const bool by_seq = nRows <= c->nSeq;
    // a wave takes one tile of a unit, two where there are work-groups for more than two rounds of the card: 48 prompts of 250 to
    // 1000 rows 42.3 -> 40.4 us, 8 prompts of up to 700 11.9 -> 13.3
    const int units = by_seq ? c->nSeq : nRows / PKV_P + c->nSeq, per = !by_seq && (long)units * c->nHead >= 8192 ? 2 : 1;
    // by sequences, up to four work-groups take turns at the units of one that has a whole prompt: 200 rows, 256 sequences in the cache
    // 27.2 us with one, 14.1 with four; a decode step's rows as long with either
    const dim3 grid(units, cdiv(2 * c->nHead, 4 * per), by_seq ? min(4, nRows / PKV_P + 1) : 1);
    const auto fn = by_seq ? k_pkv_append<true> : k_pkv_append<false>;
    hipLaunchKernelGGL(fn, grid, dim3(256), 0, stream(), *c, L, qkv, rows, nRows);
    check_launch("k_pkv_append");
}

extern "C" void gpt2_pkv_read(gpt2_half *kv, const GPT2PagedKV *c, int L, const int *rows, const int *pos, int nRows) {
    if (pkv_refused_batch(c, L, rows, nRows, "gpt2_pkv_read: bad cache, layer or rows")) return;
    if (nRows == 0) return;
    if (!kv || !aligned16(kv) || !pos || ((uintptr_t)pos & 3)) { arg_fail("gpt2_pkv_read: null/unaligned"); return; }
    hipLaunchKernelGGL(k_pkv_read, dim3(nRows / PKV_P + 2 * c->nSeq, cdiv(2 * c->nHead, 4)), dim3(256), 0, stream(), kv, *c, L, rows, pos, nRows);
    check_launch("k_pkv_read");
}

extern "C" void gpt2_pkv_fork(GPT2PagedKV *c, const int *parent) {
    if (pkv_refused(c, "gpt2_pkv_fork: bad cache")) return;
    if (!parent || ((uintptr_t)parent & 3)) { arg_fail("gpt2_pkv_fork: null/unaligned"); return; }
    hipLaunchKernelGGL(k_pkv_fork_plan, dim3(c->nSeq + 1), dim3(256), 0, stream(), *c, parent);
    hipLaunchKernelGGL(k_pkv_fork, dim3(c->nSeq, 1 + 2 * c->nLayer, cdiv(c->nHead, 4)), dim3(256), 0, stream(), *c, parent);
    check_launch("k_pkv_fork");
}

extern "C" void gpt2_pkv_compact(GPT2PagedKV *c) {
    if (pkv_refused(c, "gpt2_pkv_compact: bad cache")) return;
    const long units = (long)(c->nPages / 2) * ((2 * c->nHead + 7) / 8) * c->nLayer;   // at most: as many holes as movers
    const int copiers = (int)(units < 2048 ? units : 2048);
    hipLaunchKernelGGL(k_pkv_compact_plan, dim3(1), dim3(1024), 0, stream(), *c);
    hipLaunchKernelGGL(k_pkv_compact, dim3(copiers + cdiv((long)c->nSeq * c->maxPages, 256)), dim3(256), 0, stream(), *c, copiers);
    check_launch("k_pkv_compact");
}

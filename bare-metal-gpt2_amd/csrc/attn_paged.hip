// attn_paged.hip -- attention over the paged K/V cache (gpt2_pagedkv.h): rows of a ragged batch, a single new token or
// many a sequence, each over the tokens up to its own.
//
// att = sum_j p_j v_j / sum_j p_j, p_j = 2^(x_j - max x), x_j = (q . k_j) log2(e) / 8, with k_j = s_k q_k a page's codes and
// scale.  One pass with the running maximum and sum; scales stay out of the products (x takes s_k, the page's P.V takes s_v).
//
// A wave takes two pages at a time against 16 rows (or 32).  Scores on v_mfma_f32_16x16x32_f16 with the keys as the A operand: lane l =
// 16 g + jq names key 8 (jq / 4) + 4 t + jq % 4 of tile t, so that it receives the scores of keys 8 g .. + 7 of row jq, which
// is what the B operand of P.V holds in k-slots 8 g .. + 7; the dims are dealt so that a lane's 16 are contiguous in a K
// row (16 g .. + 15), and the V tile's order is that of the A operand of V^T (8 tokens of a dim together).  Complete pages go from
// memory to a ring in LDS, of each wave's own, by whole rows and without registers, and are made fp16, exactly, as they are taken.
// The single new token of a sequence uses two of the 16 columns; the matrix units are idle otherwise, and the sums across
// lanes that a vector form needs cost more than the empty columns.
//
// Times in this file: a launch under the tracer, the median over two sets of inputs in turn, one layer of 12 heads.
#include <cmath>

#include "pagedkv.h"

namespace g2 {

struct PagedAttn {
    GPT2PagedKV c;
    uint16_t *att;
    const uint16_t *qkv;
    const int *rows;
    int L, nRows, group, splits, per;
    float *po;      // [splits][nRows][nHead][64] unscaled sums of a split
    float4 *pml;    // [splits][nRows][nHead] their maximum and weight, and how many splits there are
};
constexpr int ATTN_SPLITS = 64;   // at most

// A page's K rows and V octets as a lane takes them.
struct PageRaw {
    i32x4 k[2], v[2];
};

// Attention of 16 rows as it accumulates: column jq is a row; o[2 i + b] element r is dim 32 i + 8 g + 2 r + b.
// m: the running maximum of x; l: the sum of the weights (in every element); o: the weighted sum of the values (both lifted).
struct AttnAcc {
    float m;
    f32x4 l, o[4];
};
__device__ __forceinline__ void attn_clear(AttnAcc &A) {
    A.m = -INFINITY;
    A.l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < 4; ++d) A.o[d] = A.l;
}

// A page (K tile, V tile) on its way to a 4 KB stage in LDS: four instructions of 1 KB, whole rows.  The 16-byte pieces of a
// K row are swizzled by the row (by choosing what each lane fetches), so that the reads below meet no bank conflict.
__device__ __forceinline__ void page_issue(const int8_t *__restrict__ k, const int8_t *__restrict__ v, char *stage) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int key = 16 * i + (lane >> 2);
        __builtin_amdgcn_global_load_lds(k + key * PKV_D + 16 * ((lane & 3) ^ (key >> 3)), G2_LDS(stage + 1024 * i), 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) __builtin_amdgcn_global_load_lds(v + 1024 * i + 16 * lane, G2_LDS(stage + PKV_TILE + 1024 * i), 16, 0, 0);
#endif
}
__device__ __forceinline__ void page_take(const char *__restrict__ stage, PageRaw &R) {
    const int lane = threadIdx.x & 63, jq = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t)
        R.k[t] = *reinterpret_cast<const i32x4 *>(stage + (8 * (jq >> 2) + 4 * t + (jq & 3)) * PKV_D + 16 * (g ^ (jq >> 2)));
#pragma unroll
    for (int i = 0; i < 2; ++i) R.v[i] = *reinterpret_cast<const i32x4 *>(stage + PKV_TILE + (g * PKV_D + 32 * i + 2 * jq) * 8);
}

// A page as the products take it: fragments of K (k[t]: dims 16 g .. + 7 and + 8 .. + 15 of the lane's key of tile t) and of V
// (v[2 i + b]: tokens 8 g .. + 7 of dim 32 i + 2 jq + b), its scales and first token.  `masked`: not every column sees all of
// it; then `only`: none does but that one (-1: all as their limits say).
struct PageFrag {
    f16x8 k[2][2], v[4];
    float sk, sv;
    int key0, only;
    bool masked;
};

// Maximum of products, as the median with infinity: fmaxf would first make each of them canonical, an instruction more.  The
// compiler does not see what `inf` is, or it would make a maximum of it.
__device__ __forceinline__ float max_by(float a, float b, float inf) { return __builtin_amdgcn_fmed3f(a, b, inf); }

// The value of the lane eight away in its row of 16.
__device__ __forceinline__ float ror8(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));
}

constexpr float ATTN_LIFT = 15.f;
// Where 8 rows or fewer are in a pass of 16 columns, column 8 + r has row r again and takes what the rounding of its weights to
// fp16 leaves in column r (AttnCols::drop is -1 there).
// N pages against Q times 16 columns, at once: a wave's chain from scores to maximum to weights to sums is what bounds it
// where few waves share a SIMD, and two pages go down it in little more than the time of one.  Column jq sees keys below lim.
template <bool SPARE, int N, int Q>
__device__ __forceinline__ void attn_pages(AttnAcc (&A)[Q], const PageFrag (&P)[N], const f16x8 (&q)[Q][2], const int (&lim)[Q], int id, float drop) {
    const int g = (threadIdx.x & 63) >> 4;
    float s[Q][N][8], scale[N], mn[Q], base[Q], inf = INFINITY;
    asm("" : "+s"(inf));
    bool moved = false;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        scale[n] = P[n].sk * (0.125f * 1.4426950408889634f);
#pragma unroll
        for (int u = 0; u < Q; ++u)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 y = __builtin_amdgcn_mfma_f32_16x16x32_f16(P[n].k[t][0], q[u][0], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(P[n].k[t][1], q[u][1], y, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[u][n][4 * t + r] = y[r];
            }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (P[n].masked)
#pragma unroll
            for (int u = 0; u < Q; ++u) {
                const int left = (P[n].only < 0 || P[n].only == id ? lim[u] : 0) - P[n].key0 - 8 * g;
#pragma unroll
                for (int e = 0; e < 8; ++e) s[u][n][e] = e < left ? s[u][n][e] : -INFINITY;
            }
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < N; ++n)
            mx = fmaxf(mx, max_by(max_by(max_by(s[u][n][0], s[u][n][1], inf), max_by(s[u][n][2], s[u][n][3], inf), inf),
                                  max_by(max_by(s[u][n][4], s[u][n][5], inf), max_by(s[u][n][6], s[u][n][7], inf), inf), inf) * scale[n]);
        mn[u] = fmaxf(A[u].m, group_max(mx));
        base[u] = mn[u] == -INFINITY ? 0.f : mn[u];   // a column that sees none of these keys
        moved |= mn[u] > A[u].m;
    }
    if (__ballot(moved)) {   // the maximum moves rarely after the first pages
#pragma unroll
        for (int u = 0; u < Q; ++u) {
            const float corr = __builtin_amdgcn_exp2f(A[u].m - base[u]);
            A[u].m = mn[u];
            A[u].l *= corr;
#pragma unroll
            for (int i = 0; i < 4; ++i) A[u].o[i] *= corr;
        }
    }
    // The weights are held 2^ATTN_LIFT times as large, the largest at 2^15, so that the many small ones of a long context stay above
    // what fp16 rounds to fewer bits (2^-29 of the largest) or to nothing (2^-40).
    // They are rounded to fp16, which with 16 or 32 rows costs an output about half as much as its own rounding (1.1e-4 of it against
    // 2.1e-4; second parts there, in products of their own, made 8 prompts of up to 600 rows take 58 us a call instead of 52).  With columns to
    // spare a second column takes what is left, w - fp16(w), which is exact in fp32: 22 bits of a weight in all, for 0.3 us of the 7.6 that
    // a call with a single token over 1000 takes.
    f16x8 p[Q][N];
    float lift[Q], rate[N];
    bool huge = false;
#pragma unroll
    for (int n = 0; n < N; ++n) rate[n] = scale[n];
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        lift[u] = ATTN_LIFT - base[u];
        huge |= fabsf(base[u]) >= 0x1p20f;
    }
    if (__ballot(huge)) {
        // The maximum is a rounded product and x an exact one, which may pass it by 2^-24 of its size: by so much that fp16 could
        // overflow.  Here x is the rounded product, too.
#pragma clang fp contract(off)
#pragma unroll
        for (int u = 0; u < Q; ++u) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = s[u][n][e] * scale[n];
                    s[u][n][e] = x - base[u];
                }
            lift[u] = ATTN_LIFT;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) rate[n] = 1.f;
    }
#pragma unroll
    for (int u = 0; u < Q; ++u)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[u][n][e], rate[n], lift[u]));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[u][n][e + 1], rate[n], lift[u]));
                const f16x2 w = {(f16)x, (f16)y};
                p[u][n][e] = SPARE ? (f16)fmaf((float)w[0], drop, x) : w[0];
                p[u][n][e + 1] = SPARE ? (f16)fmaf((float)w[1], drop, y) : w[1];
            }
    // their sum, of the fp16 values as they are multiplied, on the matrix units too: a row of ones
    const f16x8 one = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int u = 0; u < Q; ++u)
#pragma unroll
        for (int n = 0; n < N; ++n) A[u].l = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, p[u][n], A[u].l, 0, 0, 0);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < Q; ++u) {
                const f32x4 y = __builtin_amdgcn_mfma_f32_16x16x32_f16(P[n].v[i], p[u][n], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) A[u].o[i][r] = fmaf(y[r], P[n].sv, A[u].o[i][r]);
            }
}

__device__ __forceinline__ void page_widen(const PageRaw &R, PageFrag &P) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        P.k[t][0] = i8x8_to_f16x8(uint2{(uint32_t)R.k[t][0], (uint32_t)R.k[t][1]});
        P.k[t][1] = i8x8_to_f16x8(uint2{(uint32_t)R.k[t][2], (uint32_t)R.k[t][3]});
        P.v[2 * t] = i8x8_to_f16x8(uint2{(uint32_t)R.v[t][0], (uint32_t)R.v[t][1]});
        P.v[2 * t + 1] = i8x8_to_f16x8(uint2{(uint32_t)R.v[t][2], (uint32_t)R.v[t][3]});
    }
}

// The open page: fp16 in the same order; tokens at or past `used` are whatever was there, so their values are cleared.
__device__ __forceinline__ void open_take(const uint16_t *__restrict__ k, const uint16_t *__restrict__ v, int used, PageFrag &P) {
    const int lane = threadIdx.x & 63, jq = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint16_t *row = k + (8 * (jq >> 2) + 4 * t + (jq & 3)) * PKV_D + 16 * g;
        P.k[t][0] = *reinterpret_cast<const f16x8 *>(row);
        P.k[t][1] = *reinterpret_cast<const f16x8 *>(row + 8);
    }
    const int n = used - 8 * g;   // of the lane's 8 tokens, those that are there
    i32x4 keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) keep[e] = n >= 2 * e + 2 ? -1 : n == 2 * e + 1 ? 0xffff : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        P.v[i] = __builtin_bit_cast(f16x8, *reinterpret_cast<const i32x4 *>(v + (g * PKV_D + 32 * (i >> 1) + 2 * jq + (i & 1)) * 8) & keep);
    P.sk = P.sv = 1.f;
}

// What a pass goes over, as steps of a page each: the first `shared` pages of sequence seq0, for every column, then the
// pages from there on of each of `beams` sequences (lane b holds beam b's), for that beam's column alone.
struct AttnSteps {
    int seq0, len0, slot0, shared, total;
    int beams, seq, len, slot, off;   // off: own pages of the beams before
};

// One pass: Q times 16 columns (column jq: row `row` of the activations, -1 for none, which sees the keys below `lim`; every
// column sees those below `first`), one head, split z of the steps.  The W waves take steps in turn and join in LDS.
// One loop, two steps at a time, and little code around it: the instructions of a short call come from L2 (the call with one
// token took 4.4 us with 8.5 KB of code and 5.4 with 11.6).
template <int W>
constexpr int ATTN_STAGES = W > 4 ? 4 : 2;   // of 4 KB
template <int W, int Q>
struct AttnLds {
    char ring[W][ATTN_STAGES<W> * 2 * PKV_TILE];
    float m[W][16 * Q], l[W][16 * Q];
    static_assert(Q * 4 * 64 * 16 <= ATTN_STAGES<W> * 2 * PKV_TILE, "a wave's sums take its ring's place");
};
// id: which of the pass's rows or beams the column has; drop: 0, or -1 where it has the rest of that row's weights.
template <int Q>
struct AttnCols {
    int row[Q], lim[Q], first, id;
    float drop;
};
template <int W, bool BEAMS, bool SPARE, int Q>
__device__ __forceinline__ void attn_pass(const PagedAttn &a, const AttnSteps &st, int h, int z, const AttnCols<Q> &col, AttnLds<W, Q> &lds) {
    const GPT2PagedKV &c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), jq = lane & 15, g = lane >> 4;
    const int E = c.nHead * PKV_D;
    const int splits = min(a.splits, max(1, (st.total + a.per - 1) / a.per)), stride = splits * W;
    if (z >= splits) return;   // the whole work-group
    f16x8 q[Q][2] = {};
    AttnAcc A[Q];
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        const uint16_t *qrow = a.qkv + (size_t)max(col.row[u], 0) * 3 * E + h * PKV_D + 16 * g;
        if (col.row[u] >= 0) {
            q[u][0] = *reinterpret_cast<const f16x8 *>(qrow);
            q[u][1] = *reinterpret_cast<const f16x8 *>(qrow + 8);
        }
        attn_clear(A[u]);
    }

    const size_t vstep = (size_t)c.nHead * PKV_TILE;   // from a page's K tile to its V tile
    const int8_t *const layer = c.codes + pkv_tile(c, c.nPages, a.L, 0, 0, h) * PKV_TILE;
    for (int t0 = z * W + w; t0 < st.total; t0 += 64 * stride) {
        // the wave's next 64 steps, a lane each: the page's number in its sequence, whose it is, the pool's page, scales
        const int t = t0 + stride * lane;
        int b = -1, p = t, seq = st.seq0, len = st.len0;
        if constexpr (BEAMS) {
            const int u = t - st.shared;
            for (int k = 0; k < st.beams; ++k)
                if (u >= __builtin_amdgcn_readlane(st.off, k)) b = k;
            const int from = max(b, 0), off = __shfl(st.off, from, 64), s1 = __shfl(st.seq, from, 64), n1 = __shfl(st.len, from, 64);
            if (b >= 0) {
                p = st.shared + u - off;
                seq = s1;
                len = n1;
            }
        }
        const int full = len / PKV_P;
        int page = t < st.total && p < full ? c.table[(size_t)seq * c.maxPages + p] : -1;
        const bool there = pkv_page_ok(c, page);
        uint64_t opened = __ballot(t < st.total && p == full);
        float sk = 0.f, sv = 0.f;
        if (there) {
            const size_t at = pkv_tile(c, c.nPages, a.L, page, 0, h);
            sk = c.scales[at];
            sv = c.scales[at + c.nHead];
        }
        const int who = p << 5 | (b + 1);   // p < 2^25 (maxPages)
        const size_t off = (size_t)max(page, 0) * 2 * c.nHead * PKV_TILE;   // of the page in the layer, in bytes
        // complete pages through the wave's own ring of stages
        uint64_t left = __ballot(there), todo = left;
        int stage = 0, ahead = 0;   // pages under way
        char *const ring = lds.ring[w];
        auto issue = [&](int s) {
            const int j = __builtin_ctzll(todo);
            const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)off, j), hi = __builtin_amdgcn_readlane((int)(uint32_t)(off >> 32), j);
            const int8_t *k = layer + ((size_t)hi << 32 | lo);
            page_issue(k, k + vstep, ring + 2 * PKV_TILE * s);
            todo &= todo - 1;
            ++ahead;
        };
#pragma nounroll
        for (int s = 0; s < ATTN_STAGES<W> && todo; ++s) issue(s);
        asm volatile("" : "+v"(sk), "+v"(sv));   // waited for here, once, and not with every page under way in the loop
        // Two steps at a time: two complete pages, or one and an open one, or an open one; a place without a step takes
        // part with whatever the stage holds (codes are finite) and no column sees it.
        while (left | opened) {
            ahead = max(ahead - 2, 0);
            wait_tiles<4, ATTN_STAGES<W> - 2>(ahead);
            asm volatile("" ::: "memory");
            PageFrag P[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const bool open = n == 1 && !left && opened, none = !open && !left;
                const int j = open ? __builtin_ctzll(opened) : none ? 0 : __builtin_ctzll(left);
                const int x = __builtin_amdgcn_readlane(who, j), bj = (x & 31) - 1;
                P[n].key0 = (x >> 5) * PKV_P;
                P[n].only = none ? 16 : BEAMS ? bj : -1;
                P[n].masked = none || open || (BEAMS && bj >= 0) || P[n].key0 + PKV_P > col.first;
                if (open) {
                    const int slot = BEAMS && bj >= 0 ? __builtin_amdgcn_readlane(st.slot, max(bj, 0)) : st.slot0;
                    const uint16_t *k = c.open + pkv_tile(c, c.nSeq, a.L, slot, 0, h) * PKV_TILE;
                    open_take(k, k + vstep, __builtin_amdgcn_readlane(len, j) - P[n].key0, P[n]);
                    opened &= opened - 1;
                } else {
                    PageRaw R;
                    page_take(ring + 2 * PKV_TILE * (stage + n), R);
                    page_widen(R, P[n]);
                    P[n].sk = none ? 1.f : lane_f(sk, j);
                    P[n].sv = none ? 1.f : lane_f(sv, j);
                    left &= left - 1;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the stages are filled again
            if (todo) issue(stage);
            if (todo) issue(stage + 1);
            stage = (stage + 2) % ATTN_STAGES<W>;
            attn_pages<SPARE>(A, P, q, col.lim, col.id, col.drop);
        }
    }
    // the waves' sums to one maximum, then together
#pragma unroll
    for (int u = 0; u < Q; ++u)
        if (g == 0) lds.m[w][16 * u + jq] = A[u].m;
    __syncthreads();
    float mx[Q];
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        mx[u] = -INFINITY;
#pragma unroll
        for (int v = 0; v < W; ++v) mx[u] = fmaxf(mx[u], lds.m[v][16 * u + jq]);
        const float f = A[u].m != -INFINITY ? __builtin_amdgcn_exp2f(A[u].m - mx[u]) : 0.f;   // 0: the wave had no key for the column
        if (col.row[u] >= 0) {
            if (g == 0) lds.l[w][16 * u + jq] = A[u].l[0] * f;
#pragma unroll
            for (int d = 0; d < 4; ++d) reinterpret_cast<f32x4 *>(lds.ring[w])[64 * (4 * u + d) + lane] = A[u].o[d] * f;   // the ring is idle
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        // two waves a column block: dims 32 d + 8 g .. + 7 of the column's row
        const int d = w - 2 * u, row = col.row[u];
        if (d < 0 || d > 1 || row < 0) continue;
        float L = 0.f;
        f32x4 y[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const f32x4 *o = reinterpret_cast<const f32x4 *>(lds.ring[v]) + 64 * (4 * u + 2 * d) + lane;
            L += lds.l[v][16 * u + jq];
            y[0] += o[0];
            y[1] += o[64];
        }
        if constexpr (SPARE)
            if (__ballot(col.drop != 0.f)) {   // a row's two columns, eight apart, together
                L += ror8(L);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    y[0][r] += ror8(y[0][r]);
                    y[1][r] += ror8(y[1][r]);
                }
                if (col.drop != 0.f) continue;
            }
        if (a.splits == 1) {
            const float inv = L != 0.f ? 1.f / L : 0.f;   // no key: 0
            f16x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (f16)(y[e & 1][e >> 1] * inv);
            *reinterpret_cast<f16x8 *>(a.att + (size_t)row * E + h * PKV_D + 32 * d + 8 * g) = o;
        } else {
            const size_t at = ((size_t)z * a.nRows + row) * c.nHead + h;
            float *o = a.po + at * PKV_D + 32 * d + 8 * g;
            *reinterpret_cast<f32x4 *>(o) = f32x4{y[0][0], y[1][0], y[0][1], y[1][1]};
            *reinterpret_cast<f32x4 *>(o + 4) = f32x4{y[0][2], y[1][2], y[0][3], y[1][3]};
            if (d == 0 && g == 0) a.pml[at] = float4{mx[u], L, __int_as_float(splits), 0.f};
        }
    }
}

// Rows 16 Q rb .. of one sequence, 16 Q of them, as a pass; with SPARE, up to 8 in two columns each.
template <bool SPARE, int Q>
__device__ __forceinline__ AttnSteps attn_rows(const PkvSeq &s, int seq, int rb, AttnCols<Q> &col) {
    const int i0 = 16 * Q * rb, pages = (s.start + min(s.n, i0 + 16 * Q) + PKV_P - 1) / PKV_P, jq = threadIdx.x & 15;
    const bool two = SPARE && s.n <= 8;
    col.id = two ? jq & 7 : jq;
    col.drop = two && jq >= 8 ? -1.f : 0.f;
#pragma unroll
    for (int u = 0; u < Q; ++u) {
        const int i = i0 + 16 * u + col.id;
        col.row[u] = i < s.n ? s.row0 + i : -1;
        col.lim[u] = i < s.n ? s.start + i + 1 : 0;
    }
    col.first = s.start + i0 + 1;
    return {seq, s.len, s.slot, pages, pages, 0, 0, 0, 0, 0};
}

// The beams of a group, one row each at most, as a pass.  Lane b holds beam b's sequence; `on`: those with a row.
__device__ __forceinline__ AttnSteps attn_beams(const PagedAttn &a, const PkvSeq &s, int seq0, uint64_t on, AttnCols<1> &col) {
    const GPT2PagedKV &c = a.c;
    const int lane = threadIdx.x & 63, jq = lane & 15, one = __builtin_ctzll(on);
    const bool two = a.group <= 8;   // beams in two columns each
    const int id = two ? jq & 7 : jq;
    // the leading pages that all share, complete in each
    int least = s.n ? s.len / PKV_P : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));   // beams are lanes 0 .. 15
    least = __builtin_amdgcn_readfirstlane(least);
    int shared = 0;
    for (; shared < least; shared += 64) {
        const int p = shared + lane;
        bool same = p < least;
        int page[16];   // all loads under way before the first comparison
#pragma unroll
        for (int b = 0; b < 16; ++b) page[b] = c.table[(size_t)(seq0 + (on >> b & 1 ? b : one)) * c.maxPages + min(p, c.maxPages - 1)];
#pragma unroll
        for (int b = 1; b < 16; ++b) same &= page[b] == page[0];
        const uint64_t differ = __ballot(!same);
        if (differ) {
            shared += __builtin_ctzll(differ);
            break;
        }
    }
    const int own = s.n ? (s.len + PKV_P - 1) / PKV_P - shared : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const int v = __shfl_up(sum, o, 64);
        if (lane >= o) sum += v;
    }
    const int total = shared + __builtin_amdgcn_readlane(sum, 15);
    const int n = __shfl(s.n, id, 64), row = __shfl(s.row0, id, 64), len = __shfl(s.len, id, 64);
    col = {{n ? row : -1}, {n ? len : 0}, shared * PKV_P, id, two && jq >= 8 ? -1.f : 0.f};
    return {seq0 + one, __builtin_amdgcn_readlane(s.len, one), 0, shared, total, a.group, seq0 + min(lane, a.group - 1), s.len, s.slot, sum - own};
}

// One row a sequence, nearly always (no more rows than sequences): a work-group per sequence, head and split (gridDim.z of them, for
// sequences that have more than 16 rows after all).  16 contexts up to 16384 tokens: 57.8 us for 268 MB, 4.6 TB/s, bound by memory; 48
// of up to 1000 16.9; one of 1000 tokens 7.5, by the chain of loads from the books to the pages and by its code's way from L2 ...
template <int W>
__global__ __launch_bounds__(64 * W) void k_pkv_attn_one(PagedAttn a) {
    __shared__ __attribute__((aligned(1024))) AttnLds<W, 1> lds;
    const int h = blockIdx.x % a.c.nHead, seq = blockIdx.x / a.c.nHead;
    const PkvSeq s = pkv_seq(a.c, a.rows, a.nRows, seq);
#pragma nounroll
    for (int rb = blockIdx.z; 16 * rb < s.n; rb += gridDim.z) {
        if (rb >= (int)gridDim.z) __syncthreads();
        AttnCols<1> col;
        const AttnSteps st = attn_rows<true>(s, seq, rb, col);
        attn_pass<W, false, true, 1>(a, st, h, blockIdx.y, col, lds);
    }
}

// ... or per group of beams, together where they have a row each at most and there are two: shared pages are read once, and a beam is a
// column.  8 x 8 beams over 900 tokens 13.0 us, as 64 sequences of their own 14.0; bound as the single row's, with the comparison of the tables in the chain.
template <int W>
__global__ __launch_bounds__(64 * W) void k_pkv_attn_beams(PagedAttn a) {
    __shared__ __attribute__((aligned(1024))) AttnLds<W, 1> lds;
    const int h = blockIdx.x % a.c.nHead, lane = threadIdx.x & 63;
    const int seq0 = blockIdx.x / a.c.nHead * a.group;
    PkvSeq s = pkv_seq(a.c, a.rows, a.nRows, seq0 + min(lane, a.group - 1));
    if (lane >= a.group) s.n = 0;
    const uint64_t on = __ballot(s.n > 0);
    if (!on) return;
    const bool together = (on & (on - 1)) && !__ballot(s.n > 1);   // else one sequence after another
    int b = __builtin_ctzll(on), rb = 0;
    for (;;) {
        AttnSteps st;
        AttnCols<1> col;
        PkvSeq u;
        u.n = 0;
        if (together) {
            st = attn_beams(a, s, seq0, on, col);
        } else {
            u.start = __builtin_amdgcn_readlane(s.start, b);
            u.len = __builtin_amdgcn_readlane(s.len, b);
            u.row0 = __builtin_amdgcn_readlane(s.row0, b);
            u.n = __builtin_amdgcn_readlane(s.n, b);
            u.slot = __builtin_amdgcn_readlane(s.slot, b);
            st = attn_rows<true>(u, seq0 + b, rb, col);
            st.off = 0x7fffffff;   // no step is a beam's own
        }
        attn_pass<W, true, true, 1>(a, st, h, blockIdx.y, col, lds);
        if (together) break;
        if (16 * ++rb >= u.n) {
            const uint64_t more = on & ~((2ull << b) - 1);   // b < 16
            if (!more) break;
            b = __builtin_ctzll(more);
            rb = 0;
        }
        __syncthreads();
    }
}

// Any number of rows a sequence: a work-group per 16 Q of them, head and split.  8 prompts of up to 600 rows over up to 2000 tokens, Q = 2:
// 58 us (52 a call among others, whose first work-groups fill its uneven end: 0.33 PFLOP/s of what is not masked); vector instructions, 79% of
// the cycles (some 115 for 16 rows and a page), bound it, at the three waves a SIMD that its registers leave.
template <int Q>
__global__ __launch_bounds__(256) void k_pkv_attn_rows(PagedAttn a) {
    __shared__ __attribute__((aligned(1024))) AttnLds<4, Q> lds;
    const int h = blockIdx.x % a.c.nHead;
    int rb = blockIdx.x / a.c.nHead;
    const int seq = pkv_seq_of_unit(rb, a.c.nSeq, [&](int s) { return (pkv_seq(a.c, a.rows, a.nRows, s).n + 16 * Q - 1) / (16 * Q); });
    if (seq < 0) return;
    const PkvSeq s = pkv_seq(a.c, a.rows, a.nRows, seq);
    AttnCols<Q> col;
    const AttnSteps st = attn_rows<false>(s, seq, (s.n + 16 * Q - 1) / (16 * Q) - 1 - rb, col);   // the longest first
    attn_pass<4, false, false, Q>(a, st, h, blockIdx.y, col, lds);
}

// Many rows a sequence: a work-group per 64 of them and head, a wave per 16, every wave over all pages.  The four waves share
// the work of turning a page into fragments: a wave takes a quarter (a K tile's half, or 16 of V's 32 pairs of dims) from memory to
// registers, 16 bytes a lane, ATTN_AHEAD pairs of pages ahead, to fp16, and to LDS in the order in which all four read it.  16 rows a
// work-group would read each page from L2 four times as often, which bounds that form (66 us for 8 prompts of up to 600 rows over
// up to 2000 tokens).
constexpr int ATTN_AHEAD = 2;   // pairs of pages
__global__ __launch_bounds__(256, 4) void k_pkv_attn_block(PagedAttn a) {
    __shared__ __attribute__((aligned(1024))) f16x8 lds[2][2][8][64];   // two pages at a time: K (2 t + half), then V (4 + 2 i + b)
    const GPT2PagedKV &c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), jq = lane & 15, g = lane >> 4;
    const int h = blockIdx.x % c.nHead, E = c.nHead * PKV_D;
    int rb = blockIdx.x / c.nHead;
    const int seq = pkv_seq_of_unit(rb, c.nSeq, [&](int s) { return (pkv_seq(c, a.rows, a.nRows, s).n + 63) / 64; });
    if (seq < 0) return;
    const PkvSeq s = pkv_seq(c, a.rows, a.nRows, seq);
    rb = (s.n + 63) / 64 - 1 - rb;   // the longest first
    const int i0 = 64 * rb + 16 * w, i = i0 + jq, full = s.len / PKV_P;
    const int last = s.start + min(s.n, 64 * rb + 64), pages = (last + PKV_P - 1) / PKV_P;   // of the work-group's rows
    const int first = s.start + i0 + 1, lim = i < s.n ? s.start + i + 1 : 0;                 // keys that the wave's rows, and row i, see
    const int end = i0 < s.n ? s.start + min(s.n, i0 + 16) : 0;                               // ... and any of the wave's
    const uint16_t *qrow = a.qkv + (size_t)(s.row0 + min(i, s.n - 1)) * 3 * E + h * PKV_D + 16 * g;
    const f16x8 q[1][2] = {{*reinterpret_cast<const f16x8 *>(qrow), *reinterpret_cast<const f16x8 *>(qrow + 8)}};
    AttnAcc A[1];
    attn_clear(A[0]);
    const int limit[1] = {lim};

    // The wave's quarter of a page: where its 16 bytes a lane lie in the tile, and the fragments' slots that they fill.  K: wave
    // t takes keys 8 x + 4 t + y, lane 16 x + 4 y + z dims 16 z .. + 15 of one, for lane 16 z + 4 x + y of the product.
    const int from = w < 2 ? (8 * (lane >> 4) + 4 * w + ((lane >> 2) & 3)) * PKV_D + 16 * (lane & 3) : (g * PKV_D + 32 * (w - 2) + 2 * jq) * 8;
    // (swizzled: 16 lanes that write, or read, together meet no bank conflict)
    auto swizzle = [](int l) { return l ^ (l >> 4) << 2; };
    const int slot = swizzle(w < 2 ? 16 * (lane & 3) + 4 * (lane >> 4) + ((lane >> 2) & 3) : lane), mine = swizzle(lane);
    const int8_t *const quarter = c.codes + pkv_tile(c, c.nPages, a.L, 0, w >> 1, h) * PKV_TILE + from;
    uint32_t off_lo = 0, off_hi = 0;   // of the lane's page in the layer, in bytes
    int page = -1;
    float sk = 0.f, sv = 0.f;
    auto fetch = [&](int base) {   // numbers and scales of the 64 pages from `base` on, a lane each
        const int p = base + lane;
        page = p < min(pages, full) ? c.table[(size_t)seq * c.maxPages + p] : -1;
        if (!pkv_page_ok(c, page)) page = -1;
        const size_t off = (size_t)max(page, 0) * 2 * c.nHead * PKV_TILE;   // pages that are none read page 0, and are skipped below
        off_lo = (uint32_t)off;
        off_hi = (uint32_t)(off >> 32);
        sk = sv = 0.f;
        if (page >= 0) {
            const size_t at = pkv_tile(c, c.nPages, a.L, page, 0, h);
            sk = c.scales[at];
            sv = c.scales[at + c.nHead];
        }
    };
    auto part = [&](int p) {
        const uint32_t lo = __builtin_amdgcn_readlane((int)off_lo, p), hi = __builtin_amdgcn_readlane((int)off_hi, p);
        return *reinterpret_cast<const i32x4 *>(quarter + ((size_t)hi << 32 | lo));
    };
    auto put = [&](const i32x4 v, int buf, int n) {
        lds[buf][n][2 * w][slot] = i8x8_to_f16x8(uint2{(uint32_t)v[0], (uint32_t)v[1]});
        lds[buf][n][2 * w + 1][slot] = i8x8_to_f16x8(uint2{(uint32_t)v[2], (uint32_t)v[3]});
    };
    auto get = [&](int buf, int n, int p, float k, float v, PageFrag &P) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            P.k[t][0] = lds[buf][n][2 * t][mine];
            P.k[t][1] = lds[buf][n][2 * t + 1][mine];
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) P.v[d] = lds[buf][n][4 + d][mine];
        P.sk = k;
        P.sv = v;
        P.key0 = p * PKV_P;
        P.only = -1;
        P.masked = P.key0 + PKV_P > first;
    };
    const int whole = min(pages, full);
    for (int base = 0; base < whole; base += 64) {
        fetch(base);
        const int n = min(64, whole - base);
        // pairs of pages; one that is none, or past the last, takes part with no key to see (and a scale that is a number)
        i32x4 raw[ATTN_AHEAD][2];
#pragma unroll
        for (int j = 0; j < ATTN_AHEAD; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) raw[j][k] = part(min(2 * j + k, n - 1));
#pragma unroll
        for (int k = 0; k < 2; ++k) put(raw[0][k], 0, k);
        lds_barrier();
        for (int p0 = 0; p0 < n; p0 += 2 * ATTN_AHEAD) {
#pragma unroll
            for (int j = 0; j < ATTN_AHEAD; ++j) {
                const int p = p0 + 2 * j;
                if (p < n) {   // the same for all waves
#pragma unroll
                    for (int k = 0; k < 2; ++k) raw[j][k] = part(min(p + 2 * ATTN_AHEAD + k, n - 1));
                    if (p + 2 < n)
#pragma unroll
                        for (int k = 0; k < 2; ++k) put(raw[(j + 1) % ATTN_AHEAD][k], (j + 1) & 1, k);
                    if ((base + p) * PKV_P < end) {
                        PageFrag P[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int pk = p + k, at = min(pk, 63);
                            get(j & 1, k, base + pk, lane_f(sk, at), lane_f(sv, at), P[k]);
                            if (pk >= n || __builtin_amdgcn_readlane(page, at) < 0) {
                                P[k].sk = P[k].sv = 1.f;
                                P[k].only = 16;
                                P[k].masked = true;
                            }
                        }
                        attn_pages<false>(A, P, q, limit, jq, 0.f);
                    }
                    lds_barrier();
                }
            }
        }
    }
    if (pages > full) {   // the open page: fp16 as it lies, tokens that are not there cleared
        const uint16_t *tile = c.open + pkv_tile(c, c.nSeq, a.L, s.slot, w >> 1, h) * PKV_TILE + from;
        const i32x4 x = *reinterpret_cast<const i32x4 *>(tile), y = *reinterpret_cast<const i32x4 *>(tile + 8);
        const int n = w < 2 ? 8 : s.len - full * PKV_P - 8 * g;
        i32x4 keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) keep[e] = n >= 2 * e + 2 ? -1 : n == 2 * e + 1 ? 0xffff : 0;
        lds[0][0][2 * w][slot] = __builtin_bit_cast(f16x8, x & keep);
        lds[0][0][2 * w + 1][slot] = __builtin_bit_cast(f16x8, y & keep);
        lds_barrier();
        if (full * PKV_P < end) {
            PageFrag P[1];
            get(0, 0, full, 1.f, 1.f, P[0]);
            attn_pages<false>(A, P, q, limit, jq, 0.f);
        }
    }
    const float inv = A[0].l[0] != 0.f ? 1.f / A[0].l[0] : 0.f;
    if (i < s.n) {
        uint16_t *out = a.att + (size_t)(s.row0 + i) * E + h * PKV_D + 8 * g;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            f16x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (f16)(A[0].o[2 * d + (e & 1)][e >> 1] * inv);
            *reinterpret_cast<f16x8 *>(out + 32 * d) = o;
        }
    }
}

// Joins the splits: a wave per row and head; lane z holds split z's maximum and weight, then lane d dim d.  BY_SEQ: blockIdx.x
// is a sequence, with a row nearly always; else a row, whose sequence is looked up (a few dependent loads more).
template <bool BY_SEQ>
__global__ __launch_bounds__(256) void k_pkv_attn_join(PagedAttn a) {
    static_assert(ATTN_SPLITS <= 64, "a lane a split");
    const int lane = threadIdx.x & 63, h = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= a.c.nHead) return;
    const int seq = BY_SEQ ? (int)blockIdx.x : pkv_seq_of_row(a.rows, a.c.nSeq, blockIdx.x);
    if (seq < 0) return;
    const PkvSeq s = pkv_seq(a.c, a.rows, a.nRows, seq);
    if (s.n == 0) return;
    const size_t per = (size_t)a.nRows * a.c.nHead;
    const int row0 = BY_SEQ ? s.row0 : (int)blockIdx.x;
    for (int row = row0; row < (BY_SEQ ? s.row0 + s.n : row0 + 1); ++row) {
        const size_t at = (size_t)row * a.c.nHead + h;
        const int splits = max(1, min(__builtin_amdgcn_readfirstlane(__float_as_int(a.pml[at].z)), a.splits));
        const float4 ml = a.pml[at + per * min(lane, splits - 1)];
        const bool on = lane < splits && ml.y != 0.f;
        const float mx = wave_max_u(on ? ml.x : -INFINITY), f = on ? __builtin_amdgcn_exp2f(ml.x - mx) : 0.f;
        const float L = wave_sum_u(on ? ml.y * f : 0.f);
        float o = 0.f;
        for (int z = 0; z < splits; z += 8) {   // eight loads under way; f is 0 past the last split
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = a.po[(at + per * min(z + i, splits - 1)) * PKV_D + lane];
#pragma unroll
            for (int i = 0; i < 8; ++i) o = fmaf(v[i], lane_f(f, z + i), o);
        }
        a.att[at * PKV_D + lane] = f2h(L != 0.f ? o / L : 0.f);
    }
}

// How a call runs: its form, and how the steps are split over work-groups: at least `per` of them each, into `splits` at most.
//   ONE    no more rows than sequences: a sequence (or group of beams) a work-group.  Without a group up to 4 of them take turns at the
//          16-row blocks of a sequence that has a whole prompt: 200 rows after 800 tokens, 256 sequences in the cache, 80 us with one, 54 with
//          two, 31 with four; 256 single rows over up to 400 tokens 29.0, 28.7, 31.3, over up to 100 20.0, 20.0, 23.1.
//   ROWS1  16 rows a work-group, keys split over its waves.
//   ROWS2  32 of them, from 32 rows a sequence on: a page is made fp16 once for twice the rows (8 prompts of up to 600 over 2000 tokens 58 us,
//          66 with ROWS1; one of 1000 rows 11.8, 11.6 and with BLOCK 20).
//   BLOCK  64, pages shared through LDS, where that makes eight work-groups a CU: 32 prompts of up to 1000 rows 83 us, 102 with
//          ROWS2; 8 of up to 600 over 2000 tokens 62 us, 58 with ROWS2.
// No splits for caches whose sequences a work-group's waves get through in the time of a second launch, nor where the rows alone
// make one work-group a CU (8 prompts of up to 200 rows over up to 2000 tokens: 26 us, 26 + 7 with two splits).  Where splits of 64
// pages fill the card they stream best (16 contexts up to 16384 tokens: 57.8 us, 58.5 with 32 pages each, 67.3 with 96); with fewer
// sequences, or groups of beams, as many as make 512 work-groups, of 16 pages at least (8 x 8 beams over 2100 tokens: 5 splits 13.0 us,
// 2 splits 15.6, 9 splits 15.4; over 4096: 5 16.2, 3 20.0, 9 18.9).
enum AttnForm { ATTN_ONE, ATTN_ROWS1, ATTN_ROWS2, ATTN_BLOCK };
struct AttnPlan {
    AttnForm form;
    int groups, splits, per, deep;   // work-groups of a split; deep: times as many, where a sequence may have many rows
};
static AttnPlan attn_plan(const GPT2PagedKV *c, int nRows, int group) {
    AttnPlan p;
    p.form = nRows <= c->nSeq ? ATTN_ONE : nRows / 32 < c->nSeq ? ATTN_ROWS1 : (long)(nRows / 64) * c->nHead < 2048 ? ATTN_ROWS2 : ATTN_BLOCK;
    const int rows = p.form == ATTN_ROWS1 ? 16 : p.form == ATTN_ROWS2 ? 32 : 64;   // of a work-group
    p.groups = (p.form == ATTN_ONE ? c->nSeq / group : nRows / rows + c->nSeq) * c->nHead;
    p.splits = 1;
    p.per = 64;
    p.deep = p.form == ATTN_ONE && group == 1 ? min(cdiv(nRows, 16), p.groups < 2048 ? 4 : 2) : 1;
    const long busy = (long)(p.form == ATTN_ONE ? c->nSeq / group : nRows / rows + 1) * c->nHead;   // work-groups with something to do, about
    if (p.form == ATTN_BLOCK || c->maxPages <= 64 || (p.form != ATTN_ONE && busy > 256)) return p;
    const long share = 512 / max(busy, 1L);   // splits that fill the card
    p.per = min(64, max(16, share > 0 ? cdiv(c->maxPages, (int)share) : 64));
    p.splits = cdiv(c->maxPages, p.per);
    if (p.splits > ATTN_SPLITS) p.splits = ATTN_SPLITS;
    return p;
}

}  // namespace g2

using namespace g2;

extern "C" size_t gpt2_pkv_attn_ws(const GPT2PagedKV *c, int nRows) {
    if (!c || nRows < 1 || c->nHead < 1 || c->maxPages < 1) return 16;
    const int n = attn_plan(c, nRows, 16).splits;   // the most that any group has
    return n == 1 ? 16 : (size_t)n * nRows * c->nHead * (PKV_D + 4) * 4;
}

extern "C" void gpt2_pkv_attn(gpt2_half *att, const gpt2_half *qkv, const GPT2PagedKV *c, int L, const int *rows, int nRows,
                              int group, void *ws, size_t wsBytes) {
    if (pkv_refused_batch(c, L, rows, nRows, "gpt2_pkv_attn: bad cache, layer or rows")) return;
    if (nRows == 0) return;
    if (!att || !qkv || !aligned16(att) || !aligned16(qkv)) { arg_fail("gpt2_pkv_attn: null/unaligned"); return; }
    if (group < 1 || group > 16 || c->nSeq % group) { arg_fail("gpt2_pkv_attn: group must be 1 .. 16 and divide nSeq"); return; }
    if (!ws || !aligned16(ws) || wsBytes < gpt2_pkv_attn_ws(c, nRows)) { arg_fail("gpt2_pkv_attn: workspace too small or unaligned"); return; }
    PagedAttn a;
    a.c = *c;
    a.att = att;
    a.qkv = qkv;
    a.rows = rows;
    a.L = L;
    a.nRows = nRows;
    a.group = group;
    const AttnPlan p = attn_plan(c, nRows, group);
    a.splits = p.splits;
    a.per = p.per;
    a.po = (float *)ws;
    a.pml = (float4 *)(a.po + (size_t)a.splits * nRows * c->nHead * PKV_D);
    const bool wide = p.form == ATTN_ONE && p.splits == 1 && p.groups < 256;   // eight waves where that leaves CUs idle
    const auto fn = p.form == ATTN_BLOCK   ? k_pkv_attn_block
                    : p.form == ATTN_ROWS2 ? k_pkv_attn_rows<2>
                    : p.form == ATTN_ROWS1 ? k_pkv_attn_rows<1>
                    : group > 1            ? (wide ? k_pkv_attn_beams<8> : k_pkv_attn_beams<4>)
                    : wide                 ? k_pkv_attn_one<8>
                                           : k_pkv_attn_one<4>;
    hipLaunchKernelGGL(fn, dim3(p.groups, p.splits, p.deep), dim3(wide ? 512 : 256), 0, stream(), a);
    if (a.splits > 1) {
        const bool by_seq = p.form == ATTN_ONE;
        hipLaunchKernelGGL(by_seq ? k_pkv_attn_join<true> : k_pkv_attn_join<false>, dim3(by_seq ? c->nSeq : nRows, cdiv(c->nHead, 4)), dim3(256), 0,
                           stream(), a);
    }
    check_launch("k_pkv_attn");
}

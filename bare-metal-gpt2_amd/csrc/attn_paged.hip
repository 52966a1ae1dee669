// attn_paged.hip -- attention over the paged K/V cache (gpt2_pagedkv.h): rows of a ragged batch, a single new token or
// many a sequence, each over the tokens up to its own.
//
// att = sum_j p_j v_j / sum_j p_j, p_j = 2^(x_j - max x), x_j = (q . k_j) log2(e) / 8, with k_j = s_k q_k a page's codes and
// scale.  One pass with the running maximum and sum; scales stay out of the products (x takes s_k, the page's P.V takes s_v).
//
// A wave takes a page at a time against 16 rows.  Scores on v_mfma_f32_16x16x32_f16 with the keys as the A operand: lane l =
// 16 g + jq names key 8 (jq / 4) + 4 t + jq % 4 of tile t, so that it receives the scores of keys 8 g .. + 7 of row jq, which
// is what the B operand of P.V holds in k-slots 8 g .. + 7; the dims are dealt so that a lane's 16 are contiguous in a K
// row (16 g .. + 15), and the V tile's order is that of the A operand of V^T (8 tokens of a dim together).  Codes go from memory to registers 16
// bytes a lane, 1 KB an instruction, and to fp16 there, exactly: no LDS on the way.
// The single new token of a sequence uses one of the 16 columns; the matrix units are idle otherwise, and the sums across
// lanes that a vector form needs cost more than the empty columns.
#include <cmath>

#include "pagedkv.h"

namespace g2 {

struct PagedAttn {
    GPT2PagedKV c;
    uint16_t *att;
    const uint16_t *qkv;
    const int *rows;
    int L, nRows, splits;
    float *po;      // [splits][nRows][nHead][64] unscaled sums of a split
    float2 *pml;    // [splits][nRows][nHead] their maximum and weight
};

// A page in flight: its K rows and V octets as they lie.
struct PageRaw {
    i32x4 k[2], v[2];
};

// Attention of 16 rows as it accumulates: column jq is a row; o[2 i + b] element r is dim 32 i + 8 g + 2 r + b.
struct AttnAcc {
    float m, l;
    f32x4 o[4];
};

__device__ __forceinline__ void page_load(const int8_t *__restrict__ k, const int8_t *__restrict__ v, PageRaw &R) {
    const int lane = threadIdx.x & 63, jq = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t)
        R.k[t] = *reinterpret_cast<const i32x4 *>(k + (8 * (jq >> 2) + 4 * t + (jq & 3)) * PKV_D + 16 * g);
#pragma unroll
    for (int i = 0; i < 2; ++i) R.v[i] = *reinterpret_cast<const i32x4 *>(v + (g * PKV_D + 32 * i + 2 * jq) * 8);
}

// 32 tokens from `key0` on against the columns: fragments of K (kf[t]: dims 16 g .. + 7 and + 8 .. + 15 of the lane's key
// of tile t) and of V (vf[2 i + b]: tokens 8 g .. + 7 of dim 32 i + 2 jq + b); column jq sees keys below `lim`.
__device__ __forceinline__ void attn_page(AttnAcc &A, const f16x8 (&kf)[2][2], const f16x8 (&vf)[4], const f16x8 (&q)[2], float sk,
                                          float sv, int key0, int lim, bool masked) {
    const int g = (threadIdx.x & 63) >> 4;
    float x[8];
    const float scale = sk * (0.125f * 1.4426950408889634f);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        f32x4 s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][0], q[0], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][1], q[1], s, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[4 * t + r] = s[r] * scale;
    }
    if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (key0 + 8 * g + e >= lim) x[e] = -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
    const float mn = fmaxf(A.m, group_max(mx));
    const float base = mn == -INFINITY ? 0.f : mn;   // a column that sees none of these keys
    const float corr = __builtin_amdgcn_exp2f(A.m - base);
    A.m = mn;
    f16x8 p;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = (f16)__builtin_amdgcn_exp2f(x[e] - base);
    // the weights' sum is that of the fp16 values that the matrix units multiply
    float ps = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) ps = __builtin_amdgcn_fdot2(f16x2{p[e], p[e + 1]}, f16x2{1, 1}, ps, false);
    A.l = fmaf(A.l, corr, ps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 y = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[i], p, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) A.o[i][r] = fmaf(A.o[i][r], corr, y[r] * sv);
    }
}

__device__ __forceinline__ void attn_codes(AttnAcc &A, const PageRaw &R, const f16x8 (&q)[2], float sk, float sv, int key0, int lim,
                                           bool masked) {
    f16x8 kf[2][2], vf[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        kf[t][0] = i8x8_to_f16x8(uint2{(uint32_t)R.k[t][0], (uint32_t)R.k[t][1]});
        kf[t][1] = i8x8_to_f16x8(uint2{(uint32_t)R.k[t][2], (uint32_t)R.k[t][3]});
        vf[2 * t] = i8x8_to_f16x8(uint2{(uint32_t)R.v[t][0], (uint32_t)R.v[t][1]});
        vf[2 * t + 1] = i8x8_to_f16x8(uint2{(uint32_t)R.v[t][2], (uint32_t)R.v[t][3]});
    }
    attn_page(A, kf, vf, q, sk, sv, key0, lim, masked);
}

// The open page: fp16 in the same order; tokens at or past `used` are whatever was there, so their values are cleared.
__device__ __forceinline__ void attn_open(AttnAcc &A, const uint16_t *__restrict__ k, const uint16_t *__restrict__ v, int used,
                                          const f16x8 (&q)[2], int key0, int lim) {
    const int lane = threadIdx.x & 63, jq = lane & 15, g = lane >> 4;
    f16x8 kf[2][2], vf[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint16_t *row = k + (8 * (jq >> 2) + 4 * t + (jq & 3)) * PKV_D + 16 * g;
        kf[t][0] = *reinterpret_cast<const f16x8 *>(row);
        kf[t][1] = *reinterpret_cast<const f16x8 *>(row + 8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        vf[i] = *reinterpret_cast<const f16x8 *>(v + (g * PKV_D + 32 * (i >> 1) + 2 * jq + (i & 1)) * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (8 * g + e >= used) vf[i][e] = (f16)0.f;
    }
    attn_page(A, kf, vf, q, 1.f, 1.f, key0, lim, true);
}

// Rows 16 rb .. + 15 of a sequence, one head, one split of the pages; W waves take the pages in turn and join in LDS.
template <int W>
__device__ __forceinline__ void attn_rows(const PagedAttn &a, const PkvSeq &s, int seq, int h, int rb, int split) {
    __shared__ float lds_m[W][16], lds_l[W][16];
    __shared__ f32x4 lds_o[W][4][64];
    const GPT2PagedKV &c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), jq = lane & 15, g = lane >> 4;
    const int E = c.nHead * PKV_D;
    const int i0 = 16 * rb, i = i0 + jq, first = s.start + i0 + 1, lim = s.start + i + 1;   // keys that rows i0 and i see
    const int end = s.start + min(s.n, i0 + 16), pages = (end + PKV_P - 1) / PKV_P, full = s.len / PKV_P;
    const int per = (pages + a.splits - 1) / a.splits, p0 = min(pages, split * per), p1 = min(pages, p0 + per);
    const uint16_t *qrow = a.qkv + (size_t)(s.row0 + min(i, s.n - 1)) * 3 * E + h * PKV_D + 16 * g;
    const f16x8 q[2] = {*reinterpret_cast<const f16x8 *>(qrow), *reinterpret_cast<const f16x8 *>(qrow + 8)};
    AttnAcc A;
    A.m = -INFINITY;
    A.l = 0.f;
#pragma unroll
    for (int d = 0; d < 4; ++d) A.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int pc = p0 + w; pc < p1; pc += 64 * W) {
        // the wave's next 64 pages: lane l holds the number and the scales of page pc + W l
        const int mine = pc + W * lane;
        int page = mine < min(p1, full) ? c.table[(size_t)seq * c.maxPages + mine] : -1;
        if (!pkv_page_ok(c, page)) page = -1;
        float sk = 0.f, sv = 0.f;
        if (page >= 0) {
            const size_t at = pkv_tile(c, c.nPages, a.L, page, 0, h);
            sk = c.scales[at];
            sv = c.scales[at + c.nHead];
        }
        const int n = min(64, (p1 - pc + W - 1) / W);
        for (int j = 0; j < n; ++j) {
            const int p = pc + W * j, key0 = p * PKV_P, pg = __builtin_amdgcn_readlane(page, j);
            if (p == full) {
                const uint16_t *k = c.open + pkv_tile(c, c.nSeq, a.L, s.slot, 0, h) * PKV_TILE;
                attn_open(A, k, k + (size_t)c.nHead * PKV_TILE, s.len - key0, q, key0, lim);
            } else if (pg >= 0) {
                const int8_t *k = c.codes + pkv_tile(c, c.nPages, a.L, pg, 0, h) * PKV_TILE;
                PageRaw R;
                page_load(k, k + (size_t)c.nHead * PKV_TILE, R);
                attn_codes(A, R, q, lane_f(sk, j), lane_f(sv, j), key0, lim, key0 + PKV_P > first);
            }
        }
    }
    const float l = group_sum(A.l);
    if (g == 0) {
        lds_m[w][jq] = A.m;
        lds_l[w][jq] = l;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) lds_o[w][d][lane] = A.o[d];
    __syncthreads();
    if (w < 2) {   // dims 32 w + 8 g .. + 7 of row i
        float mx = -INFINITY, L = 0.f, f[W];
#pragma unroll
        for (int u = 0; u < W; ++u) mx = lds_l[u][jq] != 0.f ? fmaxf(mx, lds_m[u][jq]) : mx;
#pragma unroll
        for (int u = 0; u < W; ++u) {
            f[u] = lds_l[u][jq] != 0.f ? __builtin_amdgcn_exp2f(lds_m[u][jq] - mx) : 0.f;
            L += lds_l[u][jq] * f[u];
        }
        f32x4 y[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int u = 0; u < W; ++u)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[b][r] = fmaf(lds_o[u][2 * w + b][lane][r], f[u], y[b][r]);
        if (i < s.n) {
            const size_t row = s.row0 + i;
            if (a.splits == 1) {
                const float inv = L != 0.f ? 1.f / L : 0.f;   // no key: 0
                f16x8 o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (f16)(y[e & 1][e >> 1] * inv);
                *reinterpret_cast<f16x8 *>(a.att + row * E + h * PKV_D + 32 * w + 8 * g) = o;
            } else {
                const size_t at = ((size_t)split * a.nRows + row) * c.nHead + h;
                float *o = a.po + at * PKV_D + 32 * w + 8 * g;
                *reinterpret_cast<f32x4 *>(o) = f32x4{y[0][0], y[1][0], y[0][1], y[1][1]};
                *reinterpret_cast<f32x4 *>(o + 4) = f32x4{y[0][2], y[1][2], y[0][3], y[1][3]};
                if (w == 0 && g == 0) a.pml[at] = float2{mx, L};
            }
        }
    }
}

// BY_SEQ: a work-group takes all row blocks of a sequence (no more rows than sequences: nearly always one block).
template <int W, bool BY_SEQ>
__global__ __launch_bounds__(64 * W) void k_pkv_attn(PagedAttn a) {
    const int h = blockIdx.x % a.c.nHead, split = blockIdx.y;
    int rb = blockIdx.x / a.c.nHead;
    if constexpr (BY_SEQ) {
        const int seq = rb;
        const PkvSeq s = pkv_seq(a.c, a.rows, a.nRows, seq);
        for (rb = 0; 16 * rb < s.n; ++rb) {
            if (rb) __syncthreads();
            attn_rows<W>(a, s, seq, h, rb, split);
        }
    } else {
        const int seq = pkv_seq_of_unit(rb, a.c.nSeq, [&](int s) { return (pkv_seq(a.c, a.rows, a.nRows, s).n + 15) / 16; });
        if (seq < 0) return;
        attn_rows<W>(a, pkv_seq(a.c, a.rows, a.nRows, seq), seq, h, rb, split);
    }
}

// Joins the splits: a wave per row and head, a lane per dim.
__global__ __launch_bounds__(256) void k_pkv_attn_join(PagedAttn a) {
    const int lane = threadIdx.x & 63, h = blockIdx.y * 4 + (threadIdx.x >> 6), row = blockIdx.x;
    if (h >= a.c.nHead) return;
    const int seq = pkv_seq_of_row(a.rows, a.c.nSeq, row);
    if (seq < 0 || pkv_seq(a.c, a.rows, a.nRows, seq).n == 0) return;
    float mx = -INFINITY, L = 0.f, o = 0.f;
    for (int z = 0; z < a.splits; ++z) {
        const float2 ml = a.pml[((size_t)z * a.nRows + row) * a.c.nHead + h];
        if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
    }
    for (int z = 0; z < a.splits; ++z) {
        const size_t at = ((size_t)z * a.nRows + row) * a.c.nHead + h;
        const float2 ml = a.pml[at];
        if (ml.y == 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(ml.x - mx);
        L = fmaf(ml.y, f, L);
        o = fmaf(a.po[at * PKV_D + lane], f, o);
    }
    a.att[(size_t)row * a.c.nHead * PKV_D + h * PKV_D + lane] = f2h(L != 0.f ? o / L : 0.f);
}

// Work-groups of one split, and into how many splits the pages go.
static long attn_groups(const GPT2PagedKV *c, int nRows) {
    return (long)(nRows <= c->nSeq ? c->nSeq : nRows / 16 + c->nSeq) * c->nHead;
}
static int attn_splits(const GPT2PagedKV *c, int nRows) {
    const long groups = attn_groups(c, nRows);
    int n = (int)((1024 + groups - 1) / groups);
    const int most = cdiv(c->maxPages, 16);
    if (n > most) n = most;
    return n < 1 ? 1 : n > 32 ? 32 : n;
}

}  // namespace g2

using namespace g2;

extern "C" size_t gpt2_pkv_attn_ws(const GPT2PagedKV *c, int nRows) {
    if (!c || nRows < 1 || c->nSeq < 1 || c->nHead < 1 || c->maxPages < 1) return 16;
    const int n = attn_splits(c, nRows);
    return n == 1 ? 16 : (size_t)n * nRows * c->nHead * (PKV_D + 2) * 4;
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
    a.splits = attn_splits(c, nRows);
    a.po = (float *)ws;
    a.pml = (float2 *)(a.po + (size_t)a.splits * nRows * c->nHead * PKV_D);
    const dim3 grid((unsigned)attn_groups(c, nRows), a.splits);
    const auto fn = nRows <= c->nSeq ? k_pkv_attn<4, true> : k_pkv_attn<4, false>;
    hipLaunchKernelGGL(fn, grid, dim3(256), 0, stream(), a);
    if (a.splits > 1) hipLaunchKernelGGL(k_pkv_attn_join, dim3(nRows, cdiv(c->nHead, 4)), dim3(256), 0, stream(), a);
    check_launch("k_pkv_attn");
}

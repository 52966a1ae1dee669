// beam.hip -- beam search's selection (gpt2_pagedkv.h): of each group's beams x V continuations, the best `beams` by
// score + log_softmax.
//
// score_b + x - m_b - log(sum_b) orders a row's tokens as its logits do, so a row's candidates are its best `beams` logits:
// one pass over the logits takes each part of a row's maximum, its sum of exponentials and its best, and a second launch, a
// work-group a group, joins the parts and merges the rows' lists of candidates in fp64.  64 groups of
// 8 rows of 50257 take 18.7 us (2.8 TB/s) and 5.4; 512 groups of one row, which need no bounds, 14.0: instructions, some 14 a pair of
// logits and the bounds and sums of every wave, take longer than the reading (10 us).  Four rows take 5.2 and 3.8, the latency of
// two short launches.  (Launches under the tracer, medians over two sets of inputs in turn.)
//
// A logit and its token are one 32-bit key, (logit's bits in order) << 16 | (65535 - token): keys of a row are unique, and
// the larger key is the larger logit or, of equal ones, the lower token.  0 is no key.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "gpt2_pagedkv.h"

namespace g2 {

// Pieces of eight logits a thread, 8192 a work-group.  Half as many are slower where there are many rows (512 rows of 50257: 21.3
// us and 6.0 to join for 18.7 and 5.4; four rows 4.6 and 4.0 for 5.2 and 3.8), twice as many too (20.0; 6.2).
constexpr int BEAM_PIECES = 4;
constexpr int BEAM_PARTS = GPT2_BEAM_MAX_VOCAB / 8 / (256 * BEAM_PIECES);
struct BeamPart {
    double sum;                                         // of exp(x - m)
    float m;
    uint32_t key[GPT2_BEAM_MAX];                        // the best, in order
};
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef int i32x4_dword __attribute__((ext_vector_type(4), aligned(4)));   // at any dword

// Maximum over the wave, the same scalar for all: rows of 16 lanes by DPP, then the four rows.
__device__ __forceinline__ uint32_t wave_max_key(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));
    const uint32_t a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16), c = __builtin_amdgcn_readlane((int)v, 32),
                   d = __builtin_amdgcn_readlane((int)v, 48);
    return max(max(a, b), max(c, d));
}

// Sum over the wave in fp64, in a fixed order: rows of 16 lanes by DPP, then the four rows.
__device__ __forceinline__ double wave_sum64(double v) {
    auto add = [&](auto ctrl) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, ctrl.value, 0xF, 0xF, true);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), ctrl.value, 0xF, 0xF, true);
        v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    add(std::integral_constant<int, 0xB1>{});
    add(std::integral_constant<int, 0x4E>{});
    add(std::integral_constant<int, 0x141>{});
    add(std::integral_constant<int, 0x140>{});
    auto row = [&](int l) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
        return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    return (row(0) + row(16)) + (row(32) + row(48));
}

// Two logits as they count: NaN as -inf, +inf as 65504, -0 as +0; and their bits in order.
__device__ __forceinline__ f16x2 beam_logits(f16x2 x) {
    x = x + f16x2{(f16)0.f, (f16)0.f};
    x = __builtin_elementwise_max(x, f16x2{(f16)-INFINITY, (f16)-INFINITY});
    return __builtin_elementwise_min(x, f16x2{(f16)65504.f, (f16)65504.f});
}
__device__ __forceinline__ uint32_t beam_order(f16x2 x) {
    const i16x2 b = __builtin_bit_cast(i16x2, x);
    return __builtin_bit_cast(uint32_t, b ^ ((b >> 15) | (short)0x8000));
}
__device__ __forceinline__ float beam_key_logit(uint32_t key) {
    const uint32_t o = key >> 16;
    return h2f((uint16_t)(o & 0x8000u ? o & 0x7fffu : ~o));
}

// One part of a row: its pieces of eight [256 NV part, ...), the first part also the logits after the last whole piece.
// A row's logits go to threads and sums by their number, wherever the row begins: equal rows have equal sums, so that
// equal scores tie.  So a piece is loaded as dwords, from the one that has its first logit, and where that is a dword's upper half with
// the one past them.
//
// A thread's logits stay in registers as keys of their own, order << 16 | (63 - i) for its i-th; the tokens of a thread
// ascend with i, so its largest is its best.  A key that `beams` threads of a wave reach is a lower bound for the part's result;
// the highest such is found bit by bit, a comparison and a count each, until just `beams` reach it.  The keys at or above the
// waves' best bound (those of 4 beams threads at most) are ranked by counting.
__global__ __launch_bounds__(256) void k_beam_part(BeamPart *__restrict__ out, const uint16_t *__restrict__ logits, long ld, int V,
                                                   int beams, int parts) {
    constexpr int NV = BEAM_PIECES, N = 8 * NV;
    static_assert(N <= 64, "a thread's keys hold its index in 6 bits");
    __shared__ float lds_m[4];
    __shared__ double lds_s[4];
    __shared__ uint32_t lds_t[4], lds_k[4 * GPT2_BEAM_MAX * (N + 1)];
    __shared__ int lds_n;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, part = blockIdx.x;
    const uint16_t *x = logits + (size_t)blockIdx.y * ld;
    const int pieces = V >> 3, first = part * 256 * NV + tid, left = V & 7, odd = 8 * pieces + tid;
    const bool upper = (uintptr_t)x & 2;   // the same for the whole row
    if (tid == 0) lds_n = 0;
    f16x2 v[N / 2], vodd;
    uint32_t key[N], kodd;
    const int *dwords = reinterpret_cast<const int *>(x - upper);
    i32x4 h[NV];
    int next[NV] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        h[j] = i32x4{(int)0xfc00fc00, (int)0xfc00fc00, (int)0xfc00fc00, (int)0xfc00fc00};
        if (first + 256 * j < pieces) {
            h[j] = *reinterpret_cast<const i32x4_dword *>(dwords + 4 * (first + 256 * j));
            if (upper) next[j] = dwords[4 * (first + 256 * j) + 4];
        }
    }
    const bool has_odd = part == 0 && tid < left;
    uint16_t rest = 0xfc00;
    if (has_odd) rest = x[odd];
    if (upper)
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (first + 256 * j < pieces)
#pragma unroll
                for (int d = 0; d < 4; ++d) h[j][d] = (int)__builtin_amdgcn_alignbit((uint32_t)(d < 3 ? h[j][d + 1] : next[j]), (uint32_t)h[j][d], 16);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = __builtin_bit_cast(f16x2, (int)h[i / 4][i % 4]);
    vodd = f16x2{__builtin_bit_cast(f16, rest), (f16)-INFINITY};
    uint32_t best = 0, piece[NV] = {};   // the largest of a piece
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        v[i] = beam_logits(v[i]);
        const uint32_t o = beam_order(v[i]);
        key[2 * i] = __builtin_amdgcn_perm(o, (uint32_t)(63 - 2 * i), 0x05040100u);       // o << 16 | ..
        key[2 * i + 1] = __builtin_amdgcn_perm(o, (uint32_t)(62 - 2 * i), 0x07060100u);   // o's upper half | ..
        piece[i / 4] = max(piece[i / 4], max(key[2 * i], key[2 * i + 1]));
    }
    if (256 * NV * (part + 1) > pieces) {   // the last part: pieces that are none have no keys
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = first + 256 * (i / 8) < pieces ? key[i] : 0u;
#pragma unroll
        for (int j = 0; j < NV; ++j) piece[j] = first + 256 * j < pieces ? piece[j] : 0u;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) best = max(best, piece[j]);
    vodd = beam_logits(vodd);
    const int token0 = 8 * first;
    auto token = [&](uint32_t k) {   // of one of the thread's own keys
        const int i = 63 - (int)(k & 63u);
        return token0 + 2048 * (i >> 3) + (i & 7);
    };
    best = best >> 16 ? (best & 0xffff0000u) | (uint32_t)(65535 - token(best)) : 0u;
    kodd = has_odd ? beam_order(vodd) << 16 | (uint32_t)(65535 - odd) : 0u;
    best = max(best, kodd);

    // the wave's maximum, and the bound
    const uint32_t top = wave_max_key(best);
    const float m = top ? beam_key_logit(top) : -INFINITY;
    uint32_t bound = 0u;
    if (beams <= 4) {   // maximum after maximum is quicker for few (4 rows, 4 beams: 5.2 us, 5.5)
        bound = top;
        uint32_t rest = best;
        for (int k = 1; k < beams; ++k) {
            rest = rest == bound ? 0u : rest;
            bound = wave_max_key(rest);
        }
    } else
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            const int n = __popcll(__ballot(best >= (bound | bit)));
            if (n >= beams) bound |= bit;
            if (n == beams) break;
        }
    // exp(x - m) as 2^(x l - c), l = log2 e in fp32, c = m l rounded; what the rounding takes is put back in fp64
    constexpr float l2e = 1.4426950408889634f;
    const float c = m == -INFINITY ? 0.f : m * l2e;
    float s32 = 0.f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        s32 += __builtin_amdgcn_exp2f(fmaf((float)v[i][0], l2e, -c));
        s32 += __builtin_amdgcn_exp2f(fmaf((float)v[i][1], l2e, -c));
    }
    s32 += __builtin_amdgcn_exp2f(fmaf((float)vodd[0], l2e, -c));
    const double sum = wave_sum64((double)s32);   // 33 terms at most in fp32, the rest in fp64
    if (lane == 0) {
        lds_t[w] = bound;
        lds_m[w] = m;
        const double e = 0.6931471805599453 * ((double)c - (double)m * (double)l2e);   // 0.003 at most
        lds_s[w] = m == -INFINITY ? 0.0 : sum * (1.0 + e * (1.0 + 0.5 * e));
    }
    __syncthreads();
    bound = max(max(lds_t[0], lds_t[1]), max(lds_t[2], lds_t[3]));
    if (__ballot(best >= bound)) {   // wave-uniform; a bound of 0: every key is wanted
        // the thread's keys with the bound's order count up to the bound's token
        const int d = 65535 - (int)(bound & 0xffffu) - token0, n = d < 0 ? 0 : min(N, 8 * (d >> 11) + min((d & 2047) + 1, 8));
        const uint32_t own = bound ? (bound & 0xffff0000u) + (uint32_t)(64 - n) : 0x10000u;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (__ballot(piece[j] >= own))
#pragma unroll
                for (int i = 8 * j; i < 8 * j + 8; ++i)
                    if (key[i] >= own) lds_k[atomicAdd(&lds_n, 1)] = (key[i] & 0xffff0000u) | (uint32_t)(65535 - token(key[i]));
        if (kodd && kodd >= bound) lds_k[atomicAdd(&lds_n, 1)] = kodd;
    }
    __syncthreads();
    const int n = lds_n;
    BeamPart *o = out + (size_t)blockIdx.y * parts + part;
    if (tid < beams && tid >= n) o->key[tid] = 0u;
    for (int i = tid; i < n; i += 256) {
        const uint32_t mine = lds_k[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += lds_k[j] > mine;
        if (rank < beams) o->key[rank] = mine;
    }
    if (w == 0) {   // lane i: wave i's sum, to the largest maximum
        const float mi = lds_m[lane & 3], mx = fmaxf(fmaxf(lds_m[0], lds_m[1]), fmaxf(lds_m[2], lds_m[3]));
        const double term = mi == -INFINITY ? 0.0 : mi == mx ? lds_s[lane & 3] : lds_s[lane & 3] * exp((double)mi - (double)mx);
        const double all = (__shfl(term, 0, 64) + __shfl(term, 1, 64)) + (__shfl(term, 2, 64) + __shfl(term, 3, 64));
        if (lane == 0) {
            o->m = mx;
            o->sum = all;
        }
    }
}

// A work-group per group, a wave per row: the row's parts are joined, then one wave merges the rows' candidates.
__global__ __launch_bounds__(64 * GPT2_BEAM_MAX) void k_beam_join(int *__restrict__ token, int *__restrict__ parent, float *score_out, int *done_out,
                                                                  const BeamPart *__restrict__ part, const float *score, const int *done,
                                                                  int beams, int V, int eos, int parts) {
    constexpr int K = BEAM_PARTS / 4;   // a lane's keys, four parts each
    __shared__ double cand[GPT2_BEAM_MAX * GPT2_BEAM_MAX];
    __shared__ int tok[GPT2_BEAM_MAX * GPT2_BEAM_MAX];   // beam b's at b * beams
    const int tid = threadIdx.x, lane = tid & 63, b = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x * beams + b;
    const BeamPart *p = part + (size_t)row * parts;
    const double from = (double)score[row];
    const bool ended = eos >= 0 && done[row];
    static_assert(GPT2_BEAM_MAX == 16 && BEAM_PARTS <= 8, "16 places a part, a part a lane, two keys a lane");
    uint32_t key[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int at = 4 * i + (lane >> 4);
        key[i] = at < parts && (lane & 15) < beams ? p[at].key[lane & 15] : 0u;
    }
    const float mp = lane < parts ? p[lane].m : -INFINITY;
    const double sp = lane < parts ? p[lane].sum : 0.0;
    const float m = wave_max_u(mp);
    const double term = mp == -INFINITY ? 0.0 : mp == m ? sp : sp * exp((double)mp - (double)m);
    double sum = 0.0;
    for (int i = 0; i < parts; ++i) sum += __shfl(term, i, 64);
    const double lse = log(sum);
    uint32_t mine = 0;   // lane k: the row's k-th best
    for (int k = 0; k < beams; ++k) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < K; ++i) best = max(best, key[i]);
        const uint32_t top = wave_max_key(best);
        if (lane == k) mine = top;
#pragma unroll
        for (int i = 0; i < K; ++i) key[i] = key[i] == top ? 0u : key[i];
    }
    if (lane < beams) {
        double s = ended ? from : from + ((double)beam_key_logit(mine) - (double)m) - lse;
        if (s != s) s = -INFINITY;
        const bool there = ended ? lane == 0 : mine != 0;
        cand[b * beams + lane] = there ? s : (double)NAN;   // NaN: not there
        tok[b * beams + lane] = ended ? eos : 65535 - (int)(mine & 0xffffu);
    }
    __syncthreads();
    if (b) return;
    // the rows' lists, each in order, merged: lane r has row r's next candidate
    int at = min(lane, beams - 1) * beams, my_row = 0, my_at = 0;
    const int last = at + beams - 1;
    double next = lane < beams ? cand[at] : (double)NAN;
    for (int k = 0; k < beams; ++k) {
        double best = next;   // NaN gives way to numbers, and a number is left: every row has a candidate
        auto step = [&](auto ctrl) {
            const uint64_t v = __builtin_bit_cast(uint64_t, best);
            const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, ctrl.value, 0xF, 0xF, true);
            const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), ctrl.value, 0xF, 0xF, true);
            best = fmax(best, __builtin_bit_cast(double, (uint64_t)hi << 32 | lo));
        };
        step(std::integral_constant<int, 0xB1>{});
        step(std::integral_constant<int, 0x4E>{});
        step(std::integral_constant<int, 0x141>{});
        step(std::integral_constant<int, 0x140>{});
        const int r = __builtin_ctzll(__ballot(next == best) | 1ull << 63);   // of equal scores the lower row
        const int from = __builtin_amdgcn_readlane(at, r);
        if (lane == k) {
            my_row = r;
            my_at = from;
        }
        if (lane == r) {
            next = at < last ? cand[at + 1] : (double)NAN;
            ++at;
        }
    }
    if (lane < beams) {
        const int o = blockIdx.x * beams + lane, t = tok[my_at];
        token[o] = t;
        parent[o] = blockIdx.x * beams + my_row;
        score_out[o] = (float)cand[my_at];
        done_out[o] = eos >= 0 && t == eos;
    }
}

static int beam_parts(int V) { return V < 8 ? 1 : cdiv(V / 8, 256 * BEAM_PIECES); }

}  // namespace g2

using namespace g2;

extern "C" size_t gpt2_beam_select_ws(int groups, int beams, int V) {
    if (groups < 1 || beams < 1 || V < 1 || (long)groups * beams > 65535) return 16;
    return (size_t)groups * beams * beam_parts(V) * sizeof(BeamPart);
}

extern "C" void gpt2_beam_select(int *token, int *parent, float *score_out, int *done_out, const gpt2_half *logits, long ld,
                                 const float *score, const int *done, int groups, int beams, int V, int eos, void *ws, size_t wsBytes) {
    if (groups == 0) return;
    if (groups < 0 || beams < 1 || beams > GPT2_BEAM_MAX || (long)groups * beams > 65535 || V < 1 || V > GPT2_BEAM_MAX_VOCAB || ld < V || eos >= V) {
        arg_fail("gpt2_beam_select: sizes out of range");
        return;
    }
    if (!token || !parent || !score_out || !done_out || !logits || !score || (eos >= 0 && !done) || ((uintptr_t)logits & 1)) {
        arg_fail("gpt2_beam_select: null/unaligned");
        return;
    }
    if (!ws || !aligned16(ws) || wsBytes < gpt2_beam_select_ws(groups, beams, V)) {
        arg_fail("gpt2_beam_select: workspace too small or unaligned");
        return;
    }
    const int rows = groups * beams, parts = beam_parts(V);
    BeamPart *part = (BeamPart *)ws;
    hipLaunchKernelGGL(k_beam_part, dim3(parts, rows), dim3(256), 0, stream(), part, logits, ld, V, beams, parts);
    hipLaunchKernelGGL(k_beam_join, dim3(groups), dim3(64 * beams), 0, stream(), token, parent, score_out, done_out, part, score, done,
                       beams, V, eos, parts);
    check_launch("k_beam_select");
}

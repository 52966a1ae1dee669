// beam.hip -- beam search's selection (gpt2_pagedkv.h): of each group's beams x V continuations, the best `beams` by
// score + log_softmax.
//
// score_b + x - m_b - log(sum_b) orders a row's tokens as its logits do, so a row's candidates are its best `beams` logits:
// one pass over the logits takes each part of a row's maximum, its sum of exponentials and its best, and a second launch, a
// work-group a group, joins the parts and ranks the beams x beams candidates in fp64.  Bound by reading the logits once.
//
// A logit and its token are one 32-bit key, (logit's bits in order) << 16 | (65535 - token): keys of a row are unique, and
// the larger key is the larger logit or, of equal ones, the lower token.  0 is no key.
#include <cmath>

#include "common.h"
#include "gpt2_pagedkv.h"

namespace g2 {

constexpr int BEAM_NV = 4;                              // 16-byte pieces a thread
constexpr int BEAM_PART = 256 * BEAM_NV;                // pieces a work-group: 8192 logits
struct BeamPart {
    double sum;                                         // of exp(x - m)
    float m;
    uint32_t key[GPT2_BEAM_MAX];
};

__device__ __forceinline__ uint32_t wave_max_key(uint32_t v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// NaN counts as -inf, +inf as 65504, -0 as +0.
__device__ __forceinline__ f16 beam_logit(f16 x) {
    const float f = (float)x + 0.f;
    return f != f ? (f16)-INFINITY : (f16)fminf(f, 65504.f);
}
__device__ __forceinline__ uint32_t beam_key(f16 x, int token) {
    const uint32_t b = __builtin_bit_cast(uint16_t, x);
    const uint32_t o = b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
    return o << 16 | (uint32_t)(65535 - token);
}
__device__ __forceinline__ float beam_key_logit(uint32_t key) {
    const uint32_t o = key >> 16;
    return h2f((uint16_t)(o & 0x8000u ? o & 0x7fffu : ~o));
}

// One part of a row: its 16-byte pieces [part * BEAM_PART, ...), the first part also the logits before the first whole
// piece and after the last.
__global__ __launch_bounds__(256) void k_beam_part(BeamPart *__restrict__ out, const uint16_t *__restrict__ logits, long ld, int V,
                                                   int beams, int parts) {
    __shared__ float lds_m[4];
    __shared__ double lds_s[4];
    __shared__ uint32_t lds_k[4 * GPT2_BEAM_MAX];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, part = blockIdx.x;
    const uint16_t *x = logits + (size_t)blockIdx.y * ld;
    const int head = min(V, (int)(((16 - ((uintptr_t)x & 15)) & 15) >> 1)), pieces = (V - head) >> 3;
    f16 v[BEAM_NV * 8 + 1];
    uint32_t key[BEAM_NV * 8 + 1];
#pragma unroll
    for (int j = 0; j < BEAM_NV; ++j) {
        const int p = part * BEAM_PART + j * 256 + tid;
        f16x8 h = {};
        if (p < pieces) h = *reinterpret_cast<const f16x8 *>(x + head + 8 * p);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[8 * j + e] = p < pieces ? beam_logit(h[e]) : (f16)-INFINITY;
            key[8 * j + e] = p < pieces ? beam_key(v[8 * j + e], head + 8 * p + e) : 0u;
        }
    }
    {
        const int left = V - 8 * pieces, t = tid < head ? tid : 8 * pieces + tid;
        const bool on = part == 0 && tid < left;
        v[8 * BEAM_NV] = on ? beam_logit(__builtin_bit_cast(f16, x[t])) : (f16)-INFINITY;
        key[8 * BEAM_NV] = on ? beam_key(v[8 * BEAM_NV], t) : 0u;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i <= 8 * BEAM_NV; ++i) m = fmaxf(m, (float)v[i]);
    m = wave_max_u(m);
    if (lane == 0) lds_m[w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(lds_m[0], lds_m[1]), fmaxf(lds_m[2], lds_m[3]));
    const float base = m == -INFINITY ? 0.f : m;
    float s32 = 0.f;
#pragma unroll
    for (int i = 0; i <= 8 * BEAM_NV; ++i) s32 += __builtin_amdgcn_exp2f(((float)v[i] - base) * 1.4426950408889634f);
    double sum = s32;   // at most 33 terms in fp32, the rest in fp64
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) lds_s[w] = sum;
    // the wave's best keys
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i <= 8 * BEAM_NV; ++i) best = max(best, key[i]);
    for (int k = 0; k < beams; ++k) {
        const uint32_t top = wave_max_key(best);
        if (lane == 0) lds_k[w * GPT2_BEAM_MAX + k] = top;
        if (best == top) {
            best = 0;
#pragma unroll
            for (int i = 0; i <= 8 * BEAM_NV; ++i) best = key[i] < top ? max(best, key[i]) : best;
        }
    }
    __syncthreads();
    if (w == 0) {   // of the four waves': a lane's key has the rank of how many are larger
        BeamPart *o = out + (size_t)blockIdx.y * parts + part;
        const uint32_t mine = (lane & 15) < beams ? lds_k[lane] : 0u;
        int rank = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
            const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
            rank += other > mine || (other == mine && i < lane);
        }
        if (rank < beams) o->key[rank] = mine;
        if (lane == 0) {
            o->m = m;
            o->sum = (lds_s[0] + lds_s[1]) + (lds_s[2] + lds_s[3]);
        }
    }
}

// A work-group per group: a wave joins a row's parts, then a thread per candidate counts those ahead of it.
__global__ __launch_bounds__(256) void k_beam_join(int *__restrict__ token, int *__restrict__ parent, float *score_out, int *done_out,
                                                   const BeamPart *__restrict__ part, const float *score, const int *done, int beams,
                                                   int V, int eos, int parts) {
    __shared__ double cand[GPT2_BEAM_MAX * GPT2_BEAM_MAX];
    __shared__ int tok[GPT2_BEAM_MAX * GPT2_BEAM_MAX];   // -1: no candidate
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int row0 = blockIdx.x * beams;
    for (int i = tid; i < GPT2_BEAM_MAX * GPT2_BEAM_MAX; i += 256) tok[i] = -1;
    __syncthreads();
    for (int b = w; b < beams; b += 4) {
        const BeamPart *p = part + (size_t)(row0 + b) * parts;
        const double from = (double)score[row0 + b];
        if (eos >= 0 && done[row0 + b]) {
            if (lane == 0) {
                tok[b * GPT2_BEAM_MAX] = eos;
                cand[b * GPT2_BEAM_MAX] = from != from ? -INFINITY : from;
            }
            continue;
        }
        float m = -INFINITY;
        for (int i = 0; i < parts; ++i) m = fmaxf(m, p[i].m);
        double sum = 0.0;
        for (int i = 0; i < parts; ++i) sum += p[i].m == -INFINITY ? 0.0 : p[i].sum * exp((double)p[i].m - (double)m);
        const double lse = log(sum);
        // the best of the parts' keys, a part's own in order: 16 parts at most a lane's share is 4 keys
        const int n = parts * beams;
        for (int k = lane; k < n; k += 64) {
            const uint32_t mine = p[k / beams].key[k % beams];
            if (!mine) continue;
            int rank = 0;
            for (int i = 0; i < n; ++i) rank += p[i / beams].key[i % beams] > mine;
            if (rank < beams) {
                const double s = from + ((double)beam_key_logit(mine) - (double)m) - lse;
                tok[b * GPT2_BEAM_MAX + rank] = 65535 - (int)(mine & 0xffffu);
                cand[b * GPT2_BEAM_MAX + rank] = s != s ? -INFINITY : s;
            }
        }
    }
    __syncthreads();
    const int b = tid / GPT2_BEAM_MAX;
    if (tok[tid] < 0) return;
    const double mine = cand[tid];
    int rank = 0;
    for (int i = 0; i < beams * GPT2_BEAM_MAX; ++i)
        if (tok[i] >= 0) rank += cand[i] > mine || (cand[i] == mine && i < tid);
    if (rank < beams) {
        token[row0 + rank] = tok[tid];
        parent[row0 + rank] = row0 + b;
        score_out[row0 + rank] = (float)mine;
        done_out[row0 + rank] = eos >= 0 && tok[tid] == eos;
    }
}

static int beam_parts(int V) { return V < 8 ? 1 : cdiv(V / 8, BEAM_PART); }

}  // namespace g2

using namespace g2;

extern "C" size_t gpt2_beam_select_ws(int groups, int beams, int V) {
    if (groups < 1 || beams < 1 || V < 1) return 16;
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
    const int parts = beam_parts(V);
    BeamPart *part = (BeamPart *)ws;
    hipLaunchKernelGGL(k_beam_part, dim3(parts, groups * beams), dim3(256), 0, stream(), part, logits, ld, V, beams, parts);
    hipLaunchKernelGGL(k_beam_join, dim3(groups), dim3(256), 0, stream(), token, parent, score_out, done_out, part, score, done,
                       beams, V, eos, parts);
    check_launch("k_beam_select");
}

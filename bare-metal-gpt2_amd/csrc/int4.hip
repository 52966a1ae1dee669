// int4.hip -- weights of 4 bits with group scales (gpt2_int4.h): the quantiser, its inverse and the products.
#include <cstring>
#include <type_traits>

#include "common.h"
#include "gpt2_int4.h"

namespace g2 {

constexpr int Q4_N = 16, Q4_K = 128, Q4_TILE = 1024;   // a tile: outputs, inputs, bytes of codes

// The weights as a kernel has them.  per = 128 / group: scales of an output in a tile.
struct Q4 {
    const uint32_t *codes;
    const uint16_t *scales;
    int N, K, kb;   // kb: tiles along k
};

// Where octet o (eight consecutive k) of output n lies in a tile, in words.
__device__ __forceinline__ int q4_word(int n, int o) { return ((o & 3) * 16 + n) * 4 + (o >> 2); }

// Eight codes as exact fp16 values, in order: a code under the exponent of 1024 is 1024 + u, or with its four bits one place
// of four higher 1024 + 16 u; u = q + 8.
__device__ __forceinline__ f16x8 q4_values(uint32_t w) {
    const f16x2 lo_off = {(f16)-1032.f, (f16)-1032.f}, sixteenth = {(f16)0.0625f, (f16)0.0625f}, hi_off = {(f16)-72.f, (f16)-72.f};
    f16x2 v[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t x = w >> (8 * h);
        v[2 * h] = __builtin_bit_cast(f16x2, (x & 0x000f000fu) | 0x64006400u) + lo_off;
        v[2 * h + 1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (x & 0x00f000f0u) | 0x64006400u), sixteenth, hi_off);
    }
    return f16x8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}

// Eight consecutive halves of a row of K from k on, 0 past its end.
template <bool VEC>
__device__ __forceinline__ f16x8 q4_octet(const uint16_t *row, int k, int K) {
    f16x8 v = {};
    if constexpr (VEC) {
        if (k < K) v = *reinterpret_cast<const f16x8 *>(row + k);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) v[e] = __builtin_bit_cast(f16, row[k + e]);
    }
    return v;
}

// A work-group a tile, a thread an octet: sixteen consecutive lanes have an output's 128 k, so a group's largest value is a maximum
// over 4, 8 or 16 lanes by DPP.
template <int G, bool VEC>
__global__ __launch_bounds__(256) void k_quantize_int4(uint32_t *__restrict__ codes, uint16_t *__restrict__ scales, const uint16_t *__restrict__ src, int N,
                                                       int K, int kb) {
    constexpr int PER = Q4_K / G;
    const int tid = threadIdx.x, n = tid >> 4, o = tid & 15, tk = blockIdx.x % kb, tn = blockIdx.x / kb;
    const int row = tn * Q4_N + n, k = tk * Q4_K + 8 * o;
    f16x8 h = {};
    if (row < N) h = q4_octet<VEC>(src + (size_t)row * K, k, K);
    float x[8], peak = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = (float)h[e];
        x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -65504.f), 65504.f) : 0.f;
        peak = fmaxf(peak, fabsf(x[e]));
    }
    auto over = [&](auto f) { peak = fmaxf(peak, __int_as_float(f(__float_as_int(peak)))); };
    over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true); });
    over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true); });
    if constexpr (G >= 64) over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true); });
    if constexpr (G >= 128) over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true); });
    const f16 s16 = (f16)(peak / 7.0f);
    const float s = (float)s16 == 0.f ? 1.f : (float)s16;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int q = (int)fminf(fmaxf(rintf(x[e] / s), -7.f), 7.f);
        w |= (uint32_t)(q + 8) << (4 * (e >> 1) + 16 * (e & 1));
    }
    const size_t tile = (size_t)tn * kb + tk;
    codes[tile * (Q4_TILE / 4) + q4_word(n, o)] = w;
    if (o % (G / 8) == 0) scales[tile * (16 * PER) + ((n >> 2) * PER + o / (G / 8)) * 4 + (n & 3)] = f2h(s);
}

template <int G, bool VEC>
__global__ __launch_bounds__(256) void k_dequantize_int4(uint16_t *__restrict__ dst, const uint32_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                                         int N, int K, int kb) {
    constexpr int PER = Q4_K / G;
    const int tid = threadIdx.x, n = tid >> 4, o = tid & 15, tk = blockIdx.x % kb, tn = blockIdx.x / kb;
    const int row = tn * Q4_N + n, k = tk * Q4_K + 8 * o;
    if (row >= N || k >= K) return;
    const size_t tile = (size_t)tn * kb + tk;
    const f16x8 q = q4_values(codes[tile * (Q4_TILE / 4) + q4_word(n, o)]);
    const float s = h2f(scales[tile * (16 * PER) + ((n >> 2) * PER + o / (G / 8)) * 4 + (n & 3)]);
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (f16)((float)q[e] * s);
    uint16_t *to = dst + (size_t)row * K + k;
    if constexpr (VEC) *reinterpret_cast<f16x8 *>(to) = v;
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) to[e] = f2h((float)q[e] * s);
}

// What follows the sums, in fp32: gelu_new as v / (1 + 2^(K (v + 0.044715 v^3))), K = -2 sqrt(2 / pi) log2(e); or the residual.
__device__ __forceinline__ uint16_t q4_out(float v, int epi, const uint16_t *resid, size_t at) {
    if (epi == GPT2_EPI_GELU) {
        constexpr float K = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
        v = v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(K * __builtin_fmaf(0.044715f, v * v * v, v)));
    } else if (epi == GPT2_EPI_ADD) v = h2f(resid[at]) + v;
    return f2h(v);
}

// Any sizes and alignments: a wave 16 outputs of 16 rows.  On the matrix units the codes are the A operand (lane l: output l % 16,
// the octet l / 16 of 32 k) and the rows the B operand, so a lane ends with outputs 4 (l / 16) .. + 3 of row l % 16.  A group's products are
// summed from 0 and then added times its scale.
template <int G, bool VEC>
__global__ __launch_bounds__(256) void k_int4_any(uint16_t *C, const uint16_t *__restrict__ A, Q4 w, const uint16_t *__restrict__ bias, int M, int epi,
                                                  const uint16_t *resid) {
    constexpr int PER = Q4_K / G;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int tn = blockIdx.x, m = (blockIdx.y * 4 + (threadIdx.x >> 6)) * 16 + l16;
    const uint16_t *row = A + (size_t)min(m, M - 1) * w.K;
    f32x4 acc = {};
    for (int tk = 0; tk < w.kb; ++tk) {
        const size_t tile = (size_t)tn * w.kb + tk;
        const i32x4 c = *reinterpret_cast<const i32x4 *>(w.codes + tile * (Q4_TILE / 4) + 4 * lane);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            f32x4 part = {};
#pragma unroll
            for (int i = j * (4 / PER); i < (j + 1) * (4 / PER); ++i)
                part = __builtin_amdgcn_mfma_f32_16x16x32_f16(q4_values((uint32_t)c[i]), q4_octet<VEC>(row, tk * Q4_K + 32 * i + 8 * g, w.K), part, 0, 0, 0);
            const f16x4 s = *reinterpret_cast<const f16x4 *>(w.scales + tile * (16 * PER) + (g * PER + j) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(part[i], (float)s[i], acc[i]);
        }
    }
    if (m >= M) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = tn * Q4_N + 4 * g + i;
        if (n >= w.N) break;
        const size_t at = (size_t)m * w.N + n;
        C[at] = q4_out(acc[i] + (bias ? h2f(bias[n]) : 0.f), epi, resid, at);
    }
}

static bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
static size_t q4_tiles(int N, int K) { return (size_t)cdiv(N, Q4_N) * cdiv(K, Q4_K); }
static bool int4_refused(const GPT2Int4W *w, const char *what) {
    if (!w || !w->codes || !w->scales || !aligned16(w->codes) || !aligned16(w->scales) || w->N < 1 || w->K < 1 || !group_ok(w->group) ||
        q4_tiles(w->N, w->K) > 0xffffff)
        return arg_fail(what);
    return false;
}

// f(group as a constant, `vec` as one)
template <class F>
static void by_group(int group, bool vec, F f) {
    auto with = [&](auto g) {
        if (vec) f(g, std::true_type{});
        else f(g, std::false_type{});
    };
    if (group == 32) with(std::integral_constant<int, 32>{});
    else if (group == 64) with(std::integral_constant<int, 64>{});
    else with(std::integral_constant<int, 128>{});
}

}  // namespace g2

using namespace g2;

extern "C" size_t gpt2_int4_code_bytes(int N, int K) { return N < 1 || K < 1 ? 0 : q4_tiles(N, K) * Q4_TILE; }
extern "C" size_t gpt2_int4_scale_count(int N, int K, int group) {
    return N < 1 || K < 1 || !group_ok(group) ? 0 : q4_tiles(N, K) * (size_t)(16 * (Q4_K / group));
}

extern "C" int gpt2_int4_alloc(GPT2Int4W *w, int N, int K, int group) {
    if (!w) return arg_fail("gpt2_int4_alloc: null"), 1;
    memset(w, 0, sizeof(*w));
    if (N < 1 || K < 1 || !group_ok(group) || q4_tiles(N, K) > 0xffffff) return arg_fail("gpt2_int4_alloc: sizes out of range"), 1;
    const size_t codes = gpt2_int4_code_bytes(N, K);
    char *p = (char *)gpt2_dmalloc(codes + 2 * gpt2_int4_scale_count(N, K, group));
    if (!p) return 1;
    *w = GPT2Int4W{(uint8_t *)p, (gpt2_half *)(p + codes), N, K, group, p};
    return 0;
}

extern "C" void gpt2_int4_free(GPT2Int4W *w) {
    if (w && w->arena) {
        gpt2_dfree(w->arena);
        memset(w, 0, sizeof(*w));
    }
}

extern "C" void gpt2_quantize_int4(const GPT2Int4W *w, const gpt2_half *src) {
    if (int4_refused(w, "gpt2_quantize_int4: bad weights")) return;
    if (!src || ((uintptr_t)src & 1)) { arg_fail("gpt2_quantize_int4: null/unaligned"); return; }
    const int kb = cdiv(w->K, Q4_K);
    by_group(w->group, w->K % 8 == 0 && aligned16(src), [&](auto g, auto vec) {
        hipLaunchKernelGGL((k_quantize_int4<g.value, vec.value>), dim3((unsigned)q4_tiles(w->N, w->K)), dim3(256), 0, stream(), (uint32_t *)w->codes,
                           w->scales, src, w->N, w->K, kb);
    });
    check_launch("k_quantize_int4");
}

extern "C" void gpt2_dequantize_int4(gpt2_half *dst, const GPT2Int4W *w) {
    if (int4_refused(w, "gpt2_dequantize_int4: bad weights")) return;
    if (!dst || ((uintptr_t)dst & 1)) { arg_fail("gpt2_dequantize_int4: null/unaligned"); return; }
    const int kb = cdiv(w->K, Q4_K);
    by_group(w->group, w->K % 8 == 0 && aligned16(dst), [&](auto g, auto vec) {
        hipLaunchKernelGGL((k_dequantize_int4<g.value, vec.value>), dim3((unsigned)q4_tiles(w->N, w->K)), dim3(256), 0, stream(), dst, (const uint32_t *)w->codes,
                           w->scales, w->N, w->K, kb);
    });
    check_launch("k_dequantize_int4");
}

extern "C" void gpt2_matmul_int4(gpt2_half *C, const gpt2_half *A, const GPT2Int4W *w, const gpt2_half *bias, int M, int epi, const gpt2_half *resid) {
    if (int4_refused(w, "gpt2_matmul_int4: bad weights")) return;
    if (M < 0 || M > 1 << 21 || epi < GPT2_EPI_NONE || epi > GPT2_EPI_ADD) { arg_fail("gpt2_matmul_int4: rows or epilogue out of range"); return; }
    if (M == 0) return;
    if (!C || !A || (((uintptr_t)C | (uintptr_t)A | (uintptr_t)bias) & 1) || (epi == GPT2_EPI_ADD) != (resid != nullptr) || ((uintptr_t)resid & 1)) {
        arg_fail("gpt2_matmul_int4: null/unaligned, or a residual without its epilogue");
        return;
    }
    const Q4 q = {(const uint32_t *)w->codes, w->scales, w->N, w->K, cdiv(w->K, Q4_K)};
    by_group(w->group, w->K % 8 == 0 && aligned16(A), [&](auto g, auto vec) {
        hipLaunchKernelGGL((k_int4_any<g.value, vec.value>), dim3(cdiv(w->N, Q4_N), cdiv(M, 64)), dim3(256), 0, stream(), C, A, q, bias, M, epi, resid);
    });
    check_launch("k_int4_any");
}

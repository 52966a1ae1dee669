// int4.hip -- weights of 4 bits with group scales (gpt2_int4.h): the quantiser, its inverse and the products.
//
// A code is exact in fp16 and its products are exact in fp32, so the products run on v_mfma_f32_16x16x32_f16 with codes made fp16 in registers; a group is
// summed from 0 and added times its scale in fp32, one multiplication for each output and group.  The tiles lie as the instructions take them: a lane's
// 16 bytes are its codes for four instructions, and a load of a wave is 1 KB in one piece.
#include <cmath>
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

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Where octet o (eight consecutive k) of output n lies in a tile, in words.
__device__ __forceinline__ int q4_word(int n, int o) { return ((o & 3) * 16 + n) * 4 + (o >> 2); }

// Eight codes as exact fp16 values, in order: a code under the exponent of 1024 is 1024 + u, or with its four bits one place
// of four higher 1024 + 16 u; u = q + 8 (codes made fp16 by their exponent: Kim, Henry, Fahim, Awadalla, "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into
// Cloud Scale Production", 2022).  The masks come from registers, so that each pair takes one instruction for mask and exponent (a vector
// instruction has room for one literal): a kernel makes one Q4Bits and keeps it.
struct Q4Bits {
    uint32_t lo = 0x000f000fu, hi = 0x00f000f0u, one = 0x64006400u;
    __device__ __forceinline__ Q4Bits() { asm("" : "+s"(lo), "+s"(hi), "+v"(one)); }
};
__device__ __forceinline__ f16x8 q4_values(uint32_t w, const Q4Bits &k) {
    const f16x2 lo_off = {(f16)-1032.f, (f16)-1032.f}, sixteenth = {(f16)0.0625f, (f16)0.0625f}, hi_off = {(f16)-72.f, (f16)-72.f};
    f16x2 v[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t x = w >> (8 * h);
        v[2 * h] = __builtin_bit_cast(f16x2, (x & k.lo) | k.one) + lo_off;
        v[2 * h + 1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (x & k.hi) | k.one), sixteenth, hi_off);
    }
    return f16x8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}

// Eight consecutive halves of a row of K from k on, 0 past its end; rows at any alignment.
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef uint16_t u16x4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ f16x8 q4_eight(const uint16_t *at) { return __builtin_bit_cast(f16x8, *reinterpret_cast<const u16x8_any *>(at)); }
// Where the row ends inside the octet, its last eight are loaded and moved down.
__device__ __forceinline__ f16x8 q4_octet(const uint16_t *row, int k, int K) {
    f16x8 v = {};
    if (K >= 8) {
        const int past = k + 8 - K;   // halves past the end
        const i32x4 w = __builtin_bit_cast(i32x4, q4_eight(row + min(k, K - 8)));
        if (past <= 0) return __builtin_bit_cast(f16x8, w);
        if (past >= 8) return v;
        const uint64_t lo = (uint64_t)(uint32_t)w[1] << 32 | (uint32_t)w[0], hi = (uint64_t)(uint32_t)w[3] << 32 | (uint32_t)w[2];
        const int bits = 16 * past;
        const uint64_t a = bits < 64 ? lo >> bits | hi << (64 - bits) : hi >> (bits - 64), b = bits < 64 ? hi >> bits : 0;
        return __builtin_bit_cast(f16x8, i32x4{(int)a, (int)(a >> 32), (int)b, (int)(b >> 32)});
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < K) v[e] = __builtin_bit_cast(f16, row[k + e]);
    return v;
}

// A work-group a tile, a thread an octet: sixteen consecutive lanes have an output's 128 k, so a group's largest value is a maximum
// over 4, 8 or 16 lanes by DPP.  50257 x 768: 25.6 us under the tracer, 97 MB at 3.8 TB/s, with some 80 vector instructions an octet; work-groups that take
// several tiles with the next one's loads under way are no faster.
template <int G>
__global__ __launch_bounds__(256) void k_quantize_int4(uint32_t *__restrict__ codes, uint16_t *__restrict__ scales, const uint16_t *__restrict__ src, int N,
                                                       int K, int kb) {
    constexpr int PER = Q4_K / G;
    const int tid = threadIdx.x, n = tid >> 4, o = tid & 15;
    const int tile = blockIdx.x, row = tile / kb * Q4_N + n;
    f16x8 h = {};
    if (row < N) h = q4_octet(src + (size_t)row * K, tile % kb * Q4_K + 8 * o, K);
    auto largest = [&]() {   // of the sizes' bits
        const i32x4 b = __builtin_bit_cast(i32x4, h);
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, b[e] & 0x7fff7fff)));
        return max(m & 0xffffu, m >> 16);
    };
    uint32_t top = largest();
    if (__ballot(top >= 0x7c00u)) {   // infinities, NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = (float)h[e];
            h[e] = (f16)(v == v ? fminf(fmaxf(v, -65504.f), 65504.f) : 0.f);
        }
        top = largest();
    }
    auto over = [&](auto f) { top = max(top, (uint32_t)f((int)top)); };
    over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true); });
    over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true); });
    if constexpr (G >= 64) over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true); });
    if constexpr (G >= 128) over([](int v) { return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true); });
    const f16 s16 = (f16)(h2f((uint16_t)top) / 7.0f);
    const float s = (float)s16 == 0.f ? 1.f : (float)s16, inv = 1.0f / s;
    // x / s by a product, to the nearest whole number by what an addition of 1.5 2^23 rounds off: it is off by 2^-22 of at most 7.5, and numbers of 11 bits have quotients
    // that are n + 1/2 or 2^-13 from it, so only those that are n + 1/2 are looked at again (x - q s is exact): they go to the even one.  Past 7
    // are only quotients by scales below the normal numbers.  With eight divisions a thread the head's matrix took 38 us.
    constexpr float whole = 12582912.f;
    float q[8], off = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        q[e] = __builtin_fmaf((float)h[e], inv, whole) - whole;
        off = fmaxf(off, fabsf(__builtin_fmaf(-q[e], s, (float)h[e])));
    }
    if (__ballot(off >= 0.5f * s || s < 0x1p-14f))
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (fabsf(__builtin_fmaf(-q[e], s, (float)h[e])) == 0.5f * s) q[e] = 2.f * rintf(0.5f * ((float)h[e] * inv));
            q[e] = fminf(fmaxf(q[e], -7.f), 7.f);
        }
    float half[2] = {8.f * 0x1111, 8.f * 0x1111};   // the four codes of a half word, exact in fp32
#pragma unroll
    for (int e = 0; e < 8; ++e) half[e & 1] = __builtin_fmaf(q[e], (float)(1 << (4 * (e >> 1))), half[e & 1]);
    const uint32_t w = (uint32_t)half[0] | (uint32_t)half[1] << 16;
    codes[(size_t)tile * (Q4_TILE / 4) + q4_word(n, o)] = w;
    if (o % (G / 8) == 0) scales[(size_t)tile * (16 * PER) + ((n >> 2) * PER + o / (G / 8)) * 4 + (n & 3)] = f2h(s);
}

// 50257 x 768: 15.7 us, 97 MB at 6.2 TB/s (what is written stays in the last cache).
template <int G>
__global__ __launch_bounds__(256) void k_dequantize_int4(uint16_t *__restrict__ dst, const uint32_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                                         int N, int K, int kb) {
    constexpr int PER = Q4_K / G;
    const int tid = threadIdx.x, n = tid >> 4, o = tid & 15, tk = blockIdx.x % kb, tn = blockIdx.x / kb;
    const int row = tn * Q4_N + n, k = tk * Q4_K + 8 * o;
    if (row >= N || k >= K) return;
    const size_t tile = (size_t)tn * kb + tk;
    const f16x8 q = q4_values(codes[tile * (Q4_TILE / 4) + q4_word(n, o)], Q4Bits());
    const float s = h2f(scales[tile * (16 * PER) + ((n >> 2) * PER + o / (G / 8)) * 4 + (n & 3)]);
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (f16)((float)q[e] * s);
    uint16_t *to = dst + (size_t)row * K + k;
    if (k + 8 <= K) *reinterpret_cast<u16x8_any *>(to) = __builtin_bit_cast(u16x8_any, v);
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) to[e] = f2h((float)q[e] * s);
}

__device__ __forceinline__ int cdiv_dev(int a, int b) { return (a + b - 1) / b; }

template <int EPI>
__device__ __forceinline__ uint16_t q4_round(float v) {
    if constexpr (EPI == GPT2_EPI_GELU) {
        constexpr float K = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
        v = v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(K * __builtin_fmaf(0.044715f, v * v * v, v)));
    }
    return f2h(v);
}

// A lane's four outputs n .. n + 3 of row m: bias, what follows in fp32 (gelu_new as v / (1 + 2^(K (v + 0.044715 v^3))), K = -2 sqrt(2 / pi) log2(e);
// or the residual), one rounding.  Four halves go as one piece wherever a row begins (by halves 1059 rows of 10543 x 139 and a residual took 104 us).
template <int EPI>
__device__ __forceinline__ void q4_store(uint16_t *C, f32x4 v, int n, int m, int M, int N, const uint16_t *bias, const uint16_t *resid) {
    if (m >= M || n >= N) return;
    const size_t at = (size_t)m * N + n;
    if (n + 4 <= N) {
        u16x4_any b = {}, r = {}, o;
        if (bias) b = *reinterpret_cast<const u16x4_any *>(bias + n);
        if constexpr (EPI == GPT2_EPI_ADD) r = *reinterpret_cast<const u16x4_any *>(resid + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y = v[i] + h2f(b[i]);
            if constexpr (EPI == GPT2_EPI_ADD) y = h2f(r[i]) + y;
            o[i] = q4_round<EPI>(y);
        }
        *reinterpret_cast<u16x4_any *>(C + at) = o;
    } else
        for (int i = 0; n + i < N; ++i) {
            float y = (i == 0 ? v[0] : i == 1 ? v[1] : v[2]) + (bias ? h2f(bias[n + i]) : 0.f);
            if constexpr (EPI == GPT2_EPI_ADD) y = h2f(resid[at + i]) + y;
            C[at + i] = q4_round<EPI>(y);
        }
}
// f(epilogue as a constant)
template <class F>
__device__ __forceinline__ void by_epilogue(int epi, F f) {
    if (epi == GPT2_EPI_GELU) f(std::integral_constant<int, GPT2_EPI_GELU>{});
    else if (epi == GPT2_EPI_ADD) f(std::integral_constant<int, GPT2_EPI_ADD>{});
    else f(std::integral_constant<int, GPT2_EPI_NONE>{});
}

// On the matrix units the codes are the A operand (lane l: output l % 16, the octet l / 16 of 32 k) and rows of activations the B operand, so a
// lane ends with outputs 4 (l / 16) .. + 3 of row l % 16.  Weights rounded to fp16 with their scales would save the multiplication by group and add half as much again to
// the result's rounding.

// Up to 16 rows: the weights are a stream.  A work-group has NT tiles of 16 outputs; its KW waves take the tiles along k in turn, U at a time with the
// next U on the way.  A wave's piece of A goes through LDS of its own, 4 RQ rows of 256 bytes (16-byte octet o of row r at o ^ (r & 15), so that rows
// read together lie in different banks), so nothing is waited for but the wave's own loads; where there are fewer than 16 rows the matrix unit's other
// columns compute what nobody stores.  The waves' sums are added in wave order.
// Bound by the stream: one row of 8192 x 8192, 34.6 MB, 8.3 us (4.2 TB/s, where a copy has 5.1), of 2304 x 768 2.9 under the tracer, the latency of a launch and one
// round of loads.  A tile of codes takes 36 vector instructions to become fp16 (with both masks as literals 52: 9.2 us for 8.9).
template <int G, int RQ, int NT, int KW, int U>
__global__ __launch_bounds__(64 * KW) void k_int4_rows(uint16_t *C, const uint16_t *__restrict__ A, Q4 w, const uint16_t *__restrict__ bias, int M, int epi,
                                                       const uint16_t *resid) {
    constexpr int PER = Q4_K / G, ROWS = 4 * RQ, STAGE = ROWS * 256, SUMS = KW * NT * 1024;
    static_assert(ROWS <= 16, "rows of one tile");
    __shared__ __attribute__((aligned(1024))) char lds[KW * STAGE > SUMS ? KW * STAGE : SUMS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int tn0 = blockIdx.x * NT, tns = cdiv_dev(w.N, Q4_N);
    char *const mine = lds + wave * STAGE;
    struct Stage {
        i32x4 c[NT];
        f16x8 x[RQ];
        f16x4 s[NT][PER];
    };
    auto load = [&](Stage (&st)[U], int r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int tk = min((r * U + u) * KW + wave, w.kb - 1);
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const size_t tile = (size_t)min(tn0 + a, tns - 1) * w.kb + tk;
                st[u].c[a] = *reinterpret_cast<const i32x4 *>(w.codes + tile * (Q4_TILE / 4) + 4 * lane);
#pragma unroll
                for (int j = 0; j < PER; ++j) st[u].s[a][j] = *reinterpret_cast<const f16x4 *>(w.scales + tile * (16 * PER) + (g * PER + j) * 4);
            }
            const bool whole = tk * Q4_K + Q4_K <= w.K;
#pragma unroll
            for (int q = 0; q < RQ; ++q) {
                const uint16_t *row = A + (size_t)min(4 * q + g, M - 1) * w.K;
                if (whole) st[u].x[q] = q4_eight(row + tk * Q4_K + 8 * l16);
                else st[u].x[q] = q4_octet(row, tk * Q4_K + 8 * l16, w.K);
            }
        }
    };
    const Q4Bits bits;
    f32x4 acc[NT] = {};
    auto compute = [&](Stage (&st)[U], int r) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if ((r * U + u) * KW + wave >= w.kb) return;
#pragma unroll
            for (int q = 0; q < RQ; ++q) {
                const int row = 4 * q + g;
                *reinterpret_cast<f16x8 *>(mine + row * 256 + ((l16 ^ row) << 4)) = st[u].x[q];
            }
            asm volatile("" ::: "memory");   // other lanes' pieces are read below; a wave's LDS operations are done in order
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                f32x4 part[NT] = {};
#pragma unroll
                for (int i = j * (4 / PER); i < (j + 1) * (4 / PER); ++i) {
                    const int row = l16 & (ROWS - 1);
                    const f16x8 x = *reinterpret_cast<const f16x8 *>(mine + row * 256 + (((4 * i + g) ^ row) << 4));
#pragma unroll
                    for (int a = 0; a < NT; ++a) part[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q4_values((uint32_t)st[u].c[a][i], bits), x, part[a], 0, 0, 0);
                }
#pragma unroll
                for (int a = 0; a < NT; ++a)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[a][i] = __builtin_fmaf(part[a][i], (float)st[u].s[a][j][i], acc[a][i]);
            }
            asm volatile("" ::: "memory");
        }
    };
    const int rounds = cdiv_dev(w.kb, KW * U);
    Stage s0[U], s1[U];
    load(s0, 0);
    for (int r = 0; r < rounds; r += 2) {
        if (r + 1 < rounds) load(s1, r + 1);
        compute(s0, r);
        if (r + 1 >= rounds) break;
        if (r + 2 < rounds) load(s0, r + 2);
        compute(s1, r + 1);
    }
    __syncthreads();   // every wave is done with its piece
    f32x4 *const sums = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int a = 0; a < NT; ++a) sums[(a * KW + wave) * 64 + lane] = acc[a];
    __syncthreads();
    for (int a = wave; a < NT; a += KW) {
        f32x4 v = sums[a * KW * 64 + lane];
#pragma unroll
        for (int i = 1; i < KW; ++i) v += sums[(a * KW + i) * 64 + lane];
        by_epilogue(epi, [&](auto k) { q4_store<k.value>(C, v, (tn0 + a) * Q4_N + 4 * g, l16, M, w.N, bias, resid); });
    }
}

// Many rows: tiles of BM rows and BN outputs, 128 k at a time.  Rows of A (256 bytes, swizzled as above), the codes' tiles as they lie and the waves'
// scales go to LDS by direct loads into a ring of S stages; a wave reads its fragments, makes the codes fp16 and multiplies.  WM x WN waves share a
// stage, each with 16 TM rows and 16 TN outputs; KS such groups split K and meet in LDS.  SREG: scales in registers instead, which lets one more work-group on a
// CU (two of 128 x 128: 2 x 80 KB); !DIRECT: everything through registers, for rows that are not at 16 bytes.
// 2000 x 4096 x 4096 takes 67 to 76 us by the card (0.88 to 1.0 PFLOP/s): by the counters of its 128 x 128 form the matrix units have 48% of the cycles, other vector
// instructions 32 and LDS reads 25, without a bank conflict, so what is left is how they overlap; hints to the compiler's scheduling gave nothing, 256 x 128 tiles on eight waves took 77 for 72.  A wave takes 128 rows by 32 outputs rather
// than 64 by 64, since each wave makes its codes fp16 for itself (70 us for 76).  Products of a few hundred rows are chains of short steps: 777 rows of 768
// x 3072, six steps of 1.1 us and the launch.
__device__ __attribute__((aligned(16))) uint32_t g_q4_zero[4] = {};   // what is multiplied past K

template <int G, int BM, int BN, int WM, int WN, int KS, int S, bool SREG, bool DIRECT>
__device__ __forceinline__ void int4_tile(uint16_t *C, const uint16_t *__restrict__ A, const uint32_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                          int N, int K, int kb, const uint16_t *__restrict__ bias, int M, int epi, const uint16_t *resid, int tiles_m,
                                          int tiles, int along_n) {
#if defined(__HIP_DEVICE_COMPILE__)   // LDS address-space pointers exist only in the device pass
    constexpr int PER = Q4_K / G, NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int A_B = BM * 256, W_B = BN * 64, S_B = SREG ? 0 : NW * TN * 32 * PER, STAGE = A_B + W_B + (S_B + 255) / 256 * 256;
    constexpr int A_INS = BM / 4, W_INS = BN / 16, PIECES = (A_INS + W_INS + NW - 1) / NW, LOADS = PIECES + 1;   // a wave's loads a stage
    static_assert(!SREG || S == 2, "scales in registers are there with the only stage under way");
    static_assert(DIRECT || SREG, "without direct loads scales are in registers");
    static_assert(TN * 2 * PER <= 64 && LOADS * (S - 1) < 64, "a wave's scales are one load; loads are counted");
    constexpr int SUMS = (KS - 1) * NW * TM * TN * 1024;
    __shared__ __attribute__((aligned(1024))) char lds[KS * S * STAGE > SUMS ? KS * S * STAGE : SUMS];
    const int lane = threadIdx.x & 63, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int kg = wave_all / NW, wave = wave_all % NW;
    char *const ring = lds + kg * S * STAGE;
    // consecutive work-groups go round the eight XCDs: each XCD has one run of tiles
    int tile = blockIdx.x;
    {
        const int xcd = tile & 7, slot = tile >> 3, per = tiles >> 3, rem = tiles & 7;
        tile = xcd * per + min(xcd, rem) + slot;
    }
    const int tiles_n = tiles / tiles_m, tns = cdiv_dev(N, Q4_N);
    const int m0 = (along_n ? tile / tiles_n : tile % tiles_m) * BM, tn0 = (along_n ? tile % tiles_n : tile / tiles_m) * (BN / 16);
    const int wm0 = (wave % WM) * TM * 16, wn0 = (wave / WM) * TN;   // within the tile: rows; tiles of 16 outputs
    const int steps = cdiv_dev(kb, KS), k_first = kg * steps;        // of 128 k; the last group may have fewer

    const char *src[PIECES];
    int dst[PIECES], step_b[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int q = min(wave + NW * j, A_INS + W_INS - 1);
        if (q < A_INS) {
            const int row = 4 * q + g;
            src[j] = reinterpret_cast<const char *>(A + (size_t)min(m0 + row, M - 1) * K) + ((l16 ^ (row & 15)) << 4);
            dst[j] = q * 1024;
            step_b[j] = 256;
        } else {
            src[j] = reinterpret_cast<const char *>(codes) + (size_t)min(tn0 + q - A_INS, tns - 1) * kb * Q4_TILE + 16 * lane;
            dst[j] = A_B + (q - A_INS) * 1024;
            step_b[j] = Q4_TILE;
        }
    }
    const char *const src_s = reinterpret_cast<const char *>(scales) + (size_t)min(tn0 + wn0 + lane / (2 * PER), tns - 1) * kb * (32 * PER) + (lane % (2 * PER)) * 16;
    const bool ragged = K & 127;
    auto issue = [&](int t) {
        const int tk = min(k_first + t, kb - 1);
        char *const st = ring + (t % S) * STAGE;
        if (ragged && tk == kb - 1) {   // what is multiplied past K is 0
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                const int q = min(wave + NW * j, A_INS + W_INS - 1), row = 4 * q + g;
                const bool past = q < A_INS && tk * Q4_K + 8 * (l16 ^ (row & 15)) >= K;
                __builtin_amdgcn_global_load_lds(past ? reinterpret_cast<const char *>(g_q4_zero) : src[j] + (size_t)tk * step_b[j], G2_LDS(st + dst[j]), 16, 0, 0);
            }
        } else
#pragma unroll
            for (int j = 0; j < PIECES; ++j) __builtin_amdgcn_global_load_lds(src[j] + (size_t)tk * step_b[j], G2_LDS(st + dst[j]), 16, 0, 0);
        if (!SREG && lane < TN * 2 * PER) __builtin_amdgcn_global_load_lds(src_s + (size_t)tk * (32 * PER), G2_LDS(st + A_B + W_B + wave * TN * 32 * PER), 16, 0, 0);
    };
    const Q4Bits bits;
    f32x4 acc[TN][TM] = {};
    f16x4 s_now[SREG ? TN : 1][PER], s_next[SREG ? TN : 1][PER];
    auto load_scales = [&](f16x4 (&to)[SREG ? TN : 1][PER], int t) {
        const int tk = min(k_first + t, kb - 1);
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                to[a][j] = *reinterpret_cast<const f16x4 *>(scales + ((size_t)min(tn0 + wn0 + a, tns - 1) * kb + tk) * (16 * PER) + (g * PER + j) * 4);
    };
    auto compute = [&](int t) {
        const char *const st = ring + (t % S) * STAGE;
        i32x4 c[TN];
#pragma unroll
        for (int a = 0; a < TN; ++a) c[a] = *reinterpret_cast<const i32x4 *>(st + A_B + (wn0 + a) * 1024 + 16 * lane);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            f32x4 part[TN][TM] = {};
#pragma unroll
            for (int i = j * (4 / PER); i < (j + 1) * (4 / PER); ++i) {
                f16x8 x[TM];
#pragma unroll
                for (int b = 0; b < TM; ++b) {
                    const int row = wm0 + 16 * b + l16;
                    x[b] = *reinterpret_cast<const f16x8 *>(st + row * 256 + (((4 * i + g) ^ l16) << 4));
                }
#pragma unroll
                for (int a = 0; a < TN; ++a) {
                    const f16x8 q = q4_values((uint32_t)c[a][i], bits);
#pragma unroll
                    for (int b = 0; b < TM; ++b) part[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q, x[b], part[a][b], 0, 0, 0);
                }
            }
#pragma unroll
            for (int a = 0; a < TN; ++a) {
                f16x4 s;
                if constexpr (SREG) s = s_now[a][j];
                else s = *reinterpret_cast<const f16x4 *>(st + A_B + W_B + (wave * TN + a) * 32 * PER + (g * PER + j) * 8);
#pragma unroll
                for (int b = 0; b < TM; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][b][e] = __builtin_fmaf(part[a][b][e], (float)s[e], acc[a][b][e]);
            }
        }
    };
    auto next_scales = [&](int t) {
        if constexpr (SREG) {
#pragma unroll
            for (int a = 0; a < TN; ++a)
#pragma unroll
                for (int j = 0; j < PER; ++j) s_now[a][j] = s_next[a][j];
            load_scales(s_next, t);   // ahead of a stage's other loads
        }
    };
    if constexpr (DIRECT) {
        if constexpr (SREG) load_scales(s_next, 0);
#pragma unroll
        for (int t = 0; t < S - 1; ++t)
            if (t < steps) issue(t);
        for (int t = 0; t < steps; ++t) {
            wait_tiles<LOADS, S - 2>(min(S - 2, steps - 1 - t));   // step t's loads are in
            lds_barrier();                                        // everyone's, and everyone is done with step t - 1
            next_scales(t + 1);
            if (t + S - 1 < steps) issue(t + S - 1);
            if (KS == 1 || k_first + t < kb) compute(t);
        }
    } else {   // through registers: the next step's pieces are under way while this one is multiplied
        f16x8 piece[PIECES];
        auto fetch = [&](int t) {
            const int tk = min(k_first + t, kb - 1);
            const bool whole = tk * Q4_K + Q4_K <= K;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                const int q = min(wave + NW * j, A_INS + W_INS - 1), row = 4 * q + g;
                const char *p = src[j] + (size_t)tk * step_b[j];
                if (q >= A_INS) piece[j] = *reinterpret_cast<const f16x8 *>(p);
                else if (whole) piece[j] = q4_eight(reinterpret_cast<const uint16_t *>(p));
                else piece[j] = q4_octet(A + (size_t)min(m0 + row, M - 1) * K, tk * Q4_K + 8 * (l16 ^ (row & 15)), K);
            }
        };
        auto put = [&](int t) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) *reinterpret_cast<f16x8 *>(ring + (t % S) * STAGE + dst[j] + 16 * lane) = piece[j];
        };
        fetch(0);
        put(0);
        for (int t = 0; t < steps; ++t) {
            __syncthreads();
            load_scales(s_now, t);   // needed behind the products
            if (t + 1 < steps) fetch(t + 1);
            if (KS == 1 || k_first + t < kb) compute(t);
            if (t + 1 < steps) put(t + 1);
        }
    }
    if constexpr (KS > 1) {
        lds_barrier();
        f32x4 *const sums = reinterpret_cast<f32x4 *>(lds);
        if (kg)
#pragma unroll
            for (int a = 0; a < TN; ++a)
#pragma unroll
                for (int b = 0; b < TM; ++b) sums[(((kg - 1) * NW + wave) * TN * TM + a * TM + b) * 64 + lane] = acc[a][b];
        lds_barrier();
        if (kg) return;
#pragma unroll
        for (int i = 0; i < KS - 1; ++i)
#pragma unroll
            for (int a = 0; a < TN; ++a)
#pragma unroll
                for (int b = 0; b < TM; ++b) acc[a][b] += sums[((i * NW + wave) * TN * TM + a * TM + b) * 64 + lane];
    }
    by_epilogue(epi, [&](auto e) {
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int b = 0; b < TM; ++b) q4_store<e.value>(C, acc[a][b], (tn0 + wn0 + a) * Q4_N + 4 * g, m0 + wm0 + 16 * b + l16, M, N, bias, resid);
    });
#endif
}
// Two waves a SIMD for the form through registers with four waves, which the compiler would give up for earlier loads (1272 rows of 4742 x 517, groups of 32: 33 us for 23).
template <int G, int BM, int BN, int WM, int WN, int KS, int S, bool SREG, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN * KS, !DIRECT && WM * WN * KS == 4 ? 2 : 1) void k_int4_tile(uint16_t *C, const uint16_t *__restrict__ A, const uint32_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                          int N, int K, int kb, const uint16_t *__restrict__ bias, int M, int epi, const uint16_t *resid, int tiles_m,
                                          int tiles, int along_n) {
    int4_tile<G, BM, BN, WM, WN, KS, S, SREG, DIRECT>(C, A, codes, scales, N, K, kb, bias, M, epi, resid, tiles_m, tiles, along_n);
}

static bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
static size_t q4_tiles(int N, int K) { return (size_t)cdiv(N, Q4_N) * cdiv(K, Q4_K); }
static bool int4_refused(const GPT2Int4W *w, const char *what) {
    if (!w || !w->codes || !w->scales || !aligned16(w->codes) || !aligned16(w->scales) || w->N < 1 || w->K < 1 || !group_ok(w->group) ||
        q4_tiles(w->N, w->K) > 0xffffff)
        return arg_fail(what);
    return false;
}

// f(group as a constant)
template <class F>
static void by_group(int group, F f) {
    if (group == 32) f(std::integral_constant<int, 32>{});
    else if (group == 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

typedef void (*Q4RowsFn)(uint16_t *, const uint16_t *, Q4, const uint16_t *, int, int, const uint16_t *);
typedef void (*Q4TileFn)(uint16_t *, const uint16_t *, const uint32_t *, const uint16_t *, int, int, int, const uint16_t *, int, int, const uint16_t *, int, int, int);

// The form for up to 16 rows, NT tiles of outputs x KW waves.  us a call, one row unless said:
//   768 tiles and more: 2 x 4 (16 rows of 16400 x 768 4.4, 1 x 8 for 16000 5.0; 50257 x 4096: 24.9, 2 x 8 25.2; x 1600, 16 rows: 16.4, 2 x 8 28.5, 1 x 4 with two tiles each under way 27.2), and for 5 to 8
//   rows of five or six tiles along k, which three waves take in one round of two and four in two rounds, 2 x 3 (8 rows of 50257 x 768, groups of 128: 7.1, 2 x 4 7.7; x 640 6.7 and 7.3;
//   100000 x 768 10.5 and 11.5).  Not of four tiles or fewer (50257 x 512: 6.4, 2 x 4 5.7; x 256 5.2 and 4.5), and not in groups of 32, whose scales leave its registers two
//   work-groups a CU (50257 x 768: 8.4, 2 x 4 8.2; x 510 10.2 and 6.7);
//   fewer and long rows: 16 waves (2048 x 8192: 1 x 16 5.2, 1 x 8 6.5; 8192 x 8192: 2 x 16 8.8, 1 x 8 9.0, 1 x 16 9.6), 8 for more than eight rows, whose pieces
//   would not leave the registers; else 1 x 8.
template <int G, int RQ>
static void rows_form(const Q4 &q, Q4RowsFn &fn, int &nt, int &kw) {
    const int tiles = cdiv(q.N, Q4_N);
    auto take = [&](Q4RowsFn f, int n, int k) { fn = f, nt = n, kw = k; };
    if (tiles >= 768) {
        if constexpr (RQ == 2 && G > 32)
            if (q.kb == 5 || q.kb == 6) return take(k_int4_rows<G, RQ, 2, 3, 2>, 2, 3);
        return take(k_int4_rows<G, RQ, 2, 4, 1>, 2, 4);
    }
    if (q.kb < 32) return take(k_int4_rows<G, RQ, 1, 8, 1>, 1, 8);
    if constexpr (RQ < 4) return tiles > 256 ? take(k_int4_rows<G, RQ, 2, 16, 1>, 2, 16) : take(k_int4_rows<G, RQ, 1, 16, 1>, 1, 16);
    else return tiles > 256 ? take(k_int4_rows<G, RQ, 2, 8, 1>, 2, 8) : take(k_int4_rows<G, RQ, 1, 8, 1>, 1, 8);
}

// A form for more rows, and what it takes in us: a round of work-groups `start` and `step` for each 128 k of a group of waves; each further work-group on a CU
// that has room for `room` at once `start2` and `step2`.  Fitted to the times of 580 products, 17 to 1990 rows, N from 65 to 50257, K from 136 to 8152, each in groups of 32, 64
// and 128: the form with the smallest sum is within 0.3% of the fastest of the nine in the mean, 15% at most (fitted to the first 460, 0.5% and 12% on the others); without any one of them products
// are up to 1.16 to 1.49 times as long (the least, 64 x 64: 1.11).
struct Q4Form {
    int bm, bn, ks, threads, room;
    float start, step, start2, step2;
    Q4TileFn fn;
};
template <int G, int BM, int BN, int WM, int WN, int KS, int S, bool SREG, bool DIRECT>
static Q4Form q4_form(int room, float start, float step, float start2, float step2) {
    return {BM, BN, KS, 64 * WM * WN * KS, room, start, step, start2, step2, k_int4_tile<G, BM, BN, WM, WN, KS, S, SREG, DIRECT>};
}
template <int G>
static const Q4Form &tile_form(int M, int N, int kb, bool direct) {
    static const Q4Form by_loads[] = {
        q4_form<G, 16, 32, 1, 1, 8, 2, false, true>(1, 2.07f, 0.75f, 0.f, 0.f),    q4_form<G, 16, 64, 1, 4, 3, 3, false, true>(2, 1.63f, 0.58f, 0.29f, 0.48f),
        q4_form<G, 32, 32, 1, 2, 4, 3, false, true>(1, 1.70f, 0.66f, 0.f, 0.f),    q4_form<G, 32, 64, 1, 4, 4, 2, true, true>(1, 1.89f, 0.95f, 0.f, 0.f),
        q4_form<G, 32, 64, 1, 4, 2, 3, false, true>(2, 1.50f, 0.66f, 0.27f, 0.30f), q4_form<G, 48, 64, 1, 4, 4, 2, true, true>(1, 1.75f, 1.24f, 0.f, 0.f),
        q4_form<G, 64, 64, 1, 2, 2, 2, true, true>(2, 1.82f, 0.97f, 0.86f, 0.41f),  q4_form<G, 64, 128, 1, 4, 1, 2, true, true>(3, 1.81f, 0.76f, 0.98f, 0.37f),
        q4_form<G, 128, 128, 1, 4, 1, 2, true, true>(2, 3.77f, 1.25f, 1.85f, 0.67f)};
    // Rows that are not at 16 bytes: fitted to the times of 580 products, 17 to 2000 rows, N from 66 to 50257, K from 139 to 8175, each in groups of 32, 64 and 128: within 0.2% of the fastest of the six in the
    // mean, 13% at most; fitted to the first 460, 0.4% and 11% on the others.  Without any one of them products are up to 1.17 to 1.9 times as long.  How many
    // work-groups of 32 x 64 and 64 x 128 a CU has room for goes by the registers that a group size takes.
    static const Q4Form by_registers[] = {
        q4_form<G, 16, 32, 1, 1, 8, 2, true, false>(1, 1.79f, 1.34f, 0.f, 0.f), q4_form<G, 16, 64, 1, 4, 3, 2, true, false>(2, 1.44f, 0.60f, 0.36f, 0.42f),
        q4_form<G, 32, 64, 1, 4, 4, 2, true, false>(1, 1.56f, 1.24f, 0.f, 0.f), q4_form<G, 32, 64, 1, 4, 2, 2, true, false>(G == 64 ? 2 : 3, 1.32f, 0.75f, 0.22f, 0.35f),
        q4_form<G, 48, 64, 1, 4, 4, 2, true, false>(1, 1.89f, 1.55f, 0.f, 0.f), q4_form<G, 64, 128, 1, 4, 1, 2, true, false>(G == 128 ? 3 : 2, 2.56f, 0.93f, 1.13f, 0.33f)};
    const Q4Form *const forms = direct ? by_loads : by_registers, *best = forms;
    float least = INFINITY;
    for (const Q4Form *f = forms, *end = forms + (direct ? sizeof by_loads : sizeof by_registers) / sizeof *forms; f < end; ++f) {
        const float a_cu = ceilf((float)cdiv(M, f->bm) * cdiv(N, f->bn) / 256.f), rounds = ceilf(a_cu / f->room), steps = cdiv(kb, f->ks);
        const float us = rounds * (f->start + steps * f->step) + (a_cu - rounds) * (f->start2 + steps * f->step2);
        if (us < least) least = us, best = f;
    }
    return *best;
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
    by_group(w->group, [&](auto g) {
        hipLaunchKernelGGL(k_quantize_int4<g.value>, dim3((unsigned)q4_tiles(w->N, w->K)), dim3(256), 0, stream(), (uint32_t *)w->codes,
                           w->scales, src, w->N, w->K, kb);
    });
    check_launch("k_quantize_int4");
}

extern "C" void gpt2_dequantize_int4(gpt2_half *dst, const GPT2Int4W *w) {
    if (int4_refused(w, "gpt2_dequantize_int4: bad weights")) return;
    if (!dst || ((uintptr_t)dst & 1)) { arg_fail("gpt2_dequantize_int4: null/unaligned"); return; }
    const int kb = cdiv(w->K, Q4_K);
    by_group(w->group, [&](auto g) {
        hipLaunchKernelGGL(k_dequantize_int4<g.value>, dim3((unsigned)q4_tiles(w->N, w->K)), dim3(256), 0, stream(), dst, (const uint32_t *)w->codes,
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
    by_group(w->group, [&](auto group) {
        constexpr int G = group.value;
        if (M <= 16) {
            Q4RowsFn fn;
            int nt, kw;
            if (M <= 4) rows_form<G, 1>(q, fn, nt, kw);
            else if (M <= 8) rows_form<G, 2>(q, fn, nt, kw);
            else rows_form<G, 4>(q, fn, nt, kw);
            hipLaunchKernelGGL(fn, dim3(cdiv(cdiv(q.N, Q4_N), nt)), dim3(64 * kw), 0, stream(), C, A, q, bias, M, epi, resid);
            return;
        }
        const Q4Form &f = tile_form<G>(M, q.N, q.kb, w->K % 8 == 0 && aligned16(A));
        const int tm = cdiv(M, f.bm), tn = cdiv(q.N, f.bn);
        if ((double)tm * tn * f.threads >= 0x1p32) { arg_fail("gpt2_matmul_int4: more outputs than a launch has threads for"); return; }
        // an XCD's run of tiles goes along n where the eight of them then read less: all codes once for each of up to eight rows of tiles, or all of A once for
        // each of up to eight columns (2000 x 4096 x 4096: 64 x 128 tiles 89.3 -> 84.7 us)
        const int along_n = 2.0 * M + 0.5 * q.N * (tm < 8 ? tm : 8) < 0.5 * q.N + 2.0 * M * (tn < 8 ? tn : 8);
        hipLaunchKernelGGL(f.fn, dim3(tm * tn), dim3(f.threads), 0, stream(), C, A, q.codes, q.scales, q.N, q.K, q.kb, bias, M, epi, resid, tm, tm * tn, along_n);
    });
    check_launch("gpt2_matmul_int4");
}

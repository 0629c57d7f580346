// The paged cache in 4 bits, and how the attention works on it.
//
// A page is cut into blocks of 16 slots; a block holds, head by head, a tile: for every 32 elements of the head 16 rows of
// 16 bytes (one per slot; element 2j in the low half of byte j), then for every group of elements 16 words.  So the
// attention's tile of 16 keys of one head is one run of bytes, which one bulk copy brings, already in the order in which
// eight rows of 16 bytes meet all banks.  A word is the bits of the group's scale with the zero point in the last
// four: scales have 20 significant bits, and a scale times a difference of two 4-bit numbers is exact in fp32.
#pragma once

#include "l2d_attn.cuh"

#include <cfloat>
#include <type_traits>

namespace l2d {

constexpr int kBlockSlots = 16;
constexpr int kChunk = 32;                           // elements of a row of 16 bytes
constexpr int kChunkBytes = kBlockSlots * 16;
constexpr int kGroupBytes = kBlockSlots * 4;

// ---------------------------------------------------------------------------------------------
// Attention: one warp's part of one head group, in the kernel that l2d_attn.cuh describes.
//
// Per 16 keys of 128 elements a warp reads 2 x 1088 bytes, which an SM's share of the memory brings in about 100 cycles,
// the issue of 400 instructions; so the conversion of 4096 nibbles is what has to be cheap.  A word of eight nibbles gives
// four registers of two 16-bit numbers each: a mask and a multiply-add that takes off the zero point, and one shift for the
// upper two; the differences n - z are exact.  Scales stay outside the products: the scores of a group's elements are
// multiplied by its key's scale as fp32 sums, and weights by the value's scale before they are cut into 16-bit parts.
//
// Keys are the rows of a product with the queries of eight heads as columns: a matrix of ldmatrix (8 keys x 16 bytes) gives a
// lane word t of key g, elements 8t .. 8t + 7 of the 32, and queries are staged in the order in which two instructions meet
// them.  Elements of values are the rows of the other, with the weights as columns: the transposed load gives a lane the
// same four elements of keys 2t and 2t + 1 side by side, as an A operand wants two neighbours of a row, nibble by
// nibble; the weights come from the layout of sums to that of a B operand by movmatrix.  (With the heads as rows eight of 16 would
// be empty for groups of up to eight, or hold second parts, and their sums would take twice the registers.)
//
// Queries of 32 bits are three bf16 numbers that add up to them.  Weights times scales are three for fp32 and fp16, and two for
// bf16, which leaves 2^-16 of one, a 256th of what rounding an output to bf16 may take off; with two, one output in a hundred was
// not the nearest fp16 number (1 x 131072 keys; with three one in five hundred, as of a softmax in fp32; 47.1 us for 43.5, and 64 x
// 8192 keys 112 for 101).  In 32 bits the sums of products with each part of a query stay apart, and so do a run's products with
// weights: the instruction cuts a product off at its sum's last place, and apart the small parts lose nothing to a large sum (errors
// against 64 bits over 120 drawn fp32 cases 2.4e-7 at most, not 1.2e-6; 16 x 8192 keys, 32 / 8 heads of 128, 45 us for 42).  In 16
// bits they stay in the instruction: where all values are positive and nothing cancels, outputs over 131072 keys are 6e-6 too small
// on average, an 80th of fp16's half step (apart, 1 x 131072 keys take 50.7 us).
//
// Measured (32 query and 8 key-value heads of 128, bf16, one group a head): 64 sequences of 0 to 8192 keys 102 us, 2.8 TB/s, for
// 45 us of bytes (131 us in groups of 32); one sequence of 17 keys 6.5 us, of which a launch 4.1.  457 warp instructions per 16
// keys and values would take 53 us if they filled the issue slots; they fill 56 % of them.  What binds is the latency of one chain
// after the other (scores, their maximum, weights, values) in the 16 warps a SM that registers leave room for; the kernels of heads of
// 97 to 128 elements spill 40 (one group) to 152 bytes (groups of 32, fp16 168) a thread at their 128, of fp32 queries 84 to 128, and those of
// fp32 queries with more than eight heads and 129 elements 236 to 400 at 255.
// ---------------------------------------------------------------------------------------------

// a b + c of two pairs
template <typename T>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

// Nibbles i of both halves of a word, i = 0..3, less their zero points, times kStep<T>.  The lowest bits of a 16-bit number are a
// count of 2^-24 (fp16, eleven bits) or 2^-133 (bf16, eight): the subnormal numbers and the first normal ones.  So a nibble
// in the first place, or in the second 16-fold, is one without more than a mask.
template <typename T>
constexpr float kStep = 0x1p-6f;
template <>
constexpr float kStep<__half> = 0x1p-9f;
template <typename T>
__device__ __forceinline__ void differences(uint32_t (&r)[4], uint32_t w, uint32_t minus_zero) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr uint32_t kFirst = kHalf ? 0x78007800u : 0x7f007f00u, kSecond = kHalf ? 0x68006800u : 0x7d007d00u;  // 2^15 and 2^11, 2^127 and 2^123
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t u = w >> (4 * i);
        r[i] = fma2<T>(u & 0x000f000fu, kFirst, minus_zero);
        r[i + 1] = fma2<T>(u & 0x00f000f0u, kSecond, minus_zero);
    }
}
// Of two zero points, in the halves of z: -z kStep<T>, by way of 1024 + z or 128 + z.
template <typename T>
__device__ __forceinline__ uint32_t minus_zeros(uint32_t z) {
    if constexpr (std::is_same<T, __half>::value) return fma2<T>(0x64006400u + z, 0x98009800u, 0x40004000u);
    else return fma2<T>(0x43004300u + z, 0xbc80bc80u, 0x40004000u);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// An 8 x 8 matrix of 16-bit numbers, a row in four lanes, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}

// IO: queries and outputs; C: 32s of elements of a head, rounded up; G: of a group (C: there is one group); N: eights of
// query heads.
template <typename IO, int C, int G, int N>
struct NibbleCore {
    using Elem = IO;
    static constexpr bool kPacked = true, kScored = false;  // other scores are a branch here
    static constexpr int kWholeTiles = 3, kSwitch = 2;
    static constexpr bool kThree = sizeof(IO) == 4;         // parts of queries, and sums apart
    static constexpr bool kHalf = std::is_same<IO, __half>::value;
    using Q = typename std::conditional<kHalf, __half, __nv_bfloat16>::type;
    static constexpr int kParts = kThree ? 3 : 1, kWeightParts = kThree || kHalf ? 3 : 2;
    static constexpr int kKeys = 32, kRuns = 2;             // of a tile: two runs share what a tile costs besides its products
    static constexpr int kWarps = N == 1 || C <= 4 ? 8 : 4;  // whose sums fit an SM
    static constexpr int kBlocks = N == 1 && C <= 4 ? 2 : 1;
    static constexpr bool kWholeRows = true;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRows = 8 * N;
    static constexpr int kDim = C * kChunk;
    static constexpr int kBoxes = 0, kChunks = 0;
    static constexpr int kRunBytes = C * kChunkBytes + (C + G - 1) / G * kGroupBytes, kTileBytes = kRuns * kRunBytes;
    static constexpr int kPitch = (C * 4 + 1) * 16;         // of queries: an odd number of 16-byte chunks
    static constexpr bool kQueryInSmem = kThree || N * C > 8;
    static constexpr int kPartBytes = kRows * kPitch;
    static constexpr int kQueryBytes = kParts * kPartBytes;
    static constexpr int kWarpBytes = 0;
    static constexpr float kUnit = 0x1p-24f;                // weights and their parts are bf16 whatever IO is
    // Queries of the range of fp32 are taken 2^12 times smaller: 256 products with numbers up to 15, whose scale is yet to
    // come, then stay in it.
    static constexpr float kRoom = 8.0f;
    static constexpr float kQuery = kHalf ? 1.0f : 0x1p-12f, kScale = 1.0f / kQuery / kStep<Q>;
    // Columns are heads 8 j + 2 t + e, for which a lane keeps maximum and sum.
    uint32_t qb[kQueryInSmem ? 1 : C][N][4];
    float o[2 * C][N][4], m[N][2], l[N][2], slope[N][2];
    uint32_t query;
    int words, last;  // where a tile's words begin; the last group

    // Word w of a row's 32 elements holds two, this one and the fourth after it: word t, or 4 + t, of an instruction's eight is
    // what the lanes of column t multiply with their first, or second, register.
    static __device__ __forceinline__ int element(int w) { return 8 * (w % 4) + 2 * (w / 8) + w % 8 / 4; }

    static __device__ __forceinline__ void stage_query(const IO *q, int heads, int D, bool, bool, char *smem_q) {
        for (int e = threadIdx.x; e < kRows * kDim / 2; e += kThreads) {
            const int r = e / (kDim / 2), w = e - r * (kDim / 2), i = w / 16 * kChunk + element(w % 16);
            uint32_t *to = reinterpret_cast<uint32_t *>(smem_q + r * kPitch) + w;
            float x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = r < heads && i + 4 * h < D ? dev::widen(q[r * D + i + 4 * h]) * kQuery : 0.0f;
            if constexpr (kThree) {
                // Cut off, not rounded, so that the parts' sum is exact; a number that is not finite is its first part.
                uint32_t bits[2][3];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool finite = fabsf(x[h]) <= FLT_MAX;
#pragma unroll
                    for (int part = 0; part < 3; ++part) {
                        bits[h][part] = __float_as_uint(x[h]);
                        x[h] = finite ? x[h] - __uint_as_float(bits[h][part] & 0xffff0000u) : 0.0f;
                    }
                    if (!finite && (bits[h][0] & 0xffffu)) bits[h][0] |= 0x400000u;  // a NaN stays one
                }
#pragma unroll
                for (int part = 0; part < 3; ++part) to[part * (kPartBytes / 4)] = bits[0][part] >> 16 | (bits[1][part] & 0xffff0000u);
            } else {
                *to = pack2(dev::narrow<IO>(x[0]), dev::narrow<IO>(x[1]));
            }
        }
    }

    __device__ __forceinline__ void begin(char *smem_q, char *, const AttnArgs &a, const Scoring &sc) {
        const int t = threadIdx.x & 3;
        query = smem_addr(smem_q);
        words = (a.c.head_dim + kChunk - 1) / kChunk * kChunkBytes;
        last = (a.c.head_dim + a.c.group - 1) / a.c.group - 1;
        if constexpr (!kQueryInSmem) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < N; ++j) load_query(qb[c][j], c, j, 0);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                slope[j][e] = slope_of(sc, 8 * j + 2 * t + e);
                m[j][e] = -INFINITY;
                l[j][e] = 0.0f;
            }
#pragma unroll
            for (int n = 0; n < 2 * C; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][j][e] = 0.0f;
        }
    }

    // Eight heads' queries of 32 elements, for their two instructions.
    __device__ __forceinline__ void load_query(uint32_t (&r)[4], int c, int j, int part) const {
        const int lane = threadIdx.x & 31;
        ldmatrix4(r, query + part * kPartBytes + (8 * j + (lane & 7)) * kPitch + (4 * c + (lane >> 3)) * 16);
    }

    // Makes the words of values that do not count zeros: their weights are, and the words may hold anything.
    static __device__ __forceinline__ void clear(char *values, uint32_t live, const Cache &c) {
        const int lane = threadIdx.x & 31, first = (c.head_dim + kChunk - 1) / kChunk * kChunkBytes;
        uint32_t *word = reinterpret_cast<uint32_t *>(values + lane / 16 * kRunBytes + first) + lane % 16;
        const bool dead = !(live >> lane & 1);
#pragma unroll
        for (int k = 0; k < (C + G - 1) / G; ++k)
            if (dead && first + k * kGroupBytes < c.tile_bytes) word[k * kBlockSlots] = 0;
    }

    // Scores of a run's keys g (elements 0 and 1) and g + 8 (2 and 3), not scaled: of each group, then their sum.
    __device__ __forceinline__ void score(float (&s)[N][4], const char *ks) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        const uint32_t ka = smem_addr(ks) + lane * 16;
        float part[kParts][N][4] = {};
        uint32_t b[4], zero[2];
        float scale[2];
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c % G == 0) {
                const char *w = ks + words + min(c / G, last) * kGroupBytes + 4 * g;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t word = *reinterpret_cast<const uint32_t *>(w + 32 * h);
                    zero[h] = minus_zeros<Q>((word & 15u) * 0x10001u);
                    scale[h] = __uint_as_float(word & ~15u);
                }
            }
            if (c % 2 == 0) ldmatrix4(b, ka + c * kChunkBytes - (c + 1 == C ? (lane >> 4) * kChunkBytes : 0));
            uint32_t n[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) differences<Q>(n[h], b[2 * (c % 2) + h], zero[h]);
            const uint32_t a0[4] = {n[0][0], n[1][0], n[0][1], n[1][1]}, a1[4] = {n[0][2], n[1][2], n[0][3], n[1][3]};
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    uint32_t q[4];
                    if constexpr (kQueryInSmem) {
                        load_query(q, c, j, p);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) q[e] = qb[c][j][e];
                    }
                    mma16816<Q>(part[p][j], a0, q[0], q[1]);
                    mma16816<Q>(part[p][j], a1, q[2], q[3]);
                }
            if (c + 1 == C || (c + 1) % G == 0) {
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float sum = part[kParts - 1][j][e];
#pragma unroll
                        for (int p = kParts - 2; p >= 0; --p) sum += part[p][j][e];
#pragma unroll
                        for (int p = 0; p < kParts; ++p) part[p][j][e] = 0.0f;
                        s[j][e] = fmaf(sum, scale[e >> 1], s[j][e]);
                    }
            }
        }
    }

    // Adds a run's values: weights s with a group's scales, in parts, times the differences of its elements.
    __device__ __forceinline__ void add_values(const float (&s)[N][4], const char *vs) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const uint32_t va = smem_addr(vs) + lane * 16;
        uint32_t b[4], p[N][kWeightParts][2], zeros[2];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c % G == 0) {
                const char *w = vs + words + min(c / G, last) * kGroupBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint2 two = *reinterpret_cast<const uint2 *>(w + (8 * h + 2 * t) * 4);
                    zeros[h] = minus_zeros<__nv_bfloat16>((two.x & 15u) + ((two.y & 15u) << 16));
                    const float by = __uint_as_float(*reinterpret_cast<const uint32_t *>(w + (8 * h + g) * 4) & ~15u) * (kUnit / kStep<__nv_bfloat16>);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        float x = s[j][2 * h] * by, y = s[j][2 * h + 1] * by;
#pragma unroll
                        for (int k = 0; k < kWeightParts; ++k) {
                            const uint32_t two16 = pack_bf16(x, y);
                            p[j][k][h] = transposed(two16);
                            x -= low_of(two16);
                            y -= high_of(two16);
                        }
                    }
                }
            }
            if (c % 2 == 0) ldmatrix4_trans(b, va + c * kChunkBytes - (c + 1 == C ? (lane >> 4) * kChunkBytes : 0));
            uint32_t n[2][4];
            differences<__nv_bfloat16>(n[0], b[2 * (c % 2)], zeros[0]);
            differences<__nv_bfloat16>(n[1], b[2 * (c % 2) + 1], zeros[1]);
            const uint32_t a0[4] = {n[0][0], n[0][1], n[1][0], n[1][1]}, a1[4] = {n[0][2], n[0][3], n[1][2], n[1][3]};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if constexpr (kThree) {  // a run's products by themselves, small ones first: the long sum is rounded, not cut off
                    float sum[2][4] = {};
#pragma unroll
                    for (int k = kWeightParts - 1; k >= 0; --k) {
                        mma16816<__nv_bfloat16>(sum[0], a0, p[j][k][0], p[j][k][1]);
                        mma16816<__nv_bfloat16>(sum[1], a1, p[j][k][0], p[j][k][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[2 * c][j][e] += sum[0][e];
                        o[2 * c + 1][j][e] += sum[1][e];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < kWeightParts; ++k) {
                        mma16816<__nv_bfloat16>(o[2 * c][j], a0, p[j][k][0], p[j][k][1]);
                        mma16816<__nv_bfloat16>(o[2 * c + 1][j], a1, p[j][k][0], p[j][k][1]);
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void step(const char *ks, const char *vs, uint32_t live, const Scoring &sc, int first) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        float s[kRuns][N][4];
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
            score(s[r], ks + r * kRunBytes);
            if (sc.cap != 0.0f || sc.slopes) {
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][j][e] = score_of(sc, s[r][j][e], slope[j][e & 1], first + 16 * r + g + 8 * (e >> 1));
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[r][j][e] *= sc.scale2;
            }
        }
        if (live != 0xffffffffu) {
#pragma unroll
            for (int r = 0; r < kRuns; ++r)
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(live >> (16 * r + g + 8 * (e >> 1)) & 1)) s[r][j][e] = -INFINITY;
        }
        // Weights are relative to a score that is at most 2^kRoom below the largest so far: with eight heads a lane's maximum
        // grows in two steps of three, and taking all sums down each time cost more than the sums' range has to give.
        bool more = false;
        float top[N][2];
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[j][e] = fmaxf(fmaxf(s[0][j][e], s[0][j][2 + e]), fmaxf(s[1][j][e], s[1][j][2 + e]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top[j][e] = fmaxf(top[j][e], __shfl_xor_sync(0xffffffffu, top[j][e], d));
                more |= top[j][e] > m[j][e] + kRoom;
            }
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float now = fmaxf(top[j][e], m[j][e]), f = exp2_approx(m[j][e] - finite_base(now));
                    l[j][e] *= f;
                    m[j][e] = now;
#pragma unroll
                    for (int n = 0; n < 2 * C; ++n) {
                        o[n][j][e] *= f;
                        o[n][j][2 + e] *= f;
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = finite_base(m[j][e]);
#pragma unroll
                for (int r = 0; r < kRuns; ++r) {
                    s[r][j][e] = exp2_approx(s[r][j][e] - base);
                    s[r][j][2 + e] = exp2_approx(s[r][j][2 + e] - base);
                    l[j][e] += s[r][j][e] + s[r][j][2 + e];
                }
            }
#pragma unroll
        for (int r = 0; r < kRuns; ++r) add_values(s[r], vs + r * kRunBytes);
    }

    // This warp's sums [kRows][kDim], maxima and sums of weights [kRows] to shared memory.
    __device__ __forceinline__ void end(float *so, float *sm, float *sl) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int head = 8 * j + 2 * t + e;
                float sum = l[j][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (g == 0) {
                    sm[head] = m[j][e];
                    sl[head] = sum;
                }
#pragma unroll
                for (int c = 0; c < C; ++c)  // rows g and g + 8 of both instructions: elements 4 g .. 4 g + 3 of the 32
                    *reinterpret_cast<float4 *>(so + head * kDim + c * kChunk + 4 * g) =
                        make_float4(o[2 * c][j][e], o[2 * c][j][2 + e], o[2 * c + 1][j][e], o[2 * c + 1][j][2 + e]);
            }
    }
};

template <typename IO, int C, int G, int N>
AttnKernel nibble_kernel() {
    constexpr int kStages = 2;
    static_assert(AttnSmem<NibbleCore<IO, C, G, N>, kStages>::kBytes <= 227 * 1024, "fits an SM");
    return attn_kernel<NibbleCore<IO, C, G, N>, kStages>();
}

template <typename IO, int C, int N>
AttnKernel pick_group(int group) {
    if (group == 32) return nibble_kernel<IO, C, 1, N>();
    if (group == 64) return nibble_kernel<IO, C, 2, N>();
    if constexpr (C == 2) return nibble_kernel<IO, C, 2, N>();
    else return nibble_kernel<IO, C, C == 3 ? 3 : 4, N>();
}

template <typename IO, int N>
AttnKernel pick_nibbles(int D, int group) {
    if (D <= 64) return pick_group<IO, 2, N>(group);
    if (D <= 96) return pick_group<IO, 3, N>(group);
    if (D <= 128) return pick_group<IO, 4, N>(group);
    if (D <= 192) return pick_group<IO, 6, N>(group);
    return pick_group<IO, 8, N>(group);
}

// The kernel for one type of queries (a file each, which are compiled apart).
AttnKernel pick_kv4_half(int D, int group, int heads);
AttnKernel pick_kv4_bf16(int D, int group, int heads);
AttnKernel pick_kv4_float(int D, int group, int heads);

}  // namespace l2d

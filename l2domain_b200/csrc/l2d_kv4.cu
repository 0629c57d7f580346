// The paged cache in 4 bits: appending to it (l2d_kv4_append), and how the attention works on it.
//
// A page is cut into blocks of 16 slots; a block holds, head by head, a tile: for every 32 elements of the head 16 rows of
// 16 bytes (one per slot; element 2j in the low half of byte j), then for every group of elements 16 words.  So the
// attention's tile of 16 keys of one head is one run of bytes, which one bulk copy brings, already in the order in which
// eight rows of 16 bytes meet all banks.  A word is the bits of the group's scale with the zero point in the last
// four: scales have 20 significant bits, and a scale times a difference of two 4-bit numbers is exact in fp32.
#include "l2d_attn.cuh"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace l2d {

constexpr int kBlockSlots = 16;
constexpr int kChunk = 32;                           // elements of a row of 16 bytes
constexpr int kChunkBytes = kBlockSlots * 16;
constexpr int kGroupBytes = kBlockSlots * 4;

// ---------------------------------------------------------------------------------------------
// Appending.
//
// The same copy as to a cache of 16 or 32 bits, with a maximum and a minimum per group in between.  A thread has eight
// elements of a row (one word of nibbles), the threads of a row, a power of two of them, are neighbours in a warp and
// meet by shuffles; a thread keeps its angles for as many heads of its token as the grid leaves it.  Products,
// sums and quotients are rounded one by one to fp32, so that what is stored follows from the inputs and not from how an
// expression was compiled.
// ---------------------------------------------------------------------------------------------

constexpr int kAppend4Threads = 256;

struct Append4Args {
    AppendArgs a;
    void *k_out, *v_out;
};

// Eight elements from p on, of which those at d, d + 1, .. below D are real; by 16-byte words where WORDS.
template <typename T, bool WORDS>
__device__ __forceinline__ void load8(float (&x)[8], const T *p, int d, int D) {
    if constexpr (WORDS) {
        if (d < D) {
            const Pack<T, 8> r = load_pack<T, 8>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = dev::widen(r.v[i]);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = d + i < D ? dev::widen(p[i]) : 0.0f;
}
template <typename T, bool WORDS>
__device__ __forceinline__ void store8(T *p, const float (&x)[8], int d, int D) {
    if constexpr (WORDS) {
        Pack<T, 8> r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = dev::narrow<T>(x[i]);
        if (d < D) store_pack<T, 8>(p, r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (d + i < D) p[i] = dev::narrow<T>(x[i]);
    }
}

// lanes: threads of a row; the lanes * rows threads of a token take every rows-th of its heads.  WORDS: every row, and the
// second halves of rotated ones, on 16-byte boundaries, and angles too.
template <typename T, bool WORDS, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppend4Threads) k_append4(const __grid_constant__ Append4Args args, int lanes, int rows) {
    dev::wait_for_previous();
    const AppendArgs &a = args.a;
    const int D = a.c.head_dim, half = a.rot_dim / 2, hk = a.c.heads, heads = a.heads_q + 2 * hk;
    const int64_t thread = static_cast<int64_t>(blockIdx.x) * kAppend4Threads + threadIdx.x;
    const int64_t t = thread / (lanes * rows);
    if (t >= a.tokens) return;
    const int rest = static_cast<int>(thread - t * (lanes * rows)), row = rest / lanes, unit = rest - row * lanes, lane = threadIdx.x & 31;
    const unsigned mine = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1) << (lane & ~(lanes - 1));  // the threads of this row
    const int p = a.pos[t];
    if (p < 0) return;
    if (a.rot_dim && p >= a.max_pos) {
        if (rest == 0) report(a.c.status, L2D_KV_BAD_POSITION);
        return;
    }
    const int64_t page = page_of(a.c, a.seq ? a.seq[t] : t, p);
    if (page < 0) {
        if (rest == 0) report(a.c.status, L2D_KV_BAD_PAGE);
        return;
    }
    const int slot = p - static_cast<int>(page_index(a.c, p)) * a.c.page_size, inside = slot % kBlockSlots;
    const int chunks = (D + kChunk - 1) / kChunk, meet = min(a.c.group / 8, lanes), d = 8 * unit;
    const int64_t block = static_cast<int64_t>(slot / kBlockSlots) * hk * a.c.tile_bytes;
    const T *k = static_cast<const T *>(a.k) + t * a.k_token, *v = static_cast<const T *>(a.v) + t * a.v_token;
    const T *q = static_cast<const T *>(a.q) + t * a.q_token;
    T *q_out = static_cast<T *>(a.q_out) + t * a.q_out_token;

    // The angles of this thread's elements, and where the other elements of their pairs are: the second halves' angles
    // turn the other way.
    float cs[8], sn[8];
    int other = 0;
    if (d < a.rot_dim) {
        const float *cos = a.cos + static_cast<int64_t>(p) * half, *sin = a.sin + static_cast<int64_t>(p) * half;
        if constexpr (WORDS && !INTERLEAVED) {
            const bool second = d >= half;
            const Pack<float, 8> c8 = load_pack<float, 8>(cos + (second ? d - half : d)), s8 = load_pack<float, 8>(sin + (second ? d - half : d));
#pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = c8.v[i], sn[i] = second ? s8.v[i] : -s8.v[i];
            other = second ? -half : half;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = d + i;
                const bool in = e < a.rot_dim, second = INTERLEAVED ? e & 1 : e >= half;
                const int pair = INTERLEAVED ? e / 2 : second ? e - half : e;
                cs[i] = in ? cos[pair] : 1.0f;
                sn[i] = in ? (second ? sin[pair] : -sin[pair]) : 0.0f;
            }
        }
    }
    auto rotate = [&](float (&x)[8], const T *src) {  // src: this thread's elements
        float y[8];
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        } else if constexpr (WORDS) {
            load8<T, true>(y, src + other, 0, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = d + i;
                y[i] = e < a.rot_dim ? dev::widen(src[i + (e >= half ? -half : half)]) : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (d + i < a.rot_dim) x[i] = __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(y[i], sn[i]));
    };
    // Heads in order: queries, keys, values; a few at a time, loads first.
    constexpr int kHeads = 2;
    for (int h0 = row; h0 < heads; h0 += kHeads * rows) {
        float x[kHeads][8];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = h0 + j * rows, g = h - a.heads_q, w = g - hk;
            if (h >= heads) continue;
            const T *src = (g < 0 ? q + static_cast<int64_t>(h) * D : w < 0 ? k + static_cast<int64_t>(g) * D : v + static_cast<int64_t>(w) * D) + d;
            load8<T, WORDS>(x[j], src, d, D);
            if (w < 0 && d < a.rot_dim) rotate(x[j], src);
        }
        __syncwarp(mine);  // outputs may be the inputs
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = h0 + j * rows, g = h - a.heads_q, w = g - hk;
            if (h >= heads) continue;
            if (g < 0) {
                store8<T, WORDS>(q_out + static_cast<int64_t>(h) * D + d, x[j], d, D);
                continue;
            }
            float lo = 0.0f, hi = 0.0f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                lo = fminf(lo, x[j][i]);
                hi = fmaxf(hi, x[j][i]);
                bad |= !(fabsf(x[j][i]) <= FLT_MAX);
            }
            if (bad) hi = INFINITY;
            for (int m = 1; m < meet; m <<= 1) {
                lo = fminf(lo, __shfl_xor_sync(mine, lo, m));
                hi = fmaxf(hi, __shfl_xor_sync(mine, hi, m));
            }
            constexpr float kFifteenth = 1.0f / 15.0f;
            uint32_t word = (__float_as_uint(__fsub_rn(__fmul_rn(hi, kFifteenth), __fmul_rn(lo, kFifteenth))) + 15u) & ~15u;
            if (hi == INFINITY) word = 0x7fc00000u;
            const float s = __uint_as_float(word), by = word == 0 ? 1.0f : s;
            const float z = hi == INFINITY ? 0.0f : fminf(rintf(__fdiv_rn(-lo, by)), 15.0f);
            uint32_t nibbles = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // Of a group that is not a number every difference is 0.
                const float n = hi == INFINITY ? 0.0f : fminf(fmaxf(rintf(__fdiv_rn(x[j][i], by)) + z, 0.0f), 15.0f);
                if (d + i < D) nibbles |= static_cast<uint32_t>(n) << (4 * i);
                x[j][i] = s * (n - z);
            }
            char *tile = w < 0 ? a.c.k + page * a.c.k_page + block + static_cast<int64_t>(g) * a.c.tile_bytes
                               : a.c.v + page * a.c.v_page + block + static_cast<int64_t>(w) * a.c.tile_bytes;
            if (unit < 4 * chunks) *reinterpret_cast<uint32_t *>(tile + (unit / 4) * kChunkBytes + inside * 16 + (unit % 4) * 4) = nibbles;
            if (d < D && d % a.c.group == 0)
                *reinterpret_cast<uint32_t *>(tile + chunks * kChunkBytes + d / a.c.group * kGroupBytes + inside * 4) = word | static_cast<uint32_t>(z);
            T *out = static_cast<T *>(w < 0 ? args.k_out : args.v_out);
            if (out) store8<T, WORDS>(out + (w < 0 ? t * a.k_token + static_cast<int64_t>(g) * D : t * a.v_token + static_cast<int64_t>(w) * D) + d, x[j], d, D);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Attention: one warp's part of one head group, in the kernel that l2d_attn.cuh describes.
//
// Per 16 keys of 128 elements a warp reads 2 x 1088 bytes, which an SM's share of the memory brings in about 100 cycles,
// the issue of 400 instructions; so the conversion of 4096 nibbles is what has to be cheap.  A word of eight nibbles gives
// four registers of two 16-bit numbers each, by one mask that also sets the exponent of 2^10 (fp16) or 2^7 (bf16), and one
// subtraction that takes off this and the zero point together; the differences n - z are exact.  Scales stay outside
// the products: the scores of a group's elements are multiplied by its key's scale as fp32 sums, and weights by the
// value's scale before they are cut into 16-bit parts.
//
// Keys: a matrix of ldmatrix (8 keys x 16 bytes) gives a lane word t of key g, elements 8t .. 8t + 7 of the 32; queries are
// staged in the order in which two instructions meet them.  Values: the transposed load gives a lane the same four elements
// of keys 2t and 2t + 1 side by side, which is what a B operand needs of two neighbouring rows, nibble by nibble.
//
// Queries of 32 bits are three bf16 numbers that add up to them, and weights three; of 16 bits, weights two (2^-17 of
// a weight is left).
// ---------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t sub2_half(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// a / 16 + b
__device__ __forceinline__ uint32_t sixteenth_plus(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x2c002c00u), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t sub2_bf16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(b), "r"(0xbf80bf80u), "r"(a));
    return r;
}
// (w & mask) | bits
__device__ __forceinline__ uint32_t masked_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}

// Nibbles i of both halves of a word, i = 0..3, less their zero points.  T = bf16: zero holds 128 + z twice.
__device__ __forceinline__ void differences_bf16(uint32_t (&r)[4], uint32_t w, uint32_t zero) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = sub2_bf16(masked_or(w >> (4 * i), 0x000f000fu, 0x43004300u), zero);
}
// fp16: zero holds 1024 + z twice, and high -(64 + z): nibbles in the second place count 16-fold there.
__device__ __forceinline__ void differences_half(uint32_t (&r)[4], uint32_t w, uint32_t zero, uint32_t high) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t u = w >> (4 * i);
        r[i] = sub2_half(masked_or(u, 0x000f000fu, 0x64006400u), zero);
        r[i + 1] = sixteenth_plus(masked_or(u, 0x00f000f0u, 0x64006400u), high);
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// IO: queries and outputs; C: 32s of elements of a head, rounded up; SPLIT: groups of up to eight heads, whose other eight
// rows are the weights' second parts.
template <typename IO, int C, bool SPLIT>
struct NibbleCore {
    using Elem = IO;
    static constexpr bool kPacked = true, kScored = false;  // other scores are a branch here
    static constexpr int kWholeTiles = 6, kSwitch = 4;
    static constexpr bool kThree = sizeof(IO) == 4;         // parts of queries and weights
    static constexpr bool kHalf = std::is_same<IO, __half>::value;
    using Q = typename std::conditional<kHalf, __half, __nv_bfloat16>::type;
    static constexpr int kParts = kThree ? 3 : 1;
    static constexpr int kKeys = 16;
    static constexpr int kWarps = SPLIT || C <= 4 ? 8 : 4;  // whose sums fit an SM
    static constexpr int kBlocks = 1;
    static constexpr bool kWholeRows = true;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRows = SPLIT ? 8 : 16;
    static constexpr int kDim = C * kChunk;
    static constexpr int kBoxes = 0, kChunks = 0;
    static constexpr int kTileBytes = C * (kChunkBytes + kGroupBytes);
    static constexpr int kPitch = (C * 4 + 1) * 16;         // of queries: an odd number of 16-byte chunks
    static constexpr bool kQueryInSmem = kThree || (!SPLIT && C > 4);
    static constexpr int kPartBytes = kRows * kPitch;
    static constexpr int kQueryBytes = kParts * kPartBytes;
    static constexpr int kWarpBytes = 0;
    static constexpr float kUnit = 0x1p-24f;                // weights and their parts are bf16 whatever IO is
    // Queries of the range of fp32 are taken 2^12 times smaller: 256 products with numbers up to 15, whose scale is yet to
    // come, then stay in it.
    static constexpr float kQuery = kHalf ? 1.0f : 0x1p-12f, kScale = 1.0f / kQuery;
    uint32_t qa[kQueryInSmem ? 1 : 2 * C][SPLIT ? 2 : 4];
    float o[4 * C][4], m[2], l[2], slope[2];
    uint32_t query;
    int words, group_shift, groups;

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
        const int lane = threadIdx.x & 31;
        query = smem_addr(smem_q);
        words = (a.c.head_dim + kChunk - 1) / kChunk * kChunkBytes;
        group_shift = __ffs(a.c.group / kChunk) - 1;
        groups = (a.c.head_dim + a.c.group - 1) / a.c.group;
        for (int r = 0; r < (SPLIT ? 1 : 2); ++r) slope[r] = slope_of(sc, (lane >> 2) + 8 * r);
        if constexpr (!kQueryInSmem) {
#pragma unroll
            for (int c = 0; c < C; ++c) load_query(qa[2 * c], qa[2 * c + 1], c, 0);
        }
#pragma unroll
        for (int n = 0; n < 4 * C; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
    }

    // The queries of one 32 of elements, for its two instructions.
    template <int N>
    __device__ __forceinline__ void load_query(uint32_t (&x)[N], uint32_t (&y)[N], int c, int part) const {
        const int lane = threadIdx.x & 31;
        uint32_t r[4];
        if constexpr (SPLIT) {  // matrices of 8 heads x 8 elements
            ldmatrix4(r, query + part * kPartBytes + (lane & 7) * kPitch + (4 * c + (lane >> 3)) * 16);
            x[0] = r[0], x[1] = r[1], y[0] = r[2], y[1] = r[3];
        } else {
            const uint32_t at = query + part * kPartBytes + (((lane >> 3) & 1) * 8 + (lane & 7)) * kPitch + (lane >> 4) * 16 + c * 64;
            ldmatrix4(r, at);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = r[e];
            ldmatrix4(r, at + 32);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = r[e];
        }
    }
    template <typename T, int N>
    static __device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[N], uint32_t b0, uint32_t b1) {
        if constexpr (N == 2) {
            const uint32_t a4[4] = {a[0], 0, a[1], 0};
            mma16816<T>(c, a4, b0, b1);
        } else {
            mma16816<T>(c, a, b0, b1);
        }
    }

    // Makes the words of values that do not count zeros: their weights are, and the words may hold anything.
    static __device__ __forceinline__ void clear(char *values, uint32_t live, const Cache &c) {
        const int lane = threadIdx.x & 31;
        if (lane < kKeys && !(live >> lane & 1))
            for (int at = (c.head_dim + kChunk - 1) / kChunk * kChunkBytes; at < c.tile_bytes; at += kGroupBytes)
                *reinterpret_cast<uint32_t *>(values + at + 4 * lane) = 0;
    }

    __device__ __forceinline__ void step(const char *ks, const char *vs, uint32_t live, const Scoring &sc, int first) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const uint32_t ka = smem_addr(ks) + lane * 16, va = smem_addr(vs) + lane * 16;
        const int last = groups - 1;
        // Scores: of each group, then their sum over the groups, scaled.
        float s[2][4] = {}, part[2][4] = {};
        uint32_t b[4], zero[2], high[2];
        float2 scale[2];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c == 0 || (c & ((1 << group_shift) - 1)) == 0) {
                const char *w = ks + words + min(c >> group_shift, last) * kGroupBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t z = *reinterpret_cast<const uint32_t *>(w + (8 * h + g) * 4) & 15u;
                    zero[h] = (kHalf ? 0x64006400u : 0x43004300u) + z * 0x10001u;
                    high[h] = 0xd400d400u + z * 0x100010u;
                    const uint2 two = *reinterpret_cast<const uint2 *>(w + (8 * h + 2 * t) * 4);
                    scale[h] = make_float2(__uint_as_float(two.x & ~15u), __uint_as_float(two.y & ~15u));
                }
            }
            if (c % 2 == 0) ldmatrix4(b, ka + c * kChunkBytes - (c + 1 == C ? (lane >> 4) * kChunkBytes : 0));
            uint32_t n[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (kHalf) differences_half(n[h], b[2 * (c % 2) + h], zero[h], high[h]);
                else differences_bf16(n[h], b[2 * (c % 2) + h], zero[h]);
            }
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                uint32_t x[SPLIT ? 2 : 4], y[SPLIT ? 2 : 4];
                if constexpr (kQueryInSmem) {
                    load_query(x, y, c, p);
                } else {
#pragma unroll
                    for (int e = 0; e < (SPLIT ? 2 : 4); ++e) x[e] = qa[2 * c][e], y[e] = qa[2 * c + 1][e];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    multiply<Q>(part[h], x, n[h][0], n[h][1]);
                    multiply<Q>(part[h], y, n[h][2], n[h][3]);
                }
            }
            if (c + 1 == C || ((c + 1) & ((1 << group_shift) - 1)) == 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < (SPLIT ? 2 : 4); ++e) {
                        s[h][e] = fmaf(part[h][e], e & 1 ? scale[h].y : scale[h].x, s[h][e]);
                        part[h][e] = 0.0f;
                    }
            }
        }
        if (sc.cap != 0.0f || sc.slopes) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < (SPLIT ? 2 : 4); ++e) s[h][e] = score_of(sc, s[h][e], slope[e >> 1], first + h * 8 + 2 * t + (e & 1));
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < (SPLIT ? 2 : 4); ++e) s[h][e] *= sc.scale2;
        }
        if (live != (1u << kKeys) - 1) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < (SPLIT ? 2 : 4); ++e)
                    if (!(live >> (h * 8 + 2 * t + (e & 1)) & 1)) s[h][e] = -INFINITY;
        }
        // Weights, relative to the largest score so far.
#pragma unroll
        for (int r = 0; r < (SPLIT ? 1 : 2); ++r) {
            float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m2 = fmaxf(m[r], top), base = finite_base(m2);
            if (__any_sync(0xffffffffu, m2 != m[r])) {
                const float f = exp2_approx(m[r] - base);
                l[r] *= f;
#pragma unroll
                for (int n = 0; n < 4 * C; ++n) {
                    o[n][2 * r] *= f;
                    o[n][2 * r + 1] *= f;
                    if constexpr (SPLIT) {
                        o[n][2] *= f;
                        o[n][3] *= f;
                    }
                }
                m[r] = m2;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 2 * r; e < 2 * r + 2; ++e) s[h][e] = exp2_approx(s[h][e] - base);
            l[r] += (s[0][2 * r] + s[0][2 * r + 1]) + (s[1][2 * r] + s[1][2 * r + 1]);
        }
        // Values: weights with a group's scales, in parts, times the differences of its elements.
        uint32_t p[kThree ? 3 : 2][4], zeros[2];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c == 0 || (c & ((1 << group_shift) - 1)) == 0) {
                const char *w = vs + words + min(c >> group_shift, last) * kGroupBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint2 two = *reinterpret_cast<const uint2 *>(w + (8 * h + 2 * t) * 4);
                    zeros[h] = 0x43004300u + (two.x & 15u) + ((two.y & 15u) << 16);
                    const float sx = __uint_as_float(two.x & ~15u) * kUnit, sy = __uint_as_float(two.y & ~15u) * kUnit;
#pragma unroll
                    for (int r = 0; r < (SPLIT ? 1 : 2); ++r) {
                        float x = s[h][2 * r] * sx, y = s[h][2 * r + 1] * sy;
#pragma unroll
                        for (int k = 0; k < (kThree ? 3 : 2); ++k) {
                            const uint32_t two16 = pack_bf16(x, y);
                            x -= low_of(two16);
                            y -= high_of(two16);
                            // SPLIT: the first two parts in one instruction, a third in one of its own.
                            if (!SPLIT) p[k][r + 2 * h] = two16;
                            else if (k < 2) p[0][k + 2 * h] = two16;
                            else p[1][2 * h] = two16, p[1][1 + 2 * h] = 0;
                        }
                    }
                }
            }
            if (c % 2 == 0) ldmatrix4_trans(b, va + c * kChunkBytes - (c + 1 == C ? (lane >> 4) * kChunkBytes : 0));
            uint32_t n[2][4];
            differences_bf16(n[0], b[2 * (c % 2)], zeros[0]);
            differences_bf16(n[1], b[2 * (c % 2) + 1], zeros[1]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < (SPLIT ? (kThree ? 2 : 1) : (kThree ? 3 : 2)); ++k)
                    mma16816<__nv_bfloat16>(o[4 * c + i], p[k], n[0][i], n[1][i]);
        }
    }

    // This warp's sums [kRows][kDim], maxima and sums of weights [kRows] to shared memory.
    __device__ __forceinline__ void end(float *so, float *sm, float *sl) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int r = 0; r < (SPLIT ? 1 : 2); ++r) {
            float sum = l[r] + __shfl_xor_sync(0xffffffffu, l[r], 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (t == 0) {
                sm[g + 8 * r] = m[r];
                sl[g + 8 * r] = sum;
            }
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // columns 2t + e: elements 4 (2t + e) .. + 3 of the 32
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = o[4 * c + i][2 * r + e] + (SPLIT ? o[4 * c + i][2 + e] : 0.0f);
                    *reinterpret_cast<float4 *>(so + (g + 8 * r) * kDim + c * kChunk + 4 * (2 * t + e)) = make_float4(v[0], v[1], v[2], v[3]);
                }
        }
    }
};

template <typename IO, int C, bool SPLIT>
AttnKernel nibble_kernel() {
    constexpr int kStages = 4;
    static_assert(AttnSmem<NibbleCore<IO, C, SPLIT>, kStages>::kBytes <= 227 * 1024, "fits an SM");
    return attn_kernel<NibbleCore<IO, C, SPLIT>, kStages>();
}

template <typename IO, bool SPLIT>
AttnKernel pick_nibbles(int D) {
    if (D <= 64) return nibble_kernel<IO, 2, SPLIT>();
    if (D <= 96) return nibble_kernel<IO, 3, SPLIT>();
    if (D <= 128) return nibble_kernel<IO, 4, SPLIT>();
    if (D <= 192) return nibble_kernel<IO, 6, SPLIT>();
    return nibble_kernel<IO, 8, SPLIT>();
}

AttnKernel pick_attn_kv4(int dtype, int D, int G) {
    if (dtype == L2D_F16) return G <= 8 ? pick_nibbles<__half, true>(D) : pick_nibbles<__half, false>(D);
    if (dtype == L2D_BF16) return G <= 8 ? pick_nibbles<__nv_bfloat16, true>(D) : pick_nibbles<__nv_bfloat16, false>(D);
    return G <= 8 ? pick_nibbles<float, true>(D) : pick_nibbles<float, false>(D);
}

int check_cache4(const l2d_kv4_cache *cache, Cache *c) {
    if (!cache) return set_error(L2D_ERR_INVALID, "null cache");
    const l2d_kv4_cache &k = *cache;
    int64_t page = 0;
    int st = l2d_kv4_page_bytes(k.heads, k.head_dim, k.page_size, k.group, &page);
    if (st != L2D_OK) return st;
    // The rest is checked as of a cache of bytes whose pages are one row.
    l2d_kv_cache plain = {};
    plain.k = k.k;
    plain.v = k.v;
    plain.dtype = k.dtype;
    plain.heads = k.heads;
    plain.head_dim = k.head_dim;
    plain.page_size = k.page_size;
    plain.num_pages = k.num_pages;
    plain.table = k.table;
    plain.table_stride = k.table_stride;
    plain.num_seqs = k.num_seqs;
    plain.table_width = k.table_width;
    plain.status = k.status;
    plain.device = k.device;
    st = check_cache(&plain, c);
    if (st != L2D_OK) return st;
    c->k_page = k.k_page ? k.k_page : page;
    c->v_page = k.v_page ? k.v_page : page;
    if (c->k_page < page || c->v_page < page || c->k_page % 16 || c->v_page % 16)
        return set_error(L2D_ERR_INVALID, "pages are %lld and %lld bytes apart: at least %lld, and a multiple of 16", static_cast<long long>(c->k_page),
                         static_cast<long long>(c->v_page), static_cast<long long>(page));
    if (std::max(c->k_page, c->v_page) > (int64_t(1) << 31)) return set_error(L2D_ERR_INVALID, "cache strides too large");
    if (misaligned(k.k, 16) || misaligned(k.v, 16)) return set_error(L2D_ERR_INVALID, "keys and values in 4 bits must be aligned to 16 bytes");
    c->group = k.group;
    c->tile_bytes = static_cast<int>(page / (k.page_size / kBlockSlots) / k.heads);
    return L2D_OK;
}

}  // namespace l2d

using namespace l2d;

extern "C" {

int l2d_kv4_page_bytes(int heads, int head_dim, int page_size, int group, int64_t *bytes) {
    if (!bytes) return set_error(L2D_ERR_INVALID, "null pointer");
    if (heads < 1 || heads > 65535) return set_error(L2D_ERR_INVALID, "%d key-value heads", heads);
    if (head_dim < 1 || head_dim > kMaxHeadDim) return set_error(L2D_ERR_UNSUPPORTED, "head_dim %d: 1 to %d are supported", head_dim, kMaxHeadDim);
    if (page_size < kBlockSlots || page_size % kBlockSlots)
        return set_error(L2D_ERR_UNSUPPORTED, "pages of %d slots: a cache in 4 bits takes multiples of %d", page_size, kBlockSlots);
    if (group != 32 && group != 64 && group != 128) return set_error(L2D_ERR_UNSUPPORTED, "groups of %d elements: 32, 64 and 128 are supported", group);
    const int tile = (head_dim + kChunk - 1) / kChunk * kChunkBytes + (head_dim + group - 1) / group * kGroupBytes;
    *bytes = int64_t(page_size / kBlockSlots) * heads * tile;
    return L2D_OK;
}

int l2d_kv4_append(const l2d_kv4_cache *cache, const l2d_append_desc *desc, const void *k, const void *v, const void *q, void *q_out, void *k_out,
                   void *v_out, const int32_t *pos, const int32_t *seq, int64_t tokens, void *stream) {
    Append4Args args = {};
    AppendArgs &a = args.a;
    int st = check_cache4(cache, &a.c);
    if (st != L2D_OK) return st;
    st = check_append(desc, cache->dtype, cache->heads, cache->head_dim, cache->num_seqs, k, v, q, q_out, pos, seq, tokens, &a);
    if (st != L2D_OK || tokens == 0) return st;
    const int eb = elem_bytes(cache->dtype), D = cache->head_dim, half = a.rot_dim / 2;
    if (misaligned(k_out, eb) || misaligned(v_out, eb)) return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    int sms = 0;
    st = device_sms(cache->device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(cache->device);
    L2D_CUDA_TRY(on.err);
    args.k_out = k_out;
    args.v_out = v_out;
    // Eight elements of 16 bits, or half as many of 32, are a word; halves of heads are whole runs of eight or interleaved.
    const int64_t each = 8, in_words = 16 / eb;
    const bool words = D % each == 0 && a.rot_dim % each == 0 && (desc->interleaved || half % each == 0) && a.k_token % in_words == 0 &&
                       a.v_token % in_words == 0 && a.q_token % in_words == 0 && a.q_out_token % in_words == 0 && !misaligned(k, 16) &&
                       !misaligned(v, 16) && !misaligned(q, 16) && !misaligned(q_out, 16) && !misaligned(k_out, 16) && !misaligned(v_out, 16) &&
                       (desc->interleaved || (!misaligned(a.cos, 16) && !misaligned(a.sin, 16)));
    int lanes = 4;  // of a row, so that its groups meet by shuffles
    while (lanes * 8 < D) lanes *= 2;
    // Heads of a token in one thread: all of them, or as few as it takes for four blocks a SM.
    const int heads = desc->heads_q + 2 * cache->heads;
    const int64_t want = int64_t(sms) * 4 * kAppend4Threads, have = tokens * lanes;
    const int rows = static_cast<int>(std::min<int64_t>(heads, std::max<int64_t>(1, (want + have - 1) / have)));
    const int64_t blocks = (have * rows + kAppend4Threads - 1) / kAppend4Threads;
    if (blocks > INT32_MAX) return set_error(L2D_ERR_INVALID, "%lld tokens are too many", static_cast<long long>(tokens));
    auto pick = [&](auto type) {
        using T = decltype(type);
        if (words) return desc->interleaved ? k_append4<T, true, true> : k_append4<T, true, false>;
        return desc->interleaved ? k_append4<T, false, true> : k_append4<T, false, false>;
    };
    auto kernel = cache->dtype == L2D_F32 ? pick(float()) : cache->dtype == L2D_F16 ? pick(__half()) : pick(__nv_bfloat16());
    L2D_CUDA_TRY(launch(kernel, dim3(static_cast<unsigned>(blocks)), kAppend4Threads, 0, stream, args, lanes, rows));
    return L2D_OK;
}

}  // extern "C"

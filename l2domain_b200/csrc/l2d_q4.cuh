// The kernel of matrix-vector products with 4-bit weights and group scales.
//
//   y[b][i] = sum_j s[i][j / g] * (q[i][j] - z[i][j / g]) * x[b][j]
//
// Memory bound: a weight is half a byte and is used once per vector.  At the bandwidth of HBM an SM
// gets about 52 weights a cycle and has 128 lanes to treat them (64 of them for logic), so a weight may
// cost little over two instructions; a fused multiply-add in fp32 with its conversion would be three or
// four.  So the products run on matrix instructions, 16 rows of weights as the A operand and the vectors
// as columns of B, and everything else is arranged to spend next to nothing per weight:
//
//  * Few vectors are multiplied in integers (m16n8k32, bytes): two masks and a shift turn eight nibbles into
//    bytes.  x of each 128 columns is a 30-bit integer times a power of two, in four signed digits of 8 bits, a
//    column of B each, and one of fp32 a 60-bit integer in eight.  x is exact, and so are sums up to the end of a group.
//  * More vectors are multiplied in fp16 with fp32 sums (m16n8k16), one column a vector.  The difference q - z is
//    taken first, exactly, from 1024 + q and 1024 + z, because sum q x and z sum x may nearly cancel: where the largest
//    x meets a weight of zero, or a row has few others, their difference has few right bits left.  (A nibble masked
//    into the low mantissa bits of an fp16 number is exact as it is, and two instructions less for every two weights:
//    8 vectors 28672 x 8192 on groups of 128 took 42 us so, and take 47 with the differences.)  A mask higher up
//    gives 16 (q - z), with a sixteenth of x.  Each 128 columns of a vector are scaled by a power of two to a largest
//    value just under 2^15.
//  * fp32 vectors take two columns of fp16, 11 bits each and a sign between them: the last of 24 bits of x may be lost.
//  * Infinities and NaNs, and values so far below the largest of their 128 columns that the scaled number loses bits of
//    them, are staged as zeros, and the threads that store a vector's results add their terms at the end.  In fp16 that
//    is what is below 2^-23 of the largest (fp32), or below 2^-24 of it with bits that would be lost (16-bit vectors); in
//    integers, below 2^-36 (fp32), 2^-19 (fp16) or 2^-22 (bf16) of it with such bits.
//  * The scales are applied to the fp32 sums of each group.  One instruction sums over the four lanes of a
//    row, 128 columns; where groups are shorter, x of the different groups goes to different columns of B
//    (zeros elsewhere), so that each group still has a sum of its own: S = 128 / group columns per part.
//  * A lane's 16 bytes (32 columns of one row) are loaded straight into registers from the row-major
//    weights, a step of 512 columns ahead, in code without branches.  A product's order of columns is free,
//    so nibbles are used in the order in which masks deliver them, and x is put into that order when it is
//    staged.  A request for eight rows occupies the L1 for eight cycles whatever its width, so the scales of
//    a whole step are loaded as one word per row.  Up to 16 columns of B that fits the 128 registers that 16 warps leave,
//    but for a few words; with 17 to 32 of them 44 to 440 bytes of a thread go to local memory.
//  * A block's rows are its even share of M, in tiles of at most 16 rows of nearly equal size, so that
//    blocks finish together whatever M is; groups of its warps take a tile each, split its columns and
//    meet in shared memory at its end, in a fixed order.
//  * Where a block has few rows, or there are many vectors, staging x costs more than multiplying: a cluster
//    of blocks then takes its rows together, each block a share of the columns, and adds its sums over
//    distributed shared memory, in rank order (q4_shape() weighs it; 8 vectors of 8192 x 8192 on groups of 32:
//    37 us alone, 28.5 in pairs, 27.5 in fours).
#pragma once

#include "l2d_launch.cuh"

#include <cooperative_groups.h>

#include <cstring>

namespace l2d {

struct Q4Args {
    const uint8_t *W;
    const uint8_t *scales;
    const uint8_t *zeros;
    const void *x;
    void *y;
    int64_t M, ldw, lds, stride_x, stride_y;
    int N, vectors, dtype_x, dtype_y, dtype_s;
    int warps_k;     // warps that split a tile's columns
    int ranks;       // blocks of a cluster, which split the columns
    int stage_h;     // halves of 128 columns of x staged at a time
    int y_rows;      // rows of the block's sums kept (0: one staging and no cluster)
    int wide;        // scales and zeros of a step as one word
    // ceil(2^40 / (group / 128)): a half's group without a division.  On a 16-byte boundary, because the kernels come out
    // 2 to 5 % slower with it on another one of 8 (28672 x 8192: 28.0 us and 27.2, 16 vectors 77.7 and 72.2).
    alignas(16) uint64_t per_group;
};

constexpr int kQ4Warps = 16;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4Half = 128;       // columns of one sum: 64 bytes of each row
constexpr int kQ4Deep = 4;         // of them in a step, which a warp has in registers or on their way
constexpr int kQ4Rows = 16;
constexpr int kQ4MaxRows = 896;    // rows of a block, at most
// Bytes between columns of x in shared memory: 256 used (128 by bytes), and 64 so that two lie in other banks.
__host__ __device__ constexpr int q4_column(bool bytes) { return bytes ? 192 : 320; }

// Byte offsets in dynamic shared memory: x, its sums and factors, offsets of scales, marks of what of x is left out
// (16 bytes for 128 columns of a vector), the warps' sums, y.
struct Q4Smem {
    int sums, offsets, marks, red, y, bytes;
};
__host__ __device__ inline Q4Smem q4_smem(int tiles_n, bool bytes, int vectors, int parts, int stage_h, int y_floats) {
    Q4Smem s;
    s.sums = vectors * parts * stage_h * q4_column(bytes);
    s.offsets = s.sums + stage_h * 8 * tiles_n * 8;
    s.marks = s.offsets + (stage_h + 3) / 4 * 16;
    s.red = s.marks + vectors * stage_h * 16;
    s.y = s.red + (tiles_n == 1 ? 2 : 1) * kQ4Warps * kQ4Rows * 8 * tiles_n * 4;
    s.bytes = s.y + y_floats * 4;
    return s;
}

// c = a b, and c += a b.
__device__ __forceinline__ void q4_mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void q4_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c += a b in integers: a unsigned, b signed bytes, 32 columns.
__device__ __forceinline__ void q4_mma_bytes(uint32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes of shared memory where `real`; v stays as it is elsewhere.
__device__ __forceinline__ void load_if(uint4 &v, const char *p, bool real) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %5, 0;\n@p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
        : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
        : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(static_cast<uint32_t>(real)));
}

__device__ __forceinline__ uint32_t sub_half2(uint32_t a, uint32_t b) {
    __half2 x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    x = __hsub2(x, y);
    memcpy(&a, &x, 4);
    return a;
}

// Eight nibbles as fp16 numbers, p[i] nibbles i and i + 4: q - z, and 16 (q - z) in p[1] and p[3].
__device__ __forceinline__ void unpack_less(uint32_t w, uint32_t z, uint32_t (&p)[4]) {
    const uint32_t lo = (0x6400 | z) * 0x10001u, hi = (0x6400 | z << 4) * 0x10001u;  // 1024 + z, 1024 + 16 z
    p[0] = sub_half2((w & 0x000F000F) | 0x64006400, lo);
    p[1] = sub_half2((w & 0x00F000F0) | 0x64006400, hi);
    w >>= 8;
    p[2] = sub_half2((w & 0x000F000F) | 0x64006400, lo);
    p[3] = sub_half2((w & 0x00F000F0) | 0x64006400, hi);
}

__device__ __forceinline__ uint4 load_weights(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Of x, by ordinary loads: the kernel before may still have been writing it when this one's blocks became resident, so
// it is no read-only data.
__device__ __forceinline__ uint4 load_words(const char *p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_word(const char *p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_short(const char *p) {
    uint16_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}

// 16 bytes at any address, of which `left` belong to the row (zeros after them), inside [begin, end): from the
// two aligned ones around them where those are inside too, else byte by byte.
__device__ __forceinline__ uint4 load_any(const uint8_t *p, int left, const uint8_t *begin, const uint8_t *end) {
    if (left >= 16 && p >= begin + 16 && p + 32 <= end) {
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15;
        const uint4 *q = reinterpret_cast<const uint4 *>(p - off);
        const uint4 a = __ldg(q), b = off ? __ldg(q + 1) : a;
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (off & 8) {
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
        }
        if (off & 4) {
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
        }
        const uint32_t s = (off & 3) * 8;
        return make_uint4(__funnelshift_r(w[0], w[1], s), __funnelshift_r(w[1], w[2], s), __funnelshift_r(w[2], w[3], s),
                          __funnelshift_r(w[3], w[4], s));
    }
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < left) v[i >> 2] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// What a warp holds of 128 columns of a tile: this lane's 16 bytes of rows g and g + 8.
struct Q4Part {
    uint4 w[2];
};
// And of a step of four such halves: the scales and zeros of its columns 2t, 2t + 1 of C for both rows, as
// stored.  Two to a word (zeros: bytes); S = 0: those of the first and of the last half.
template <int S, bool ZEROS>
struct Q4Scales {
    uint32_t s[2][S > 1 ? 4 : 2];
    uint32_t z[2][!ZEROS ? 1 : S == 4 ? 4 : 2];
    int from;  // S = 0: the first half whose scale is the last one's
};

__device__ __forceinline__ float scale_value(uint32_t word, bool high, bool is_half) {
    const float wide = __uint_as_float(high ? word & 0xffff0000u : word << 16);
    return is_half ? __half2float(__ushort_as_half(static_cast<unsigned short>(high ? word >> 16 : word))) : wide;
}

// S: columns of B per part of a vector (4, 2, 1 for groups of 32, 64, 128 columns), 0 for longer groups.
// WORDS: every row of W is whole 16-byte words on 16-byte boundaries, and the 16-bit scales (and zeros) of a step
// can be read in words.
// KIND: how products are taken, in fp16 or by bytes, and whether vectors have 16 or 32 bits.
enum Q4Kind { kQ4Half16, kQ4Half32, kQ4Bytes16, kQ4Bytes32 };
// Columns of x per vector.
__host__ __device__ constexpr int q4_parts(Q4Kind kind) { return kind == kQ4Bytes32 ? 8 : kind == kQ4Bytes16 ? 4 : kind == kQ4Half32 ? 2 : 1; }
template <int NT, int S, bool ZEROS, bool WORDS, Q4Kind KIND>
__global__ void __launch_bounds__(kQ4Threads, 1) k_q4_gemv(Q4Args a) {
    constexpr bool BYTES = KIND == kQ4Bytes16 || KIND == kQ4Bytes32, FP32 = KIND == kQ4Half32 || KIND == kQ4Bytes32;
    constexpr int PARTS = q4_parts(KIND);
    constexpr int SUB = S > 1 ? S : 1, kShift = S == 4 ? 2 : S == 2 ? 1 : 0, E = S > 1 ? 2 : 1, kColumn = q4_column(BYTES);
    constexpr float kUnit = BYTES ? 0x1p16f : 0x1p12f;  // of the sums: those of (q - z) x may pass the range before their scale
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in all lanes
    const int columns = a.vectors * PARTS;                 // of x in shared memory
    const Q4Smem lay = q4_smem(NT, BYTES, a.vectors, PARTS, a.stage_h, a.y_rows * a.vectors);
    float2 *sums = reinterpret_cast<float2 *>(smem + lay.sums);
    int *offsets = reinterpret_cast<int *>(smem + lay.offsets);
    uint8_t *marks = reinterpret_cast<uint8_t *>(smem + lay.marks);
    float *red = reinterpret_cast<float *>(smem + lay.red), *ysum = reinterpret_cast<float *>(smem + lay.y);
    // This block's rows, and its halves of 128 columns.
    const int shares = gridDim.x / a.ranks, share = blockIdx.x / a.ranks, rank = blockIdx.x % a.ranks;
    const int64_t r0 = a.M * share / shares;
    const int rows = static_cast<int>(a.M * (share + 1) / shares - r0);
    const int all_h = (a.N + kQ4Half - 1) / kQ4Half, all_steps = (all_h + kQ4Deep - 1) / kQ4Deep;
    const int h_lo = static_cast<int>(static_cast<int64_t>(all_steps) * rank / a.ranks) * kQ4Deep;
    const int h_hi = min(all_h, static_cast<int>(static_cast<int64_t>(all_steps) * (rank + 1) / a.ranks) * kQ4Deep);
    // This warp's group: its rows, in tiles of q or q + 1 rows.
    const int wk = warp & (a.warps_k - 1), wm = warp / a.warps_k, warps_m = kQ4Warps / a.warps_k;
    const int g0 = rows * wm / warps_m, g_rows = rows * (wm + 1) / warps_m - g0;
    const int tiles = (g_rows + kQ4Rows - 1) / kQ4Rows, tile_q = tiles ? g_rows / tiles : 0, tile_rest = g_rows - tiles * tile_q;
    auto first_row = [&](int tile) { return g0 + tile * tile_q + min(tile, tile_rest); };
    const int row_bytes = (a.N + 1) / 2;
    const uint8_t *w_end = a.W + (a.M - 1) * a.ldw + row_bytes;
    // The group of a column: group / 128 is 1 or more, or groups are 32 or 64 columns.
    auto group_of = [&](int col) {
        return S > 1 ? col >> (7 - kShift) : static_cast<int>(static_cast<uint64_t>(col >> 7) * a.per_group >> 40);
    };
    dev::wait_for_previous();

    // The column of x that this lane feeds into column g of each n-tile: part (8 n + g) / S, if the lane's columns
    // of W belong to that column's subgroup.  b stays zero where it feeds none.
    constexpr int kAhead = NT == 1 ? 2 : 1;
    bool feeds[NT];
    uint4 b[NT][kAhead];
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        feeds[n] = (g & (SUB - 1)) == (t * SUB >> 2) && ((8 * n + g) >> kShift) < columns;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) b[n][e] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
    }
    const char *x_lane = smem + (g >> kShift) * kColumn + t * 16;
    const int x_half = columns * kColumn;
    const bool is_half = a.dtype_s == L2D_F16;

    // Adds the products of half `half` of the staging: scales s and zeros z of [row][column of C].
    auto multiply = [&](const Q4Part &part, int half, const float (&s)[2][E], const uint32_t (&z)[2][E]) {
        const uint32_t w0[4] = {part.w[0].x, part.w[0].y, part.w[0].z, part.w[0].w}, w1[4] = {part.w[1].x, part.w[1].y, part.w[1].z, part.w[1].w};
        float sum[NT][4];
        const char *x = x_lane + half * x_half;
        if constexpr (BYTES) {
            // Sums of products of bytes, on top of the bits of 1.5 * 2^23: as a float they are that much more.
            uint32_t c[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0x4b400000u;
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const uint32_t a0[4] = {w0[j] & 0x0F0F0F0F, w1[j] & 0x0F0F0F0F, w0[j] >> 4 & 0x0F0F0F0F, w1[j] >> 4 & 0x0F0F0F0F};
                const uint32_t a1[4] = {w0[j + 1] & 0x0F0F0F0F, w1[j + 1] & 0x0F0F0F0F, w0[j + 1] >> 4 & 0x0F0F0F0F, w1[j + 1] >> 4 & 0x0F0F0F0F};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint4 &bb = b[n][j / 2 % kAhead];
                    load_if(bb, x + n * (8 >> kShift) * kColumn + j * 32, feeds[n]);
                    q4_mma_bytes(c[n], a0, bb.x, bb.y);
                    q4_mma_bytes(c[n], a1, bb.z, bb.w);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[n][e] = __uint_as_float(c[n][e]);
        } else {
            uint32_t z0 = z[0][0], z1 = z[1][0];  // of this lane's own columns, which the lane of their subgroup's sum has
            if constexpr (ZEROS && S > 1) {
                const int own = t * SUB >> 2, from = (lane & ~3) | own >> 1;
                uint32_t v[2][2];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e / 2][e % 2] = __shfl_sync(0xffffffffu, z[e / 2][e % E], from);
                z0 = v[0][own & 1];
                z1 = v[1][own & 1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t p0[4], p1[4];
                unpack_less(w0[j], z0, p0);
                unpack_less(w1[j], z1, p1);
                const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint4 &bb = b[n][j % kAhead];
                    load_if(bb, x + n * (8 >> kShift) * kColumn + j * 64, feeds[n]);
                    if (j == 0) q4_mma_first(sum[n], a0, bb.x, bb.y);
                    else q4_mma(sum[n], a0, bb.x, bb.y);
                    q4_mma(sum[n], a1, bb.z, bb.w);
                }
            }
        }
        const float4 *xs = reinterpret_cast<const float4 *>(sums + half * 8 * NT) + t;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float4 f = xs[4 * n];  // sum and factor of columns 2t and 2t + 1
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // By bytes all of this is integers below 2^24, and exact (without zeros the sum is 8 of it and the bias).
                const float xsum = e & 1 ? f.z : f.x;
                const float v = BYTES ? sum[n][e] - (ZEROS ? fmaf(static_cast<float>(z[e >> 1][(e & 1) % E]), xsum, 12582912.0f) : xsum) : sum[n][e];
                acc[n][e] = fmaf(s[e >> 1][(e & 1) % E], v * fabsf(e & 1 ? f.w : f.y), acc[n][e]);
            }
        }
    };
    // Half h of a step.
    auto multiply_of = [&](const Q4Part &c, const Q4Scales<S, ZEROS> &q, int h, int half) {
        float s[2][E];
        uint32_t z[2][E];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const bool second = S == 0 && h >= q.from;
            const uint32_t word = S == 0 ? (second ? q.s[r][1] : q.s[r][0]) : q.s[r][S == 1 ? h / 2 : h];
#pragma unroll
            for (int e = 0; e < E; ++e) s[r][e] = scale_value(word, S == 1 ? h & 1 : e, is_half);
            uint32_t zeros = 0;
            if constexpr (ZEROS) zeros = S == 0 ? (second ? q.z[r][1] : q.z[r][0]) : S == 1 ? q.z[r][h / 2] >> (8 * (h & 1)) : S == 2 ? q.z[r][h / 2] >> (16 * (h & 1)) : q.z[r][h];
#pragma unroll
            for (int e = 0; e < E; ++e) z[r][e] = ZEROS ? zeros >> (8 * e) & 15 : 8;
        }
        multiply(c, half, s, z);
    };

    // Where this lane reads: rows g and g + 8 of a tile, or the tile's last row where it has fewer (their sums are
    // dropped), from half `half` of all on.
    struct Rows {
        const uint8_t *w[2], *s[2], *z[2];
    };
    // Scales of the columns 2t, 2t + 1 of C, which belong to the subgroups (2t) % S and (2t + 1) % S.
    const int sub = S == 4 ? (2 * t) & 3 : 0;
    auto rows_of = [&](int tile, int half) {
        Rows at;
        const int last = first_row(tile + 1) - 1, lo = first_row(tile);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t row = r0 + min(lo + g + 8 * r, last), first = S ? half * SUB + sub : 0;
            at.w[r] = a.W + row * a.ldw + half * 64 + 16 * t;
            at.s[r] = a.scales + (row * a.lds + first) * 2;
            at.z[r] = ZEROS ? a.zeros + row * a.lds + first : nullptr;
        }
        return at;
    };
    auto load = [&](Q4Part &c, const Rows &at, int h) {
#pragma unroll
        for (int r = 0; r < 2; ++r) c.w[r] = load_weights(at.w[r] + h * 64);
    };
    // The scales of the step from half `half` of the staging on.
    auto load_scales = [&](Q4Scales<S, ZEROS> &q, const Rows &at, int half) {
        const int first = S == 0 ? offsets[half] : 0, last = S == 0 ? offsets[half + kQ4Deep - 1] : 0;
        if (S == 0) q.from = offsets[half + 1] != first ? 1 : offsets[half + 2] != first ? 2 : 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if constexpr (S == 0) {
                q.s[r][0] = __ldg(reinterpret_cast<const uint16_t *>(at.s[r]) + first);
                q.s[r][1] = __ldg(reinterpret_cast<const uint16_t *>(at.s[r]) + last);
                if constexpr (ZEROS) q.z[r][0] = __ldg(at.z[r] + first), q.z[r][1] = __ldg(at.z[r] + last);
            } else if constexpr (S == 1) {
                if (a.wide) {
                    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(at.s[r]));
                    q.s[r][0] = v.x, q.s[r][1] = v.y;
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) q.s[r][i] = __ldg(reinterpret_cast<const uint32_t *>(at.s[r]) + i);
                }
                if constexpr (ZEROS) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) q.z[r][i] = __ldg(reinterpret_cast<const uint16_t *>(at.z[r]) + i);
                }
            } else if constexpr (S == 2) {
                if (a.wide) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(at.s[r]));
                    q.s[r][0] = v.x, q.s[r][1] = v.y, q.s[r][2] = v.z, q.s[r][3] = v.w;
                    if constexpr (ZEROS) {
                        const uint2 u = __ldg(reinterpret_cast<const uint2 *>(at.z[r]));
                        q.z[r][0] = u.x, q.z[r][1] = u.y;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(at.s[r]) + i);
                        q.s[r][2 * i] = v.x, q.s[r][2 * i + 1] = v.y;
                        if constexpr (ZEROS) q.z[r][i] = __ldg(reinterpret_cast<const uint32_t *>(at.z[r]) + i);
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < kQ4Deep; ++h) {
                    q.s[r][h] = __ldg(reinterpret_cast<const uint32_t *>(at.s[r]) + 2 * h);
                    if constexpr (ZEROS) q.z[r][h] = __ldg(reinterpret_cast<const uint16_t *>(at.z[r]) + 2 * h);
                }
            }
        }
    };
    // One half by itself, whatever its alignment, and be it the last one of a row that is not whole: fewer bytes,
    // fewer groups (scales past the last column belong to sums that are zero).
    struct Alone {
        Q4Part c;
        uint32_t s[2][E], z[2][E];
    };
    auto load_alone = [&](Alone &x, int tile, int half) {
        const int col = half * kQ4Half, left = row_bytes - (col >> 1) - 16 * t;
        const int last = first_row(tile + 1) - 1, lo = first_row(tile);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t row = r0 + min(lo + g + 8 * r, last);
            x.c.w[r] = load_any(a.W + row * a.ldw + (col >> 1) + 16 * t, left, a.W, w_end);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int64_t i = row * a.lds + group_of(min(col + (S > 1 ? (sub + e) * (kQ4Half / SUB) : 0), a.N - 1));
                x.s[r][e] = a.dtype_s == L2D_F32 ? __ldg(reinterpret_cast<const uint32_t *>(a.scales) + i)
                                                 : __ldg(reinterpret_cast<const uint16_t *>(a.scales) + i);
                x.z[r][e] = a.zeros ? __ldg(a.zeros + i) : 8;
            }
        }
    };
    auto multiply_alone = [&](const Alone &x, int half) {
        float s[2][E];
        uint32_t z[2][E];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s[r][e] = a.dtype_s == L2D_F32 ? __uint_as_float(x.s[r][e]) : scale_value(x.s[r][e], false, is_half);
                z[r][e] = x.z[r][e] & 15;
            }
        multiply(x.c, half, s, z);
    };

    // x of one staging: 16 lanes take 128 columns of one vector, eight columns each.  16 bytes hold columns
    // (0, 4) (1, 5) (2, 6) (3, 7) of eight; [half][column of x][word j][lane t].
    auto stage = [&](int kb) {
        bool any_odd = false;
        const int first = h_lo + kb * a.stage_h, halves = min(h_hi - first, a.stage_h);
        const int u = lane & 15, units = halves * a.vectors;
        // Eight columns of x as stored: 16 bytes, or 32 of fp32.
        struct Raw {
            uint4 lo, hi;
        };
        struct Unit {
            int v, half;
        };
        auto step = [&](Unit &e) {
            for (e.half += kQ4Warps * 2; e.half >= halves; e.half -= halves) ++e.v;
        };
        auto fetch = [&](const Unit &e) {
            Raw r = {};
            if (e.v >= a.vectors) return r;
            const int v = e.v, col = (first + e.half) * kQ4Half + 8 * u, size = FP32 ? 4 : 2;
            const char *src = static_cast<const char *>(a.x) + (v * a.stride_x + col) * size;
            if (col + 8 <= a.N && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                r.lo = load_words(src);
                if (size == 4) r.hi = load_words(src + 16);
                return r;
            }
            uint32_t w[8] = {};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (col + i >= a.N) continue;
                if (size == 4) w[i] = load_word(src + 4 * i);
                else w[i / 2] |= load_short(src + 2 * i) << (16 * (i & 1));
            }
            r.lo = make_uint4(w[0], w[1], w[2], w[3]);
            r.hi = make_uint4(w[4], w[5], w[6], w[7]);
            return r;
        };
        const int mine = warp * 2 + (lane >> 4);
        Unit at = {mine / halves, mine % halves};
        Raw ahead = fetch(at);
        for (int e = mine; e - (lane >> 4) < units; e += kQ4Warps * 2) {
            const Raw r = ahead;
            const bool real = e < units;
            const int v = real ? at.v : 0, half = real ? at.half : 0, column = v * PARTS, tt = u >> 2, j = u & 3;
            float2 *to = sums + half * 8 * NT + (column << kShift) + u / (16 / SUB);
            const bool stores_sums = real && u % (16 / SUB) == 0;
            step(at);
            ahead = fetch(at);
            if constexpr (KIND == kQ4Half16) {  // the same as below in fewer instructions
                uint32_t w[4] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w};
                const bool is_fp16 = a.dtype_x == L2D_F16;
                const uint32_t inf = is_fp16 ? 0x7c00u : 0x7f80u;
                auto largest = [&] {
                    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
                    return max(m & 0xffffu, m >> 16);
                };
                uint32_t top = largest(), mark = 0;
                if (top >= inf) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if ((w[i] & 0x7fffu) >= inf) w[i] &= 0xffff0000u, mark |= 1u << 2 * i;
                        if ((w[i] >> 16 & 0x7fffu) >= inf) w[i] &= 0xffffu, mark |= 2u << 2 * i;
                    }
                    top = largest();
                }
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                const uint32_t p = min(268u - (__float_as_uint(scale_value(top, false, is_fp16)) >> 23), 254u);
                const float up = __uint_as_float(p << 23), back = __uint_as_float((266u - p) << 23) * 0x1p-24f;
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = scale_value(w[i / 2], i & 1, is_fp16) * up;
                // All 11 bits of a value are above 2^-24, sixteenths included, down to 2^-10; each that is not is looked at.
                const uint32_t m = __vminu2(__vminu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vminu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
                if ((__float_as_uint(scale_value(min(m & 0xffffu, m >> 16), false, is_fp16)) >> 23) + p < 244) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float g = i & 1 ? f[i] * 0.0625f : f[i];
                        if (__half2float(__float2half_rn(g)) != g || (g == 0.0f && scale_value(w[i / 2], i & 1, is_fp16) != 0.0f)) f[i] = 0.0f, mark |= 1u << i;
                    }
                }
                const bool odd = __ballot_sync(0xffffffffu, mark != 0) >> (lane & 16) & 0xffff;  // in these 128 columns
                any_odd = any_odd || (real && odd);
                uint32_t out[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __half2 h = i & 1 ? __floats2half2_rn(f[i] * 0.0625f, f[i + 4] * 0.0625f) : __floats2half2_rn(f[i], f[i + 4]);
                    memcpy(&out[i], &h, 4);
                }
                if (real) reinterpret_cast<uint4 *>(smem + (half * columns + column) * kColumn)[j * 4 + tt] = make_uint4(out[0], out[1], out[2], out[3]);
                if (stores_sums) to[0] = make_float2(0.0f, odd ? -back : back);  // the sign: see add_odd_ones()
                if (real && odd) marks[(half * a.vectors + v) * 16 + u] = static_cast<uint8_t>(mark);
                continue;
            }
            const uint32_t raw[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
            float f[8];
            uint32_t top = 0, mark = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = FP32 ? __uint_as_float(raw[i]) : scale_value(raw[i / 2], i & 1, a.dtype_x == L2D_F16);
                const uint32_t m = __float_as_uint(f[i]) & 0x7fffffffu;
                if (m < 0x7f800000u) top = max(top, m);
                else f[i] = 0.0f, mark |= 1u << i;
            }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
            if constexpr (BYTES) {
                // 2^(p - 127) takes the largest to [2^29, 2^30); four signed digits of 8 bits, a column each, and for fp32
                // four more of the next 30 bits.  The factor back is short of 2^16, which the end makes good.
                const uint32_t p = min(283u - (top >> 23), 253u);
                const float up = __uint_as_float(p << 23), back = __uint_as_float((254u - p) << 23) * 0x1p-16f;
                // All bits of a value are there from 2^-7 on (fp32) or 2^10 (16 bits); each that is below is looked at.
                bool far = false;
                if constexpr (FP32) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) far = far || (fabsf(f[i] * up) < 0x1p-7f && f[i] != 0.0f);
                } else {
                    const uint32_t m = __vminu2(__vminu2(raw[0] & 0x7fff7fffu, raw[1] & 0x7fff7fffu), __vminu2(raw[2] & 0x7fff7fffu, raw[3] & 0x7fff7fffu));
                    far = (__float_as_uint(scale_value(min(m & 0xffffu, m >> 16), false, a.dtype_x == L2D_F16)) >> 23) + p < 264;
                }
                if (far) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float n = f[i] * up;
                        float left = n - rintf(n);
                        if (FP32) left = left * 0x1p30f - rintf(left * 0x1p30f);
                        if (left != 0.0f || (n == 0.0f && f[i] != 0.0f)) f[i] = 0.0f, mark |= 1u << i;
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] *= up;
                const bool odd = __ballot_sync(0xffffffffu, mark != 0) >> (lane & 16) & 0xffff;
                any_odd = any_odd || (real && odd);
                if (real && odd) marks[(half * a.vectors + v) * 16 + u] = static_cast<uint8_t>(mark);
                auto four_digits = [&](int part, float unit) {
                    uint32_t digits[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) digits[i] = (static_cast<uint32_t>(__float2int_rn(f[i])) + 0x00808080u) ^ 0x00808080u;
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const uint32_t pick = d | (4 + d) << 4;
                        const uint32_t even = __byte_perm(__byte_perm(digits[0], digits[2], pick), __byte_perm(digits[4], digits[6], pick), 0x5410);
                        const uint32_t odds = __byte_perm(__byte_perm(digits[1], digits[3], pick), __byte_perm(digits[5], digits[7], pick), 0x5410);
                        if (real)
                            *reinterpret_cast<uint2 *>(smem + (half * columns + column + part + d) * kColumn + (j >> 1) * 64 + tt * 16 + (j & 1) * 8) = make_uint2(even, odds);
                        int total = __dp4a(static_cast<int>(even), 0x01010101, __dp4a(static_cast<int>(odds), 0x01010101, 0));
#pragma unroll
                        for (int o = 1; o < 16 / SUB; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
                        const float factor = unit * static_cast<float>(1 << 8 * d);
                        if (stores_sums)
                            to[(part + d) << kShift] = make_float2(ZEROS ? static_cast<float>(total) : 12582912.0f + 8.0f * static_cast<float>(total),
                                                                   odd && part + d == 0 ? -factor : factor);  // the sign: see add_odd_ones()
                    }
                };
                four_digits(0, back);
                if constexpr (FP32) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = (f[i] - rintf(f[i])) * 0x1p30f;
                    four_digits(4, back * 0x1p-30f);
                }
                continue;
            }
            // 2^(p - 127) takes the largest to [2^14, 2^15); the factor back is short of 2^12, which the end makes good.
            const uint32_t p = min(268u - (top >> 23), 254u);
            const float up = __uint_as_float(p << 23), back = __uint_as_float((266u - p) << 23) * 0x1p-24f;
            // The two parts keep 23 bits of what is not below 2^-13, sixteenths included.
            bool far = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) far = far || (fabsf(f[i] * up) < (i & 1 ? 0x1p-9f : 0x1p-13f) && f[i] != 0.0f);
            if (far) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (fabsf(f[i] * up) < (i & 1 ? 0x1p-9f : 0x1p-13f) && f[i] != 0.0f) f[i] = 0.0f, mark |= 1u << i;
            }
            const bool odd = __ballot_sync(0xffffffffu, mark != 0) >> (lane & 16) & 0xffff;
            any_odd = any_odd || (real && odd);
            if (real && odd) marks[(half * a.vectors + v) * 16 + u] = static_cast<uint8_t>(mark);
            uint32_t hi[8], lo[8];  // lo: what the first part leaves, 2^11 times as large
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] *= i & 1 ? up * 0.0625f : up;
                const __half h = __float2half_rn(f[i]);
                hi[i] = __half_as_ushort(h);
                lo[i] = __half_as_ushort(__float2half_rn((f[i] - __half2float(h)) * 2048.0f));
            }
            uint4 *dst = reinterpret_cast<uint4 *>(smem + (half * columns + column) * kColumn) + j * 4 + tt;
            if (real) {
                dst[0] = make_uint4(hi[0] | hi[4] << 16, hi[1] | hi[5] << 16, hi[2] | hi[6] << 16, hi[3] | hi[7] << 16);
                dst[kColumn / 16] = make_uint4(lo[0] | lo[4] << 16, lo[1] | lo[5] << 16, lo[2] | lo[6] << 16, lo[3] | lo[7] << 16);
            }
            if (stores_sums) {
                to[0] = make_float2(0.0f, odd ? -back : back);
                to[SUB] = make_float2(0.0f, back * 0x1p-11f);
            }
        }
        // Columns of B without a vector: their sums are dropped, but stay finite.
        const int used = columns << kShift, unused = 8 * NT - used;
        for (int e = tid; e < halves * unused; e += kQ4Threads) sums[e / unused * 8 * NT + used + e % unused] = make_float2(0.0f, 0.0f);
        return any_odd;
    };

    bool odd_vectors = false;
    // The terms of what of x was left out of this staging, for one result: row of the block, vector v.
    auto add_odd_ones = [&](float sum, int kb, int row, int v) {
        const int first = h_lo + kb * a.stage_h, halves = min(h_hi - first, a.stage_h);
        for (int half = 0; half < halves; ++half) {
            if (!(sums[half * 8 * NT + ((v * PARTS) << kShift)].y < 0.0f)) continue;
            const uint32_t *bits = reinterpret_cast<const uint32_t *>(marks + (half * a.vectors + v) * 16);
            for (int w = 0; w < 4; ++w) {  // 32 columns, of one group
                uint32_t left = bits[w];
                if (!left) continue;
                const int col = (first + half) * kQ4Half + 32 * w;
                const int64_t i = (r0 + row) * a.lds + group_of(col);
                const uint4 q = load_any(a.W + (r0 + row) * a.ldw + col / 2, row_bytes - col / 2, a.W, w_end);
                const float s = dev::load_as_float(a.scales, a.dtype_s, i), z = a.zeros ? a.zeros[i] & 15 : 8;
                for (; left; left &= left - 1) {
                    const int j = __ffs(left) - 1;
                    const uint32_t eight = j < 16 ? (j < 8 ? q.x : q.y) : j < 24 ? q.z : q.w;
                    sum += s * ((static_cast<float>(eight >> (4 * (j & 7)) & 15) - z) * dev::load_as_float(a.x, a.dtype_x, v * a.stride_x + col + j));
                }
            }
        }
        return sum;
    };

    // A tile is done: its warps' sums meet, in warp order.
    int buffer = 0;
    auto meet = [&] {
        if (a.warps_k == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(wm + 1), "r"(a.warps_k * 32) : "memory");
    };
    auto finish = [&](int kb, int tile) {
        if (NT > 1) meet();  // the sums before have been read
        float *mine = red + (buffer * kQ4Warps + warp) * kQ4Rows * 8 * NT;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * 8 * NT + 8 * n + 2 * t) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * 8 * NT + 8 * n + 2 * t) = make_float2(acc[n][2], acc[n][3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
        }
        meet();
        const int lo = first_row(tile), n = first_row(tile + 1) - lo;
        // Another warp of the group begins each time.
        for (int e = ((wk + tile) & (a.warps_k - 1)) * 32 + lane; e < kQ4Rows * a.vectors; e += a.warps_k * 32) {
            const int v = e / kQ4Rows, r = e % kQ4Rows, row = lo + r;
            if (r >= n) continue;
            const float *p = red + ((buffer * kQ4Warps + wm * a.warps_k) * kQ4Rows + r) * 8 * NT + v * PARTS * SUB;
            float sum = 0.0f;
            for (int w = 0; w < a.warps_k; ++w, p += kQ4Rows * 8 * NT)
                for (int i = 0; i < PARTS; ++i)
#pragma unroll
                    for (int c = 0; c < SUB; ++c) sum += p[i * SUB + c];
            if (odd_vectors) sum = add_odd_ones(sum * kUnit, kb, row, v) / kUnit;
            if (a.y_rows) {
                float *y = ysum + row * a.vectors + v;
                sum += kb ? *y : 0.0f;
                *y = sum;  // this thread again the next time
            }
            if (h_lo + (kb + 1) * a.stage_h >= h_hi && a.ranks == 1) dev::store_as(a.y, a.dtype_y, v * a.stride_y + r0 + row, sum * kUnit);
        }
        if (NT == 1) buffer ^= 1;
    };

    for (int kb = 0; h_lo + kb * a.stage_h < h_hi; ++kb) {
        // The staging's halves: whole steps, an even share for each warp, and what is left, a half for a warp.
        const int first = h_lo + kb * a.stage_h, n = min(h_hi - first, a.stage_h);
        const bool cut = (first + n) * kQ4Half > a.N;  // the last half is not whole
        const int whole = WORDS ? (n - (cut ? 1 : 0)) / kQ4Deep : 0, rest = n - whole * kQ4Deep;
        const int k0 = whole * wk / a.warps_k, mine = whole * (wk + 1) / a.warps_k - k0;
        Q4Part part[kQ4Deep] = {};
        Q4Scales<S, ZEROS> now = {}, next = {};
        Rows at = {};
        if (S == 0) {  // the offsets of the scales are needed before the first load
            if (kb) __syncthreads();
            for (int h = tid; h < n; h += kQ4Threads) offsets[h] = group_of(min((first + h) * kQ4Half, a.N - 1));
            __syncthreads();
        }
        if (tiles && mine) {
            at = rows_of(0, first + k0 * kQ4Deep);
#pragma unroll
            for (int h = 0; h < kQ4Deep; ++h) load(part[h], at, h);
            load_scales(now, at, k0 * kQ4Deep);
        }
        if (S && kb) __syncthreads();  // all are done with the x before
        odd_vectors = __syncthreads_or(stage(kb)) != 0;

        for (int tile = 0; tile < tiles; ++tile) {
            for (int i = (wk + tile) & (a.warps_k - 1); i < rest; i += 2 * a.warps_k) {
                const int half = whole * kQ4Deep + i, other = half + a.warps_k;
                Alone x, y;
                load_alone(x, tile, first + half);
                if (other < n) load_alone(y, tile, first + other);
                multiply_alone(x, half);
                if (other < n) multiply_alone(y, other);
            }
            for (int i = 0; i < mine; ++i) {
                const bool end = i == mine - 1;
                const int half = (k0 + i) * kQ4Deep;
                if (!(end && tile == tiles - 1)) {
                    if (end) {
                        at = rows_of(tile + 1, first + k0 * kQ4Deep);
                    } else {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            at.w[r] += 64 * kQ4Deep;
                            if (S) at.s[r] += SUB * kQ4Deep * 2;
                            if (S && ZEROS) at.z[r] += SUB * kQ4Deep;
                        }
                    }
                    load_scales(next, at, end ? k0 * kQ4Deep : half + kQ4Deep);
#pragma unroll
                    for (int h = 0; h < kQ4Deep; ++h) {
                        multiply_of(part[h], now, h, half + h);
                        load(part[h], at, h);
                    }
                    now = next;
                } else {
#pragma unroll
                    for (int h = 0; h < kQ4Deep; ++h) multiply_of(part[h], now, h, half + h);
                }
            }
            finish(kb, tile);
        }
    }

    if (a.ranks > 1) {  // the ranks' sums, each rank for its share of the rows
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int lo = rows * rank / a.ranks, n = rows * (rank + 1) / a.ranks - lo;
        for (int e = tid; e < n * a.vectors; e += kQ4Threads) {
            const int v = e / n, row = lo + e - v * n;
            float sum = 0.0f;
            for (int r = 0; r < a.ranks; ++r) sum += cluster.map_shared_rank(ysum, r)[row * a.vectors + v];
            dev::store_as(a.y, a.dtype_y, v * a.stride_y + r0 + row, sum * kUnit);
        }
        cluster.sync();  // nobody leaves while its sums are read
    }
}

using Q4Kernel = void (*)(Q4Args);
struct Q4Entry {
    Q4Kernel run;
    std::atomic<uint64_t> *smem_set;
};

template <int NT, int S, bool ZEROS, bool WORDS, Q4Kind KIND>
Q4Entry q4_entry() {
    static std::atomic<uint64_t> set{0};
    return {k_q4_gemv<NT, S, ZEROS, WORDS, KIND>, &set};
}
template <int NT, int S, Q4Kind KIND>
Q4Entry q4_entry(bool zeros, bool words) {
    if (words) return zeros ? q4_entry<NT, S, true, true, KIND>() : q4_entry<NT, S, false, true, KIND>();
    return q4_entry<NT, S, true, false, KIND>();
}
template <int NT, Q4Kind KIND>
Q4Entry q4_entry(int group, bool zeros, bool words) {
    if (group == 32) return q4_entry<NT, 4, KIND>(zeros, words);
    if (group == 64) return q4_entry<NT, 2, KIND>(zeros, words);
    return group == 128 ? q4_entry<NT, 1, KIND>(zeros, words) : q4_entry<NT, 0, KIND>(zeros, words);
}
// The kernels of one kind each, compiled apart; tiles_n: how many eights of columns B has (1, 2 or 4; by bytes 1).
Q4Entry q4_entry_half(int tiles_n, int group, bool zeros, bool words);
Q4Entry q4_entry_float(int tiles_n, int group, bool zeros, bool words);
Q4Entry q4_entry_bytes(bool fp32, int group, bool zeros, bool words);

}  // namespace l2d

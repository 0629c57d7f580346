// Matrix-vector products with 4-bit weights and group scales (l2d_q4_gemv).
//
//   y[b][i] = sum_j s[i][j / g] * (q[i][j] - z[i][j / g]) * x[b][j]
//
// Memory bound: a weight is half a byte and is used once per vector.  At the bandwidth of HBM an SM
// gets about 52 weights a cycle and has 128 lanes to treat them, so a weight may cost two instructions;
// a fused multiply-add in fp32 alone would be one, with its conversion three.  So the products run on
// matrix instructions (m16n8k16, fp32 sums): 16 rows of weights are the A operand, turned from nibbles
// into exact 16-bit integers q - z in about 1.2 instructions a weight, the vectors are the columns of B,
// and the scales are applied to the fp32 sums of each group, so nothing is rounded before the end.
//
//  * A lane's 16 bytes (32 columns of one row) are loaded straight into registers from the row-major
//    weights.  A product's order of columns is free, so the lane's nibbles are used in the order in
//    which masks deliver them, and x is put into that order when it is staged in shared memory.
//  * One instruction sums over the four lanes of a row, 128 columns.  Where groups are shorter, x of
//    the different groups goes to different columns of B (zeros elsewhere), so that each group still has
//    a sum of its own: S = 128 / group columns per vector.
//  * fp32 vectors are split into three bf16 parts, 8 bits each, which hold all 24 bits: three columns.
//  * A block's rows are its even share of M, in tiles of at most 16 rows of nearly equal size, so that
//    blocks finish together whatever M is; its warps split the columns of a tile (or, where rows are
//    short, several tiles) and meet in shared memory once per tile, in a fixed order.
#include "l2d_launch.cuh"

#include <algorithm>
#include <cstring>

namespace l2d {

struct Q4Args {
    const uint8_t *W;
    const uint8_t *scales;
    const uint8_t *zeros;
    const void *x;
    void *y;
    int64_t M, ldw, lds, stride_x, stride_y;
    int N, vectors, group, dtype_x, dtype_y, dtype_s;
    int aligned;     // rows of W on 16-byte boundaries
    int sub_shift;   // log2 of S, columns of B per vector part
    int parts;       // columns of B per vector for its precision: 3 for fp32, else 1
    int warps_k;     // warps that split a tile's columns
    int block_k;     // columns of x staged at a time
    int blocks_k;    // how many times
    int y_rows;      // rows of the block's sums kept over several stagings (0: one staging)
};

constexpr int kQ4Warps = 8;
constexpr int kQ4Threads = kQ4Warps * 32;
constexpr int kQ4Chunk = 256;      // columns a warp takes at a time: 128 bytes of each row
constexpr int kQ4Rows = 16;
constexpr int kQ4MaxRows = 512;    // rows of a block, at most

// Byte offsets in dynamic shared memory.
struct Q4Smem {
    int red, y, bytes;
};
__host__ __device__ inline Q4Smem q4_smem(int tiles_n, int columns, int block_k, int y_rows) {
    Q4Smem s;
    s.red = columns * block_k * 2;
    s.y = s.red + 2 * kQ4Warps * kQ4Rows * 8 * tiles_n * 4;
    s.bytes = s.y + y_rows * columns * 4;
    return s;
}

template <typename T>
struct MmaType { using type = T; };
template <>
struct MmaType<float> { using type = __nv_bfloat16; };

template <typename T>
__device__ __forceinline__ void q4_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename H2>
__device__ __forceinline__ uint32_t bits_of(H2 v) {
    uint32_t r;
    memcpy(&r, &v, 4);
    return r;
}
template <typename H2>
__device__ __forceinline__ H2 from_bits(uint32_t r) {
    H2 v;
    memcpy(&v, &r, 4);
    return v;
}

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t set) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(set));
    return d;
}

// Eight nibbles to q - z: p[i] holds nibbles i and i + 4.  A nibble or-ed into the low mantissa bits of
// 2^n is 2^n + q; subtracting 2^n + z is exact.  z: that subtrahend, one per type (see zero_of).
template <typename T>
struct Nibbles;
template <>
struct Nibbles<__half> {
    // 1024 + q from bits 0-3; 1024 + 16 q from bits 4-7, a sixteenth of which is 64 + q.
    static __device__ __forceinline__ void unpack(uint32_t w, uint32_t z, uint32_t (&p)[4]) {
        const __half2 lo = from_bits<__half2>(z);  // 1024 + z
        const __half2 hi = __hsub2(__half2half2(__ushort_as_half(0x6380)), lo);  // 960 - (1024 + z) = -(64 + z)
        const __half2 r16 = __half2half2(__ushort_as_half(0x2c00));              // 1 / 16
        p[0] = bits_of(__hsub2(from_bits<__half2>(and_or(w, 0x000F000F, 0x64006400)), lo));
        p[1] = bits_of(__hfma2(from_bits<__half2>(and_or(w, 0x00F000F0, 0x64006400)), r16, hi));
        w >>= 8;
        p[2] = bits_of(__hsub2(from_bits<__half2>(and_or(w, 0x000F000F, 0x64006400)), lo));
        p[3] = bits_of(__hfma2(from_bits<__half2>(and_or(w, 0x00F000F0, 0x64006400)), r16, hi));
    }
    static __device__ __forceinline__ uint32_t zero_of(uint32_t z) { return (0x6400 | z) * 0x10001u; }
};
template <>
struct Nibbles<__nv_bfloat16> {
    // Seven mantissa bits: 128 + q, one nibble position at a time.
    static __device__ __forceinline__ void unpack(uint32_t w, uint32_t z, uint32_t (&p)[4]) {
        const __nv_bfloat162 lo = from_bits<__nv_bfloat162>(z);  // 128 + z
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = bits_of(__hsub2(from_bits<__nv_bfloat162>(and_or(w >> (4 * i), 0x000F000F, 0x43004300)), lo));
    }
    static __device__ __forceinline__ uint32_t zero_of(uint32_t z) { return (0x4300 | z) * 0x10001u; }
};

__device__ __forceinline__ uint4 load_weights(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The first n (0..16) bytes at p, zeros after them.
__device__ __noinline__ uint4 load_bytes(const uint8_t *p, int n) {
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < n) v[i >> 2] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// 16 bytes at any address, from the two aligned ones around them.
__device__ __forceinline__ uint4 load_unaligned(const uint8_t *p) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15;
    const uint4 *q = reinterpret_cast<const uint4 *>(p - off);
    const uint4 a = __ldg(q);
    const uint4 b = off ? __ldg(q + 1) : a;
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

// What a warp holds of one chunk (two halves of 128 columns) of a tile: this lane's 16 bytes of rows g
// and g + 8, the scales of those rows' sums and the zeros of its columns.
template <bool SUB, bool ZEROS>
struct Q4Chunk {
    uint4 w[2][2];                          // [half][row]
    uint32_t s[2][2][SUB ? 2 : 1];          // [half][row][column of C], as stored
    uint32_t z[2][ZEROS ? 2 : 1];
};

template <typename X, int NT, bool SUB, bool ZEROS>
__global__ void __launch_bounds__(kQ4Threads, 2) k_q4_gemv(Q4Args a) {
    using T = typename MmaType<X>::type;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int columns = a.vectors * a.parts;  // columns of x in shared memory
    const Q4Smem lay = q4_smem(NT, columns, a.block_k, a.y_rows);
    float *red = reinterpret_cast<float *>(smem + lay.red), *ysum = reinterpret_cast<float *>(smem + lay.y);
    const int64_t r0 = a.M * blockIdx.x / gridDim.x;
    const int rows = static_cast<int>(a.M * (blockIdx.x + 1) / gridDim.x - r0), tiles = (rows + kQ4Rows - 1) / kQ4Rows;
    const int wk = warp % a.warps_k, wm = warp / a.warps_k, warps_m = kQ4Warps / a.warps_k;
    const int rounds = (tiles + warps_m - 1) / warps_m;  // of one tile for each group of warps
    const int row_bytes = (a.N + 1) / 2;
    const uint8_t *w_end = a.W + (a.M - 1) * a.ldw + row_bytes;
    const int S = 1 << a.sub_shift;
    dev::wait_for_previous();

    auto chunks_in = [&](int kb) {  // chunks of a staging that fall to each warp
        const int n = min(a.N - kb * a.block_k, a.block_k);
        return ((n + kQ4Chunk - 1) / kQ4Chunk + a.warps_k - 1) / a.warps_k;
    };
    struct At {
        int kb, round, i, n;
    };
    auto advance = [&](At &at) {
        if (++at.i == at.n) {
            at.i = 0;
            if (++at.round == rounds) {
                at.round = 0;
                if (++at.kb < a.blocks_k) at.n = chunks_in(at.kb);
            }
        }
    };
    auto first_row = [&](int tile) { return tile * rows / tiles; };

    auto load = [&](Q4Chunk<SUB, ZEROS> &c, const At &at) {
        const int tile = at.round * warps_m + wm;
        const int col = at.kb * a.block_k + (at.i * a.warps_k + wk) * kQ4Chunk;
        if (at.kb >= a.blocks_k || tile >= tiles || col >= min(a.N, (at.kb + 1) * a.block_k)) return;
        const int lo = first_row(tile), hi = first_row(tile + 1);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = lo + g + 8 * r;
            const bool real = row < hi;
            const uint8_t *base = a.W + (r0 + row) * a.ldw;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at_byte = col / 2 + 64 * h + 16 * t, left = row_bytes - at_byte;
                const uint8_t *p = base + at_byte;
                c.w[h][r] = make_uint4(0, 0, 0, 0);
                if (real && left > 0) {
                    if (a.aligned && left >= 16) c.w[h][r] = load_weights(p);
                    else if (left >= 16 && p >= a.W + 16 && p + 32 <= w_end) c.w[h][r] = load_unaligned(p);
                    else c.w[h][r] = load_bytes(p, min(left, 16));
                }
                // Scales: of the columns 2t, 2t + 1 of C, which belong to the subgroups (2t) % S and (2t + 1) % S.
                const int half = col + 128 * h;
                const int64_t s_row = (r0 + row) * a.lds;
#pragma unroll
                for (int e = 0; e < (SUB ? 2 : 1); ++e) {
                    const int at_col = half + ((2 * t + e) & (S - 1)) * a.group;
                    c.s[h][r][e] = 0;
                    if (real && at_col < a.N) {
                        const int64_t i = s_row + (SUB ? at_col / 32 >> (2 - a.sub_shift) : at_col / a.group);
                        c.s[h][r][e] = a.dtype_s == L2D_F32 ? reinterpret_cast<const uint32_t *>(a.scales)[i]
                                                            : reinterpret_cast<const uint16_t *>(a.scales)[i];
                    }
                }
                if constexpr (ZEROS) {
                    const int mine = half + 32 * t;
                    c.z[h][r] = 0;
                    if (real && mine < a.N) c.z[h][r] = a.zeros[s_row + (SUB ? mine / 32 >> (2 - a.sub_shift) : mine / a.group)];
                }
            }
        }
    };

    auto scale = [&](uint32_t v) {
        if (a.dtype_s == L2D_F32) return __uint_as_float(v);
        if (a.dtype_s == L2D_BF16) return __uint_as_float(v << 16);
        return __half2float(__ushort_as_half(static_cast<unsigned short>(v)));
    };

    // The column of x that this lane feeds into column g of each n-tile: vector part (8 n + g) / S, if its
    // own columns of W belong to that column's subgroup.
    const bool feeds = (g & (S - 1)) == (t * S >> 2);
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;

    auto consume = [&](const Q4Chunk<SUB, ZEROS> &c, const At &at) {
        const int tile = at.round * warps_m + wm;
        const int k = (at.i * a.warps_k + wk) * kQ4Chunk;  // in the staged columns
        if (tile >= tiles || at.kb * a.block_k + k >= min(a.N, (at.kb + 1) * a.block_k)) return;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float sum[NT][4] = {};
            const uint4 *x = reinterpret_cast<const uint4 *>(smem) + static_cast<int64_t>(k / 128 + h) * columns * 16 + t;
            const uint32_t z0 = Nibbles<T>::zero_of(ZEROS ? c.z[h][0] & 15 : 8), z1 = Nibbles<T>::zero_of(ZEROS ? c.z[h][ZEROS ? 1 : 0] & 15 : 8);
            const uint32_t w0[4] = {c.w[h][0].x, c.w[h][0].y, c.w[h][0].z, c.w[h][0].w};
            const uint32_t w1[4] = {c.w[h][1].x, c.w[h][1].y, c.w[h][1].z, c.w[h][1].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t p0[4], p1[4];
                Nibbles<T>::unpack(w0[j], z0, p0);
                Nibbles<T>::unpack(w1[j], z1, p1);
                const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int column = (8 * n + g) >> a.sub_shift;
                    uint4 b = make_uint4(0, 0, 0, 0);
                    if (feeds && column < columns) b = x[(j * columns + column) * 4];
                    q4_mma<T>(sum[n], a0, b.x, b.y);
                    q4_mma<T>(sum[n], a1, b.z, b.w);
                }
            }
            const float s00 = scale(c.s[h][0][0]), s10 = scale(c.s[h][1][0]);
            const float s01 = SUB ? scale(c.s[h][0][SUB ? 1 : 0]) : s00, s11 = SUB ? scale(c.s[h][1][SUB ? 1 : 0]) : s10;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                acc[n][0] = fmaf(s00, sum[n][0], acc[n][0]);
                acc[n][1] = fmaf(s01, sum[n][1], acc[n][1]);
                acc[n][2] = fmaf(s10, sum[n][2], acc[n][2]);
                acc[n][3] = fmaf(s11, sum[n][3], acc[n][3]);
            }
        }
    };

    // x of one staging, in the order of the nibbles: 16 bytes hold columns (0, 4) (1, 5) (2, 6) (3, 7) of eight;
    // [128 columns][word j][column of B][lane t].
    auto stage = [&](int kb) {
        const int k0 = kb * a.block_k, n = (min(a.N - k0, a.block_k) + kQ4Chunk - 1) / kQ4Chunk * (kQ4Chunk / 8);
        for (int e = tid; e < n * a.vectors; e += kQ4Threads) {
            const int v = e / n, u = e - v * n, col = k0 + 8 * u;  // eight columns from col
            const X *src = static_cast<const X *>(a.x) + v * a.stride_x + col;
            const int half = u >> 4, tt = (u >> 2) & 3, j = u & 3;
            uint4 *dst = reinterpret_cast<uint4 *>(smem) + (static_cast<int64_t>(half) * columns * 16 + (j * columns + v * a.parts) * 4 + tt);
            if constexpr (sizeof(X) == 2) {
                uint32_t h[8];
                if (col + 8 <= a.N && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                    const uint4 q = *reinterpret_cast<const uint4 *>(src);
                    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[i] = w[i >> 1] >> (16 * (i & 1)) & 0xffff;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[i] = col + i < a.N ? reinterpret_cast<const uint16_t *>(src)[i] : 0;
                }
                *dst = make_uint4(h[0] | h[4] << 16, h[1] | h[5] << 16, h[2] | h[6] << 16, h[3] | h[7] << 16);
            } else {
                // fp32 into three bf16 parts by truncation: each takes the next 8 bits, so the three add up exactly.
                // Infinities and NaNs stay whole in the first part.
                uint32_t f[8];
                if (col + 8 <= a.N && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                    const uint4 q = *reinterpret_cast<const uint4 *>(src), r = *reinterpret_cast<const uint4 *>(src + 4);
                    f[0] = q.x, f[1] = q.y, f[2] = q.z, f[3] = q.w, f[4] = r.x, f[5] = r.y, f[6] = r.z, f[7] = r.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = col + i < a.N ? reinterpret_cast<const uint32_t *>(src)[i] : 0;
                }
                uint32_t part[3][8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool finite = (f[i] & 0x7f800000u) != 0x7f800000u;
                    if (!finite && (f[i] & 0x007fffffu)) f[i] |= 0x00400000u;
                    const float rest = finite ? __uint_as_float(f[i]) - __uint_as_float(f[i] & 0xffff0000u) : 0.0f;
                    const uint32_t m = __float_as_uint(rest);
                    const float last = rest - __uint_as_float(m & 0xffff0000u);
                    part[0][i] = f[i] >> 16;
                    part[1][i] = m >> 16;
                    part[2][i] = __float_as_uint(last) >> 16;
                }
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    dst[4 * q] = make_uint4(part[q][0] | part[q][4] << 16, part[q][1] | part[q][5] << 16, part[q][2] | part[q][6] << 16,
                                            part[q][3] | part[q][7] << 16);
            }
        }
    };

    // One tile for each group of warps is done: their sums meet, in warp order.
    int buffer = 0;
    auto finish = [&](const At &at) {
        float *mine = red + (buffer * kQ4Warps + warp) * kQ4Rows * 8 * NT;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * 8 * NT + 8 * n + 2 * t) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * 8 * NT + 8 * n + 2 * t) = make_float2(acc[n][2], acc[n][3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
        }
        __syncthreads();
        const int per_vector = a.parts << a.sub_shift;
        for (int e = tid; e < warps_m * kQ4Rows * a.vectors; e += kQ4Threads) {
            const int v = e / (warps_m * kQ4Rows), rest = e - v * warps_m * kQ4Rows, m = rest / kQ4Rows, r = rest % kQ4Rows;
            const int tile = at.round * warps_m + m;
            if (tile >= tiles) continue;
            const int row = first_row(tile) + r;
            if (row >= first_row(tile + 1)) continue;
            const float *p = red + ((buffer * kQ4Warps + m * a.warps_k) * kQ4Rows + r) * 8 * NT + v * per_vector;
            float sum = 0.0f;
            for (int w = 0; w < a.warps_k; ++w)
                for (int i = 0; i < per_vector; ++i) sum += p[w * kQ4Rows * 8 * NT + i];
            if (a.y_rows) {
                float *y = ysum + row * a.vectors + v;
                sum += at.kb ? *y : 0.0f;
                *y = sum;  // this thread again the next time
            }
            if (at.kb == a.blocks_k - 1) dev::store_as(a.y, a.dtype_y, v * a.stride_y + r0 + row, sum);
        }
        buffer ^= 1;
    };

    Q4Chunk<SUB, ZEROS> even, odd;
    At now = {0, 0, 0, chunks_in(0)}, next = now;
    load(even, next);
    advance(next);
    load(odd, next);
    advance(next);
    auto step = [&](Q4Chunk<SUB, ZEROS> &c) {
        if (now.i == 0 && now.round == 0) {
            if (now.kb) __syncthreads();
            stage(now.kb);
            __syncthreads();
        }
        consume(c, now);
        load(c, next);
        advance(next);
        if (now.i == now.n - 1) finish(now);
        advance(now);
        return now.kb < a.blocks_k;
    };
    while (step(even) && step(odd)) {
    }
}

using Q4Kernel = void (*)(Q4Args);
struct Q4Entry {
    Q4Kernel run;
    std::atomic<uint64_t> *smem_set;
};

template <typename X, int NT, bool SUB, bool ZEROS>
Q4Entry q4_entry() {
    static std::atomic<uint64_t> set{0};
    return {k_q4_gemv<X, NT, SUB, ZEROS>, &set};
}
template <typename X, int NT>
Q4Entry q4_entry(bool sub, bool zeros) {
    if (sub) return zeros ? q4_entry<X, NT, true, true>() : q4_entry<X, NT, true, false>();
    return zeros ? q4_entry<X, NT, false, true>() : q4_entry<X, NT, false, false>();
}
template <typename X>
Q4Entry q4_entry(int nt, bool sub, bool zeros) {
    if (nt == 1) return q4_entry<X, 1>(sub, zeros);
    return nt == 2 ? q4_entry<X, 2>(sub, zeros) : q4_entry<X, 4>(sub, zeros);
}

// No columns: every sum is empty.
__global__ void k_q4_zero(Q4Args a) {
    dev::wait_for_previous();
    for (int64_t e = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; e < a.M * a.vectors; e += int64_t(gridDim.x) * blockDim.x)
        dev::store_as(a.y, a.dtype_y, e / a.M * a.stride_y + e % a.M, 0.0f);
}

}  // namespace l2d

using namespace l2d;

extern "C" {

int l2d_q4_gemv(const l2d_q4_desc *desc, const void *x, int64_t stride_x, void *y, int64_t stride_y, int64_t vectors,
                void *stream) {
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    const l2d_q4_desc &d = *desc;
    constexpr int64_t kMax = int64_t(1) << 31;
    if (d.M < 0 || d.N < 0 || d.M >= kMax || d.N >= kMax / 2)
        return set_error(L2D_ERR_INVALID, "M = %lld, N = %lld: M below 2^31 and N below 2^30 are supported",
                         static_cast<long long>(d.M), static_cast<long long>(d.N));
    if (vectors < 0 || vectors >= kMax) return set_error(L2D_ERR_INVALID, "%lld vectors", static_cast<long long>(vectors));
    if (!valid_dtype(d.dtype_x) || !valid_dtype(d.dtype_y) || !valid_dtype(d.dtype_s))
        return set_error(L2D_ERR_INVALID, "bad dtype (x %d, y %d, scales %d)", d.dtype_x, d.dtype_y, d.dtype_s);
    if (d.group != 32 && d.group != 64 && (d.group <= 0 || d.group % 128))
        return set_error(L2D_ERR_INVALID, "group %d: 32, 64 or a multiple of 128", d.group);
    const int64_t groups = (d.N + d.group - 1) / d.group;
    const int64_t ldw = d.ldw ? d.ldw : (d.N + 1) / 2, lds = d.lds ? d.lds : groups;
    if (ldw < (d.N + 1) / 2 || lds < groups)
        return set_error(L2D_ERR_INVALID, "ldw %lld or lds %lld is shorter than a row", static_cast<long long>(ldw),
                         static_cast<long long>(lds));
    if (!stride_x) stride_x = d.N;
    if (!stride_y) stride_y = d.M;
    if (vectors > 1 && (stride_x < d.N || stride_y < d.M)) return set_error(L2D_ERR_INVALID, "vector strides overlap");
    constexpr int64_t kFar = int64_t(1) << 60;  // byte offsets stay far inside 64 bits
    if ((d.M && (ldw > kFar / d.M || lds > kFar / d.M)) ||
        (vectors > 1 && (stride_x > kFar / vectors || stride_y > kFar / vectors)))
        return set_error(L2D_ERR_INVALID, "strides too large");
    if (d.M == 0 || vectors == 0) return L2D_OK;
    if (!y || (d.N && (!x || !d.W || !d.scales))) return set_error(L2D_ERR_INVALID, "null pointer");
    if (reinterpret_cast<uintptr_t>(x) % elem_bytes(d.dtype_x) || reinterpret_cast<uintptr_t>(y) % elem_bytes(d.dtype_y) ||
        reinterpret_cast<uintptr_t>(d.scales) % elem_bytes(d.dtype_s))
        return set_error(L2D_ERR_INVALID, "x, y and scales must be aligned to their elements");
    int sms = 0;
    const int st = device_sms(d.device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(d.device);
    L2D_CUDA_TRY(on.err);
    Q4Args a = {};
    a.W = static_cast<const uint8_t *>(d.W);
    a.scales = static_cast<const uint8_t *>(d.scales);
    a.zeros = static_cast<const uint8_t *>(d.zeros);
    a.M = d.M;
    a.N = static_cast<int>(d.N);
    a.ldw = ldw;
    a.lds = lds;
    a.stride_x = stride_x;
    a.stride_y = stride_y;
    a.group = d.group;
    a.dtype_x = d.dtype_x;
    a.dtype_y = d.dtype_y;
    a.dtype_s = d.dtype_s;
    a.aligned = reinterpret_cast<uintptr_t>(d.W) % 16 == 0 && ldw % 16 == 0;
    a.sub_shift = d.group == 32 ? 2 : d.group == 64 ? 1 : 0;
    a.parts = d.dtype_x == L2D_F32 ? 3 : 1;
    const int each = a.parts << a.sub_shift;  // columns of B per vector
    const int most = 32 / each;               // vectors of one pass over the weights
    const int64_t chunks = (d.N + kQ4Chunk - 1) / kQ4Chunk;
    a.warps_k = 1;
    while (a.warps_k < kQ4Warps && a.warps_k < chunks) a.warps_k *= 2;
    const int64_t blocks = std::max<int64_t>(std::min<int64_t>(d.M, 2 * sms), (d.M + kQ4MaxRows - 1) / kQ4MaxRows);
    for (int64_t v = 0; v < vectors; v += most) {
        a.vectors = static_cast<int>(std::min<int64_t>(most, vectors - v));
        a.x = static_cast<const char *>(x) + v * stride_x * elem_bytes(d.dtype_x);
        a.y = static_cast<char *>(y) + v * stride_y * elem_bytes(d.dtype_y);
        if (d.N == 0) {
            L2D_CUDA_TRY(launch(k_q4_zero, dim3(2 * sms), 256, 0, stream, a));
            continue;
        }
        const int tiles_n = a.vectors * each <= 8 ? 1 : a.vectors * each <= 16 ? 2 : 4;
        const int columns = a.vectors * a.parts;
        // x is staged whole where two blocks with it fit an SM, else as many times as it takes.
        const int rows = static_cast<int>((d.M + blocks - 1) / blocks);
        constexpr int kRoom = 112 * 1024;
        const int64_t whole = chunks * kQ4Chunk;
        if (whole * columns * 2 <= kRoom - q4_smem(tiles_n, columns, 0, 0).bytes) {
            a.block_k = static_cast<int>(whole);
            a.blocks_k = 1;
            a.y_rows = 0;
        } else {
            const int step = kQ4Chunk * a.warps_k;
            const int fits = (kRoom - q4_smem(tiles_n, columns, 0, rows).bytes) / (columns * 2) / step * step;
            a.block_k = std::max(fits, step);
            a.blocks_k = static_cast<int>((d.N + a.block_k - 1) / a.block_k);
            a.y_rows = rows;
        }
        const int smem = q4_smem(tiles_n, columns, a.block_k, a.y_rows).bytes;
        const bool sub = a.sub_shift > 0, zeros = d.zeros != nullptr;
        const Q4Entry k = d.dtype_x == L2D_F32 ? q4_entry<float>(tiles_n, sub, zeros)
                          : d.dtype_x == L2D_F16 ? q4_entry<__half>(tiles_n, sub, zeros)
                                                 : q4_entry<__nv_bfloat16>(tiles_n, sub, zeros);
        L2D_CUDA_TRY(allow_smem(k.run, 227 * 1024, d.device, *k.smem_set));
        L2D_CUDA_TRY(launch(k.run, dim3(static_cast<unsigned>(blocks)), kQ4Threads, smem, stream, a));
    }
    return L2D_OK;
}

}  // extern "C"

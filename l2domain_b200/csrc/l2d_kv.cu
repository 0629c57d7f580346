// The paged cache of keys and values: appending with rotation (l2d_kv_append) and attention of one new
// token per sequence over it (l2d_attn_*).
#include "l2d_launch.cuh"

#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

namespace l2d {

constexpr int kMaxHeadDim = 256;

// A checked cache description with every stride filled in.
struct Cache {
    char *k, *v;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    const int32_t *table;
    int64_t table_stride, num_pages;
    int num_seqs, table_width, page_size, heads, head_dim;
    int page_shift;  // log2 of page_size, -1 if it is no power of two
    uint32_t *status;
};

struct AppendArgs {
    Cache c;
    const void *k, *v, *q;
    void *q_out;
    const float *cos, *sin;
    const int32_t *pos, *seq;
    int64_t tokens, max_pos, k_token, v_token, q_token, q_out_token;
    int heads_q, rot_dim, interleaved;
};

struct AttnArgs {
    Cache c;
    const void *q;
    void *out;
    float *lse;
    const int32_t *lens;
    int64_t q_token, out_token;
    int heads_q, window, batch;
    float scale;
};

// The page of its sequence that holds a position.
__device__ __forceinline__ unsigned page_index(const Cache &c, unsigned pos) {
    return c.page_shift >= 0 ? pos >> c.page_shift : pos / static_cast<unsigned>(c.page_size);
}

__device__ __forceinline__ void report(uint32_t *status, uint32_t bit) {
    if (status) atomicOr(status, bit);
}

// The page of position p of sequence s, or -1 if it has none.
__device__ __forceinline__ int64_t page_of(const Cache &c, int64_t s, int p) {
    const int i = static_cast<int>(page_index(c, p));
    if (s < 0 || s >= c.num_seqs || i >= c.table_width) return -1;
    const int32_t page = c.table[s * c.table_stride + i];
    return page >= 0 && page < c.num_pages ? page : -1;
}

// ---------------------------------------------------------------------------------------------
// Appending.
//
// A copy with a few multiplications: every element is read once and written once.  A head is cut into units
// of VEC pairs (the rotated part: for the half layout VEC elements and their VEC partners, for the interleaved
// one 2 VEC elements side by side) and of 2 VEC elements (the rest, and values), so that a thread moves 32 bytes
// of 16-bit elements.  A thread keeps its unit's cosines and sines for as many heads of its token as the grid
// leaves it: heads are split over blocks only while there are too few tokens to fill the GPU.
// ---------------------------------------------------------------------------------------------

template <typename T, int N>
struct Pack {
    T v[N];
};

// N consecutive elements; one load or store of up to 16 bytes each where N > 1 (the host checked the alignment).
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    Pack<T, N> r;
    if constexpr (N * sizeof(T) >= 16) {
#pragma unroll
        for (int i = 0; i < N * static_cast<int>(sizeof(T)) / 16; ++i) {
            const uint4 x = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p) + 16 * i);
            memcpy(reinterpret_cast<char *>(r.v) + 16 * i, &x, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = p[i];
    }
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r) {
    if constexpr (N * sizeof(T) >= 16) {
#pragma unroll
        for (int i = 0; i < N * static_cast<int>(sizeof(T)) / 16; ++i) {
            uint4 x;
            memcpy(&x, reinterpret_cast<const char *>(r.v) + 16 * i, 16);
            *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p) + 16 * i) = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = r.v[i];
    }
}

constexpr int kAppendThreads = 256;

// units: rotated units of a head (rot_units), then plain ones.  A thread's unit is fixed; the threads of a token
// for which `rows` are left take every rows-th of its heads.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads) k_append(const __grid_constant__ AppendArgs a, int units, int rot_units, int rows) {
    dev::wait_for_previous();
    const int D = a.c.head_dim, half = a.rot_dim / 2, hk = a.c.heads, heads = a.heads_q + 2 * hk;
    const int64_t thread = static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x;
    const int64_t t = thread / (units * rows);
    if (t >= a.tokens) return;
    const int rest = static_cast<int>(thread - t * (units * rows)), row = rest / units, unit = rest - row * units;
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
    const int slot = p - static_cast<int>(page_index(a.c, p)) * a.c.page_size;
    const T *k = static_cast<const T *>(a.k) + t * a.k_token, *v = static_cast<const T *>(a.v) + t * a.v_token;
    const T *q = static_cast<const T *>(a.q) + t * a.q_token;
    T *q_out = static_cast<T *>(a.q_out) + t * a.q_out_token;
    T *kc = reinterpret_cast<T *>(a.c.k) + page * a.c.k_page + slot * a.c.k_slot;
    T *vc = reinterpret_cast<T *>(a.c.v) + page * a.c.v_page + slot * a.c.v_slot;

    // Where the unit's two halves are, and its angles.
    const bool rotated = unit < rot_units;
    const int pair = unit * VEC;  // first pair of a rotated unit
    const int first = !rotated ? a.rot_dim + (unit - rot_units) * 2 * VEC : INTERLEAVED ? 2 * pair : pair;
    const int second = rotated && !INTERLEAVED ? pair + half : first + VEC;
    const bool both = rotated || second < D;  // the plain part may end with one half
    float c[VEC], s[VEC];
    if (rotated) {
        const Pack<float, VEC> cc = load_pack<float, VEC>(a.cos + static_cast<int64_t>(p) * half + pair);
        const Pack<float, VEC> ss = load_pack<float, VEC>(a.sin + static_cast<int64_t>(p) * half + pair);
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = cc.v[i], s[i] = ss.v[i];
    }
    // Heads in order: queries, keys, values; a few at a time, loads first.
    auto at = [&](int h, const T *&src, T *&dst) {
        const int g = h - a.heads_q, w = g - hk;
        if (g < 0) src = q + static_cast<int64_t>(h) * D, dst = q_out + static_cast<int64_t>(h) * D;
        else if (w < 0) src = k + static_cast<int64_t>(g) * D, dst = kc + g * a.c.k_head;
        else src = v + static_cast<int64_t>(w) * D, dst = vc + w * a.c.v_head;
    };
    constexpr int kHeads = 4;
    for (int h0 = row; h0 < heads; h0 += kHeads * rows) {
        Pack<T, VEC> x[kHeads], y[kHeads];
        T *dst[kHeads];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const T *src = nullptr;
            dst[j] = nullptr;
            if (h0 + j * rows >= heads) continue;
            at(h0 + j * rows, src, dst[j]);
            x[j] = load_pack<T, VEC>(src + first);
            if (both) y[j] = load_pack<T, VEC>(src + second);
        }
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            if (h0 + j * rows >= heads) continue;
            if (rotated && h0 + j * rows < a.heads_q + hk) {
                float u[2 * VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) u[i] = dev::widen(x[j].v[i]), u[VEC + i] = dev::widen(y[j].v[i]);
                T r[2 * VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int lo = INTERLEAVED ? 2 * i : i, hi = INTERLEAVED ? 2 * i + 1 : VEC + i;
                    r[lo] = dev::narrow<T>(fmaf(u[lo], c[i], -(u[hi] * s[i])));
                    r[hi] = dev::narrow<T>(fmaf(u[hi], c[i], u[lo] * s[i]));
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[j].v[i] = r[i], y[j].v[i] = r[VEC + i];
            }
            store_pack<T, VEC>(dst[j] + first, x[j]);
            if (both) store_pack<T, VEC>(dst[j] + second, y[j]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Attention of one token over the cache.
//
// Memory bound: each key and value is read once, for all query heads of its group.  A block of
// eight warps (four for heads of more than 128 elements, whose rings would not fit) works on one
// key-value head of one sequence at a time; each warp streams its own 16 keys (8 of 32 bits) of every 128 (64 with four
// warps or 32 bits, 32 with both) through a ring of shared memory of its own (no block-wide barrier in the loop) and
// keeps a running maximum and sum per query head, so the data is passed over once.  16-bit caches feed matrix
// instructions with the query heads as the 16 rows; 32-bit caches use fp32 fused multiply-adds.
//
// A tile of 16 keys that lies in one page is one box of a tensor map over the cache (elements, heads,
// slots, pages), and one thread starts its copies; with a page size that is no multiple of 16, or rows off
// 16-byte boundaries, the lanes look up the page of each key and copy its rows themselves.
//
// The tiles of all sequences and heads, and kSwitch units before each head's, form one line that is cut into
// equal pieces, one per resident block, whatever the lengths are: a long sequence is split over many blocks and a block may take
// several short ones.  A piece that ends inside a sequence leaves its unnormalised sums in the plan's
// scratch, and the last piece of that sequence to arrive adds them in piece order, so the result does
// not depend on which block came last.
//
// Measured (32 query and 8 key-value heads of 128, bf16): 64 sequences of 0 to 8192 keys 170-182 us, 6.0-6.4
// TB/s of keys and values; 64 x 2048 91 us, 5.9 TB/s; one sequence of 17 keys 5.9 us, of which a launch 4.1.
// ---------------------------------------------------------------------------------------------

constexpr int kMaxRows = 16;    // query heads a block works on
// Heads of sequences of up to so many tiles are not split, the block in whose piece their first unit lies does them
// whole: a tile takes about 1.2 us of its block, and joining pieces 4 us (8 key-value heads of 128; one sequence of 300
// keys 8.4 us whole and 9.8 us split, of 500 keys 9.8 and 9.6, of 1000 keys 14.3 and 9.9; ragged 30 x 380 with 4 heads
// 10.2 and 15.5, 200 x 300 61 and 63; ragged 100 x 1000 is 56.5 us with 3 here, 54.8 with 5).
constexpr int kWholeTiles = 3;
// What a block spends on a head of a sequence besides its tiles (finding it, its first pages and queries, the sum over
// the warps), as so many tiles of the line that the blocks share evenly.  With none, blocks of many short sequences end
// last; 0, 1, 2, 3, 4 (8 key-value heads of 128, ragged): 64 x 8192 keys 195, 180, 174, 172, 172 us; 32 x 4000 71, 56,
// 53, 52, 52; 100 x 1000 82, 62, 56, 57, 57; 200 x 300 77, 66, 63, 65, 66; equal lengths 64 x 2048 89, 92, 90, 91, 92.
constexpr int kSwitch = 2;

__host__ __device__ __forceinline__ int64_t units_of(int64_t tiles) { return tiles ? tiles + kSwitch : 0; }

struct AttnScratch {
    float *part;         // [grid][2][kMaxRows][head_dim padded] unnormalised sums
    float *ml;           // [grid][2][2][kMaxRows] their maxima (log2) and sums of weights
    unsigned *arrived;   // [max_batch * heads * m_tiles], zero between calls
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// 16 bytes to shared memory; none are read, and zeros stored, where `real` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A box of a tensor map to shared memory, counted by a barrier there.
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap *map, int x, int head, int slot, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(head), "r"(slot), "r"(page), "r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void barrier_expect(uint32_t bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits for the barrier's phase of this parity; false if it does not come in about two seconds (a try suspends the
// thread for up to 4 us).
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
    uint32_t done = 0;
    for (int i = 0; i < (1 << 19) && !done; ++i)
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
// What this thread did to shared memory comes before copies of boxes that are started after the next barrier.
__device__ __forceinline__ void before_boxes() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Rows of keys and values in shared memory: boxes of 128 bytes a row, 16-byte chunks exchanged by the row
// (chunk ^ row, as the tensor map's 128-byte swizzle has it), so that eight rows' chunks meet all banks.
template <int ROWS>
__device__ __forceinline__ int chunk_at(int row, int chunk) {
    return (chunk >> 3) * (ROWS * 128) + row * 128 + (((chunk ^ row) & 7) << 4);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(T lo, T hi) {
    static_assert(sizeof(T) == 2, "16-bit types");
    uint16_t a, b;
    memcpy(&a, &lo, 2);
    memcpy(&b, &hi, 2);
    return static_cast<uint32_t>(a) | static_cast<uint32_t>(b) << 16;
}

// A running softmax's maximum, and what exponents are taken relative to: never -inf.
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.0f : m; }

// What the weights, 1 for the largest score, are multiplied by before they meet the values, and the sums of values with
// them until they are divided by the sum of weights: fp16 ends at 2^-24, so there small weights need it; bf16 and fp32
// values may be so large that only sums of fractions of them stay in the range.
template <typename T>
constexpr float kWeightUnit = 0x1p-24f;
template <>
constexpr float kWeightUnit<__half> = 0x1p15f;

// One warp's part of one head group of a 16-bit cache: KS steps of 16 elements of the head, the query
// heads as the rows of m16n8k16.  Groups of up to eight heads (SPLIT) use the other eight rows for the
// low halves of the weights: p = hi + lo in two 16-bit numbers, which leaves 2^-17 of p (bf16), or 2^-23 of it and
// at least 2^-51 of the largest (fp16, whose low halves are taken another 2^11 times as large).
// Larger groups multiply twice, by hi and by lo, into the same sums, which for fp16 leaves at least 2^-40 of the largest.
template <typename T, int KS, bool SPLIT>
struct MmaCore {
    using Elem = T;
    static constexpr int kKeys = 16;                       // keys of a warp's tile
    static constexpr int kWarps = KS <= 8 ? 8 : 4;         // whose rings fit an SM
    static constexpr bool kWholeRows = true;               // products reach the padding of a row
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRows = SPLIT ? 8 : 16;           // query heads
    static constexpr int kDim = KS * 16;                   // head_dim, padded
    static constexpr int kBoxes = (KS + 3) / 4;            // of 64 elements
    static constexpr int kChunks = kBoxes * 8;             // 16-byte chunks of a row, padding included
    static constexpr int kPitch = (KS * 2 + 1) * 16;       // of queries: an odd number of chunks
    static constexpr bool kQueryInSmem = !SPLIT && KS > 8; // registers would not hold queries and sums
    static constexpr int kQueryBytes = kRows * kPitch;
    static constexpr int kWarpBytes = 0;
    static constexpr float kUnit = kWeightUnit<T>;
    static constexpr float kLow = SPLIT && kUnit > 1.0f ? 0x1p11f : 1.0f;  // of low halves, beyond kUnit
    uint32_t qa[kQueryInSmem ? 1 : KS][SPLIT ? 2 : 4];
    float o[2 * KS][4], m[2], l[2];
    uint32_t query;

    // q: this group's first head; `heads` rows are real, `flip` takes their negatives.  All threads of the block call
    // it, and wait for their copies (copies_wait) and for each other before begin().
    static __device__ __forceinline__ void stage_query(const T *q, int heads, int D, bool aligned, bool flip, char *smem_q) {
        const uint16_t sign = flip ? 0x8000 : 0;
        if (aligned && !flip) {
            for (int e = threadIdx.x; e < kRows * KS * 2; e += kThreads) {
                const int r = e / (KS * 2), ch = e - r * (KS * 2);
                const bool real = r < heads && ch * 8 < D;
                copy16(smem_addr(smem_q + r * kPitch + ch * 16), real ? q + r * D + ch * 8 : q, real);
            }
        } else {
            for (int e = threadIdx.x; e < kRows * kDim; e += kThreads) {
                const int r = e / kDim, i = e - r * kDim;
                const uint16_t x = r < heads && i < D ? reinterpret_cast<const uint16_t *>(q)[r * D + i] : 0;
                reinterpret_cast<uint16_t *>(smem_q + r * kPitch)[i] = static_cast<uint16_t>(x ^ sign);
            }
        }
    }

    __device__ __forceinline__ void begin(char *smem_q, char *, int) {
        const int lane = threadIdx.x & 31;
        query = smem_addr(smem_q);
        if constexpr (SPLIT) {  // matrices of 8 heads x 8 elements, two steps of 16 at once
            uint32_t r[4];
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                ldmatrix4(r, query + (lane & 7) * kPitch + min(2 * k + (lane >> 3), KS * 2 - 1) * 16);
                qa[k][0] = r[0];
                qa[k][1] = r[1];
                if (k + 1 < KS) {
                    qa[k + 1][0] = r[2];
                    qa[k + 1][1] = r[3];
                }
            }
        } else if constexpr (!kQueryInSmem) {
#pragma unroll
            for (int k = 0; k < KS; ++k) load_query(qa[k], k);
        }
#pragma unroll
        for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
    }

    __device__ __forceinline__ void load_query(uint32_t (&a)[4], int k) const {
        const int lane = threadIdx.x & 31;
        ldmatrix4(a, query + (((lane >> 3) & 1) * 8 + (lane & 7)) * kPitch + (lane >> 4) * 16 + k * 32);
    }

    // One tile: keys at ks, values at vs (shared memory), bit j of live: key j counts.  scale2 > 0.  Scores are scaled,
    // and rounded, before the maximum is taken and taken off: the largest is then 0 whatever its size.  With one
    // rounding fewer, by a fused multiply-add on the unscaled ones, it would be what that rounding left: hundreds for
    // scores of 2^31.
    __device__ __forceinline__ void step(const char *ks, const char *vs, uint32_t live, float scale2) {
        const int lane = threadIdx.x & 31, t = lane & 3;
        // Chunk 2k + hi of row r is at chunk_at(r, hi) ^ (2k & 7) * 16, in box k / 4.
        const uint32_t ka = smem_addr(ks) + chunk_at<kKeys>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
        const uint32_t va = smem_addr(vs) + chunk_at<kKeys>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
        float s[2][4] = {}, s2[2][4] = {};  // of even and odd steps: shorter chains
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t a[4], b[4];
            if constexpr (kQueryInSmem) {
                load_query(a, k);
            } else if constexpr (SPLIT) {
                a[0] = qa[k][0];
                a[1] = 0;
                a[2] = qa[k][1];
                a[3] = 0;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = qa[k][e];
            }
            ldmatrix4(b, (ka ^ ((2 * k & 7) << 4)) + (k / 4) * (kKeys * 128));
            mma16816<T>(k & 1 ? s2[0] : s[0], a, b[0], b[1]);
            mma16816<T>(k & 1 ? s2[1] : s[1], a, b[2], b[3]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] = (s[e >> 2][e & 3] + s2[e >> 2][e & 3]) * scale2;
        if (live != (1u << kKeys) - 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (!(live >> ((e >> 2) * 8 + 2 * t + (e & 1)) & 1)) s[e >> 2][e & 3] = -INFINITY;
        }
        uint32_t p[4], lo[SPLIT ? 1 : 4];
#pragma unroll
        for (int r = 0; r < (SPLIT ? 1 : 2); ++r) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = s[e >> 1][2 * r + (e & 1)];
            float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m2 = fmaxf(m[r], top), base = finite_base(m2);
            if (__any_sync(0xffffffffu, m2 != m[r])) {
                const float f = exp2_approx(m[r] - base);
                l[r] *= f;
#pragma unroll
                for (int n = 0; n < 2 * KS; ++n) {
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
            for (int e = 0; e < 4; ++e) x[e] = exp2_approx(x[e] - base);
            l[r] += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float u = x[2 * h] * kUnit, v = x[2 * h + 1] * kUnit;
                const T a = dev::narrow<T>(u), b = dev::narrow<T>(v);
                p[r + 2 * h] = pack2(a, b);
                (SPLIT ? p[1 + 2 * h] : lo[r + 2 * h]) = pack2(dev::narrow<T>((u - dev::widen(a)) * kLow), dev::narrow<T>((v - dev::widen(b)) * kLow));
            }
        }
#pragma unroll
        for (int n = 0; n < KS; ++n) {
            uint32_t b[4];
            ldmatrix4_trans(b, (va ^ ((2 * n & 7) << 4)) + (n / 4) * (kKeys * 128));
            mma16816<T>(o[2 * n], p, b[0], b[1]);
            mma16816<T>(o[2 * n + 1], p, b[2], b[3]);
            if constexpr (!SPLIT) {
                mma16816<T>(o[2 * n], lo, b[0], b[1]);
                mma16816<T>(o[2 * n + 1], lo, b[2], b[3]);
            }
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
            for (int n = 0; n < 2 * KS; ++n) {
                float2 v = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if constexpr (SPLIT) v = make_float2(fmaf(o[n][2], 1.0f / kLow, v.x), fmaf(o[n][3], 1.0f / kLow, v.y));
                *reinterpret_cast<float2 *>(so + (g + 8 * r) * kDim + 8 * n + 2 * t) = v;
            }
        }
    }
};

// The same for a 32-bit cache: GT query heads, DV x 128 elements of the head.  Scores: a lane per key
// (two or four lanes share one, each every second or fourth chunk of the row), values: a lane per four
// elements of the head, the weights passed through shared memory.
template <int GT, int DV>
struct SimdCore {
    using Elem = float;
    static constexpr int kKeys = 8;
    static constexpr int kWarps = DV == 1 ? 8 : 4;
    static constexpr bool kWholeRows = false;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRows = GT;
    static constexpr int kDim = DV * 128;
    static constexpr int kBoxes = kDim / 32;
    static constexpr int kChunks = kDim / 4;
    static constexpr int kQueryBytes = GT * kDim * 4;
    static constexpr int kWarpBytes = GT * kKeys * 4;  // weights of the warp's tile
    static constexpr int kParts = 32 / kKeys;
    float o[GT][DV][4], m[GT], l[GT];
    const float *query;
    float *weights;
    int chunks;

    static __device__ __forceinline__ void stage_query(const float *q, int heads, int D, bool aligned, bool flip, char *smem_q) {
        if (aligned && !flip) {
            for (int e = threadIdx.x; e < GT * kDim / 4; e += kThreads) {
                const int r = e / (kDim / 4), i = (e - r * (kDim / 4)) * 4;
                const bool real = r < heads && i < D;
                copy16(smem_addr(smem_q + e * 16), real ? q + r * D + i : q, real);
            }
            return;
        }
        for (int e = threadIdx.x; e < GT * kDim; e += kThreads) {
            const int r = e / kDim, i = e - r * kDim;
            const float x = r < heads && i < D ? q[r * D + i] : 0.0f;
            reinterpret_cast<float *>(smem_q)[e] = flip ? -x : x;
        }
    }

    __device__ __forceinline__ void begin(char *smem_q, char *warp_smem, int D) {
        query = reinterpret_cast<float *>(smem_q);
        weights = reinterpret_cast<float *>(warp_smem);
        chunks = (D + 3) / 4;
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.0f;
#pragma unroll
            for (int v = 0; v < DV; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[g][v][e] = 0.0f;
        }
    }

    __device__ __forceinline__ void step(const char *ks, const char *vs, uint32_t live, float scale2) {
        const int lane = threadIdx.x & 31, key = lane % kKeys, sub = lane / kKeys;
        float s[GT] = {};
        for (int c = sub; c < chunks; c += kParts) {
            const float4 k = *reinterpret_cast<const float4 *>(ks + chunk_at<kKeys>(key, c));
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float4 q = reinterpret_cast<const float4 *>(query + g * kDim)[c];
                s[g] = fmaf(q.x, k.x, s[g]);
                s[g] = fmaf(q.y, k.y, s[g]);
                s[g] = fmaf(q.z, k.z, s[g]);
                s[g] = fmaf(q.w, k.w, s[g]);
            }
        }
        const bool ok = live >> key & 1;
#pragma unroll
        for (int g = 0; g < GT; ++g) {
#pragma unroll
            for (int d = kKeys; d < 32; d <<= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], d);
            s[g] *= scale2;
            float top = ok ? s[g] : -INFINITY;
#pragma unroll
            for (int d = 1; d < kKeys; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float m2 = fmaxf(m[g], top), base = finite_base(m2), f = exp2_approx(m[g] - base);
            const float w = ok ? exp2_approx(s[g] - base) : 0.0f;
            l[g] = fmaf(l[g], f, w);
            m[g] = m2;
            if (sub == 0) weights[g * kKeys + key] = w * kWeightUnit<float>;
#pragma unroll
            for (int v = 0; v < DV; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[g][v][e] *= f;
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kKeys; j += 4) {
#pragma unroll
            for (int v = 0; v < DV; ++v) {
                if (lane + 32 * v >= chunks) continue;
                float4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4 *>(vs + chunk_at<kKeys>(j + i, lane + 32 * v));
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    const float4 w = *reinterpret_cast<const float4 *>(weights + g * kKeys + j);
                    const float ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[g][v][0] = fmaf(ww[i], x[i].x, o[g][v][0]);
                        o[g][v][1] = fmaf(ww[i], x[i].y, o[g][v][1]);
                        o[g][v][2] = fmaf(ww[i], x[i].z, o[g][v][2]);
                        o[g][v][3] = fmaf(ww[i], x[i].w, o[g][v][3]);
                    }
                }
            }
        }
        __syncwarp();
    }

    __device__ __forceinline__ void end(float *so, float *sm, float *sl) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            float sum = l[g];
#pragma unroll
            for (int d = 1; d < kKeys; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) {
                sm[g] = m[g];
                sl[g] = sum;
            }
#pragma unroll
            for (int v = 0; v < DV; ++v)
                *reinterpret_cast<float4 *>(so + g * kDim + 4 * (lane + 32 * v)) = make_float4(o[g][v][0], o[g][v][1], o[g][v][2], o[g][v][3]);
        }
    }
};

// Shared memory of a block: the rings, stage by stage (the last one, which the first tiles of the next piece do
// not need, is reused for the warps' sums at the end of a piece), queries, the
// cores' own words, barriers, live bits, maxima and sums.
constexpr int kJoin = 64;  // pieces whose factors are held at a time when a sequence's pieces are joined
template <typename Core, int STAGES>
struct AttnSmem {
    static constexpr int kTile = Core::kKeys * 128 * Core::kBoxes;  // of keys, and of values
    static constexpr int kStage = 2 * kTile;  // of one warp
    static constexpr int kRing = Core::kWarps * STAGES * kStage;
    static constexpr int kSums = Core::kWarps * (STAGES - 1) * kStage;
    static constexpr int kFactors = kSums + Core::kWarps * Core::kRows * Core::kDim * 4;
    static constexpr int kEnd = kFactors + 2 * kJoin * kMaxRows * 4;
    static constexpr int kQuery = kRing > kEnd ? kRing : kEnd;
    static constexpr int kWarp = kQuery + 2 * Core::kQueryBytes;  // of this piece and of the next one
    static constexpr int kBars = kWarp + Core::kWarps * Core::kWarpBytes;
    static constexpr int kLive = kBars + Core::kWarps * STAGES * 8;
    static constexpr int kMl = kLive + Core::kWarps * STAGES * 4;
    static constexpr int kFlag = kMl + Core::kWarps * 2 * kMaxRows * 4;
    static constexpr int kBytes = kFlag + 16;
};

// How keys and values come to shared memory: as boxes, as 16-byte chunks, or element by element.
enum { kBoxes = 2, kWords = 1, kElements = 0 };

struct AttnMaps {
    CUtensorMap k, v;
};

// A warp's view of the keys of one sequence and head.  Page lookups run one tile ahead of the copies.
template <typename Core, int STAGES>
struct Stream {
    using T = typename Core::Elem;
    using Sm = AttnSmem<Core, STAGES>;
    const Cache &c;
    const AttnMaps &maps;
    int how, head;
    const int32_t *table;
    char *ring;
    uint32_t bars;
    uint32_t *live;
    uint32_t phases;      // parity of each stage's barrier; kLate: a box did not come
    int64_t next;         // the first key of the tile whose pages are in `page`
    int lo, len, step;    // keys lo .. len - 1 count; keys between this warp's tiles
    int slot, page;       // of this lane's key (lanes kLanes j .. kLanes j + kLanes - 1: key j); with boxes, of the tile's first
    bool wanted;          // that key, or one of the tile's, counts
    static constexpr int kLanes = 32 / Core::kKeys;
    static constexpr uint32_t kLate = 1u << 31;

    // The entry is not looked at before the next tile is started: an instruction that used it here would wait for
    // it, and the products with it.
    __device__ __forceinline__ void lookup() {
        const int64_t key = how == kBoxes ? next : next + (threadIdx.x & 31) / kLanes;
        wanted = key < len && (how == kBoxes ? key + Core::kKeys : key + 1) > lo;
        const unsigned i = page_index(c, static_cast<unsigned>(key));
        slot = static_cast<int>(static_cast<unsigned>(key) - i * static_cast<unsigned>(c.page_size));
        if (wanted) page = __ldg(table + i);
    }

    // Starts the copies of the next tile into a stage of the ring.
    __device__ __forceinline__ void issue(int stage) {
        const int lane = threadIdx.x & 31;
        constexpr uint32_t kAll = (1u << Core::kKeys) - 1;
        const bool real = wanted && page >= 0 && page < c.num_pages;
        if (wanted && !real) report(c.status, L2D_KV_BAD_PAGE);
        char *tile = ring + stage * (Core::kWarps * Sm::kStage);
        if (how == kBoxes) {
            uint32_t bits = 0;
            if (real) {
                bits = kAll;
                if (next < lo) bits &= kAll << (lo - static_cast<int>(next));  // by less than kKeys: lookup()
                if (next + Core::kKeys > len) bits &= kAll >> (static_cast<int>(next) + Core::kKeys - len);
            }
            if (lane == 0) {
                live[stage] = bits;
                if (bits) {
                    const uint32_t bar = bars + 8 * stage, to = smem_addr(tile);
                    barrier_expect(bar, Sm::kStage);
#pragma unroll
                    for (int b = 0; b < Core::kBoxes; ++b) {
                        const int x = b * (128 / static_cast<int>(sizeof(T)));
                        copy_box(to + b * Core::kKeys * 128, &maps.k, x, head, slot, page, bar);
                        copy_box(to + Sm::kTile + b * Core::kKeys * 128, &maps.v, x, head, slot, page, bar);
                    }
                }
            }
        } else {
            // Bit kLanes j of the vote to bit j.
            const uint32_t vote = __ballot_sync(0xffffffffu, real);
            const uint32_t bits = __ballot_sync(0xffffffffu, lane < Core::kKeys && (vote >> (lane * kLanes & 31) & 1));
            if (lane == 0) live[stage] = bits;
            if (bits) {
                constexpr int64_t eb = sizeof(T);
                const int r = lane / kLanes, first = lane % kLanes;
                const char *k = c.k, *v = c.v;
                if (real) {
                    k += (page * c.k_page + slot * c.k_slot + head * c.k_head) * eb;
                    v += (page * c.v_page + slot * c.v_slot + head * c.v_head) * eb;
                }
                if (how == kWords) {
                    const int have = c.head_dim * static_cast<int>(eb) / 16, need = Core::kWholeRows ? Core::kDim / 8 : have;
                    const uint32_t to = smem_addr(tile);
#pragma unroll 4
                    for (int ch = first; ch < need; ch += kLanes) {
                        const bool in = real && ch < have;
                        const int off = in ? ch * 16 : 0;
                        copy16(to + chunk_at<Core::kKeys>(r, ch), k + off, in);
                        copy16(to + Sm::kTile + chunk_at<Core::kKeys>(r, ch), v + off, in);
                    }
                } else {
                    constexpr int kPer = 16 / static_cast<int>(sizeof(T));
                    const int need = Core::kWholeRows ? Core::kDim : (c.head_dim + 3) / 4 * 4;
                    for (int i = first; i < need; i += kLanes) {
                        const bool in = real && i < c.head_dim;
                        const int dst = chunk_at<Core::kKeys>(r, i / kPer) + i % kPer * static_cast<int>(eb);
                        *reinterpret_cast<T *>(tile + dst) = in ? reinterpret_cast<const T *>(k)[i] : dev::narrow<T>(0.0f);
                        *reinterpret_cast<T *>(tile + Sm::kTile + dst) = in ? reinterpret_cast<const T *>(v)[i] : dev::narrow<T>(0.0f);
                    }
                }
            }
            copies_commit();
        }
        next += step;
        lookup();
    }

    // A box did not come: no more are started (lane 0 starts them), and the ones under way are waited for.
    __device__ __forceinline__ void give_up(int stage) {
        report(c.status, L2D_KV_TIMEOUT);
        phases |= kLate;
        len = 0;
        wanted = false;
        if (threadIdx.x & 31) return;
#pragma unroll 1
        for (int j = 1; j < STAGES - 1; ++j) {
            const int s = (stage + j) % STAGES;
            if (live[s]) barrier_wait(bars + 8 * s, phases >> s & 1);
            live[s] = 0;
        }
    }

    // The live bits of a stage, once its copies are there.  Values of keys that do not count are made zeros, as
    // their weights are: slots that were never written may hold anything.
    __device__ __forceinline__ uint32_t take(int stage) {
        if (how != kBoxes) copies_wait<STAGES - 2>();
        __syncwarp();
        const uint32_t bits = live[stage];
        if (how == kBoxes && bits) {
            if (!barrier_wait(bars + 8 * stage, phases >> stage & 1)) give_up(stage);
            phases ^= 1u << stage;
            if (bits != (1u << Core::kKeys) - 1) {
                char *values = ring + stage * (Core::kWarps * Sm::kStage) + Sm::kTile;
                for (int r = 0; r < Core::kKeys; ++r)
                    if (!(bits >> r & 1))
                        for (int ch = threadIdx.x & 31; ch < Core::kChunks; ch += 32)
                            *reinterpret_cast<uint4 *>(values + chunk_at<Core::kKeys>(r, ch)) = make_uint4(0, 0, 0, 0);
                before_boxes();
                __syncwarp();
            }
        }
        return bits;
    }
};

struct Span {
    int lo, len;      // the keys that count
    int from, tiles;  // tiles from a multiple of their size on
};

template <int TILE>
__device__ __forceinline__ Span span_of(const AttnArgs &a, int b) {
    Span s;
    const int room = a.c.table_width * a.c.page_size;  // below 2^31
    s.len = min(max(a.lens[b], 0), room);
    s.lo = a.window && s.len > a.window ? s.len - a.window : 0;
    s.from = s.lo & ~(TILE - 1);
    s.tiles = s.len > s.lo ? (s.len - s.from) / TILE + ((s.len - s.from) % TILE != 0) : 0;
    return s;
}

// a / b of two non-negative numbers, mostly below 2^32.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// Where a head's row of the output and its log-sum-exp go.
template <typename T>
__device__ __forceinline__ void store_row4(const AttnArgs &a, int b, int h, int i, int D, float4 x, float base, float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / kWeightUnit<T> / sum;
    const float v[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    T *out = static_cast<T *>(a.out) + b * a.out_token + static_cast<int64_t>(h) * D + i;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < D) out[e] = dev::narrow<T>(sum == 0.0f ? 0.0f : v[e]);
    if (i == 0 && a.lse) a.lse[static_cast<int64_t>(b) * a.heads_q + h] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
}

// Joins the pieces c0..c1 of one item: piece q's sums are in slot 2q, the first one's in slot 2 c0 + odd.
template <typename Core>
__device__ __forceinline__ void join(const AttnArgs &a, const AttnScratch &sc, int c0, int c1, int odd, int b, int head0, int rows,
                                     float *sums, float *factors, float *sm_m, float *sm_l) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.c.head_dim, n = c1 - c0 + 1;
    auto slot = [&](int j) { return static_cast<int64_t>(c0 + j) * 2 + (j == 0 ? odd : 0); };
    float *weights = factors + kJoin * kMaxRows;  // the pieces' sums of weights
    // The sums, warps over the pieces, up to 1024 elements (of whole rows' float4s) at a time; kJoin pieces at a
    // time, relative to the largest maximum so far.
    constexpr int kQuads = Core::kRows * Core::kDim / 4, kEach = kQuads % 256 == 0 ? 8 : kQuads % 128 == 0 ? 4 : 1, kRowQuads = Core::kDim / 4;
    static_assert(kQuads % (32 * kEach) == 0, "every lane has as many");
    for (int first = 0; first < kQuads; first += 32 * kEach) {
        float4 acc[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) acc[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (tid < kMaxRows) {
            sm_m[tid] = -INFINITY;
            sm_l[tid] = 0.0f;
        }
        for (int p0 = 0; p0 < n; p0 += kJoin) {
            const int pn = min(n - p0, kJoin);
            __syncthreads();
#pragma unroll 4
            for (int e = tid; e < pn * kMaxRows; e += Core::kThreads) {
                const int j = e / kMaxRows, r = e % kMaxRows;
                const float *ml = sc.ml + slot(p0 + j) * 2 * kMaxRows + r;
                factors[e] = r < rows ? __ldcg(ml) : -INFINITY;
                weights[e] = r < rows ? __ldcg(ml + kMaxRows) : 0.0f;
            }
            __syncthreads();
            for (int r = warp; r < kMaxRows; r += Core::kWarps) {  // a warp a row, lanes over the pieces
                const float was = sm_m[r], m0 = lane < pn ? factors[lane * kMaxRows + r] : -INFINITY,
                            m1 = lane + 32 < pn ? factors[(lane + 32) * kMaxRows + r] : -INFINITY;
                float top = fmaxf(was, fmaxf(m0, m1));
#pragma unroll
                for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float base = finite_base(top), f0 = exp2_approx(m0 - base), f1 = exp2_approx(m1 - base);
                float sum = (lane < pn ? f0 * weights[lane * kMaxRows + r] : 0.0f) + (lane + 32 < pn ? f1 * weights[(lane + 32) * kMaxRows + r] : 0.0f);
                if (lane < pn) factors[lane * kMaxRows + r] = f0;
                if (lane + 32 < pn) factors[(lane + 32) * kMaxRows + r] = f1;
#pragma unroll
                for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                __syncwarp();
                if (lane == 0) {
                    const float f = exp2_approx(was - base);  // what the pieces before are worth now
                    sm_m[r] = top;
                    sm_l[r] = fmaf(sm_l[r], f, sum);
                    sm_m[kMaxRows + r] = f;
                }
            }
            __syncthreads();
            if (p0) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const float f = sm_m[kMaxRows + (first + lane + 32 * i) / kRowQuads];
                    acc[i] = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
                }
            }
            // Four pieces' loads at a time (rows that are not real: of anything, and dropped).
            constexpr int kPieces = 4;
            for (int j0 = warp; j0 < pn; j0 += kPieces * Core::kWarps) {
                float4 x[kPieces][kEach];
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    const int j = min(j0 + k * Core::kWarps, pn - 1);
                    const float4 *part = reinterpret_cast<const float4 *>(sc.part + slot(p0 + j) * kMaxRows * Core::kDim) + first + lane;
#pragma unroll
                    for (int i = 0; i < kEach; ++i) x[k][i] = __ldcg(part + 32 * i);
                }
#pragma unroll
                for (int k = 0; k < kPieces; ++k) {
                    const int j = j0 + k * Core::kWarps;
                    if (j >= pn) break;
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        const float f = factors[j * kMaxRows + (first + lane + 32 * i) / kRowQuads];
                        acc[i] = make_float4(fmaf(f, x[k][i].x, acc[i].x), fmaf(f, x[k][i].y, acc[i].y), fmaf(f, x[k][i].z, acc[i].z), fmaf(f, x[k][i].w, acc[i].w));
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            reinterpret_cast<float4 *>(sums)[warp * kQuads + first + lane + 32 * i] = acc[i];
    }
    __syncthreads();
    for (int q = tid; q < rows * kRowQuads; q += Core::kThreads) {
        const int r = q / kRowQuads, i = (q - r * kRowQuads) * 4;
        if (i >= D) continue;
        float4 x = reinterpret_cast<const float4 *>(sums)[q];
#pragma unroll
        for (int w = 1; w < Core::kWarps; ++w) {
            const float4 y = reinterpret_cast<const float4 *>(sums)[w * kQuads + q];
            x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        store_row4<typename Core::Elem>(a, b, head0 + r, i, D, x, finite_base(sm_m[r]), sm_l[r]);
    }
}

template <typename Core, int STAGES>
__global__ void __launch_bounds__(Core::kThreads, 1) k_attn(const __grid_constant__ AttnArgs a, const __grid_constant__ AttnMaps maps, AttnScratch sc, int m_tiles, int how, bool q_aligned) {
    using T = typename Core::Elem;
    using Sm = AttnSmem<Core, STAGES>;
    constexpr int TILE = Core::kWarps * Core::kKeys;
    extern __shared__ __align__(1024) char smem[];
    float *sm_m = reinterpret_cast<float *>(smem + Sm::kMl), *sm_l = sm_m + Core::kWarps * kMaxRows;
    int *flag = reinterpret_cast<int *>(smem + Sm::kFlag);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int D = a.c.head_dim, G = a.heads_q / a.c.heads, items = a.c.heads * m_tiles;
    // What needs nothing of the kernels before: the maps' way to the copy unit, and the barriers.
    const uint32_t bars = smem_addr(smem + Sm::kBars) + warp * STAGES * 8;
    if (how == kBoxes && tid < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(tid ? &maps.v : &maps.k) : "memory");
    if (lane < STAGES) barrier_init(bars + 8 * lane);
    before_boxes();
    dev::wait_for_previous();

    // All units of one head, and rows without a position.
    int64_t total = 0;
    for (int b = lane; b < a.batch; b += 32) total += units_of(span_of<TILE>(a, b).tiles);
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (tid == 0 && a.lens[b] > a.c.table_width * a.c.page_size) report(a.c.status, L2D_KV_BAD_PAGE);
        if (span_of<TILE>(a, b).tiles) continue;
        for (int i = tid; i < a.heads_q * D; i += Core::kThreads) static_cast<T *>(a.out)[b * a.out_token + i] = dev::narrow<T>(0.0f);
        if (a.lse)
            for (int h = tid; h < a.heads_q; h += Core::kThreads) a.lse[static_cast<int64_t>(b) * a.heads_q + h] = -INFINITY;
    }

    // This block's piece of the line of units, and the sequence it starts in (every warp looks for itself).
    total *= items;
    const int64_t per = max(quotient(total + gridDim.x - 1, gridDim.x), static_cast<int64_t>(1));
    const int64_t first_unit = blockIdx.x * per, stop = min(total, first_unit + per);
    if (first_unit >= stop) return;
    int64_t before = 0;  // units of one head in the sequences before b
    int b = 0;
    for (;; b += 32) {
        const int64_t n = b + lane < a.batch ? units_of(span_of<TILE>(a, b + lane).tiles) : 0;
        int64_t upto = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += x;
        }
        upto += before;
        const unsigned found = __ballot_sync(0xffffffffu, n && first_unit < upto * items);
        if (found) {
            const int l = __ffs(found) - 1;
            before = __shfl_sync(0xffffffffu, upto - n, l);
            b += l;
            break;
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
    }

    const float scale2 = fabsf(a.scale) * 1.4426950408889634f;  // a negative one turns the queries' signs
    Stream<Core, STAGES> in{a.c, maps, how};
    in.ring = smem + warp * Sm::kStage;
    in.bars = bars;
    in.live = reinterpret_cast<uint32_t *>(smem + Sm::kLive) + warp * STAGES;
    in.phases = 0;
    in.page = -1;
    __syncwarp();
    // What a block does at a time: n tiles from t0 of one head group of a sequence, whose first tile is unit u0.
    struct Piece {
        Span s;
        int b, item, t0, n, head0, rows;
        int64_t u0;
    };
    auto find = [&](int64_t at_unit) {  // the first piece from that unit on; n = 0: none
        Piece p;
        p.n = 0;
        while (at_unit < stop) {
            p.s = span_of<TILE>(a, b);
            const int64_t units = units_of(p.s.tiles), at = at_unit - before * items;
            if (at >= units * items) {
                before += units;
                ++b;
                continue;
            }
            p.b = b;
            p.item = static_cast<int>(quotient(at, units));
            p.u0 = before * items + p.item * units + kSwitch;
            if (p.s.tiles <= kWholeTiles) {
                if (at_unit > p.u0 - kSwitch) {  // the block before has it
                    at_unit = p.u0 + p.s.tiles;
                    continue;
                }
                p.t0 = 0;
                p.n = p.s.tiles;
            } else {
                p.t0 = static_cast<int>(max(at_unit - p.u0, static_cast<int64_t>(0)));
                p.n = static_cast<int>(max(min(static_cast<int64_t>(p.s.tiles), stop - p.u0) - p.t0, static_cast<int64_t>(0)));
            }
            const int hk = p.item / m_tiles, row0 = (p.item - hk * m_tiles) * Core::kRows;
            p.rows = min(G - row0, Core::kRows);
            p.head0 = hk * G + row0;
            break;  // without a tile it is at its end
        }
        return p;
    };
    auto start = [&](const Piece &p) {  // its first tiles
        in.head = p.item / m_tiles;
        in.table = a.c.table + p.b * a.c.table_stride;
        in.lo = p.s.lo;
        in.len = static_cast<int>(min(static_cast<int64_t>(p.s.len), p.s.from + static_cast<int64_t>(p.t0 + p.n) * TILE));
        if (in.phases & in.kLate) in.len = 0;
        in.next = p.s.from + static_cast<int64_t>(p.t0) * TILE + warp * Core::kKeys;
        in.step = TILE;
        in.lookup();
#pragma unroll 1
        for (int i = 0; i < STAGES - 1; ++i) in.issue(i);
    };
    auto stage_query = [&](const Piece &p, char *to) {
        Core::stage_query(static_cast<const T *>(a.q) + p.b * a.q_token + static_cast<int64_t>(p.head0) * D, p.rows, D, q_aligned, a.scale < 0.0f,
                          to);
    };

    Core core;
    Piece p = find(first_unit);
    if (p.n == 0) return;
    start(p);
    char *query = smem + Sm::kQuery, *next_query = query + Core::kQueryBytes;
    stage_query(p, query);
    copies_commit();
    copies_wait<0>();
    __syncthreads();
    for (;;) {
        core.begin(query, smem + Sm::kWarp + warp * Core::kWarpBytes, D);
        // While the first tiles come: what follows, and its queries (with those loaded while the sums meet, 32 x 4096 keys
        // with 16 heads of 256 elements took 3 us more).
        Piece following = find(p.u0 + p.t0 + p.n);
        const bool more = following.n;
        if (more) stage_query(following, next_query);
        int stage = 0;
#pragma unroll 1
        for (int i = 0; i < p.n; ++i) {
            const uint32_t live = in.take(stage);
            in.issue(stage == 0 ? STAGES - 1 : stage - 1);  // every lane is done with that one: take()
            const char *ks = in.ring + stage * (Core::kWarps * Sm::kStage);
            if (live) core.step(ks, ks + Sm::kTile, live, scale2);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        copies_commit();
        copies_wait<0>();
        // The next piece's first tiles are on their way while this one's sums meet.
        before_boxes();
        __syncwarp();
        if (more) start(following);
        __syncthreads();

        // The warps' sums meet.
        const Span s = p.s;
        const int n = p.n, t0 = p.t0, item = p.item, head0 = p.head0, rows = p.rows;
        float *sums = reinterpret_cast<float *>(smem + Sm::kSums);
        core.end(sums + warp * Core::kRows * Core::kDim, sm_m + warp * kMaxRows, sm_l + warp * kMaxRows);
        __syncthreads();
        const bool whole = n == s.tiles;
        const int64_t u0 = p.u0, slot = static_cast<int64_t>(blockIdx.x) * 2 + (u0 + t0 != first_unit);
        constexpr int kRowQuads = Core::kDim / 4;
        for (int q = tid; q < rows * kRowQuads; q += Core::kThreads) {
            const int r = q / kRowQuads, i = (q - r * kRowQuads) * 4;
            if (i >= D) continue;
            float top = sm_m[r];
#pragma unroll
            for (int w = 1; w < Core::kWarps; ++w) top = fmaxf(top, sm_m[w * kMaxRows + r]);
            const float base = finite_base(top);
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < Core::kWarps; ++w) {
                const float f = exp2_approx(sm_m[w * kMaxRows + r] - base);
                const float4 y = *reinterpret_cast<const float4 *>(sums + (w * Core::kRows + r) * Core::kDim + i);
                x = make_float4(fmaf(f, y.x, x.x), fmaf(f, y.y, x.y), fmaf(f, y.z, x.z), fmaf(f, y.w, x.w));
                sum = fmaf(f, sm_l[w * kMaxRows + r], sum);
            }
            if (whole) {
                store_row4<T>(a, p.b, head0 + r, i, D, x, base, sum);
            } else {
                *reinterpret_cast<float4 *>(sc.part + (slot * kMaxRows + r) * Core::kDim + i) = x;
                if (i == 0) {
                    sc.ml[slot * 2 * kMaxRows + r] = top;
                    sc.ml[(slot * 2 + 1) * kMaxRows + r] = sum;
                }
            }
        }
        if (!whole) {
            const int c0 = static_cast<int>(quotient(u0, per)), c1 = static_cast<int>(quotient(u0 + s.tiles - 1, per));
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                unsigned *count = sc.arrived + static_cast<int64_t>(p.b) * items + item;
                const bool last = atomicAdd(count, 1u) == static_cast<unsigned>(c1 - c0);
                if (last) *count = 0;
                *flag = last;
            }
            __syncthreads();
            if (*flag) {
                __threadfence();
                join<Core>(a, sc, c0, c1, u0 != c0 * per, p.b, head0, rows, sums, reinterpret_cast<float *>(smem + Sm::kFactors), sm_m, sm_l);
            }
        }
        before_boxes();
        __syncthreads();  // the last stage holds sums until here
        if (!more) break;
        p = following;
        char *const used = query;
        query = next_query;
        next_query = used;
    }
}

struct AttnKernel {
    void (*run)(AttnArgs, AttnMaps, AttnScratch, int, int, bool);
    int smem, threads, rows, dim, tile, keys;
};

template <typename Core, int STAGES>
AttnKernel attn_kernel() {
    return {k_attn<Core, STAGES>, AttnSmem<Core, STAGES>::kBytes, Core::kThreads, Core::kRows, Core::kDim, Core::kWarps * Core::kKeys, Core::kKeys};
}

template <typename T, bool SPLIT>
AttnKernel pick_mma(int D) {
    if (D <= 64) return attn_kernel<MmaCore<T, 4, SPLIT>, 3>();
    if (D <= 80) return attn_kernel<MmaCore<T, 5, SPLIT>, 3>();
    if (D <= 96) return attn_kernel<MmaCore<T, 6, SPLIT>, 3>();
    if (D <= 128) return attn_kernel<MmaCore<T, 8, SPLIT>, 3>();
    if (D <= 192) return attn_kernel<MmaCore<T, 12, SPLIT>, 3>();
    return attn_kernel<MmaCore<T, 16, SPLIT>, 3>();
}

AttnKernel pick_attn(int dtype, int D, int G) {
    if (dtype == L2D_F16) return G <= 8 ? pick_mma<__half, true>(D) : pick_mma<__half, false>(D);
    if (dtype == L2D_BF16) return G <= 8 ? pick_mma<__nv_bfloat16, true>(D) : pick_mma<__nv_bfloat16, false>(D);
    if (D <= 128) {
        if (G == 1) return attn_kernel<SimdCore<1, 1>, 3>();
        if (G <= 4) return attn_kernel<SimdCore<4, 1>, 3>();
        if (G <= 8) return attn_kernel<SimdCore<8, 1>, 3>();
        return attn_kernel<SimdCore<16, 1>, 3>();
    }
    if (G == 1) return attn_kernel<SimdCore<1, 2>, 3>();
    if (G <= 4) return attn_kernel<SimdCore<4, 2>, 3>();
    return attn_kernel<SimdCore<8, 2>, 3>();
}

// Checks a cache description and fills in its strides.
int check_cache(const l2d_kv_cache *cache, Cache *c) {
    if (!cache) return set_error(L2D_ERR_INVALID, "null cache");
    const l2d_kv_cache &k = *cache;
    if (!valid_dtype(k.dtype)) return set_error(L2D_ERR_INVALID, "bad dtype %d", k.dtype);
    if (k.heads < 1 || k.heads > 65535) return set_error(L2D_ERR_INVALID, "%d key-value heads", k.heads);
    if (k.head_dim < 1 || k.head_dim > kMaxHeadDim)
        return set_error(L2D_ERR_UNSUPPORTED, "head_dim %d: 1 to %d are supported", k.head_dim, kMaxHeadDim);
    if (k.page_size < 1 || k.num_pages < 0 || k.num_pages > INT32_MAX)
        return set_error(L2D_ERR_INVALID, "%lld pages of %d slots", static_cast<long long>(k.num_pages), k.page_size);
    if (k.num_seqs < 0 || k.table_width < 0) return set_error(L2D_ERR_INVALID, "page table of %d x %d", k.num_seqs, k.table_width);
    if (int64_t(k.table_width) * k.page_size > INT32_MAX)
        return set_error(L2D_ERR_INVALID, "positions of a sequence (%d pages of %d) must stay below 2^31", k.table_width, k.page_size);
    c->k = static_cast<char *>(k.k);
    c->v = static_cast<char *>(k.v);
    const int64_t slot = int64_t(k.heads) * k.head_dim;
    c->k_head = k.k_head ? k.k_head : k.head_dim;
    c->v_head = k.v_head ? k.v_head : k.head_dim;
    c->k_slot = k.k_slot ? k.k_slot : slot;
    c->v_slot = k.v_slot ? k.v_slot : slot;
    c->k_page = k.k_page ? k.k_page : slot * k.page_size;
    c->v_page = k.v_page ? k.v_page : slot * k.page_size;
    c->table = k.table;
    c->table_stride = k.table_stride ? k.table_stride : k.table_width;
    c->num_pages = k.num_pages;
    c->num_seqs = k.num_seqs;
    c->table_width = k.table_width;
    c->page_size = k.page_size;
    c->page_shift = k.page_size & (k.page_size - 1) ? -1 : __builtin_ctz(static_cast<unsigned>(k.page_size));
    c->heads = k.heads;
    c->head_dim = k.head_dim;
    c->status = k.status;
    const int64_t least = std::min({c->k_head, c->v_head, c->k_slot, c->v_slot, c->k_page, c->v_page});
    if (least < k.head_dim || c->table_stride < k.table_width)
        return set_error(L2D_ERR_INVALID, "cache strides overlap (the least of them is %lld elements)", static_cast<long long>(least));
    const int64_t most = std::max({c->k_page, c->v_page, c->k_slot, c->v_slot, c->k_head, c->v_head, c->table_stride});
    if (most > (int64_t(1) << 40)) return set_error(L2D_ERR_INVALID, "cache strides too large");
    const bool used = k.num_seqs && k.table_width;  // the table is read then, and pages where there are any
    if (used && (!k.table || (k.num_pages && (!k.k || !k.v)))) return set_error(L2D_ERR_INVALID, "null cache pointer");
    const uintptr_t align = elem_bytes(k.dtype) - 1;
    if ((reinterpret_cast<uintptr_t>(k.k) & align) || (reinterpret_cast<uintptr_t>(k.v) & align) ||
        (reinterpret_cast<uintptr_t>(k.table) & 3) || (reinterpret_cast<uintptr_t>(k.status) & 3))
        return set_error(L2D_ERR_INVALID, "cache pointers must be aligned to their elements");
    return L2D_OK;
}

}  // namespace l2d

using namespace l2d;

namespace l2d {

// A tensor map over keys or values: boxes of 128 bytes by `keys` slots of one head in one page.  Fetching 256 bytes
// at a time into L2 costs 20 % where a row has only 128 (32 x 4096 keys of 64 fp16 elements: 127 us, 104 us without).
bool encode_map(CUtensorMap *map, void *base, int dtype, const Cache &c, int64_t head, int64_t slot, int64_t page, int keys) {
    static const auto encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(f);
    }();
    if (!encode) return false;
    const cuuint64_t eb = elem_bytes(dtype);
    const cuuint64_t sizes[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.heads), static_cast<cuuint64_t>(c.page_size),
                                 static_cast<cuuint64_t>(c.num_pages)};
    const cuuint64_t strides[3] = {head * eb, slot * eb, page * eb};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / eb), 1, static_cast<cuuint32_t>(keys), 1}, ones[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = dtype == L2D_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == L2D_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 4, base, sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  c.head_dim * eb >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace l2d

struct l2d_attn_plan {
    Cache cache;
    l2d_attn_desc desc;
    int dtype, device, grid, m_tiles;
    int how;
    AttnMaps maps;
    AttnKernel kernel;
    AttnScratch scratch;
    void *memory;
};

extern "C" {

int l2d_kv_append(const l2d_kv_cache *cache, const l2d_append_desc *desc, const void *k, const void *v, const void *q,
                  void *q_out, const int32_t *pos, const int32_t *seq, int64_t tokens, void *stream) {
    AppendArgs a = {};
    int st = check_cache(cache, &a.c);
    if (st != L2D_OK) return st;
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    const l2d_append_desc &d = *desc;
    const int D = cache->head_dim;
    if (d.heads_q < 0 || d.heads_q > 65535) return set_error(L2D_ERR_INVALID, "%d query heads", d.heads_q);
    if (d.rot_dim < 0 || d.rot_dim > D || d.rot_dim % 2)
        return set_error(L2D_ERR_INVALID, "rot_dim %d: an even number up to head_dim = %d", d.rot_dim, D);
    if (tokens < 0) return set_error(L2D_ERR_INVALID, "%lld tokens", static_cast<long long>(tokens));
    const int64_t kv_row = int64_t(cache->heads) * D, q_row = int64_t(d.heads_q) * D;
    a.k_token = d.k_token ? d.k_token : kv_row;
    a.v_token = d.v_token ? d.v_token : kv_row;
    a.q_token = d.q_token ? d.q_token : q_row;
    a.q_out_token = d.q_out_token ? d.q_out_token : q_row;
    if (a.k_token < kv_row || a.v_token < kv_row || a.q_token < q_row || a.q_out_token < q_row)
        return set_error(L2D_ERR_INVALID, "a token's stride is shorter than its heads");
    if (tokens && std::max({a.k_token, a.v_token, a.q_token, a.q_out_token}) > (int64_t(1) << 58) / tokens)
        return set_error(L2D_ERR_INVALID, "token strides too large");
    if (!seq && tokens > cache->num_seqs)
        return set_error(L2D_ERR_INVALID, "%lld tokens without seq, and a page table of %d sequences", static_cast<long long>(tokens), cache->num_seqs);
    if (tokens == 0) return L2D_OK;
    if (!k || !v || !pos || (d.heads_q && (!q || !q_out)) || (d.rot_dim && (!d.cos || !d.sin)))
        return set_error(L2D_ERR_INVALID, "null pointer");
    const int eb = elem_bytes(cache->dtype);
    if (misaligned(k, eb) || misaligned(v, eb) || misaligned(q, eb) || misaligned(q_out, eb) || misaligned(pos, 4) ||
        misaligned(seq, 4) || misaligned(d.cos, 4) || misaligned(d.sin, 4))
        return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    if (d.heads_q && q == q_out && tokens > 1 && a.q_token != a.q_out_token)
        return set_error(L2D_ERR_INVALID, "q_out is q, but q_token is %lld and q_out_token %lld", static_cast<long long>(a.q_token),
                         static_cast<long long>(a.q_out_token));
    if (d.rot_dim && d.max_pos < 0) return set_error(L2D_ERR_INVALID, "max_pos %lld", static_cast<long long>(d.max_pos));
    int sms = 0;
    st = device_sms(cache->device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(cache->device);
    L2D_CUDA_TRY(on.err);
    a.k = k;
    a.v = v;
    a.q = q;
    a.q_out = q_out;
    a.cos = d.cos;
    a.sin = d.sin;
    a.pos = pos;
    a.seq = seq;
    a.tokens = tokens;
    a.max_pos = d.max_pos;
    a.heads_q = d.heads_q;
    a.rot_dim = d.rot_dim;
    a.interleaved = d.interleaved;
    // Units of 16-byte words where everything is aligned to them.
    const int vec = 16 / eb, half = d.rot_dim / 2;
    int64_t all = D | a.k_token | a.v_token | a.c.k_page | a.c.k_slot | a.c.k_head | a.c.v_page | a.c.v_slot | a.c.v_head | half;
    if (d.heads_q) all |= a.q_token | a.q_out_token;
    const bool words = all % vec == 0 && !misaligned(k, 16) && !misaligned(v, 16) && !misaligned(q, 16) && !misaligned(q_out, 16) &&
                       !misaligned(a.c.k, 16) && !misaligned(a.c.v, 16) && !misaligned(d.cos, 16) && !misaligned(d.sin, 16);
    const int each = words ? vec : 1, rot_units = half / each, units = rot_units + (D - d.rot_dim + 2 * each - 1) / (2 * each);
    // Heads of a token in one thread: all of them, or as few as it takes for two blocks a SM.
    const int heads = d.heads_q + 2 * cache->heads;
    const int64_t want = int64_t(sms) * 2 * kAppendThreads, have = tokens * units;
    const int rows = static_cast<int>(std::min<int64_t>(heads, std::max<int64_t>(1, (want + have - 1) / have)));
    const int64_t blocks = (have * rows + kAppendThreads - 1) / kAppendThreads;
    if (blocks > INT32_MAX) return set_error(L2D_ERR_INVALID, "%lld tokens are too many", static_cast<long long>(tokens));
    auto pick = [&](auto type) {
        using T = decltype(type);
        constexpr int kVec = 16 / sizeof(T);
        if (words) return d.interleaved ? k_append<T, kVec, true> : k_append<T, kVec, false>;
        return d.interleaved ? k_append<T, 1, true> : k_append<T, 1, false>;
    };
    auto kernel = cache->dtype == L2D_F32 ? pick(float()) : cache->dtype == L2D_F16 ? pick(__half()) : pick(__nv_bfloat16());
    L2D_CUDA_TRY(launch(kernel, dim3(static_cast<unsigned>(blocks)), kAppendThreads, 0, stream, a, units, rot_units, rows));
    return L2D_OK;
}

int l2d_attn_plan_create(const l2d_kv_cache *cache, const l2d_attn_desc *desc, l2d_attn_plan **plan) {
    if (!plan) return set_error(L2D_ERR_INVALID, "null plan pointer");
    *plan = nullptr;
    Cache c;
    int st = check_cache(cache, &c);
    if (st != L2D_OK) return st;
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    l2d_attn_desc d = *desc;
    if (d.heads_q < 1 || d.heads_q > 65535 || d.heads_q % cache->heads)
        return set_error(L2D_ERR_INVALID, "%d query heads for %d key-value heads", d.heads_q, cache->heads);
    if (d.window < 0) return set_error(L2D_ERR_INVALID, "window %d", d.window);
    if (!std::isfinite(d.scale)) return set_error(L2D_ERR_INVALID, "scale is not finite");
    if (!std::isfinite(d.scale * 1.4426950408889634f)) return set_error(L2D_ERR_INVALID, "scale %g is too large", d.scale);
    if (d.max_batch < 0 || d.max_batch > cache->num_seqs)
        return set_error(L2D_ERR_INVALID, "max_batch %d for a page table of %d sequences", d.max_batch, cache->num_seqs);
    if (!d.max_batch) d.max_batch = cache->num_seqs;
    if (int64_t(d.max_batch) * d.heads_q > INT32_MAX) return set_error(L2D_ERR_INVALID, "max_batch * heads_q must stay below 2^31");
    const int64_t row = int64_t(d.heads_q) * cache->head_dim;
    if (!d.q_token) d.q_token = row;
    if (!d.out_token) d.out_token = row;
    if (d.q_token < row || d.out_token < row) return set_error(L2D_ERR_INVALID, "a sequence's stride is shorter than its heads");
    if (std::max(d.q_token, d.out_token) > (int64_t(1) << 40)) return set_error(L2D_ERR_INVALID, "strides too large");
    if (d.scale == 0.0f) d.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(cache->head_dim)));
    int sms = 0;
    st = device_sms(cache->device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(cache->device);
    L2D_CUDA_TRY(on.err);
    const int G = d.heads_q / cache->heads;
    const AttnKernel k = pick_attn(cache->dtype, cache->head_dim, G);
    const int m_tiles = (G + k.rows - 1) / k.rows;
    int blocks = 0;
    L2D_CUDA_TRY(cudaFuncSetAttribute(k.run, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem));
    L2D_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, k.run, k.threads, k.smem));
    if (blocks < 1) return set_error(L2D_ERR_CUDA, "the attention kernel does not fit an SM");
    const int grid = sms * blocks;
    const size_t part = size_t(grid) * 2 * kMaxRows * k.dim * 4, ml = size_t(grid) * 4 * kMaxRows * 4;
    const size_t arrived = size_t(d.max_batch) * cache->heads * m_tiles * 4;
    void *memory = nullptr;
    L2D_CUDA_TRY(cudaMalloc(&memory, part + ml + arrived + 4));
    // The counters are set on a stream of their own, so that nothing else on the device is waited for.
    cudaStream_t own = nullptr;
    cudaError_t e = cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking);
    if (e == cudaSuccess) {
        e = cudaMemsetAsync(static_cast<char *>(memory) + part + ml, 0, arrived + 4, own);
        if (e == cudaSuccess) e = cudaStreamSynchronize(own);
        cudaStreamDestroy(own);
    }
    if (e != cudaSuccess) {
        cudaFree(memory);
        return set_error(L2D_ERR_CUDA, "attention scratch: %s", cudaGetErrorString(e));
    }
    l2d_attn_plan *p = new (std::nothrow) l2d_attn_plan();
    if (!p) {
        cudaFree(memory);
        return set_error(L2D_ERR_INVALID, "out of host memory");
    }
    char *base = static_cast<char *>(memory);
    p->cache = c;
    p->desc = d;
    p->dtype = cache->dtype;
    p->device = cache->device;
    p->grid = grid;
    p->m_tiles = m_tiles;
    p->kernel = k;
    p->scratch = {reinterpret_cast<float *>(base), reinterpret_cast<float *>(base + part), reinterpret_cast<unsigned *>(base + part + ml)};
    p->memory = memory;
    // 16-byte copies need rows of whole 16-byte words on 16-byte boundaries; boxes also pages of whole tiles.
    const int64_t eb = elem_bytes(cache->dtype);
    const int64_t any = cache->head_dim | c.k_page | c.k_slot | c.k_head | c.v_page | c.v_slot | c.v_head;
    p->how = (any * eb) % 16 || misaligned(c.k, 16) || misaligned(c.v, 16) ? kElements : kWords;
    if (p->how == kWords && cache->page_size % k.keys == 0 && c.num_pages > 0) {
        const bool ok = encode_map(&p->maps.k, c.k, cache->dtype, c, c.k_head, c.k_slot, c.k_page, k.keys) &&
                        encode_map(&p->maps.v, c.v, cache->dtype, c, c.v_head, c.v_slot, c.v_page, k.keys);
        if (ok) p->how = kBoxes;
    }
    *plan = p;
    return L2D_OK;
}

int l2d_attn_decode(l2d_attn_plan *p, const void *q, void *out, float *lse, const int32_t *lens, int batch, void *stream) {
    if (!p) return set_error(L2D_ERR_INVALID, "null plan");
    if (batch < 0 || batch > p->desc.max_batch) return set_error(L2D_ERR_INVALID, "batch %d of at most %d", batch, p->desc.max_batch);
    if (batch == 0) return L2D_OK;
    if (!q || !out || !lens) return set_error(L2D_ERR_INVALID, "null pointer");
    const int eb = elem_bytes(p->dtype);
    if (misaligned(q, eb) || misaligned(out, eb) || misaligned(lse, 4) || misaligned(lens, 4))
        return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    OnDevice on(p->device);
    L2D_CUDA_TRY(on.err);
    const bool q_aligned = !misaligned(q, 16) && (p->desc.q_token * eb) % 16 == 0 && (p->cache.head_dim * eb) % 16 == 0;
    // No more blocks than pieces the page table leaves room for.
    const int64_t room = int64_t(p->cache.table_width) * p->cache.page_size, tiles = (room + p->kernel.tile - 1) / p->kernel.tile;
    const int64_t most = (tiles <= kWholeTiles ? 1 : units_of(tiles)) * batch * p->cache.heads * p->m_tiles;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(p->grid, most)));
    AttnArgs a = {p->cache, q, out, lse, lens, p->desc.q_token, p->desc.out_token, p->desc.heads_q, p->desc.window, batch, p->desc.scale};
    L2D_CUDA_TRY(launch(p->kernel.run, grid, p->kernel.threads, p->kernel.smem, stream, a, p->maps, p->scratch, p->m_tiles, p->how, q_aligned));
    return L2D_OK;
}

int l2d_attn_plan_destroy(l2d_attn_plan *p) {
    if (!p) return L2D_OK;
    OnDevice on(p->device);
    cudaError_t e = cudaFree(p->memory);  // waits for the device
    delete p;
    if (e != cudaSuccess) return set_error(L2D_ERR_CUDA, "attn_plan_destroy: %s", cudaGetErrorString(e));
    return L2D_OK;
}

}  // extern "C"

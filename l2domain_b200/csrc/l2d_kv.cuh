// The paged cache as the kernels see it, and wide loads and stores.
#pragma once

#include "l2d_launch.cuh"

#include <cstring>

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
    int group, tile_bytes;  // of a cache in 4 bits: elements of a scale, bytes of 16 slots of one head
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

// ---------------------------------------------------------------------------------------------
// Appending.
//
// A copy with a few multiplications: every element is read once and written once.  A head is cut into units
// of VEC pairs (the rotated part: for the half layout VEC elements and their VEC partners, for the interleaved
// one 2 VEC elements side by side) and of 2 VEC elements (the rest, and values), so that a thread moves 32 bytes
// of 16-bit elements.  A thread keeps its unit's cosines and sines for as many heads of its token as the grid
// leaves it: heads are split over blocks only while there are too few tokens to fill the GPU.
// ---------------------------------------------------------------------------------------------

constexpr int kAppendThreads = 256;

// The first `heads` of a token: queries, keys, values.  units: rotated units of a head (rot_units), then plain ones.  A thread's unit is fixed; the threads of a token
// for which `rows` are left take every rows-th of its heads.
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void append_heads(const AppendArgs &a, unsigned block, int units, int rot_units, int rows, int heads) {
    const int D = a.c.head_dim, half = a.rot_dim / 2, hk = a.c.heads;
    const int64_t thread = static_cast<int64_t>(block) * kAppendThreads + threadIdx.x;
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

// How an append's heads are cut into units: of 16-byte words where everything is aligned to them (`words`).
struct AppendUnits {
    int units, rot_units;
};
inline AppendUnits append_units(bool words, int elem, int head_dim, int rot_dim) {
    const int each = words ? 16 / elem : 1, rot = rot_dim / 2 / each;
    return {rot + (head_dim - rot_dim + 2 * each - 1) / (2 * each), rot};
}

// Checks a cache description and fills in its strides (l2d_kv.cu).
int check_cache(const l2d_kv_cache *cache, Cache *c);
// The same of a cache in 4 bits (l2d_kv4.cu).
int check_cache4(const l2d_kv4_cache *cache, Cache *c);
// Checks what an append needs besides its cache and fills it in; `tokens` may be 0.
int check_append(const l2d_append_desc *desc, int dtype, int heads, int head_dim, int num_seqs, const void *k, const void *v, const void *q,
                 void *q_out, const int32_t *pos, const int32_t *seq, int64_t tokens, AppendArgs *a);

}  // namespace l2d

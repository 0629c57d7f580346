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

// Checks a cache description and fills in its strides (l2d_kv.cu).
int check_cache(const l2d_kv_cache *cache, Cache *c);
// The same of a cache in 4 bits (l2d_kv4.cu).
int check_cache4(const l2d_kv4_cache *cache, Cache *c);
// Checks what an append needs besides its cache and fills it in; `tokens` may be 0.
int check_append(const l2d_append_desc *desc, int dtype, int heads, int head_dim, int num_seqs, const void *k, const void *v, const void *q,
                 void *q_out, const int32_t *pos, const int32_t *seq, int64_t tokens, AppendArgs *a);

}  // namespace l2d

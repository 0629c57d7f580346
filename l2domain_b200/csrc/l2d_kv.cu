// The paged cache of keys and values: appending with rotation (l2d_kv_append) and attention of one new
// token per sequence over it (l2d_attn_*).
#include "l2d_launch.cuh"

#include <algorithm>
#include <cmath>
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

__device__ __forceinline__ void report(uint32_t *status, uint32_t bit) {
    if (status) atomicOr(status, bit);
}

// The page of position p of sequence s, or -1 if it has none.
__device__ __forceinline__ int64_t page_of(const Cache &c, int64_t s, int p) {
    const int i = p / c.page_size;
    if (s < 0 || s >= c.num_seqs || i >= c.table_width) return -1;
    const int32_t page = c.table[s * c.table_stride + i];
    return page >= 0 && page < c.num_pages ? page : -1;
}

// One block per token; a thread takes single elements (of a pair, the first one and its partner).
template <typename T>
__global__ void __launch_bounds__(256) k_append(AppendArgs a) {
    dev::wait_for_previous();
    const int D = a.c.head_dim, half = a.rot_dim / 2, hk = a.c.heads;
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int p = a.pos[t];
        if (p < 0) continue;
        if (a.rot_dim && p >= a.max_pos) {
            if (threadIdx.x == 0) report(a.c.status, L2D_KV_BAD_POSITION);
            continue;
        }
        const int64_t page = page_of(a.c, a.seq ? a.seq[t] : t, p);
        if (page < 0) {
            if (threadIdx.x == 0) report(a.c.status, L2D_KV_BAD_PAGE);
            continue;
        }
        const int slot = p % a.c.page_size;
        T *kc = reinterpret_cast<T *>(a.c.k) + page * a.c.k_page + slot * a.c.k_slot;
        T *vc = reinterpret_cast<T *>(a.c.v) + page * a.c.v_page + slot * a.c.v_slot;
        for (int e = threadIdx.x; e < hk * D; e += blockDim.x) {
            const int h = e / D, i = e - h * D;
            vc[h * a.c.v_head + i] = static_cast<const T *>(a.v)[t * a.v_token + e];
        }
        for (int e = threadIdx.x; e < (a.heads_q + hk) * D; e += blockDim.x) {
            const int hh = e / D, i = e - hh * D;
            const bool is_q = hh < a.heads_q;
            const int h = is_q ? hh : hh - a.heads_q;
            const T *src = is_q ? static_cast<const T *>(a.q) + t * a.q_token + int64_t(h) * D
                                : static_cast<const T *>(a.k) + t * a.k_token + int64_t(h) * D;
            T *dst = is_q ? static_cast<T *>(a.q_out) + t * a.q_out_token + int64_t(h) * D : kc + h * a.c.k_head;
            if (i >= a.rot_dim) {
                dst[i] = src[i];
                continue;
            }
            if (a.interleaved ? (i & 1) : i >= half) continue;
            const int j = a.interleaved ? i + 1 : i + half, r = a.interleaved ? i / 2 : i;
            const float c = a.cos[int64_t(p) * half + r], s = a.sin[int64_t(p) * half + r];
            const float u = dev::widen(src[i]), w = dev::widen(src[j]);
            dst[i] = dev::narrow<T>(fmaf(u, c, -(w * s)));
            dst[j] = dev::narrow<T>(fmaf(w, c, u * s));
        }
    }
}

// One block of four warps per sequence and query head; a warp takes every fourth key, a lane every 32nd
// element of the head; the warps' parts meet in shared memory.
template <typename T>
__global__ void __launch_bounds__(128) k_attn(AttnArgs a) {
    dev::wait_for_previous();
    const int D = a.c.head_dim, h = blockIdx.x % a.heads_q, b = blockIdx.x / a.heads_q;
    const int hk = h / (a.heads_q / a.c.heads), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int E = kMaxHeadDim / 32;
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = lane + 32 * e;
        q[e] = i < D ? dev::widen(static_cast<const T *>(a.q)[b * a.q_token + int64_t(h) * D + i]) * a.scale : 0.0f;
        o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    int64_t len = a.lens[b];
    const int64_t room = int64_t(a.c.table_width) * a.c.page_size;
    if (len > room) {
        len = room;
        if (threadIdx.x == 0) report(a.c.status, L2D_KV_BAD_PAGE);
    }
    for (int64_t p = (a.window && len > a.window ? len - a.window : 0) + warp; p < len; p += 4) {
        const int64_t page = page_of(a.c, b, static_cast<int>(p));
        if (page < 0) {
            if (lane == 0) report(a.c.status, L2D_KV_BAD_PAGE);
            continue;
        }
        const int slot = static_cast<int>(p % a.c.page_size);
        const T *k = reinterpret_cast<const T *>(a.c.k) + page * a.c.k_page + slot * a.c.k_slot + hk * a.c.k_head;
        const T *v = reinterpret_cast<const T *>(a.c.v) + page * a.c.v_page + slot * a.c.v_slot + hk * a.c.v_head;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < D) s = fmaf(q[e], dev::widen(k[lane + 32 * e]), s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float m2 = fmaxf(m, s), base = m2 == -INFINITY ? 0.0f : m2;
        const float f = expf(m - base), w = expf(s - base);
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < D) o[e] = fmaf(w, dev::widen(v[lane + 32 * e]), o[e] * f);
        m = m2;
    }
    __shared__ float part[4][kMaxHeadDim], pm[4], pl[4];
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][lane + 32 * e] = o[e];
    if (lane == 0) {
        pm[warp] = m;
        pl[warp] = l;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = expf(pm[w] - base);
        sum += f[w] * pl[w];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int i = threadIdx.x; i < D; i += 128) {
        float r = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) r = fmaf(f[w], part[w][i], r);
        static_cast<T *>(a.out)[b * a.out_token + int64_t(h) * D + i] = dev::narrow<T>(r * inv);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[int64_t(b) * a.heads_q + h] = sum == 0.0f ? -INFINITY : base + logf(sum);
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
    c->heads = k.heads;
    c->head_dim = k.head_dim;
    c->status = k.status;
    const int64_t least = std::min({c->k_head, c->v_head, c->k_slot, c->v_slot, c->k_page, c->v_page});
    if (least < k.head_dim || c->table_stride < k.table_width)
        return set_error(L2D_ERR_INVALID, "cache strides overlap (the least of them is %lld elements)", static_cast<long long>(least));
    const int64_t most = std::max({c->k_page, c->v_page, c->k_slot, c->v_slot, c->k_head, c->v_head, c->table_stride});
    if (most > (int64_t(1) << 40)) return set_error(L2D_ERR_INVALID, "cache strides too large");
    const bool used = k.num_seqs && k.table_width && k.num_pages;
    if (used && (!k.k || !k.v || !k.table)) return set_error(L2D_ERR_INVALID, "null cache pointer");
    const uintptr_t align = elem_bytes(k.dtype) - 1;
    if ((reinterpret_cast<uintptr_t>(k.k) & align) || (reinterpret_cast<uintptr_t>(k.v) & align) ||
        (reinterpret_cast<uintptr_t>(k.table) & 3) || (reinterpret_cast<uintptr_t>(k.status) & 3))
        return set_error(L2D_ERR_INVALID, "cache pointers must be aligned to their elements");
    return L2D_OK;
}

bool misaligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace l2d

using namespace l2d;

struct l2d_attn_plan {
    Cache cache;
    l2d_attn_desc desc;
    int dtype, device, sms;
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
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(tokens, int64_t(sms) * 64)));
    auto kernel = cache->dtype == L2D_F32 ? k_append<float> : cache->dtype == L2D_F16 ? k_append<__half> : k_append<__nv_bfloat16>;
    L2D_CUDA_TRY(launch(kernel, grid, 256, 0, stream, a));
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
    l2d_attn_plan *p = new (std::nothrow) l2d_attn_plan();
    if (!p) return set_error(L2D_ERR_INVALID, "out of host memory");
    p->cache = c;
    p->desc = d;
    p->dtype = cache->dtype;
    p->device = cache->device;
    p->sms = sms;
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
    AttnArgs a = {p->cache, q, out, lse, lens, p->desc.q_token, p->desc.out_token, p->desc.heads_q, p->desc.window, batch, p->desc.scale};
    const dim3 grid(static_cast<unsigned>(batch) * p->desc.heads_q);
    auto kernel = p->dtype == L2D_F32 ? k_attn<float> : p->dtype == L2D_F16 ? k_attn<__half> : k_attn<__nv_bfloat16>;
    L2D_CUDA_TRY(launch(kernel, grid, 128, 0, stream, a));
    return L2D_OK;
}

int l2d_attn_plan_destroy(l2d_attn_plan *p) {
    delete p;
    return L2D_OK;
}

}  // extern "C"

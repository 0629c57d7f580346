// The paged cache of keys and values: appending with rotation (l2d_kv_append) and attention of one new
// token per sequence over it (l2d_attn_*).
#include "l2d_attn.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <new>

namespace l2d {

template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads) k_append(const __grid_constant__ AppendArgs a, int units, int rot_units, int rows) {
    dev::wait_for_previous();
    append_heads<T, VEC, INTERLEAVED>(a, blockIdx.x, units, rot_units, rows, a.heads_q + 2 * a.c.heads);
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

int check_append(const l2d_append_desc *desc, int dtype, int heads, int head_dim, int num_seqs, const void *k, const void *v, const void *q,
                 void *q_out, const int32_t *pos, const int32_t *seq, int64_t tokens, AppendArgs *args) {
    AppendArgs &a = *args;
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    const l2d_append_desc &d = *desc;
    if (d.heads_q < 0 || d.heads_q > 65535) return set_error(L2D_ERR_INVALID, "%d query heads", d.heads_q);
    if (d.rot_dim < 0 || d.rot_dim > head_dim || d.rot_dim % 2)
        return set_error(L2D_ERR_INVALID, "rot_dim %d: an even number up to head_dim = %d", d.rot_dim, head_dim);
    if (tokens < 0) return set_error(L2D_ERR_INVALID, "%lld tokens", static_cast<long long>(tokens));
    const int64_t kv_row = int64_t(heads) * head_dim, q_row = int64_t(d.heads_q) * head_dim;
    a.k_token = d.k_token ? d.k_token : kv_row;
    a.v_token = d.v_token ? d.v_token : kv_row;
    a.q_token = d.q_token ? d.q_token : q_row;
    a.q_out_token = d.q_out_token ? d.q_out_token : q_row;
    if (a.k_token < kv_row || a.v_token < kv_row || a.q_token < q_row || a.q_out_token < q_row)
        return set_error(L2D_ERR_INVALID, "a token's stride is shorter than its heads");
    if (tokens && std::max({a.k_token, a.v_token, a.q_token, a.q_out_token}) > (int64_t(1) << 58) / tokens)
        return set_error(L2D_ERR_INVALID, "token strides too large");
    if (!seq && tokens > num_seqs)
        return set_error(L2D_ERR_INVALID, "%lld tokens without seq, and a page table of %d sequences", static_cast<long long>(tokens), num_seqs);
    if (tokens == 0) return L2D_OK;
    if (!k || !v || !pos || (d.heads_q && (!q || !q_out)) || (d.rot_dim && (!d.cos || !d.sin)))
        return set_error(L2D_ERR_INVALID, "null pointer");
    const int eb = elem_bytes(dtype);
    if (misaligned(k, eb) || misaligned(v, eb) || misaligned(q, eb) || misaligned(q_out, eb) || misaligned(pos, 4) ||
        misaligned(seq, 4) || misaligned(d.cos, 4) || misaligned(d.sin, 4))
        return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    if (d.heads_q && q == q_out && tokens > 1 && a.q_token != a.q_out_token)
        return set_error(L2D_ERR_INVALID, "q_out is q, but q_token is %lld and q_out_token %lld", static_cast<long long>(a.q_token),
                         static_cast<long long>(a.q_out_token));
    if (d.rot_dim && d.max_pos < 0) return set_error(L2D_ERR_INVALID, "max_pos %lld", static_cast<long long>(d.max_pos));
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
    return L2D_OK;
}

}  // namespace l2d

struct l2d_attn_plan {
    Cache cache;
    l2d_attn_desc desc;
    l2d_attn_scores scores;
    int dtype, device, grid, m_tiles;
    int how;
    AttnMaps maps;
    AttnKernel kernel;
    AttnScratch scratch;
    void *memory;
};

namespace l2d {

AttnKernel pick_attn(int dtype, int D, int G) { return pick_dense<false>(dtype, D, G); }

// A plan over a checked cache, without its way of copying.
int make_plan(const Cache &c, int dtype, int device, const l2d_attn_desc *desc, const l2d_attn_scores *scores, l2d_attn_plan **plan) {
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    l2d_attn_desc d = *desc;
    if (d.heads_q < 1 || d.heads_q > 65535 || d.heads_q % c.heads)
        return set_error(L2D_ERR_INVALID, "%d query heads for %d key-value heads", d.heads_q, c.heads);
    if (d.window < 0) return set_error(L2D_ERR_INVALID, "window %d", d.window);
    if (!std::isfinite(d.scale)) return set_error(L2D_ERR_INVALID, "scale is not finite");
    if (!std::isfinite(d.scale * 1.4426950408889634f)) return set_error(L2D_ERR_INVALID, "scale %g is too large", d.scale);
    if (d.max_batch < 0 || d.max_batch > c.num_seqs)
        return set_error(L2D_ERR_INVALID, "max_batch %d for a page table of %d sequences", d.max_batch, c.num_seqs);
    if (!d.max_batch) d.max_batch = c.num_seqs;
    if (int64_t(d.max_batch) * d.heads_q > INT32_MAX) return set_error(L2D_ERR_INVALID, "max_batch * heads_q must stay below 2^31");
    const int64_t row = int64_t(d.heads_q) * c.head_dim;
    if (!d.q_token) d.q_token = row;
    if (!d.out_token) d.out_token = row;
    if (d.q_token < row || d.out_token < row) return set_error(L2D_ERR_INVALID, "a sequence's stride is shorter than its heads");
    if (std::max(d.q_token, d.out_token) > (int64_t(1) << 40)) return set_error(L2D_ERR_INVALID, "strides too large");
    const l2d_attn_scores s = scores ? *scores : l2d_attn_scores{};
    if (!(s.cap == 0.0f || (s.cap >= FLT_MIN && std::isfinite(s.cap * 1.4426950408889634f))))
        return set_error(L2D_ERR_INVALID, "cap %g: 0 or a positive number whose reciprocal and logarithm's base leave it one", s.cap);
    if (misaligned(s.slopes, 4)) return set_error(L2D_ERR_INVALID, "slopes must be aligned to their elements");
    if (d.scale == 0.0f) d.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(c.head_dim)));
    int sms = 0;
    int st = device_sms(device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(device);
    L2D_CUDA_TRY(on.err);
    const int G = d.heads_q / c.heads;
    const bool scored = s.cap != 0.0f || s.slopes;
    const AttnKernel k = c.group ? pick_attn_kv4(dtype, c.head_dim, c.group, G) : scored ? pick_attn_scored(dtype, c.head_dim, G) : pick_attn(dtype, c.head_dim, G);
    if (!std::isfinite(d.scale * 1.4426950408889634f * k.scale)) return set_error(L2D_ERR_INVALID, "scale %g is too large", d.scale);
    const int m_tiles = (G + k.rows - 1) / k.rows;
    int blocks = 0;
    L2D_CUDA_TRY(cudaFuncSetAttribute(k.run, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem));
    L2D_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, k.run, k.threads, k.smem));
    if (blocks < 1) return set_error(L2D_ERR_CUDA, "the attention kernel does not fit an SM");
    const int grid = sms * blocks;
    const size_t part = size_t(grid) * 2 * kMaxRows * k.dim * 4, ml = size_t(grid) * 4 * kMaxRows * 4;
    const size_t arrived = size_t(d.max_batch) * c.heads * m_tiles * 4;
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
    p->scores = s;
    p->dtype = dtype;
    p->device = device;
    p->grid = grid;
    p->m_tiles = m_tiles;
    p->kernel = k;
    p->scratch = {reinterpret_cast<float *>(base), reinterpret_cast<float *>(base + part), reinterpret_cast<unsigned *>(base + part + ml)};
    p->memory = memory;
    *plan = p;
    return L2D_OK;
}

}  // namespace l2d

extern "C" {

int l2d_kv_append(const l2d_kv_cache *cache, const l2d_append_desc *desc, const void *k, const void *v, const void *q,
                  void *q_out, const int32_t *pos, const int32_t *seq, int64_t tokens, void *stream) {
    AppendArgs a = {};
    int st = check_cache(cache, &a.c);
    if (st != L2D_OK) return st;
    st = check_append(desc, cache->dtype, cache->heads, cache->head_dim, cache->num_seqs, k, v, q, q_out, pos, seq, tokens, &a);
    if (st != L2D_OK || tokens == 0) return st;
    const l2d_append_desc &d = *desc;
    const int D = cache->head_dim, eb = elem_bytes(cache->dtype);
    int sms = 0;
    st = device_sms(cache->device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(cache->device);
    L2D_CUDA_TRY(on.err);
    // Units of 16-byte words where everything is aligned to them.
    const int vec = 16 / eb, half = d.rot_dim / 2;
    int64_t all = D | a.k_token | a.v_token | a.c.k_page | a.c.k_slot | a.c.k_head | a.c.v_page | a.c.v_slot | a.c.v_head | half;
    if (d.heads_q) all |= a.q_token | a.q_out_token;
    const bool words = all % vec == 0 && !misaligned(k, 16) && !misaligned(v, 16) && !misaligned(q, 16) && !misaligned(q_out, 16) &&
                       !misaligned(a.c.k, 16) && !misaligned(a.c.v, 16) && !misaligned(d.cos, 16) && !misaligned(d.sin, 16);
    const auto [units, rot_units] = append_units(words, eb, D, d.rot_dim);
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
    return l2d_attn_plan_create_scored(cache, desc, nullptr, plan);
}

int l2d_attn_plan_create_scored(const l2d_kv_cache *cache, const l2d_attn_desc *desc, const l2d_attn_scores *scores, l2d_attn_plan **plan) {
    if (!plan) return set_error(L2D_ERR_INVALID, "null plan pointer");
    *plan = nullptr;
    Cache c;
    int st = check_cache(cache, &c);
    if (st != L2D_OK) return st;
    c.group = 0;
    st = make_plan(c, cache->dtype, cache->device, desc, scores, plan);
    if (st != L2D_OK) return st;
    l2d_attn_plan *p = *plan;
    // 16-byte copies need rows of whole 16-byte words on 16-byte boundaries; boxes also pages of whole tiles.
    const int64_t eb = elem_bytes(cache->dtype);
    const int64_t any = cache->head_dim | c.k_page | c.k_slot | c.k_head | c.v_page | c.v_slot | c.v_head;
    p->how = (any * eb) % 16 || misaligned(c.k, 16) || misaligned(c.v, 16) ? kElements : kWords;
    if (p->how == kWords && cache->page_size % p->kernel.keys == 0 && c.num_pages > 0) {
        const bool ok = encode_map(&p->maps.k, c.k, cache->dtype, c, c.k_head, c.k_slot, c.k_page, p->kernel.keys) &&
                        encode_map(&p->maps.v, c.v, cache->dtype, c, c.v_head, c.v_slot, c.v_page, p->kernel.keys);
        if (ok) p->how = kBoxes;
    }
    return L2D_OK;
}

int l2d_attn_plan_create_kv4(const l2d_kv4_cache *cache, const l2d_attn_desc *desc, const l2d_attn_scores *scores, l2d_attn_plan **plan) {
    if (!plan) return set_error(L2D_ERR_INVALID, "null plan pointer");
    *plan = nullptr;
    Cache c;
    const int st = check_cache4(cache, &c);
    if (st != L2D_OK) return st;
    return make_plan(c, cache->dtype, cache->device, desc, scores, plan);
}

int l2d_attn_decode(l2d_attn_plan *p, const void *q, void *out, float *lse, const int32_t *lens, int batch, void *stream) {
    return l2d_attn_decode_from(p, q, out, lse, lens, nullptr, batch, stream);
}

int l2d_attn_decode_from(l2d_attn_plan *p, const void *q, void *out, float *lse, const int32_t *lens, const int32_t *starts, int batch, void *stream) {
    if (!p) return set_error(L2D_ERR_INVALID, "null plan");
    if (batch < 0 || batch > p->desc.max_batch) return set_error(L2D_ERR_INVALID, "batch %d of at most %d", batch, p->desc.max_batch);
    if (batch == 0) return L2D_OK;
    if (!q || !out || !lens) return set_error(L2D_ERR_INVALID, "null pointer");
    const int eb = elem_bytes(p->dtype);
    if (misaligned(q, eb) || misaligned(out, eb) || misaligned(lse, 4) || misaligned(lens, 4) || misaligned(starts, 4))
        return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    OnDevice on(p->device);
    L2D_CUDA_TRY(on.err);
    const bool q_aligned = !misaligned(q, 16) && (p->desc.q_token * eb) % 16 == 0 && (p->cache.head_dim * eb) % 16 == 0;
    // No more blocks than pieces the page table leaves room for.
    const int64_t room = int64_t(p->cache.table_width) * p->cache.page_size, tiles = (room + p->kernel.tile - 1) / p->kernel.tile;
    const int64_t most = (tiles <= p->kernel.whole_tiles ? 1 : units_of(tiles, p->kernel.before)) * batch * p->cache.heads * p->m_tiles;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(p->grid, most)));
    AttnArgs a = {p->cache, q, out, lse, lens, p->desc.q_token, p->desc.out_token, p->desc.heads_q, p->desc.window, batch, p->desc.scale, starts,
                  p->scores.cap, p->scores.slopes};
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
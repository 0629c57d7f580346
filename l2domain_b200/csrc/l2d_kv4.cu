// The paged cache in 4 bits: appending to it (l2d_kv4_append), and its checks.
#include "l2d_kv4.cuh"

#include <algorithm>

namespace l2d {

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

AttnKernel pick_attn_kv4(int dtype, int D, int group, int G) {
    if (dtype == L2D_F16) return pick_kv4_half(D, group, G);
    return dtype == L2D_BF16 ? pick_kv4_bf16(D, group, G) : pick_kv4_float(D, group, G);
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

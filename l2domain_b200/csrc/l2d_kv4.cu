// The paged cache in 4 bits: appending to it (l2d_kv4_append), and its checks.
#include "l2d_kv4.cuh"

#include <algorithm>

namespace l2d {

// ---------------------------------------------------------------------------------------------
// Appending.
//
// Queries are rotated as beside a cache of 16 or 32 bits.  Keys and values: a copy with a maximum and a minimum per group in
// between.  A thread has eight
// elements of a row (one word of nibbles), the threads of a row, a power of two of them, are neighbours in a warp and
// meet by shuffles; a thread keeps its angles for as many heads of its token as the grid leaves it.  Products,
// sums and quotients are rounded one by one to fp32, so that what is stored follows from the inputs and not from how an
// expression was compiled.
//
// Measured (32 query and 8 key-value heads of 128): 8192 tokens of fp16 in groups of 32, with what is held written out, 64 us,
// 3.4 TB/s, for 34 us of bytes; 32 tokens 6 us, of which a launch 4.1.  Some 400 warp instructions per 256 elements use half of the
// issue slots; what binds is the loads of the next head, which begin after this one is stored.  bf16 takes 98 us: at the 80
// registers of three blocks a SM its kernels spill 172 bytes and more a thread, those of fp16 16 (67 us with four blocks).
// ---------------------------------------------------------------------------------------------

// Two numbers at a time, each rounded as by itself.
__device__ __forceinline__ unsigned long long bits_of(float2 v) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 two_of(unsigned long long b) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(b));
    return v;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return two_of(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return two_of(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
    return two_of(r);
}

struct Append4Args {
    AppendArgs a;
    void *k_out, *v_out;
};

// Eight elements from p on, of which those at d, d + 1, .. below D are real; by 16-byte words where WORDS.
template <typename T, bool WORDS>
__device__ __forceinline__ Pack<T, 8> load8(const T *p, int d, int D) {
    Pack<T, 8> r;
    if constexpr (WORDS) {
        if (d < D) return load_pack<T, 8>(p);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = d + i < D ? p[i] : dev::narrow<T>(0.0f);
    return r;
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
__device__ __forceinline__ void append4(const Append4Args &args, unsigned block_at, int lanes, int rows) {
    const AppendArgs &a = args.a;
    const int D = a.c.head_dim, half = a.rot_dim / 2, hk = a.c.heads;
    const int64_t thread = static_cast<int64_t>(block_at) * kAppendThreads + threadIdx.x;
    const int64_t t = quotient(thread, lanes * rows);
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

    // The angles of this thread's elements, and where the other elements of their pairs are: the second halves' angles
    // turn the other way.
    const bool rotated = d < a.rot_dim;
    float cs[8], sn[8];
    int other[WORDS ? 1 : 8] = {};
    if (rotated) {
        const float *cos = a.cos + static_cast<int64_t>(p) * half, *sin = a.sin + static_cast<int64_t>(p) * half;
        if constexpr (WORDS && !INTERLEAVED) {
            const bool second = d >= half;
            const Pack<float, 8> c8 = load_pack<float, 8>(cos + (second ? d - half : d)), s8 = load_pack<float, 8>(sin + (second ? d - half : d));
#pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = c8.v[i], sn[i] = second ? s8.v[i] : -s8.v[i];
            other[0] = second ? -half : half;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = d + i;
                const bool in = e < a.rot_dim, second = INTERLEAVED ? e & 1 : e >= half;
                const int pair = INTERLEAVED ? e / 2 : second ? e - half : e;
                cs[i] = in ? cos[pair] : 1.0f;
                sn[i] = in ? (second ? sin[pair] : -sin[pair]) : 0.0f;
                if constexpr (!WORDS) other[i] = !in ? 0 : second ? -half : half;
            }
        }
    }
    // This thread's elements of a head at src, and the others of their pairs.
    auto load = [&](Pack<T, 8> &own, Pack<T, 8> &pair, const T *src, bool turn) {
        own = load8<T, WORDS>(src, d, D);
        if constexpr (!INTERLEAVED) {
            if (!turn || !rotated) return;
            if constexpr (WORDS) {
                pair = load_pack<T, 8>(src + other[0]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) pair.v[i] = d + i < D ? src[i + other[i]] : dev::narrow<T>(0.0f);
            }
        }
    };
    auto rotate = [&](float (&x)[8], const Pack<T, 8> &own, const Pack<T, 8> &pair) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float2 u = make_float2(dev::widen(own.v[i]), dev::widen(own.v[i + 1]));
            if (rotated) {
                const float2 y = INTERLEAVED ? make_float2(u.y, u.x) : make_float2(dev::widen(pair.v[i]), dev::widen(pair.v[i + 1]));
                // (The sum of two products taken as one multiply-add would be rounded once.)
                const float2 one = mul2(u, make_float2(cs[i], cs[i + 1])), two = mul2(y, make_float2(sn[i], sn[i + 1]));
                const float2 turned = make_float2(__fadd_rn(one.x, two.x), __fadd_rn(one.y, two.y));
                if (WORDS || d + i < a.rot_dim) u.x = turned.x;
                if (WORDS || d + i + 1 < a.rot_dim) u.y = turned.y;
            }
            x[i] = u.x;
            x[i + 1] = u.y;
        }
    };
    // Holds a head's elements x in the tile, and leaves in x what they stand for.
    auto hold = [&](float (&x)[8], char *tile) {
        float lo = 0.0f, hi = 0.0f;
        float2 odd = make_float2(0.0f, 0.0f);  // 0 times an infinity or a NaN is one
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            lo = fminf(lo, fminf(x[i], x[i + 1]));
            hi = fmaxf(hi, fmaxf(x[i], x[i + 1]));
            odd = fma2(make_float2(x[i], x[i + 1]), make_float2(0.0f, 0.0f), odd);
        }
        if (!(odd.x + odd.y == 0.0f)) hi = INFINITY;
        for (int m = 1; m < meet; m <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(mine, lo, m));
            hi = fmaxf(hi, __shfl_xor_sync(mine, hi, m));
        }
        constexpr float kFifteenth = 1.0f / 15.0f;
        uint32_t word = (__float_as_uint(__fsub_rn(__fmul_rn(hi, kFifteenth), __fmul_rn(lo, kFifteenth))) + 15u) & ~15u;
        const bool bad = hi == INFINITY;
        const float by = word == 0 ? 1.0f : __uint_as_float(word), inverse = 1.0f / by;
        float z = fminf(rintf(__fdiv_rn(-lo, by)), 15.0f), s = __uint_as_float(word);
        // x / s rounded to a whole number.  By the reciprocal it is off by less than 2^-19, two roundings of up to 15, and the
        // quotient rounded to fp32, which decides, by 2^-20 more: where a half is nearer than 2^-17, and where the reciprocal is no
        // number, the quotient itself is taken.  Adding 1.5 * 2^23 rounds to whole numbers.
        constexpr float kWhole = 12582912.0f;
        float2 near[4];
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 r = mul2(make_float2(x[2 * i], x[2 * i + 1]), make_float2(inverse, inverse));
            near[i] = add2(add2(r, make_float2(kWhole, kWhole)), make_float2(-kWhole, -kWhole));
            const float2 off = fma2(near[i], make_float2(-1.0f, -1.0f), r);
            far = fmaxf(far, fmaxf(fabsf(off.x), fabsf(off.y)));
        }
        if (!(far < 0.5f - 0x1p-17f) || !(inverse <= FLT_MAX)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) near[i] = make_float2(rintf(__fdiv_rn(x[2 * i], by)), rintf(__fdiv_rn(x[2 * i + 1], by)));
        }
        if (bad) {  // every number is 0, and stands for NaN
            word = 0x7fc00000u;
            s = __uint_as_float(word);
            z = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) near[i] = make_float2(0.0f, 0.0f);
        }
        // Four numbers of 0..15 are one below 2^16.
        float four[2] = {};
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            float2 n = add2(near[i], make_float2(z, z));
            n = make_float2(fminf(fmaxf(n.x, 0.0f), 15.0f), fminf(fmaxf(n.y, 0.0f), 15.0f));
            if (!WORDS) n = make_float2(d + 2 * i < D ? n.x : 0.0f, d + 2 * i + 1 < D ? n.y : 0.0f);
            four[i / 2] = fmaf(four[i / 2], 16.0f, n.y);
            four[i / 2] = fmaf(four[i / 2], 16.0f, n.x);
            const float2 stands = mul2(make_float2(s, s), add2(n, make_float2(-z, -z)));
            x[2 * i] = stands.x;
            x[2 * i + 1] = stands.y;
        }
        const uint32_t nibbles = __byte_perm(__float_as_uint(four[0] + kWhole), __float_as_uint(four[1] + kWhole), 0x5410);
        if (unit < 4 * chunks) *reinterpret_cast<uint32_t *>(tile + (unit / 4) * kChunkBytes + inside * 16 + (unit % 4) * 4) = d < D ? nibbles : 0;
        if (d < D && d % a.c.group == 0)
            *reinterpret_cast<uint32_t *>(tile + chunks * kChunkBytes + d / a.c.group * kGroupBytes + inside * 4) = word | static_cast<uint32_t>(z);
    };
    // Every rows-th head is this thread's, one at a time (two, loads first, took registers that a block more makes better use of).
    // The barrier: outputs may be the inputs.
    const int64_t block = static_cast<int64_t>(slot / kBlockSlots) * hk * a.c.tile_bytes;
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {  // keys, then values
        const int64_t at = t * (which ? a.v_token : a.k_token) + d;
        const T *from = static_cast<const T *>(which ? a.v : a.k) + at;
        T *out = static_cast<T *>(which ? args.v_out : args.k_out);
        const bool tell = out;
        out += at;
        char *tiles = (which ? a.c.v + page * a.c.v_page : a.c.k + page * a.c.k_page) + block;
#pragma unroll 1
        for (int h = row; h < hk; h += rows) {
            Pack<T, 8> own, pair;
            load(own, pair, from + h * D, !which);
            __syncwarp(mine);
            float x[8];
            if (!which) {
                rotate(x, own, pair);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = dev::widen(own.v[i]);
            }
            hold(x, tiles + h * a.c.tile_bytes);
            if (tell) store8<T, WORDS>(out + h * D, x, d, D);
        }
    }
}

// Queries, as a cache of 16 or 32 bits has them, in the first `query.blocks` blocks; keys and values.
struct QueryBlocks {
    unsigned blocks;
    int units, rot_units, rows;
};
template <typename T, bool WORDS, bool INTERLEAVED, bool QUERY_WORDS>
__global__ void __launch_bounds__(kAppendThreads, 3) k_append4(const __grid_constant__ Append4Args args, QueryBlocks query, int lanes, int rows) {
    dev::wait_for_previous();
    constexpr int kVec = QUERY_WORDS ? 16 / static_cast<int>(sizeof(T)) : 1;
    if (blockIdx.x < query.blocks) append_heads<T, kVec, INTERLEAVED>(args.a, blockIdx.x, query.units, query.rot_units, query.rows, args.a.heads_q);
    else append4<T, WORDS, INTERLEAVED>(args, blockIdx.x - query.blocks, lanes, rows);
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
    // Runs of eight elements, in whole words.
    const int in_words = 16 / eb;
    const bool words = D % 8 == 0 && a.rot_dim % 8 == 0 && (desc->interleaved || half % 8 == 0) && a.k_token % in_words == 0 &&
                       a.v_token % in_words == 0 && !misaligned(k, 16) && !misaligned(v, 16) && !misaligned(k_out, 16) && !misaligned(v_out, 16) &&
                       !misaligned(a.cos, 16) && !misaligned(a.sin, 16);
    const bool query_words = desc->heads_q && (D | half | a.q_token | a.q_out_token) % in_words == 0 && !misaligned(q, 16) && !misaligned(q_out, 16) &&
                             !misaligned(a.cos, 16) && !misaligned(a.sin, 16);
    int lanes = 4;  // of a row, so that its groups meet by shuffles
    while (lanes * 8 < D) lanes *= 2;
    // Heads of a token in one thread: all of them, or as few as it takes for eight blocks a SM (two of queries).
    auto rows_of = [&](int heads, int64_t threads, int per_sm) {
        return static_cast<int>(std::min<int64_t>(heads, std::max<int64_t>(1, (int64_t(sms) * per_sm * kAppendThreads + threads - 1) / threads)));
    };
    if (tokens > INT32_MAX) return set_error(L2D_ERR_INVALID, "%lld tokens are too many", static_cast<long long>(tokens));
    int rows = rows_of(cache->heads, tokens * lanes, 8);
    while (cache->heads % rows) ++rows;  // so that neighbours in a warp have as many heads
    int64_t blocks = (tokens * lanes * rows + kAppendThreads - 1) / kAppendThreads;
    QueryBlocks query = {};
    if (desc->heads_q) {
        const AppendUnits u = append_units(query_words, eb, D, a.rot_dim);
        query.units = u.units;
        query.rot_units = u.rot_units;
        query.rows = rows_of(desc->heads_q, tokens * u.units, 2);
        const int64_t n = (tokens * u.units * query.rows + kAppendThreads - 1) / kAppendThreads;
        blocks += n;
        query.blocks = static_cast<unsigned>(std::min<int64_t>(n, INT32_MAX));
    }
    if (blocks > INT32_MAX) return set_error(L2D_ERR_INVALID, "%lld tokens are too many", static_cast<long long>(tokens));
    auto pick_query = [&](auto type, auto in_runs, auto interleaved) {
        using T = decltype(type);
        return query_words ? k_append4<T, decltype(in_runs)::value, decltype(interleaved)::value, true> : k_append4<T, decltype(in_runs)::value, decltype(interleaved)::value, false>;
    };
    auto pick = [&](auto type) {
        if (words) return desc->interleaved ? pick_query(type, std::true_type(), std::true_type()) : pick_query(type, std::true_type(), std::false_type());
        return desc->interleaved ? pick_query(type, std::false_type(), std::true_type()) : pick_query(type, std::false_type(), std::false_type());
    };
    auto kernel = cache->dtype == L2D_F32 ? pick(float()) : cache->dtype == L2D_F16 ? pick(__half()) : pick(__nv_bfloat16());
    L2D_CUDA_TRY(launch(kernel, dim3(static_cast<unsigned>(blocks)), kAppendThreads, 0, stream, args, query, lanes, rows));
    return L2D_OK;
}

}  // extern "C"

// A mixture-of-experts layer for a few tokens (l2d_moe_*): the router, the chosen experts' products, their weighted sum.
//
// Memory bound: the weights of every chosen expert are read once and meet one token or a few.  Four launches, each of which
// waits for the one before on the device and not on the host:
//   k_route    a router row and up to four tokens per block; the last block of these tokens chooses their experts, the last of
//              all sorts (token, choice) pairs ("slots") into entries: an expert and up to so many slots as one pass takes
//   k_experts  gate and up: silu(gate x) * (up x) of every slot, to scratch
//   k_experts  down: of every slot, to scratch
//   k_combine  the weighted sum over a token's slots, in their order
// (Measured and dropped for a token or a few: choosing in every block of gate and up, which saves a meeting of blocks, 8 us
// there for 6.6 here; summing in the blocks of down, which saves a launch, with whole tiles of rows to a block: 20.6 us for
// 17 + 5 at 4096 x 1536, and 45 for 30 in all at 1001 x 333.)
// Nothing depends on the order in which blocks come: a slot's sums are its own.
//
// Measured (bf16): 32 tokens, 4 of 64 experts of 4096 x 1024, 250 to 265 us under the power cap, 5.6 to 5.3 TB/s, for 220 us
// of bytes at a copy's rate; one token, 4 of 32 of 4096 x 1536, 45 us for 24: the chain of launches and, in each, some
// microseconds until its rows come.
#include "l2d_launch.cuh"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstring>
#include <new>
#include <type_traits>

namespace l2d {

constexpr int kMaxExperts = 512;
constexpr int kMoeThreads = 256, kMoeWarps = kMoeThreads / 32;
constexpr int kRouteTokens = 4;  // of a block of the router
constexpr int kRouteExperts = 2; // where there are tokens for blocks enough

struct MoeArgs {
    const void *x, *router, *gate, *up, *down;
    void *y;
    int32_t *ids_out;
    float *weights_out;
    int64_t x_token, y_token, router_row, gate_row, up_row, down_row, gate_expert, up_expert, down_expert;
    int tokens, hidden, inner, experts, top, normalize, per_entry;
    // The plan's scratch.
    double *logits;       // [tokens][experts]
    int *ids;             // [slots], slot = token * top + choice
    float *weights;       // [slots]
    uint32_t *largest;    // [slots] bits of the largest |silu(gate x) (up x)| (fp16; bf16: of one that is not finite, or 0)
    int *sorted;          // [slots], by expert
    int4 *entries;        // expert, first place in sorted, slots
    int *num_entries;     // and whether an inner value is not finite (bf16)
    unsigned *arrived;    // [token tiles + 1], zero between calls
    float *inner_out;     // [slots][inner_row]
    float *part;          // [slots][hidden]
    int64_t inner_row;
};

// ---------------------------------------------------------------------------------------------
// Router.  Its sums are 64-bit ones: they choose, and two experts whose scores differ by less than a 32-bit sum is off would be
// chosen by the order of addition.  A router row's numbers are made 64-bit ones once for up to four tokens.
// ---------------------------------------------------------------------------------------------

template <typename T>
struct Eight {
    T v[8];
};
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T *p) {
    Eight<T> r;
    const uint4 *from = reinterpret_cast<const uint4 *>(p);
    uint4 *to = reinterpret_cast<uint4 *>(&r);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) to[i] = from[i];
    return r;
}

// Chooses the experts of one token: a warp, `top` rounds over kEach scores a lane, as numbers whose order is that of whole
// numbers (fp64 comparisons took ten times as long).  What is no number comes last.  Weights are computed in 64 bits and rounded
// once (in fp32 they were off by up to 2^-21.9, now 2^-24, for at most half a microsecond less).
template <int kEach>
__device__ __forceinline__ void choose_of(const MoeArgs &a, int token) {
    const int lane = threadIdx.x & 31;
    const double *logits = a.logits + static_cast<int64_t>(token) * a.experts;
    double v[kEach];
    uint32_t high[kEach], low[kEach];
    uint32_t open = 0;  // this lane's experts that are not chosen yet
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int e = lane + 32 * i;
        v[i] = 0.0;
        if (e < a.experts) {
            v[i] = __ldcg(logits + e) + 0.0;  // one zero
            open |= 1u << i;
        }
        const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v[i])), order = bits >> 63 ? ~bits : bits | 1ull << 63;
        const bool number = (bits & 0x7fffffffffffffffull) <= 0x7ff0000000000000ull;
        high[i] = number ? static_cast<uint32_t>(order >> 32) : 0;
        low[i] = number ? static_cast<uint32_t>(order) : 0;
    }
    int mine = 0;
    double score = 0.0, first = 0.0;  // of the choice that this lane keeps, and of the first
    for (int k = 0; k < a.top; ++k) {
        uint32_t h = 0, l = 0;
        int at = INT_MAX;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if ((open >> i & 1) && (at == INT_MAX || high[i] > h || (high[i] == h && low[i] > l))) h = high[i], l = low[i], at = lane + 32 * i;
        const uint32_t top_high = __reduce_max_sync(0xffffffffu, h);
        const bool with_high = at != INT_MAX && h == top_high;
        const uint32_t top_low = __reduce_max_sync(0xffffffffu, with_high ? l : 0);
        const int won = static_cast<int>(__reduce_min_sync(0xffffffffu, with_high && l == top_low ? static_cast<uint32_t>(at) : static_cast<uint32_t>(INT_MAX)));
        double given = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (won == lane + 32 * i) {
                open &= ~(1u << i);
                given = v[i];
            }
        given = __shfl_sync(0xffffffffu, given, won & 31);
        if (k == 0) first = given;
        if (k == lane) mine = won, score = given;
    }
    const double e = lane < a.top ? exp(score - first) : 0.0;
    double sum = 0.0;
    if (a.normalize) {
        sum = e;
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (lane + 32 * i < a.experts) sum += exp(v[i] - first);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane < a.top) {
        const int64_t slot = static_cast<int64_t>(token) * a.top + lane;
        const float w = static_cast<float>(e / sum);
        a.ids[slot] = mine;
        a.weights[slot] = w;
        if (a.ids_out) a.ids_out[slot] = mine;
        if (a.weights_out) a.weights_out[slot] = w;
    }
}
__device__ __forceinline__ void choose(const MoeArgs &a, int token) {
    if (a.experts <= 32) choose_of<1>(a, token);
    else if (a.experts <= 128) choose_of<4>(a, token);
    else choose_of<kMaxExperts / 32>(a, token);
}

// Sorts the slots by expert, and cuts each expert's into entries.
__device__ __forceinline__ void sort_slots(const MoeArgs &a) {
    __shared__ int count[kMaxExperts], place[kMaxExperts], entry[kMaxExperts];
    const int tid = threadIdx.x, slots = a.tokens * a.top;
    const int mine = tid < slots ? __ldcg(a.ids + tid) : 0;
    for (int e = tid; e < kMaxExperts; e += kMoeThreads) count[e] = 0;
    __syncthreads();
    for (int s = tid; s < slots; s += kMoeThreads) atomicAdd(&count[s == tid ? mine : __ldcg(a.ids + s)], 1);
    __syncthreads();
    if (tid < 32) {  // places and entries before each expert's: as many experts a lane
        const int kEach = (a.experts + 31) / 32;
        int here = 0, entries = 0;
        for (int i = 0; i < kEach; ++i) {
            const int n = count[tid * kEach + i];
            here += n;
            entries += (n + a.per_entry - 1) / a.per_entry;
        }
        int upto = here, upto_entries = entries;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, d), y = __shfl_up_sync(0xffffffffu, upto_entries, d);
            if (tid >= d) upto += x, upto_entries += y;
        }
        if (tid == 31) a.num_entries[0] = upto_entries, a.num_entries[1] = 0;
        upto -= here;
        upto_entries -= entries;
        for (int i = 0; i < kEach; ++i) {
            const int n = count[tid * kEach + i];
            place[tid * kEach + i] = upto;
            entry[tid * kEach + i] = upto_entries;
            upto += n;
            upto_entries += (n + a.per_entry - 1) / a.per_entry;
        }
    }
    __syncthreads();
    for (int e = tid; e < a.experts; e += kMoeThreads)
        for (int done = 0, i = entry[e]; done < count[e]; done += a.per_entry, ++i)
            a.entries[i] = make_int4(e, place[e] + done, min(count[e] - done, a.per_entry), 0);
    __syncthreads();
    for (int s = tid; s < slots; s += kMoeThreads) a.sorted[atomicAdd(&place[s == tid ? mine : __ldcg(a.ids + s)], 1)] = s;
}

// Whether this block is the last of `n` to come here; what the others wrote before is then visible.
__device__ __forceinline__ bool last_of(unsigned *arrived, unsigned n) {
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();  // after the barrier, for the whole block
        last = atomicAdd(arrived, 1u) == n - 1;
        if (last) *arrived = 0;
        __threadfence();
    }
    __syncthreads();
    return last;
}

// EXPERTS: router rows of a block.  More of them read the tokens, and make them 64-bit numbers, less often.
template <typename T, bool WORDS, int EXPERTS>
__global__ void __launch_bounds__(kMoeThreads) k_route(const __grid_constant__ MoeArgs a) {
    dev::wait_for_previous();
    __shared__ double sums[kMoeWarps][EXPERTS * kRouteTokens];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e = blockIdx.x * EXPERTS, t0 = blockIdx.y * kRouteTokens;
    const int n = min(a.tokens - t0, kRouteTokens), experts = min(a.experts - e, EXPERTS);
    const T *w = static_cast<const T *>(a.router) + e * a.router_row, *x = static_cast<const T *>(a.x) + t0 * a.x_token;
    double acc[EXPERTS][kRouteTokens] = {};
    constexpr int kEach = WORDS ? 8 : 1;
    for (int k = kEach * tid; k < a.hidden; k += kEach * kMoeThreads) {
        double wide[EXPERTS][kEach];
#pragma unroll
        for (int j = 0; j < EXPERTS; ++j) {
            const T *row = w + min(j, experts - 1) * a.router_row + k;  // past the last: nobody's sum
            if constexpr (WORDS) {
                const Eight<T> r = load_eight(row);
#pragma unroll
                for (int i = 0; i < 8; ++i) wide[j][i] = dev::widen(r.v[i]);
            } else {
                wide[j][0] = dev::widen(*row);
            }
        }
#pragma unroll
        for (int t = 0; t < kRouteTokens; ++t) {
            if (t >= n) break;
            T v[kEach];
            if constexpr (WORDS) {
                const Eight<T> r = load_eight(x + t * a.x_token + k);
                memcpy(v, &r, sizeof r);
            } else {
                v[0] = x[t * a.x_token + k];
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const double y = dev::widen(v[i]);
#pragma unroll
                for (int j = 0; j < EXPERTS; ++j) acc[j][t] = fma(wide[j][i], y, acc[j][t]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kRouteTokens; ++t) {
        if (t >= n) break;
#pragma unroll
        for (int j = 0; j < EXPERTS; ++j) {
#pragma unroll
            for (int d = 16; d; d >>= 1) acc[j][t] += __shfl_xor_sync(0xffffffffu, acc[j][t], d);
            if (lane == 0) sums[warp][j * kRouteTokens + t] = acc[j][t];
        }
    }
    __syncthreads();
    if (const int j = tid / kRouteTokens, t = tid % kRouteTokens; j < experts && t < n) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < kMoeWarps; ++i) s += sums[i][tid];
        a.logits[static_cast<int64_t>(t0 + t) * a.experts + e + j] = s;
    }
    if (e == 0)
        for (int i = tid; i < n * a.top; i += kMoeThreads) a.largest[static_cast<int64_t>(t0) * a.top + i] = 0;
    if (!last_of(a.arrived + 1 + blockIdx.y, gridDim.x)) return;
    if (warp < n) choose(a, t0 + warp);
    if (gridDim.y > 1) {
        if (!last_of(a.arrived, gridDim.y)) return;
    } else {
        __syncthreads();
    }
    sort_slots(a);
}

// ---------------------------------------------------------------------------------------------
// The experts' products.
//
// 16 bits: a warp works on 16 rows of a matrix (eight of gate and the same eight of up, or 16 of down) and the slots of an
// entry, the columns of m16n8k16.  A lane brings 16 bytes of rows g and g + 8 at a time, elements 8t .. 8t + 7 of 32: any order
// of the sum's terms will do as long as both sides have it, and so no lane needs what another one brought.  Rows go through a
// ring of shared memory of the lane's own (asynchronous copies, no barrier), which keeps kDepth steps on their way across
// the ends of items; columns are read from L1 or L2 a step ahead.  Where there are few items, their rows are cut into S
// parts for as many warps of a block.
//
// silu(gate x) (up x) is held in fp32 and cut on the way to the down product: for bf16 into three numbers that add up to it (two, made
// once by the first product, took 1.5 us less for one token and 16 of 253 for 156, and 2^-16 of each), for fp16
// into two, relative to the slot's largest, which only the whole first product knows: 2^-22 of it is left, 2^-11 of what rounding
// an output to fp16 may take off.
//
// The products of a step are added to the sum in fp32: the instruction cuts them off at its sum's last place (no change in time).
//
// 32 bits: a warp works on four rows (two of gate and of up) with the lanes along them, by fused multiply-adds.
// ---------------------------------------------------------------------------------------------

constexpr int kDepth32 = 4;               // steps in a ring, all but one of them on their way
constexpr int kRowBytes = 2048;           // of a step: 16 rows of 128 bytes, or four of 512
constexpr int kCached = 128, kCachedSlots = 1024;  // entries and slots that a block keeps in shared memory
// How rows come: 16 bytes at a time; 4; 4, of rows of 16-bit elements that may begin in the middle of a word; one element.
enum { kBy16 = 0, kBy4 = 1, kByHalves = 2, kByElement = 3 };

__device__ __forceinline__ uint32_t smem_at(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 16 bytes of a row, of which `n` elements are real.  L2 fetches 256 at a time: each step takes 128 of sixteen rows, and a memory
// page's other half would be a row's next step (32 tokens 263 us, 243 so; bursts of steps bring less).
template <typename T, int COPY>
__device__ __forceinline__ void bring(char *to, const T *from, int n) {
    constexpr int kEach = 16 / static_cast<int>(sizeof(T));
    if constexpr (COPY == kBy16) {
        asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(smem_at(to)), "l"(from), "r"(n * static_cast<int>(sizeof(T))) : "memory");
    } else if constexpr (COPY == kBy4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int have = min(max(n * static_cast<int>(sizeof(T)) - 4 * i, 0), 4);
            const char *p = have ? reinterpret_cast<const char *>(from) + 4 * i : reinterpret_cast<const char *>(from);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_at(to + 4 * i)), "l"(p), "r"(have) : "memory");
        }
    } else {
        T v[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = i < n ? from[i] : dev::narrow<T>(0.0f);
        memcpy(to, v, 16);
    }
}

// Eight 16-bit elements, of which `n` are real, as the four words that they lie in, and the fifth where they begin in the middle
// of one: what is before them in their first word is the row before's last element.
template <typename T>
__device__ __forceinline__ void bring_halves(char *to, char *fifth, const T *from, int n, const T *none) {
    const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(from) & 2);
    const char *p = n ? reinterpret_cast<const char *>(from) - skip : reinterpret_cast<const char *>(none);  // nothing is read there
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        if (i == 4 && !skip) break;
        const int have = n ? min(max(skip + 2 * n - 4 * i, 0), 4) : 0;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_at(i < 4 ? to + 4 * i : fifth)), "l"(have ? p + 4 * i : p), "r"(have) : "memory");
    }
}
// The elements of such words.
__device__ __forceinline__ uint4 from_halves(const char *at, const char *fifth, bool skip) {
    uint4 w = *reinterpret_cast<const uint4 *>(at);
    if (skip) {
        const uint32_t last = *reinterpret_cast<const uint32_t *>(fifth);
        w = make_uint4(w.x >> 16 | w.y << 16, w.y >> 16 | w.z << 16, w.z >> 16 | w.w << 16, w.w >> 16 | last << 16);
    }
    return w;
}

template <typename T, int COPY>
__device__ __forceinline__ void bring_all(char *to, const T *from) {
    if constexpr (COPY == kBy16) asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(smem_at(to)), "l"(from) : "memory");
    else bring<T, COPY>(to, from, 16 / static_cast<int>(sizeof(T)));
}

// Sixteen bytes by way of L1, for what all warps of an SM read: of rows, which are read once, L1 keeps nothing.  (Past L1 the few
// lines of one token's columns were all SMs' at once, and its down product took 59 us for 17.)
__device__ __forceinline__ void bring_shared(char *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_at(to)), "l"(from) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The items of a launch, and this group of warps' share of them: entry by entry for gate and up, whose columns are the same for
// all rows of an entry; tile of rows by tile for down.
struct Items {
    int tiles, entries, first, stop;
    __device__ __forceinline__ void split(int item, bool by_entry, int &entry, int &tile) const {
        entry = by_entry ? item / tiles : item % entries;
        tile = by_entry ? item - entry * tiles : item / entries;
    }
};
// Even shares to within one item.
__device__ __forceinline__ Items items_of(int entries, int tiles, int groups, int group) {
    const int64_t total = static_cast<int64_t>(tiles) * entries;
    return {tiles, entries, static_cast<int>(total * group / groups), static_cast<int>(total * (group + 1) / groups)};
}

__device__ __forceinline__ float silu_times(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    uint32_t r;
    memcpy(&r, &h, 4);
    return r;
}

// What a slot's numbers are multiplied by before they become fp16: the largest then lies in 2^14 .. 2^15.  Beside an infinity
// or a NaN the finite ones only have to stay finite, whatever they are: every output is that one's.
__device__ __forceinline__ float to_half_range(uint32_t largest_bits) {
    const int exponent = static_cast<int>(largest_bits >> 23);  // 255: not finite
    if (exponent == 255 || exponent == 0) return exponent ? 0x1p-113f : 0x1p100f;
    return __uint_as_float(static_cast<uint32_t>(min(127 + 14 - (exponent - 127), 254)) << 23);
}

// The entries and the slots behind them: a block's own copy where they are few.
struct Lists {
    const int4 *entries;
    const int *sorted;
    int num;
    bool odd;  // an inner value is not finite
};
__device__ __forceinline__ Lists lists_of(const MoeArgs &a) {
    __shared__ int4 kept_entries[kCached];
    __shared__ int kept_sorted[kCachedSlots];
    const int slots = a.tokens * a.top;
    const int2 two = *reinterpret_cast<const int2 *>(a.num_entries);
    const int num = two.x;
    if (num > kCached || slots > kCachedSlots) return {a.entries, a.sorted, num, two.y != 0};
    for (int i = threadIdx.x; i < num; i += kMoeThreads) kept_entries[i] = a.entries[i];
    for (int i = threadIdx.x; i < slots; i += kMoeThreads) kept_sorted[i] = a.sorted[i];
    __syncthreads();
    return {kept_entries, kept_sorted, num, two.y != 0};
}

// A warp's ring: a step's rows, then its columns (16 bytes a lane of each eight and run, of four-byte elements twice), as deep as
// sixteen warps an SM leave room for (eight of many columns).
template <int N, bool DOWN, bool HALVES>
struct ExpertsRing {
    static constexpr int kWords = kRowBytes + N * (DOWN ? 2048 : 1024);
    static constexpr int kStep = kWords + (HALVES ? 128 * (4 + (DOWN ? 0 : 2 * N)) : 0);  // and fifth words, four bytes a lane
    static constexpr int kBlocks = N == 4 || (N == 2 && HALVES) ? 1 : 2;
    static constexpr int kDepth = 12 * 1024 * (3 - kBlocks) / kStep;
    static constexpr int kBytes = kDepth * kStep;
    static_assert(kDepth >= 2, "one step on its way");
};

// N: eights of columns; DOWN: the second product.  S: warps that share an item.
template <typename T, int N, bool DOWN, int COPY>
__global__ void __launch_bounds__(kMoeThreads, ExpertsRing<N, DOWN, COPY == kByHalves>::kBlocks) k_experts(const __grid_constant__ MoeArgs a, int S) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kK = 64;                           // elements of a step: two runs of 32
    constexpr int kCuts = kHalf ? 2 : 3;             // 16-bit numbers of an inner value
    using Ring = ExpertsRing<N, DOWN, COPY == kByHalves>;
    extern __shared__ __align__(128) char smem[];
    dev::wait_for_previous();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int K = DOWN ? a.inner : a.hidden, rows = DOWN ? a.hidden : a.inner, per_tile = DOWN ? 16 : 8;
    const int part = warp % S, groups = kMoeWarps / S, group = warp / S;
    const Lists lists = lists_of(a);
    const Items items = items_of(lists.num, (rows + per_tile - 1) / per_tile, gridDim.x * groups, blockIdx.x * groups + group);
    // This warp's part of K.  Only the last step of all may be short.
    const int all = (K + kK - 1) / kK, each = (all + S - 1) / S, begin = min(part * each, all), steps = min(begin + each, all) - begin;
    const bool short_end = begin + steps == all && K % kK;
    const int n_end[2] = {min(max(K - (all - 1) * kK - 8 * t, 0), 8), min(max(K - (all - 1) * kK - 32 - 8 * t, 0), 8)};
    const int first_k = begin * kK + 8 * t;
    char *ring = smem + warp * Ring::kBytes + lane * 16;
    const int fifths = Ring::kWords - lane * 12;  // of a step's words, where this lane's fifth words begin
    float *meet = reinterpret_cast<float *>(smem + kMoeWarps * Ring::kBytes);  // [warp][4 N][lane]

    // What is brought next: rows g and g + 8 from p0 and p1 on, and column g of each eight, `left` steps of them.
    using X = typename std::conditional<DOWN, float, T>::type;
    constexpr int kRun = DOWN ? 2 : 1;  // 16-byte words of eight elements of a column
    int item = items.first, left = 0, in_at = 0, in_count = 0;
    const T *p0 = nullptr, *p1 = nullptr;
    const X *column[N] = {};
    auto point = [&] {  // rows past the last are the last one's, and so are columns: their sums go nowhere
        int at, tile;
        items.split(item, !DOWN, at, tile);
        const int4 entry = lists.entries[at];
        const int expert = entry.x;
        in_count = entry.z;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int slot = lists.sorted[entry.y + min(8 * j + g, entry.z - 1)];
            if constexpr (DOWN) column[j] = a.inner_out + slot * a.inner_row + first_k;
            else column[j] = static_cast<const T *>(a.x) + slot / a.top * a.x_token + first_k;
        }
        if constexpr (DOWN) {
            const T *w = static_cast<const T *>(a.down) + expert * a.down_expert + first_k;
            p0 = w + min(tile * 16 + g, rows - 1) * a.down_row;
            p1 = w + min(tile * 16 + g + 8, rows - 1) * a.down_row;
        } else {
            const int r = min(tile * 8 + g, rows - 1);
            p0 = static_cast<const T *>(a.gate) + expert * a.gate_expert + r * a.gate_row + first_k;
            p1 = static_cast<const T *>(a.up) + expert * a.up_expert + r * a.up_row + first_k;
        }
        left = steps;
    };
    // Where a copy of no elements points: its address has to be aligned as any other's, so it is one of a matrix that the width
    // of the copies was chosen by.
    const T *none = static_cast<const T *>(DOWN ? a.down : a.gate);
    auto bring_step = [&] {
        if (left) {
            char *to = ring + in_at;
            const bool end = short_end && left == 1;
            if constexpr (COPY == kByHalves) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int n = end ? n_end[h] : 8;
                    bring_halves(to + 1024 * h, to + fifths + 256 * h, p0 + 32 * h, n, none);
                    bring_halves(to + 1024 * h + 512, to + fifths + 256 * h + 128, p1 + 32 * h, n, none);
                    if constexpr (!DOWN) {
#pragma unroll
                        for (int j = 0; j < N; ++j)
                            if (j == 0 || 8 * j < in_count)
                                bring_halves(to + kRowBytes + 1024 * j + 512 * h, to + fifths + 512 + 256 * j + 128 * h, column[j] + 32 * h, n, none);
                    }
                }
            } else if (end) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // nothing is read of a run without elements, whose first may lie anywhere
                    bring<T, COPY>(to + 1024 * h, n_end[h] ? p0 + 32 * h : none, n_end[h]);
                    bring<T, COPY>(to + 1024 * h + 512, n_end[h] ? p1 + 32 * h : none, n_end[h]);
                    if constexpr (!DOWN) {
#pragma unroll
                        for (int j = 0; j < N; ++j)
                            if (j == 0 || 8 * j < in_count) bring<T, COPY>(to + kRowBytes + 1024 * j + 512 * h, n_end[h] ? column[j] + 32 * h : none, n_end[h]);
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bring_all<T, COPY>(to + 1024 * h, p0 + 32 * h);
                    bring_all<T, COPY>(to + 1024 * h + 512, p1 + 32 * h);
                    if constexpr (!DOWN) {
#pragma unroll
                        for (int j = 0; j < N; ++j)
                            if (j == 0 || 8 * j < in_count) {
                                char *x = to + kRowBytes + 1024 * j + 512 * h;
                                if constexpr (COPY == kBy16) bring_shared(x, column[j] + 32 * h);
                                else bring_all<T, COPY>(x, column[j] + 32 * h);
                            }
                    }
                }
            }
            if constexpr (DOWN) {  // rows of the scratch are padded with zeros, and aligned
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j == 0 || 8 * j < in_count)
#pragma unroll
                        for (int h = 0; h < 4; ++h)
                            bring_shared(to + kRowBytes + 2048 * j + 512 * h, column[j] + 32 * (h / 2) + 4 * (h % 2));
            }
            p0 += kK;
            p1 += kK;
#pragma unroll
            for (int j = 0; j < N; ++j) column[j] += kK;
            if (--left == 0 && ++item < items.stop) point();
        }
        copy_commit();
        in_at = in_at + Ring::kStep == Ring::kBytes ? 0 : in_at + Ring::kStep;
    };
    if (item < items.stop && steps) point();
#pragma unroll 1
    for (int i = 0; i < Ring::kDepth - 1; ++i) bring_step();

    int out_at = 0;
#pragma unroll 1
    for (int now = items.first; now < items.stop; ++now) {
        int at, tile;
        items.split(now, !DOWN, at, tile);
        const int4 entry = lists.entries[at];
        float factor[N];  // what makes this lane's columns fp16
        uint32_t low_mask[N];
        if constexpr (DOWN) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t bits = kHalf || lists.odd ? a.largest[lists.sorted[entry.y + min(8 * j + g, entry.z - 1)]] : 0;
                if constexpr (kHalf) factor[j] = to_half_range(bits);
                low_mask[j] = bits >= 0x7f800000u ? 0 : 0xffffffffu;  // beside an infinity or a NaN first numbers alone
            }
        }
        // Which rows and columns begin in the middle of a word: the products' matrices begin at one.
        bool skip[2] = {}, skip_x[N] = {};
        if constexpr (COPY == kByHalves) {
            const int r0 = DOWN ? min(tile * 16 + g, rows - 1) : min(tile * 8 + g, rows - 1), r1 = DOWN ? min(tile * 16 + g + 8, rows - 1) : r0;
            skip[0] = (entry.x * (DOWN ? a.down_expert : a.gate_expert) + r0 * (DOWN ? a.down_row : a.gate_row)) & 1;
            skip[1] = (entry.x * (DOWN ? a.down_expert : a.up_expert) + r1 * (DOWN ? a.down_row : a.up_row)) & 1;
            if constexpr (!DOWN)
#pragma unroll
                for (int j = 0; j < N; ++j) skip_x[j] = (lists.sorted[entry.y + min(8 * j + g, entry.z - 1)] / a.top * a.x_token) & 1;
        }
        float acc[N][4] = {};
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            copy_wait<Ring::kDepth - 2>();
            const char *from = ring + out_at;
            uint4 r[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (COPY == kByHalves) r[h][i] = from_halves(from + 1024 * h + 512 * i, from + fifths + 256 * h + 128 * i, skip[i]);
                    else r[h][i] = *reinterpret_cast<const uint4 *>(from + 1024 * h + 512 * i);
                }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (j && 8 * j >= entry.z) break;
                float sum[4] = {};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 &r0 = r[h][0], &r1 = r[h][1];
                    const uint4 *x = reinterpret_cast<const uint4 *>(from + kRowBytes + 1024 * kRun * j + 512 * kRun * h);
                    uint4 u;
                    if constexpr (!DOWN && COPY == kByHalves) u = from_halves(reinterpret_cast<const char *>(x), from + fifths + 512 + 256 * j + 128 * h, skip_x[j]);
                    else u = x[0];
                    if constexpr (!DOWN) {
                        mma<T>(sum, r0.x, r1.x, r0.y, r1.y, u.x, u.y);
                        mma<T>(sum, r0.z, r1.z, r0.w, r1.w, u.z, u.w);
                    } else {
                        const uint4 v = x[32];
                        const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                        uint32_t cut[kCuts][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float one = __uint_as_float(w[2 * i]), two = __uint_as_float(w[2 * i + 1]);
                            if constexpr (kHalf) {
                                one *= factor[j], two *= factor[j];
                                cut[0][i] = pack_half(one, two);
                                __half2 halves;
                                memcpy(&halves, &cut[0][i], 4);
                                cut[1][i] = pack_half(one - __low2float(halves), two - __high2float(halves)) & low_mask[j];
                            } else {  // cut off, not rounded: what is left is exact, and the largest number's first part finite
#pragma unroll
                                for (int part = 0; part < kCuts; ++part) {
                                    const uint32_t low = __float_as_uint(one), high = __float_as_uint(two);
                                    cut[part][i] = __byte_perm(low, high, 0x7632);
                                    one -= __uint_as_float(low & 0xffff0000u);
                                    two -= __uint_as_float(high & 0xffff0000u);
                                }
                            }
                        }
#pragma unroll
                        for (int part = 0; part < kCuts; ++part) {
                            if (!kHalf && part && lists.odd) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) cut[part][i] &= low_mask[j];
                            }
                            mma<T>(sum, r0.x, r1.x, r0.y, r1.y, cut[part][0], cut[part][1]);
                            mma<T>(sum, r0.z, r1.z, r0.w, r1.w, cut[part][2], cut[part][3]);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j][e] += sum[e];
            }
            bring_step();  // into the step before's place, which this lane has read
            out_at = out_at + Ring::kStep == Ring::kBytes ? 0 : out_at + Ring::kStep;
        }
        // The parts' sums meet, in their order, in the group's first warp.
        if (S > 1) {
            const int bar = 1 + group;
            asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(32 * S) : "memory");  // the item before is done with
            if (part) {
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) meet[(warp * 4 * N + 4 * j + e) * 32 + lane] = acc[j][e];
            }
            asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(32 * S) : "memory");
            if (part) continue;
            for (int p = 1; p < S; ++p)
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] += meet[((warp + p) * 4 * N + 4 * j + e) * 32 + lane];
        }
        // Columns 2 t and 2 t + 1 of rows g and g + 8.
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (8 * j >= entry.z) break;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = 8 * j + 2 * t + e;
                const int slot = lists.sorted[entry.y + min(c, entry.z - 1)];
                if constexpr (DOWN) {
                    float back = 1.0f;
                    if constexpr (kHalf) back = 1.0f / to_half_range(a.largest[slot]);
                    float *to = a.part + static_cast<int64_t>(slot) * a.hidden + tile * 16 + g;
                    if (c < entry.z && tile * 16 + g < rows) to[0] = acc[j][e] * back;
                    if (c < entry.z && tile * 16 + g + 8 < rows) to[8] = acc[j][2 + e] * back;
                } else {
                    const int row = tile * 8 + g;
                    const bool real = c < entry.z && row < rows;
                    const float h = real ? silu_times(acc[j][e], acc[j][2 + e]) : 0.0f;
                    if (real) a.inner_out[slot * a.inner_row + row] = h;
                    if constexpr (kHalf) {
                        uint32_t top = __float_as_uint(h) & 0x7fffffffu;
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                        if (g == 0 && c < entry.z && top) atomicMax(a.largest + slot, top);
                    } else if (!(fabsf(h) <= FLT_MAX)) {  // not of a row or column that is not real: those are 0
                        atomicMax(a.largest + slot, __float_as_uint(h) & 0x7fffffffu);
                        a.num_entries[1] = 1;
                    }
                }
            }
        }
    }
}

// The same of 32 bits: rows 0 and 1 of gate and 2 and 3 of up, or four of down, up to eight columns.  Elements of a step that
// a lane has: four side by side, or every 32nd where they come one by one.
template <bool DOWN, int COPY>
__global__ void __launch_bounds__(kMoeThreads, 2) k_experts32(const __grid_constant__ MoeArgs a, int S) {
    constexpr int kK = 128, kOne = COPY == kBy16 ? 1 : 32;  // elements of a step, and between two of a lane's
    extern __shared__ __align__(128) char smem[];
    dev::wait_for_previous();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int K = DOWN ? a.inner : a.hidden, rows = DOWN ? a.hidden : a.inner, per_tile = DOWN ? 4 : 2;
    const int part = warp % S, groups = kMoeWarps / S, group = warp / S;
    const Lists lists = lists_of(a);
    const Items items = items_of(lists.num, (rows + per_tile - 1) / per_tile, gridDim.x * groups, blockIdx.x * groups + group);
    const int all = (K + kK - 1) / kK, each = (all + S - 1) / S, begin = min(part * each, all), steps = min(begin + each, all) - begin;
    const int first_k = begin * kK + (COPY == kBy16 ? 4 * lane : lane);
    char *ring = smem + warp * kDepth32 * kRowBytes + lane * 16;
    float *meet = reinterpret_cast<float *>(smem + kMoeWarps * kDepth32 * kRowBytes);  // [warp][lane]

    int item = items.first, left = 0, in_at = 0, in_k = first_k;
    const float *p[4] = {};
    uint32_t in = 0;
    auto point = [&] {
        int at, tile;
        items.split(item, !DOWN, at, tile);
        const int expert = lists.entries[at].x;
        in = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = tile * per_tile + (DOWN ? i : i & 1);
            const float *w = DOWN ? static_cast<const float *>(a.down) + expert * a.down_expert
                             : i < 2 ? static_cast<const float *>(a.gate) + expert * a.gate_expert : static_cast<const float *>(a.up) + expert * a.up_expert;
            const int64_t row = DOWN ? a.down_row : i < 2 ? a.gate_row : a.up_row;
            p[i] = w;
            if (r < rows) {
                p[i] += r * row;
                in |= 1u << i;
            }
        }
        left = steps;
        in_k = first_k;
    };
    auto bring_step = [&] {
        if (left) {
            char *to = ring + in_at;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (COPY == kBy16) {
                    const int n = in >> i & 1 ? min(max(K - in_k, 0), 4) : 0;
                    bring<float, kBy16>(to + 512 * i, p[i] + (n ? in_k : 0), n);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool real = (in >> i & 1) && in_k + 32 * e < K;
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_at(to + 512 * i + 4 * e)), "l"(real ? p[i] + in_k + 32 * e : p[i]),
                                     "r"(real ? 4 : 0) : "memory");
                    }
                }
            }
            in_k += kK;
            if (--left == 0 && ++item < items.stop) point();
        }
        copy_commit();
        in_at = in_at + kRowBytes == kDepth32 * kRowBytes ? 0 : in_at + kRowBytes;
    };
    if (item < items.stop && steps) point();
#pragma unroll 1
    for (int i = 0; i < kDepth32 - 1; ++i) bring_step();

    int out_at = 0;
#pragma unroll 1
    for (int now = items.first; now < items.stop; ++now) {
        int at, tile;
        items.split(now, !DOWN, at, tile);
        const int4 entry = lists.entries[at];
        const float *column[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int slot = lists.sorted[entry.y + min(c, entry.z - 1)];
            column[c] = DOWN ? a.inner_out + slot * a.inner_row : static_cast<const float *>(a.x) + slot / a.top * a.x_token;
        }
        float acc[32] = {};  // [row][column]
        int k = first_k;
#pragma unroll 1
        for (int step = 0; step < steps; ++step, k += kK) {
            float4 x[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                x[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c >= entry.z) break;
                const float *q = column[c] + k;
                if constexpr (COPY == kBy16) {  // whole words: of K, or of the scratch's rows, which are padded with zeros
                    if (k < K) x[c] = *reinterpret_cast<const float4 *>(q);
                } else {
                    if (k < K) x[c].x = q[0];
                    if (k + kOne < K) x[c].y = q[kOne];
                    if (k + 2 * kOne < K) x[c].z = q[2 * kOne];
                    if (k + 3 * kOne < K) x[c].w = q[3 * kOne];
                }
            }
            copy_wait<kDepth32 - 2>();
            const char *from = ring + out_at;
            float4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4 *>(from + 512 * i);
            bring_step();
            out_at = out_at + kRowBytes == kDepth32 * kRowBytes ? 0 : out_at + kRowBytes;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c >= entry.z) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float s = acc[8 * i + c];
                    s = fmaf(w[i].x, x[c].x, s);
                    s = fmaf(w[i].y, x[c].y, s);
                    s = fmaf(w[i].z, x[c].z, s);
                    acc[8 * i + c] = fmaf(w[i].w, x[c].w, s);
                }
            }
        }
        // Lane l gets the sum of row l / 8 and column l % 8: halves exchanged until one is left.
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const bool upper = lane & d;
#pragma unroll
            for (int i = 0; i < d; ++i) {
                const float give = upper ? acc[i] : acc[i + d], keep = upper ? acc[i + d] : acc[i];
                acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
            }
        }
        float s = acc[0];
        if (S > 1) {
            const int bar = 1 + group;
            asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(32 * S) : "memory");
            if (part) meet[warp * 32 + lane] = s;
            asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(32 * S) : "memory");
            if (part) continue;
            for (int i = 1; i < S; ++i) s += meet[(warp + i) * 32 + lane];
        }
        const int c = lane % 8, row = lane / 8;
        if constexpr (DOWN) {
            if (c < entry.z && tile * 4 + row < rows) a.part[static_cast<int64_t>(lists.sorted[entry.y + c]) * a.hidden + tile * 4 + row] = s;
        } else {
            const float up = __shfl_down_sync(0xffffffffu, s, 16);
            if (row < 2 && c < entry.z && tile * 2 + row < rows)
                a.inner_out[lists.sorted[entry.y + c] * a.inner_row + tile * 2 + row] = silu_times(s, up);
        }
    }
}

// The sum over a token's slots.
template <typename T>
__global__ void __launch_bounds__(kMoeThreads) k_combine(const __grid_constant__ MoeArgs a) {
    dev::wait_for_previous();
    const int h = blockIdx.x * kMoeThreads + threadIdx.x, t = blockIdx.y;
    if (h >= a.hidden) return;
    const float *part = a.part + static_cast<int64_t>(t) * a.top * a.hidden + h, *w = a.weights + t * a.top;
    float y = 0.0f;
    for (int k0 = 0; k0 < a.top; k0 += 4) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = k0 + k < a.top ? part[static_cast<int64_t>(k0 + k) * a.hidden] : 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k0 + k < a.top) y = fmaf(w[k0 + k], v[k], y);
    }
    static_cast<T *>(a.y)[t * a.y_token + h] = dev::narrow<T>(y);
}

struct MoeKernels {
    void (*route)(MoeArgs);
    void (*gate_up)(MoeArgs, int);
    void (*down)(MoeArgs, int);
    void (*combine)(MoeArgs);
    int smem[2], blocks[2];  // of gate and up, and of down: bytes of a block, blocks an SM
};

template <typename T, int N, bool DOWN>
int experts_smem(int copy) {
    return kMoeWarps * (sizeof(T) == 4 ? kDepth32 * kRowBytes + 128 : (copy == kByHalves ? ExpertsRing<N, DOWN, true>::kBytes : ExpertsRing<N, DOWN, false>::kBytes) + 4 * N * 128);
}

template <typename T, int N>
int experts_blocks(int copy) {
    return sizeof(T) == 4 ? 2 : copy == kByHalves ? ExpertsRing<N, false, true>::kBlocks : ExpertsRing<N, false, false>::kBlocks;
}

template <typename T, int N, int COPY>
void (*pick_experts(bool down))(MoeArgs, int) {
    if constexpr (sizeof(T) == 4) return down ? k_experts32<true, COPY> : k_experts32<false, COPY>;
    else return down ? k_experts<T, N, true, COPY> : k_experts<T, N, false, COPY>;
}

template <typename T, int N>
void (*pick_copy(bool down, int copy))(MoeArgs, int) {
    if (copy == kBy16) return pick_experts<T, N, kBy16>(down);
    if (copy == kBy4 || sizeof(T) == 4) return pick_experts<T, N, kBy4>(down);
    if constexpr (sizeof(T) == 2) return copy == kByHalves ? pick_experts<T, N, kByHalves>(down) : pick_experts<T, N, kByElement>(down);
    else return nullptr;
}

template <typename T, int N>
MoeKernels moe_kernels(int tokens, bool route_words, int copy_up, int copy_down) {
    auto route = tokens >= 16 ? (route_words ? k_route<T, true, kRouteExperts> : k_route<T, false, kRouteExperts>)
                              : (route_words ? k_route<T, true, 1> : k_route<T, false, 1>);
    return {route, pick_copy<T, N>(false, copy_up), pick_copy<T, N>(true, copy_down), k_combine<T>,
            {experts_smem<T, N, false>(copy_up), experts_smem<T, N, true>(copy_down)},
            {experts_blocks<T, N>(copy_up), experts_blocks<T, N>(copy_down)}};
}

template <typename T>
MoeKernels pick_moe(int eights, int tokens, bool route_words, int copy_up, int copy_down) {
    if constexpr (sizeof(T) == 4) return moe_kernels<T, 1>(tokens, route_words, copy_up, copy_down);
    else
        return eights == 1   ? moe_kernels<T, 1>(tokens, route_words, copy_up, copy_down)
               : eights == 2 ? moe_kernels<T, 2>(tokens, route_words, copy_up, copy_down)
                             : moe_kernels<T, 4>(tokens, route_words, copy_up, copy_down);
}

}  // namespace l2d

using namespace l2d;

struct l2d_moe_plan {
    l2d_moe_desc desc;
    int sms;
    MoeArgs args;
    void *memory;
    void (*allowed[2])(MoeArgs, int);  // the kernels whose shared memory limit was raised last
};

namespace l2d {

// How rows of a matrix can be brought: by what they and their strides are aligned to.
int copy_of(const void *p, int64_t row, int64_t expert, int eb) {
    const uintptr_t any = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row * eb) | static_cast<uintptr_t>(expert * eb);
    return any % 16 == 0 ? kBy16 : any % 4 == 0 ? kBy4 : misaligned(p, 4) ? kByElement : kByHalves;
}

// Warps that share an item: so many that every warp of the GPU has two, as long as each has a few steps of it.
int parts_of(int64_t items, int warps, int steps) {
    int s = 1;
    while (s < kMoeWarps && items * s < 2 * warps && steps >= 8 * s) s *= 2;
    return s;
}

}  // namespace l2d

extern "C" {

int l2d_moe_plan_create(const l2d_moe_desc *desc, l2d_moe_plan **plan) {
    if (!plan) return set_error(L2D_ERR_INVALID, "null plan pointer");
    *plan = nullptr;
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    l2d_moe_desc d = *desc;
    if (!valid_dtype(d.dtype)) return set_error(L2D_ERR_INVALID, "bad dtype %d", d.dtype);
    constexpr int64_t kMost = 1 << 24;
    if (d.hidden < 1 || d.hidden > kMost || d.inner < 1 || d.inner > kMost)
        return set_error(L2D_ERR_INVALID, "hidden %lld and inner %lld: 1 to 2^24 are supported", static_cast<long long>(d.hidden), static_cast<long long>(d.inner));
    if (d.experts < 1 || d.experts > kMaxExperts) return set_error(L2D_ERR_UNSUPPORTED, "%d experts: 1 to %d are supported", d.experts, kMaxExperts);
    if (d.top < 1 || d.top > d.experts || d.top > 32) return set_error(L2D_ERR_UNSUPPORTED, "top %d of %d experts: 1 to 32 are supported", d.top, d.experts);
    if (d.max_tokens < 1 || d.max_tokens > 65535) return set_error(L2D_ERR_INVALID, "max_tokens %d: 1 to 65535 are supported", d.max_tokens);
    if (!d.x_token) d.x_token = d.hidden;
    if (!d.y_token) d.y_token = d.hidden;
    if (!d.router_row) d.router_row = d.hidden;
    if (!d.gate_row) d.gate_row = d.hidden;
    if (!d.up_row) d.up_row = d.hidden;
    if (!d.down_row) d.down_row = d.inner;
    const int64_t least = std::min({d.x_token, d.y_token, d.router_row, d.gate_row, d.up_row});
    if (least < d.hidden || d.down_row < d.inner) return set_error(L2D_ERR_INVALID, "a stride is shorter than its row");
    if (std::max({d.x_token, d.y_token, d.router_row, d.gate_row, d.up_row, d.down_row}) > (int64_t(1) << 32)) return set_error(L2D_ERR_INVALID, "strides too large");
    if (!d.gate_expert) d.gate_expert = d.gate_row * d.inner;
    if (!d.up_expert) d.up_expert = d.up_row * d.inner;
    if (!d.down_expert) d.down_expert = d.down_row * d.hidden;
    // Experts of one matrix after the other, or row by row beside another's: no row may lie in two.
    if (std::min({d.gate_expert, d.up_expert}) < d.hidden || d.down_expert < d.inner)
        return set_error(L2D_ERR_INVALID, "experts' strides are shorter than a row");
    if (std::max({d.gate_expert, d.up_expert, d.down_expert}) > (int64_t(1) << 48)) return set_error(L2D_ERR_INVALID, "strides too large");
    if (!d.router || !d.gate || !d.up || !d.down) return set_error(L2D_ERR_INVALID, "null pointer");
    const int eb = elem_bytes(d.dtype);
    if (misaligned(d.router, eb) || misaligned(d.gate, eb) || misaligned(d.up, eb) || misaligned(d.down, eb))
        return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    const int64_t slots = int64_t(d.max_tokens) * d.top, inner_row = (d.inner + 127) / 128 * 128;
    if (int64_t(std::max(d.hidden, d.inner)) * std::min<int64_t>(slots, d.experts + slots / 8) > INT32_MAX)
        return set_error(L2D_ERR_INVALID, "rows of all experts' entries must stay below 2^31");
    int sms = 0;
    int st = device_sms(d.device, &sms);
    if (st != L2D_OK) return st;
    OnDevice on(d.device);
    L2D_CUDA_TRY(on.err);
    // Sixteen-byte rows of numbers first.
    size_t bytes = 0;
    auto take = [&](size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    };
    const size_t tiles = (d.max_tokens + kRouteTokens - 1) / kRouteTokens, entries = d.experts + slots / 8 + 1;
    const size_t inner_at = take(slots * inner_row * 4), part_at = take(slots * d.hidden * 4), logits_at = take(size_t(d.max_tokens) * d.experts * 8),
                 ids_at = take(slots * 4), weights_at = take(slots * 4), largest_at = take(slots * 4), sorted_at = take(slots * 4),
                 entries_at = take(entries * 16), num_at = take(8), arrived_at = take((tiles + 1) * 4);
    void *memory = nullptr;
    cudaError_t e = cudaMalloc(&memory, bytes);
    if (e != cudaSuccess) {
        cudaGetLastError();  // not the next caller's error
        return set_error(L2D_ERR_CUDA, "experts' scratch of %zu bytes: %s", bytes, cudaGetErrorString(e));
    }
    // Counters, and what pads the rows of inner_out, on a stream of their own, so that nothing else on the device is waited for.
    cudaStream_t own = nullptr;
    e = cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking);
    if (e == cudaSuccess) {
        if (inner_row > d.inner)
            e = cudaMemset2DAsync(static_cast<char *>(memory) + inner_at + d.inner * 4, inner_row * 4, 0, (inner_row - d.inner) * 4, slots, own);
        if (e == cudaSuccess) e = cudaMemsetAsync(static_cast<char *>(memory) + arrived_at, 0, (tiles + 1) * 4, own);
        if (e == cudaSuccess) e = cudaStreamSynchronize(own);
        cudaStreamDestroy(own);
    }
    l2d_moe_plan *p = e == cudaSuccess ? new (std::nothrow) l2d_moe_plan() : nullptr;
    if (!p) {
        cudaFree(memory);
        return e != cudaSuccess ? set_error(L2D_ERR_CUDA, "experts' scratch: %s", cudaGetErrorString(e)) : set_error(L2D_ERR_INVALID, "out of host memory");
    }
    char *base = static_cast<char *>(memory);
    p->desc = d;
    p->sms = sms;
    p->memory = memory;
    MoeArgs &a = p->args;
    a.router = d.router;
    a.gate = d.gate;
    a.up = d.up;
    a.down = d.down;
    a.x_token = d.x_token;
    a.y_token = d.y_token;
    a.router_row = d.router_row;
    a.gate_row = d.gate_row;
    a.up_row = d.up_row;
    a.down_row = d.down_row;
    a.gate_expert = d.gate_expert;
    a.up_expert = d.up_expert;
    a.down_expert = d.down_expert;
    a.hidden = static_cast<int>(d.hidden);
    a.inner = static_cast<int>(d.inner);
    a.experts = d.experts;
    a.top = d.top;
    a.normalize = d.normalize;
    a.inner_out = reinterpret_cast<float *>(base + inner_at);
    a.part = reinterpret_cast<float *>(base + part_at);
    a.logits = reinterpret_cast<double *>(base + logits_at);
    a.ids = reinterpret_cast<int *>(base + ids_at);
    a.weights = reinterpret_cast<float *>(base + weights_at);
    a.largest = reinterpret_cast<uint32_t *>(base + largest_at);
    a.sorted = reinterpret_cast<int *>(base + sorted_at);
    a.entries = reinterpret_cast<int4 *>(base + entries_at);
    a.num_entries = reinterpret_cast<int *>(base + num_at);
    a.arrived = reinterpret_cast<unsigned *>(base + arrived_at);
    a.inner_row = inner_row;
    *plan = p;
    return L2D_OK;
}

int l2d_moe_forward(l2d_moe_plan *p, const void *x, void *y, int32_t *ids, float *weights, int tokens, void *stream) {
    if (!p) return set_error(L2D_ERR_INVALID, "null plan");
    const l2d_moe_desc &d = p->desc;
    if (tokens < 0 || tokens > d.max_tokens) return set_error(L2D_ERR_INVALID, "%d tokens of at most %d", tokens, d.max_tokens);
    if (tokens == 0) return L2D_OK;
    if (!x || !y) return set_error(L2D_ERR_INVALID, "null pointer");
    const int eb = elem_bytes(d.dtype);
    if (misaligned(x, eb) || misaligned(y, eb) || misaligned(ids, 4) || misaligned(weights, 4))
        return set_error(L2D_ERR_INVALID, "pointers must be aligned to their elements");
    OnDevice on(d.device);
    L2D_CUDA_TRY(on.err);
    MoeArgs a = p->args;
    a.x = x;
    a.y = y;
    a.ids_out = ids;
    a.weights_out = weights;
    a.tokens = tokens;
    // An expert with more slots than an entry takes is read again for the next one, mostly from L2.
    const int64_t likely = int64_t(tokens) * d.top / d.experts;
    const int eights = eb == 4 || tokens <= 8 || likely <= 3 ? 1 : tokens <= 16 || likely <= 8 ? 2 : 4;
    a.per_entry = 8 * eights;
    const int x_copy = copy_of(x, d.x_token, 0, eb), whole = eb == 4 && d.hidden % 4 ? kBy4 : kBy16;
    const int copy_up = std::max({copy_of(d.gate, d.gate_row, d.gate_expert, eb), copy_of(d.up, d.up_row, d.up_expert, eb), x_copy, whole});
    const int copy_down = copy_of(d.down, d.down_row, d.down_expert, eb);
    const bool route_words = x_copy == kBy16 && d.hidden % 8 == 0 && copy_of(d.router, d.router_row, 0, eb) == kBy16;
    const MoeKernels k = d.dtype == L2D_F32   ? pick_moe<float>(eights, tokens, route_words, copy_up, copy_down)
                         : d.dtype == L2D_F16 ? pick_moe<__half>(eights, tokens, route_words, copy_up, copy_down)
                                              : pick_moe<__nv_bfloat16>(eights, tokens, route_words, copy_up, copy_down);
    const int up_rows = eb == 4 ? 2 : 8, down_rows = eb == 4 ? 4 : 16, step = eb == 4 ? 128 : 64;
    const int64_t tiles_up = (d.inner + up_rows - 1) / up_rows, tiles_down = (d.hidden + down_rows - 1) / down_rows;
    L2D_CUDA_TRY(launch(k.route, dim3(tokens >= 16 ? (d.experts + kRouteExperts - 1) / kRouteExperts : d.experts, (tokens + kRouteTokens - 1) / kRouteTokens), kMoeThreads, 0, stream, a));
    const int64_t entries = std::min<int64_t>(int64_t(tokens) * d.top, d.experts);
    const int grid_up = k.blocks[0] * p->sms, grid_down = k.blocks[1] * p->sms;
    const int s_up = parts_of(entries * tiles_up, grid_up * kMoeWarps, static_cast<int>((d.hidden + step - 1) / step));
    const int s_down = parts_of(entries * tiles_down, grid_down * kMoeWarps, static_cast<int>((d.inner + step - 1) / step));
    if (p->allowed[0] != k.gate_up) L2D_CUDA_TRY(cudaFuncSetAttribute(k.gate_up, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem[0]));
    if (p->allowed[1] != k.down) L2D_CUDA_TRY(cudaFuncSetAttribute(k.down, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem[1]));
    p->allowed[0] = k.gate_up;
    p->allowed[1] = k.down;
    L2D_CUDA_TRY(launch(k.gate_up, dim3(grid_up), kMoeThreads, k.smem[0], stream, a, s_up));
    L2D_CUDA_TRY(launch(k.down, dim3(grid_down), kMoeThreads, k.smem[1], stream, a, s_down));
    L2D_CUDA_TRY(launch(k.combine, dim3((a.hidden + kMoeThreads - 1) / kMoeThreads, tokens), kMoeThreads, 0, stream, a));
    return L2D_OK;
}

int l2d_moe_plan_destroy(l2d_moe_plan *p) {
    if (!p) return L2D_OK;
    OnDevice on(p->desc.device);
    cudaError_t e = cudaFree(p->memory);  // waits for the device
    delete p;
    if (e != cudaSuccess) return set_error(L2D_ERR_CUDA, "moe_plan_destroy: %s", cudaGetErrorString(e));
    return L2D_OK;
}

}  // extern "C"

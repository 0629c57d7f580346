// Matrix-vector products with 4-bit weights and group scales (l2d_q4_gemv): the choice of a kernel and its
// shape, and the entry point.  The kernel itself is in l2d_q4.cuh.
#include "l2d_q4.cuh"

#include <algorithm>

namespace l2d {

// No columns: every sum is empty.
__global__ void k_q4_zero(Q4Args a) {
    dev::wait_for_previous();
    for (int64_t e = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; e < a.M * a.vectors; e += int64_t(gridDim.x) * blockDim.x)
        dev::store_as(a.y, a.dtype_y, e / a.M * a.stride_y + e % a.M, 0.0f);
}

// How many clusters of 1, 2, 4 and 8 blocks of one SM each run at the same time; looked up once per device, and kept
// as four numbers of 16 bits in one word.
int q4_clusters(int device, const Q4Entry &k, int (&clusters)[4]) {
    static std::atomic<uint64_t> known[kMaxDevices];
    uint64_t word = known[device].load(std::memory_order_relaxed);
    if (!word) {
        for (int i = 0; i < 4; ++i) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1u << i;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3(1u << i);
            cfg.blockDim = dim3(kQ4Threads);
            cfg.dynamicSmemBytes = 200 * 1024;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int found = 0;
            L2D_CUDA_TRY(cudaOccupancyMaxActiveClusters(&found, k.run, &cfg));
            word |= static_cast<uint64_t>(std::min(found, 0xffff)) << (16 * i);
        }
        known[device].store(word, std::memory_order_relaxed);
    }
    for (int i = 0; i < 4; ++i) clusters[i] = static_cast<int>(word >> (16 * i) & 0xffff);
    return L2D_OK;
}

// Blocks of a cluster and warps of a tile: the choice that gives a warp the least to do, in units of 128 columns
// of a tile of fp16 products in one n-tile.  Measured with every choice forced on 14 shapes of 360 x 171 to
// 28672 x 8192 and 1 to 16 vectors: this picks the fastest of them or one within 3 %, but 9 % for 8 vectors of
// 28672 x 8192 (46.8 us, and 43.1 in pairs).
struct Q4Shape {
    int ranks, warps_k, rows;
    int64_t shares;
};
Q4Shape q4_shape(int64_t M, int halves, int vectors, int tiles_n, bool bytes, int deep, const int *clusters) {
    constexpr double kStage = 2.4;    // 128 columns of two vectors staged
    constexpr double kCluster = 2.4;  // two barriers and the sums' way over distributed shared memory
    constexpr double kEnd = 2.0;      // a tile's end
    const double unit = bytes ? 0.6 : tiles_n == 1 ? 1.0 : tiles_n == 2 ? 1.5 : 2.4;
    Q4Shape best = {};
    double least = 1e300;
    for (int i = 0; i < 4; ++i) {
        const int ranks = 1 << i, steps = (halves + kQ4Deep - 1) / kQ4Deep;
        if (ranks > steps || (i && clusters[i] < 1)) break;
        const int64_t shares = std::max<int64_t>(std::min<int64_t>(M, std::max(1, clusters[i])), (M + kQ4MaxRows - 1) / kQ4MaxRows);
        const int rows = static_cast<int>((M + shares - 1) / shares), mine = std::min(halves, (steps + ranks - 1) / ranks * kQ4Deep);
        const double stage = (int64_t(mine) * vectors + 2 * kQ4Warps - 1) / (2 * kQ4Warps) * kStage + (i ? kCluster : 0.0);
        for (int wk = 1; wk <= kQ4Warps; wk *= 2) {
            const int groups = kQ4Warps / wk, each = (rows + groups - 1) / groups;
            const int share = (mine / deep + wk - 1) / wk * deep + (mine % deep + wk - 1) / wk;
            const int64_t waves = (shares + std::max(1, clusters[i]) - 1) / std::max(1, clusters[i]);
            const double work = waves * (stage + ((each + kQ4Rows - 1) / kQ4Rows) * (share * unit + kEnd));
            if (work < least) {
                least = work;
                best = {ranks, wk, rows, shares};
            }
        }
    }
    return best;
}

}  // namespace l2d

using namespace l2d;

extern "C" {

int l2d_q4_gemv(const l2d_q4_desc *desc, const void *x, int64_t stride_x, void *y, int64_t stride_y, int64_t vectors,
                void *stream) {
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    const l2d_q4_desc &d = *desc;
    constexpr int64_t kMax = int64_t(1) << 31;
    if (d.M < 0 || d.N < 0 || d.M >= kMax || d.N >= kMax / 16)
        return set_error(L2D_ERR_INVALID, "M = %lld, N = %lld: M below 2^31 and N below 2^27 are supported",
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
    if (misaligned(x, elem_bytes(d.dtype_x)) || misaligned(y, elem_bytes(d.dtype_y)) || misaligned(d.scales, elem_bytes(d.dtype_s)))
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
    a.dtype_x = d.dtype_x;
    a.dtype_y = d.dtype_y;
    a.dtype_s = d.dtype_s;
    a.per_group = ((uint64_t(1) << 40) + d.group / 128 - 1) / std::max(d.group / 128, 1);
    // Scales that are read together: at least `word` of them, and twice as many where they are aligned to that.
    const int word = d.group == 32 ? 2 : d.group == 64 ? 4 : d.group == 128 ? 2 : 1;
    auto together = [&](int n) { return lds % n == 0 && !misaligned(d.scales, 2 * n) && !misaligned(d.zeros, n); };
    const bool words = !misaligned(d.W, 16) && ldw % 16 == 0 && d.dtype_s != L2D_F32 && together(word);
    a.wide = together(2 * word);
    const int sub = d.group == 32 ? 4 : d.group == 64 ? 2 : 1;
    const bool fp32 = d.dtype_x == L2D_F32;
    const bool bytes = vectors * sub * q4_parts(fp32 ? kQ4Bytes32 : kQ4Bytes16) <= 8;  // columns of B
    const int parts = q4_parts(bytes ? fp32 ? kQ4Bytes32 : kQ4Bytes16 : fp32 ? kQ4Half32 : kQ4Half16);
    const int each = parts * sub;                                           // columns of B per vector
    const int most = 32 / each;                                             // vectors of one pass over the weights
    const int halves = static_cast<int>((d.N + kQ4Half - 1) / kQ4Half);
    for (int64_t v = 0; v < vectors; v += most) {
        a.vectors = static_cast<int>(std::min<int64_t>(most, vectors - v));
        a.x = static_cast<const char *>(x) + v * stride_x * elem_bytes(d.dtype_x);
        a.y = static_cast<char *>(y) + v * stride_y * elem_bytes(d.dtype_y);
        if (d.N == 0) {
            L2D_CUDA_TRY(launch(k_q4_zero, dim3(2 * sms), 256, 0, stream, a));
            continue;
        }
        const int tiles_n = a.vectors * each <= 8 ? 1 : a.vectors * each <= 16 ? 2 : 4;
        const bool zeros = d.zeros != nullptr;
        const Q4Entry k = bytes  ? q4_entry_bytes(fp32, d.group, zeros, words)
                          : fp32 ? q4_entry_float(tiles_n, d.group, zeros, words)
                                 : q4_entry_half(tiles_n, d.group, zeros, words);
        L2D_CUDA_TRY(allow_smem(k.run, 227 * 1024, d.device, *k.smem_set));
        int clusters[4];
        const int known = q4_clusters(d.device, k, clusters);
        if (known != L2D_OK) return known;
        const Q4Shape shape = q4_shape(d.M, halves, a.vectors, tiles_n, bytes, words ? kQ4Deep : 1, clusters);
        a.ranks = shape.ranks;
        a.warps_k = shape.warps_k;
        const int rows = shape.rows;
        // x is staged whole where it fits, else in as many parts as it takes.
        constexpr int kRoom = 227 * 1024 - 64;
        const int mine = ((halves + kQ4Deep - 1) / kQ4Deep + a.ranks - 1) / a.ranks * kQ4Deep;  // of a block
        a.y_rows = a.ranks > 1 ? rows : 0;
        const int per_half = q4_smem(tiles_n, bytes, a.vectors, parts, 4, 0).bytes - q4_smem(tiles_n, bytes, a.vectors, parts, 0, 0).bytes;  // four of them
        int fits = (kRoom - q4_smem(tiles_n, bytes, a.vectors, parts, 0, a.y_rows * a.vectors).bytes) / per_half * 4;
        if (fits < mine) {
            a.y_rows = rows;
            fits = (kRoom - q4_smem(tiles_n, bytes, a.vectors, parts, 0, rows * a.vectors).bytes) / per_half * 4;
            const int times = (mine + fits - 1) / fits;
            fits = ((mine + times - 1) / times + kQ4Deep - 1) / kQ4Deep * kQ4Deep;
        }
        a.stage_h = std::min(fits, mine);
        const int smem = q4_smem(tiles_n, bytes, a.vectors, parts, a.stage_h, a.y_rows * a.vectors).bytes;
        L2D_CUDA_TRY(launch_clusters(k.run, dim3(static_cast<unsigned>(shape.shares * a.ranks)), a.ranks, kQ4Threads, smem, stream, a));
    }
    return L2D_OK;
}

}  // extern "C"

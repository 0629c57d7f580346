// Matrix-vector products with 4-bit weights and group scales (l2d_q4_gemv).
//
//   y[b][i] = sum_j s[i][j / g] * (q[i][j] - z[i][j / g]) * x[b][j]
//
// One warp per row and vector; a lane takes every 32nd packed byte (two columns).
#include "l2d_launch.cuh"

#include <algorithm>

namespace l2d {

struct Q4Args {
    const uint8_t *W;
    const void *scales;
    const uint8_t *zeros;
    const void *x;
    void *y;
    int64_t M, N, ldw, lds, stride_x, stride_y, vectors;
    int group, dtype_x, dtype_y, dtype_s;
};

constexpr int kQ4Threads = 256;

__global__ void __launch_bounds__(kQ4Threads) k_q4_gemv(Q4Args a) {
    dev::wait_for_previous();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kQ4Threads / 32) + (threadIdx.x >> 5);
    if (row >= a.M) return;
    const uint8_t *w = a.W + row * a.ldw;
    for (int64_t b = blockIdx.y; b < a.vectors; b += gridDim.y) {
        float sum = 0.0f;
        for (int64_t j = lane; 2 * j < a.N; j += 32) {
            const int64_t g = row * a.lds + 2 * j / a.group;
            const float z = a.zeros ? static_cast<float>(a.zeros[g] & 15) : 8.0f;
            const uint32_t byte = w[j];
            float t = (static_cast<float>(byte & 15) - z) * dev::load_as_float(a.x, a.dtype_x, b * a.stride_x + 2 * j);
            if (2 * j + 1 < a.N)
                t = fmaf(static_cast<float>(byte >> 4) - z,
                         dev::load_as_float(a.x, a.dtype_x, b * a.stride_x + 2 * j + 1), t);
            sum = fmaf(dev::load_as_float(a.scales, a.dtype_s, g), t, sum);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) dev::store_as(a.y, a.dtype_y, b * a.stride_y + row, sum);
    }
}

}  // namespace l2d

using namespace l2d;

extern "C" {

int l2d_q4_gemv(const l2d_q4_desc *desc, const void *x, int64_t stride_x, void *y, int64_t stride_y, int64_t vectors,
                void *stream) {
    if (!desc) return set_error(L2D_ERR_INVALID, "null descriptor");
    const l2d_q4_desc &d = *desc;
    constexpr int64_t kMax = int64_t(1) << 31;
    if (d.M < 0 || d.N < 0 || d.M >= kMax || d.N >= kMax - 256)
        return set_error(L2D_ERR_INVALID, "M = %lld, N = %lld: 0 to 2^31 - 257 are supported",
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
    Q4Args a = {static_cast<const uint8_t *>(d.W), d.scales, static_cast<const uint8_t *>(d.zeros), x, y, d.M, d.N, ldw,
                lds, stride_x, stride_y, vectors, d.group, d.dtype_x, d.dtype_y, d.dtype_s};
    const dim3 grid(static_cast<unsigned>((d.M + kQ4Threads / 32 - 1) / (kQ4Threads / 32)),
                    static_cast<unsigned>(std::min<int64_t>(vectors, 65535)));
    L2D_CUDA_TRY(launch(k_q4_gemv, grid, kQ4Threads, 0, stream, a));
    return L2D_OK;
}

}  // extern "C"

// The fp16 kernels of the 4-bit products for fp32 vectors.
#include "l2d_q4.cuh"

namespace l2d {

Q4Entry q4_entry_float(int tiles_n, int group, bool zeros, bool words) {
    if (tiles_n == 1) return q4_entry<1, kQ4Half32>(group, zeros, words);
    return tiles_n == 2 ? q4_entry<2, kQ4Half32>(group, zeros, words) : q4_entry<4, kQ4Half32>(group, zeros, words);
}

}  // namespace l2d

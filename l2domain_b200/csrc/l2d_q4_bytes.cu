// The integer kernels of the 4-bit products, for few vectors.
#include "l2d_q4.cuh"

namespace l2d {

Q4Entry q4_entry_bytes(bool fp32, int group, bool zeros, bool words) {
    if (!fp32) return q4_entry<1, kQ4Bytes16>(group, zeros, words);
    return group == 128 ? q4_entry<1, 1, kQ4Bytes32>(zeros, words) : q4_entry<1, 0, kQ4Bytes32>(zeros, words);  // its eight columns are one group's
}

}  // namespace l2d

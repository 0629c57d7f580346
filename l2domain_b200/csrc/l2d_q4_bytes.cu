// The integer kernels of the 4-bit products, for few vectors.
#include "l2d_q4.cuh"

namespace l2d {

Q4Entry q4_entry_bytes(bool fp32, int group, bool zeros, bool words) {
    if (group == 64) return q4_entry<1, 2, kQ4Bytes16>(zeros, words);  // fp32, or shorter groups, take more than eight columns
    if (group == 128) return fp32 ? q4_entry<1, 1, kQ4Bytes32>(zeros, words) : q4_entry<1, 1, kQ4Bytes16>(zeros, words);
    return fp32 ? q4_entry<1, 0, kQ4Bytes32>(zeros, words) : q4_entry<1, 0, kQ4Bytes16>(zeros, words);
}

}  // namespace l2d

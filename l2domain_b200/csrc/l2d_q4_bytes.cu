// The integer kernels of the 4-bit products, for few vectors.
#include "l2d_q4.cuh"

namespace l2d {

Q4Entry q4_entry_bytes(int group, bool zeros, bool words) { return q4_entry<1, kQ4Bytes>(group, zeros, words); }

}  // namespace l2d

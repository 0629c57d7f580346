// Attention over a cache in 4 bits, fp32 queries.
#include "l2d_kv4.cuh"

namespace l2d {

AttnKernel pick_kv4_float(int D, int group, int heads) { return heads <= 8 ? pick_nibbles<float, 1>(D, group) : pick_nibbles<float, 2>(D, group); }

}  // namespace l2d

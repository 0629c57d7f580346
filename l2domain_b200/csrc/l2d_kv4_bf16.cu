// Attention over a cache in 4 bits, bf16 queries.
#include "l2d_kv4.cuh"

namespace l2d {

AttnKernel pick_kv4_bf16(int D, int group, int heads) { return heads <= 8 ? pick_nibbles<__nv_bfloat16, 1>(D, group) : pick_nibbles<__nv_bfloat16, 2>(D, group); }

}  // namespace l2d

// Attention over caches of 32 and 16 bits with other scores (l2d_attn_plan_create_scored): kernels of their own, so that
// plain scores keep theirs.  Four tanh (of fp32, as the scores are) per lane and 16 keys: 16 sequences of 4096 keys, 32 query and
// 8 key-value heads of 128, bf16, take 55 us, 4.9 TB/s, for 42 us of bytes.
#include "l2d_attn.cuh"

namespace l2d {

AttnKernel pick_attn_scored(int dtype, int D, int G) { return pick_dense<true>(dtype, D, G); }

}  // namespace l2d

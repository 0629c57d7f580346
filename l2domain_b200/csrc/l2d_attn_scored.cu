// Attention over caches of 32 and 16 bits with other scores (l2d_attn_plan_create_scored): kernels of their own, so that
// plain scores keep theirs.
#include "l2d_attn.cuh"

namespace l2d {

AttnKernel pick_attn_scored(int dtype, int D, int G) { return pick_dense<true>(dtype, D, G); }

}  // namespace l2d

// the backward walk over the rows of differential attention, bf16
#include "diff_attn.cuh"

namespace fmm {
namespace attn {

int walk_rows_bf16(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_walk<__nv_bfloat16, BackwardRows, false>(s, p, st); }

}  // namespace attn
}  // namespace fmm

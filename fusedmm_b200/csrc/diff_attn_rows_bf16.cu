// the backward walk over the rows of differential attention, bf16
#include "diff_attn_mma.cuh"

namespace fmm {
namespace attn {

int walk_rows_bf16(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_mma<__nv_bfloat16, true, BackwardRowsMma>(s, p, st); }

}  // namespace attn
}  // namespace fmm

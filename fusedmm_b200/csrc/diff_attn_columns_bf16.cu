// the backward walk over the columns of differential attention, bf16
#include "diff_attn_mma.cuh"

namespace fmm {
namespace attn {

int walk_columns_bf16(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_mma<__nv_bfloat16, false, BackwardColumnsMma>(s, p, st); }

}  // namespace attn
}  // namespace fmm

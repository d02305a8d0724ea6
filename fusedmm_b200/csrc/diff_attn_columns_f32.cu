// the backward walk over the columns of differential attention, f32
#include "diff_attn.cuh"

namespace fmm {
namespace attn {

int walk_columns_f32(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_walk<float, BackwardColumns, true>(s, p, st); }

}  // namespace attn
}  // namespace fmm

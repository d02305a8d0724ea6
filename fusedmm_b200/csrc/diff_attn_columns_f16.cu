// the backward walk over the columns of differential attention, f16
#include "diff_attn.cuh"

namespace fmm {
namespace attn {

int walk_columns_f16(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_walk<__half, BackwardColumns, true>(s, p, st); }

}  // namespace attn
}  // namespace fmm

// the forward walk of differential attention, f32
#include "diff_attn.cuh"

namespace fmm {
namespace attn {

int walk_forward_f32(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_walk<float, Forward, false>(s, p, st); }

}  // namespace attn
}  // namespace fmm

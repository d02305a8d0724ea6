// the forward walk of differential attention, f16
#include "diff_attn_mma.cuh"

namespace fmm {
namespace attn {

int walk_forward_f16(const WalkShape &s, const AttnParams &p, cudaStream_t st) { return launch_mma<__half, true, ForwardMma>(s, p, st); }

}  // namespace attn
}  // namespace fmm

// Score attention on the tensor cores for bf16 (score_tc.cuh).
#include "score_tc.cuh"

namespace fpk {
namespace score {

int launch_tc_bf16(const Params& p, int D, cudaStream_t s) { return launch_tc_type<__nv_bfloat16>(p, D, s); }

}  // namespace score
}  // namespace fpk

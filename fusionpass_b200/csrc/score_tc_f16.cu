// Score attention on the tensor cores for f16 (score_tc.cuh).
#include "score_tc.cuh"

namespace fpk {
namespace score {

int launch_tc_f16(const Params& p, int D, cudaStream_t s) { return launch_tc_type<__half>(p, D, s); }

}  // namespace score
}  // namespace fpk

// Tree attention on the tensor cores in bf16 (tree_tc.cuh).
#include "tree_tc.cuh"

namespace fpk {
namespace tree {

int launch_tc_bf16(const Params& p, int D, cudaStream_t s) { return tc::launch_type<__nv_bfloat16>(p, D, s); }

}  // namespace tree
}  // namespace fpk

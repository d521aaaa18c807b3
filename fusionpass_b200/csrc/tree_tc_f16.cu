// Tree attention on the tensor cores in f16 (tree_tc.cuh).
#include "tree_tc.cuh"

namespace fpk {
namespace tree {

int launch_tc_f16(const Params& p, int D, cudaStream_t s) { return tc::launch_type<__half>(p, D, s); }

}  // namespace tree
}  // namespace fpk

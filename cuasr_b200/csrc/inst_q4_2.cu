// Products with 4-bit weights, 16 columns at a time, 8 warps to a block.
#include "q4_launch.cuh"
namespace cuasr_b200 {
template cudaError_t launch_q4_columns<2, 1, 16>(int, bool, const CUtensorMap&, const Q4Params&, const Q4Launch&);
}  // namespace cuasr_b200

// Linear layers with 4-bit weights in groups of 64, without minima (q4_rows.cuh).
#include "q4_launch.cuh"

namespace sdb {

template int q4_launch<64, false>(const Q4Args&, const Q4Plan&, cudaStream_t);

}  // namespace sdb

// Linear layers with 4-bit weights in groups of 32, with minima (q4_rows.cuh).
#include "q4_launch.cuh"

namespace sdb {

template int q4_launch<32, true>(const Q4Args&, const Q4Plan&, cudaStream_t);

}  // namespace sdb

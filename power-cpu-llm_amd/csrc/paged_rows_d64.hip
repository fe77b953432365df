// The chunk kernels of many query rows of a step's new tokens at padded head dim 64.
#include "paged_rows.hpp"

template hipError_t pcl::launch_paged_rows<64>(const TreeParams &, int, bool, int64_t, int64_t,
                                                hipStream_t);

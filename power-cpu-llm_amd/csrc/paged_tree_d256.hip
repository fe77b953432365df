// The chunk kernels of the attention of a step's new tokens at padded head dim 256.
#include "paged_kv.hpp"

template hipError_t pcl::launch_paged_tree<256>(const TreeParams &, const TreeVariant &, bool,
                                                int64_t, int64_t, hipStream_t);

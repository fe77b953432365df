// The paged attention's chunk kernels at padded head dim 512.
#include "paged_kv.hpp"

template hipError_t pcl::launch_paged_kv<512>(const PagedParams &, bool, int64_t, hipStream_t);

#include "dh_product.h"

template int dhp::launch<float>(const dhp::Launch&, bool, bool, bool, const dhp::Shape&, hipStream_t);
template int dhp::launch_slope<float>(const void*, const void*, void*, void*, int64_t, int64_t, int64_t, int, float*, hipStream_t);

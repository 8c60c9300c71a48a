#include "wide.h"

template hipError_t tg::launch_wide<96>(const Attention&, int64_t, int, bool, hipStream_t);

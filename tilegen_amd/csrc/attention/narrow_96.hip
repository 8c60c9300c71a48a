#include "narrow.h"

template hipError_t tg::launch_narrow<96>(const Attention&, int64_t, int, bool, hipStream_t);

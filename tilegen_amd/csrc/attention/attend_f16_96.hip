#include "attend.h"

template hipError_t tg::launch_parts<_Float16, 96>(const Attention&, int, int, hipStream_t);

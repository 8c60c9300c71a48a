#include "attend.h"

template hipError_t tg::launch_parts<_Float16, 64>(const Attention&, int, int, hipStream_t);

#include "attend.h"

template hipError_t tg::launch_parts<_Float16, 64>(const Attention&, int, int, hipStream_t);
template hipError_t tg::launch_whole<_Float16, 64>(const Attention&, hipStream_t);

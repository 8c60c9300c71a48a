#include "attend.h"

template hipError_t tg::launch_parts<__bf16, 128>(const Attention&, int, int, hipStream_t);
template hipError_t tg::launch_whole<__bf16, 128>(const Attention&, hipStream_t);

// multi_kernel for heads of 64 and int8 codes.
#define FATHOM_ROWS8_MULTI_KERNEL
#include "rows8_multi.hpp"

void fathom::rows8::launch_multi_d64_int8(const MultiArgs &a, int q_dtype, hipStream_t st) { launch_multi<64, true>(a, q_dtype, st); }

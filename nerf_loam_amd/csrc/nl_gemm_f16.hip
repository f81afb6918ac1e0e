// nl_gemm_f16.hip -- the tiled product of nl_gemm.h for float16
#include "nl_gemm.h"

void nl_gemm_f16(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st) { nl_gemm_layout<_Float16>(g, layout, tile, grid, st); }

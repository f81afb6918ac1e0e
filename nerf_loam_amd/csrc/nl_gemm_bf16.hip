// nl_gemm_bf16.hip -- the tiled product of nl_gemm.h for bfloat16
#include "nl_gemm.h"

void nl_gemm_bf16(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st) { nl_gemm_layout<__bf16>(g, layout, tile, grid, st); }

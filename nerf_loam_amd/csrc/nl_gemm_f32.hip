// nl_gemm_f32.hip -- the tiled product of nl_gemm.h for float32 (six bf16 products of exact splits)
#include "nl_gemm.h"

void nl_gemm_f32(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st) { nl_gemm_layout<__bf16, true>(g, layout, tile, grid, st); }

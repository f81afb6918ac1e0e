// nl_gemm_f32.hip -- the tiled product of nl_gemm.h for float32 (six bf16 products of exact splits)
#include "nl_gemm.h"

void nl_gemm_f32(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st)
{
    if (layout == 0) nl_gemm_tile_f32<false, false>(g, tile, grid, st);
    else if (layout == 1) nl_gemm_tile_f32<false, true>(g, tile, grid, st);
    else nl_gemm_tile_f32<true, true>(g, tile, grid, st);
}
void nl_gemm_f32_to16(const NlGemm& g, int dt, int layout, dim3 grid, hipStream_t st)
{
    if (dt == NL_DT_BF16 && layout == 1) hipLaunchKernelGGL((k_gemm_f32<false, true, 64, NL_DT_BF16>), grid, dim3(256), 0, st, g);
    else if (dt == NL_DT_BF16) hipLaunchKernelGGL((k_gemm_f32<true, true, 64, NL_DT_BF16>), grid, dim3(256), 0, st, g);
    else if (layout == 1) hipLaunchKernelGGL((k_gemm_f32<false, true, 64, NL_DT_F16>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_gemm_f32<true, true, 64, NL_DT_F16>), grid, dim3(256), 0, st, g);
}

// nl_checkpoint.hip -- activations kept in 8 bits: e4m3 codes with a power of two per 32 neighbouring features (include/nerfloam_hip.h nl_mx8_*).
#include "nl_layers.h"

// A thread: eight neighbouring elements; four threads share a block of 32 and find its maximum among themselves.
__global__ __launch_bounds__(256) void k_mx8_encode(const void* x, long long ldx, long long M, int K, int dt, unsigned char* codes, unsigned char* exps, long long pitch)
{
    const long long per_row = pitch / 8, total = M * per_row;
    const bool row_aligned = (ldx & 3) == 0 && ((uintptr_t)x & (dt == NL_DT_F32 ? 15 : 7)) == 0;
    // whole blocks of threads run every round: the four threads of a 32-block stay together
    for (long long t0 = (long long)blockIdx.x * 256; t0 < total; t0 += (long long)gridDim.x * 256) {
        const long long t = t0 + threadIdx.x;
        const long long m = t / per_row;
        const int k = (int)(t - m * per_row) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
        if (t < total) {
            if (row_aligned && k + 7 < K) {
                const nl_f32x4 a = nl_load4(x, m * ldx + k, dt), b = nl_load4(x, m * ldx + k + 4, dt);
#pragma unroll
                for (int j = 0; j < 4; j++) { v[j] = a[j]; v[4 + j] = b[j]; }
            } else
#pragma unroll
                for (int j = 0; j < 8; j++) if (k + j < K) v[j] = nl_load_elem(x, m * ldx + k + j, dt);
        }
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) amax = fmaxf(amax, nl_finite_abs(v[j]));
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const int e = nl_mx_exponent(amax);
        const float s = nl_pow2(-e);
        if (t < total) {
            *reinterpret_cast<nl_i32x2*>(codes + m * pitch + k) = nl_i32x2{(int)nl_mx_encode4(v[0], v[1], v[2], v[3], s), (int)nl_mx_encode4(v[4], v[5], v[6], v[7], s)};
            if ((threadIdx.x & 3) == 0) exps[m * (pitch / 32) + (k >> 5)] = (unsigned char)(e + 127);
        }
    }
}

__global__ __launch_bounds__(256) void k_mx8_decode(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps, long long M, int K, int dt, void* out, long long pitch)
{
    const long long per_row = (K + 7) / 8, total = M * per_row;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const long long m = t / per_row;
        const int k = (int)(t - m * per_row) * 8;
        const nl_i32x2 c = *reinterpret_cast<const nl_i32x2*>(codes + m * pitch + k);
        const float s = nl_mx_scale(exps[m * (pitch / 32) + (k >> 5)]);
        const nl_f32x4 a = nl_mx_decode4((unsigned)c[0], s, nl_dtype_max(dt)), b = nl_mx_decode4((unsigned)c[1], s, nl_dtype_max(dt));
        if ((K & 3) == 0) {
            nl_store4(out, m * K + k, dt, a);
            if (k + 7 < K) nl_store4(out, m * K + k + 4, dt, b);
        } else
#pragma unroll
            for (int j = 0; j < 8; j++) if (k + j < K) nl_store_elem(out, m * K + k + j, dt, j < 4 ? a[j & 3] : b[j & 3]);
    }
}

static unsigned mx_grid(long long threads) { const long long b = (threads + 255) / 256; return (unsigned)(b < 8192 ? b : 8192); }

extern "C" {

int nl_mx8_encode(const void* x, long long ldx, long long M, int K, int dtype, unsigned char* codes, unsigned char* exps, void* stream)
{
    if (!nl_dtype_ok(dtype) || M < 0 || K < 1 || ldx < K) return NL_ERR_INVALID_ARG;
    if (M == 0) return NL_OK;
    if (!x || !codes || !exps || ((uintptr_t)codes & 7) || ((uintptr_t)x & (nl_dtype_size(dtype) - 1))) return NL_ERR_INVALID_ARG;
    const long long pitch = nl_up(K, NL_MX_BLOCK);
    hipLaunchKernelGGL(k_mx8_encode, dim3(mx_grid(M * (pitch / 8))), dim3(256), 0, (hipStream_t)stream, x, ldx, M, K, dtype, codes, exps, pitch);
    NL_LAUNCH_CHECK();
    return NL_OK;
}

int nl_mx8_decode(const unsigned char* codes, const unsigned char* exps, long long M, int K, int dtype, void* out, void* stream)
{
    if (!nl_dtype_ok(dtype) || M < 0 || K < 1) return NL_ERR_INVALID_ARG;
    if (M == 0) return NL_OK;
    if (!codes || !exps || !out || ((uintptr_t)codes & 7) || ((uintptr_t)out & 15)) return NL_ERR_INVALID_ARG;
    hipLaunchKernelGGL(k_mx8_decode, dim3(mx_grid(M * ((K + 7) / 8))), dim3(256), 0, (hipStream_t)stream, codes, exps, M, K, dtype, out, nl_up(K, NL_MX_BLOCK));
    NL_LAUNCH_CHECK();
    return NL_OK;
}

}  // extern "C"

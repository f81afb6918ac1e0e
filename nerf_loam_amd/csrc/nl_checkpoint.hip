// nl_checkpoint.hip -- activations kept in 8 bits: e4m3 codes with a power of two per 32 neighbouring features (include/nerfloam_hip.h nl_mx8_*).
#include "nl_layers.h"

// A thread: eight neighbouring elements; four threads share a block of 32 and find its maximum among themselves.  Bound by memory: 131072 x 1024 bf16, 268 MB read and
// 138 MB written, encoded in 87 us and decoded in 68 (4.7 and 6.0 TB/s; a large copy: 5.1).
template <int DT>
__global__ __launch_bounds__(256) void k_mx8_encode(const void* __restrict__ x, long long ldx, long long M, int K, unsigned char* codes, unsigned char* exps, long long pitch)
{
    const long long per_row = pitch / 8, total = M * per_row;
    // whole blocks of threads run every round: the four threads of a 32-block stay together
    for (long long t0 = (long long)blockIdx.x * 256; t0 < total; t0 += (long long)gridDim.x * 256) {
        const long long t = t0 + threadIdx.x;
        const long long m = t / per_row;
        const int k = (int)(t - m * per_row) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.0f;
        if (t < total) nl_load8<DT>(v, x, m * ldx + k, K - k);
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

template <int DT>
__global__ __launch_bounds__(256) void k_mx8_decode(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps, long long M, int K, void* __restrict__ out, long long pitch)
{
    const long long per_row = (K + 7) / 8, total = M * per_row;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const long long m = t / per_row;
        const int k = (int)(t - m * per_row) * 8;
        const nl_i32x2 c = *reinterpret_cast<const nl_i32x2*>(codes + m * pitch + k);
        const float s = nl_mx_scale(exps[m * (pitch / 32) + (k >> 5)]);
        const nl_f32x4 a = nl_mx_decode4((unsigned)c[0], s, nl_dtype_max(DT)), b = nl_mx_decode4((unsigned)c[1], s, nl_dtype_max(DT));
        const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        nl_store8<DT>(out, m * K + k, v, K - k);
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
    NL_WITH_DTYPE(dtype, hipLaunchKernelGGL(k_mx8_encode<DT>, dim3(mx_grid(M * (pitch / 8))), dim3(256), 0, (hipStream_t)stream, x, ldx, M, K, codes, exps, pitch));
    NL_LAUNCH_CHECK();
    return NL_OK;
}

int nl_mx8_decode(const unsigned char* codes, const unsigned char* exps, long long M, int K, int dtype, void* out, void* stream)
{
    if (!nl_dtype_ok(dtype) || M < 0 || K < 1) return NL_ERR_INVALID_ARG;
    if (M == 0) return NL_OK;
    if (!codes || !exps || !out || ((uintptr_t)codes & 7) || ((uintptr_t)out & 15)) return NL_ERR_INVALID_ARG;
    NL_WITH_DTYPE(dtype, hipLaunchKernelGGL(k_mx8_decode<DT>, dim3(mx_grid(M * ((K + 7) / 8))), dim3(256), 0, (hipStream_t)stream, codes, exps, M, K, out, nl_up(K, NL_MX_BLOCK)));
    NL_LAUNCH_CHECK();
    return NL_OK;
}

}  // extern "C"

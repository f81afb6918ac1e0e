// nl_layers.h -- shared by the layer operators (nl_linear*.hip, nl_checkpoint.hip, nl_embedding.hip): element types, activations, the 8-bit
// block format, the argument blocks of the matrix-product kernels and of their epilogue.
#pragma once
#include "nl_common.h"
#include "../../include/nerfloam_hip.h"

#define NL_MX_BLOCK 32                  // elements that share one power of two in the 8-bit format
#define NL_MX_EXP_MIN (-126)            // 2^-e stays a finite fp32 number

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 nl_bf16x8;
typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 nl_f16x8;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short nl_s16x4;
typedef __attribute__((__vector_size__(8 * sizeof(short)))) short nl_s16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float nl_f32x4;
typedef __attribute__((__vector_size__(4 * sizeof(int)))) int nl_i32x4;
typedef __attribute__((__vector_size__(2 * sizeof(int)))) int nl_i32x2;

static inline bool nl_dtype_ok(int dt) { return dt == NL_DT_F32 || dt == NL_DT_BF16 || dt == NL_DT_F16; }
static inline int nl_dtype_size(int dt) { return dt == NL_DT_F32 ? 4 : 2; }
static inline long long nl_up(long long a, long long b) { return (a + b - 1) / b * b; }

// operand of a product as it lies in memory: element (i, k) - i the row or column of the result, k the contraction index - at p + i si + k sk.
// NL_DT_MX8: 8-bit codes, whose power of two is e[k se + i / 32] (the blocks run along i).
#define NL_DT_MX8 3
struct NlOperand { const void* p; const unsigned char* e; long long si, sk, se; int type; };

// what happens to an element of the product: y = act(v + b) + r, and what the backward pass keeps of z = v + b
struct NlEpilogue {
    const void* b; const void* r; void* y; void* z;
    unsigned* bits; unsigned char* z8; unsigned char* z8e;
    float* part;                                   // partial sums of a split contraction, [split][M][N] fp32 (everything else unused then)
    long long ldr, ldy, ldz, ldbits, ldz8, ldz8e;
    int dt, act;
};

#ifdef __HIPCC__
__device__ __forceinline__ float nl_bf2f(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ unsigned short nl_f2bf(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }     // to nearest, ties to even
__device__ __forceinline__ float nl_h2f(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ unsigned short nl_f2h(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

__device__ __forceinline__ float nl_load_elem(const void* p, long long i, int dt)
{
    if (dt == NL_DT_F32) return ((const float*)p)[i];
    const unsigned short v = ((const unsigned short*)p)[i];
    return dt == NL_DT_BF16 ? nl_bf2f(v) : nl_h2f(v);
}
__device__ __forceinline__ void nl_store_elem(void* p, long long i, int dt, float v)
{
    if (dt == NL_DT_F32) ((float*)p)[i] = v;
    else ((unsigned short*)p)[i] = dt == NL_DT_BF16 ? nl_f2bf(v) : nl_f2h(v);
}
// four consecutive elements, aligned to four elements
__device__ __forceinline__ nl_f32x4 nl_load4(const void* p, long long i, int dt)
{
    if (dt == NL_DT_F32) return *reinterpret_cast<const nl_f32x4*>((const float*)p + i);
    const ushort4 u = *reinterpret_cast<const ushort4*>((const unsigned short*)p + i);
    if (dt == NL_DT_BF16) return nl_f32x4{nl_bf2f(u.x), nl_bf2f(u.y), nl_bf2f(u.z), nl_bf2f(u.w)};
    return nl_f32x4{nl_h2f(u.x), nl_h2f(u.y), nl_h2f(u.z), nl_h2f(u.w)};
}
__device__ __forceinline__ void nl_store4(void* p, long long i, int dt, nl_f32x4 v)
{
    if (dt == NL_DT_F32) { *reinterpret_cast<nl_f32x4*>((float*)p + i) = v; return; }
    ushort4 u;
    if (dt == NL_DT_BF16) u = make_ushort4(nl_f2bf(v[0]), nl_f2bf(v[1]), nl_f2bf(v[2]), nl_f2bf(v[3]));
    else u = make_ushort4(nl_f2h(v[0]), nl_f2h(v[1]), nl_f2h(v[2]), nl_f2h(v[3]));
    *reinterpret_cast<ushort4*>((unsigned short*)p + i) = u;
}

// activations and their slopes.  erff, not the tanh form: the exact definition is what a checkpoint or another framework's model was trained with.
__device__ __forceinline__ float nl_act(float z, int act)
{
    if (act == NL_ACT_RELU) return z < 0.0f ? 0.0f : z;                       // (a NaN stays one)
    if (act == NL_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    if (act == NL_ACT_SILU) return z / (1.0f + expf(-z));
    return z;
}
__device__ __forceinline__ float nl_act_slope(float z, int act)
{
    if (act == NL_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == NL_ACT_GELU) return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    if (act == NL_ACT_SILU) { const float s = 1.0f / (1.0f + expf(-z)); return s * (1.0f + z * (1.0f - s)); }
    return 1.0f;
}

// ---- the 8-bit format ----
// A block of 32 elements shares 2^e, e the smallest exponent with max |x| <= 448 2^e (448 = 1.75 2^8 is the largest e4m3 number); a code is x / 2^e to
// nearest, ties to even.  x / 2^e is exact (a power of two, nothing overflows: |x / 2^e| <= 448; what underflows is below the smallest code's half).
// Infinities and NaN do not enter the maximum and become the code of NaN.
__device__ __forceinline__ int nl_mx_exponent(float amax)
{
    const unsigned u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);     // (a denormal amax reads as exponent -127: clipped below)
    return e < NL_MX_EXP_MIN ? NL_MX_EXP_MIN : e;
}
__device__ __forceinline__ float nl_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }      // -126 <= e <= 127
__device__ __forceinline__ float nl_finite_abs(float v) { const unsigned u = __float_as_uint(v) & 0x7FFFFFFFu; return u < 0x7F800000u ? __uint_as_float(u) : 0.0f; }
// four codes in a word; scale = 2^-e
__device__ __forceinline__ unsigned nl_mx_encode4(float a, float b, float c, float d, float scale)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * scale, b * scale, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c * scale, d * scale, w, true);
    unsigned u = (unsigned)w;
    if (!(fabsf(a) < INFINITY)) u |= 0x7Fu;
    if (!(fabsf(b) < INFINITY)) u |= 0x7F00u;
    if (!(fabsf(c) < INFINITY)) u |= 0x7F0000u;
    if (!(fabsf(d) < INFINITY)) u |= 0x7F000000u;
    return u;
}
__device__ __forceinline__ float nl_mx_scale(unsigned char e) { return __uint_as_float((unsigned)e << 23); }      // the stored byte is e + 127, 1 .. 254
// A value next to the type's largest one may round up to a code beyond it (fp16: from 63488 on, 65536): such a code decodes to the type's largest number
__device__ __forceinline__ float nl_dtype_max(int dt) { return dt == NL_DT_F16 ? NL_F16_MAX : dt == NL_DT_BF16 ? 3.38953139e38f : 3.40282347e38f; }
__device__ __forceinline__ float nl_mx_clip(float v, float most) { return fabsf(v) > most ? copysignf(most, v) : v; }

__device__ __forceinline__ nl_f32x4 nl_mx_decode4(unsigned w, float scale, float most)
{
    return nl_f32x4{nl_mx_clip(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * scale, most), nl_mx_clip(__builtin_amdgcn_cvt_f32_fp8((int)w, 1) * scale, most),
                    nl_mx_clip(__builtin_amdgcn_cvt_f32_fp8((int)w, 2) * scale, most), nl_mx_clip(__builtin_amdgcn_cvt_f32_fp8((int)w, 3) * scale, most)};
}

// ---- epilogue ----
// One call: a wave's 16 rows x 32 columns of the result.  Lane l holds, of row m = m0 + (l & 15), the columns n0 + 4 (l >> 4) + 0..3 in a and the same + 16
// in b (the matrix instruction gets the column operand as its first one: four neighbouring columns of a row per lane, one 8- or 16-byte store each).
__device__ __forceinline__ void nl_epilogue_pair(const NlEpilogue& ep, nl_f32x4 va, nl_f32x4 vb, long long m0, int n0, long long M, int N, long long split_off)
{
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const long long m = m0 + (lane & 15);
    const bool row = m < M;
    if (n0 >= N) return;                                          // (uniform over the wave)
    if (ep.part) {
        if (!row) return;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int n = n0 + 16 * h + 4 * g;
            const nl_f32x4 v = h ? vb : va;
            float* o = ep.part + split_off + m * N + n;
            if ((N & 3) == 0 && n < N) *reinterpret_cast<nl_f32x4*>(o) = v;
            else {
#pragma unroll
                for (int j = 0; j < 4; j++) if (n + j < N) o[j] = v[j];
            }
        }
        return;
    }
    float z[8];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int n = n0 + 16 * h + 4 * g;
        const nl_f32x4 v = h ? vb : va;
#pragma unroll
        for (int j = 0; j < 4; j++) z[4 * h + j] = v[j] + ((ep.b && n + j < N) ? nl_load_elem(ep.b, n + j, ep.dt) : 0.0f);
    }
    if (ep.bits) {                                                // one bit per element: z > 0
        unsigned w = 0;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 4; j++) w |= (unsigned)(z[4 * h + j] > 0.0f && n0 + 16 * h + 4 * g + j < N) << (16 * h + 4 * g + j);
        w |= __shfl_xor(w, 16);
        w |= __shfl_xor(w, 32);
        if (row && g == 0) ep.bits[m * ep.ldbits + (n0 >> 5)] = w;
    }
    if (ep.z8) {                                                  // z in 8 bits, from the fp32 values
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) amax = fmaxf(amax, n0 + 16 * (j >> 2) + 4 * g + (j & 3) < N ? nl_finite_abs(z[j]) : 0.0f);
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        const int e = nl_mx_exponent(amax);
        const float s = nl_pow2(-e);
        if (row) {
#pragma unroll
            for (int h = 0; h < 2; h++) {                         // (rows of codes are padded to whole blocks: always a whole word; columns behind N hold zeros)
                const int n = n0 + 16 * h + 4 * g;
                *reinterpret_cast<unsigned*>(ep.z8 + m * ep.ldz8 + n) =
                    nl_mx_encode4(n < N ? z[4 * h] : 0.0f, n + 1 < N ? z[4 * h + 1] : 0.0f, n + 2 < N ? z[4 * h + 2] : 0.0f, n + 3 < N ? z[4 * h + 3] : 0.0f, s);
            }
            if (g == 0) ep.z8e[m * ep.ldz8e + (n0 >> 5)] = (unsigned char)(e + 127);
        }
    }
    if (!row) return;
    const int es = ep.dt == NL_DT_F32 ? 16 : 8;                   // bytes of four elements
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int n = n0 + 16 * h + 4 * g;
        if (n >= N) continue;
        const bool whole = n + 3 < N;
        if (ep.z) {
            const nl_f32x4 v = {z[4 * h], z[4 * h + 1], z[4 * h + 2], z[4 * h + 3]};
            if (whole && (ep.ldz & 3) == 0) nl_store4(ep.z, m * ep.ldz + n, ep.dt, v);
            else {
#pragma unroll
                for (int j = 0; j < 4; j++) if (n + j < N) nl_store_elem(ep.z, m * ep.ldz + n + j, ep.dt, v[j]);
            }
        }
        nl_f32x4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = nl_act(z[4 * h + j], ep.act);
        if (ep.r) {
            if (whole && (ep.ldr & 3) == 0 && ((uintptr_t)ep.r & (es - 1)) == 0) o += nl_load4(ep.r, m * ep.ldr + n, ep.dt);
            else {
#pragma unroll
                for (int j = 0; j < 4; j++) if (n + j < N) o[j] += nl_load_elem(ep.r, m * ep.ldr + n + j, ep.dt);
            }
        }
        if (whole && (ep.ldy & 3) == 0 && ((uintptr_t)ep.y & (es - 1)) == 0) nl_store4(ep.y, m * ep.ldy + n, ep.dt, o);
        else {
#pragma unroll
            for (int j = 0; j < 4; j++) if (n + j < N) nl_store_elem(ep.y, m * ep.ldy + n + j, ep.dt, o[j]);
        }
    }
}
#endif

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

#define NL_DT_MX8 3                     // 8-bit codes with their powers of two, as an operand of a product

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

// Elements of a type that is known at compile time (DT: NL_DT_*).  A type looked up at run time puts every load into a branch of its own, and a branch's end waits for
// what it loaded: one access in flight.
template <int DT> __device__ __forceinline__ float nl_load_elem(const void* p, long long i)
{
    if (DT == NL_DT_F32) return ((const float*)p)[i];
    const unsigned short v = ((const unsigned short*)p)[i];
    return DT == NL_DT_BF16 ? nl_bf2f(v) : nl_h2f(v);
}
template <int DT> __device__ __forceinline__ void nl_store_elem(void* p, long long i, float v)
{
    if (DT == NL_DT_F32) ((float*)p)[i] = v;
    else ((unsigned short*)p)[i] = DT == NL_DT_BF16 ? nl_f2bf(v) : nl_f2h(v);
}
// Eight elements of a row as they lie in memory, wherever they begin (global memory takes accesses of 16 bytes at any address): fetched early, converted where used.
// 1003 x 1001 -> 777 bf16 with residual, no row aligned: 14.1 us, element by element 18.1.
typedef __attribute__((__vector_size__(4 * sizeof(int)), __aligned__(2))) int nl_i32x4_at2;
typedef __attribute__((__vector_size__(4 * sizeof(int)), __aligned__(4))) int nl_i32x4_at4;
template <int DT> struct NlRaw8 { nl_i32x4 w[DT == NL_DT_F32 ? 2 : 1]; };
template <int DT> __device__ __forceinline__ NlRaw8<DT> nl_raw8(const void* p, long long i)
{
    NlRaw8<DT> o;
    if constexpr (DT == NL_DT_F32) {
        const nl_i32x4_at4* q = reinterpret_cast<const nl_i32x4_at4*>((const float*)p + i);
        o.w[0] = q[0]; o.w[1] = q[1];
    } else o.w[0] = *reinterpret_cast<const nl_i32x4_at2*>((const unsigned short*)p + i);
    return o;
}
template <int DT> __device__ __forceinline__ void nl_unraw8(float* v, const NlRaw8<DT>& r)
{
    if constexpr (DT == NL_DT_F32) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = __int_as_float(r.w[j >> 2][j & 3]);
    } else {
        const nl_s16x8 u = __builtin_bit_cast(nl_s16x8, r.w[0]);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = DT == NL_DT_BF16 ? nl_bf2f((unsigned short)u[j]) : nl_h2f((unsigned short)u[j]);
    }
}
// four neighbouring elements
typedef __attribute__((__vector_size__(2 * sizeof(int)), __aligned__(2))) int nl_i32x2_at2;
template <int DT> __device__ __forceinline__ nl_f32x4 nl_load4(const void* p, long long i)
{
    if constexpr (DT == NL_DT_F32) return __builtin_bit_cast(nl_f32x4, (nl_i32x4)*reinterpret_cast<const nl_i32x4_at4*>((const float*)p + i));
    else {
        const nl_s16x4 u = __builtin_bit_cast(nl_s16x4, (nl_i32x2)*reinterpret_cast<const nl_i32x2_at2*>((const unsigned short*)p + i));
        nl_f32x4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = DT == NL_DT_BF16 ? nl_bf2f((unsigned short)u[j]) : nl_h2f((unsigned short)u[j]);
        return o;
    }
}
template <int DT> __device__ __forceinline__ void nl_store4(void* p, long long i, nl_f32x4 v)
{
    if constexpr (DT == NL_DT_F32) *reinterpret_cast<nl_i32x4_at4*>((float*)p + i) = __builtin_bit_cast(nl_i32x4, v);
    else {
        nl_s16x4 u;
#pragma unroll
        for (int j = 0; j < 4; j++) u[j] = (short)(DT == NL_DT_BF16 ? nl_f2bf(v[j]) : nl_f2h(v[j]));
        *reinterpret_cast<nl_i32x2_at2*>((unsigned short*)p + i) = __builtin_bit_cast(nl_i32x2, u);
    }
}
// `left` of the eight are inside the row (zeros behind them)
template <int DT> __device__ __forceinline__ void nl_load8(float* v, const void* p, long long i, int left)
{
    if (left >= 8) { nl_unraw8<DT>(v, nl_raw8<DT>(p, i)); return; }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < left ? nl_load_elem<DT>(p, i + j) : 0.0f;
}
template <int DT> __device__ __forceinline__ void nl_store8(void* p, long long i, const float* v, int left)
{
    if (left < 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) if (j < left) nl_store_elem<DT>(p, i + j, v[j]);
        return;
    }
    if constexpr (DT == NL_DT_F32) {
        nl_i32x4_at4* q = reinterpret_cast<nl_i32x4_at4*>((float*)p + i);
        q[0] = __builtin_bit_cast(nl_i32x4, nl_f32x4{v[0], v[1], v[2], v[3]});
        q[1] = __builtin_bit_cast(nl_i32x4, nl_f32x4{v[4], v[5], v[6], v[7]});
    } else {
        nl_s16x8 u;
#pragma unroll
        for (int j = 0; j < 8; j++) u[j] = (short)(DT == NL_DT_BF16 ? nl_f2bf(v[j]) : nl_f2h(v[j]));
        *reinterpret_cast<nl_i32x4_at2*>((unsigned short*)p + i) = __builtin_bit_cast(nl_i32x4, u);
    }
}

// activations and their slopes.  Products whose epilogue or dz pass calls erff and expf are bound by vector arithmetic (dz of 16384 x 4096 gelu: 157 us, where
// memory takes 78), so both come from one hardware exponential and one hardware reciprocal.
// Phi(z) = (1 + erf(z / sqrt 2)) / 2 after Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26: with x = |z| / sqrt 2 and t = 1 / (1 + 0.3275911 x),
// erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2) to 1.5e-7; the same exponential is the density of gelu's slope.
__device__ __forceinline__ float nl_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ void nl_normal(float z, float& cdf, float& e)          // e = exp(-z^2 / 2)
{
    const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
    e = nl_exp(-x * x);
    float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
    p = __builtin_fmaf(p, t, 1.421413741f);
    p = __builtin_fmaf(p, t, -0.284496736f);
    p = __builtin_fmaf(p, t, 0.254829592f);
    const float tail = 0.5f * p * t * e;                                           // 1 - Phi(|z|)
    cdf = z < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ float nl_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + nl_exp(-z)); }
__device__ __forceinline__ float nl_act(float z, int act)
{
    if (act == NL_ACT_RELU) return z < 0.0f ? 0.0f : z;                       // (a NaN stays one)
    if (act == NL_ACT_GELU) { float c, e; nl_normal(z, c, e); return z * c; }
    if (act == NL_ACT_SILU) return z * nl_sigmoid(z);
    return z;
}
__device__ __forceinline__ float nl_act_slope(float z, int act)
{
    if (act == NL_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == NL_ACT_GELU) { float c, e; nl_normal(z, c, e); return __builtin_fmaf(z * e, 0.39894228040143268f, c); }
    if (act == NL_ACT_SILU) { const float s = nl_sigmoid(z); return s * __builtin_fmaf(z, 1.0f - s, 1.0f); }
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
// A lane holds eight neighbouring columns n .. n + 7 (n a multiple of 8) of row m of the product; four neighbouring lanes hold 32 columns from a multiple of 32 on.
// Every lane of a wave calls (rows and columns beyond the result do not store).
__device__ __forceinline__ void nl_act8(float* v, int act)
{
    if (act == NL_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = nl_act(v[j], NL_ACT_RELU);
    } else if (act == NL_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = nl_act(v[j], NL_ACT_GELU);
    } else if (act == NL_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = nl_act(v[j], NL_ACT_SILU);
    }
}
// b, r: the bias and the residual of the eight columns, zeros where there is none.  INSIDE: the wave's rows and columns all are inside the result, no lane asks
template <int DT, bool INSIDE> __device__ __forceinline__ void nl_epilogue8(const NlEpilogue& ep, float* v, const float* b, const float* r, long long m, int n, long long M, int N, long long split_off)
{
    const bool row = INSIDE || m < M, live = INSIDE || (row && n < N);
    const int lane = threadIdx.x & 63, left = INSIDE ? 8 : N - n;
    if (ep.part) {
        if (live) nl_store8<NL_DT_F32>(ep.part + split_off, m * N + n, v, left);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += b[j];
    if (ep.bits) {                                                // one bit per element: z > 0
        unsigned w = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) w |= (unsigned)(v[j] > 0.0f && j < left) << j;
        w <<= 8 * (lane & 3);
        w |= __shfl_xor(w, 1);
        w |= __shfl_xor(w, 2);
        if (live && (lane & 3) == 0) ep.bits[m * ep.ldbits + (n >> 5)] = w;
    }
    if (ep.z8) {                                                  // z in 8 bits, from the fp32 values; rows of codes are padded to whole blocks with zeros
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) { if (j >= left) v[j] = 0.0f; amax = fmaxf(amax, nl_finite_abs(v[j])); }
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const int e = nl_mx_exponent(amax);
        const float s = nl_pow2(-e);
        if (row && n < ep.ldz8) {
            *reinterpret_cast<nl_i32x2*>(ep.z8 + m * ep.ldz8 + n) = nl_i32x2{(int)nl_mx_encode4(v[0], v[1], v[2], v[3], s), (int)nl_mx_encode4(v[4], v[5], v[6], v[7], s)};
            if ((lane & 3) == 0) ep.z8e[m * ep.ldz8e + (n >> 5)] = (unsigned char)(e + 127);
        }
    }
    if (!live) return;
    if (ep.z) nl_store8<DT>(ep.z, m * ep.ldz + n, v, left);      // (rounded to the type: half the bytes; only slopes are taken of it)
    nl_act8(v, ep.act);
    if (ep.r) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] += r[j];
    }
    nl_store8<DT>(ep.y, m * ep.ldy + n, v, left);
}
// the same with bias and residual fetched on the spot
template <int DT> __device__ __forceinline__ void nl_epilogue8_fetch(const NlEpilogue& ep, float* v, long long m, int n, long long M, int N, long long split_off)
{
    float b[8] = {}, r[8] = {};
    if (!ep.part && m < M && n < N) {
        if (ep.r) nl_load8<DT>(r, ep.r, m * ep.ldr + n, N - n);
        if (ep.b) nl_load8<DT>(b, ep.b, n, N - n);
    }
    nl_epilogue8<DT, false>(ep, v, b, r, m, n, M, N, split_off);
}
// Workgroups in one row as long as a launch takes it (a grid's axis has at most 2^32 - 1 threads), else in several; the number of a workgroup
__device__ __forceinline__ long long nl_block() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }
inline dim3 nl_blocks(long long n) { const long long row = 1 << 22; return n <= row ? dim3((unsigned)n) : dim3((unsigned)row, (unsigned)((n + row - 1) / row)); }
// a kernel launch (or any statement) with the type as a compile-time constant DT
#define NL_WITH_DTYPE(dt, ...)                                                            \
    do {                                                                                  \
        if ((dt) == NL_DT_F32) { constexpr int DT = NL_DT_F32; __VA_ARGS__; }             \
        else if ((dt) == NL_DT_BF16) { constexpr int DT = NL_DT_BF16; __VA_ARGS__; }      \
        else { constexpr int DT = NL_DT_F16; __VA_ARGS__; }                               \
    } while (0)
#endif

// nl_linear.hip -- one linear layer: z = x w^T + b, y = act(z) + r, and its backward pass (include/nerfloam_hip.h NlLinear).
//
// Reference behaviour: torch.nn.Linear + ReLU of the decoder (/root/reference/src/variations/lidar.py:105-123), any width, any depth.
#include "nl_layers.h"

// ---------------------------------------------------------------------------------------------
// k_linear_any: any strides, any alignment, any element type.  64 x 64 results per workgroup of four waves, contraction steps of 32; both operands are read
// element by element where nothing better is known of them, rounded or split to 16-bit planes and staged in LDS.
// fp32 (PL = 3): x = h + m + l, three bf16 numbers to nearest, exact (8 bits each of 24); of the nine products the six down to 2^-18 are summed, the
// smallest first: l h, h l, m m, m h, h m, h h.  What is dropped (m l, l m, l l) is below 2^-26 |x||w|.
// ---------------------------------------------------------------------------------------------
#define ANY_T 64
#define ANY_K 32
#define ANY_PITCH 40            // 16-bit elements per row of a staged plane: 80 bytes, so that the 16 rows of a fragment start in different banks

template <class T> struct NlMma;
template <> struct NlMma<__bf16> {
    typedef nl_bf16x8 V;
    static __device__ __forceinline__ nl_f32x4 mma(nl_s16x8 a, nl_s16x8 b, nl_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0); }
};
template <> struct NlMma<_Float16> {
    typedef nl_f16x8 V;
    static __device__ __forceinline__ nl_f32x4 mma(nl_s16x8 a, nl_s16x8 b, nl_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0); }
};

// x = h + m + l; a value whose rounding would overflow is cut instead, an infinity or NaN stays in h alone
__device__ __forceinline__ void nl_split3(float x, unsigned short& h, unsigned short& m, unsigned short& l)
{
    h = nl_f2bf(x);
    if ((h & 0x7F80) == 0x7F80) {
        if (!(fabsf(x) < INFINITY)) { m = l = 0; return; }
        h = (unsigned short)(__float_as_uint(x) >> 16);
    }
    const float r = x - nl_bf2f(h);
    m = nl_f2bf(r);
    l = nl_f2bf(r - nl_bf2f(m));
}

__device__ __forceinline__ float any_elem(const NlOperand& o, long long i, long long k, float most)
{
    if (o.type == NL_DT_MX8) {
        return nl_mx_clip(__builtin_amdgcn_cvt_f32_fp8((int)((const unsigned char*)o.p)[i * o.si + k * o.sk], 0) * nl_mx_scale(o.e[k * o.se + (i >> 5)]), most);
    }
    return nl_load_elem(o.p, i * o.si + k * o.sk, o.type);
}

template <class T, int PL>
__device__ __forceinline__ void any_stage(const NlOperand& o, long long i0, long long I, long long k0, long long k1, unsigned short* lds)
{
    const int t = threadIdx.x;
    const float most = nl_dtype_max(PL == 3 ? NL_DT_F32 : __is_same(T, _Float16) ? NL_DT_F16 : NL_DT_BF16);
    const bool along_k = o.sk == 1;
    const int i = along_k ? t >> 2 : 8 * (t & 7), k = along_k ? 8 * (t & 3) : t >> 3;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int ii = along_k ? i : i + j, kk = along_k ? k + j : k;
        const float v = (i0 + ii < I && k0 + kk < k1) ? any_elem(o, i0 + ii, k0 + kk, most) : 0.0f;
        unsigned short* d = lds + ii * ANY_PITCH + kk;
        if (PL == 3) nl_split3(v, d[0], d[ANY_T * ANY_PITCH], d[2 * ANY_T * ANY_PITCH]);
        else d[0] = __is_same(T, _Float16) ? nl_f2h(v) : nl_f2bf(v);
    }
}

template <class T, int PL>
__global__ __launch_bounds__(256) void k_linear_any(NlOperand A, NlOperand B, long long M, int N, long long K, int tiles_n, long long kchunk, NlEpilogue ep)
{
    __shared__ __align__(16) unsigned short s_a[PL * ANY_T * ANY_PITCH], s_b[PL * ANY_T * ANY_PITCH];
    const long long m0 = (long long)(blockIdx.x / tiles_n) * ANY_T;
    const int n0 = (int)(blockIdx.x % tiles_n) * ANY_T;
    const long long k0 = blockIdx.y * kchunk, k1 = k0 + kchunk < K ? k0 + kchunk : K;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = 32 * (wave >> 1), wn = 32 * (wave & 1);
    nl_f32x4 acc[2][2] = {};
    for (long long k = k0; k < k1; k += ANY_K) {
        any_stage<T, PL>(A, m0, M, k, k1, s_a);
        any_stage<T, PL>(B, n0, N, k, k1, s_b);
        __syncthreads();
        nl_s16x8 fa[2][PL], fb[2][PL];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int p = 0; p < PL; p++) {
                const int at = p * ANY_T * ANY_PITCH + (lane & 15) * ANY_PITCH + 8 * (lane >> 4) + 16 * s * ANY_PITCH;
                fa[s][p] = *reinterpret_cast<const nl_s16x8*>(s_a + at + wm * ANY_PITCH);
                fb[s][p] = *reinterpret_cast<const nl_s16x8*>(s_b + at + wn * ANY_PITCH);
            }
#pragma unroll
        for (int sum = PL == 3 ? 2 : 0; sum >= 0; sum--)              // planes p + q = sum: products of one order of magnitude, the smallest first
#pragma unroll
            for (int p = 0; p <= sum; p++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) acc[i][j] = NlMma<T>::mma(fb[j][sum - p], fa[i][p], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; i++) nl_epilogue_pair(ep, acc[i][0], acc[i][1], m0 + wm + 16 * i, n0 + wn, M, N, (long long)blockIdx.y * M * N);
}

// ---------------------------------------------------------------------------------------------
// k_linear_join: sums the pieces of a split contraction in their order and runs the epilogue.  One wave: 16 rows x 32 columns.
// ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_linear_join(const float* __restrict__ part, int splits, long long M, int N, int tiles_n, NlEpilogue ep)
{
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long m0 = tile / tiles_n * 16;
    const int n0 = (int)(tile % tiles_n) * 32, lane = threadIdx.x & 63;
    if (m0 >= M) return;                                          // (the whole wave)
    const long long m = m0 + (lane & 15);
    nl_f32x4 v[2] = {};
    if (m < M)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int n = n0 + 16 * h + 4 * (lane >> 4);
            if (n >= N) continue;
            const float* p = part + m * N + n;
            for (int s = 0; s < splits; s++, p += M * N) {
                if ((N & 3) == 0) v[h] += *reinterpret_cast<const nl_f32x4*>(p);
                else {
#pragma unroll
                    for (int j = 0; j < 4; j++) if (n + j < N) v[h][j] += p[j];
                }
            }
        }
    nl_epilogue_pair(ep, v[0], v[1], m0, n0, M, N, 0);
}

// ---------------------------------------------------------------------------------------------
// k_linear_dz: dz = gy act'(z) for the two products of the backward pass, and the sums of dz over a chunk of rows for the bias (unrounded).
// A workgroup: 256 columns (four to a thread) x rows_per_chunk rows, four rows at a time.
// ---------------------------------------------------------------------------------------------
struct NlDz {
    const void* gy; const void* z; const unsigned* bits; const unsigned char* z8; const unsigned char* z8e;
    void* dz; float* part;
    long long M, ldgy, ldz, ldbits, ldz8, ldz8e, lddz, rows_per_chunk;
    int N, dt, act;
};
__global__ __launch_bounds__(256) void k_linear_dz(NlDz a)
{
    __shared__ nl_f32x4 s_sum[256];
    const int n = blockIdx.x * 256 + 4 * (threadIdx.x & 63), grp = threadIdx.x >> 6;
    const long long m1 = (blockIdx.y + 1) * a.rows_per_chunk < a.M ? (blockIdx.y + 1) * a.rows_per_chunk : a.M;
    const bool vec = n + 3 < a.N && (a.ldgy & 3) == 0 && ((uintptr_t)a.gy & (a.dt == NL_DT_F32 ? 15 : 7)) == 0 && (!a.z || (a.ldz & 3) == 0);
    nl_f32x4 sum = {};
    if (n < a.N)
        for (long long m = blockIdx.y * a.rows_per_chunk + grp; m < m1; m += 4) {
            nl_f32x4 g = {}, z = {};
            if (vec) {
                g = nl_load4(a.gy, m * a.ldgy + n, a.dt);
                if (a.z) z = nl_load4(a.z, m * a.ldz + n, a.dt);
            } else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (n + j < a.N) {
                        g[j] = nl_load_elem(a.gy, m * a.ldgy + n + j, a.dt);
                        if (a.z) z[j] = nl_load_elem(a.z, m * a.ldz + n + j, a.dt);
                    }
            if (a.z8) {
                z = nl_mx_decode4(*reinterpret_cast<const unsigned*>(a.z8 + m * a.ldz8 + n), nl_mx_scale(a.z8e[m * a.ldz8e + (n >> 5)]), nl_dtype_max(a.dt));
            }
            if (a.bits) {
                const unsigned w = a.bits[m * a.ldbits + (n >> 5)] >> (n & 31);
#pragma unroll
                for (int j = 0; j < 4; j++) g[j] = (w >> j & 1) ? g[j] : 0.0f;
            } else if (a.act != NL_ACT_NONE)
#pragma unroll
                for (int j = 0; j < 4; j++) g[j] *= nl_act_slope(z[j], a.act);
            sum += g;
            if (a.dz) nl_store4(a.dz, m * a.lddz + n, a.dt, g);                // (rows of dz are padded to eight elements)
        }
    if (!a.part) return;
    s_sum[threadIdx.x] = sum;
    __syncthreads();
    if (grp == 0 && n < a.N) {
        sum = (s_sum[threadIdx.x] + s_sum[threadIdx.x + 64]) + (s_sum[threadIdx.x + 128] + s_sum[threadIdx.x + 192]);
        float* o = a.part + (long long)blockIdx.y * a.N + n;
#pragma unroll
        for (int j = 0; j < 4; j++) if (n + j < a.N) o[j] = sum[j];
    }
}

// gb[n] = sum over the chunks: 32 columns x 8 runs of chunks per workgroup, joined in order
__global__ __launch_bounds__(256) void k_linear_gb(const float* __restrict__ part, int chunks, int N, void* gb, int dt)
{
    __shared__ float s_sum[256];
    const int n = blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5;
    const int per = (chunks + 7) / 8, c1 = (run + 1) * per < chunks ? (run + 1) * per : chunks;
    float s = 0.0f;
    if (n < N)
        for (int c = run * per; c < c1; c++) s += part[(long long)c * N + n];
    s_sum[threadIdx.x] = s;
    __syncthreads();
    if (run != 0 || n >= N) return;
    for (int r = 1; r < 8; r++) s += s_sum[threadIdx.x + 32 * r];
    nl_store_elem(gb, n, dt, s);
}

__global__ __launch_bounds__(256) void k_linear_zero(unsigned char* p, long long bytes)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (long long)gridDim.x * 256) p[i] = 0;
}

// ---------------------------------------------------------------------------------------------
// host: plans and launches
// ---------------------------------------------------------------------------------------------
#define NL_LINEAR_MAX_WIDTH (1 << 22)
#define NL_LINEAR_MAX_ROWS (1LL << 36)

// one product [M,N] over K: how it is cut
struct NlProduct { int splits; long long kchunk, part_bytes; };
static NlProduct nl_plan_product(long long M, long long N, long long K)
{
    const long long tiles = nl_up(M, ANY_T) / ANY_T * (nl_up(N, ANY_T) / ANY_T);
    long long s = 1;
    while (s < 64 && tiles * s < 512 && K / (2 * s) >= 4 * ANY_K) s *= 2;
    NlProduct p;
    p.kchunk = nl_up((K + s - 1) / s, ANY_K);
    p.splits = (int)((K + p.kchunk - 1) / p.kchunk);
    p.part_bytes = p.splits > 1 ? nl_up(4LL * p.splits * M * N, 256) : 0;
    return p;
}

static int nl_launch_product(const NlOperand& A, const NlOperand& B, long long M, long long N, long long K, NlEpilogue ep, char* ws, hipStream_t st)
{
    const NlProduct p = nl_plan_product(M, N, K);
    const long long tn = nl_up(N, ANY_T) / ANY_T, tiles = nl_up(M, ANY_T) / ANY_T * tn;
    if (tiles > 0x7FFFFFFF) return NL_ERR_INVALID_ARG;
    NlEpilogue e = ep;
    if (p.splits > 1) { e = NlEpilogue{}; e.part = (float*)ws; }
    const dim3 grid((unsigned)tiles, (unsigned)p.splits);
    if (ep.dt == NL_DT_F32) hipLaunchKernelGGL((k_linear_any<__bf16, 3>), grid, dim3(256), 0, st, A, B, M, (int)N, K, (int)tn, p.kchunk, e);
    else if (ep.dt == NL_DT_BF16) hipLaunchKernelGGL((k_linear_any<__bf16, 1>), grid, dim3(256), 0, st, A, B, M, (int)N, K, (int)tn, p.kchunk, e);
    else hipLaunchKernelGGL((k_linear_any<_Float16, 1>), grid, dim3(256), 0, st, A, B, M, (int)N, K, (int)tn, p.kchunk, e);
    if (p.splits > 1) {
        const long long jn = nl_up(N, 32) / 32, jt = nl_up(nl_up(M, 16) / 16 * jn, 4) / 4;
        if (jt > 0x7FFFFFFF) return NL_ERR_INVALID_ARG;
        hipLaunchKernelGGL(k_linear_join, dim3((unsigned)jt), dim3(256), 0, st, (const float*)ws, p.splits, M, (int)N, (int)jn, ep);
    }
    NL_LAUNCH_CHECK();
    return NL_OK;
}

struct NlDzPlan { int colblocks, chunks; long long rows, part_bytes, lddz, dz_bytes; };
static NlDzPlan nl_plan_dz(const NlLinear* d)
{
    NlDzPlan p;
    p.colblocks = (d->N + 255) / 256;
    long long want = 1024 / p.colblocks, most = nl_up(d->M, 16) / 16;
    if (want < 1) want = 1;
    if (want > most) want = most;
    p.rows = nl_up((d->M + want - 1) / (want > 0 ? want : 1), 4);
    p.chunks = (int)((d->M + p.rows - 1) / p.rows);
    p.part_bytes = d->gb ? nl_up(4LL * p.chunks * d->N, 256) : 0;
    p.lddz = nl_up(d->N, 8);
    p.dz_bytes = d->act != NL_ACT_NONE && (d->gx || d->gw) ? nl_up(d->M * p.lddz * nl_dtype_size(d->dtype), 256) : 0;
    return p;
}

static int nl_linear_check(const NlLinear* d, int backward)
{
    if (!d || d->struct_size != (int)sizeof(NlLinear) || !nl_dtype_ok(d->dtype) || d->act < NL_ACT_NONE || d->act > NL_ACT_SILU) return NL_ERR_INVALID_ARG;
    if (d->M < 0 || d->M > NL_LINEAR_MAX_ROWS || d->K < 1 || d->N < 1 || d->K > NL_LINEAR_MAX_WIDTH || d->N > NL_LINEAR_MAX_WIDTH) return NL_ERR_INVALID_ARG;
    const uintptr_t mis = nl_dtype_size(d->dtype) - 1;
    const void* const el[] = {d->x, d->w, d->b, d->r, d->y, d->z, d->gy, d->gx, d->gw, d->gb};
    for (const void* p : el) if ((uintptr_t)p & mis) return NL_ERR_INVALID_ARG;
    if (d->M == 0) return NL_OK;                                  // (tensors without elements have no address)
    if (((uintptr_t)d->z & 15) || ((uintptr_t)d->bits & 3) || ((uintptr_t)d->z8 & 15) || ((uintptr_t)d->x8 & 15)) return NL_ERR_INVALID_ARG;
    if (!backward) {
        if (!d->x || !d->w || !d->y || d->ldx < d->K || d->ldw < d->K || d->ldy < d->N || (d->r && d->ldr < d->N)) return NL_ERR_INVALID_ARG;
        if ((!d->z8) != (!d->z8e)) return NL_ERR_INVALID_ARG;
        return NL_OK;
    }
    if (!d->gy || d->ldgy < d->N) return NL_ERR_INVALID_ARG;
    if (d->gx && (!d->w || d->ldw < d->K)) return NL_ERR_INVALID_ARG;
    if (d->gw && (d->x8 ? !d->x8e : (!d->x || d->ldx < d->K))) return NL_ERR_INVALID_ARG;
    if (d->act == NL_ACT_RELU ? !d->bits : d->act != NL_ACT_NONE && (d->z8 ? !d->z8e : !d->z)) return NL_ERR_INVALID_ARG;
    return NL_OK;
}

extern "C" {

long long nl_linear_workspace(const NlLinear* d, int backward)
{
    if (nl_linear_check(d, backward) != NL_OK) return -1;
    if (d->M == 0) return 0;
    if (!backward) return nl_plan_product(d->M, d->N, d->K).part_bytes;
    const NlDzPlan z = nl_plan_dz(d);
    const long long a = d->gx ? nl_plan_product(d->M, d->K, d->N).part_bytes : 0, b = d->gw ? nl_plan_product(d->N, d->K, d->M).part_bytes : 0;
    return z.part_bytes + z.dz_bytes + (a > b ? a : b);
}

int nl_linear_forward(const NlLinear* d, void* stream)
{
    if (nl_linear_check(d, 0) != NL_OK) return NL_ERR_INVALID_ARG;
    if (d->M == 0) return NL_OK;
    const long long need = nl_linear_workspace(d, 0);
    if (need > 0 && (!d->ws || d->ws_bytes < need || ((uintptr_t)d->ws & 255))) return NL_ERR_INVALID_ARG;
    NlEpilogue ep = {};
    ep.b = d->b; ep.r = d->r; ep.ldr = d->ldr; ep.y = d->y; ep.ldy = d->ldy; ep.dt = d->dtype; ep.act = d->act;
    ep.z = d->z; ep.ldz = d->N;
    ep.bits = d->bits; ep.ldbits = nl_up(d->N, 32) / 32;
    ep.z8 = d->z8; ep.z8e = d->z8e; ep.ldz8 = nl_up(d->N, 32); ep.ldz8e = ep.ldz8 / 32;
    const NlOperand A = {d->x, nullptr, d->ldx, 1, 0, d->dtype}, B = {d->w, nullptr, d->ldw, 1, 0, d->dtype};
    return nl_launch_product(A, B, d->M, d->N, d->K, ep, (char*)d->ws, (hipStream_t)stream);
}

int nl_linear_backward(const NlLinear* d, void* stream)
{
    if (nl_linear_check(d, 1) != NL_OK) return NL_ERR_INVALID_ARG;
    hipStream_t st = (hipStream_t)stream;
    const int es = nl_dtype_size(d->dtype);
    if (d->M == 0) {
        if (d->gw) hipLaunchKernelGGL(k_linear_zero, dim3(256), dim3(256), 0, st, (unsigned char*)d->gw, (long long)d->N * d->K * es);
        if (d->gb) hipLaunchKernelGGL(k_linear_zero, dim3(4), dim3(256), 0, st, (unsigned char*)d->gb, (long long)d->N * es);
        NL_LAUNCH_CHECK();
        return NL_OK;
    }
    const long long need = nl_linear_workspace(d, 1);
    if (need > 0 && (!d->ws || d->ws_bytes < need || ((uintptr_t)d->ws & 255))) return NL_ERR_INVALID_ARG;
    const NlDzPlan zp = nl_plan_dz(d);
    char* ws = (char*)d->ws;
    const void* dz = d->gy;
    long long lddz = d->ldgy;
    if (zp.dz_bytes || zp.part_bytes) {
        NlDz a = {};
        a.gy = d->gy; a.ldgy = d->ldgy; a.M = d->M; a.N = d->N; a.dt = d->dtype; a.act = d->act; a.rows_per_chunk = zp.rows;
        if (d->act == NL_ACT_RELU) { a.bits = d->bits; a.ldbits = nl_up(d->N, 32) / 32; }
        else if (d->act != NL_ACT_NONE && d->z8) { a.z8 = d->z8; a.z8e = d->z8e; a.ldz8 = nl_up(d->N, 32); a.ldz8e = a.ldz8 / 32; }
        else if (d->act != NL_ACT_NONE) { a.z = d->z; a.ldz = d->N; }
        a.part = zp.part_bytes ? (float*)ws : nullptr;
        if (zp.dz_bytes) { a.dz = ws + zp.part_bytes; a.lddz = zp.lddz; dz = a.dz; lddz = zp.lddz; }
        hipLaunchKernelGGL(k_linear_dz, dim3(zp.colblocks, zp.chunks), dim3(256), 0, st, a);
        if (d->gb) hipLaunchKernelGGL(k_linear_gb, dim3((d->N + 31) / 32), dim3(256), 0, st, a.part, zp.chunks, d->N, d->gb, d->dtype);
        NL_LAUNCH_CHECK();
    }
    ws += zp.part_bytes + zp.dz_bytes;
    NlEpilogue ep = {};
    ep.dt = d->dtype; ep.act = NL_ACT_NONE; ep.ldy = d->K;
    if (d->gx) {
        ep.y = d->gx;
        const NlOperand A = {dz, nullptr, lddz, 1, 0, d->dtype}, B = {d->w, nullptr, 1, d->ldw, 0, d->dtype};
        const int rc = nl_launch_product(A, B, d->M, d->K, d->N, ep, ws, st);
        if (rc != NL_OK) return rc;
    }
    if (d->gw) {
        ep.y = d->gw;
        const NlOperand A = {dz, nullptr, 1, lddz, 0, d->dtype};
        const NlOperand B = d->x8 ? NlOperand{d->x8, d->x8e, 1, nl_up(d->K, 32), nl_up(d->K, 32) / 32, NL_DT_MX8} : NlOperand{d->x, nullptr, 1, d->ldx, 0, d->dtype};
        return nl_launch_product(A, B, d->N, d->K, d->M, ep, ws, st);
    }
    return NL_OK;
}

}  // extern "C"

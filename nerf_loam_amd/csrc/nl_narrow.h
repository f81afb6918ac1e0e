// nl_narrow.h -- products of many rows with a weight of at most 256 x 256 in 16 bits (a decoder's layers over a scan's samples): C[m,n] = sum_k A(m,k) B(n,k).
//
// Such a product moves its rows and little else.  As tiles every workgroup fetches its rows, multiplies for a moment and stores, one after the other; here a workgroup
// keeps the weight in registers (a wave 16 columns of it), stays, and streams rows of A through LDS, 32 at a time: tiles are on their way while one multiplies and the one
// before it leaves.  The data gradient makes dz = gy act'(z) of a tile in LDS on its way, writes it out for the weight gradient and sums it for
// the bias: no pass over gy and z of its own.
// Bound by memory: 200000 x 256 -> 256 bf16 with residual and relu 313 MB in 75 us (4.2 TB/s; as tiles of 128 99), with the codes of x 365 MB in 95 (107); data gradient
// 205 MB in 43 us (4.7 TB/s; 57), with dz and the bias sums 312 MB in 75 (95 in two passes); a large copy reaches 5.1 TB/s.
#pragma once
#include "nl_gemm.h"

// dz: how the rows of A (of gy, b_slow) become gy act'(z).  0: they are multiplied as they are; 1: z > 0 in bits; 2: z in the type; 3: z in 8-bit codes.  With 0 the results have more than 128 columns
#define NL_NARROW_ROWS 32
void nl_narrow_bf16(const NlGemm& g, const NlDz& z, int act, bool b_slow, int dz, unsigned grid, hipStream_t st);
void nl_narrow_f16(const NlGemm& g, const NlDz& z, int act, bool b_slow, int dz, unsigned grid, hipStream_t st);

#ifdef __HIPCC__
// A workgroup of 16 waves, one to a compute unit.  Iteration i, one barrier each: tile i + 1 becomes dz in LDS, the results of tile i - 1 leave, the loads of tile i + 3
// begin, tile i is multiplied into the exchange.  KS: 32 contraction indices each, NW: columns, 16 to a wave.
template <class T, int KS, int NW, bool B_SLOW, bool ENC, int DZ>
__global__ __launch_bounds__(1024) void k_narrow(NlGemm g, NlDz z, int act)
{
    constexpr int DT = __is_same(T, _Float16) ? NL_DT_F16 : NL_DT_BF16;
    constexpr int ROWS = NL_NARROW_ROWS, BUF = ROWS * KS * 64, CHUNKS = BUF / 16, WN = NW / 16, RW = ROWS * WN / 16, FM = RW / 16, EX = ROWS * NW * 4;
    static_assert(CHUNKS <= 1024 && EX / 32 <= 1024 && FM >= 1, "a thread has at most one chunk of a tile and eight results");
    typedef GemmSide<false, ROWS, 256> Quarter;                       // 64 contraction indices of a tile
    __shared__ __align__(256) char s_buf[4 * BUF];
    __shared__ __align__(256) char s_ex[2 * EX];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wm = (wave / WN) * RW, wn = (wave % WN) * 16;
    const int tiles = (int)((g.M + ROWS - 1) / ROWS), G = (int)gridDim.x;

    // ---- the weight: 16 columns, 32 KS contraction indices a wave ----
    nl_s16x8 w[KS];
    if constexpr (B_SLOW) {
        typedef GemmSide<true, NW, NW * 4, 32> SB;                    // 16 bytes a thread
        constexpr int SLOTS = 4 * BUF / SB::BYTES < KS ? 4 * BUF / SB::BYTES : KS;
        SB b;
        b.init(g.B, g.ldb, 0, g.N, 0, g.K);
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += SLOTS) {
            if (t < NW * 4)
#pragma unroll
                for (int k = k0; k < KS && k < k0 + SLOTS; k++) b.load(s_buf + (k - k0) * SB::BYTES, k * b.step, g.K - 32 * k);
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
            for (int k = k0; k < KS && k < k0 + SLOTS; k++) w[k] = SB::frag(s_buf + (k - k0) * SB::BYTES, wn, 0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
    } else {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)g.B, 0, (int)GEMM_RANGE, 0x00020000);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int n = wn + (lane & 15), c = 32 * k + 8 * (lane >> 4);
            w[k] = __builtin_bit_cast(nl_s16x8, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(n < g.N && c < g.K ? (unsigned)(n * g.ldb + 2 * c) : GEMM_OUT_OF_RANGE), 0, 0));
        }
    }

    // ---- the rows: a thread's chunk of eight elements; in LDS a quarter is GemmSide's [32][64] ----
    const int row = (t >> 3) & 31, c8 = (t & 7) ^ (row & 7), kc = (t >> 8) * 64 + 8 * c8;
    const bool mine = t < CHUNKS && kc < g.K;
    auto load = [&](int tile, int buf) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(g.A + (long long)tile * ROWS * g.lda), 0, (int)GEMM_RANGE, 0x00020000);
        if (wave < CHUNKS / 64)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(s_buf + buf * BUF + wave * 1024), 16,
                                                     (int)(mine && (long long)tile * ROWS + row < g.M ? (unsigned)(row * g.lda + 2 * kc) : GEMM_OUT_OF_RANGE), 0, 0, 0);
    };
    nl_i32x4 zr = {};
    unsigned ze = 0;
    float sum[8] = {};
    auto z_fetch = [&](int tile) {                                    // what a later tile's dz needs of z
        const long long m = (long long)tile * ROWS + row;
        if (!mine || m >= g.M) return;
        if (DZ == 1) zr[0] = (int)z.bits[m * z.ldbits + (kc >> 5)];
        if (DZ == 2) zr = *reinterpret_cast<const nl_i32x4*>((const unsigned short*)z.z + m * z.ldz + kc);
        if (DZ == 3) {
            const nl_i32x2 c = *reinterpret_cast<const nl_i32x2*>(z.z8 + m * z.ldz8 + kc);
            zr[0] = c[0]; zr[1] = c[1];
            ze = z.z8e[m * z.ldz8e + (kc >> 5)];
        }
    };
    auto make_dz = [&](int tile, int buf) {                           // gy -> dz where it lies, to memory, and into the bias sums (unrounded)
        const long long m = (long long)tile * ROWS + row;
        if (!mine || m >= g.M) return;
        nl_i32x4* const at = reinterpret_cast<nl_i32x4*>(s_buf + buf * BUF + t * 16);
        float v[8];
        nl_unraw8<DT>(v, NlRaw8<DT>{{*at}});
        if (DZ == 1) {
            const unsigned on = (unsigned)zr[0] >> (kc & 31);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (on >> j & 1) ? v[j] : 0.0f;
        } else {
            float y[8];
            if (DZ == 2) nl_unraw8<DT>(y, NlRaw8<DT>{{zr}});
            else {
                const float s = nl_mx_scale((unsigned char)ze);
                const nl_f32x4 p = nl_mx_decode4((unsigned)zr[0], s, nl_dtype_max(DT)), q = nl_mx_decode4((unsigned)zr[1], s, nl_dtype_max(DT));
#pragma unroll
                for (int j = 0; j < 4; j++) { y[j] = p[j]; y[4 + j] = q[j]; }
            }
            if (act == NL_ACT_GELU) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] *= nl_act_slope(y[j], NL_ACT_GELU);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] *= nl_act_slope(y[j], NL_ACT_SILU);
            }
        }
        nl_s16x8 u;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            sum[j] += v[j];
            u[j] = (short)(DT == NL_DT_BF16 ? nl_f2bf(v[j]) : nl_f2h(v[j]));
        }
        *at = __builtin_bit_cast(nl_i32x4, u);
        if (z.dz) *reinterpret_cast<nl_s16x8*>((unsigned short*)z.dz + m * z.pitch + kc) = u;
    };

    auto encode = [&](int tile, const char* a) {                      // the tile in 8-bit codes, as k_mx8_encode: four neighbouring threads have a block of 32
        const long long m = (long long)tile * ROWS + row;
        if (t >= CHUNKS) return;                                      // (whole waves)
        typedef __attribute__((__vector_size__(4))) unsigned short U2;
        const nl_i32x4 raw = *reinterpret_cast<const nl_i32x4*>(a + t * 16);
        // magnitudes of 16-bit patterns have the patterns' order
        U2 two = __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(U2, raw[0] & 0x7FFF7FFF), __builtin_bit_cast(U2, raw[1] & 0x7FFF7FFF)),
                                           __builtin_elementwise_max(__builtin_bit_cast(U2, raw[2] & 0x7FFF7FFF), __builtin_bit_cast(U2, raw[3] & 0x7FFF7FFF)));
        unsigned top = max((unsigned)two[0], (unsigned)two[1]);
        top = max(top, (unsigned)__shfl_xor((int)top, 1));
        top = max(top, (unsigned)__shfl_xor((int)top, 2));
        float v[8], amax = DT == NL_DT_BF16 ? nl_bf2f((unsigned short)top) : nl_h2f((unsigned short)top);
        nl_unraw8<DT>(v, NlRaw8<DT>{{raw}});
        const bool finite = amax < INFINITY;
        if (!finite) {                                                // (all four threads)
            amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) amax = fmaxf(amax, nl_finite_abs(v[j]));
            amax = fmaxf(amax, __shfl_xor(amax, 1));
            amax = fmaxf(amax, __shfl_xor(amax, 2));
        }
        const int e = nl_mx_exponent(amax);
        const float s = nl_pow2(-e);
        if (m >= g.M || kc >= g.ld8) return;
        nl_i32x2 code;
        if (finite) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                code[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * s, v[4 * h + 1] * s, 0, false);
                code[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * s, v[4 * h + 3] * s, code[h], true);
            }
        } else code = nl_i32x2{(int)nl_mx_encode4(v[0], v[1], v[2], v[3], s), (int)nl_mx_encode4(v[4], v[5], v[6], v[7], s)};
        *reinterpret_cast<nl_i32x2*>(g.A8 + m * g.ld8 + kc) = code;
        if ((c8 & 3) == 0) g.A8e[m * (g.ld8 / 32) + (kc >> 5)] = (unsigned char)(e + 127);
    };

    // ---- the results: a thread's eight columns of one row ----
    const NlEpilogue& ep = g.ep;
    const int orow = t / (NW / 8), col = 8 * (t % (NW / 8));
    const bool leaves = t < EX / 32, whole = (g.N & 7) == 0;
    const bool residual = !B_SLOW && whole && ep.r;                   // (a data gradient is stored as it is)
    NlRaw8<DT> bias = {}, res = {};
    if (!B_SLOW && whole && ep.b && col < g.N) bias = nl_raw8<DT>(ep.b, col);
    auto results = [&](int tile, const char* ex) {
        const long long m = (long long)tile * ROWS + orow;
        const char* const from = ex + orow * (NW * 4);
        const nl_f32x4 p = *reinterpret_cast<const nl_f32x4*>(from + ((col / 4) ^ (orow & 15)) * 16);
        const nl_f32x4 q = *reinterpret_cast<const nl_f32x4*>(from + ((col / 4 + 1) ^ (orow & 15)) * 16);
        float v[8] = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
        if constexpr (B_SLOW) {
            if (m < g.M && col < g.N) nl_store8<DT>(ep.y, m * ep.ldy + col, v, g.N - col);
        } else if (whole) {
            float b[8], x[8];
            nl_unraw8<DT>(b, bias);
            nl_unraw8<DT>(x, res);
            nl_epilogue8<DT, false>(ep, v, b, x, m, col, g.M, g.N, 0);
        } else nl_epilogue8_fetch<DT>(ep, v, m, col, g.M, g.N, 0);
    };

    const int first = blockIdx.x;
    if (DZ) z_fetch(first);
    load(first, 0);
    load(first + G, 1);
    load(first + 2 * G, 2);
    if (DZ) {
        asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
        make_dz(first, 0);
        z_fetch(first + G);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    constexpr int ZS = DZ == 3 ? 2 : 1;                               // loads of z_fetch
    const bool fetches = __ballot(mine) != 0;
    for (int tile = first, i = 0;; tile += G, i++) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (DZ && tile + G < tiles) make_dz(tile + G, (i + 1) & 3);
        if (i > 0 && leaves) results(tile - G, s_ex + ((i - 1) & 1) * EX);
        if (tile >= tiles) break;
        const char* const a = s_buf + (i & 3) * BUF;
        if (ENC) encode(tile, a);
        if (DZ) z_fetch(tile + 2 * G);
        if (residual) {
            const long long m = (long long)tile * ROWS + orow;
            if (leaves && m < g.M && col < g.N) res = nl_raw8<DT>(ep.r, m * ep.ldr + col);
        }
        load(tile + 3 * G, (i + 3) & 3);
        nl_f32x4 acc[FM] = {};
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int f = 0; f < FM; f++) acc[f] = NlMma<T>::mma(w[k], Quarter::frag(a + (k >> 1) * Quarter::BYTES, wm + 16 * f, k & 1), acc[f]);
#pragma unroll
        for (int f = 0; f < FM; f++) {
            const int r = wm + 16 * f + (lane & 15), c = (wn / 4 + (lane >> 4)) ^ (r & 15);
            *reinterpret_cast<nl_f32x4*>(s_ex + (i & 1) * EX + r * (NW * 4) + c * 16) = acc[f];
        }
        // loads of tile i + 2 and all before them have landed; in flight stay at most tile i + 3's and what this iteration fetched beside it.  (A wave whose columns lie
        // behind the contraction fetches nothing of z; one without results no residual, and then waits for tile i + 1's at least, which is what it needs.)
        if (residual || (DZ && fetches)) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(DZ ? 1 + ZS : 2) : "memory");
        else asm volatile("s_waitcnt vmcnt(1)" ::: "memory");
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");       // (all loads, the ones of zeros behind the last tile too)
    if (DZ && z.part) {
        // a column's threads in the order of their rows
        float (*const s_sum)[KS * 32 + 1] = (float (*)[KS * 32 + 1])s_buf;
        if (t < CHUNKS)
#pragma unroll
            for (int j = 0; j < 8; j++) s_sum[row][kc + j] = sum[j];
        __syncthreads();
        if (t < g.K) {
            float s = 0.0f;
            for (int r = 0; r < ROWS; r++) s += s_sum[r][t];
            z.part[(long long)blockIdx.x * g.K + t] = s;
        }
    }
}

template <class T, int KS, int NW>
static void nl_narrow_sized(const NlGemm& g, const NlDz& z, int act, bool b_slow, int dz, unsigned grid, hipStream_t st)
{
    if (dz == 1) hipLaunchKernelGGL((k_narrow<T, KS, NW, true, false, 1>), dim3(grid), dim3(1024), 0, st, g, z, act);
    else if (dz == 2) hipLaunchKernelGGL((k_narrow<T, KS, NW, true, false, 2>), dim3(grid), dim3(1024), 0, st, g, z, act);
    else if (dz == 3) hipLaunchKernelGGL((k_narrow<T, KS, NW, true, false, 3>), dim3(grid), dim3(1024), 0, st, g, z, act);
    else if constexpr (NW == 256) {                                   // (without dz only wide results come here)
        if (b_slow) hipLaunchKernelGGL((k_narrow<T, KS, NW, true, false, 0>), dim3(grid), dim3(1024), 0, st, g, z, act);
        else if (g.A8) hipLaunchKernelGGL((k_narrow<T, KS, NW, false, true, 0>), dim3(grid), dim3(1024), 0, st, g, z, act);
        else hipLaunchKernelGGL((k_narrow<T, KS, NW, false, false, 0>), dim3(grid), dim3(1024), 0, st, g, z, act);
    }
}
template <class T>
static void nl_narrow_launch(const NlGemm& g, const NlDz& z, int act, bool b_slow, int dz, unsigned grid, hipStream_t st)
{
    if (g.K <= 128 && g.N <= 128) nl_narrow_sized<T, 4, 128>(g, z, act, b_slow, dz, grid, st);
    else if (g.K <= 128) nl_narrow_sized<T, 4, 256>(g, z, act, b_slow, dz, grid, st);
    else if (g.N <= 128) nl_narrow_sized<T, 8, 128>(g, z, act, b_slow, dz, grid, st);
    else nl_narrow_sized<T, 8, 256>(g, z, act, b_slow, dz, grid, st);
}
#endif

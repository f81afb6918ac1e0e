// nl_gemm.h -- the tiled 16-bit matrix product behind nl_linear_*: C[m,n] = sum_k A(m,k) B(n,k), fp32 sums, then the epilogue of nl_layers.h.
//
// An operand lies either with the contraction index fastest (rows of k: x, weights, dz of the forward / data-gradient products) or slowest (rows of m or n: both
// operands of the weight gradient, the weight of the data gradient).  Both go from global memory straight into LDS, 16 bytes a lane, without passing through
// registers; the second kind is transposed on the way out of LDS (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 elements and receive a column of 4 each), so
// no product needs a transposed copy of anything.
#pragma once
#include "nl_layers.h"

#define GEMM_BK 64                     // contraction step: two matrix instructions of 32

struct NlGemm {
    const char* A; const char* B;      // 16-byte aligned, rows 16-byte aligned
    long long lda, ldb;                // bytes between rows
    long long a_plane, b_plane;        // bytes between the planes of a split fp32 operand
    long long M, K;
    int N, tiles_m, tiles_n, split;    // fp32: split = 1, the six plane products follow each other along one contraction
    long long kchunk;                  // contraction indices per split, a multiple of GEMM_BK
    NlEpilogue ep;
};

// layout 0: both operands' rows run along k; 1: B's rows are k; 2: both operands' rows are k.  tile 0: 256 x 256, 1: 128 x 128, 2: 64 x 64.
void nl_gemm_bf16(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st);
void nl_gemm_f16(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st);
void nl_gemm_f32(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st);

#ifdef __HIPCC__
template <class T> struct NlMma;
template <> struct NlMma<__bf16> {
    static __device__ __forceinline__ nl_f32x4 mma(nl_s16x8 a, nl_s16x8 b, nl_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(nl_bf16x8, a), __builtin_bit_cast(nl_bf16x8, b), c, 0, 0, 0); }
};
template <> struct NlMma<_Float16> {
    static __device__ __forceinline__ nl_f32x4 mma(nl_s16x8 a, nl_s16x8 b, nl_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(nl_f16x8, a), __builtin_bit_cast(nl_f16x8, b), c, 0, 0, 0); }
};

#define GEMM_OUT_OF_RANGE 0x80000000u   // a buffer load from here returns zeros: beyond every tile's range (at most GEMM_RANGE bytes)
#define GEMM_RANGE 0x7FFFFFF0LL

// One operand of a workgroup: R rows or columns (of C) x GEMM_BK contraction indices per step, NT threads.
//   fast (k fastest):  LDS [R][64], 16-byte chunks of a row XORed with row & 7: the 16 rows of a fragment start in different banks
//   slow (k slowest):  LDS [64][R], pairs of chunks XORed with k & 3 and, where a row has 16 chunks, k >> 3 & 1: the rows that one transposing read touches lie
//                      in different banks
template <bool SLOW, int R, int NT>
struct GemmSide {
    static constexpr int BYTES = R * GEMM_BK * 2, LOADS = BYTES / (16 * NT), CH = R / 8;
    unsigned off[LOADS];               // byte offset of the thread's chunks from the tile's first byte; GEMM_OUT_OF_RANGE: outside the operand
    int kk[LOADS];                     // contraction index of the chunk inside a step
    const char* base; long long step, room;

    static __device__ __forceinline__ int swz(int k) { return CH >= 16 ? ((k & 3) | ((k >> 1) & 4)) : (k & 3); }

    // p: the operand, ld: bytes per row, i0: first row / column of the tile, I: how many there are, k0: first contraction index
    __device__ __forceinline__ void init(const char* p, long long ld, long long i0, long long I, long long k0, long long K)
    {
        const int t = threadIdx.x;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const int s = l * NT + t;
            if (SLOW) {
                const int k = s / CH, c = (s % CH) ^ (swz(k) << 1);
                kk[l] = k;
                off[l] = i0 + 8 * c < I ? (unsigned)(k * ld + 16 * c) : GEMM_OUT_OF_RANGE;
            } else {
                const int r = s >> 3, c = (s & 7) ^ (r & 7);
                kk[l] = 8 * c;
                off[l] = i0 + r < I ? (unsigned)(r * ld + 16 * c) : GEMM_OUT_OF_RANGE;
            }
        }
        base = SLOW ? p + k0 * ld + 2 * i0 : p + i0 * ld + 2 * k0;
        step = SLOW ? GEMM_BK * ld : GEMM_BK * 2;
    }
    // one step into LDS: kleft contraction indices are left (chunks behind them read zeros); adv: bytes from the first step's place
    __device__ __forceinline__ void load(char* lds, long long adv, long long kleft) const
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + adv), 0, (int)GEMM_RANGE, 0x00020000);
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const unsigned o = kleft >= GEMM_BK || kk[l] < kleft ? off[l] : GEMM_OUT_OF_RANGE;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + (l * NT + wave * 64) * 16), 16, (int)o, 0, 0, 0);
        }
    }
    // fragment of 16 rows / columns from i on, contraction indices 32 ks .. 32 ks + 31 of the step: lane l gets row i + (l & 15), indices 8 (l >> 4) + 0..7
    static __device__ __forceinline__ nl_s16x8 frag(const char* lds, int i, int ks)
    {
        const int l = threadIdx.x & 63;
        if (SLOW) {
            typedef __attribute__((address_space(3))) nl_s16x4* P;
            const int k = 8 * (l >> 4) + ((l & 15) >> 2);
            const int at = (k + 32 * ks) * (R * 2) + ((((i >> 4) ^ swz(k)) << 1) + ((l >> 1) & 1)) * 16 + (l & 1) * 8;
            const nl_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(nl_s16x4*)(lds + at));
            const nl_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(nl_s16x4*)(lds + at + 4 * R * 2));
            return nl_s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
        const int row = i + (l & 15), c = (4 * ks + (l >> 4)) ^ (l & 7);
        return *reinterpret_cast<const nl_s16x8*>(lds + row * (GEMM_BK * 2) + c * 16);
    }
};

template <class T, bool PLANES, bool A_SLOW, bool B_SLOW, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_gemm(NlGemm g)
{
    constexpr int DT = PLANES ? NL_DT_F32 : __is_same(T, _Float16) ? NL_DT_F16 : NL_DT_BF16;
    constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef GemmSide<A_SLOW, BM, NT> SA;
    typedef GemmSide<B_SLOW, BN, NT> SB;
    __shared__ __align__(256) char s_mem[2 * (SA::BYTES + SB::BYTES)];
    char* const s_a = s_mem;
    char* const s_b = s_mem + 2 * SA::BYTES;
    // workgroups go to the eight dies in turn: give each die neighbouring tiles, four tile rows at a time, so that its L2 holds what it shares
    const unsigned tiles = (unsigned)g.tiles_m * g.tiles_n, q = tiles >> 3, rem = tiles & 7, die = blockIdx.x & 7;
    unsigned pid = die * q + (die < rem ? die : rem) + (blockIdx.x >> 3);
    const unsigned per_group = 4u * g.tiles_n, grp = pid / per_group, first = 4 * grp, rows = min(4u, (unsigned)g.tiles_m - first);
    pid -= grp * per_group;
    const long long m0 = (long long)(first + pid % rows) * BM;
    const int n0 = (int)(pid / rows) * BN;
    const long long k0 = (long long)blockIdx.y * g.kchunk, k1 = min(k0 + g.kchunk, g.K);
    const int ksteps = (int)((k1 - k0 + GEMM_BK - 1) / GEMM_BK), steps = PLANES ? 6 * ksteps : ksteps;
    SA a; SB b;
    a.init(g.A, g.lda, m0, g.M, k0, g.K);
    b.init(g.B, g.ldb, n0, g.N, k0, g.K);
    const int wave = threadIdx.x >> 6, wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    nl_f32x4 acc[FM][FN] = {};
    auto fetch = [&](int s) {
        const int pair = PLANES ? s / ksteps : 0, k = PLANES ? s - pair * ksteps : s;
        // planes h, m, l = 0, 1, 2; the products by rising size: (l,h) (h,l) (m,m) (m,h) (h,m) (h,h)
        const int qa = PLANES ? (pair == 0 ? 2 : pair == 2 || pair == 3 ? 1 : 0) : 0, qb = PLANES ? (pair == 1 ? 2 : pair == 2 || pair == 4 ? 1 : 0) : 0;
        const long long left = k1 - k0 - (long long)k * GEMM_BK;
        a.load(s_a + (s & 1) * SA::BYTES, k * a.step + qa * g.a_plane, left);
        b.load(s_b + (s & 1) * SB::BYTES, k * b.step + qb * g.b_plane, left);
    };
    fetch(0);
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    for (int s = 0; s < steps; s++) {
        if (s + 1 < steps) fetch(s + 1);
        const char* la = s_a + (s & 1) * SA::BYTES;
        const char* lb = s_b + (s & 1) * SB::BYTES;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            nl_s16x8 fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; i++) fa[i] = SA::frag(la, wm + 16 * i, ks);
#pragma unroll
            for (int j = 0; j < FN; j++) fb[j] = SB::frag(lb, wn + 16 * j, ks);
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = NlMma<T>::mma(fb[j], fa[i], acc[i][j]);
        }
        __syncthreads();
    }
    // results: a wave passes its rows through its own part of LDS, RP at a time, and leaves with eight neighbouring columns in a lane (16-byte stores, and the
    // neighbours that bits and 8-bit blocks need).  16-byte chunks XORed with the row: neither side of the exchange has bank conflicts.
    constexpr int WC = BN / WN, RP = BM / WM < 64 ? BM / WM : 64, CX = WC / 4 - 1;
    static_assert((CX & (CX + 1)) == 0 && RP * WC * 4 * WM * WN <= 2 * (SA::BYTES + SB::BYTES), "the exchange fits into the operand buffers");
    char* const mine = s_mem + wave * (RP * WC * 4);
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int half = 0; half < BM / WM / RP; half++) {
#pragma unroll
        for (int i = 0; i < RP / 16; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) {
                const int r = 16 * i + (lane & 15), c = (4 * j + (lane >> 4)) ^ (r & CX);
                *reinterpret_cast<nl_f32x4*>(mine + r * (WC * 4) + c * 16) = acc[half * (RP / 16) + i][j];
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int t = lane; t < RP * WC / 8; t += 64) {
            const int r = t / (WC / 8), c = 2 * (t % (WC / 8));
            const nl_f32x4 p = *reinterpret_cast<const nl_f32x4*>(mine + r * (WC * 4) + (c ^ (r & CX)) * 16);
            const nl_f32x4 q = *reinterpret_cast<const nl_f32x4*>(mine + r * (WC * 4) + ((c + 1) ^ (r & CX)) * 16);
            float v[8] = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
            nl_epilogue8<DT>(g.ep, v, m0 + wm + half * RP + r, n0 + wn + 4 * c, g.M, g.N, (long long)blockIdx.y * g.M * g.N);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <class T, bool PLANES, bool A_SLOW, bool B_SLOW>
static void nl_gemm_tile(const NlGemm& g, int tile, dim3 grid, hipStream_t st)
{
    if (tile == 0) hipLaunchKernelGGL((k_gemm<T, PLANES, A_SLOW, B_SLOW, 256, 256, 2, 4>), grid, dim3(512), 0, st, g);
    else if (tile == 1) hipLaunchKernelGGL((k_gemm<T, PLANES, A_SLOW, B_SLOW, 128, 128, 2, 2>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_gemm<T, PLANES, A_SLOW, B_SLOW, 64, 64, 2, 2>), grid, dim3(256), 0, st, g);
}
template <class T, bool PLANES>
static void nl_gemm_layout(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st)
{
    if (layout == 0) nl_gemm_tile<T, PLANES, false, false>(g, tile, grid, st);
    else if (layout == 1) nl_gemm_tile<T, PLANES, false, true>(g, tile, grid, st);
    else nl_gemm_tile<T, PLANES, true, true>(g, tile, grid, st);
}
#endif

// nl_gemm.h -- the tiled 16-bit matrix product behind nl_linear_*: C[m,n] = sum_k A(m,k) B(n,k), fp32 sums, then the epilogue of nl_layers.h.
//
// An operand lies either with the contraction index fastest (rows of k: x, weights, dz of the forward / data-gradient products) or slowest (rows of m or n: both
// operands of the weight gradient, the weight of the data gradient).  Both go from global memory straight into LDS, 16 bytes a lane, without passing through
// registers; the second kind is transposed on the way out of LDS (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 elements and receive a column of 4 each), so
// no product needs a transposed copy of anything.
#pragma once
#include "nl_layers.h"

#define GEMM_BK 64                     // contraction step: two matrix instructions of 32
#define NL_GEMM_FEW_SQUARES 512        // workgroups of 64 x 64 with four buffers that run at a time (two to a compute unit)

struct NlGemm {
    const char* A; const char* B;      // 16-byte aligned, rows 16-byte aligned
    const unsigned char* Be;           // B in 8-bit codes: its powers of two, ldb / 32 bytes between rows
    unsigned char* A8; unsigned char* A8e;      // layout 4: where A's codes go, ld8 and ld8 / 32 bytes between rows
    long long ld8, plane;              // plane: bytes between the planes of a split B (0: B is fp32)
    long long lda, ldb;                // bytes between rows
    long long M, K;
    int N, tiles_m, tiles_n;
    long long kchunk;                  // contraction indices per split, a multiple of GEMM_BK
    NlEpilogue ep;
};

struct NlDz {                          // dz = gy act'(z): where gy and z are, where dz and the bias' partial sums go
    const void* gy; const void* z; const unsigned* bits; const unsigned char* z8; const unsigned char* z8e;
    void* dz; float* part;
    long long M, ldgy, ldz, ldbits, ldz8, ldz8e, pitch, rows_per_chunk;
    int N;
};

// layout 0: both operands' rows run along k; 1: B's rows are k; 2: both operands' rows are k; 3: the same with B in 8-bit codes;
// 4: layout 0, and A is written out in 8-bit codes (both for 16-bit types only).  tile 0: 256 x 256 (16 bits only), 1: 128 x 128, 2: 64 x 64.
void nl_gemm_bf16(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st);
void nl_gemm_f16(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st);
void nl_gemm_f32(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st);
void nl_gemm_f32_to16(const NlGemm& g, int dt, int layout, dim3 grid, hipStream_t st);      // A fp32, B and the result of dt; layouts 1 and 2, squares of 64

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

// One operand of a workgroup: R rows or columns (of C) x BK contraction indices per step, NT threads.
//   fast (k fastest):  LDS [R][BK], 16-byte chunks of a row XORed with row & 7 (BK 32: row >> 1 & 3): eight rows of a fragment cover all banks
//   slow (k slowest):  LDS [BK][R], pairs of chunks XORed with k & 3 and, where a row has 16 chunks, k >> 3 & 1: the rows that one transposing read touches lie
//                      in different banks
template <bool SLOW, int R, int NT, int BK = GEMM_BK>
struct GemmSide {
    static constexpr int BYTES = R * BK * 2, LOADS = BYTES / (16 * NT), CH = R / 8;
    unsigned off[LOADS];               // byte offset of the thread's chunks from the tile's first byte; GEMM_OUT_OF_RANGE: outside the operand
    int kk[LOADS];                     // contraction index of the chunk inside a step
    const char* base; long long step, room;

    static __device__ __forceinline__ int swz(int k) { return CH >= 16 ? ((k & 3) | ((k >> 1) & 4)) : (k & 3); }
    static __device__ __forceinline__ int swz_row(int r) { return BK == 64 ? r & 7 : (r >> 1) & 3; }

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
                const int r = s / (BK / 8), c = (s % (BK / 8)) ^ swz_row(r);
                kk[l] = 8 * c;
                off[l] = i0 + r < I ? (unsigned)(r * ld + 16 * c) : GEMM_OUT_OF_RANGE;
            }
        }
        base = SLOW ? p + k0 * ld + 2 * i0 : p + i0 * ld + 2 * k0;
        step = SLOW ? BK * ld : BK * 2;
    }
    // one step into LDS: kleft contraction indices are left (chunks behind them read zeros); adv: bytes from the first step's place
    __device__ __forceinline__ void load(char* lds, long long adv, long long kleft) const
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + adv), 0, (int)GEMM_RANGE, 0x00020000);
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int l = 0; l < LOADS; l++) {
            const unsigned o = kleft >= BK || kk[l] < kleft ? off[l] : GEMM_OUT_OF_RANGE;
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
        const int row = i + (l & 15), c = (4 * ks + (l >> 4)) ^ swz_row(l & 15);
        return *reinterpret_cast<const nl_s16x8*>(lds + row * (BK * 2) + c * 16);
    }
};

// Workgroups go to the eight dies in turn: give each die neighbouring work - the tiles of one piece of the contraction, four tile rows at a time - so that its L2 holds
// what it shares (256 x 256 over 200000 in 64 pieces, squares of 64, pieces dealt out across dies: 114 us).  -> the piece
template <int BM, int BN> __device__ __forceinline__ unsigned gemm_tile_of(const NlGemm& g, long long& m0, int& n0)
{
    const unsigned tiles = (unsigned)g.tiles_m * g.tiles_n, total = tiles * gridDim.y, id = blockIdx.y * tiles + blockIdx.x;
    const unsigned q = total >> 3, rem = total & 7, die = id & 7, at = die * q + (die < rem ? die : rem) + (id >> 3);
    const unsigned piece = at / tiles;
    unsigned pid = at - piece * tiles;
    const unsigned per_group = 4u * g.tiles_n, grp = pid / per_group, first = 4 * grp, rows = min(4u, (unsigned)g.tiles_m - first);
    pid -= grp * per_group;
    m0 = (long long)(first + pid % rows) * BM;
    n0 = (int)(pid / rows) * BN;
    return piece;
}

// Results of a wave, WR rows x WC columns from (m, n) on: it passes them through its own part of LDS, RP rows at a time, and leaves with eight neighbouring columns
// in a lane (16-byte stores, and the neighbours that bits and 8-bit blocks need).  16-byte chunks XORed with the row: neither side of the exchange has bank conflicts.
template <int DT, int WR, int WC, int WAVES, int LDS>
__device__ __forceinline__ void gemm_results(const NlGemm& g, nl_f32x4 (&acc)[WR / 16][WC / 16], char* s_mem, long long m, int n, unsigned piece)
{
    constexpr int RP = WR < 64 ? WR : (WAVES * 64 * WC * 4 > LDS ? 32 : 64), CX = WC / 4 - 1;
    static_assert((CX & (CX + 1)) == 0 && RP * WC * 4 * WAVES <= LDS, "the exchange fits into the operand buffers");
    constexpr int TURNS = RP * WC / 512, BATCH = TURNS < 4 ? TURNS : 4;
    static_assert(64 % (WC / 8) == 0 && TURNS % BATCH == 0, "a lane keeps its columns");
    const NlEpilogue& ep = g.ep;
    const int lane = threadIdx.x & 63, col = n + 8 * (lane % (WC / 8));
    char* const mine = s_mem + (threadIdx.x >> 6) * (RP * WC * 4);
    const bool inside = m + WR <= g.M && n + WC <= g.N;
    float bias[8] = {};
    if (inside && !ep.part && ep.b) nl_unraw8<DT>(bias, nl_raw8<DT>(ep.b, col));
#pragma unroll
    for (int half = 0; half < WR / RP; half++) {
#pragma unroll
        for (int i = 0; i < RP / 16; i++)
#pragma unroll
            for (int j = 0; j < WC / 16; j++) {
                const int r = 16 * i + (lane & 15), c = (4 * j + (lane >> 4)) ^ (r & CX);
                *reinterpret_cast<nl_f32x4*>(mine + r * (WC * 4) + c * 16) = acc[half * (RP / 16) + i][j];
            }
        __builtin_amdgcn_wave_barrier();
        auto value = [&](int t, float* v) {
            const int r = t / (WC / 8), c = 2 * (t % (WC / 8));
            const nl_f32x4 p = *reinterpret_cast<const nl_f32x4*>(mine + r * (WC * 4) + (c ^ (r & CX)) * 16);
            const nl_f32x4 q = *reinterpret_cast<const nl_f32x4*>(mine + r * (WC * 4) + ((c + 1) ^ (r & CX)) * 16);
#pragma unroll
            for (int j = 0; j < 4; j++) { v[j] = p[j]; v[4 + j] = q[j]; }
        };
        const long long off = (long long)piece * g.M * g.N;
        if (inside) {
            // four rows of residuals in flight: one load and its use at a time leaves a memory latency per row (200000 x 256 x 256 with residual: 137 us)
#pragma unroll 1
            for (int t0 = lane; t0 < RP * WC / 8; t0 += 64 * BATCH) {
                NlRaw8<DT> raw[BATCH];
                if (ep.r) {
#pragma unroll
                    for (int u = 0; u < BATCH; u++) raw[u] = nl_raw8<DT>(ep.r, (m + half * RP + (t0 + 64 * u) / (WC / 8)) * ep.ldr + col);
                }
#pragma unroll
                for (int u = 0; u < BATCH; u++) {
                    float v[8], r[8];
                    value(t0 + 64 * u, v);
                    if (ep.r) nl_unraw8<DT>(r, raw[u]);
                    nl_epilogue8<DT, true>(ep, v, bias, r, m + half * RP + (t0 + 64 * u) / (WC / 8), col, g.M, g.N, off);
                }
            }
        } else {
#pragma unroll 1
            for (int t = lane; t < RP * WC / 8; t += 64) {
                float v[8];
                value(t, v);
                nl_epilogue8_fetch<DT>(ep, v, m + half * RP + t / (WC / 8), col, g.M, g.N, off);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// An operand in 8-bit codes whose rows are the contraction: R columns x 64 indices per step.  A thread fetches 16 neighbouring codes and their power of two while the
// step before multiplies, decodes them (exactly: four significant bits) and writes them where GemmSide would have put the 16-bit elements
// (half the bytes: 256 x 256 over 200000 52 us).
template <class T, int R, int NT>
struct GemmSideMx8 {
    typedef GemmSide<true, R, NT> Plane;
    static constexpr int BYTES = Plane::BYTES, UNITS = R * GEMM_BK / (16 * NT), CH = R / 16;
    unsigned off[UNITS], eoff[UNITS]; int kk[UNITS], lds[UNITS];
    nl_i32x4 v[UNITS]; unsigned char e[UNITS];
    const char* base; const unsigned char* ebase; long long step;

    __device__ __forceinline__ void init(const char* p, const unsigned char* pe, long long ld, long long i0, long long I, long long k0)
    {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int s = u * NT + threadIdx.x, k = s / CH, c = s % CH;
            const bool in = i0 + 16 * c < I;                          // (rows of codes are whole blocks of 32)
            kk[u] = k;
            off[u] = in ? (unsigned)(k * ld + 16 * c) : GEMM_OUT_OF_RANGE;
            eoff[u] = in ? (unsigned)(k * (ld / 32) + c / 2) : GEMM_OUT_OF_RANGE;
            lds[u] = k * (R * 2) + ((2 * c) ^ (Plane::swz(k) << 1)) * 16;
        }
        base = p + k0 * ld + i0; ebase = pe + k0 * (ld / 32) + i0 / 32;
        step = GEMM_BK * ld;
    }
    __device__ __forceinline__ void fetch(int s, long long kleft)
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + s * step), 0, (int)GEMM_RANGE, 0x00020000);
        const __amdgpu_buffer_rsrc_t re = __builtin_amdgcn_make_buffer_rsrc((void*)(ebase + s * (step / 32)), 0, (int)GEMM_RANGE, 0x00020000);
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const bool in = kleft >= GEMM_BK || kk[u] < kleft;
            v[u] = __builtin_bit_cast(nl_i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(in ? off[u] : GEMM_OUT_OF_RANGE), 0, 0));
            e[u] = __builtin_amdgcn_raw_buffer_load_b8(re, (int)(in ? eoff[u] : GEMM_OUT_OF_RANGE), 0, 0);
        }
    }
    __device__ __forceinline__ void put(char* mem) const
    {
        constexpr bool F16 = __is_same(T, _Float16);
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const float s = nl_mx_scale(e[u]);
            nl_i32x4 o[2];
            if (e[u] < (F16 ? 127 + 8 : 127 + 120)) {                 // 448 2^e is inside the type
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int h = 0; h < 2; h++) o[j >> 1][2 * (j & 1) + h] = F16 ? __builtin_bit_cast(int, h ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[u][j], s, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[u][j], s, false))
                                                                                 : __builtin_bit_cast(int, h ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[u][j], s, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[u][j], s, false));
            } else
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const nl_f32x4 f = nl_mx_decode4((unsigned)v[u][j], s, nl_dtype_max(F16 ? NL_DT_F16 : NL_DT_BF16));
#pragma unroll
                    for (int h = 0; h < 2; h++) o[j >> 1][2 * (j & 1) + h] = (int)(F16 ? (unsigned)nl_f2h(f[2 * h]) | (unsigned)nl_f2h(f[2 * h + 1]) << 16 : (unsigned)nl_f2bf(f[2 * h]) | (unsigned)nl_f2bf(f[2 * h + 1]) << 16);
                }
            *reinterpret_cast<nl_i32x4*>(mem + lds[u]) = o[0];
            *reinterpret_cast<nl_i32x4*>(mem + lds[u] + 16) = o[1];
        }
    }
};

// A step's rows of A in 8-bit codes, from LDS (GemmSide's fast layout): a thread takes a block of 32.  With a value that is not finite in the block every element is asked
// (nl_mx_encode4 as in k_mx8_encode: the same codes); otherwise the largest magnitude is found among the 16-bit patterns, whose order is that of the magnitudes.
// 200000 x 256: the product takes 14 us more, a pass of its own over x 30; 32768 x 2048: 16 and 41.
template <class T>
__device__ __forceinline__ void gemm_encode_block(const NlGemm& g, const char* lds, int row, int half, long long m, long long k)      // half: which 32 of the 64 from k on
{
    constexpr int DT = __is_same(T, _Float16) ? NL_DT_F16 : NL_DT_BF16;
    typedef __attribute__((__vector_size__(4))) unsigned short U2;
    if (m >= g.M || k + 32 * half >= g.ld8) return;
    nl_i32x4 raw[4];
    U2 top = {};
#pragma unroll
    for (int q = 0; q < 4; q++) {
        raw[q] = *reinterpret_cast<const nl_i32x4*>(lds + row * (GEMM_BK * 2) + ((4 * half + q) ^ (row & 7)) * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) top = __builtin_elementwise_max(top, __builtin_bit_cast(U2, raw[q][j] & 0x7FFF7FFF));
    }
    const unsigned short most = top[0] > top[1] ? top[0] : top[1];
    float amax = DT == NL_DT_BF16 ? nl_bf2f(most) : nl_h2f(most);
    if (!(amax < INFINITY)) {
        amax = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float v[8];
            nl_unraw8<DT>(v, NlRaw8<DT>{{raw[q]}});
#pragma unroll
            for (int j = 0; j < 8; j++) amax = fmaxf(amax, nl_finite_abs(v[j]));
        }
    }
    const int e = nl_mx_exponent(amax);
    const float s = nl_pow2(-e);
    unsigned char* const to = g.A8 + m * g.ld8 + k + 32 * half;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float v[16];
        nl_unraw8<DT>(v, NlRaw8<DT>{{raw[2 * h]}});
        nl_unraw8<DT>(v + 8, NlRaw8<DT>{{raw[2 * h + 1]}});
        nl_i32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (int)nl_mx_encode4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], s);
        *reinterpret_cast<nl_i32x4*>(to + 16 * h) = w;
    }
    g.A8e[m * (g.ld8 / 32) + (k >> 5) + half] = (unsigned char)(e + 127);
}
template <class T, int BM, int NT>
__device__ __forceinline__ void gemm_encode(const NlGemm& g, const char* lds, long long m0, long long k)
{
#pragma unroll
    for (int u = 0; u < (2 * BM + NT - 1) / NT; u++) {
        const int at = u * NT + threadIdx.x;
        if (at < 2 * BM) gemm_encode_block<T>(g, lds, at >> 1, at & 1, m0 + (at >> 1), k);
    }
}

// RING: LDS buffers.  2: the next step arrives while one multiplies.  4 (squares of 64 while they leave compute units idle anyway): three steps are on their way;
// a step of such a tile multiplies for 130 cycles and waits for memory the rest of the time.  One barrier per step, in front of it every wave waits for its own loads of
// the step (the RING - 2 later ones stay in flight) and for its fragment reads of the step before, whose buffer the loads behind the barrier overwrite.
//
// The compiler lets a transposing read wait for every load into LDS that may write the same array.  Where a step has such reads behind the next step's loads, the buffers
// therefore are arrays of their own and the steps are written out one per buffer (APART); otherwise each step waits in its middle for loads that it does not need
// (4096 x 4096 x 16384, both operands transposed: 456 us, APART 416; 8192^3: 898, 820).  With only B transposed its reads simply come first (8192^3: 878, now 805).
// Bound: 256 x 256 x 64 steps take 1.47 us, 1460 TFLOP/s, at the clock that the power limit leaves (the library's best here: 1475); a tile's beginning and end add 11 us.
template <class T, bool A_SLOW, bool B_SLOW, bool B_MX8, int BM, int BN, int WM, int WN, int RING, bool ENC = false>
__global__ __launch_bounds__(64 * WM * WN) void k_gemm(NlGemm g)
{
    constexpr int DT = __is_same(T, _Float16) ? NL_DT_F16 : NL_DT_BF16;
    constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef GemmSide<A_SLOW, BM, NT> SA;
    typedef GemmSide<B_SLOW, BN, NT> SB;
    static_assert(RING == 2 || (RING == 4 && !B_MX8 && !ENC), "buffers are taken in turn by the low bits of the step");
    constexpr bool APART = A_SLOW || (B_SLOW && RING == 4), B_FIRST = B_SLOW && !APART, MIX = FM * FN == 32 && !B_FIRST;      // (MIX: 32768 x 2048 x 2048 225 -> 220 us)
    constexpr int BUF = SA::BYTES + SB::BYTES, LDS = APART ? BUF : RING * BUF;
    __shared__ __align__(256) char s_mem[LDS];
    __shared__ __align__(256) char s_1[BUF];                          // (APART; the last two with RING 4)
    __shared__ __align__(256) char s_2[BUF];
    __shared__ __align__(256) char s_3[BUF];
    long long m0; int n0;
    const unsigned piece = gemm_tile_of<BM, BN>(g, m0, n0);
    const long long k0 = (long long)piece * g.kchunk, k1 = min(k0 + g.kchunk, g.K);
    const int steps = (int)((k1 - k0 + GEMM_BK - 1) / GEMM_BK);
    SA a; SB b;
    GemmSideMx8<T, BN, NT> b8;
    a.init(g.A, g.lda, m0, g.M, k0, g.K);
    if (B_MX8) b8.init(g.B, g.Be, g.ldb, n0, g.N, k0);
    else b.init(g.B, g.ldb, n0, g.N, k0, g.K);
    const int wave = threadIdx.x >> 6, wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
    nl_f32x4 acc[FM][FN] = {};
    // the tiles of a row of tiles take turns at writing A's codes: tile column c the steps c, c + tiles_n, .. of the contraction
    int mine = 0;
    if (ENC) { const int past = (int)((k0 / GEMM_BK) % g.tiles_n); mine = n0 / BN - past; if (mine < 0) mine += g.tiles_n; }
    auto fetch = [&](int s, char* to) {
        const long long left = k1 - k0 - (long long)s * GEMM_BK;
        a.load(to, s * a.step, left);
        if (B_MX8) b8.fetch(s, left);
        else b.load(to + SA::BYTES, s * b.step, left);
    };
    auto step = [&](int s, char* buf, char* next) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * (SA::LOADS + SB::LOADS)) : "memory");
        const char* la = buf;
        const char* lb = buf + SA::BYTES;
        // fragments of both halves of the step, the loads of a later step between them: behind all fragment reads they come late (8192^3 / 16384 x 4096 x 4096,
        // layout 1 and 2: -10 %), in front of them they hold up the reads that the first matrix instructions wait for
        nl_s16x8 fa[2][FM], fb[2][FN];
#pragma unroll
        for (int j = 0; j < FN; j++) fb[0][j] = SB::frag(lb, wn + 16 * j, 0);
#pragma unroll
        for (int i = 0; i < FM; i++) fa[0][i] = SA::frag(la, wm + 16 * i, 0);
        if (B_FIRST) {
#pragma unroll
            for (int j = 0; j < FN; j++) fb[1][j] = SB::frag(lb, wn + 16 * j, 1);
        }
        if (RING > 2 || s + 1 < steps) fetch(s + RING - 1, next);
        if constexpr (MIX) __builtin_amdgcn_sched_barrier(0);
        if (!B_FIRST) {
#pragma unroll
            for (int j = 0; j < FN; j++) fb[1][j] = SB::frag(lb, wn + 16 * j, 1);
        }
#pragma unroll
        for (int i = 0; i < FM; i++) fa[1][i] = SA::frag(la, wm + 16 * i, 1);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = NlMma<T>::mma(fb[0][j], fa[0][i], acc[i][j]);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = NlMma<T>::mma(fb[1][j], fa[1][i], acc[i][j]);
        if constexpr (MIX) {                                          // the second half's reads among the first half's products, not where they are used
#pragma unroll
            for (int q = 0; q < FM + FN; q++) { __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); }
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * FM * FN - FM - FN, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (ENC && s == mine) {
            gemm_encode<T, BM, NT>(g, la, m0, k0 + (long long)s * GEMM_BK);
            mine += g.tiles_n;
        }
        if (B_MX8 && s + 1 < steps) b8.put(next + SA::BYTES);
    };
    // (behind the last step nothing is inside: zeros)
    fetch(0, s_mem);
    if constexpr (RING == 4) { fetch(1, APART ? s_1 : s_mem + BUF); fetch(2, APART ? s_2 : s_mem + 2 * BUF); }
    if (B_MX8) b8.put(s_mem + SA::BYTES);
    if constexpr (!APART) {
        for (int s = 0; s < steps; s++) step(s, s_mem + (s & (RING - 1)) * BUF, s_mem + ((s + RING - 1) & (RING - 1)) * BUF);
    } else if constexpr (RING == 2) {
        for (int s = 0; s < steps; s += 2) {
            step(s, s_mem, s_1);
            if (s + 1 < steps) step(s + 1, s_1, s_mem);
        }
    } else {
        for (int s = 0; s < steps; s += 4) {
            step(s, s_mem, s_3);
            if (s + 1 < steps) step(s + 1, s_1, s_mem);
            if (s + 2 < steps) step(s + 2, s_2, s_1);
            if (s + 3 < steps) step(s + 3, s_3, s_2);
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");        // (all loads, the ones of zeros too: the results pass through the same memory)
    gemm_results<DT, BM / WM, BN / WN, WM * WN, LDS>(g, acc, s_mem, m0 + wm, n0 + wn, piece);
}

// ---------------------------------------------------------------------------------------------
// k_gemm_f32: fp32 operands.  x = h + m + l, three bf16 numbers to nearest, exact (8 bits each of 24) from |x| = 2^-110 on: the
// last bit of such a number is 2^-133 at least, bf16's smallest, which the matrix unit does not flush; below that x is off by at most 2^-134.  Of the nine products of two such numbers the six down to
// 2^-18 are summed, per step of 32 contraction indices the smallest first (l h, h l, m m, m h, h m, h h).  What is dropped (m l, l m, l l) is below 2^-26 |x||w|.
// The split happens on the way into LDS: no operand is written to memory a second time (split planes in memory: 262144 x 256 x 256 spends 118 us on writing and
// 50 us more on reading them).  A thread fetches a step's elements into registers while the step before it multiplies, splits them and writes three planes; two
// workgroups share a compute unit, so that one splits (vector unit) while the other multiplies.  Six products: at most a sixth of the bf16 rate, 246 TFLOP/s.
// 4096^3: 699 us, 197 TFLOP/s, 209 with B split beforehand (the library's fp32 product: 151); 262144 x 256 x 256: 226 us, 152 TFLOP/s (library 97) - eight steps per tile, whose loads and stores
// (537 MB, 105 us) overlap only with the other workgroup's steps.  Starting the second workgroup of a unit later changes nothing.
// ---------------------------------------------------------------------------------------------
// two values to bf16, to nearest, in the halves of a word
__device__ __forceinline__ unsigned gemm_pack2(float a, float b)
{
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float F2;
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 B2;
    return __builtin_bit_cast(unsigned, __builtin_convertvector((F2{a, b}), B2));
}
__device__ __forceinline__ void gemm_split8(const float* x, nl_i32x4& h, nl_i32x4& m, nl_i32x4& l)
{
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int j = 0; j < 4; j++) {                                     // 11 instructions a pair
        const unsigned a = gemm_pack2(x[2 * j], x[2 * j + 1]);
        const float r0 = x[2 * j] - __uint_as_float(a << 16), r1 = x[2 * j + 1] - __uint_as_float(a & 0xFFFF0000u);
        const unsigned b = gemm_pack2(r0, r1);
        h[j] = (int)a; m[j] = (int)b;
        l[j] = (int)gemm_pack2(r0 - __uint_as_float(b << 16), r1 - __uint_as_float(b & 0xFFFF0000u));
    }
    if (top < 0x7F7F8000u) return;
    // rounding overflows, an infinity or a NaN somewhere: the first part cut instead of rounded (as exact); what is not finite stays in it alone
#pragma unroll
    for (int j = 0; j < 4; j++) {
        unsigned a[2];
        float r[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float v = x[2 * j + i];
            const unsigned u = __float_as_uint(v);
            const bool finite = (u & 0x7F800000u) != 0x7F800000u;
            a[i] = finite ? u >> 16 : (unsigned)nl_f2bf(v);
            r[i] = finite ? v - __uint_as_float(u & 0xFFFF0000u) : 0.0f;
        }
        const unsigned b = gemm_pack2(r[0], r[1]);
        h[j] = (int)(a[0] | a[1] << 16); m[j] = (int)b;
        l[j] = (int)gemm_pack2(r[0] - __uint_as_float(b << 16), r[1] - __uint_as_float(b & 0xFFFF0000u));
    }
}

// One operand: R rows or columns x 32 contraction indices per step, 256 threads; the planes' layout in LDS is GemmSide's.  SRC: its elements' type in memory
template <bool SLOW, int R, int SRC>
struct GemmSide32 {
    typedef GemmSide<SLOW, R, 256, 32> Plane;
    static constexpr int UNITS = R * 32 / (8 * 256), BYTES = 3 * Plane::BYTES, ES = SRC == NL_DT_F32 ? 4 : 2;       // a unit: eight neighbouring elements in memory
    unsigned off[UNITS]; int kk[UNITS], lds[UNITS]; bool half[UNITS];                   // half: only the first four elements are inside (fp32, slow: columns)
    NlRaw8<SRC> v[UNITS];
    const char* base; long long step;

    __device__ __forceinline__ void init(const char* p, long long ld, long long i0, long long I, long long k0)
    {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int s = u * 256 + threadIdx.x;
            if (SLOW) {
                const int k = s / (R / 8), c = s % (R / 8);
                kk[u] = k; half[u] = i0 + 8 * c + 4 >= I;
                off[u] = i0 + 8 * c < I ? (unsigned)(k * ld + 8 * ES * c) : GEMM_OUT_OF_RANGE;
                lds[u] = k * (R * 2) + (c ^ (Plane::swz(k) << 1)) * 16;
            } else {
                const int r = s >> 2, c = s & 3;
                kk[u] = 8 * c; half[u] = false;
                off[u] = i0 + r < I ? (unsigned)(r * ld + 8 * ES * c) : GEMM_OUT_OF_RANGE;
                lds[u] = r * 64 + (c ^ Plane::swz_row(r)) * 16;
            }
        }
        base = SLOW ? p + k0 * ld + ES * i0 : p + i0 * ld + ES * k0;
        step = SLOW ? 32 * ld : 32 * ES;
    }
    __device__ __forceinline__ void fetch(long long adv, long long kleft)
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + adv), 0, (int)GEMM_RANGE, 0x00020000);
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const bool in = kk[u] < kleft, in2 = SLOW ? in && !half[u] : kk[u] + 4 < kleft;
            v[u].w[0] = __builtin_bit_cast(nl_i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(in ? off[u] : GEMM_OUT_OF_RANGE), 0, 0));
            if constexpr (SRC == NL_DT_F32)
                v[u].w[1] = __builtin_bit_cast(nl_i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(in2 && off[u] != GEMM_OUT_OF_RANGE ? off[u] + 16 : GEMM_OUT_OF_RANGE), 0, 0));
        }
    }
    __device__ __forceinline__ void put(char* mem) const
    {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            float x[8];
            nl_i32x4 p[3];
            nl_unraw8<SRC>(x, v[u]);
            gemm_split8(x, p[0], p[1], p[2]);
#pragma unroll
            for (int q = 0; q < 3; q++) *reinterpret_cast<nl_i32x4*>(mem + q * Plane::BYTES + lds[u]) = p[q];
        }
    }
};

// DT: the type of B's elements and of the results; A's are fp32 (a 16-bit DT: small backward products whose dz is not rounded)
template <bool A_SLOW, bool B_SLOW, int BT, int DT>
__global__ __launch_bounds__(256, 2) void k_gemm_f32(NlGemm g)
{
    typedef GemmSide32<A_SLOW, BT, NL_DT_F32> SA;
    typedef GemmSide32<B_SLOW, BT, DT> SB;
    constexpr int F = BT / 32, LDS = SA::BYTES + SB::BYTES;
    __shared__ __align__(256) char s_mem[LDS > BT * BT * 2 ? LDS : BT * BT * 2];
    char* const s_b = s_mem + SA::BYTES;
    long long m0; int n0;
    const unsigned piece = gemm_tile_of<BT, BT>(g, m0, n0);
    const long long k0 = (long long)piece * g.kchunk, k1 = min(k0 + g.kchunk, g.K), span = k1 - k0;
    const int steps = (int)((span + 31) / 32);
    SA a; SB b;
    a.init(g.A, g.lda, m0, g.M, k0);
    b.init(g.B, g.ldb, n0, g.N, k0);
    const int wave = threadIdx.x >> 6, wm = (wave >> 1) * (BT / 2), wn = (wave & 1) * (BT / 2);
    nl_f32x4 acc[F][F] = {};
    a.fetch(0, span);
    b.fetch(0, span);
    for (int s = 0; s < steps; s++) {
        a.put(s_mem);
        b.put(s_b);
        nl_lds_barrier();
        if (s + 1 < steps) {
            a.fetch((s + 1) * a.step, span - (s + 1) * 32LL);
            b.fetch((s + 1) * b.step, span - (s + 1) * 32LL);
        }
        __builtin_amdgcn_sched_barrier(0);
        nl_s16x8 fb[3][F];
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int j = 0; j < F; j++) fb[p][j] = SB::Plane::frag(s_b + p * SB::Plane::BYTES, wn + 16 * j, 0);
#pragma unroll
        for (int i = 0; i < F; i++) {
            nl_s16x8 fa[3];
#pragma unroll
            for (int p = 0; p < 3; p++) fa[p] = SA::Plane::frag(s_mem + p * SA::Plane::BYTES, wm + 16 * i, 0);
#pragma unroll
            for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                for (int p = sum; p >= 0; p--)
#pragma unroll
                    for (int j = 0; j < F; j++) acc[i][j] = NlMma<__bf16>::mma(fb[sum - p][j], fa[p], acc[i][j]);
        }
        nl_lds_barrier();
    }
    gemm_results<DT, BT / 2, BT / 2, 4, sizeof(s_mem)>(g, acc, s_mem, m0 + wm, n0 + wn, piece);
}

// The same with B already split, in three planes g.plane bytes apart (nl_linear.hip splits a weight once where many rows of tiles would split it again each): its planes go
// straight into LDS, into two buffers in turn (arrays of their own, as in k_gemm), and only A passes through registers.  4096^3: 658 us, 209 TFLOP/s, 699 without.
template <bool A_SLOW, bool B_SLOW, int BT>
__global__ __launch_bounds__(256, 2) void k_gemm_f32_planes(NlGemm g)
{
    typedef GemmSide32<A_SLOW, BT, NL_DT_F32> SA;
    typedef GemmSide<B_SLOW, BT, 256, 32> PB;
    constexpr int F = BT / 32;
    __shared__ __align__(256) char s_mem[SA::BYTES + 3 * PB::BYTES];
    __shared__ __align__(256) char s_1[3 * PB::BYTES];
    long long m0; int n0;
    const unsigned piece = gemm_tile_of<BT, BT>(g, m0, n0);
    const long long k0 = (long long)piece * g.kchunk, k1 = min(k0 + g.kchunk, g.K), span = k1 - k0;
    const int steps = (int)((span + 31) / 32);
    SA a; PB b;
    a.init(g.A, g.lda, m0, g.M, k0);
    b.init(g.B, g.ldb, n0, g.N, k0, g.K);
    const int wave = threadIdx.x >> 6, wm = (wave >> 1) * (BT / 2), wn = (wave & 1) * (BT / 2);
    nl_f32x4 acc[F][F] = {};
    auto fetch = [&](int s, char* to) {
        a.fetch(s * a.step, span - s * 32LL);
#pragma unroll
        for (int q = 0; q < 3; q++) b.load(to + q * PB::BYTES, s * b.step + q * g.plane, span - s * 32LL);
    };
    auto step = [&](int s, const char* buf, char* next) {
        a.put(s_mem);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        nl_s16x8 fb[3][F];
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int j = 0; j < F; j++) fb[p][j] = PB::frag(buf + p * PB::BYTES, wn + 16 * j, 0);
        if (s + 1 < steps) fetch(s + 1, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < F; i++) {
            nl_s16x8 fa[3];
#pragma unroll
            for (int p = 0; p < 3; p++) fa[p] = SA::Plane::frag(s_mem + p * SA::Plane::BYTES, wm + 16 * i, 0);
#pragma unroll
            for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                for (int p = sum; p >= 0; p--)
#pragma unroll
                    for (int j = 0; j < F; j++) acc[i][j] = NlMma<__bf16>::mma(fb[sum - p][j], fa[p], acc[i][j]);
        }
        nl_lds_barrier();
    };
    fetch(0, s_mem + SA::BYTES);
    for (int s = 0; s < steps; s += 2) {
        step(s, s_mem + SA::BYTES, s_1);
        if (s + 1 < steps) step(s + 1, s_1, s_mem + SA::BYTES);
    }
    gemm_results<NL_DT_F32, BT / 2, BT / 2, 4, sizeof(s_mem)>(g, acc, s_mem, m0 + wm, n0 + wn, piece);
}

template <bool A_SLOW, bool B_SLOW>
static void nl_gemm_tile_f32(const NlGemm& g, int tile, dim3 grid, hipStream_t st)
{
    if constexpr (!A_SLOW) {
        if (g.plane) { hipLaunchKernelGGL((k_gemm_f32_planes<A_SLOW, B_SLOW, 128>), grid, dim3(256), 0, st, g); return; }
    }
    if (tile == 1) hipLaunchKernelGGL((k_gemm_f32<A_SLOW, B_SLOW, 128, NL_DT_F32>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_gemm_f32<A_SLOW, B_SLOW, 64, NL_DT_F32>), grid, dim3(256), 0, st, g);
}

template <class T, bool A_SLOW, bool B_SLOW, bool B_MX8, bool ENC = false>
static void nl_gemm_tile(const NlGemm& g, int tile, dim3 grid, hipStream_t st)
{
    if (tile == 0) hipLaunchKernelGGL((k_gemm<T, A_SLOW, B_SLOW, B_MX8, 256, 256, 2, 4, 2, ENC>), grid, dim3(512), 0, st, g);
    else if (tile == 1) hipLaunchKernelGGL((k_gemm<T, A_SLOW, B_SLOW, B_MX8, 128, 128, 2, 2, 2, ENC>), grid, dim3(256), 0, st, g);
    else {
        if constexpr (!B_MX8 && !ENC) {
            if ((long long)grid.x * grid.y <= NL_GEMM_FEW_SQUARES) { hipLaunchKernelGGL((k_gemm<T, A_SLOW, B_SLOW, false, 64, 64, 2, 2, 4>), grid, dim3(256), 0, st, g); return; }
        }
        hipLaunchKernelGGL((k_gemm<T, A_SLOW, B_SLOW, B_MX8, 64, 64, 2, 2, 2, ENC>), grid, dim3(256), 0, st, g);
    }
}
template <class T>
static void nl_gemm_layout(const NlGemm& g, int layout, int tile, dim3 grid, hipStream_t st)
{
    if (layout == 0) nl_gemm_tile<T, false, false, false>(g, tile, grid, st);
    else if (layout == 1) nl_gemm_tile<T, false, true, false>(g, tile, grid, st);
    else if (layout == 2) nl_gemm_tile<T, true, true, false>(g, tile, grid, st);
    else if (layout == 3) nl_gemm_tile<T, true, true, true>(g, tile, grid, st);
    else nl_gemm_tile<T, false, false, false, true>(g, tile, grid, st);
}
#endif

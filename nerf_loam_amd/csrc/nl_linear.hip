// nl_linear.hip -- one linear layer: z = x w^T + b, y = act(z) + r, and its backward pass (include/nerfloam_hip.h NlLinear).
//
// Reference behaviour: torch.nn.Linear + ReLU of the decoder (/root/reference/src/variations/lidar.py:105-123), any width, any depth.
#include "nl_narrow.h"

#include <math.h>

// ---------------------------------------------------------------------------------------------
// k_linear_pack: an operand as the tiled products want it - rows of up(cols, 8) elements with zeros behind the last column - from rows of any stride and
// alignment, or from 8-bit codes (for fp32 arithmetic).  Runs only where the operand does not lie that way already
// (1003 x 1001 and 777 x 1001 bf16, odd rows: 4.9 us in one launch, the product behind it 10.3).
// ---------------------------------------------------------------------------------------------
struct NlPack { const void* src; const unsigned char* e; void* dst; long long rows, ld, pitch; int cols; };
struct NlPack2 { NlPack p[2]; };                                     // one launch for both operands of a product, or both of a backward pass

template <int DT>
__global__ __launch_bounds__(256) void k_linear_pack(NlPack2 both)
{
    const NlPack a = both.p[blockIdx.y];
    const long long per_row = a.pitch / 8, total = a.rows * per_row;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const long long r = t / per_row;
        const int c = (int)(t - r * per_row) * 8;
        float v[8];
        if (a.e) {
            const nl_i32x2 w = *reinterpret_cast<const nl_i32x2*>((const unsigned char*)a.src + r * a.ld + c);       // (rows of codes are whole blocks of 32, zeros behind the last)
            const float s = nl_mx_scale(a.e[r * (a.ld / 32) + (c >> 5)]);
            const nl_f32x4 p = nl_mx_decode4((unsigned)w[0], s, nl_dtype_max(DT)), q = nl_mx_decode4((unsigned)w[1], s, nl_dtype_max(DT));
#pragma unroll
            for (int j = 0; j < 4; j++) { v[j] = p[j]; v[4 + j] = q[j]; }
        } else nl_load8<DT>(v, a.src, r * a.ld + c, a.cols - c);
        nl_store8<DT>(a.dst, r * a.pitch + c, v, 8);
    }
}

// A weight in three bf16 planes [3][rows][pitch] for k_gemm_f32_planes, zeros behind the last column (512 x 256: 4 us)
__global__ __launch_bounds__(256) void k_linear_split(const float* src, long long ld, long long rows, int cols, unsigned short* dst, long long pitch)
{
    const long long per_row = pitch / 8, total = rows * per_row;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const long long r = t / per_row;
        const int c = (int)(t - r * per_row) * 8;
        float v[8];
        nl_i32x4 p[3];
        nl_load8<NL_DT_F32>(v, src, r * ld + c, cols - c);
        gemm_split8(v, p[0], p[1], p[2]);
#pragma unroll
        for (int q = 0; q < 3; q++) *reinterpret_cast<nl_i32x4*>(dst + (q * rows + r) * pitch + c) = p[q];
    }
}

// ---------------------------------------------------------------------------------------------
// k_linear_rows: at most ROWS_MOST rows of x (the call that answers single queries) or of the weight (a last layer with one output), nothing kept for a backward pass.
// It reads the other operand once and computes little, so no tile: a group of `lanes` threads takes two rows of the many, eight neighbouring elements a thread at a
// time, several loads in flight, and sums across its threads at the end.  One launch (1 x 4096 x 4096 bf16: 6.4 us, as tiles of 64 cut 16 times and joined 9.7).
// SWAP: the few rows are the weight's, the many are x's.
// ---------------------------------------------------------------------------------------------
#define ROWS_MOST 8
struct NlRows { const void* few; const void* many; long long ldf, ldm, nmany; int nfew, K, lanes; };
template <int DT, int MR, bool SWAP>
__global__ __launch_bounds__(256) void k_linear_rows(NlRows g, NlEpilogue ep)
{
    constexpr int R = 2, U = MR == 1 ? 4 : MR <= 4 ? 2 : 1;
    const int lanes = g.lanes, lane = threadIdx.x & (lanes - 1), K = g.K;
    const long long n0 = (nl_block() * (256 / lanes) + threadIdx.x / lanes) * R;
    if (n0 >= g.nmany) return;                                        // (a whole group)
    const long long n1 = n0 + 1 < g.nmany ? n0 + 1 : n0;
    float acc[MR][R] = {};
    int k = lane * 8;
    for (; k + (U - 1) * lanes * 8 + 8 <= K; k += U * lanes * 8) {
        NlRaw8<DT> a[U][R], b[U][MR];
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u][0] = nl_raw8<DT>(g.many, n0 * g.ldm + k + u * lanes * 8);
            a[u][1] = nl_raw8<DT>(g.many, n1 * g.ldm + k + u * lanes * 8);
#pragma unroll
            for (int m = 0; m < MR; m++) b[u][m] = nl_raw8<DT>(g.few, (m < g.nfew ? m : 0) * g.ldf + k + u * lanes * 8);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float p[R][8];
            nl_unraw8<DT>(p[0], a[u][0]);
            nl_unraw8<DT>(p[1], a[u][1]);
#pragma unroll
            for (int m = 0; m < MR; m++) {
                float q[8];
                nl_unraw8<DT>(q, b[u][m]);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[m][r] = __builtin_fmaf(p[r][j], q[j], acc[m][r]);
            }
        }
    }
    for (; k < K; k += lanes * 8) {
        float p[R][8];
        nl_load8<DT>(p[0], g.many, n0 * g.ldm + k, K - k);
        nl_load8<DT>(p[1], g.many, n1 * g.ldm + k, K - k);
#pragma unroll
        for (int m = 0; m < MR; m++) {
            float q[8];
            nl_load8<DT>(q, g.few, (m < g.nfew ? m : 0) * g.ldf + k, K - k);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int j = 0; j < 8; j++) acc[m][r] = __builtin_fmaf(p[r][j], q[j], acc[m][r]);
        }
    }
#pragma unroll
    for (int f = 0; f < MR; f++)
#pragma unroll
        for (int r = 0; r < R; r++) {
            float v = acc[f][r];
            for (int off = lanes >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off);
            if (lane != 0 || f >= g.nfew || n0 + r >= g.nmany) continue;
            const long long m = SWAP ? n0 + r : f, n = SWAP ? f : n0 + r;
            if (ep.b) v += nl_load_elem<DT>(ep.b, n);
            v = nl_act(v, ep.act);
            if (ep.r) v += nl_load_elem<DT>(ep.r, m * ep.ldr + n);
            nl_store_elem<DT>(ep.y, m * ep.ldy + n, v);
        }
}
template <int DT, bool SWAP> static int nl_launch_rows(const NlLinear* d, const NlEpilogue& ep, hipStream_t st)
{
    NlRows g = SWAP ? NlRows{d->w, d->x, d->ldw, d->ldx, d->M, d->N, d->K, 8} : NlRows{d->x, d->w, d->ldx, d->ldw, d->N, (int)d->M, d->K, 8};
    while (g.lanes < 64 && g.lanes * 8 < d->K) g.lanes *= 2;
    const long long blocks = (g.nmany + 2 * (256 / g.lanes) - 1) / (2 * (256 / g.lanes));
    const dim3 grid = nl_blocks(blocks);
    if (g.nfew == 1) hipLaunchKernelGGL((k_linear_rows<DT, 1, SWAP>), grid, dim3(256), 0, st, g, ep);
    else if (g.nfew == 2) hipLaunchKernelGGL((k_linear_rows<DT, 2, SWAP>), grid, dim3(256), 0, st, g, ep);
    else if (g.nfew <= 4) hipLaunchKernelGGL((k_linear_rows<DT, 4, SWAP>), grid, dim3(256), 0, st, g, ep);
    else hipLaunchKernelGGL((k_linear_rows<DT, 8, SWAP>), grid, dim3(256), 0, st, g, ep);
    return NL_OK;
}

// gb[n] = sum over the chunks of k_linear_dz: four columns a workgroup, 256 runs of neighbouring chunks, the runs joined pairwise (2048 chunks x 256: 6 us, latency)
struct NlGb { const float* part; void* gb; int chunks, N, blocks; };      // blocks: workgroups that it takes
template <int DT>
__device__ __forceinline__ void nl_gb_block(const NlGb& a, int block, nl_f32x4* s_sum)
{
    const int n = block * 4, run = threadIdx.x, N = a.N;
    const int per = (a.chunks + 255) / 256, c1 = (run + 1) * per < a.chunks ? (run + 1) * per : a.chunks;
    nl_f32x4 s = {};
    if ((N & 3) == 0) {
#pragma unroll 4
        for (int c = run * per; c < c1; c++) s += *reinterpret_cast<const nl_f32x4*>(a.part + (long long)c * N + n);
    } else
        for (int c = run * per; c < c1; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) if (n + j < N) s[j] += a.part[(long long)c * N + n + j];
    s_sum[run] = s;
    for (int off = 128; off >= 1; off >>= 1) {
        __syncthreads();
        if (run < off) s_sum[run] += s_sum[run + off];
    }
    if (run != 0) return;
#pragma unroll
    for (int j = 0; j < 4; j++) if (n + j < N) nl_store_elem<DT>(a.gb, n + j, s_sum[0][j]);
}
template <int DT>
__global__ __launch_bounds__(256) void k_linear_gb(NlGb a)
{
    __shared__ nl_f32x4 s_sum[256];
    nl_gb_block<DT>(a, blockIdx.x, s_sum);
}

// ---------------------------------------------------------------------------------------------
// k_linear_join: sums the pieces of a split contraction and runs the epilogue.  Eight columns a thread, whole blocks of 32 columns.  With few results and many pieces
// one thread per result group would walk all pieces one memory latency after the other (256 x 256 results in 64 pieces: 30 us): then RUNS threads sum a run of
// neighbouring pieces each and the runs are added in order (the same in 128 pieces: 11 us, bound by latency; 2048 x 2048 in 4 pieces, 76 MB: 17 us).  The first gb.blocks workgroups sum a bias gradient: one launch less where a weight gradient is joined.
// ---------------------------------------------------------------------------------------------
template <int DT, int RUNS>
__global__ __launch_bounds__(256) void k_linear_join(const float* __restrict__ part, int splits, long long M, int N, NlEpilogue ep, NlGb gb)
{
    constexpr int POS = 256 / RUNS;
    __shared__ __align__(16) char s_mem[RUNS > 1 ? RUNS * POS * 9 * 4 : 256 * 16];
    if ((int)blockIdx.x < gb.blocks) { nl_gb_block<DT>(gb, blockIdx.x, (nl_f32x4*)s_mem); return; }
    float (*const s_sum)[POS][9] = (float (*)[POS][9])s_mem;
    const unsigned block = blockIdx.x - gb.blocks, blocks = gridDim.x - gb.blocks;
    const int at = threadIdx.x % POS, run = threadIdx.x / POS, per = (splits + RUNS - 1) / RUNS;
    const int s0 = run * per, s1 = s0 + per < splits ? s0 + per : splits;
    const long long per_row = (N + 31) / 32 * 4, total = M * per_row;
    for (long long t0 = (long long)block * POS; t0 < total; t0 += (long long)blocks * POS) {
        const long long t = t0 + at, m = t / per_row;
        const int n = (int)(t - m * per_row) * 8;
        float v[8] = {};
        if (m < M) {
            const float* p = part + (long long)s0 * M * N + m * N + n;
            if (n + 7 < N && (N & 3) == 0) {
#pragma unroll 4
                for (int s = s0; s < s1; s++, p += M * N) {
                    const nl_f32x4 a = *reinterpret_cast<const nl_f32x4*>(p), b = *reinterpret_cast<const nl_f32x4*>(p + 4);
#pragma unroll
                    for (int j = 0; j < 4; j++) { v[j] += a[j]; v[4 + j] += b[j]; }
                }
            } else
                for (int s = s0; s < s1; s++, p += M * N)
#pragma unroll
                    for (int j = 0; j < 8; j++) if (n + j < N) v[j] += p[j];
        }
        if (RUNS > 1) {
#pragma unroll
            for (int j = 0; j < 8; j++) s_sum[run][at][j] = v[j];
            __syncthreads();
            if (run == 0) {
#pragma unroll
                for (int r = 1; r < RUNS; r++)
#pragma unroll
                    for (int j = 0; j < 8; j++) v[j] += s_sum[r][at][j];
                nl_epilogue8_fetch<DT>(ep, v, m, n, M, N, 0);
            }
            __syncthreads();
        } else nl_epilogue8_fetch<DT>(ep, v, m, n, M, N, 0);
    }
}

// ---------------------------------------------------------------------------------------------
// k_linear_dz: dz = gy act'(z), packed for the two products of the backward pass, and the sums of dz over a chunk of rows for the bias (unrounded).
// A workgroup: 256 columns (eight to a thread) x rows_per_chunk rows, eight rows at a time.  dz is rounded to the tensors' type because that is what the matrix unit
// multiplies (OUT fp32 where nl_wide says so).  Bound by memory: 16384 x 4096 bf16 gelu 403 MB in 78 us, 65536 x 512 fp32 silu 403 MB in 79 us, 5.1 TB/s, what a large
// copy reaches; hence one exponential and one reciprocal per element.
// ---------------------------------------------------------------------------------------------
template <int DT, int ACT, int OUT>
__global__ __launch_bounds__(256) void k_linear_dz(NlDz a)
{
    __shared__ float s_sum[8][257];
    const int c8 = threadIdx.x & 31, n = blockIdx.x * 256 + 8 * c8, grp = threadIdx.x >> 5;
    const long long m1 = (blockIdx.y + 1) * a.rows_per_chunk < a.M ? (blockIdx.y + 1) * a.rows_per_chunk : a.M;
    constexpr float most = DT == NL_DT_F16 ? NL_F16_MAX : DT == NL_DT_BF16 ? 3.38953139e38f : 3.40282347e38f;
    float sum[8] = {};
    if (n < a.N)
        for (long long m = blockIdx.y * a.rows_per_chunk + grp; m < m1; m += 8) {
            float g[8], z[8];
            nl_load8<DT>(g, a.gy, m * a.ldgy + n, a.N - n);
            if (ACT == NL_ACT_RELU) {
                const unsigned w = a.bits[m * a.ldbits + (n >> 5)] >> (n & 31);
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] = (w >> j & 1) ? g[j] : 0.0f;
            } else if (ACT != NL_ACT_NONE) {
                if (a.z8) {
                    const nl_i32x2 w = *reinterpret_cast<const nl_i32x2*>(a.z8 + m * a.ldz8 + n);
                    const float s = nl_mx_scale(a.z8e[m * a.ldz8e + (n >> 5)]);
                    const nl_f32x4 p = nl_mx_decode4((unsigned)w[0], s, most), q = nl_mx_decode4((unsigned)w[1], s, most);
#pragma unroll
                    for (int j = 0; j < 4; j++) { z[j] = p[j]; z[4 + j] = q[j]; }
                } else nl_load8<DT>(z, a.z, m * a.ldz + n, a.N - n);
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] = n + j < a.N ? g[j] * nl_act_slope(z[j], ACT) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) sum[j] += g[j];
            if (a.dz) nl_store8<OUT>(a.dz, m * a.pitch + n, g, 8);
        }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < 8; j++) s_sum[grp][8 * c8 + j] = sum[j];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= a.N) return;
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; r++) s += s_sum[r][threadIdx.x];
    a.part[(long long)blockIdx.y * a.N + col] = s;
}

__global__ __launch_bounds__(256) void k_linear_zero(unsigned char* p, long long bytes)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (long long)gridDim.x * 256) p[i] = 0;
}

// ---------------------------------------------------------------------------------------------
// host: plans and launches.  Every function below runs twice: first without a workspace, to say how much it takes, then with it, to launch.
// ---------------------------------------------------------------------------------------------
#define NL_LINEAR_MAX_WIDTH (1 << 22)
#define NL_LINEAR_MAX_ROWS (1LL << 30)

struct NlWork {
    char* base; long long used; hipStream_t st; bool dry; int rc;
    NlPack2 pack; int packs;                                      // noted by nl_packed, launched by nl_pack
    char* take(long long bytes) { char* p = base + used; used += nl_up(bytes, 256); return p; }
};

// a packed operand: rows `pitch` elements apart, zeros behind the last column up to a multiple of 8 (4 where an fp32 operand is used in place)
struct NlPacked { const void* p; long long pitch; const unsigned char* e; long long plane; };      // e: 8-bit codes and their powers of two instead; plane: bytes between bf16 planes instead

static unsigned nl_grid(long long threads) { const long long b = (threads + 255) / 256; return (unsigned)(b < 1 ? 1 : b < 16384 ? b : 16384); }

static bool nl_in_place(const void* p, int cols, long long ld, int dt)
{
    const int v = dt == NL_DT_F32 ? 4 : 8;
    return ld % v == 0 && cols % v == 0 && ld <= NL_LINEAR_MAX_WIDTH && ((uintptr_t)p & 15) == 0;
}
static void nl_pack(NlWork& w, int dt)
{
    if (!w.packs) return;
    long long most = 0;
    for (int i = 0; i < w.packs; i++) { const long long t = w.pack.p[i].rows * (w.pack.p[i].pitch / 8); if (t > most) most = t; }
    if (!w.dry) NL_WITH_DTYPE(dt, hipLaunchKernelGGL(k_linear_pack<DT>, dim3(nl_grid(most), w.packs), dim3(256), 0, w.st, w.pack));
    w.packs = 0;
}
static NlPacked nl_packed(NlWork& w, const void* p, const unsigned char* e, long long rows, int cols, long long ld, int type, int dt)
{
    if (type == dt && nl_in_place(p, cols, ld, dt)) return NlPacked{p, ld, nullptr};
    NlPack a = {};
    a.src = p; a.e = e; a.rows = rows; a.cols = cols; a.ld = ld;
    a.pitch = nl_up(cols, 8);
    a.dst = w.take(rows * a.pitch * nl_dtype_size(dt));
    w.pack.p[w.packs++] = a;
    return NlPacked{a.dst, a.pitch, nullptr};
}

// How a product [M,N] over K is cut: the tile, and into how many pieces the contraction goes.  The estimate: rounds of as many workgroups as run at a time, each with
// its contraction steps of 64 (alone on a compute unit / with as many neighbours as fit) and what surrounds them; for a cut contraction the pieces' way through memory
// and the launch that joins them.  Measured, in microseconds, on operands of numbers (zeros draw less power: 4096^3 takes 95 and 576 of them) (bf16, 4096^3: 111 in squares of 256, 124 of 128, 193 of 64;
// 2048 x 256 x 256: 14, 7.2, 4.3; 256 x 256 x 200000: 55 in 256 pieces of the first, 47 in 128 of the second, 50 in 32 of the third, 4000 uncut; 8-bit codes, 256 x 256 x 200000
// from memory: 73 in 64 pieces of the second, 52 in 128, 80 in squares of 64; fp32 4096^3: 680 in squares of 128, 864 of 64, 2048 x 256 x 256: 20, 9.6).  At 23 shapes of either kind
// the estimate's choice is the best of all tiles and powers of two or within 6 % of it, but for 256 x 4096 x 4096 (20 and 16 %), 256 x 256 x 200000 bf16 (11), 512^3 and 2048^3 fp32
// (12 and 16) and 128 x 128 x 4096 bf16 (13.2 instead of 8.8).
struct NlCut { int tile, splits; long long kchunk; };
static NlCut nl_cut(long long M, long long N, long long K, int dt, int layout, int largest)
{
    struct Tile { int size, at_a_time; double alone, full, rest, codes; };      // codes: on the steps of layout 3 (a thread decodes as much, the tile multiplies less)
    static const Tile T16[3] = {{256, 256, 1.33, 1.40, 9.0, 1.0}, {128, 512, 0.70, 0.87, 4.0, 1.0}, {64, 1024, 0.50, 0.67, 2.0, 1.6}};
    static const Tile T32[3] = {{256, 0, 0, 0, 0, 0}, {128, 512, 3.95, 4.50, 4.0, 1.0}, {64, 1024, 1.67, 2.60, 2.5, 1.0}};
    const Tile* T = dt == NL_DT_F32 ? T32 : T16;
    const long long ksteps = (K + GEMM_BK - 1) / GEMM_BK;
    const double memory = ((double)nl_dtype_size(dt) * (M * K + M * N) + (layout == 3 ? 1.0 : nl_dtype_size(dt)) * N * K) / 4.5e6;
    NlCut best = {2, 1, ksteps * GEMM_BK};
    double least = 1e300;
    for (int t = largest; t < 3; t++) {
        const double tiles = (double)(nl_up(M, T[t].size) / T[t].size) * (double)(nl_up(N, T[t].size) / T[t].size);
        for (int s = 1; s <= 256 && s <= ksteps; s *= 2) {
            if (s > 1 && 4.0 * s * M * N > 1.5e9) break;
            const long long per = (ksteps + s - 1) / s;
            const double at = tiles * s / T[t].at_a_time, full = at < 1.0 ? at : 1.0, rounds = at < 1.0 ? 1.0 : at < 4.0 ? ceil(at) : at + 0.5;
            const bool ring = t == 2 && dt != NL_DT_F32 && layout < 3 && tiles * s <= NL_GEMM_FEW_SQUARES;      // (four buffers)
            // two buffers: one workgroup to a compute unit draws half of the bandwidth (of squares of 256 all of it)
            const double alone = ring ? 0.28 : T[t].alone, draws = tiles * s / (t == 0 ? 256 : 512), reach = ring || draws > 1.0 ? 1.0 : draws;
            double us = rounds * (per * (alone + (T[t].full - alone) * full) * (layout == 3 ? T[t].codes : 1.0) + T[t].rest * (0.5 + 0.5 * full));
            if (us < memory / reach) us = memory / reach;
            if (s > 1) us += 5.0 + 4.0 * s * M * N / 4.0e6;
            if (us < least) { least = us; best = NlCut{t, s, per * GEMM_BK}; }
        }
    }
    best.splits = (int)((K + best.kchunk - 1) / best.kchunk);
    return best;
}

// The weight of an fp32 product, split beforehand where that saves more than it costs: every row of tiles splits it again otherwise (4096^3 699 -> 658 us, 65536 x 512 -> 256
// 100 -> 93, 262144 x 256 -> 256 226 -> 226, 4096 x 512 -> 2048 54 -> 54); the pass over the weight takes a launch, 5 us, and 10 bytes an element.  M, N, K: the product's; squares of 128 only
static NlPacked nl_weight(NlWork& w, const NlLinear* d, long long M, int N, int K, int layout)
{
    if (d->dtype != NL_DT_F32 || M < 4096 || K < 512 || (double)M * N * K < 4e9 || nl_cut(M, N, K, NL_DT_F32, layout, 1).tile != 1)
        return nl_packed(w, d->w, nullptr, d->N, d->K, d->ldw, d->dtype, d->dtype);
    const long long pitch = nl_up(d->K, 8);
    unsigned short* const to = (unsigned short*)w.take(6 * d->N * pitch);
    if (!w.dry) hipLaunchKernelGGL(k_linear_split, dim3(nl_grid(d->N * (pitch / 8))), dim3(256), 0, w.st, (const float*)d->w, d->ldw, (long long)d->N, d->K, to, pitch);
    return NlPacked{to, pitch, nullptr, 2 * d->N * pitch};
}

// C[M,N] = sum_k A(m,k) B(n,k), layouts as in nl_gemm.h.  A8, A8e: layout 4's codes.  gb: a bias gradient to sum in the same launch if there is one; then it is cleared.
// wide: A is fp32 whatever the type
static void nl_product(NlWork& w, const NlPacked& A, const NlPacked& B, int layout, long long M, int N, long long K, const NlEpilogue& ep, unsigned char* A8, unsigned char* A8e, NlGb* gb, bool wide)
{
    const NlCut c = nl_cut(M, N, K, wide ? NL_DT_F32 : ep.dt, layout == 4 ? 0 : layout, wide ? 2 : ep.dt == NL_DT_F32 ? 1 : 0);      // (the codes do not change the sums)
    static const int size[3] = {256, 128, 64};
    NlGemm g = {};
    g.A = (const char*)A.p; g.B = (const char*)B.p; g.Be = B.e; g.lda = (wide ? 4 : nl_dtype_size(ep.dt)) * A.pitch; g.ldb = layout == 3 ? B.pitch : nl_dtype_size(ep.dt) * B.pitch;
    if (B.plane) { g.plane = B.plane; g.ldb = 2 * B.pitch; }
    g.A8 = A8; g.A8e = A8e; g.ld8 = nl_up(K, NL_MX_BLOCK);
    g.M = M; g.N = N; g.K = K; g.kchunk = c.kchunk;
    const long long tm = nl_up(M, size[c.tile]) / size[c.tile], tn = nl_up(N, size[c.tile]) / size[c.tile];
    if (tm * tn * (c.tile == 0 ? 512 : 256) > 0xFFFFFFFFLL) {      // (a grid's axis)
        w.rc = NL_ERR_INVALID_ARG; return; }
    g.tiles_m = (int)tm; g.tiles_n = (int)tn;
    g.ep = ep;
    if (c.splits > 1) { g.ep = NlEpilogue{}; g.ep.part = (float*)w.take(4LL * c.splits * M * N); }
    if (w.dry) return;
    const dim3 grid((unsigned)(tm * tn), (unsigned)c.splits);
    if (wide) nl_gemm_f32_to16(g, ep.dt, layout, grid, w.st);
    else if (ep.dt == NL_DT_F32) nl_gemm_f32(g, layout, c.tile, grid, w.st);
    else if (ep.dt == NL_DT_BF16) nl_gemm_bf16(g, layout, c.tile, grid, w.st);
    else nl_gemm_f16(g, layout, c.tile, grid, w.st);
    if (c.splits > 1) {
        const long long groups = M * ((N + 31) / 32 * 4);
        const NlGb bias = gb ? *gb : NlGb{};
        if (gb) *gb = NlGb{};
        if (c.splits >= 8 && groups < 131072) NL_WITH_DTYPE(ep.dt, hipLaunchKernelGGL((k_linear_join<DT, 8>), dim3(nl_grid(8 * groups) + bias.blocks), dim3(256), 0, w.st, g.ep.part, c.splits, M, N, ep, bias));
        else NL_WITH_DTYPE(ep.dt, hipLaunchKernelGGL((k_linear_join<DT, 1>), dim3(nl_grid(groups) + bias.blocks), dim3(256), 0, w.st, g.ep.part, c.splits, M, N, ep, bias));
    }
    if (hipGetLastError() != hipSuccess) w.rc = NL_ERR_LAUNCH;
}

// A weight of at most 256 x 256 in 16 bits: when the product streams (nl_narrow.h).  K: the contraction, N: the results' columns; dz: the data gradient that makes dz on
// its way, which saves a pass and a launch.  Without dz it pays for wide results that do not stay in the caches (bf16, us, tiles / streaming: 262144 x 256 -> 256 relu 90 / 74,
// 262144 x 16 -> 256 55 / 44, 65536 x 256 -> 256 22.3 / 23.8, 262144 x 64 -> 160 39 / 44; 262144 x 256 -> 64 45 / 47, 262144 x 64 -> 64 17 / 39); with it everywhere (all gradients, relu:
// 64 x 256 -> 256 24 / 21, 4096 x 256 -> 256 24.5 / 22.0, 65536 x 256 -> 256 58 / 46, 262144 x 256 -> 64 121 / 103; only 262144 x 64 -> 64 52 / 54).
static int nl_stream_groups(long long M) { const long long tiles = (M + NL_NARROW_ROWS - 1) / NL_NARROW_ROWS; return tiles < 256 ? (int)tiles : 256; }      // one to a compute unit
static bool nl_streams(long long M, int K, int N, int dt, bool dz)
{
    if (dt == NL_DT_F32 || K > 256 || N > 256) return false;
    return dz || (M >= 65536 && N > 128);
}
static void nl_stream(NlWork& w, const NlPacked& A, const NlPacked& B, bool b_slow, long long M, int N, int K, const NlEpilogue& ep, unsigned char* A8, unsigned char* A8e, const NlDz& z, int act, int dz)
{
    if (w.dry) return;
    NlGemm g = {};
    g.A = (const char*)A.p; g.B = (const char*)B.p; g.lda = 2 * A.pitch; g.ldb = 2 * B.pitch;
    g.A8 = A8; g.A8e = A8e; g.ld8 = nl_up(K, NL_MX_BLOCK);
    g.M = M; g.N = N; g.K = K; g.ep = ep;
    if (ep.dt == NL_DT_BF16) nl_narrow_bf16(g, z, act, b_slow, dz, (unsigned)nl_stream_groups(M), w.st);
    else nl_narrow_f16(g, z, act, b_slow, dz, (unsigned)nl_stream_groups(M), w.st);
    if (hipGetLastError() != hipSuccess) w.rc = NL_ERR_LAUNCH;
}

// what a pass runs as: few rows without tiles; the streaming product (backward: the data gradient as one)
static bool nl_forward_rows(const NlLinear* d) { return (d->M <= ROWS_MOST || d->N <= ROWS_MOST) && !d->z && !d->bits && !d->z8; }
static bool nl_forward_streams(const NlLinear* d) { return !nl_forward_rows(d) && nl_streams(d->M, d->K, d->N, d->dtype, false); }

static void nl_forward_run(const NlLinear* d, NlWork& w)
{
    NlEpilogue ep = {};
    ep.b = d->b; ep.r = d->r; ep.ldr = d->ldr; ep.y = d->y; ep.ldy = d->ldy; ep.dt = d->dtype; ep.act = d->act;
    ep.z = d->z; ep.ldz = d->N;
    ep.bits = d->bits; ep.ldbits = nl_up(d->N, 32) / 32;
    ep.z8 = d->z8; ep.z8e = d->z8e; ep.ldz8 = nl_up(d->N, 32); ep.ldz8e = ep.ldz8 / 32;
    const bool rows = nl_forward_rows(d);
    // the codes of x come out of the product's own tiles; fp32's are split there, and few rows have no tiles: a pass of their own
    const bool codes = d->x8 && d->dtype != NL_DT_F32 && !rows;
    if (d->x8 && !codes && !w.dry) {
        w.rc = nl_mx8_encode(d->x, d->ldx, d->M, d->K, d->dtype, d->x8, d->x8e, w.st);
        if (w.rc != NL_OK) return;
    }
    if (rows) {
        if (!w.dry) NL_WITH_DTYPE(d->dtype, w.rc = d->M <= ROWS_MOST ? nl_launch_rows<DT, false>(d, ep, w.st) : nl_launch_rows<DT, true>(d, ep, w.st));
        return;
    }
    const NlPacked x = nl_packed(w, d->x, nullptr, d->M, d->K, d->ldx, d->dtype, d->dtype), wt = nl_weight(w, d, d->M, d->N, d->K, 0);
    nl_pack(w, d->dtype);
    if (nl_forward_streams(d)) nl_stream(w, x, wt, false, d->M, d->N, d->K, ep, d->x8, d->x8e, NlDz{}, 0, 0);
    else nl_product(w, x, wt, codes ? 4 : 0, d->M, d->N, d->K, ep, d->x8, d->x8e, nullptr, false);
}

// dz = gy act'(z) in 16 bits is a second rounding of half a step besides the gradients' own (1.41 times the error of one, 1.45 with z kept in the type, whose rounding costs the bias'
// gradient 5 %; with few results up to 1.9 times).  Where the
// products are short, and launches are what the pass takes, dz stays in fp32 and the products run as fp32's do (2^22 multiplications in either, both products, bf16: 18.5
// instead of 13.7 us of a pass that takes 70 from autograd; 2^25 in either: 21 instead of 15.5).
#define NL_WIDE_MOST (1LL << 23)
static bool nl_wide(const NlLinear* d)
{
    return d->dtype != NL_DT_F32 && (d->act == NL_ACT_GELU || d->act == NL_ACT_SILU) && (double)d->M * d->N * d->K <= (double)NL_WIDE_MOST;
}

static bool nl_backward_streams(const NlLinear* d)
{
    return d->gx && !nl_wide(d) && nl_streams(d->M, d->N, d->K, d->dtype, d->act != NL_ACT_NONE) && nl_in_place(d->gy, d->N, d->ldgy, d->dtype) && (d->K & 7) == 0;
}

static void nl_backward_run(const NlLinear* d, NlWork& w)
{
    const bool in_place = d->act == NL_ACT_NONE && nl_in_place(d->gy, d->N, d->ldgy, d->dtype);
    const bool products = d->gx || d->gw, wide = nl_wide(d);
    NlPacked dz = {d->gy, d->ldgy, nullptr};
    NlGb gb = {};
    // the streaming data gradient makes dz on its way
    const bool streams = nl_backward_streams(d);
    const int on_its_way = !streams || d->act == NL_ACT_NONE ? 0 : d->act == NL_ACT_RELU ? 1 : d->z8 ? 3 : 2;
    NlDz a = {};
    if (d->gb || (products && !in_place)) {
        a.gy = d->gy; a.ldgy = d->ldgy; a.M = d->M; a.N = d->N;
        if (d->act == NL_ACT_RELU) { a.bits = d->bits; a.ldbits = nl_up(d->N, 32) / 32; }
        else if (d->act != NL_ACT_NONE && d->z8) { a.z8 = d->z8; a.z8e = d->z8e; a.ldz8 = nl_up(d->N, 32); a.ldz8e = a.ldz8 / 32; }
        else if (d->act != NL_ACT_NONE) { a.z = d->z; a.ldz = d->N; }
        const int colblocks = (d->N + 255) / 256;
        long long chunks = 2048 / colblocks, most = nl_up(d->M, 16) / 16;       // (16 rows are two per thread)
        chunks = chunks < 1 ? 1 : chunks > most ? most : chunks;
        if (chunks > 32768) chunks = 32768;
        a.rows_per_chunk = nl_up((d->M + chunks - 1) / chunks, 8);
        chunks = on_its_way ? nl_stream_groups(d->M) : (d->M + a.rows_per_chunk - 1) / a.rows_per_chunk;
        if (d->gb) a.part = (float*)w.take(4LL * chunks * d->N);
        if (on_its_way ? d->gw != nullptr : products && !in_place) {
            a.pitch = nl_up(d->N, 8);
            a.dz = w.take(d->M * a.pitch * (wide ? 4 : nl_dtype_size(d->dtype)));
            dz = NlPacked{a.dz, a.pitch, nullptr};
        }
        if (!w.dry && !on_its_way) {
            const dim3 grid(colblocks, (unsigned)chunks);
            NL_WITH_DTYPE(d->dtype, if (d->act == NL_ACT_NONE) hipLaunchKernelGGL((k_linear_dz<DT, NL_ACT_NONE, DT>), grid, dim3(256), 0, w.st, a);
                                    else if (d->act == NL_ACT_RELU) hipLaunchKernelGGL((k_linear_dz<DT, NL_ACT_RELU, DT>), grid, dim3(256), 0, w.st, a);
                                    else if (d->act == NL_ACT_GELU && wide) hipLaunchKernelGGL((k_linear_dz<DT, NL_ACT_GELU, NL_DT_F32>), grid, dim3(256), 0, w.st, a);
                                    else if (d->act == NL_ACT_GELU) hipLaunchKernelGGL((k_linear_dz<DT, NL_ACT_GELU, DT>), grid, dim3(256), 0, w.st, a);
                                    else if (wide) hipLaunchKernelGGL((k_linear_dz<DT, NL_ACT_SILU, NL_DT_F32>), grid, dim3(256), 0, w.st, a);
                                    else hipLaunchKernelGGL((k_linear_dz<DT, NL_ACT_SILU, DT>), grid, dim3(256), 0, w.st, a));
        }
        if (d->gb) gb = NlGb{a.part, d->gb, (int)chunks, d->N, (d->N + 3) / 4};
    }
    NlEpilogue ep = {};
    ep.dt = d->dtype; ep.act = NL_ACT_NONE; ep.ldy = d->K;
    NlPacked wt = {}, x = {};
    const bool codes = d->gw && d->x8 && d->dtype != NL_DT_F32 && !wide;  // (fp32 arithmetic splits its operands: codes are decoded first)
    if (d->gx) wt = nl_weight(w, d, d->M, d->K, d->N, 1);
    if (codes) x = NlPacked{d->x8, nl_up(d->K, 32), d->x8e};
    else if (d->gw) x = d->x8 ? nl_packed(w, d->x8, d->x8e, d->M, d->K, nl_up(d->K, 32), NL_DT_MX8, d->dtype) : nl_packed(w, d->x, nullptr, d->M, d->K, d->ldx, d->dtype, d->dtype);
    nl_pack(w, d->dtype);
    const long long keep = w.used;
    long long most = keep;
    if (d->gx) {
        ep.y = d->gx;
        if (streams) nl_stream(w, NlPacked{d->gy, d->ldgy, nullptr}, wt, true, d->M, d->K, d->N, ep, nullptr, nullptr, a, d->act, on_its_way);
        else nl_product(w, dz, wt, 1, d->M, d->K, d->N, ep, nullptr, nullptr, nullptr, wide);
        most = w.used;
        w.used = keep;                                               // (the second product follows on the stream: it takes the same place)
    }
    if (d->gw) {
        ep.y = d->gw;
        nl_product(w, dz, x, codes ? 3 : 2, d->N, d->K, d->M, ep, nullptr, nullptr, &gb, wide);
    }
    if (gb.blocks && !w.dry) NL_WITH_DTYPE(d->dtype, hipLaunchKernelGGL(k_linear_gb<DT>, dim3(gb.blocks), dim3(256), 0, w.st, gb));
    if (w.used < most) w.used = most;
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
        if ((!d->z8) != (!d->z8e) || (!d->x8) != (!d->x8e)) return NL_ERR_INVALID_ARG;
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
    NlWork w = {};
    w.dry = true;
    if (backward) nl_backward_run(d, w); else nl_forward_run(d, w);
    return w.rc == NL_OK ? w.used : -1;
}

int nl_linear_streams(const NlLinear* d, int backward)
{
    if (nl_linear_check(d, backward) != NL_OK) return -1;
    return d->M > 0 && (backward ? nl_backward_streams(d) : nl_forward_streams(d));
}

static int nl_linear_run(const NlLinear* d, int backward, void* stream)
{
    const long long need = nl_linear_workspace(d, backward);
    if (need < 0 || (need > 0 && (!d->ws || d->ws_bytes < need || ((uintptr_t)d->ws & 255)))) return NL_ERR_INVALID_ARG;
    NlWork w = {};
    w.base = (char*)d->ws; w.st = (hipStream_t)stream;
    if (backward) nl_backward_run(d, w); else nl_forward_run(d, w);
    if (w.rc != NL_OK) return w.rc;
    NL_LAUNCH_CHECK();
    return NL_OK;
}

int nl_linear_forward(const NlLinear* d, void* stream)
{
    if (nl_linear_check(d, 0) != NL_OK) return NL_ERR_INVALID_ARG;
    if (d->M == 0) return NL_OK;
    return nl_linear_run(d, 0, stream);
}

int nl_linear_backward(const NlLinear* d, void* stream)
{
    if (nl_linear_check(d, 1) != NL_OK) return NL_ERR_INVALID_ARG;
    if (d->M == 0) {
        const int es = nl_dtype_size(d->dtype);
        hipStream_t st = (hipStream_t)stream;
        if (d->gw) hipLaunchKernelGGL(k_linear_zero, dim3(256), dim3(256), 0, st, (unsigned char*)d->gw, (long long)d->N * d->K * es);
        if (d->gb) hipLaunchKernelGGL(k_linear_zero, dim3(4), dim3(256), 0, st, (unsigned char*)d->gb, (long long)d->N * es);
        NL_LAUNCH_CHECK();
        return NL_OK;
    }
    return nl_linear_run(d, 1, stream);
}

}  // extern "C"

// nl_embedding.hip -- embedding lookup with scaling and its gradient by sorted ids (include/nerfloam_hip.h nl_embedding_*).
//
// Reference behaviour: F.embedding of the voxels' corner rows and the weighted sum over the eight corners (/root/reference/src/variations/render_helpers.py:40-89);
// torch's embedding backward adds with atomics.  Here the lookups are sorted by id (a stable radix sort, eight bits a pass) and a row's gradient is a sum over
// neighbouring entries in ascending position: pieces of a fixed number of entries, the pieces of a row that spans several joined in order, level by level.
#include "nl_layers.h"

// Sorted entries per run-summing group: 16 while that leaves at most EMB_THREADS threads of eight columns, so that there are enough of them, else 64, so that there
// are fewer pieces (table's gradient, bf16: 16384 lookups x 1024 50 us with 16, 58 with 64; 2.1 M x 16 135, 142; 262144 x 256 98, 86; 131072 x 1024 160, 143).
// Pieces of a row that crosses such chunks are joined in blocks of EMB_BLOCK neighbours, level by level.
#define EMB_CHUNK_FEW 16
#define EMB_CHUNK_MANY 64
#define EMB_THREADS (1 << 18)
#define EMB_BLOCK 64
#define EMB_BATCH 8             // rows in flight together
// A sorting pass takes 1024 keys a workgroup (4 waves x 4 rounds x 64 lanes) up to RS_FEW keys, else 4096 and puts them in order in LDS first, so that what it writes
// lies in runs of 16 keys on average (2.1 M keys, a pass: 18 us and 5 for the scan, 40 and 14 in workgroups of 1024).  There the weights of bags move along: 7 us a
// pass, and the sums fetch a line of 128 bytes less per lookup (2.1 M x 16 bf16: 43 us instead of 69).  Whole gradient in workgroups of 4096 / 1024: 2.1 M weighted lookups x 16
// 135 / 205 us, 131072 lookups x 256 77 / 57, 32768 60 / 40: RS_FEW lies below where they cross.  Up to RS_FEW_BLOCKS workgroups the scatter sums the histograms
// itself: a launch less per pass.
#define RS_FEW 65536
#define RS_FEW_BLOCKS 64
#define RS_SMALL 4096           // up to here one workgroup sorts everything in LDS: one launch instead of three per pass

__device__ __forceinline__ long long emb_id(const void* ids, int id64, long long i) { return id64 ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i]; }

// VEC neighbouring columns of a row as fp32 (VEC 1, 4, 8, at most D).  Where VEC does not divide D the last thread of a row takes the row's last VEC columns: what two
// threads have both compute alike (27525 bags of two rows of 733 fp16: forward 50 us, gradients 76 and 24; element by element 91, 104 and 40)
template <int VEC> struct EmbVec { float v[VEC]; };
template <int VEC, int DT>
__device__ __forceinline__ EmbVec<VEC> emb_load(const void* p, long long i)
{
    EmbVec<VEC> o;
    if constexpr (VEC == 1) o.v[0] = nl_load_elem<DT>(p, i);
    else if constexpr (VEC == 8) nl_load8<DT>(o.v, p, i, 8);
    else {
        const nl_f32x4 a = nl_load4<DT>(p, i);
#pragma unroll
        for (int j = 0; j < 4; j++) o.v[j] = a[j];
    }
    return o;
}
template <int VEC, int DT>
__device__ __forceinline__ void emb_store(void* p, long long i, const EmbVec<VEC>& a)
{
    if constexpr (VEC == 1) nl_store_elem<DT>(p, i, a.v[0]);
    else if constexpr (VEC == 8) nl_store8<DT>(p, i, a.v, 8);
    else nl_store4<DT>(p, i, nl_f32x4{a.v[0], a.v[1], a.v[2], a.v[3]});
}

// VEC neighbouring columns from a byte offset into a table of less than 2 GB; an offset from 2^31 on reads zeros
template <int VEC, int DT>
__device__ __forceinline__ EmbVec<VEC> emb_fetch(__amdgpu_buffer_rsrc_t r, unsigned at)
{
    EmbVec<VEC> o;
    if constexpr (VEC == 4 && DT != NL_DT_F32) {
        const nl_s16x4 u = __builtin_bit_cast(nl_s16x4, __builtin_amdgcn_raw_buffer_load_b64(r, (int)at, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; j++) o.v[j] = DT == NL_DT_BF16 ? nl_bf2f((unsigned short)u[j]) : nl_h2f((unsigned short)u[j]);
    } else {
        const nl_i32x4 w = __builtin_bit_cast(nl_i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0));
        if constexpr (DT == NL_DT_F32) {
#pragma unroll
            for (int j = 0; j < VEC; j++) o.v[j] = __int_as_float(w[j]);
        } else nl_unraw8<DT>(o.v, NlRaw8<DT>{{w}});
    }
    return o;
}

// One group of `lanes` threads (a power of two, at most 256) per output row.  The ids of a bag are read BAG at a time and their rows fetched together: what bounds
// a small row is the way id -> row, once per batch instead of once per lookup.
// EIGHT: bags of eight 32-bit ids and weights, both 16-byte aligned (a voxel's corners).  Two neighbouring threads load half of them each and exchange them, past the
// caches that the table's rows should stay in, as the results are stored: 262144 rows of 16 bf16 from a table of 1.7 MB 11.5 us on the same inputs again and again, 14.4 on
// inputs that change; with every thread loading all eight through the caches 13.5 (from cold ones 16.5, 21.3).  Of it 3.4 us are the streams; the rest is 2.1 M lookups of 32 bytes that move a line of 128 from L2 to L1 each.
// The table is below 2 GB: 32-bit offsets, and an id without a row reads zeros from behind the buffer's range.
template <int DT, int VEC, int BAG, bool EIGHT>
__global__ __launch_bounds__(256) void k_emb_forward(const void* __restrict__ table, long long V, int D, const void* __restrict__ ids, int id64,
                                                     const float* __restrict__ weights, long long M, int bag, float scale, void* __restrict__ out, int lanes)
{
    const int log2 = __builtin_ctz(lanes);                            // (a division costs more than the rest of a short row's address)
    const long long m = (nl_block() << (8 - log2)) + (threadIdx.x >> log2);
    if (m >= M) return;
    const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc((void*)table, 0, 0x7FFFFFF0, 0x00020000);
    nl_i32x4 i8[2];
    nl_f32x4 w8[2];
    if (EIGHT) {                                                      // (a group's threads all are here: they exchange before some have no columns)
        const bool second = threadIdx.x & 1;
        const nl_i32x4 mi = __builtin_nontemporal_load(reinterpret_cast<const nl_i32x4*>(ids) + 2 * m + second);
        const nl_f32x4 mw = __builtin_nontemporal_load(reinterpret_cast<const nl_f32x4*>(weights) + 2 * m + second);
        nl_i32x4 oi;
        nl_f32x4 ow;
#pragma unroll
        for (int j = 0; j < 4; j++) {                                 // the neighbour's (lanes 1 0 3 2)
            oi[j] = __builtin_amdgcn_mov_dpp(mi[j], 0xB1, 0xF, 0xF, true);
            ow[j] = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(mw[j]), 0xB1, 0xF, 0xF, true));
        }
        i8[0] = second ? oi : mi; i8[1] = second ? mi : oi;
        w8[0] = second ? ow : mw; w8[1] = second ? mw : ow;
    }
    for (int d0 = (threadIdx.x & (lanes - 1)) * VEC; d0 < D; d0 += lanes * VEC) {
        const int d = d0 < D - VEC ? d0 : D - VEC;
        EmbVec<VEC> acc = {};
        for (int k0 = 0; k0 < bag; k0 += BAG) {
            long long id[BAG];
            float w[BAG];
            EmbVec<VEC> r[BAG];
#pragma unroll
            for (int k = 0; k < BAG; k++) {
                if constexpr (EIGHT) {
                    const unsigned i = (unsigned)i8[k >> 2][k & 3];
                    r[k] = emb_fetch<VEC, DT>(rows, i < (unsigned)V ? (i * (unsigned)D + d) * (DT == NL_DT_F32 ? 4 : 2) : 0x80000000u);
                    w[k] = i < (unsigned)V ? w8[k >> 2][k & 3] : 0.0f;
                    continue;
                }
                const bool in = k0 + k < bag;
                id[k] = in ? emb_id(ids, id64, m * bag + k0 + k) : -1;
                w[k] = in && weights ? weights[m * bag + k0 + k] : 1.0f;
            }
#pragma unroll
            for (int k = 0; k < BAG; k++) {
                if (EIGHT) break;
                const bool in = id[k] >= 0 && id[k] < V;
                r[k] = emb_load<VEC, DT>(table, (in ? id[k] : 0) * D + d);
                if (!in) {                                            // no row: its place in memory may hold anything
#pragma unroll
                    for (int j = 0; j < VEC; j++) r[k].v[j] = 0.0f;
                    w[k] = 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < BAG; k++)
#pragma unroll
                for (int j = 0; j < VEC; j++) acc.v[j] = __builtin_fmaf(w[k], r[k].v[j], acc.v[j]);
            if (EIGHT) break;
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) acc.v[j] *= scale;
        if constexpr (EIGHT && VEC == 8) {
            nl_s16x8 u;
#pragma unroll
            for (int j = 0; j < 8; j++) u[j] = (short)(DT == NL_DT_BF16 ? nl_f2bf(acc.v[j]) : nl_f2h(acc.v[j]));
            __builtin_nontemporal_store(u, reinterpret_cast<nl_s16x8*>((unsigned short*)out + m * D + d));
        } else emb_store<VEC, DT>(out, m * D + d, acc);
    }
}
template <int VEC> static void emb_forward(dim3 grid, hipStream_t st, const void* table, long long V, int D, int dt, const void* ids, int id64, const float* weights, long long M, int bag,
                                           float scale, void* out, int lanes)
{
    const bool eight = VEC > 1 && lanes > 1 && bag == 8 && weights && !id64 && D % VEC == 0 && (((uintptr_t)ids | (uintptr_t)weights | (uintptr_t)table | (uintptr_t)out) & 15) == 0 && V * D * nl_dtype_size(dt) <= 0x7FFFFFF0;
    NL_WITH_DTYPE(dt, if (bag == 1) hipLaunchKernelGGL((k_emb_forward<DT, VEC, 1, false>), grid, dim3(256), 0, st, table, V, D, ids, id64, weights, M, bag, scale, out, lanes);
                      else if (eight) hipLaunchKernelGGL((k_emb_forward<DT, VEC, 8, (VEC > 1)>), grid, dim3(256), 0, st, table, V, D, ids, id64, weights, M, bag, scale, out, lanes);
                      else hipLaunchKernelGGL((k_emb_forward<DT, VEC, 8, false>), grid, dim3(256), 0, st, table, V, D, ids, id64, weights, M, bag, scale, out, lanes));
}

// g_weights[i,k] = scale <g[i], table[ids[i,k]]>: one group of at most 64 lanes per lookup (2.1 M lookups of 16 bf16: 18 us, 32768 of 1024: 17 us; a line of 128 bytes per
// short row, the rows' bytes for long ones)
template <int DT, int VEC>
__global__ __launch_bounds__(256) void k_emb_gweights(const void* __restrict__ table, long long V, int D, const void* __restrict__ ids, int id64, long long L,
                                                      int bag, float scale, const void* __restrict__ g, float* __restrict__ gw, int lanes)
{
    const int per = 256 / lanes, grp = threadIdx.x / lanes;
    const long long i = nl_block() * per + grp;
    if (i >= L) return;
    const long long id = emb_id(ids, id64, i);
    float s = 0.0f;
    if (id >= 0 && id < V)
        for (int d0 = (threadIdx.x & (lanes - 1)) * VEC; d0 < D; d0 += lanes * VEC) {
            const int d = d0 < D - VEC ? d0 : D - VEC;
            const EmbVec<VEC> a = emb_load<VEC, DT>(g, (i / bag) * D + d), b = emb_load<VEC, DT>(table, id * D + d);
#pragma unroll
            for (int j = 0; j < VEC; j++) s += d + j >= d0 ? a.v[j] * b.v[j] : 0.0f;
        }
    for (int off = lanes >> 1; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & (lanes - 1)) == 0) gw[i] = s * scale;
}

// ---- stable radix sort of (id, position), eight bits a pass ----
// The first pass reads the ids themselves: an id that selects no row sorts behind all others (key V).
struct RsArgs {
    const void* ids; int id64; long long V;            // first pass
    const unsigned* keys; const unsigned* pos;         // later passes
    unsigned* out_keys; unsigned* out_pos;
    const float* w; float* out_w;                      // weights that go along (staged passes; null: none)
    int* hist;                                         // [nblk][256], then (k_rs_scan) its exclusive sums over the blocks
    int* totals;                                       // [256]; null: every workgroup of the scatter sums what is in front of it
    int L, nblk, shift;                                // nblk workgroups of 256 ROUNDS keys
    unsigned* zero; long long zero_words;              // first pass: the launch's workgroups behind the sorting ones clear these (the gradient's rows)
};
__device__ __forceinline__ bool rs_zero(const RsArgs& a, int sorting)
{
    if ((int)blockIdx.x < sorting) return false;
    const long long step = (long long)(gridDim.x - sorting) * blockDim.x;
    for (long long i = (long long)(blockIdx.x - sorting) * blockDim.x + threadIdx.x; i < a.zero_words; i += step) a.zero[i] = 0;
    return true;
}
__device__ __forceinline__ unsigned rs_key(const RsArgs& a, int i)
{
    if (!a.ids) return a.keys[i];
    const long long id = emb_id(a.ids, a.id64, i);
    return id < 0 || id >= a.V ? (unsigned)a.V : (unsigned)id;
}
template <int ROUNDS>
__global__ __launch_bounds__(256) void k_rs_hist(RsArgs a)
{
    __shared__ int s_h[256];
    if (rs_zero(a, a.nblk)) return;
    s_h[threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * (256 * ROUNDS);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = base + r * 256 + threadIdx.x;
        if (i < a.L) atomicAdd(&s_h[rs_key(a, i) >> a.shift & 255], 1);       // (whole numbers: the order does not matter)
    }
    __syncthreads();
    a.hist[blockIdx.x * 256 + threadIdx.x] = s_h[threadIdx.x];
}
// one workgroup per digit: exclusive sums of the digit's column of the histogram, and its total
__global__ __launch_bounds__(256) void k_rs_scan(RsArgs a)
{
    __shared__ int s_w[4];
    if (rs_zero(a, 256)) return;
    int* col = a.hist + blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int run = 0;
    for (int b = 0; b < a.nblk; b += 256) {
        const int i = b + threadIdx.x;
        const int v = i < a.nblk ? col[(long long)i * 256] : 0;
        int s = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(s, off); if (lane >= off) s += t; }
        if (lane == 63) s_w[wave] = s;
        __syncthreads();
        int before = run;
        for (int w = 0; w < wave; w++) before += s_w[w];
        if (i < a.nblk) col[(long long)i * 256] = before + s - v;
        run += s_w[0] + s_w[1] + s_w[2] + s_w[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.totals[blockIdx.x] = run;
}
template <int ROUNDS>
__global__ __launch_bounds__(256) void k_rs_scatter(RsArgs a)
{
    constexpr bool STAGE = ROUNDS > 4;
    __shared__ int s_cnt[4][256], s_base[256], s_w[4];
    __shared__ unsigned s_key[STAGE ? 256 * ROUNDS : 1], s_pos[STAGE ? 256 * ROUNDS : 1];
    __shared__ float s_wt[STAGE ? 256 * ROUNDS : 1];
    if (rs_zero(a, a.nblk)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d0 = threadIdx.x;
    // where the digit begins: sums of the totals in front of it
    {
        int v = 0, front = 0;
        if (a.totals) { v = a.totals[d0]; front = a.hist[(long long)blockIdx.x * 256 + d0]; }
        else
#pragma unroll 8
            for (int b = 0; b < a.nblk; b++) { const int c = a.hist[(long long)b * 256 + d0]; front += b < (int)blockIdx.x ? c : 0; v += c; }
        int s = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(s, off); if (lane >= off) s += t; }
        if (lane == 63) s_w[wave] = s;
        __syncthreads();
        for (int w = 0; w < wave; w++) s += s_w[w];
        s_base[d0] = s - v + front;
    }
#pragma unroll
    for (int w = 0; w < 4; w++) s_cnt[w][d0] = 0;
    __syncthreads();
    // a wave ranks its neighbouring keys, 64 at a time: lanes with the same digit find each other by eight ballots
    unsigned key[ROUNDS], rank[ROUNDS];
    const int tile = blockIdx.x * (256 * ROUNDS), first = tile + wave * (64 * ROUNDS);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = first + r * 64 + lane;
        const bool in = i < a.L;
        key[r] = in ? rs_key(a, i) : 0;
        const unsigned d = key[r] >> a.shift & 255;
        unsigned long long same = __ballot(in);
#pragma unroll
        for (int b = 0; b < 8; b++) { const unsigned long long m = __ballot(d >> b & 1); same &= (d >> b & 1) ? m : ~m; }
        const unsigned long long below = same & ((1ull << lane) - 1);
        const int seen = s_cnt[wave][d];
        rank[r] = seen + __popcll(below);
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) s_cnt[wave][d] = seen + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    if constexpr (STAGE) {
        // in LDS a digit's keys begin behind those of the smaller digits of the tile; from there on they lie as they will in memory
        int total = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) total += s_cnt[w][d0];
        int s = total;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(s, off); if (lane >= off) s += t; }
        if (lane == 63) s_w[wave] = s;
        __syncthreads();
        for (int w = 0; w < wave; w++) s += s_w[w];
        int before = s - total;
        s_base[d0] -= before;                                         // place in memory minus place in the tile
#pragma unroll
        for (int w = 0; w < 4; w++) { const int c = s_cnt[w][d0]; s_cnt[w][d0] = before; before += c; }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const int i = first + r * 64 + lane;
            if (i >= a.L) continue;
            const unsigned to = s_cnt[wave][key[r] >> a.shift & 255] + rank[r];
            s_key[to] = key[r];
            s_pos[to] = a.ids ? (unsigned)i : a.pos[i];
            if (a.w) s_wt[to] = a.w[i];
        }
        __syncthreads();
        const int n = a.L - tile < 256 * ROUNDS ? a.L - tile : 256 * ROUNDS;
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += 256) {
            const unsigned k = s_key[i];
            const int to = s_base[k >> a.shift & 255] + i;
            a.out_keys[to] = k;
            a.out_pos[to] = s_pos[i];
            if (a.w) a.out_w[to] = s_wt[i];
        }
    } else {
        int before = s_base[d0];
#pragma unroll
        for (int w = 0; w < 4; w++) { const int c = s_cnt[w][d0]; s_cnt[w][d0] = before; before += c; }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const int i = first + r * 64 + lane;
            if (i >= a.L) continue;
            const unsigned to = s_cnt[wave][key[r] >> a.shift & 255] + rank[r];
            a.out_keys[to] = key[r];
            a.out_pos[to] = a.ids ? (unsigned)i : a.pos[i];
        }
    }
}

// All passes of at most RS_SMALL keys by one workgroup of 16 waves, keys and positions in LDS (512 keys below 1000, two passes: 8.6 us, latency of barriers and LDS)
__global__ __launch_bounds__(1024) void k_rs_small(RsArgs a, int passes)
{
    constexpr int R = RS_SMALL / 1024;
    __shared__ unsigned s_key[RS_SMALL], s_pos[RS_SMALL];
    __shared__ int s_cnt[16][256], s_w[4];
    if (rs_zero(a, 1)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave * (64 * R);
    unsigned key[R], pos[R], rank[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = first + r * 64 + lane;
        key[r] = i < a.L ? rs_key(a, i) : 0; pos[r] = i;
    }
    for (int p = 0; p < passes; p++) {
        const int shift = 8 * p;
        for (int i = threadIdx.x; i < 16 * 256; i += 1024) s_cnt[0][i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const bool in = first + r * 64 + lane < a.L;
            const unsigned d = key[r] >> shift & 255;
            unsigned long long same = __ballot(in);
#pragma unroll
            for (int b = 0; b < 8; b++) { const unsigned long long m = __ballot(d >> b & 1); same &= (d >> b & 1) ? m : ~m; }
            const unsigned long long below = same & ((1ull << lane) - 1);
            const int seen = s_cnt[wave][d];
            rank[r] = seen + __popcll(below);
            __builtin_amdgcn_wave_barrier();
            if (in && below == 0) s_cnt[wave][d] = seen + __popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        int total = 0, incl = 0;
        if (threadIdx.x < 256) {
            for (int w = 0; w < 16; w++) total += s_cnt[w][threadIdx.x];
            incl = total;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(incl, off); if (lane >= off) incl += t; }
            if (lane == 63) s_w[wave] = incl;
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            int before = incl - total;
            for (int w = 0; w < wave; w++) before += s_w[w];
            for (int w = 0; w < 16; w++) { const int c = s_cnt[w][threadIdx.x]; s_cnt[w][threadIdx.x] = before; before += c; }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++)
            if (first + r * 64 + lane < a.L) {
                const unsigned to = s_cnt[wave][key[r] >> shift & 255] + rank[r];
                s_key[to] = key[r]; s_pos[to] = pos[r];
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int i = first + r * 64 + lane;
            if (i < a.L) { key[r] = s_key[i]; pos[r] = s_pos[i]; }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = first + r * 64 + lane;
        if (i < a.L) { a.out_keys[i] = key[r]; a.out_pos[i] = pos[r]; }
    }
}

// ---- sums of neighbouring entries with one key ----
// k_emb_sum: a group of `lanes` threads walks one chunk of the sorted list.  A run of equal keys that begins and ends inside the chunk is a finished row of the
// gradient; a run that a chunk border cuts becomes a piece.  A chunk leaves its first and last key and at most two pieces: slot 0 of its first run, slot 1 of its last.
// k_emb_join: the pieces of a row stand in neighbouring chunks, slot 1 (or the slot 0 of a chunk that is one run) of the first, then slots 0.  A group per chunk sums
// the row that begins there, within a block of EMB_BLOCK chunks; a row that leaves the block becomes a piece of the block, and blocks are the next level's chunks.
// What bounds both is the way position -> row: EMB_BATCH rows are fetched together.  32768 lookups x 1024 bf16: sums 21 us (67 MB read and up to 67 written: at the rate of
// a copy), joins 8 us a level; 2.1 M x 16: sums 43 us, of every line of 128 bytes that an XCD's L2 fetches 32 are used.
struct EmbPieces { unsigned* keys; unsigned char* any; float* piece; };        // [n][2] keys (first, last), [n][2] flags, [n][2][D] fp32
struct EmbSum {
    const unsigned* keys; const unsigned* pos; const void* g; const float* weights; bool sorted;      // sorted: the weights lie as the keys do
    EmbPieces out; void* g_table; long long V;
    int L, D, bag, chunk; float scale;
};
template <int DT, int VEC>
__global__ __launch_bounds__(256) void k_emb_sum(EmbSum a, int lanes)
{
    const int per = 256 / lanes, chunk = (int)(blockIdx.x * per + threadIdx.x / lanes);
    const long long s0 = (long long)chunk * a.chunk;
    if (s0 >= a.L) return;
    const int s = (int)s0, e = s + a.chunk < a.L ? s + a.chunk : a.L;
    const int d0 = (int)(blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * VEC, d = d0 < a.D - VEC ? d0 : a.D - VEC;
    const bool lead = d0 == 0, col = d0 < a.D;
    const unsigned k_first = a.keys[s], k_last = a.keys[e - 1];
    const bool open_l = s > 0 && a.keys[s - 1] == k_first, open_r = e < a.L && a.keys[e] == k_last;
    EmbVec<VEC> acc = {};
    bool any0 = false, any1 = false, in_first = true;
    unsigned cur = k_first;
    // the run of `cur` ends, at the chunk's end or before it
    auto flush = [&](bool at_end) {
        if (cur >= a.V) return;
        if (!((in_first && open_l) || (at_end && open_r))) { if (col) emb_store<VEC, DT>(a.g_table, (long long)cur * a.D + d, acc); return; }
        if (in_first) any0 = true; else any1 = true;
        if (col) emb_store<VEC, NL_DT_F32>(a.out.piece, (2LL * chunk + (in_first ? 0 : 1)) * a.D + d, acc);
    };
    unsigned nkey[EMB_BATCH], npos[EMB_BATCH];
    int at[EMB_BATCH];
    auto look = [&](int j0) {                                         // keys and positions of the next batch; behind the chunk's end its last entry again
#pragma unroll
        for (int b = 0; b < EMB_BATCH; b++) {
            const int j = j0 + b < e ? j0 + b : e - 1;
            nkey[b] = a.keys[j];
            npos[b] = a.pos[j];
            at[b] = j;
        }
    };
    look(s);
    for (int j0 = s; j0 < e; j0 += EMB_BATCH) {
        unsigned key[EMB_BATCH];
        float w[EMB_BATCH];
        EmbVec<VEC> r[EMB_BATCH];
#pragma unroll
        for (int b = 0; b < EMB_BATCH; b++) {
            // every row is fetched, also where it does not count (a load under a condition is waited for where the branch ends)
            key[b] = nkey[b];
            w[b] = a.weights ? a.scale * a.weights[a.sorted ? (unsigned)at[b] : npos[b]] : a.scale;
            r[b] = emb_load<VEC, DT>(a.g, (long long)(npos[b] / (unsigned)a.bag) * a.D + (col ? d : 0));
        }
        if (j0 + EMB_BATCH < e) look(j0 + EMB_BATCH);
#pragma unroll
        for (int b = 0; b < EMB_BATCH; b++) {
            if (key[b] != cur) {
                flush(false);
                acc = EmbVec<VEC>{};
                in_first = false; cur = key[b];
            }
            if (j0 + b < e)
#pragma unroll
                for (int q = 0; q < VEC; q++) acc.v[q] += w[b] * r[b].v[q];
        }
    }
    flush(true);
    if (lead && a.out.keys) {
        a.out.keys[2 * chunk] = k_first; a.out.keys[2 * chunk + 1] = k_last;
        a.out.any[2 * chunk] = any0; a.out.any[2 * chunk + 1] = any1;
    }
}

// n chunks of one level; out.keys null: they are one block, nothing leaves it
template <int DT, int VEC>
__global__ __launch_bounds__(256) void k_emb_join(EmbPieces in, EmbPieces out, int n, int D, void* g_table, int lanes)
{
    const int per = 256 / lanes, c = (int)(blockIdx.x * per + threadIdx.x / lanes);
    if (c >= n) return;
    const int d0 = (int)(blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * VEC, d = d0 < D - VEC ? d0 : D - VEC;
    const bool lead = d0 == 0, col = d0 < D;
    const int block = c / EMB_BLOCK, b0 = block * EMB_BLOCK, b1 = b0 + EMB_BLOCK < n ? b0 + EMB_BLOCK : n;
    const unsigned block_first = in.keys[2 * b0], block_last = in.keys[2 * b1 - 1];
    const unsigned first = in.keys[2 * c], last = in.keys[2 * c + 1];
    const bool open_l = c > 0 && in.keys[2 * c - 1] == first;
    const bool any0 = in.any[2 * c], any1 = in.any[2 * c + 1];
    if (out.keys && lead && c == b0) {
        const bool from_l = b0 > 0 && in.keys[2 * b0 - 1] == block_first, to_r = b1 < n && in.keys[2 * b1] == block_last, one = block_first == block_last;
        out.keys[2 * block] = block_first; out.keys[2 * block + 1] = block_last;
        out.any[2 * block] = any0 && (from_l || (one && to_r));
        out.any[2 * block + 1] = !one && to_r && in.any[in.keys[2 * b1 - 2] == block_last ? 2 * b1 - 2 : 2 * b1 - 1];
    }
    // at most two sums begin here: of the first run (it comes from the left and the block begins, or the chunk is one run and the row begins with it), of the last one
#pragma unroll 1
    for (int which = 0; which < 2; which++) {
        const bool mine = which == 0 ? any0 && (open_l ? c == b0 : first == last) : any1;
        if (!mine) continue;
        const unsigned key = which == 0 ? first : last;
        // how far the row goes: the chunks behind c whose first key is its key (keys are sorted: they follow each other), eight looked at together
        int more = 0;
        for (bool full = true; full;) {
            bool same[EMB_BATCH];
#pragma unroll
            for (int i = 0; i < EMB_BATCH; i++) { const int j = c + 1 + more + i; same[i] = in.keys[2 * (j < b1 ? j : c)] == key && j < b1; }
#pragma unroll
            for (int i = 0; i < EMB_BATCH; i++) { full = full && same[i]; more += full; }
        }
        const bool goes_on = more > 0 ? in.keys[2 * (c + more) + 1] == key : which == 1 || first == last;
        EmbVec<VEC> acc = emb_load<VEC, NL_DT_F32>(in.piece, (2LL * c + which) * D + (col ? d : 0));
        for (int j0 = 0; j0 < more; j0 += EMB_BATCH) {
            EmbVec<VEC> r[EMB_BATCH];
#pragma unroll
            for (int b = 0; b < EMB_BATCH; b++) r[b] = emb_load<VEC, NL_DT_F32>(in.piece, 2LL * (c + 1 + (j0 + b < more ? j0 + b : more - 1)) * D + (col ? d : 0));
#pragma unroll
            for (int b = 0; b < EMB_BATCH; b++)
                if (j0 + b < more)
#pragma unroll
                    for (int q = 0; q < VEC; q++) acc.v[q] += r[b].v[q];
        }
        const bool from_left = which == 0 && open_l, to_right = goes_on && c + more + 1 == b1 && b1 < n && in.keys[2 * b1] == key;
        if (!from_left && !to_right) { if (col) emb_store<VEC, DT>(g_table, (long long)key * D + d, acc); }
        else if (col) emb_store<VEC, NL_DT_F32>(out.piece, (2LL * block + (key == block_first ? 0 : 1)) * D + d, acc);
    }
}

__global__ __launch_bounds__(256) void k_emb_zero(unsigned* p, long long words)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < words; i += (long long)gridDim.x * 256) p[i] = 0;
}
__global__ void k_emb_zero_tail(unsigned short* p) { *p = 0; }

// ---- host ----
#define EMB_MAX_LOOKUPS ((1LL << 30) - EMB_CHUNK_MANY)      // below 2^24 chunks: a launch with a workgroup for each has fewer than 2^32 threads
struct EmbPlan { bool carry; int L, nblk, rounds, passes, chunk, levels; long long keys, hist, key_l[2], any_l[2], piece_l[2], total; };      // levels: launches of k_emb_join
static EmbPlan emb_plan(long long V, int D, long long L, int bag)
{
    EmbPlan p = {};
    p.L = (int)L;
    p.rounds = L <= RS_FEW ? 4 : 16;
    p.nblk = (int)((L + 256 * p.rounds - 1) / (256 * p.rounds));
    p.passes = 1;
    while (p.passes < 4 && (V >> (8 * p.passes)) != 0) p.passes++;
    p.keys = nl_up(4 * L, 256);
    p.hist = nl_up(4LL * 256 * p.nblk + 1024, 256);
    p.carry = bag > 1 && p.rounds > 4;                                // (a weight fetched by position moves a line of 128 bytes)
    p.total = (p.carry ? 6 : 4) * p.keys + p.hist;
    p.chunk = L / EMB_CHUNK_FEW * ((D + 7) / 8) <= EMB_THREADS ? EMB_CHUNK_FEW : EMB_CHUNK_MANY;
    for (long long n = (L + p.chunk - 1) / p.chunk; n > 1; n = (n + EMB_BLOCK - 1) / EMB_BLOCK) {        // levels take two buffers in turn
        if (p.levels < 2) {
            const int i = p.levels;
            p.key_l[i] = nl_up(8 * n, 256); p.any_l[i] = nl_up(2 * n, 256); p.piece_l[i] = nl_up(8 * n * D, 256);
            p.total += p.key_l[i] + p.any_l[i] + p.piece_l[i];
        }
        p.levels++;
    }
    return p;
}
static int emb_lanes(int D, int vec, int most)
{
    int l = 1;
    while (l < most && l * vec < D) l *= 2;
    return l;
}
static int emb_vec(int D, int dt) { return dt != NL_DT_F32 && D >= 8 ? 8 : D >= 4 ? 4 : 1; }
static int emb_check(const void* table, long long V, int D, int dtype, const void* ids, int id64, long long M, int bag)
{
    if (!nl_dtype_ok(dtype) || V < 1 || V > 0x7FFFFFFF || D < 1 || D > (1 << 20) || M < 0 || bag < 1 || M > EMB_MAX_LOOKUPS / bag) return NL_ERR_INVALID_ARG;
    if (M > 0 && (!ids || ((uintptr_t)ids & (id64 ? 7 : 3)))) return NL_ERR_INVALID_ARG;
    if ((uintptr_t)table & (nl_dtype_size(dtype) - 1)) return NL_ERR_INVALID_ARG;
    return NL_OK;
}
static unsigned emb_zero_blocks(long long words, int threads)
{
    const long long b = (words + 8LL * threads - 1) / (8LL * threads);
    return (unsigned)(b < 2048 ? b : 2048);
}
template <int VEC> static void emb_sums(const EmbPlan& p, EmbSum a, const EmbPieces* buf, int dt, hipStream_t st)
{
    const int lanes = emb_lanes(a.D, VEC, 256), per = 256 / lanes;
    const unsigned cols = (unsigned)((a.D + lanes * VEC - 1) / (lanes * VEC));
    int n = (a.L + p.chunk - 1) / p.chunk;
    if (p.levels > 0) a.out = buf[0];
    NL_WITH_DTYPE(dt, hipLaunchKernelGGL((k_emb_sum<DT, VEC>), dim3((n + per - 1) / per, cols), dim3(256), 0, st, a, lanes));
    for (int l = 0; l < p.levels; l++) {
        const EmbPieces out = l + 1 < p.levels ? buf[(l + 1) & 1] : EmbPieces{};
        NL_WITH_DTYPE(dt, hipLaunchKernelGGL((k_emb_join<DT, VEC>), dim3((n + per - 1) / per, cols), dim3(256), 0, st, buf[l & 1], out, n, a.D, a.g_table, lanes));
        n = (n + EMB_BLOCK - 1) / EMB_BLOCK;
    }
}

extern "C" {

long long nl_embedding_workspace(long long V, int D, long long M, int bag)
{
    if (V < 1 || V > 0x7FFFFFFF || D < 1 || D > (1 << 20) || M < 0 || bag < 1 || M > EMB_MAX_LOOKUPS / bag) return -1;
    return M == 0 ? 0 : emb_plan(V, D, M * bag, bag).total;
}

int nl_embedding_forward(const void* table, long long V, int D, int dtype, const void* ids, int id64, const float* weights, long long M, int bag, float scale,
                         void* out, void* stream)
{
    if (emb_check(table, V, D, dtype, ids, id64, M, bag) != NL_OK || !table) return NL_ERR_INVALID_ARG;
    if (M == 0) return NL_OK;
    if (!out || ((uintptr_t)out & (nl_dtype_size(dtype) - 1)) || ((uintptr_t)weights & 3)) return NL_ERR_INVALID_ARG;
    hipStream_t st = (hipStream_t)stream;
    const int vec = emb_vec(D, dtype), lanes = emb_lanes(D, vec, 256), per = 256 / lanes;
    const dim3 grid = nl_blocks((M + per - 1) / per);
    if (vec == 8) emb_forward<8>(grid, st, table, V, D, dtype, ids, id64, weights, M, bag, scale, out, lanes);
    else if (vec == 4) emb_forward<4>(grid, st, table, V, D, dtype, ids, id64, weights, M, bag, scale, out, lanes);
    else emb_forward<1>(grid, st, table, V, D, dtype, ids, id64, weights, M, bag, scale, out, lanes);
    NL_LAUNCH_CHECK();
    return NL_OK;
}

int nl_embedding_backward(const void* table, long long V, int D, int dtype, const void* ids, int id64, const float* weights, long long M, int bag, float scale,
                          const void* g_out, void* g_table, float* g_weights, void* ws, long long ws_bytes, void* stream)
{
    if (emb_check(table, V, D, dtype, ids, id64, M, bag) != NL_OK) return NL_ERR_INVALID_ARG;
    const uintptr_t mis = nl_dtype_size(dtype) - 1;
    if ((M > 0 && !g_out) || ((uintptr_t)g_out & mis) || ((uintptr_t)g_table & 3) || ((uintptr_t)g_weights & 3) || ((uintptr_t)weights & 3) || (g_weights && M > 0 && !table))
        return NL_ERR_INVALID_ARG;
    hipStream_t st = (hipStream_t)stream;
    const long long L = M * bag;
    if (g_table && M > 0 && (!ws || ws_bytes < emb_plan(V, D, L, bag).total || ((uintptr_t)ws & 255))) return NL_ERR_INVALID_ARG;      // (before anything is written)
    if (g_weights && M > 0) {
        const int vec = emb_vec(D, dtype), lanes = emb_lanes(D, vec, 64), per = 256 / lanes;
        const dim3 grid = nl_blocks((L + per - 1) / per);
        if (vec == 8) NL_WITH_DTYPE(dtype, hipLaunchKernelGGL((k_emb_gweights<DT, 8>), grid, dim3(256), 0, st, table, V, D, ids, id64, L, bag, scale, g_out, g_weights, lanes));
        else if (vec == 4) NL_WITH_DTYPE(dtype, hipLaunchKernelGGL((k_emb_gweights<DT, 4>), grid, dim3(256), 0, st, table, V, D, ids, id64, L, bag, scale, g_out, g_weights, lanes));
        else NL_WITH_DTYPE(dtype, hipLaunchKernelGGL((k_emb_gweights<DT, 1>), grid, dim3(256), 0, st, table, V, D, ids, id64, L, bag, scale, g_out, g_weights, lanes));
    }
    if (!g_table) { NL_LAUNCH_CHECK(); return NL_OK; }
    const long long bytes = V * D * nl_dtype_size(dtype);
    if (bytes & 3) hipLaunchKernelGGL(k_emb_zero_tail, dim3(1), dim3(1), 0, st, (unsigned short*)((char*)g_table + bytes - 2));
    if (M == 0) {
        hipLaunchKernelGGL(k_emb_zero, dim3((unsigned)(bytes / 4 < 256 * 2048 ? bytes / 1024 + 1 : 2048)), dim3(256), 0, st, (unsigned*)g_table, bytes / 4);
        NL_LAUNCH_CHECK();
        return NL_OK;
    }
    const EmbPlan p = emb_plan(V, D, L, bag);
    char* w = (char*)ws;
    unsigned* keys[2] = {(unsigned*)w, (unsigned*)(w + p.keys)};
    unsigned* pos[2] = {(unsigned*)(w + 2 * p.keys), (unsigned*)(w + 3 * p.keys)};
    w += 4 * p.keys;
    float* const moved[2] = {(float*)w, (float*)(w + p.keys)};
    const bool carry = p.carry && weights;
    if (p.carry) w += 2 * p.keys;
    RsArgs r = {};
    r.totals = p.nblk <= RS_FEW_BLOCKS ? nullptr : (int*)w; r.hist = (int*)(w + 1024); r.L = p.L; r.nblk = p.nblk; r.V = V;
    w += p.hist;
    // the gradient's rows are cleared beside the first sorting pass, an equal part by each of its launches
    const long long words = bytes / 4, launches = p.nblk <= RS_FEW_BLOCKS ? 2 : 3, part = (words / launches + 63) / 64 * 64;
    if (p.L <= RS_SMALL) {
        r.ids = ids; r.id64 = id64; r.out_keys = keys[(p.passes - 1) & 1]; r.out_pos = pos[(p.passes - 1) & 1];
        r.zero = (unsigned*)g_table; r.zero_words = words;
        hipLaunchKernelGGL(k_rs_small, dim3(1 + emb_zero_blocks(words, 1024)), dim3(1024), 0, st, r, p.passes);
    } else
        for (int i = 0; i < p.passes; i++) {
            r.ids = i == 0 ? ids : nullptr; r.id64 = id64; r.shift = 8 * i;
            r.keys = keys[(i + 1) & 1]; r.pos = pos[(i + 1) & 1]; r.out_keys = keys[i & 1]; r.out_pos = pos[i & 1];
            if (carry) { r.w = i == 0 ? weights : moved[(i + 1) & 1]; r.out_w = moved[i & 1]; }
            for (int k = 0; k < 3; k++) {
                if (k == 1 && p.nblk <= RS_FEW_BLOCKS) continue;
                const long long nth = k == 2 ? launches - 1 : k, z0 = nth * part < words ? nth * part : words, z1 = k == 2 ? words : z0 + part < words ? z0 + part : words;
                r.zero = (unsigned*)g_table + z0; r.zero_words = i == 0 ? z1 - z0 : 0;
                const dim3 grid((k == 1 ? 256 : p.nblk) + emb_zero_blocks(r.zero_words, 256));
                if (k == 1) hipLaunchKernelGGL(k_rs_scan, grid, dim3(256), 0, st, r);
                else if (k == 0 && p.rounds == 4) hipLaunchKernelGGL(k_rs_hist<4>, grid, dim3(256), 0, st, r);
                else if (k == 0) hipLaunchKernelGGL(k_rs_hist<16>, grid, dim3(256), 0, st, r);
                else if (p.rounds == 4) hipLaunchKernelGGL(k_rs_scatter<4>, grid, dim3(256), 0, st, r);
                else hipLaunchKernelGGL(k_rs_scatter<16>, grid, dim3(256), 0, st, r);
            }
        }
    EmbPieces buf[2] = {};
    for (int i = 0; i < 2; i++) {
        buf[i] = EmbPieces{(unsigned*)w, (unsigned char*)(w + p.key_l[i]), (float*)(w + p.key_l[i] + p.any_l[i])};
        w += p.key_l[i] + p.any_l[i] + p.piece_l[i];
    }
    EmbSum a = {};
    a.keys = keys[(p.passes - 1) & 1]; a.pos = pos[(p.passes - 1) & 1]; a.g = g_out; a.weights = carry ? moved[(p.passes - 1) & 1] : weights; a.sorted = carry; a.g_table = g_table; a.V = V; a.L = p.L; a.D = D;
    a.bag = bag; a.scale = scale; a.chunk = p.chunk;
    const int vec = emb_vec(D, dtype);
    if (vec == 8) emb_sums<8>(p, a, buf, dtype, st);
    else if (vec == 4) emb_sums<4>(p, a, buf, dtype, st);
    else emb_sums<1>(p, a, buf, dtype, st);
    NL_LAUNCH_CHECK();
    return NL_OK;
}

}  // extern "C"

// nl_embedding.hip -- embedding lookup with scaling and its gradient by sorted ids (include/nerfloam_hip.h nl_embedding_*).
//
// Reference behaviour: F.embedding of the voxels' corner rows and the weighted sum over the eight corners (/root/reference/src/variations/render_helpers.py:40-89);
// torch's embedding backward adds with atomics.  Here the lookups are sorted by id (a stable radix sort, eight bits a pass) and a row's gradient is a sum over
// neighbouring entries in ascending position: pieces of at most EMB_CHUNK entries, the pieces of a row that spans several joined in order, level by level.
#include "nl_layers.h"

#define EMB_CHUNK 64            // sorted entries per run-summing group
#define RS_TILE 2048            // keys per workgroup of a sorting pass: 4 waves x 8 rounds x 64 lanes
#define RS_ROUNDS (RS_TILE / 256)

__device__ __forceinline__ long long emb_id(const void* ids, int id64, long long i) { return id64 ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i]; }

// VEC neighbouring columns of a row as fp32 (VEC 1, 4, 8; 4 and 8 need D divisible by it)
template <int VEC> struct EmbVec { float v[VEC]; };
template <int VEC>
__device__ __forceinline__ EmbVec<VEC> emb_load(const void* p, long long i, int dt)
{
    EmbVec<VEC> o;
    if (VEC == 1) { o.v[0] = nl_load_elem(p, i, dt); return o; }
#pragma unroll
    for (int h = 0; h < VEC / 4; h++) {
        const nl_f32x4 a = nl_load4(p, i + 4 * h, dt);
#pragma unroll
        for (int j = 0; j < 4; j++) o.v[(4 * h + j) % VEC] = a[j];
    }
    return o;
}
template <int VEC>
__device__ __forceinline__ void emb_store(void* p, long long i, int dt, const EmbVec<VEC>& a)
{
    if (VEC == 1) { nl_store_elem(p, i, dt, a.v[0]); return; }
#pragma unroll
    for (int h = 0; h < VEC / 4; h++) nl_store4(p, i + 4 * h, dt, nl_f32x4{a.v[4 * h % VEC], a.v[(4 * h + 1) % VEC], a.v[(4 * h + 2) % VEC], a.v[(4 * h + 3) % VEC]});
}

// One group of `lanes` threads (a power of two, at most 256) per output row
template <int VEC>
__global__ __launch_bounds__(256) void k_emb_forward(const void* __restrict__ table, long long V, int D, int dt, const void* __restrict__ ids, int id64,
                                                     const float* __restrict__ weights, long long M, int bag, float scale, void* __restrict__ out, int lanes)
{
    const int per = 256 / lanes, grp = threadIdx.x / lanes;
    const long long m = (long long)blockIdx.x * per + grp;
    if (m >= M) return;
    for (int d = (threadIdx.x & (lanes - 1)) * VEC; d < D; d += lanes * VEC) {
        EmbVec<VEC> acc = {};
        for (int k = 0; k < bag; k++) {
            const long long id = emb_id(ids, id64, m * bag + k);
            if (id < 0 || id >= V) continue;
            const float w = weights ? weights[m * bag + k] : 1.0f;
            const EmbVec<VEC> r = emb_load<VEC>(table, id * D + d, dt);
#pragma unroll
            for (int j = 0; j < VEC; j++) acc.v[j] += w * r.v[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) acc.v[j] *= scale;
        emb_store<VEC>(out, m * D + d, dt, acc);
    }
}

// g_weights[i,k] = scale <g[i], table[ids[i,k]]>: one group of at most 64 lanes per lookup
template <int VEC>
__global__ __launch_bounds__(256) void k_emb_gweights(const void* __restrict__ table, long long V, int D, int dt, const void* __restrict__ ids, int id64, long long L,
                                                      int bag, float scale, const void* __restrict__ g, float* __restrict__ gw, int lanes)
{
    const int per = 256 / lanes, grp = threadIdx.x / lanes;
    const long long i = (long long)blockIdx.x * per + grp;
    if (i >= L) return;
    const long long id = emb_id(ids, id64, i);
    float s = 0.0f;
    if (id >= 0 && id < V)
        for (int d = (threadIdx.x & (lanes - 1)) * VEC; d < D; d += lanes * VEC) {
            const EmbVec<VEC> a = emb_load<VEC>(g, (i / bag) * D + d, dt), b = emb_load<VEC>(table, id * D + d, dt);
#pragma unroll
            for (int j = 0; j < VEC; j++) s += a.v[j] * b.v[j];
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
    int* hist;                                         // [256][nblk], then its exclusive sums along a row
    int* totals;                                       // [256]
    int L, nblk, shift;
};
__device__ __forceinline__ unsigned rs_key(const RsArgs& a, int i)
{
    if (!a.ids) return a.keys[i];
    const long long id = emb_id(a.ids, a.id64, i);
    return id < 0 || id >= a.V ? (unsigned)a.V : (unsigned)id;
}
__global__ __launch_bounds__(256) void k_rs_hist(RsArgs a)
{
    __shared__ int s_h[256];
    s_h[threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * RS_TILE;
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; r++) {
        const int i = base + r * 256 + threadIdx.x;
        if (i < a.L) atomicAdd(&s_h[rs_key(a, i) >> a.shift & 255], 1);       // (whole numbers: the order does not matter)
    }
    __syncthreads();
    a.hist[threadIdx.x * a.nblk + blockIdx.x] = s_h[threadIdx.x];
}
// one workgroup per digit: exclusive sums along the digit's row of the histogram, and its total
__global__ __launch_bounds__(256) void k_rs_scan(RsArgs a)
{
    __shared__ int s_w[4];
    int* row = a.hist + (long long)blockIdx.x * a.nblk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int run = 0;
    for (int b = 0; b < a.nblk; b += 256) {
        const int i = b + threadIdx.x;
        const int v = i < a.nblk ? row[i] : 0;
        int s = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(s, off); if (lane >= off) s += t; }
        if (lane == 63) s_w[wave] = s;
        __syncthreads();
        int before = run;
        for (int w = 0; w < wave; w++) before += s_w[w];
        if (i < a.nblk) row[i] = before + s - v;
        run += s_w[0] + s_w[1] + s_w[2] + s_w[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.totals[blockIdx.x] = run;
}
__global__ __launch_bounds__(256) void k_rs_scatter(RsArgs a)
{
    __shared__ int s_cnt[4][256], s_base[256], s_w[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d0 = threadIdx.x;
    // where the digit begins: sums of the totals in front of it
    {
        const int v = a.totals[d0];
        int s = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(s, off); if (lane >= off) s += t; }
        if (lane == 63) s_w[wave] = s;
        __syncthreads();
        for (int w = 0; w < wave; w++) s += s_w[w];
        s_base[d0] = s - v + a.hist[(long long)d0 * a.nblk + blockIdx.x];
    }
#pragma unroll
    for (int w = 0; w < 4; w++) s_cnt[w][d0] = 0;
    __syncthreads();
    // a wave ranks its 512 neighbouring keys, 64 at a time: lanes with the same digit find each other by eight ballots
    unsigned key[RS_ROUNDS], rank[RS_ROUNDS];
    const int first = blockIdx.x * RS_TILE + wave * (RS_TILE / 4);
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; r++) {
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
    int before = s_base[d0];
#pragma unroll
    for (int w = 0; w < 4; w++) { const int c = s_cnt[w][d0]; s_cnt[w][d0] = before; before += c; }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RS_ROUNDS; r++) {
        const int i = first + r * 64 + lane;
        if (i >= a.L) continue;
        const unsigned to = s_cnt[wave][key[r] >> a.shift & 255] + rank[r];
        a.out_keys[to] = key[r];
        a.out_pos[to] = a.ids ? (unsigned)i : a.pos[i];
    }
}

// ---- sums of neighbouring entries with one key ----
// A group of `lanes` threads walks one chunk of the sorted list.  A run of equal keys that begins and ends inside the chunk is a finished row of the gradient;
// a run that touches a chunk border which the row crosses becomes a piece.  Every chunk leaves two entries for the next level, its first and its last run's key
// (a chunk of one run: the same key twice), each with a flag that says whether a piece stands behind it: the keys of the next level are sorted again.
struct EmbSum {
    const unsigned* keys; const unsigned char* any;    // any: null at level 0 (every entry counts)
    const unsigned* pos; const void* g; const float* weights;      // level 0: rows of the output gradient
    const float* piece;                                // later levels
    unsigned* out_keys; unsigned char* out_any; float* out_piece;  // null: this level is the last one
    void* g_table; long long V;
    int L, D, dt, bag; float scale;
};
template <int VEC, bool LEVEL0>
__global__ __launch_bounds__(256) void k_emb_sum(EmbSum a, int lanes)
{
    const int per = 256 / lanes, chunk = (int)(blockIdx.x * per + threadIdx.x / lanes);
    const int s = chunk * EMB_CHUNK;
    if (s >= a.L) return;
    const int e = s + EMB_CHUNK < a.L ? s + EMB_CHUNK : a.L;
    const int d = (int)(blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * VEC;
    const bool lead = d == 0, col = d < a.D;
    const unsigned k_first = a.keys[s], k_last = a.keys[e - 1];
    const bool open_l = s > 0 && a.keys[s - 1] == k_first, open_r = e < a.L && a.keys[e] == k_last;
    EmbVec<VEC> acc = {};
    bool some = false, any0 = false, any1 = false;
    unsigned cur = k_first;
    bool in_first = true;
    for (int j = s; j <= e; j++) {
        const unsigned k = j < e ? a.keys[j] : ~0u;
        if (k != cur) {
            // the run of `cur` ends at j
            const bool cut = (in_first && open_l) || (j == e && open_r);
            if (some && cur < a.V) {
                if (!cut) { if (col) emb_store<VEC>(a.g_table, (long long)cur * a.D + d, a.dt, acc); }
                else {
                    const int slot = in_first ? 0 : 1;
                    if (in_first) any0 = true; else any1 = true;
                    if (col) {
                        float* o = a.out_piece + (2LL * chunk + slot) * a.D + d;
#pragma unroll
                        for (int q = 0; q < VEC; q++) o[q] = acc.v[q];
                    }
                }
            }
            if (j == e) break;
            acc = EmbVec<VEC>{};
            some = false; in_first = false; cur = k;
        }
        if (!LEVEL0 && !a.any[j]) continue;
        some = true;
        if (!col || cur >= a.V) continue;
        if (LEVEL0) {
            const unsigned p = a.pos[j];
            const EmbVec<VEC> r = emb_load<VEC>(a.g, (long long)(p / (unsigned)a.bag) * a.D + d, a.dt);
            const float w = a.weights ? a.scale * a.weights[p] : a.scale;
#pragma unroll
            for (int q = 0; q < VEC; q++) acc.v[q] += w * r.v[q];
        } else {
            const float* r = a.piece + (long long)j * a.D + d;
#pragma unroll
            for (int q = 0; q < VEC; q++) acc.v[q] += r[q];
        }
    }
    if (lead && a.out_keys) {
        a.out_keys[2 * chunk] = k_first; a.out_keys[2 * chunk + 1] = k_last;
        a.out_any[2 * chunk] = any0; a.out_any[2 * chunk + 1] = any1;
    }
}

__global__ __launch_bounds__(256) void k_emb_zero(unsigned* p, long long words)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < words; i += (long long)gridDim.x * 256) p[i] = 0;
}
__global__ void k_emb_zero_tail(unsigned short* p) { *p = 0; }

// ---- host ----
#define EMB_MAX_LOOKUPS 0x7FFF0000LL
struct EmbPlan { int L, nblk, passes, levels; long long keys, hist, key_l[2], any_l[2], piece_l[2], total; };
static EmbPlan emb_plan(long long V, int D, long long L)
{
    EmbPlan p = {};
    p.L = (int)L;
    p.nblk = (int)((L + RS_TILE - 1) / RS_TILE);
    p.passes = 1;
    while (p.passes < 4 && (V >> (8 * p.passes)) != 0) p.passes++;
    p.keys = nl_up(4 * L, 256);
    p.hist = nl_up(4LL * 256 * p.nblk + 1024, 256);
    p.total = 4 * p.keys + p.hist;
    for (long long n = L; n > EMB_CHUNK;) {                                    // two entries per chunk for the next level; levels take two buffers in turn
        n = 2 * ((n + EMB_CHUNK - 1) / EMB_CHUNK);
        if (p.levels < 2) {
            const int i = p.levels;
            p.key_l[i] = nl_up(4 * n, 256); p.any_l[i] = nl_up(n, 256); p.piece_l[i] = nl_up(4 * n * D, 256);
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
static int emb_vec(int D, int dt, const void* a, const void* b)
{
    const uintptr_t m = (uintptr_t)a | (uintptr_t)b;
    if (dt != NL_DT_F32 && (D & 7) == 0 && (m & 7) == 0) return 8;
    if ((D & 3) == 0 && (m & (dt == NL_DT_F32 ? 15 : 7)) == 0) return 4;
    return 1;
}
static int emb_check(const void* table, long long V, int D, int dtype, const void* ids, int id64, long long M, int bag)
{
    if (!nl_dtype_ok(dtype) || V < 1 || V > 0x7FFFFFFF || D < 1 || D > (1 << 20) || M < 0 || bag < 1 || M > EMB_MAX_LOOKUPS / bag) return NL_ERR_INVALID_ARG;
    if (M > 0 && (!ids || ((uintptr_t)ids & (id64 ? 7 : 3)))) return NL_ERR_INVALID_ARG;
    if ((uintptr_t)table & (nl_dtype_size(dtype) - 1)) return NL_ERR_INVALID_ARG;
    return NL_OK;
}
template <int VEC> static void emb_level(const EmbSum& a, bool level0, hipStream_t st)
{
    const int lanes = emb_lanes(a.D, VEC, 256), per = 256 / lanes, chunks = (a.L + EMB_CHUNK - 1) / EMB_CHUNK;
    const dim3 grid((chunks + per - 1) / per, (a.D + lanes * VEC - 1) / (lanes * VEC));
    if (level0) hipLaunchKernelGGL((k_emb_sum<VEC, true>), grid, dim3(256), 0, st, a, lanes);
    else hipLaunchKernelGGL((k_emb_sum<VEC, false>), grid, dim3(256), 0, st, a, lanes);
}

extern "C" {

long long nl_embedding_workspace(long long V, int D, long long M, int bag)
{
    if (V < 1 || V > 0x7FFFFFFF || D < 1 || D > (1 << 20) || M < 0 || bag < 1 || M > EMB_MAX_LOOKUPS / bag) return -1;
    return M == 0 ? 0 : emb_plan(V, D, M * bag).total;
}

int nl_embedding_forward(const void* table, long long V, int D, int dtype, const void* ids, int id64, const float* weights, long long M, int bag, float scale,
                         void* out, void* stream)
{
    if (emb_check(table, V, D, dtype, ids, id64, M, bag) != NL_OK || !table) return NL_ERR_INVALID_ARG;
    if (M == 0) return NL_OK;
    if (!out || ((uintptr_t)out & (nl_dtype_size(dtype) - 1)) || ((uintptr_t)weights & 3)) return NL_ERR_INVALID_ARG;
    hipStream_t st = (hipStream_t)stream;
    const int vec = emb_vec(D, dtype, table, out), lanes = emb_lanes(D, vec, 256), per = 256 / lanes;
    const dim3 grid((unsigned)((M + per - 1) / per));
    if (vec == 8) hipLaunchKernelGGL(k_emb_forward<8>, grid, dim3(256), 0, st, table, V, D, dtype, ids, id64, weights, M, bag, scale, out, lanes);
    else if (vec == 4) hipLaunchKernelGGL(k_emb_forward<4>, grid, dim3(256), 0, st, table, V, D, dtype, ids, id64, weights, M, bag, scale, out, lanes);
    else hipLaunchKernelGGL(k_emb_forward<1>, grid, dim3(256), 0, st, table, V, D, dtype, ids, id64, weights, M, bag, scale, out, lanes);
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
    if (g_weights && M > 0) {
        const int vec = emb_vec(D, dtype, table, g_out), lanes = emb_lanes(D, vec, 64), per = 256 / lanes;
        const dim3 grid((unsigned)((L + per - 1) / per));
        if (vec == 8) hipLaunchKernelGGL(k_emb_gweights<8>, grid, dim3(256), 0, st, table, V, D, dtype, ids, id64, L, bag, scale, g_out, g_weights, lanes);
        else if (vec == 4) hipLaunchKernelGGL(k_emb_gweights<4>, grid, dim3(256), 0, st, table, V, D, dtype, ids, id64, L, bag, scale, g_out, g_weights, lanes);
        else hipLaunchKernelGGL(k_emb_gweights<1>, grid, dim3(256), 0, st, table, V, D, dtype, ids, id64, L, bag, scale, g_out, g_weights, lanes);
    }
    if (!g_table) { NL_LAUNCH_CHECK(); return NL_OK; }
    const long long bytes = V * D * nl_dtype_size(dtype);
    hipLaunchKernelGGL(k_emb_zero, dim3((unsigned)(bytes / 4 < 256 * 2048 ? bytes / 1024 + 1 : 2048)), dim3(256), 0, st, (unsigned*)g_table, bytes / 4);
    if (bytes & 3) hipLaunchKernelGGL(k_emb_zero_tail, dim3(1), dim3(1), 0, st, (unsigned short*)((char*)g_table + bytes - 2));
    if (M == 0) { NL_LAUNCH_CHECK(); return NL_OK; }
    const EmbPlan p = emb_plan(V, D, L);
    if (!ws || ws_bytes < p.total || ((uintptr_t)ws & 255)) return NL_ERR_INVALID_ARG;
    char* w = (char*)ws;
    unsigned* keys[2] = {(unsigned*)w, (unsigned*)(w + p.keys)};
    unsigned* pos[2] = {(unsigned*)(w + 2 * p.keys), (unsigned*)(w + 3 * p.keys)};
    w += 4 * p.keys;
    RsArgs r = {};
    r.totals = (int*)w; r.hist = (int*)(w + 1024); r.L = p.L; r.nblk = p.nblk; r.V = V;
    w += p.hist;
    for (int i = 0; i < p.passes; i++) {
        r.ids = i == 0 ? ids : nullptr; r.id64 = id64; r.shift = 8 * i;
        r.keys = keys[(i + 1) & 1]; r.pos = pos[(i + 1) & 1]; r.out_keys = keys[i & 1]; r.out_pos = pos[i & 1];
        hipLaunchKernelGGL(k_rs_hist, dim3(p.nblk), dim3(256), 0, st, r);
        hipLaunchKernelGGL(k_rs_scan, dim3(256), dim3(256), 0, st, r);
        hipLaunchKernelGGL(k_rs_scatter, dim3(p.nblk), dim3(256), 0, st, r);
    }
    unsigned* lk[2]; unsigned char* la[2]; float* lp[2];
    for (int i = 0; i < 2; i++) {
        lk[i] = (unsigned*)w; la[i] = (unsigned char*)(w + p.key_l[i]); lp[i] = (float*)(w + p.key_l[i] + p.any_l[i]);
        w += p.key_l[i] + p.any_l[i] + p.piece_l[i];
    }
    const int vec = emb_vec(D, dtype, g_out, g_table);
    EmbSum a = {};
    a.keys = keys[(p.passes - 1) & 1]; a.pos = pos[(p.passes - 1) & 1]; a.g = g_out; a.weights = weights; a.g_table = g_table; a.V = V; a.L = p.L; a.D = D; a.dt = dtype;
    a.bag = bag; a.scale = scale;
    for (int lev = 0; lev <= p.levels; lev++) {
        const bool last = lev == p.levels;
        a.out_keys = last ? nullptr : lk[lev & 1]; a.out_any = last ? nullptr : la[lev & 1]; a.out_piece = last ? nullptr : lp[lev & 1];
        if (vec == 8) emb_level<8>(a, lev == 0, st);
        else if (vec == 4) emb_level<4>(a, lev == 0, st);
        else emb_level<1>(a, lev == 0, st);
        a.keys = a.out_keys; a.any = a.out_any; a.piece = a.out_piece; a.pos = nullptr;
        a.L = 2 * ((a.L + EMB_CHUNK - 1) / EMB_CHUNK);
    }
    NL_LAUNCH_CHECK();
    return NL_OK;
}

}  // extern "C"

// Embedding lookup and its gradient.
//
// Forward: y_i = s T[id_i] (zeros where id_i is outside the table). Backward: dT_v = s sum over {i : id_i = v} of dy_i.
// Bound: HBM (one multiply per element moved); the sort in front of the gradient by latency.
//
// The gradient adds rows up in a fixed order and without atomics: the positions are sorted by index (a stable radix sort),
// so that the rows of one table row are neighbours, and each run of neighbours is summed in registers.
#ifndef CVCUDA_B200_EMBEDDING_KERNELS_CUH
#define CVCUDA_B200_EMBEDDING_KERNELS_CUH

#include "row_math.cuh"

#include <cooperative_groups.h>

namespace b200pp {

struct EmbeddingKParams
{
    RowMap   indices, table, dst;
    int      indexType, tableType, dstType;
    unsigned count;
    int      rows, cols;
    float    scale;
    unsigned blocks; // of a row
};

// `blockDim.x` lanes of a warp per row, R rows for each; a lane moves U vectors of W neighbouring elements of each, one block of
// blockDim.x * U vectors of the row. All loads go out before the first is used, and none is conditional: past the row's end its last
// vector is loaded again, for an index outside the table the first row. What bounds the kernel is how many bytes it has under way
// and, for short rows, how many instructions a row takes (3.3 million rows of nine: 155 us with each lane of a row reading the
// index, now 81), so a warp reads 32 indices at a time and hands them out. 65536 rows of 1024 bfloat16: 29.3 us, 5.7 TB/s, 0.88 of a
// copy's rate. DST: the output's type, -1 for any. Eight vectors per lane, four where they have eight elements (58000 rows of 512
// floats: 24.9 us, with eight 28.4; narrower ones, 400000 rows of 75 bfloat16: 57 us, with four 81).
template<int W>
constexpr int kLookupVectors = W == 8 ? 4 : 8; // U * R

template<int TABLE, int DST, int W, int U>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbeddingKParams p)
{
    constexpr int  R    = kLookupVectors<W> / U;
    const unsigned tile = blockIdx.x / p.blocks;
    const int      span = blockDim.x * W, tid = threadIdx.y * blockDim.x + threadIdx.x;
    const int      c0   = static_cast<int>(blockIdx.x - tile * p.blocks) * (span * U) + threadIdx.x * W;
    const int      rowsAtATime = 32 / blockDim.x, g = (tid & 31) / blockDim.x; // of the warp
    // below 2^31 + 256 * 8
    const unsigned base = (tile * 8 + (tid >> 5)) * (R * rowsAtATime);
    int            id[R], mine = -1;
    Vec<TABLE, W>  raw[R][U];
#pragma unroll
    for (int k = 0; k < R; ++k)
    {
        if ((k * rowsAtATime & 31) == 0)
            mine = load_index(p.indices, p.indexType, min(base + k * rowsAtATime + (tid & 31), p.count - 1), p.rows);
        id[k] = __shfl_sync(0xffffffffu, mine, (k * rowsAtATime & 31) + g);
    }
    if (p.rows > 0)
    {
#pragma unroll
        for (int k = 0; k < R; ++k)
        {
            const uint8_t *t = p.table.at(max(id[k], 0));
#pragma unroll
            for (int u = 0; u < U; ++u)
                raw[k][u] = load_raw<kElemBytes<TABLE> * W>(t + static_cast<long long>(min(c0 + u * span, p.cols - W)) * kElemBytes<TABLE>);
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k)
    {
        const unsigned r = base + k * rowsAtATime + g;
        if (r >= p.count)
            return;
        float v[U * W];
#pragma unroll
        for (int u = 0; u < U; ++u) unpack<TABLE, W>(raw[k][u], v + u * W);
#pragma unroll
        for (int i = 0; i < U * W; ++i) v[i] = id[k] < 0 ? 0.0f : v[i] * p.scale;
        if constexpr (DST < 0)
            store_vecs<W, U>(p.dst.at(r), p.dstType, c0, span, p.cols, v);
        else
            store_vecs<DST, W, U>(p.dst.at(r), c0, span, p.cols, v);
    }
}

// Rows of C elements (a palette's colours) that follow one another without gaps. A thread makes R rows, R * C elements of 16 * C
// bytes in all (R = 8 for 16-bit elements, 4 for 32-bit ones), and the warp stores its 512 * C bytes from shared memory as whole
// lines. SHARED: the table's rows, times the scale and rounded to the output's type, are copied to shared memory first, with a row of
// zeros for indices outside the table. Gathers bound this kernel: from L1 a warp's 32 addresses take a cycle for each 128-byte line
// they touch (114 us for 16.6 million indices and a palette of 256 x 3 floats), from shared memory one for each clash of banks, which
// 16-bit rows read whole (8 bytes for three) have half as many of as three floats read one by one (26 us, 4.4 TB/s, against 37).
constexpr int kShortTable = 16384; // bytes of a table that is copied to shared memory

// Elements a row takes there: 16-bit rows a power of two, float32 rows an odd number, so that they start in all banks.
template<int C, int R>
constexpr int kShortStride = R == 4 ? C | 1 : C <= 2 ? C : C <= 4 ? 4 : 8;

template<int IT, int R>
__device__ __forceinline__ void load_short_indices(const EmbeddingKParams &p, unsigned r0, int none, int *id)
{
    typedef typename Index<IT>::type T;
    if (IT == B200PP_U8 && R == 8 && p.indices.n2 == 0 && p.indices.s2 == 1 && (reinterpret_cast<uintptr_t>(p.indices.base) & 7) == 0
        && r0 + 8 <= p.count) // r0 is a multiple of eight
    {
        const uint2 v = *reinterpret_cast<const uint2 *>(p.indices.base + r0);
#pragma unroll
        for (int k = 0; k < R; ++k)
        {
            id[k] = static_cast<int>((k < 4 ? v.x : v.y) >> (k % 4 * 8) & 0xffu);
            id[k] = id[k] < p.rows ? id[k] : none;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < R; ++k)
    {
        id[k] = none;
        if (r0 + k < p.count)
        {
            const long long v = *reinterpret_cast<const T *>(p.indices.at(r0 + k));
            id[k]             = v >= 0 && v < p.rows ? static_cast<int>(v) : none;
        }
    }
}

template<int C, int R, bool SHARED>
__global__ void __launch_bounds__(256) embedding_short_rows_kernel(const EmbeddingKParams p)
{
    constexpr int            S = kShortStride<C, R>;
    extern __shared__ uint4  short_smem[]; // [8 warps][32 * C], then the table
    uint8_t                 *table = reinterpret_cast<uint8_t *>(short_smem + 8 * 32 * C);
    const int                lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint4                   *mine = short_smem + warp * (32 * C);
    if constexpr (SHARED)
    {
        for (int i = threadIdx.x; i < (p.rows + 1) * C; i += 256)
            store_elem_as(table, i / C * S + i % C, p.dstType,
                          i / C < p.rows ? load_elem(p.table.at(i / C), i % C, p.tableType) * p.scale : 0.0f);
        __syncthreads();
    }
    constexpr unsigned kWarpRows = 32 * R;
    for (unsigned long long w0 = (static_cast<unsigned long long>(blockIdx.x) * 8 + warp) * kWarpRows; w0 < p.count;
         w0 += static_cast<unsigned long long>(gridDim.x) * 8 * kWarpRows)
    {
        const unsigned r0 = static_cast<unsigned>(w0) + lane * R;
        const int      none = SHARED ? p.rows : -1;
        int            id[R];
        if (p.indexType == B200PP_U8)
            load_short_indices<B200PP_U8, R>(p, r0, none, id);
        else if (p.indexType == B200PP_S32)
            load_short_indices<B200PP_S32, R>(p, r0, none, id);
        else
            load_short_indices<B200PP_S64, R>(p, r0, none, id);
        uint4 line[C]; // the thread's 16 * C bytes
        if constexpr (SHARED && R == 8)
        {
            unsigned short h[8 * C];
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                const RawVec<2 * S> e = load_raw<2 * S>(table + id[k] * (2 * S));
#pragma unroll
                for (int c = 0; c < C; ++c) h[k * C + c] = static_cast<unsigned short>(S == 1 ? e.w[0] : e.w[c / 2] >> (c % 2 * 16));
            }
#pragma unroll
            for (int i = 0; i < C; ++i)
                line[i] = make_uint4(h[8 * i] | h[8 * i + 1] << 16, h[8 * i + 2] | h[8 * i + 3] << 16, h[8 * i + 4] | h[8 * i + 5] << 16,
                                     h[8 * i + 6] | h[8 * i + 7] << 16);
        }
        else
        {
            float v[R * C];
#pragma unroll
            for (int k = 0; k < R; ++k)
            {
                const uint8_t *row = SHARED ? nullptr : p.table.at(max(id[k], 0));
#pragma unroll
                for (int c = 0; c < C; ++c)
                {
                    if constexpr (SHARED)
                        v[k * C + c] = reinterpret_cast<const float *>(table)[id[k] * S + c];
                    else
                    {
                        v[k * C + c] = 0.0f;
                        if (id[k] >= 0)
                            v[k * C + c] = load_elem(row, c, p.tableType) * p.scale;
                    }
                }
            }
            if constexpr (R == 4)
            {
#pragma unroll
                for (int i = 0; i < C; ++i)
                    line[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                                         __float_as_uint(v[4 * i + 3]));
            }
            else
            {
#pragma unroll
                for (int i = 0; i < C; ++i)
                {
                    const RawVec<16> r = p.dstType == B200PP_BF16 ? pack<B200PP_BF16, 8>(v + 8 * i) : pack<B200PP_F16, 8>(v + 8 * i);
                    line[i]            = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
                }
            }
        }
        __syncwarp(); // the lines of the turn before are stored
#pragma unroll
        for (int i = 0; i < C; ++i) mine[lane * C + i] = line[i];
        __syncwarp();
        constexpr int kElem = 16 / R; // bytes: 2 or 4
        uint8_t      *y     = p.dst.base + w0 * (C * kElem);
        if (w0 + kWarpRows <= p.count)
        {
#pragma unroll
            for (int i = 0; i < C; ++i) reinterpret_cast<uint4 *>(y)[i * 32 + lane] = mine[i * 32 + lane];
        }
        else
        {
            const int bytes = static_cast<int>(p.count - w0) * (C * kElem);
            for (int i = lane * 2; i < bytes; i += 64)
                *reinterpret_cast<unsigned short *>(y + i) = *reinterpret_cast<unsigned short *>(reinterpret_cast<uint8_t *>(mine) + i);
        }
    }
}

struct EmbeddingGradKParams
{
    RowMap    grad, indices, dtable;
    int       gradType, indexType, dtableType;
    unsigned  count;
    int       rows, cols;
    float     scale;
    int       accumulate;
    int       padding;            // -1: none
    uint2    *entries[2];         // (index, position), count each; entries[0] holds the sorted ones
    int       passes, digitBits, sortWarps;
    unsigned  span;      // positions of a warp that sorts
    int       zeroWidth; // of the vectors that clear the table
    float    *partials;                       // [groups][2][cols]
    unsigned  units, groups;                  // of kGradUnit and kShortRun sorted positions
    unsigned  blocks;                         // column blocks of kGradCols<W>
};

// ---- first kernel: sort the positions 0..count-1 by index, stable; indices that take no part get the key `rows` and end up last.
//
// A least-significant-digit radix sort by one CTA or one cluster. Each warp owns a contiguous range of the positions and counts its
// digits in a table of its own; a prefix over the warps, the CTAs (through distributed shared memory) and the digits turns the
// counts into the places each warp writes to. The arrays between the passes are in global memory (they stay in L2); the cluster
// barrier orders the passes. One cluster, because a grid-wide sort takes three launches a pass, and clearing the table goes on at the
// same time. Few indices (of tables so large that the one kernel in embedding_grad_direct.cuh is not for them) cost latency -- the
// trips to memory, the barriers, code that is fetched to run once (8 us for 1000) -- many the scattered stores and the ballots (25 us
// for 65536 of 50000, 59 us for 262144 of 128000, sixteen CTAs). A match instruction instead of the ballots takes a turn for each
// different digit of a warp (43 us for the 65536 with eight CTAs, where ballots take 34).
constexpr int kSortThreads = 1024;
constexpr int kSortMaxBits = 10;
constexpr int kSortMaxCtas = 16;
constexpr int kSortKeys    = 2; // keys a lane holds at a time: the code is short, most of it runs once and is waited for

inline size_t sort_smem_words(int warps, int bins)
{
    return static_cast<size_t>(bins) * warps + bins + 32;
}

__global__ void __launch_bounds__(kSortThreads, 1) embedding_sort_kernel(const EmbeddingGradKParams p)
{
    namespace cg = cooperative_groups;
    extern __shared__ unsigned smem[];
    cudaTriggerProgrammaticLaunchCompletion(); // the table may be cleared meanwhile
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned    rank = cluster.block_rank(), ctas = cluster.num_blocks();
    const int         lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = kSortThreads, warps = p.sortWarps;
    const int         bins  = 1 << p.digitBits;
    unsigned         *hist  = smem;                // [warps][bins]
    unsigned         *total = smem + warps * bins; // [bins], read by the other CTAs
    unsigned         *wsum  = total + bins;        // [32]
    unsigned         *mine  = hist + warp * bins;

    constexpr unsigned kTile = 32 * kSortKeys;
    const unsigned     i0    = warp < warps ? min(p.count, (rank * warps + warp) * p.span) : p.count, i1 = min(p.count, i0 + p.span);

    for (int pass = 0; pass < p.passes; ++pass)
    {
        const int    to    = (p.passes - 1 - pass) & 1; // the last pass writes to array 0
        const uint2 *from  = p.entries[to ^ 1];
        const int    shift = pass * p.digitBits;
        uint2        entry[kSortKeys];
        auto         load = [&](unsigned tile) {
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k)
            {
                const unsigned i = tile + 32 * k + lane;
                entry[k]         = make_uint2(0, 0);
                if (i < i1)
                {
                    if (pass > 0)
                        entry[k] = from[i];
                    else
                    {
                        const int id = load_index(p.indices, p.indexType, i, p.rows);
                        entry[k]     = make_uint2(static_cast<unsigned>(id < 0 || id == p.padding ? p.rows : id), i);
                    }
                }
            }
        };
        for (int b = threadIdx.x; b < warps * bins; b += threads) hist[b] = 0;
        __syncthreads();
        for (unsigned tile = i0; tile < i1; tile += kTile)
        {
            load(tile);
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k)
                if (tile + 32 * k + lane < i1)
                    atomicAdd(mine + ((entry[k].x >> shift) & (bins - 1)), 1u); // counts: their order does not matter
        }
        __syncthreads();
        // thread b: digit b (there are at most as many as threads). Its counts over the warps before each, and over all
        const bool has = static_cast<int>(threadIdx.x) < bins;
        unsigned  *col = hist + threadIdx.x;
        if (has)
        {
            unsigned sum = 0;
#pragma unroll 4
            for (int w = 0; w < warps; ++w)
            {
                const unsigned n = col[w * bins];
                col[w * bins]    = sum;
                sum += n;
            }
            total[threadIdx.x] = sum;
        }
        cluster.sync();
        // where the digit starts for this CTA: the digits below it everywhere, and its own in the CTAs before
        unsigned before = 0, all = 0;
        if (has)
        {
            unsigned n[kSortMaxCtas];
#pragma unroll
            for (unsigned c = 0; c < kSortMaxCtas; ++c) n[c] = c < ctas ? cluster.map_shared_rank(total, c)[threadIdx.x] : 0;
#pragma unroll
            for (unsigned c = 0; c < kSortMaxCtas; ++c)
            {
                before += c < rank ? n[c] : 0;
                all += n[c];
            }
        }
        unsigned incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
            incl += lane >= o ? up : 0;
        }
        if (lane == 31)
            wsum[warp] = incl;
        __syncthreads();
        if (warp == 0)
        {
            unsigned v = lane < threads >> 5 ? wsum[lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
            {
                const unsigned up = __shfl_up_sync(0xffffffffu, v, o);
                v += lane >= o ? up : 0;
            }
            wsum[lane] = v;
        }
        __syncthreads();
        if (has)
        {
            const unsigned base = incl - all + (warp > 0 ? wsum[warp - 1] : 0) + before;
#pragma unroll 4
            for (int w = 0; w < warps; ++w) col[w * bins] += base;
        }
        __syncthreads();
        for (unsigned tile = i0; tile < i1; tile += kTile)
        {
            if (i1 - i0 > kTile)
                load(tile); // otherwise the entries are still there
            // lanes with the same digit find one another bit by bit; the first of them takes as many places as they are. The
            // barriers of the warp keep the steps' atomics in order; their results are not waited for until all are under way.
            unsigned same[kSortKeys], place[kSortKeys];
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k) same[k] = __ballot_sync(0xffffffffu, tile + 32 * k + lane < i1);
#pragma unroll 1
            for (int b = shift; b < shift + p.digitBits; ++b)
#pragma unroll
                for (int k = 0; k < kSortKeys; ++k)
                {
                    const bool     one  = entry[k].x >> b & 1;
                    const unsigned ones = __ballot_sync(0xffffffffu, one);
                    same[k] &= one ? ones : ~ones;
                }
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k)
                if (tile + 32 * k + lane >= i1)
                    same[k] = 0xffffffffu; // nobody
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k)
            {
                place[k] = 0;
                if (tile + 32 * k + lane < i1 && lane == __ffs(same[k]) - 1)
                    place[k] = atomicAdd(mine + ((entry[k].x >> shift) & (bins - 1)), static_cast<unsigned>(__popc(same[k])));
                __syncwarp();
            }
#pragma unroll
            for (int k = 0; k < kSortKeys; ++k)
            {
                const unsigned at = __shfl_sync(0xffffffffu, place[k], __ffs(same[k]) - 1) + __popc(same[k] & ((1u << lane) - 1));
                if (tile + 32 * k + lane < i1)
                    p.entries[to][at] = entry[k];
            }
        }
        cluster.sync(); // the next pass reads what this one wrote; also keeps `total` until every CTA has read it
    }
}

template<int W>
__device__ __forceinline__ void embedding_clear_row(const EmbeddingGradKParams &p, unsigned r)
{
    uint8_t *d    = p.dtable.at(r);
    float    z[W] = {};
    for (long long c = static_cast<int>(threadIdx.x & 31) * W; c < p.cols; c += 32 * W)
        store_vecs<W, 1>(d, p.dtableType, static_cast<int>(c), 0, p.cols, z);
}

// ---- beside it: clears the table, launched while the sort runs, on the SMs that leaves. All rows: rows that are written again
// soon are still in L2 then, and finding out which those are took longer (a bit per row, 65536 indices of 50000: 86 us).
constexpr int kZeroThreads = 256;

__global__ void __launch_bounds__(kZeroThreads) embedding_clear_kernel(const EmbeddingGradKParams p)
{
    cudaTriggerProgrammaticLaunchCompletion();
    for (unsigned r = blockIdx.x * (kZeroThreads / 32) + (threadIdx.x >> 5); r < static_cast<unsigned>(p.rows); r += gridDim.x * (kZeroThreads / 32))
    {
        if (p.zeroWidth == 8)
            embedding_clear_row<8>(p, r);
        else if (p.zeroWidth == 4)
            embedding_clear_row<4>(p, r);
        else if (p.zeroWidth == 2)
            embedding_clear_row<2>(p, r);
        else
            embedding_clear_row<1>(p, r);
    }
    cudaGridDependencySynchronize(); // whoever waits for this kernel waits for the sort
}

// ---- second kernel: sums the runs of equal keys among the sorted positions, a warp for kGradCols<W> columns of each job.
//  - Runs of up to kShortRun positions belong to the warp in whose unit of kGradUnit positions they start, wherever they end. It has
//    the rows of a unit in flight at once; larger units left the GPU with little more than one wave of long-lived warps.
//  - Longer runs are summed by groups of kShortRun positions into `partials` -- slot 0 for the run that comes from the group before,
//    slot 1 for the one that starts in the group, a job each -- and joined by the third kernel.
// 16384 indices of 32000 x 1024, bfloat16 to float32: 20 of 52 us; the sort takes 15 and the clearing beside it 22, the join 6.
constexpr int kGradUnit  = 8;
constexpr int kShortRun  = 32;
template<int W>
constexpr int kGradCols = W >= 4 ? 256 : 128; // eight per lane, four where they are narrow vectors
constexpr int kGradAhead = 8; // rows loaded before the first is added

// Puts a lane's sums where they belong: into `partial` or, if that is null, into the table. Not inlined: it would be there once for
// each of the rows a warp has in flight, and code that runs once is as slow as it can be fetched (32 us instead of 19 for 5003 rows of
// 333 floats). `N` values as vectors of W, `step` elements apart.
template<int W, int N>
__device__ __noinline__ void embedding_grad_put(const EmbeddingGradKParams &p, float *partial, unsigned key, int c, int step, float s0,
                                                float s1, float s2, float s3, float s4, float s5, float s6, float s7)
{
    // vectors of four at most: 256-bit accesses in a function that is not inlined end this ptxas (12.9) with a segmentation fault
    constexpr int P    = W == 8 ? 4 : W, M = N / P;
    const int     by   = W == 8 ? 4 : step;
    float         v[8] = {s0, s1, s2, s3, s4, s5, s6, s7};
    if (partial)
    {
        store_vecs<B200PP_F32, P, M>(reinterpret_cast<uint8_t *>(partial), c, by, p.cols, v);
        return;
    }
    uint8_t *d = p.dtable.at(key);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= p.scale;
    if (p.accumulate)
    {
        float old[8];
        load_vecs<P, M>(d, p.dtableType, c, by, p.cols, old);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += old[i];
    }
    store_vecs<P, M>(d, p.dtableType, c, by, p.cols, v);
}

template<int GRAD, int W>
__global__ void __launch_bounds__(256, GRAD == B200PP_F32 && W >= 4 ? 2 : 3) embedding_grad_runs_kernel(const __grid_constant__ EmbeddingGradKParams p)
{
    constexpr int            N = kGradCols<W> / 32, V = N / W, kAhead = kGradAhead;
    constexpr unsigned       kAll = 0xffffffffu;
    const int                lane = threadIdx.x & 31;
    const unsigned long long job  = blockIdx.x * 8ull + (threadIdx.x >> 5);
    const unsigned           item = static_cast<unsigned>(job / p.blocks); // the groups' slots, then the units
    if (item >= 2 * p.groups + p.units)
        return;
    const int      c0    = static_cast<int>(job - static_cast<unsigned long long>(item) * p.blocks) * kGradCols<W> + lane * W;
    const bool     whole = item < 2 * p.groups;
    const unsigned i0    = whole ? item / 2 * kShortRun : (item - 2 * p.groups) * kGradUnit;
    const int      n     = static_cast<int>(min(p.count - i0, static_cast<unsigned>(whole ? kShortRun : kGradUnit)));
    const unsigned none  = static_cast<unsigned>(p.rows);
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    // keys of the 32 positions before (lane l: i0 - 1 - l), of the 32 from i0 on and of the 32 after those
    const unsigned i     = i0 + lane;
    const unsigned bk    = static_cast<unsigned>(lane) < i0 ? p.entries[0][i0 - 1 - lane].x : none;
    const uint2    e0    = i < p.count ? p.entries[0][i] : make_uint2(none, 0);
    const uint2    e1    = i + 32u < p.count ? p.entries[0][i + 32] : make_uint2(none, 0);
    const unsigned first = __shfl_sync(kAll, e0.x, 0);
    if (first == none)
        return;
    const int valid = __popc(__ballot_sync(kAll, e0.x != none)) + __popc(__ballot_sync(kAll, e1.x != none));
    // the run at the start: `back` positions of it lie before (32: at least), it goes on for `on` (64: at least)
    const unsigned other = __ballot_sync(kAll, bk != first);
    const int      back  = other ? __ffs(other) - 1 : 32;
    const unsigned d0 = __ballot_sync(kAll, e0.x != first), d1 = __ballot_sync(kAll, e1.x != first);
    const int      on    = d0 ? __ffs(d0) - 1 : d1 ? 31 + __ffs(d1) : 64;
    // the run at the end: from position `start`, as far as it starts here, up to `stop` (beyond n if it goes on)
    const unsigned endKey = __shfl_sync(kAll, e0.x, n - 1);
    const unsigned m0 = __ballot_sync(kAll, e0.x == endKey), m1 = __ballot_sync(kAll, e1.x == endKey);
    const int      start = __ffs(m0) - 1, stop = start + __popc(m0) + (start + __popc(m0) == 32 ? __popc(m1) : 0);
    const bool     goes = endKey != none && stop > n, ours = start > 0 || back == 0; // it goes on; it starts here
    const bool     tail = goes && ours && stop - start > kShortRun;
    // what this job sums: positions from..to, counted from i0
    int from, to;
    if (whole)
    {
        if (item & 1)
        {
            if (!tail)
                return;
            from = start, to = n;
        }
        else
        {
            if (back == 0 || back + on <= kShortRun)
                return;
            from = 0, to = min(on, n);
        }
    }
    else
    {
        from = back > 0 ? on : 0; // a run from before is done by the warp it starts with, or by groups
        to   = min(tail ? start : goes && ours ? stop : n, valid);
        if (from >= min(to, n))
            return;
    }
    // bit j of ends: position j is the last of its run, as far as this job goes
    const unsigned     f0 = __shfl_down_sync(kAll, e0.x, 1), f1 = __shfl_down_sync(kAll, e1.x, 1), g1 = __shfl_sync(kAll, e1.x, 0);
    unsigned long long ends = __ballot_sync(kAll, e0.x != (lane < 31 ? f0 : g1));
    ends |= static_cast<unsigned long long>(__ballot_sync(kAll, e1.x != f1 || lane == 31)) << 32;
    ends |= 1ull << (to - 1);
    float *const part   = whole ? p.partials + static_cast<long long>(item) * p.cols : nullptr;
    float        acc[8] = {};
    for (int j = from; j < to; j += kAhead)
    {
        // nothing conditional about the loads, so that they all go out together: past the last row it is loaded again, past the
        // last column the last vector is
        Vec<GRAD, W> raw[kAhead][V];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
        {
            const int      at = min(j + a, to - 1);
            const unsigned o0 = __shfl_sync(kAll, e0.y, at & 31), o1 = __shfl_sync(kAll, e1.y, at & 31);
            const uint8_t *row = p.grad.at(at < 32 ? o0 : o1);
#pragma unroll
            for (int v = 0; v < V; ++v)
                raw[a][v] = load_raw<kElemBytes<GRAD> * W>(row + static_cast<long long>(min(c0 + v * 32 * W, p.cols - W)) * kElemBytes<GRAD>);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
        {
            const int q = j + a;
            if (q >= to)
                break;
#pragma unroll
            for (int v = 0; v < V; ++v)
            {
                float g[W];
                unpack<GRAD, W>(raw[a][v], g);
#pragma unroll
                for (int k = 0; k < W; ++k) acc[v * W + k] += g[k];
            }
            if (!((ends >> q) & 1))
                continue;
            embedding_grad_put<W, N>(p, part, __shfl_sync(kAll, q < 32 ? e0.x : e1.x, q & 31), c0, 32 * W, acc[0], acc[1], acc[2], acc[3],
                                     acc[4], acc[5], acc[6], acc[7]);
#pragma unroll
            for (int z = 0; z < N; ++z) acc[z] = 0.0f;
        }
    }
}

// ---- third kernel: the runs longer than kShortRun. A CTA looks after eight groups, a warp each: it finds out whether such a run
// starts in its group and adds up the run's parts for kJoinCols columns. Runs of more than kJoinAlone groups are left to the whole CTA,
// each warp a contiguous share of the groups, the warps one after another. (16384 indices of 32000 x 1024, all kernels: 54.1 us; left to
// the CTA from six groups on 51.7, from 66 on 61.1. 65536 of 50 x 512: 43.1, 43.1 and 55.1 us.)
constexpr int      kJoinCols  = 256;
constexpr unsigned kJoinAlone = 16;

// Adds the parts from..to of the run that starts in group u: 0 is slot 1 of that group, k slot 0 of group u + k.
__device__ __forceinline__ void embedding_add_parts(const EmbeddingGradKParams &p, unsigned u, unsigned from, unsigned to, int c0, float (&s)[8])
{
#pragma unroll 2
    for (unsigned m = from; m < to; ++m)
    {
        const float *part = p.partials + (static_cast<unsigned long long>(u + m) * 2 + (m == 0 ? 1 : 0)) * p.cols;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += part[min(c0 + 32 * j, p.cols - 1)];
    }
}

__global__ void __launch_bounds__(256) embedding_grad_join_kernel(const __grid_constant__ EmbeddingGradKParams p)
{
    __shared__ float    sums[8][kJoinCols];
    __shared__ unsigned keys[8], parts[8]; // of the runs left to the whole CTA
    constexpr unsigned  kAll = 0xffffffffu;
    const unsigned      none = static_cast<unsigned>(p.rows);
    const int           lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.y * kJoinCols + lane;
    cudaGridDependencySynchronize();
    {
        const unsigned u = blockIdx.x * 8 + warp;
        unsigned       k = none, more = 0; // the run's key, the groups it goes on in
        if (u + 1 < p.groups) // not the last group, so it is full
        {
            const unsigned first = u * kShortRun;
            const unsigned mine = p.entries[0][first + lane].x, prev = first > 0 ? p.entries[0][first - 1].x : none;
            const unsigned last = __shfl_sync(kAll, mine, 31), after = p.entries[0][first + kShortRun].x;
            const unsigned start = first + __ffs(__ballot_sync(kAll, mine == last)) - 1;
            if (last != none && after == last && !(start == first && prev == last) && start + kShortRun < p.count
                && p.entries[0][start + kShortRun].x == last)
                k = last;
        }
        while (k != none)
        {
            const unsigned long long at = (static_cast<unsigned long long>(u) + 1 + more + lane) * kShortRun;
            const unsigned           on = __ballot_sync(kAll, at < p.count && p.entries[0][at].x == k);
            more += on == kAll ? 32 : __ffs(~on) - 1;
            if (on != kAll)
                break;
        }
        if (k != none && more <= kJoinAlone)
        {
            float s[8] = {};
            embedding_add_parts(p, u, 0, more + 1, c0, s);
            embedding_grad_put<1, 8>(p, nullptr, k, c0, 32, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]);
            k = none;
        }
        if (lane == 0)
            keys[warp] = k, parts[warp] = more + 1;
    }
    __syncthreads();
    for (int l = 0; l < 8; ++l)
    {
        const unsigned k = keys[l];
        if (k == none)
            continue;
        const unsigned per = (parts[l] + 7) / 8, from = min(parts[l], warp * per), to = min(parts[l], from + per);
        float          s[8] = {};
        embedding_add_parts(p, blockIdx.x * 8 + l, from, to, c0, s);
        __syncthreads(); // the sums of the run before are taken
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[warp][lane + 32 * j] = s[j];
        __syncthreads();
        // the first warp hands the totals over: lane l has columns l, l + 32, ...
        if (warp == 0)
        {
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                s[j] = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) s[j] += sums[w][lane + 32 * j];
            }
            embedding_grad_put<1, 8>(p, nullptr, k, c0, 32, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]);
        }
    }
}

} // namespace b200pp

#endif

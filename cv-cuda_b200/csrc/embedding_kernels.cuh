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

// blockDim.x lanes of a warp per row, blockDim.y rows per CTA; a lane moves up to U vectors of W neighbouring elements, one
// block of blockDim.x * U vectors of the row at a time. All loads of a block are issued before the first is used.
template<int TABLE, int W, int U>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbeddingKParams p)
{
    const unsigned long long job = static_cast<unsigned long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const unsigned           r   = static_cast<unsigned>(p.blocks == 1 ? job : job / p.blocks);
    if (job >= static_cast<unsigned long long>(p.count) * p.blocks)
        return;
    const int      span = blockDim.x * W;
    const int      c0   = static_cast<int>(job - static_cast<unsigned long long>(r) * p.blocks) * (span * U) + threadIdx.x * W;
    const int      id   = load_index(p.indices, p.indexType, r, p.rows);
    uint8_t       *y    = p.dst.at(r);
    const uint8_t *t    = p.table.at(max(id, 0));
    Vec<TABLE, W>  raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
    {
        const int c = c0 + u * span;
        raw[u]      = zero_raw<kElemBytes<TABLE> * W>();
        if (id >= 0 && c < p.cols)
            raw[u] = load_raw<kElemBytes<TABLE> * W>(t + static_cast<long long>(c) * kElemBytes<TABLE>);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
    {
        const int c = c0 + u * span;
        float     v[W];
        unpack<TABLE, W>(raw[u], v);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = id < 0 ? 0.0f : v[i] * p.scale;
        if (c < p.cols)
            store_vec<W>(y, c, p.dstType, v);
    }
}

// Rows of a few elements that follow one another without gaps (a palette's colours): a thread makes eight neighbouring elements of
// the output, whichever rows they belong to, and stores them as one vector.
__global__ void __launch_bounds__(256) embedding_short_rows_kernel(const EmbeddingKParams p)
{
    const unsigned long long total = static_cast<unsigned long long>(p.count) * p.cols;
    const unsigned long long e0    = (static_cast<unsigned long long>(blockIdx.x) * blockDim.x + threadIdx.x) * 8;
    if (e0 >= total)
        return;
    unsigned       r  = static_cast<unsigned>(e0 / p.cols);
    int            c  = static_cast<int>(e0 - static_cast<unsigned long long>(r) * p.cols);
    int            id = load_index(p.indices, p.indexType, r, p.rows);
    const uint8_t *t  = p.table.at(max(id, 0));
    float          v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        v[i] = 0.0f;
        if (e0 + i < total)
        {
            if (id >= 0)
                v[i] = load_elem(t, c, p.tableType) * p.scale;
            if (++c == p.cols && e0 + i + 1 < total)
            {
                c  = 0;
                id = load_index(p.indices, p.indexType, ++r, p.rows);
                t  = p.table.at(max(id, 0));
            }
        }
    }
    if (e0 + 8 <= total)
        store_vec<8>(p.dst.base, e0, p.dstType, v);
    else
        for (int i = 0; i < 8 && e0 + i < total; ++i) store_elem_as(p.dst.base, e0 + i, p.dstType, v[i]);
}

struct EmbeddingGradKParams
{
    RowMap    grad, indices, dtable;
    int       gradType, indexType, dtableType;
    unsigned  count;
    int       rows, cols;
    float     scale;
    int       accumulate;
    int       padding; // -1: none
    unsigned *keys[2], *order[2]; // count entries each; the sorted ones are keys[0], order[0]
    int       passes, digitBits;
    float    *partials; // [units][2][cols]
    unsigned  unit;     // sorted positions per unit
};

// ---- sort: positions 0..count-1 by index, stable; indices that take no part get the key `rows` and end up last.
//
// One cluster of kSortCtas CTAs, a least-significant-digit radix sort. Each warp owns a contiguous range of the positions
// and counts its digits in a table of its own (lanes with equal digits find one another with a match instruction, so no
// atomics and a fixed order); a prefix over the warps, the CTAs (through distributed shared memory) and the digits turns the
// counts into the places each warp writes to. The arrays between the passes are in global memory (they stay in L2); the
// cluster barrier orders the passes.
constexpr int kSortCtas    = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortMaxBits = 10;

inline size_t sort_smem_words(int bins)
{
    return static_cast<size_t>(bins) * (kSortThreads / 32) + bins + 32;
}

__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads, 1) embedding_sort_kernel(const EmbeddingGradKParams p)
{
    namespace cg = cooperative_groups;
    extern __shared__ unsigned smem[];
    cg::cluster_group          cluster = cg::this_cluster();
    const unsigned             rank    = cluster.block_rank();
    const int                  lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int              kWarps = kSortThreads / 32;
    const int                  bins   = 1 << p.digitBits;
    unsigned                  *hist   = smem;                 // [warps][bins]
    unsigned                  *total  = smem + kWarps * bins; // [bins], read by the other CTAs
    unsigned                  *wsum   = total + bins;         // [32]

    const unsigned long long perWarp = ((static_cast<unsigned long long>(p.count) + kSortCtas * kWarps - 1) / (kSortCtas * kWarps) + 31) / 32 * 32;
    const unsigned long long first   = (static_cast<unsigned long long>(rank) * kWarps + warp) * perWarp;
    const unsigned           i0      = static_cast<unsigned>(first < p.count ? first : p.count);
    const unsigned           i1      = static_cast<unsigned>(first + perWarp < p.count ? first + perWarp : p.count);
    unsigned                *mine    = hist + warp * bins;

    for (int pass = 0; pass < p.passes; ++pass)
    {
        // the last pass writes to array 0
        const int       to    = (p.passes - 1 - pass) & 1;
        const unsigned *keys  = p.keys[to ^ 1];
        const unsigned *order = p.order[to ^ 1];
        const int       shift = pass * p.digitBits;
        auto            key_at = [&](unsigned i) {
            if (pass > 0)
                return keys[i];
            const int id = load_index(p.indices, p.indexType, i, p.rows);
            return id < 0 || id == p.padding ? static_cast<unsigned>(p.rows) : static_cast<unsigned>(id);
        };
        for (int b = threadIdx.x; b < kWarps * bins; b += kSortThreads) hist[b] = 0;
        __syncthreads();
        for (unsigned i = i0 + lane; i - lane < i1; i += 32)
        {
            const bool     in    = i < i1;
            const unsigned digit = in ? (key_at(i) >> shift) & (bins - 1) : bins;
            const unsigned same  = __match_any_sync(0xffffffffu, digit);
            if (in && lane == __ffs(same) - 1)
                mine[digit] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        // bins <= threads: thread b does digit b
        unsigned sum = 0;
        if (static_cast<int>(threadIdx.x) < bins)
        {
            for (int w = 0; w < kWarps; ++w)
            {
                const unsigned n                = hist[w * bins + threadIdx.x];
                hist[w * bins + threadIdx.x] = sum;
                sum += n;
            }
            total[threadIdx.x] = sum;
        }
        cluster.sync();
        unsigned before = 0, all = 0;
        if (static_cast<int>(threadIdx.x) < bins)
            for (unsigned c = 0; c < kSortCtas; ++c)
            {
                const unsigned n = cluster.map_shared_rank(total, c)[threadIdx.x];
                before += c < rank ? n : 0;
                all += n;
            }
        // exclusive prefix of `all` over the digits
        unsigned incl = all;
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
            unsigned v = wsum[lane];
            for (int o = 1; o < 32; o <<= 1)
            {
                const unsigned up = __shfl_up_sync(0xffffffffu, v, o);
                v += lane >= o ? up : 0;
            }
            wsum[lane] = v;
        }
        __syncthreads();
        const unsigned base = incl - all + (warp > 0 ? wsum[warp - 1] : 0) + before;
        if (static_cast<int>(threadIdx.x) < bins)
            for (int w = 0; w < kWarps; ++w) hist[w * bins + threadIdx.x] += base;
        __syncthreads();
        for (unsigned i = i0 + lane; i - lane < i1; i += 32)
        {
            const bool     in    = i < i1;
            const unsigned key   = in ? key_at(i) : 0;
            const unsigned pos   = in ? (pass > 0 ? order[i] : i) : 0;
            const unsigned digit = in ? (key >> shift) & (bins - 1) : bins;
            const unsigned same  = __match_any_sync(0xffffffffu, digit);
            if (in)
            {
                const unsigned at = mine[digit] + __popc(same & ((1u << lane) - 1));
                p.keys[to][at]    = key;
                p.order[to][at]   = pos;
            }
            __syncwarp();
            if (in && lane == __ffs(same) - 1)
                mine[digit] += __popc(same);
            __syncwarp();
        }
        cluster.sync(); // also keeps `total` until every CTA has read it
    }
}

__global__ void __launch_bounds__(256) embedding_zero_kernel(const EmbeddingGradKParams p)
{
    for (unsigned r = blockIdx.x; r < static_cast<unsigned>(p.rows); r += gridDim.x)
    {
        uint8_t *d = p.dtable.at(r);
        for (long long c = threadIdx.x; c < p.cols; c += blockDim.x) store_elem_as(d, c, p.dtableType, 0.0f);
    }
}

__device__ __forceinline__ void embedding_grad_store(const EmbeddingGradKParams &p, unsigned key, long long c, float sum)
{
    uint8_t *d = p.dtable.at(key);
    float    v = sum * p.scale;
    if (p.accumulate)
        v += load_elem(d, c, p.dtableType);
    store_elem_as(d, c, p.dtableType, v);
}

// A warp sums the runs of equal keys among `unit` neighbouring sorted positions, for 256 columns. A run that lies inside the
// unit goes to the table; what belongs to a run that crosses the unit's ends goes to `partials`: slot 0 the run that comes
// from the unit before, slot 1 the one that starts here and goes on.
__global__ void __launch_bounds__(256) embedding_grad_runs_kernel(const EmbeddingGradKParams p)
{
    const int          lane   = threadIdx.x & 31;
    const unsigned     blocks = (p.cols + 255u) / 256u;
    const unsigned     units  = (p.count + p.unit - 1) / p.unit;
    unsigned long long job    = blockIdx.x * 8ull + (threadIdx.x >> 5);
    if (job >= static_cast<unsigned long long>(units) * blocks)
        return;
    const unsigned  u  = static_cast<unsigned>(job / blocks);
    const long long c0 = static_cast<long long>(job % blocks) * 256 + lane;
    const unsigned  i0 = u * p.unit, i1 = min(p.count, i0 + p.unit);
    float           acc[8] = {};
    unsigned        cur    = p.keys[0][i0];
    bool            head   = i0 > 0 && p.keys[0][i0 - 1] == cur;
    for (unsigned i = i0; i < i1; ++i)
    {
        if (cur == static_cast<unsigned>(p.rows))
            return;
        const uint8_t *g = p.grad.at(p.order[0][i]);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c0 + 32 * k < p.cols)
                acc[k] += load_elem(g, c0 + 32 * k, p.gradType);
        const unsigned next = i + 1 < p.count ? p.keys[0][i + 1] : static_cast<unsigned>(p.rows);
        if (next == cur && i + 1 < i1)
            continue;
        const bool tail = next == cur;
#pragma unroll
        for (int k = 0; k < 8; ++k)
        {
            if (c0 + 32 * k < p.cols)
            {
                if (head || tail)
                    p.partials[(static_cast<long long>(u) * 2 + (head ? 0 : 1)) * p.cols + c0 + 32 * k] = acc[k];
                else
                    embedding_grad_store(p, cur, c0 + 32 * k, acc[k]);
            }
            acc[k] = 0.0f;
        }
        head = false;
        cur  = next;
    }
}

// The runs that cross units: the unit a run starts in adds up its parts, in order.
__global__ void __launch_bounds__(256) embedding_grad_join_kernel(const EmbeddingGradKParams p)
{
    const unsigned  u    = blockIdx.x;
    const unsigned  last = min(p.count, (u + 1) * p.unit) - 1; // its last position
    const unsigned  key  = p.keys[0][last];
    const long long c    = static_cast<long long>(blockIdx.y) * 256 + threadIdx.x;
    if (last + 1 >= p.count || key == static_cast<unsigned>(p.rows) || p.keys[0][last + 1] != key)
        return; // nothing goes on
    const unsigned first = u * p.unit;
    if (p.keys[0][first] == key && first > 0 && p.keys[0][first - 1] == key)
        return; // it started before
    if (c >= p.cols)
        return;
    float sum = p.partials[(static_cast<long long>(u) * 2 + 1) * p.cols + c];
    for (unsigned long long i = last + 1ull; i < p.count && p.keys[0][i] == key; i += p.unit)
        sum += p.partials[static_cast<long long>(i / p.unit) * 2 * p.cols + c];
    embedding_grad_store(p, key, c, sum);
}

} // namespace b200pp

#endif

// The embedding lookup's gradient for few indices: one kernel, no workspace.
#ifndef CVCUDA_B200_EMBEDDING_GRAD_DIRECT_CUH
#define CVCUDA_B200_EMBEDDING_GRAD_DIRECT_CUH

#include "row_math.cuh"

namespace b200pp {

struct EmbeddingDirectKParams
{
    RowMap   grad, indices, dtable;
    int      gradType, indexType, dtableType;
    unsigned count;
    int      rows, cols;
    float    scale;
    int      accumulate;
    unsigned ranges;                   // of table rows: a CTA for each, times the blocks of columns
    int      most, rest;               // rows of the ranges below `rest`, one less in the others
    unsigned inverse;                  // of the odd factor of ranges, modulo 2^32
    int      twos;                     // ranges has the factor 2^twos
    unsigned paddingRange, paddingRow; // the row that is left out; ranges: none
};

constexpr int      kDirectThreads = 512, kDirectWarps = kDirectThreads / 32;
constexpr unsigned kDirectCount   = 8192; // indices. With more, all CTAs' reading of them takes longer than the sort
constexpr int      kDirectRows    = 2048; // table rows of a CTA
constexpr int      kDirectTile    = 4;    // indices a thread holds at a time, and as many are on the way
// Runs, positions that name the same row, of up to so many are summed by a group of lanes; by a warp; put in order by a warp.
constexpr int kDirectShort = 32, kDirectLong = 128, kDirectLongest = 1024;

// Lanes of a group that sums a row, a vector of W elements each: 128 bytes of it, or a warp's width of rows without vectors.
template<int GRAD, int W>
constexpr int kDirectLanes = W == 1 ? 32 : 128 / (W * kElemBytes<GRAD>) < 32 ? 128 / (W * kElemBytes<GRAD>) : 32;

// Bytes of the list, whose memory later takes the maps of bits, then the sums of the longest runs.
inline __host__ __device__ unsigned direct_list_bytes(unsigned count)
{
    return count * 4 > 8192 ? (count * 4 + 15) / 16 * 16 : 8192;
}

inline size_t direct_smem(unsigned count, int most)
{
    return direct_list_bytes(count) + (most + 7) / 8 * 48 + 16 + (count + 7) / 8 * 16;
}

// A CTA owns the table rows v with v % ranges = its own and a block of columns. It
//  1. goes through all indices and lists the positions of those that name its rows, in order;
//  2. deals the list out to its rows in whatever order that happens, and puts each row's positions into theirs: by counting the
//     smaller ones in short runs, through a map of bits in long ones, out of the list once more in the longest;
//  3. writes zeros to the rows that nobody names, and lists the others;
//  4. sums each row's positions in their order: short runs by a group of lanes each, longer ones by a warp, the longest by the CTA,
//     in contiguous shares that are added in a fixed order.
// No CTA waits for another, nothing goes through memory twice and the table is written once, where the kernels for many indices are
// a chain of four. What bounds it is latency -- 4000 of 14000 cycles go to the indices, 5000 to the loads of the rows, for 5003 of
// 1000 rows of 333 floats (16.4 -> 9.0 us) -- and, with a large table, writing that (64 of 32000 x 1024: 32 -> 26 us, 131 MB). Every
// CTA reads all the indices, so their number ends it: at 8192 of 50000 x 256 floats it takes 24 us and the chain 36, at 16384 of
// 32000 x 1024 bfloat16 59 and 54. The worst are many indices of very few, narrow rows, which few CTAs sum: 8192 of one row of 64,
// 30 us where the chain takes 23.
template<int GRAD, int W>
__global__ void __launch_bounds__(kDirectThreads, 2) embedding_grad_direct_kernel(const __grid_constant__ EmbeddingDirectKParams p)
{
    constexpr unsigned kAll = 0xffffffffu;
    constexpr int      L = kDirectLanes<GRAD, W>, C = L * W, kGroups = kDirectThreads / L, kPerWarp = 32 / L;
    extern __shared__ __align__(16) uint8_t pool[];
    __shared__ unsigned       counted[2][kDirectWarps], sums[kDirectWarps], lists[3];
    __shared__ unsigned short longs[kDirectCount / kDirectShort], longest[kDirectCount / kDirectLong]; // rows with such runs
    const int           lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned      mine = blockIdx.y;
    const int           c    = static_cast<int>(blockIdx.x) * C + lane % L * W;
    const int           own  = p.most - (mine >= static_cast<unsigned>(p.rest)); // rows

    const int       room  = (p.most + 7) / 8 * 8;
    unsigned       *list  = reinterpret_cast<unsigned *>(pool); // position | row << 16
    unsigned short *count = reinterpret_cast<unsigned short *>(pool + direct_list_bytes(p.count));
    unsigned short *start = count + room;     // [own + 1]
    unsigned short *named = start + room + 8; // rows with short runs
    unsigned short *order = named + room;     // positions by row
    for (int i = threadIdx.x; i < room / 2; i += kDirectThreads) reinterpret_cast<unsigned *>(count)[i] = 0;
    if (threadIdx.x < 3)
        lists[threadIdx.x] = 0;

    // 1. v = mine + q * ranges for a whole q exactly if (v - mine) / ranges comes out below `own` when divided modulo 2^32: by
    // the inverse of the odd factor, and by a rotation, which puts what a power of two leaves over on top
    const unsigned offset = 0u - mine * p.inverse;
    const unsigned left   = p.paddingRange == mine ? p.paddingRow : 0xffffffffu;
    const unsigned below  = (1u << lane) - 1;
    unsigned       total  = 0;
    uint2          next[kDirectTile]; // the indices of the turn to come, halves
    auto           fetch = [&](unsigned i0) {
        const bool whole = i0 - lane + 32 * kDirectTile <= p.count && p.indices.n2 == 0;
        if (whole && p.indexType == B200PP_S64 && p.indices.s2 == 8)
        {
#pragma unroll
            for (int k = 0; k < kDirectTile; ++k) next[k] = reinterpret_cast<const uint2 *>(p.indices.base)[i0 + 32 * k];
        }
        else if (whole && p.indexType == B200PP_S32 && p.indices.s2 == 4)
        {
#pragma unroll
            for (int k = 0; k < kDirectTile; ++k) next[k] = make_uint2(reinterpret_cast<const unsigned *>(p.indices.base)[i0 + 32 * k], 0);
        }
        else
        {
#pragma unroll
            for (int k = 0; k < kDirectTile; ++k)
            {
                next[k] = make_uint2(0, 0xffffffffu);
                if (i0 + 32 * k >= p.count)
                    continue;
                const uint8_t *at = p.indices.at(i0 + 32 * k);
                if (p.indexType == B200PP_S64)
                    next[k] = *reinterpret_cast<const uint2 *>(at);
                else
                    next[k] = make_uint2(p.indexType == B200PP_S32 ? *reinterpret_cast<const unsigned *>(at) : *at, 0);
            }
        }
    };
    fetch(warp * (32 * kDirectTile) + lane);
    for (unsigned tile = 0, turn = 0; tile < p.count; tile += kDirectThreads * kDirectTile, turn ^= 1)
    {
        uint2          v[kDirectTile];
        const unsigned i0 = tile + warp * (32 * kDirectTile) + lane;
#pragma unroll
        for (int k = 0; k < kDirectTile; ++k) v[k] = next[k];
        fetch(i0 + kDirectThreads * kDirectTile);
        unsigned keep[kDirectTile], n = 0;
        bool     ours[kDirectTile];
#pragma unroll
        for (int k = 0; k < kDirectTile; ++k)
        {
            const unsigned x = v[k].x * p.inverse + offset;
            v[k].x           = __funnelshift_r(x, x, p.twos);
            ours[k]          = v[k].y == 0 && v[k].x < static_cast<unsigned>(own) && v[k].x != left;
            keep[k]          = __ballot_sync(kAll, ours[k]);
            n += __popc(keep[k]);
        }
        if (lane == 0)
            counted[turn][warp] = n;
        __syncthreads();
        unsigned all = lane < kDirectWarps ? counted[turn][lane] : 0, before = lane < warp ? all : 0;
        all    = __reduce_add_sync(kAll, all);
        before = __reduce_add_sync(kAll, before) + total;
        total += all;
#pragma unroll
        for (int k = 0; k < kDirectTile; ++k)
        {
            if (ours[k])
                list[before + __popc(keep[k] & below)] = (i0 + 32 * k) | v[k].x << 16;
            before += __popc(keep[k]);
        }
    }
    __syncthreads();

    // 2.
    // (many equal rows cost no more here than others: counting them warp by warp first was slower in every case)
    for (unsigned i = threadIdx.x; i < total; i += kDirectThreads)
    {
        const unsigned row = list[i] >> 16;
        atomicAdd(reinterpret_cast<unsigned *>(count) + row / 2, 1u << row % 2 * 16); // up to 8192: no carry
    }
    __syncthreads();
    {
        constexpr int kEach = kDirectRows / kDirectThreads;
        const int     each  = (own + kDirectThreads - 1) / kDirectThreads;
        unsigned      n[kEach], sum = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k)
        {
            const int r = threadIdx.x * each + k;
            n[k]        = k < each && r < own ? count[r] : 0;
            sum += n[k];
        }
        unsigned incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const unsigned up = __shfl_up_sync(kAll, incl, o);
            incl += lane >= o ? up : 0;
        }
        if (lane == 31)
            sums[warp] = incl;
        __syncthreads();
        unsigned at = __reduce_add_sync(kAll, lane < warp ? sums[lane & (kDirectWarps - 1)] : 0) + incl - sum;
#pragma unroll
        for (int k = 0; k < kEach; ++k)
        {
            const int r = threadIdx.x * each + k;
            if (k < each && r < own)
            {
                start[r] = count[r] = static_cast<unsigned short>(at);
                at += n[k];
                if (r == own - 1)
                    start[own] = static_cast<unsigned short>(at);
            }
        }
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < total; i += kDirectThreads)
    {
        const unsigned entry = list[i], row = entry >> 16, half = row % 2 * 16;
        const unsigned at = atomicAdd(reinterpret_cast<unsigned *>(count) + row / 2, 1u << half) >> half & 0xffffu;
        order[at]         = static_cast<unsigned short>(entry);
    }

    // 3.
    const int  group = threadIdx.x / L;
    const bool inside = c < p.cols;
    for (int r = group; r < own; r += kGroups)
    {
        if (start[r] == start[r + 1])
        {
            if (!p.accumulate && inside)
            {
                float zero[W] = {};
                store_vecs<W, 1>(p.dtable.at(mine + r * p.ranges), p.dtableType, c, 0, p.cols, zero);
            }
        }
        else if (threadIdx.x % L == 0)
        {
            const int n = start[r + 1] - start[r];
            if (n <= kDirectShort)
                named[atomicAdd(lists, 1u)] = static_cast<unsigned short>(r);
            else if (n <= kDirectLong)
                longs[atomicAdd(lists + 1, 1u)] = static_cast<unsigned short>(r);
            else
                longest[atomicAdd(lists + 2, 1u)] = static_cast<unsigned short>(r);
        }
    }
    __syncthreads();

    // 2. again: short runs
    for (unsigned i = threadIdx.x; i < total; i += kDirectThreads)
    {
        const unsigned entry = list[i], row = entry >> 16, at = entry & 0xffffu, from = start[row], to = start[row + 1];
        if (to - from > kDirectShort)
            list[i] = entry | 0x80000000u; // rows are below 2048, places below 8192
        else
        {
            unsigned place = from;
            for (unsigned j = from; j < to; ++j) place += order[j] < at;
            list[i] = at | place << 16;
        }
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < total; i += kDirectThreads)
    {
        const unsigned entry = list[i];
        if (!(entry >> 31))
            order[entry >> 16] = static_cast<unsigned short>(entry);
    }
    __syncthreads();
    // the longest ones are taken out of the list again, each warp a share of it; there are few of those
    const unsigned nlongest = lists[2];
    for (unsigned k = 0; k < nlongest; ++k)
    {
        const unsigned r = longest[k], share = (total + kDirectThreads - 1) / kDirectThreads * 32, i0 = warp * share, i1 = min(total, i0 + share);
        if (start[r + 1] - start[r] <= kDirectLongest)
            continue;
        unsigned n = 0;
        for (unsigned i = i0 + lane; i - lane < i1; i += 32) n += __popc(__ballot_sync(kAll, i < i1 && list[i] >> 16 == (r | 0x8000u)));
        if (lane == 0)
            sums[warp] = n;
        __syncthreads();
        unsigned at = start[r] + __reduce_add_sync(kAll, lane < warp ? sums[lane & (kDirectWarps - 1)] : 0);
        for (unsigned i = i0 + lane; i - lane < i1; i += 32)
        {
            const unsigned entry = i < i1 ? list[i] : 0;
            const bool     in    = entry >> 16 == (r | 0x8000u);
            const unsigned all   = __ballot_sync(kAll, in);
            if (in)
                order[at + __popc(all & below)] = static_cast<unsigned short>(entry);
            at += __popc(all);
        }
        __syncthreads();
    }
    // and long ones, a warp each: the list is done with, its memory takes a map of the positions for every warp
    const unsigned words = (p.count + 31) / 32;
    unsigned      *map   = list + warp * words;
    auto           sort  = [&](unsigned from, unsigned to) {
        for (unsigned w = lane; w < words; w += 32) map[w] = 0;
        __syncwarp();
        for (unsigned j = from + lane; j < to; j += 32) atomicOr(map + order[j] / 32, 1u << order[j] % 32);
        __syncwarp();
        for (unsigned w0 = 0; w0 < words; w0 += 32)
        {
            unsigned word = w0 + lane < words ? map[w0 + lane] : 0, incl = __popc(word);
            unsigned at   = from - incl;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
            {
                const unsigned up = __shfl_up_sync(kAll, incl, o);
                incl += lane >= o ? up : 0;
            }
            at += incl;
            from += __shfl_sync(kAll, incl, 31);
            for (; word; word &= word - 1) order[at++] = static_cast<unsigned short>((w0 + lane) * 32 + __ffs(word) - 1);
        }
        __syncwarp();
    };

    // 4.
    auto add = [&](unsigned from, unsigned to, float(&acc)[W]) {
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] = 0.0f;
        constexpr int kAhead = 8;
        for (unsigned j = from; j < to; j += kAhead)
        {
            Vec<GRAD, W> raw[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
            {
                raw[a] = zero_raw<kElemBytes<GRAD> * W>();
                if (j + a < to && inside)
                    raw[a] = load_raw<kElemBytes<GRAD> * W>(p.grad.at(order[j + a]) + static_cast<long long>(c) * kElemBytes<GRAD>);
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
            {
                float g[W];
                unpack<GRAD, W>(raw[a], g);
#pragma unroll
                for (int k = 0; k < W; ++k) acc[k] += g[k];
            }
        }
    };
    auto put = [&](int r, float(&acc)[W]) {
        if (!inside)
            return;
        uint8_t *d = p.dtable.at(mine + r * p.ranges);
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] *= p.scale;
        if (p.accumulate)
        {
            float old[W];
            load_vecs<W, 1>(d, p.dtableType, c, 0, p.cols, old);
#pragma unroll
            for (int k = 0; k < W; ++k) acc[k] += old[k];
        }
        store_vecs<W, 1>(d, p.dtableType, c, 0, p.cols, acc);
    };
    // the sums of a warp's groups, in the lanes of the first
    auto fold = [&](float(&acc)[W]) {
#pragma unroll
        for (int o = L; o < 32; o <<= 1)
#pragma unroll
            for (int k = 0; k < W; ++k) acc[k] += __shfl_down_sync(kAll, acc[k], o);
    };
    float          acc[W];
    const unsigned rows = lists[0], nlong = lists[1];
    for (unsigned i = kDirectWarps - 1 - warp; i < nlongest; i += kDirectWarps)
    {
        const unsigned r = longest[i];
        if (start[r + 1] - start[r] <= kDirectLongest)
            sort(start[r], start[r + 1]);
    }
    for (unsigned i = warp; i < nlong; i += kDirectWarps)
    {
        const int      r    = longs[i];
        const unsigned from = start[r], n = start[r + 1] - from, sub = lane / L;
        sort(from, from + n);
        add(from + n * sub / kPerWarp, from + n * (sub + 1) / kPerWarp, acc);
        fold(acc);
        if (lane < L)
            put(r, acc);
    }
    for (unsigned i = group; i < rows; i += kGroups)
    {
        const int r = named[i];
        add(start[r], start[r + 1], acc);
        put(r, acc);
    }
    if (nlongest == 0)
        return;
    __syncthreads();
    float *join = reinterpret_cast<float *>(list); // [kDirectWarps][C]
    for (unsigned i = 0; i < nlongest; ++i)
    {
        const int      r    = longest[i];
        const unsigned from = start[r], n = start[r + 1] - from;
        add(from + n * group / kGroups, from + n * (group + 1) / kGroups, acc);
        fold(acc);
        __syncthreads(); // the sums before are read
        if (lane < L)
#pragma unroll
            for (int k = 0; k < W; ++k) join[warp * C + lane * W + k] = acc[k];
        __syncthreads();
        if (threadIdx.x < L)
        {
#pragma unroll
            for (int k = 0; k < W; ++k)
            {
                acc[k] = 0.0f;
                for (int w = 0; w < kDirectWarps; ++w) acc[k] += join[w * C + lane * W + k];
            }
            put(r, acc);
        }
    }
}

// padding: the row that is left out, -1 for none.
int embedding_grad_direct(EmbeddingDirectKParams &p, int width, int padding, cudaStream_t stream);

} // namespace b200pp

#endif

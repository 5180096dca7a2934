// LayerNorm.
//
// Per row of D values: m = sum(x) / D, v = sum((x - m)^2) / D, r = 1 / sqrt(v + epsilon), y = (x - m) r w + b.
// Bound: HBM (about one operation per byte moved).
#ifndef CVCUDA_B200_LAYERNORM_KERNELS_CUH
#define CVCUDA_B200_LAYERNORM_KERNELS_CUH

#include "row_math.cuh"

#include <cooperative_groups.h>

namespace b200pp {

struct LayerNormKParams
{
    RowMap         src, dst;
    unsigned       rows;
    int            cols;
    int            dstType, weightType, biasType;
    const uint8_t *weight, *bias;
    float          epsilon, fcols, invCols; // the number of columns and its reciprocal
    float         *mean, *rstd;
    unsigned       chunks;   // of a long row
    float2        *partials; // [rows][chunks]
};

// Elements a thread's vectors are made of: W, or pairs where rows start anywhere (W = 0).
template<int W>
constexpr int kStep = W ? W : 2;

// Sum over the `lanes` neighbouring lanes (a power of two) a row has in a warp, or over the block.
template<bool BLOCK>
__device__ __forceinline__ float row_sum(float v, int lanes, float *scratch)
{
    if constexpr (!BLOCK)
    {
        for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    else
    {
        // one barrier per sum: consecutive sums use different halves of the scratch memory
        v = warp_sum(v);
        if ((threadIdx.x & 31) == 0)
            scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        const float s = (threadIdx.x & 31) < ((blockDim.x + 31) >> 5) ? scratch[threadIdx.x & 31] : 0.0f;
        return warp_sum(s);
    }
}

// Weights and biases of eight values (1 and 0 where there are none).
template<int W>
__device__ __forceinline__ void layernorm_affine(const LayerNormKParams &p, int c, int step, int end, f32x2 *w, f32x2 *b)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = both(1.0f), b[i] = both(0.0f);
    if (p.weight)
        load_param<W>(p.weight, p.weightType, c, step, end, w);
    if (p.bias)
        load_param<W>(p.bias, p.biasType, c, step, end, b);
}

// Sum of a thread's values; the values that lie behind the row's end are zero.
template<int E>
__device__ __forceinline__ float sum_pairs(const f32x2 *x)
{
    f32x2 a = x[0], b = x[1];
#pragma unroll
    for (int i = 2; i < E / 2; i += 2)
    {
        a = add2(a, x[i]);
        b = add2(b, x[i + 1]);
    }
    a = add2(a, b);
    return lo2(a) + hi2(a);
}

// Replaces a thread's values by their distances to the mean (0 behind the row's end) and gives the sum of the squares.
template<int E, int W>
__device__ __forceinline__ float centre(f32x2 *x, float mean, int c, int step, int end)
{
    if (c + (E / W - 1) * step + W > end) // part of them lies behind the end
    {
        float v[E];
        singles<E>(x, v);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c + e / W * step + e % W >= end)
                v[e] = mean;
        pairs<E>(v, x);
    }
    f32x2 a = both(0.0f), b = both(0.0f);
#pragma unroll
    for (int i = 0; i < E / 2; i += 2)
    {
        x[i]     = add2(x[i], both(-mean));
        x[i + 1] = add2(x[i + 1], both(-mean));
        a        = fma2(x[i], x[i], a);
        b        = fma2(x[i + 1], x[i + 1], b);
    }
    a = add2(a, b);
    return lo2(a) + hi2(a);
}

// Forward, `blockDim.x` lanes of a warp per row (a power of two), blockDim.y rows per CTA, E values per lane. A warp walks down its
// share of the rows with the weights in registers; the rows ahead are on their way through shared memory. The statistics come from
// the registers (the variance about the mean), so the row is read once.
constexpr int kWarpStages = 3;

template<int E>
constexpr int kWarpCtas = E <= 8 ? 4 : E <= 16 ? 3 : 2; // of 256 threads on an SM, by the registers the launch bound leaves

template<int SRC, int E, int W>
__global__ void __launch_bounds__(256, kWarpCtas<E>) layernorm_warp_kernel(const LayerNormKParams p)
{
    typedef RowStage<SRC, E, W> Stage;
    extern __shared__ uint4     ring[];
    const int                   lanes = E == 32 ? 32 : blockDim.x, stageBytes = Stage::bytes(lanes, blockDim.y);
    const RowThread             k     = row_thread<E, W, E == 32>(threadIdx.x, lanes, threadIdx.y, blockDim.y);
    const unsigned              ring0 = static_cast<unsigned>(__cvta_generic_to_shared(ring));
    f32x2                       w[E / 2], b[E / 2];
#pragma unroll
    for (int i = 0; i < E / 8; ++i)
        layernorm_affine<W>(p, k.c + 8 / kStep<W> * i * k.step, k.step, p.cols, w + 4 * i, b + 4 * i);
    const unsigned long long step = static_cast<unsigned long long>(gridDim.x) * blockDim.y;
    const unsigned long long r0   = static_cast<unsigned long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    auto row = [&](unsigned long long r) { return r < p.rows ? p.src.at(static_cast<unsigned>(r)) : static_cast<const uint8_t *>(nullptr); };
#pragma unroll
    for (int s = 0; s < kWarpStages - 1; ++s)
    {
        Stage::fetch(ring0 + s * stageBytes, k, row(r0 + s * step), p.cols);
        copies_commit();
    }
    int stage = 0;
    // the lanes of a warp take the same number of turns: those of the warp's first row
    for (unsigned long long r = r0, first = r0 - threadIdx.y % (32u / lanes); first < p.rows; r += step, first += step)
    {
        Stage::fetch(ring0 + (stage == 0 ? kWarpStages - 1 : stage - 1) * stageBytes, k, row(r + (kWarpStages - 1) * step), p.cols);
        copies_commit();
        copies_wait<kWarpStages - 1>();
        if (W == 0)
            __syncwarp();
        f32x2 x[E / 2];
        Stage::take(reinterpret_cast<const uint8_t *>(ring) + stage * stageBytes, k, row(r), p.cols, x);
        stage = stage == kWarpStages - 1 ? 0 : stage + 1;
        if (W == 0)
            __syncwarp();
        const float mean = divide_count(row_sum<false>(sum_pairs<E>(x), lanes, nullptr), p.fcols, p.invCols);
        const float q    = centre<E, kStep<W>>(x, mean, k.c, k.step, p.cols);
        const float rstd = rsqrtf(row_sum<false>(q, lanes, nullptr) * p.invCols + p.epsilon);
        if (r >= p.rows)
            continue;
        if (k.t == 0)
        {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i) x[i] = fma2(mul2(x[i], both(rstd)), w[i], b[i]);
        store_row<E, W>(p.dst.at(static_cast<unsigned>(r)), p.dstType, k, p.cols, x);
    }
}

// Forward, longer rows: a CTA per row, or a cluster of up to eight CTAs with `span` columns each, which walk down their share of the
// rows together. Each CTA takes the mean and the squares of its part; the parts are joined as Chan, Golub and LeVeque do (the mean
// weighted by length, the squares plus the distances of the means) after one exchange through distributed shared memory. With
// sixteen values per thread the weights stay in registers; thirty-two are for rows that sixteen do not reach.
template<int E>
constexpr int kClusterThreads = E <= 16 ? 512 : 768; // most threads of a CTA, by the registers they need
template<int E>
constexpr int kClusterStages = E <= 16 ? 3 : 2;

template<int SRC, int E, int W>
__global__ void __launch_bounds__(kClusterThreads<E>, 1) layernorm_cluster_kernel(const LayerNormKParams p, int span)
{
    namespace cg = cooperative_groups;
    typedef RowStage<SRC, E, W> Stage;
    constexpr int               kStages = kClusterStages<E>;
    extern __shared__ uint4     ring[];
    __shared__ float            scratch[2][32];
    __shared__ float2           parts[2][8];
    cg::cluster_group           cluster = cg::this_cluster();
    const int                   ctas = cluster.num_blocks(), rank = cluster.block_rank(), stageBytes = Stage::bytes(blockDim.x, 1);
    const int                   from = rank * span, end = min(p.cols - from, span); // this CTA's columns
    const RowThread             k     = row_thread<E, W, true>(threadIdx.x, blockDim.x, 0, 1);
    const unsigned              ring0 = static_cast<unsigned>(__cvta_generic_to_shared(ring));
    f32x2                       w[E <= 16 ? E / 2 : 4], b[E <= 16 ? E / 2 : 4];
    if constexpr (E <= 16)
    {
#pragma unroll
        for (int i = 0; i < E / 8; ++i)
            layernorm_affine<W>(p, from + k.c + 8 / kStep<W> * i * k.step, k.step, from + end, w + 4 * i, b + 4 * i);
    }
    const unsigned long long step = gridDim.x / ctas;
    unsigned long long       r    = blockIdx.x / ctas;
    auto                     row  = [&](unsigned long long n) {
        return n < p.rows ? p.src.at(static_cast<unsigned>(n)) + static_cast<long long>(from) * kElemBytes<SRC> : static_cast<const uint8_t *>(nullptr);
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
    {
        Stage::fetch(ring0 + s * stageBytes, k, row(r + s * step), end);
        copies_commit();
    }
    const float n     = static_cast<float>(end), inv = 1.0f / n;
    int         stage = 0, half = 0;
    for (; r < p.rows; r += step)
    {
        // the stage before was read by every thread before a barrier of the last turn
        Stage::fetch(ring0 + (stage == 0 ? kStages - 1 : stage - 1) * stageBytes, k, row(r + (kStages - 1) * step), end);
        copies_commit();
        copies_wait<kStages - 1>();
        if (W == 0)
            __syncthreads();
        f32x2 x[E / 2];
        Stage::take(reinterpret_cast<const uint8_t *>(ring) + stage * stageBytes, k, row(r), end, x);
        stage        = stage == kStages - 1 ? 0 : stage + 1;
        float mean   = divide_count(row_sum<true>(sum_pairs<E>(x), 0, scratch[0]), n, inv);
        float q      = row_sum<true>(centre<E, kStep<W>>(x, mean, k.c, k.step, end), 0, scratch[1]);
        float centre = 0.0f; // distance of this CTA's mean to the row's
        if (ctas > 1)
        {
            if (static_cast<int>(threadIdx.x) < ctas)
                *cluster.map_shared_rank(&parts[half][rank], threadIdx.x) = make_float2(mean, q);
            cluster.sync();
            float sum = 0.0f;
            for (int c = 0; c < ctas; ++c) sum += parts[half][c].x * static_cast<float>(min(p.cols - c * span, span));
            const float whole = divide_count(sum, p.fcols, p.invCols);
            q                 = 0.0f;
            for (int c = 0; c < ctas; ++c)
            {
                const float d = parts[half][c].x - whole;
                q += parts[half][c].y + d * d * static_cast<float>(min(p.cols - c * span, span));
            }
            centre = mean - whole;
            mean   = whole;
            half ^= 1; // the next turn's parts come while slower CTAs read these
        }
        const float rstd = rsqrtf(q * p.invCols + p.epsilon);
        if (rank == 0 && threadIdx.x == 0)
        {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
        uint8_t *y = p.dst.at(static_cast<unsigned>(r)) + static_cast<long long>(from) * (p.dstType == B200PP_F32 ? 4 : 2);
        if constexpr (E <= 16)
        {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) x[i] = fma2(mul2(add2(x[i], both(centre)), both(rstd)), w[i], b[i]);
        }
        else
        {
#pragma unroll
            for (int j = 0; j < E / 8; ++j)
            {
                if (p.weight || p.bias)
                    layernorm_affine<W>(p, from + k.c + 8 / kStep<W> * j * k.step, k.step, from + end, w, b);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    const f32x2 h = mul2(add2(x[4 * j + i], both(centre)), both(rstd));
                    x[4 * j + i]  = p.weight || p.bias ? fma2(h, w[i], b[i]) : h;
                }
            }
        }
        store_row<E, W>(y, p.dstType, k, end, x);
    }
    if (ctas > 1)
        cluster.sync(); // no CTA leaves while another may still write to it
}

// Forward, a CTA per row and eight values per thread, for so few rows that only latency counts: the weights are fetched at the same
// time as the row.
template<int SRC, int W>
__global__ void __launch_bounds__(512) layernorm_few_kernel(const LayerNormKParams p)
{
    __shared__ float scratch[2][32];
    const unsigned   r = blockIdx.x;
    const RowThread  k = row_thread<8, W, true>(threadIdx.x, blockDim.x, 0, 1);
    f32x2            x[4], w[4], b[4];
    float            v[8];
    load_vecs<SRC, W, 8 / W>(p.src.at(r), k.c, k.step, p.cols, v);
    layernorm_affine<W>(p, k.c, k.step, p.cols, w, b);
    pairs<8>(v, x);
    const float mean = divide_count(row_sum<true>(sum_pairs<8>(x), 0, scratch[0]), p.fcols, p.invCols);
    const float q    = centre<8, W>(x, mean, k.c, k.step, p.cols);
    const float rstd = rsqrtf(row_sum<true>(q, 0, scratch[1]) * p.invCols + p.epsilon);
    if (threadIdx.x == 0)
    {
        if (p.mean)
            p.mean[r] = mean;
        if (p.rstd)
            p.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fma2(mul2(x[i], both(rstd)), w[i], b[i]);
    singles<8>(x, v);
    store_vecs<W, 8 / W>(p.dst.at(r), p.dstType, k.c, k.step, p.cols, v);
}

// Forward, rows too long for that, or long and few: two kernels over chunks of kChunk values. The first leaves each chunk's mean and
// sum of squared distances to it; the second joins those of its row, likewise, and normalises its chunk. It takes the
// chunks in reverse order, so that the ones read last by the first kernel are still in L2.
constexpr int kChunk        = 8192;
constexpr int kChunkThreads = 256;

template<int SRC, int W>
__global__ void __launch_bounds__(kChunkThreads) layernorm_chunk_stats_kernel(const LayerNormKParams p)
{
    __shared__ float scratch[2][32];
    constexpr int    E   = kChunk / kChunkThreads;
    const unsigned   r   = blockIdx.x / p.chunks;
    const long long  at  = static_cast<long long>(blockIdx.x - r * p.chunks) * kChunk;
    const int        c0  = static_cast<int>(at);
    const int        end = min(static_cast<long long>(p.cols), at + kChunk);
    const RowThread           span = row_thread<E, W, true>(threadIdx.x, kChunkThreads, 0, 1);
    f32x2                     x[E / 2];
    {
        float v[E];
        load_vecs<SRC, W, E / W>(p.src.at(r), c0 + span.c, span.step, end, v);
        pairs<E>(v, x);
    }
    const float mean = row_sum<true>(sum_pairs<E>(x), 0, scratch[0]) / static_cast<float>(end - c0);
    const float q    = row_sum<true>(centre<E, W>(x, mean, c0 + span.c, span.step, end), 0, scratch[1]);
    if (threadIdx.x == 0)
        p.partials[blockIdx.x] = make_float2(mean, q);
}

template<int SRC, int W>
__global__ void __launch_bounds__(kChunkThreads) layernorm_chunk_apply_kernel(const LayerNormKParams p)
{
    __shared__ float scratch[2][32];
    constexpr int    E   = kChunk / kChunkThreads;
    const unsigned   job = gridDim.x - 1 - blockIdx.x;
    const unsigned   r   = job / p.chunks;
    const long long  at  = static_cast<long long>(job - r * p.chunks) * kChunk;
    const int        c0  = static_cast<int>(at);
    const int        end = min(static_cast<long long>(p.cols), at + kChunk);
    const RowThread           span = row_thread<E, W, true>(threadIdx.x, kChunkThreads, 0, 1);
    f32x2                     x[E / 2];
    {
        float v[E];
        load_vecs<SRC, W, E / W>(p.src.at(r), c0 + span.c, span.step, end, v);
        pairs<E>(v, x);
    }
    const float2 *part = p.partials + static_cast<unsigned long long>(r) * p.chunks;
    const float   tail = static_cast<float>(p.cols - static_cast<long long>(p.chunks - 1) * kChunk); // length of the last chunk
    float         s    = 0.0f;
    for (unsigned k = threadIdx.x; k < p.chunks; k += kChunkThreads) s += part[k].x * (k + 1 < p.chunks ? static_cast<float>(kChunk) : tail);
    const float mean = divide_count(row_sum<true>(s, 0, scratch[0]), p.fcols, p.invCols);
    float       q    = 0.0f;
    for (unsigned k = threadIdx.x; k < p.chunks; k += kChunkThreads)
    {
        const float d = part[k].x - mean;
        q += part[k].y + d * d * (k + 1 < p.chunks ? static_cast<float>(kChunk) : tail);
    }
    const float rstd = rsqrtf(row_sum<true>(q, 0, scratch[1]) * p.invCols + p.epsilon);
    if (c0 == 0 && threadIdx.x == 0)
    {
        if (p.mean)
            p.mean[r] = mean;
        if (p.rstd)
            p.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) x[i] = add2(x[i], both(-mean));
    uint8_t *y = p.dst.at(r);
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
    {
        const int c = c0 + span.c + 8 / W * j * span.step;
        f32x2     w[4], b[4];
        float     v[8];
        layernorm_affine<W>(p, c, span.step, end, w, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fma2(mul2(x[4 * j + i], both(rstd)), w[i], b[i]);
        singles<8>(w, v);
        store_vecs<W, 8 / W>(y, p.dstType, c, span.step, end, v);
    }
}

} // namespace b200pp

#endif

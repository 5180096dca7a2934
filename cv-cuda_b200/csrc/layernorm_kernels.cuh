// LayerNorm.
//
// Per row of D values: m = sum(x) / D, v = sum((x - m)^2) / D, r = 1 / sqrt(v + epsilon), y = (x - m) r w + b.
// Bound: HBM (about one operation per byte moved).
#ifndef CVCUDA_B200_LAYERNORM_KERNELS_CUH
#define CVCUDA_B200_LAYERNORM_KERNELS_CUH

#include "row_math.cuh"

namespace b200pp {

struct LayerNormKParams
{
    RowMap         src, dst;
    unsigned       rows;
    int            cols;
    int            dstType, weightType, biasType;
    const uint8_t *weight, *bias;
    float          epsilon, fcols; // fcols: the number of columns
    float         *mean, *rstd;
    unsigned       chunks;   // of a long row
    float2        *partials; // [rows][chunks]
};

// A thread holds E values of its row, as vectors of W neighbouring elements: lane l of warp k of the row has vectors l, l + 32, ...
// of the warp's 32 E elements, so that every load and store of a warp covers one contiguous span, at offsets known at compile
// time. (Rows of fewer than 32 lanes: l, l + lanes, ...)
template<int E, int W, bool BLOCK>
struct RowSpan
{
    int c, step; // first element of the thread, distance to its next vector

    __device__ __forceinline__ explicit RowSpan(int t)
        : c(BLOCK ? (t >> 5) * (32 * E) + (t & 31) * W : t * W)
        , step(BLOCK || E > 8 ? 32 * W : static_cast<int>(blockDim.x) * W)
    {
    }
};

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
__device__ __forceinline__ void layernorm_affine(const LayerNormKParams &p, int c, int step, int end, float *w, float *b)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.0f, b[i] = 0.0f;
    if (p.weight)
        load_vecs<W, 8 / W>(p.weight, p.weightType, c, step, end, w);
    if (p.bias)
        load_vecs<W, 8 / W>(p.bias, p.biasType, c, step, end, b);
}

// y of a thread's values, eight at a time.
template<int E, int W>
__device__ __forceinline__ void layernorm_store(const LayerNormKParams &p, uint8_t *y, const float *x, float mean, float rstd, int c,
                                                int step, int end)
{
#pragma unroll
    for (int k = 0; k < E / 8; ++k, c += 8 / W * step)
    {
        float w[8], b[8];
        layernorm_affine<W>(p, c, step, end, w, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = fmaf((x[k * 8 + i] - mean) * rstd, w[i], b[i]);
        store_vecs<W, 8 / W>(y, p.dstType, c, step, end, b);
    }
}

// Forward, rows that fit into registers. BLOCK: one CTA per row; otherwise blockDim.x lanes of a warp per row and
// blockDim.y rows per CTA. The statistics come from the registers (the variance about the mean), so the row is read once.
template<int SRC, int E, int W, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? (E <= 16 ? 512 : 1024) : 256) layernorm_kernel(const LayerNormKParams p)
{
    __shared__ float scratch[2][32];
    const int        t = threadIdx.x, threads = blockDim.x;
    const unsigned   r = BLOCK ? blockIdx.x : blockIdx.x * blockDim.y + threadIdx.y;
    if (!BLOCK && r - threadIdx.y % (32u / threads) >= p.rows) // all rows of the warp
        return;
    const bool                 live = BLOCK || r < p.rows;
    const RowSpan<E, W, BLOCK> at(t);
    float                      xv[E], s = 0.0f;
    load_vecs<SRC, W, E / W>(p.src.at(live ? r : p.rows - 1), at.c, at.step, p.cols, xv);
    // with eight values there are registers left to fetch the weights at the same time as the row
    float w[8], b[8];
    if constexpr (E == 8)
        layernorm_affine<W>(p, at.c, at.step, p.cols, w, b);
#pragma unroll
    for (int e = 0; e < E; ++e) s += xv[e];
    const float mean = row_sum<BLOCK>(s, threads, scratch[0]) / p.fcols;
    float       q    = 0.0f;
#pragma unroll
    for (int v = 0; v < E / W; ++v)
        if (at.c + v * at.step < p.cols)
        {
#pragma unroll
            for (int i = 0; i < W; ++i)
            {
                const float d = xv[v * W + i] - mean;
                q             = fmaf(d, d, q);
            }
        }
    const float rstd = 1.0f / sqrtf(row_sum<BLOCK>(q, threads, scratch[1]) / p.fcols + p.epsilon);
    if (!live)
        return;
    if (t == 0)
    {
        if (p.mean)
            p.mean[r] = mean;
        if (p.rstd)
            p.rstd[r] = rstd;
    }
    if constexpr (E == 8)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = fmaf((xv[i] - mean) * rstd, w[i], b[i]);
        store_vecs<W, 8 / W>(p.dst.at(r), p.dstType, at.c, at.step, p.cols, b);
    }
    else
        layernorm_store<E, W>(p, p.dst.at(r), xv, mean, rstd, at.c, at.step, p.cols);
}

// Forward, longer rows: two kernels over chunks of kChunk values. The first leaves each chunk's mean and sum of squared distances
// to it; the second joins those of its row (as Chan, Golub and LeVeque do for two sets) and normalises its chunk. It takes the
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
    float            xv[E], s = 0.0f, q = 0.0f;
    const RowSpan<E, W, true> span(threadIdx.x);
    load_vecs<SRC, W, E / W>(p.src.at(r), c0 + span.c, span.step, end, xv);
#pragma unroll
    for (int e = 0; e < E; ++e) s += xv[e];
    const float mean = row_sum<true>(s, 0, scratch[0]) / static_cast<float>(end - c0);
#pragma unroll
    for (int v = 0; v < E / W; ++v)
        if (c0 + span.c + v * span.step < end)
        {
#pragma unroll
            for (int i = 0; i < W; ++i)
            {
                const float d = xv[v * W + i] - mean;
                q             = fmaf(d, d, q);
            }
        }
    q = row_sum<true>(q, 0, scratch[1]);
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
    float            xv[E];
    const RowSpan<E, W, true> span(threadIdx.x);
    load_vecs<SRC, W, E / W>(p.src.at(r), c0 + span.c, span.step, end, xv);
    const float2 *part = p.partials + static_cast<unsigned long long>(r) * p.chunks;
    const float   tail = static_cast<float>(p.cols - static_cast<long long>(p.chunks - 1) * kChunk); // length of the last chunk
    float         s    = 0.0f;
    for (unsigned k = threadIdx.x; k < p.chunks; k += kChunkThreads) s += part[k].x * (k + 1 < p.chunks ? static_cast<float>(kChunk) : tail);
    const float mean = row_sum<true>(s, 0, scratch[0]) / p.fcols;
    float       q    = 0.0f;
    for (unsigned k = threadIdx.x; k < p.chunks; k += kChunkThreads)
    {
        const float d = part[k].x - mean;
        q += part[k].y + d * d * (k + 1 < p.chunks ? static_cast<float>(kChunk) : tail);
    }
    const float rstd = 1.0f / sqrtf(row_sum<true>(q, 0, scratch[1]) / p.fcols + p.epsilon);
    if (c0 == 0 && threadIdx.x == 0)
    {
        if (p.mean)
            p.mean[r] = mean;
        if (p.rstd)
            p.rstd[r] = rstd;
    }
    layernorm_store<E, W>(p, p.dst.at(r), xv, mean, rstd, c0 + span.c, span.step, end);
}

} // namespace b200pp

#endif

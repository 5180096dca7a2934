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
    float          epsilon, fcols, invCols; // the number of columns and its reciprocal
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
__device__ __forceinline__ void layernorm_affine(const LayerNormKParams &p, int c, int step, int end, f32x2 *w, f32x2 *b)
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = both(1.0f), b[i] = both(0.0f);
    if (p.weight)
    {
        load_vecs<W, 8 / W>(p.weight, p.weightType, c, step, end, v);
        pairs<8>(v, w);
    }
    if (p.bias)
    {
        load_vecs<W, 8 / W>(p.bias, p.biasType, c, step, end, v);
        pairs<8>(v, b);
    }
}

// y of eight values, given their distances d to the mean.
template<int W>
__device__ __forceinline__ void layernorm_store(const LayerNormKParams &p, uint8_t *y, const f32x2 *d, float rstd, const f32x2 *w,
                                                const f32x2 *b, int c, int step, int end)
{
    f32x2 o[4];
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fma2(mul2(d[i], both(rstd)), w[i], b[i]);
    singles<8>(o, v);
    store_vecs<W, 8 / W>(y, p.dstType, c, step, end, v);
}

// y of a thread's values, eight at a time.
template<int E, int W>
__device__ __forceinline__ void layernorm_store(const LayerNormKParams &p, uint8_t *y, const f32x2 *d, float rstd, int c, int step, int end)
{
#pragma unroll
    for (int k = 0; k < E / 8; ++k, c += 8 / W * step)
    {
        f32x2 w[4], b[4];
        layernorm_affine<W>(p, c, step, end, w, b);
        layernorm_store<W>(p, y, d + 4 * k, rstd, w, b, c, step, end);
    }
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
    if (c + (E / W - 1) * step >= end) // part of them lies behind the end
    {
        float v[E];
        singles<E>(x, v);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c + e / W * step >= end)
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

// Forward, a warp per row, or part of one for up to 256 columns (eight values a lane): blockDim.x lanes per row, blockDim.y rows
// per CTA. A warp walks down its share of the rows with the weights in registers; the rows ahead are on their way through shared
// memory. The statistics come from the registers (the variance about the mean), so the row is read once.
constexpr int kWarpStages = 3;

template<int E>
constexpr int kWarpCtas = E <= 8 ? 4 : E <= 16 ? 3 : 2; // of 256 threads on an SM, by the registers the launch bound leaves

template<int SRC, int E, int W>
__global__ void __launch_bounds__(256, kWarpCtas<E>) layernorm_warp_kernel(const LayerNormKParams p)
{
    typedef RowStage<SRC, W, E / W> Stage;
    extern __shared__ uint4         ring[];
    constexpr int                   kStage = Stage::kThread * 256;
    const int                       t = threadIdx.x, lanes = E > 8 ? 32 : blockDim.x, tid = threadIdx.y * lanes + t;
    const RowSpan<E, W, false>      at(t);
    const unsigned                  ring0 = static_cast<unsigned>(__cvta_generic_to_shared(ring));
    f32x2                           w[E / 2], b[E / 2];
#pragma unroll
    for (int k = 0; k < E / 8; ++k)
        layernorm_affine<W>(p, at.c + 8 / W * k * at.step, at.step, p.cols, w + 4 * k, b + 4 * k);
    const unsigned long long step = static_cast<unsigned long long>(gridDim.x) * blockDim.y;
    const unsigned long long r0   = static_cast<unsigned long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    auto                     row  = [&](unsigned long long r) { return r < p.rows ? p.src.at(static_cast<unsigned>(r)) : nullptr; };
    if constexpr (Stage::kStaged)
    {
#pragma unroll
        for (int s = 0; s < kWarpStages - 1; ++s)
        {
            Stage::fetch(ring0 + s * kStage, tid, 256, row(r0 + s * step), p.src.base, at.c, at.step, p.cols);
            copies_commit();
        }
    }
    int stage = 0;
    // the lanes of a warp take the same number of turns: those of the warp's first row
    for (unsigned long long r = r0, first = r0 - threadIdx.y % (32u / lanes); first < p.rows; r += step, first += step)
    {
        f32x2 x[E / 2];
        {
            float v[E];
            if constexpr (Stage::kStaged)
            {
                const int ahead = stage == 0 ? kWarpStages - 1 : stage - 1;
                Stage::fetch(ring0 + ahead * kStage, tid, 256, row(r + (kWarpStages - 1) * step), p.src.base, at.c, at.step, p.cols);
                copies_commit();
                copies_wait<kWarpStages - 1>();
            }
            Stage::take(reinterpret_cast<const uint8_t *>(ring) + stage * kStage, tid, 256, Stage::kStaged ? nullptr : row(r), at.c, at.step,
                        p.cols, v);
            stage = stage == kWarpStages - 1 ? 0 : stage + 1;
            pairs<E>(v, x);
        }
        const float mean = divide_count(row_sum<false>(sum_pairs<E>(x), lanes, nullptr), p.fcols, p.invCols);
        const float q    = centre<E, W>(x, mean, at.c, at.step, p.cols);
        const float rstd = rsqrtf(row_sum<false>(q, lanes, nullptr) * p.invCols + p.epsilon);
        if (r >= p.rows)
            continue;
        if (t == 0)
        {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
        float v[E];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) x[i] = fma2(mul2(x[i], both(rstd)), w[i], b[i]);
        singles<E>(x, v);
        store_vecs<W, E / W>(p.dst.at(static_cast<unsigned>(r)), p.dstType, at.c, at.step, p.cols, v);
    }
}

// Forward, a CTA per row.
template<int SRC, int E, int W>
__global__ void __launch_bounds__(E <= 16 ? 512 : 1024) layernorm_block_kernel(const LayerNormKParams p)
{
    __shared__ float          scratch[2][32];
    const unsigned            r = blockIdx.x;
    const RowSpan<E, W, true> at(threadIdx.x);
    f32x2                     x[E / 2];
    {
        float v[E];
        load_vecs<SRC, W, E / W>(p.src.at(r), at.c, at.step, p.cols, v);
        pairs<E>(v, x);
    }
    // with eight values there are registers left to fetch the weights at the same time as the row
    f32x2 w[4], b[4];
    if constexpr (E == 8)
        layernorm_affine<W>(p, at.c, at.step, p.cols, w, b);
    const float mean = divide_count(row_sum<true>(sum_pairs<E>(x), 0, scratch[0]), p.fcols, p.invCols);
    const float q    = centre<E, W>(x, mean, at.c, at.step, p.cols);
    const float rstd = rsqrtf(row_sum<true>(q, 0, scratch[1]) * p.invCols + p.epsilon);
    if (threadIdx.x == 0)
    {
        if (p.mean)
            p.mean[r] = mean;
        if (p.rstd)
            p.rstd[r] = rstd;
    }
    if constexpr (E == 8)
        layernorm_store<W>(p, p.dst.at(r), x, rstd, w, b, at.c, at.step, p.cols);
    else
        layernorm_store<E, W>(p, p.dst.at(r), x, rstd, at.c, at.step, p.cols);
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
    const RowSpan<E, W, true> span(threadIdx.x);
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
    const RowSpan<E, W, true> span(threadIdx.x);
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
    layernorm_store<E, W>(p, p.dst.at(r), x, rstd, c0 + span.c, span.step, end);
}

} // namespace b200pp

#endif

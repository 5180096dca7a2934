// LayerNorm.
//
// Per row of D values: m = sum(x) / D, v = sum((x - m)^2) / D, r = 1 / sqrt(v + epsilon), y = (x - m) r w + b. r comes from rsqrtf,
// which is off by two units in the last place at most; a rounded root and a rounded division would leave one.
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
    int            chunk;    // values of a chunk
    int            shift0, shift; // RAGGED: row r starts (shift0 + r * shift) % W elements after the boundary of a vector
};

// RAGGED kernels are for rows that are no whole vectors of W, which start anywhere. A thread counts its columns from the boundary of a
// vector at or before the row's start; only the first and the last vector are not whole. All rows that a thread goes through start alike,
// so that its weights stay in registers. (The other way, W = 0, picks pairs of elements out of the rows' lines: 390000 rows of 77 float16
// take 81 us instead of 44, 116731 of 257 72 instead of 47; 300 uint8 rows of 77777, in chunks value by value, 63 instead of 24.)
template<bool RAGGED, int W>
__device__ __forceinline__ int columns_before(const LayerNormKParams &p, unsigned r)
{
    return RAGGED ? (p.shift0 + static_cast<int>(r % 8u) * p.shift) & (W - 1) : 0;
}

// Elements a thread's vectors are made of: W, or pairs where rows start anywhere (W = 0).
template<int W>
constexpr int kStep = W ? W : 2;

// Sum over the `lanes` neighbouring lanes (a power of two) a row has in a warp, or over the block.
template<bool BLOCK>
__device__ __forceinline__ float row_sum(float v, int lanes, float *scratch)
{
    if constexpr (!BLOCK)
    {
        if (lanes == 32)
            return warp_sum(v);
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

// Weights and biases of eight values (1 and 0 where there are none). RAGGED: of columns c and so on of the weights, wherever they lie.
template<int W, bool RAGGED = false>
__device__ __forceinline__ void layernorm_affine(const LayerNormKParams &p, int c, int step, int end, f32x2 *w, f32x2 *b)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = both(1.0f), b[i] = both(0.0f);
    if constexpr (RAGGED)
    {
        float f[8];
        auto  at = [&](int i) { return c + i / W * step + i % W; };
        if (p.weight)
        {
            load_scattered<8>(p.weight, p.weightType, p.cols, f, at);
            pairs<8>(f, w);
        }
        if (p.bias)
        {
            load_scattered<8>(p.bias, p.biasType, p.cols, f, at);
            pairs<8>(f, b);
        }
        return;
    }
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

// Replaces a thread's values by their distances to the mean (0 behind the row's end and before its begin) and gives the sum of the
// squares.
template<int E, int W>
__device__ __forceinline__ float centre(f32x2 *x, float mean, int c, int step, int end, int begin = 0)
{
    if (c + (E / W - 1) * step + W > end || c < begin) // part of them lies outside
    {
        float v[E];
        singles<E>(x, v);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c + e / W * step + e % W >= end || c + e / W * step + e % W < begin)
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
// the registers (the variance about the mean), so the row is read once. 50176 rows of 768 float16: 28.5 us, 5.4 TB/s, 0.84 of a copy's
// rate; the rest is the start and the end, about 4 us, at sixteen warps per SM.
constexpr int kWarpStages = 3;

template<int E>
constexpr int kWarpCtas = E <= 8 ? 4 : E <= 16 ? 3 : 2; // of 256 threads on an SM, by the registers the launch bound leaves

// FULL: 32 lanes per row.
template<int SRC, int E, int W, bool FULL, bool RAGGED>
__global__ void __launch_bounds__(256, kWarpCtas<E>) layernorm_warp_kernel(const LayerNormKParams p)
{
    typedef RowStage<SRC, E, W> Stage;
    extern __shared__ uint4     ring[];
    const int                   lanes = FULL ? 32 : blockDim.x, groups = FULL ? 8 : blockDim.y, stageBytes = Stage::bytes(lanes, groups);
    const RowThread             k     = row_thread<E, W, FULL>(threadIdx.x, lanes, threadIdx.y, groups);
    uint8_t                    *ring8 = reinterpret_cast<uint8_t *>(ring);
    const unsigned              ring0 = static_cast<unsigned>(__cvta_generic_to_shared(ring));
    f32x2                       w[E / 2], b[E / 2];
    const unsigned              step = gridDim.x * groups, r0 = blockIdx.x * groups + threadIdx.y; // a multiple of eight
    const int                   begin = columns_before<RAGGED, W>(p, r0), end = p.cols + begin;
#pragma unroll
    for (int i = 0; i < E / 8; ++i)
        layernorm_affine<W, RAGGED>(p, k.c - begin + 8 / kStep<W> * i * k.step, k.step, p.cols, w + 4 * i, b + 4 * i);
    auto source = [&](unsigned n) { return p.src.at(n) - begin * kElemBytes<SRC>; };
#pragma unroll
    for (int s = 0; s < kWarpStages; ++s) Stage::clear(ring8 + s * stageBytes, k, end);
#pragma unroll
    for (int s = 0; s < kWarpStages - 1; ++s)
    {
        if (r0 + s * step < p.rows)
            Stage::template fetch<RAGGED>(ring0 + s * stageBytes, k, source(r0 + s * step), end);
        copies_commit();
    }
    int stage = 0;
    // the lanes of a warp take the same number of turns: those of the warp's first row
    for (unsigned r = r0, first = r0 - threadIdx.y % (32u / lanes); first < p.rows; r += step, first += step)
    {
        const unsigned ahead = r + (kWarpStages - 1) * step;
        if (ahead < p.rows)
            Stage::template fetch<RAGGED>(ring0 + (stage == 0 ? kWarpStages - 1 : stage - 1) * stageBytes, k, source(ahead), end);
        copies_commit();
        copies_wait<kWarpStages - 1>();
        if (W == 0)
            __syncwarp();
        f32x2 x[E / 2];
        Stage::take(ring8 + stage * stageBytes, k, W == 0 ? p.src.at(min(r, p.rows - 1)) : nullptr, x, begin);
        stage = stage == kWarpStages - 1 ? 0 : stage + 1;
        if (W == 0)
            __syncwarp();
        const float mean = divide_count(row_sum<false>(sum_pairs<E>(x), lanes, nullptr), p.fcols, p.invCols);
        const float q    = centre<E, kStep<W>>(x, mean, k.c, k.step, end, begin);
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
        store_row<E, W, RAGGED>(p.dst.at(r) - begin * (p.dstType == B200PP_F32 ? 4 : 2), p.dstType, k, end, x, begin);
    }
}

// Forward, longer rows: a CTA per row, sixteen values per thread (15000 rows of 2048 float16: 25 us, 4.9 TB/s).
// (Clusters of CTAs for rows that do not fit into one were slower than
// the two kernels over chunks below: 72 against 37.5 us for 256 uint8 images of 224 x 224 x 3. A CTA of so many threads is alone on
// its SM, and nothing goes on there while it waits for its barriers.)
constexpr int kBlockCols     = 16 * 512;
constexpr int kBlockResident = 768; // threads that fit on an SM, by the registers per thread the launch bound leaves (80)

template<int SRC, int W, bool RAGGED>
__global__ void __launch_bounds__(kBlockResident) layernorm_block_kernel(const LayerNormKParams p)
{
    constexpr int               E = 16, kStages = 3;
    typedef RowStage<SRC, E, W> Stage;
    extern __shared__ uint4     ring[];
    __shared__ float            scratch[2][32];
    const int                   stageBytes = Stage::bytes(blockDim.x, 1);
    const RowThread             k     = row_thread<E, W, true>(threadIdx.x, blockDim.x, 0, 1);
    uint8_t                    *ring8 = reinterpret_cast<uint8_t *>(ring);
    const unsigned              ring0 = static_cast<unsigned>(__cvta_generic_to_shared(ring));
    f32x2                       w[E / 2], b[E / 2];
    const int                   begin = columns_before<RAGGED, W>(p, blockIdx.x), end = p.cols + begin;
#pragma unroll
    for (int i = 0; i < E / 8; ++i)
        layernorm_affine<W, RAGGED>(p, k.c - begin + 8 / kStep<W> * i * k.step, k.step, p.cols, w + 4 * i, b + 4 * i);
    const unsigned step   = gridDim.x; // RAGGED: a multiple of eight
    auto           source = [&](unsigned n) { return p.src.at(n) - begin * kElemBytes<SRC>; };
#pragma unroll
    for (int s = 0; s < kStages; ++s) Stage::clear(ring8 + s * stageBytes, k, end);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
    {
        if (blockIdx.x + s * step < p.rows)
            Stage::template fetch<RAGGED>(ring0 + s * stageBytes, k, source(blockIdx.x + s * step), end);
        copies_commit();
    }
    int stage = 0;
    for (unsigned r = blockIdx.x; r < p.rows; r += step)
    {
        // the stage this goes to was read by every thread before a barrier of the last turn
        const unsigned ahead = r + (kStages - 1) * step;
        if (ahead < p.rows)
            Stage::template fetch<RAGGED>(ring0 + (stage == 0 ? kStages - 1 : stage - 1) * stageBytes, k, source(ahead), end);
        copies_commit();
        copies_wait<kStages - 1>();
        if (W == 0)
            __syncthreads();
        f32x2 x[E / 2];
        Stage::take(ring8 + stage * stageBytes, k, W == 0 ? p.src.at(r) : nullptr, x, begin);
        stage            = stage == kStages - 1 ? 0 : stage + 1;
        const float mean = divide_count(row_sum<true>(sum_pairs<E>(x), 0, scratch[0]), p.fcols, p.invCols);
        const float q    = centre<E, kStep<W>>(x, mean, k.c, k.step, end, begin);
        const float rstd = rsqrtf(row_sum<true>(q, 0, scratch[1]) * p.invCols + p.epsilon);
        if (threadIdx.x == 0)
        {
            if (p.mean)
                p.mean[r] = mean;
            if (p.rstd)
                p.rstd[r] = rstd;
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i) x[i] = fma2(mul2(x[i], both(rstd)), w[i], b[i]);
        store_row<E, W, RAGGED>(p.dst.at(r) - begin * (p.dstType == B200PP_F32 ? 4 : 2), p.dstType, k, end, x, begin);
    }
}

// Forward, a CTA per row and eight values per thread, for so few rows that only latency counts: the weights are fetched at the same
// time as the row (one row of 4096 bfloat16: 2.6 us).
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

// Forward, rows too long for that: two kernels over chunks of kChunk values. The first leaves each chunk's mean and
// sum of squared distances to it; the second joins those of its row, likewise, and normalises its chunk. It takes the
// chunks in reverse order, so that the ones read last by the first kernel are still in L2. Chunks of rows that are no whole vectors
// are eight values shorter, for the vector that the first one lies in. 256 uint8 images of 224 x 224 x 3 to float32: 37.5 us, of which the
// first reading takes 9; 5.1 TB/s of what has to be moved.
constexpr int kChunk        = 8192;
constexpr int kChunkThreads = 256;

// Vectors `step` elements apart, zeros outside begin..end; those that are not whole element by element.
template<int DT, int W, int N>
__device__ __forceinline__ void load_ragged(const uint8_t *row, int c, int step, int begin, int end, Vec<DT, W> *raw)
{
    constexpr int kSize = kElemBytes<DT>, kPer = 4 / kSize; // elements of a word
#pragma unroll
    for (int v = 0; v < N; ++v)
    {
        const int at = c + v * step;
        raw[v]       = zero_raw<kSize * W>();
        if (at >= begin && at + W <= end)
            raw[v] = load_raw<kSize * W>(row + static_cast<long long>(at) * kSize);
        else
        {
#pragma unroll
            for (int e = 0; e < W; ++e)
                if (at + e >= begin && at + e < end)
                    raw[v].w[e / kPer] |= load_raw<kSize>(row + static_cast<long long>(at + e) * kSize).w[0] << (e % kPer * 8 * kSize);
        }
    }
}

template<int SRC, int W, bool RAGGED>
__global__ void __launch_bounds__(kChunkThreads) layernorm_chunk_stats_kernel(const LayerNormKParams p)
{
    cudaTriggerProgrammaticLaunchCompletion();
    constexpr int   E   = kChunk / kChunkThreads;
    const unsigned  r   = blockIdx.x / p.chunks;
    const long long at  = static_cast<long long>(blockIdx.x - r * p.chunks) * p.chunk;
    const int       len = static_cast<int>(min(static_cast<long long>(p.cols) - at, static_cast<long long>(p.chunk)));
    const int       begin = columns_before<RAGGED, W>(p, r), end = len + begin;
    const uint8_t  *x8  = p.src.at(r) + (at - begin) * kElemBytes<SRC>;
    const RowThread k   = row_thread<E, W, true>(threadIdx.x, kChunkThreads, 0, 1);
    Vec<SRC, W>     raw[E / W];
    if constexpr (RAGGED)
        load_ragged<SRC, W, E / W>(x8, k.c, k.step, begin, end, raw);
    else
    {
#pragma unroll
        for (int v = 0; v < E / W; ++v)
        {
            raw[v] = zero_raw<kElemBytes<SRC> * W>();
            if (k.c + v * k.step < end)
                raw[v] = load_raw<kElemBytes<SRC> * W>(x8 + (k.c + v * k.step) * kElemBytes<SRC>);
        }
    }
    if constexpr (SRC == B200PP_U8 && W >= 4)
    {
        // whole numbers: sum and sum of squares (at most 8192 * 255^2 < 2^32) by the four-way dot product, exact
        __shared__ unsigned total[2][8];
        unsigned            s = 0, q = 0;
#pragma unroll
        for (int v = 0; v < E / W; ++v)
#pragma unroll
            for (int i = 0; i < W / 4; ++i)
            {
                s = __dp4a(raw[v].w[i], 0x01010101u, s);
                q = __dp4a(raw[v].w[i], raw[v].w[i], q);
            }
        s = __reduce_add_sync(0xffffffffu, s);
        q = __reduce_add_sync(0xffffffffu, q);
        if ((threadIdx.x & 31) == 0)
            total[0][threadIdx.x >> 5] = s, total[1][threadIdx.x >> 5] = q;
        __syncthreads();
        if (threadIdx.x == 0)
        {
            s = q = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += total[0][i], q += total[1][i];
            // n sum(x^2) - sum(x)^2, both below 2^46
            const unsigned long long d = static_cast<unsigned long long>(len) * q - static_cast<unsigned long long>(s) * s;
            const float              n = static_cast<float>(len);
            p.partials[blockIdx.x]     = make_float2(static_cast<float>(s) / n, static_cast<float>(d) / n);
        }
    }
    else
    {
        __shared__ float scratch[2][32];
        f32x2            x[E / 2];
        {
            float v[E];
#pragma unroll
            for (int i = 0; i < E / W; ++i) unpack<SRC, W>(raw[i], v + i * W);
            pairs<E>(v, x);
        }
        const float mean = row_sum<true>(sum_pairs<E>(x), 0, scratch[0]) / static_cast<float>(len);
        const float q    = row_sum<true>(centre<E, W>(x, mean, k.c, k.step, end, begin), 0, scratch[1]);
        if (threadIdx.x == 0)
            p.partials[blockIdx.x] = make_float2(mean, q);
    }
}

template<int SRC, int W, bool RAGGED>
__global__ void __launch_bounds__(kChunkThreads) layernorm_chunk_apply_kernel(const LayerNormKParams p)
{
    constexpr int   E   = kChunk / kChunkThreads;
    const unsigned  job = gridDim.x - 1 - blockIdx.x, r = job / p.chunks;
    const long long at  = static_cast<long long>(job - r * p.chunks) * p.chunk;
    const int       len = static_cast<int>(min(static_cast<long long>(p.cols) - at, static_cast<long long>(p.chunk)));
    const int       begin = columns_before<RAGGED, W>(p, r), end = len + begin;
    const uint8_t  *x8  = p.src.at(r) + (at - begin) * kElemBytes<SRC>;
    uint8_t        *y   = p.dst.at(r) + (at - begin) * (p.dstType == B200PP_F32 ? 4 : 2);
    const RowThread k   = row_thread<E, W, true>(threadIdx.x, kChunkThreads, 0, 1);
    Vec<SRC, W>     raw[E / W];
    if constexpr (RAGGED)
        load_ragged<SRC, W, E / W>(x8, k.c, k.step, begin, end, raw);
    else
    {
#pragma unroll
        for (int v = 0; v < E / W; ++v)
        {
            raw[v] = zero_raw<kElemBytes<SRC> * W>();
            if (k.c + v * k.step < end)
                raw[v] = load_raw<kElemBytes<SRC> * W>(x8 + (k.c + v * k.step) * kElemBytes<SRC>);
        }
    }
    cudaGridDependencySynchronize(); // launched early: the values are on their way, the statistics may not be there yet
    // every warp joins the parts for itself: no barrier
    const int     lane = threadIdx.x & 31;
    const float2 *part = p.partials + static_cast<unsigned long long>(r) * p.chunks;
    const float   full = static_cast<float>(p.chunk), tail = static_cast<float>(p.cols - static_cast<long long>(p.chunks - 1) * p.chunk);
    float         s    = 0.0f;
    for (unsigned i = lane; i < p.chunks; i += 32) s += part[i].x * (i + 1 < p.chunks ? full : tail);
    const float mean = divide_count(warp_sum(s), p.fcols, p.invCols);
    float       q    = 0.0f;
    for (unsigned i = lane; i < p.chunks; i += 32)
    {
        const float d = part[i].x - mean;
        q += part[i].y + d * d * (i + 1 < p.chunks ? full : tail);
    }
    const float rstd = rsqrtf(warp_sum(q) * p.invCols + p.epsilon);
    if (at == 0 && threadIdx.x == 0)
    {
        if (p.mean)
            p.mean[r] = mean;
        if (p.rstd)
            p.rstd[r] = rstd;
    }
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
    {
        const int c = k.c + 8 / W * j * k.step;
        f32x2     x[4], w[4], b[4];
        float     v[8];
#pragma unroll
        for (int i = 0; i < 8 / W; ++i) unpack<SRC, W>(raw[j * (8 / W) + i], v + i * W);
        pairs<8>(v, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = mul2(add2(x[i], both(-mean)), both(rstd));
        if (p.weight || p.bias)
        {
            layernorm_affine<W, RAGGED>(p, static_cast<int>(at) - begin + c, k.step, static_cast<int>(at) + end, w, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fma2(x[i], w[i], b[i]);
        }
        const RowThread part = {k.t, k.threads, 0, 1, c, k.step};
        store_row<8, W, RAGGED>(y, p.dstType, part, end, x, begin);
    }
}

} // namespace b200pp

#endif

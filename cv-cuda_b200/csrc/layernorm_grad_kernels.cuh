// Gradient of LayerNorm: h = (x - m) r, g = dy w, dx = r (g - mean(g) - h mean(g h)); dw = sum over the rows of dy h, db = sum over
// the rows of dy. Bound: HBM (two tensors read, one written, about one operation per byte).
//
// The sums over the rows are split over a fixed number of parts, added up by a second kernel in a fixed order: no atomics, equal
// inputs give equal bits.
#ifndef CVCUDA_B200_LAYERNORM_GRAD_KERNELS_CUH
#define CVCUDA_B200_LAYERNORM_GRAD_KERNELS_CUH

#include "layernorm_kernels.cuh"

#include <cooperative_groups.h>

namespace b200pp {

struct LayerNormGradKParams
{
    RowMap         grad, src, dsrc;
    unsigned       rows;
    int            cols;
    int            gradType, dsrcType, weightType, dweightType, dbiasType;
    const uint8_t *weight;
    const float   *mean, *rstd;
    float          fcols, invCols;
    uint8_t       *dweight, *dbias;
    float         *partials; // [parts][2][cols]
    int            parts;
    int            shift0, shift; // row r starts (shift0 + r * shift) % W elements after the boundary of a vector, in all tensors
    int            ownWeights;    // a copy of the weights for each row group, whose rows start like one another
};

// All gradients in one pass over the data. WARP: blockDim.x lanes of a warp per row (a power of two) and blockDim.y rows per CTA at a
// time; otherwise whole warps per row, blockDim.y rows per CTA at a time, or -- for longer rows -- a cluster of up to eight CTAs with
// `span` columns each per row. CTAs (clusters) walk down their share of the rows; each thread keeps its columns of the sums over the
// rows in registers, and the rows ahead are on their way through shared memory. What a row costs besides its values -- addresses,
// shuffles, the barrier -- is why a thread has up to 24 values. 50176 rows of 768 bfloat16: 44 us with the join, 5.3 TB/s, 0.81 of a copy's
// rate. Short of that by waiting: the sums leave registers for sixteen warps per SM (5003 rows of 2051 float16, eleven rows for each
// CTA: 28 us, issue slots 0.41 used).
constexpr int kGradResident = 512; // threads that fit on an SM, by the registers per thread the launch bound leaves (128)

template<int SRC, int GRAD, int E, int W>
struct GradRing
{
    typedef RowStage<SRC, E, W>  X;
    typedef RowStage<GRAD, E, W> G;

    static constexpr int kThread = E * (kElemBytes<SRC> + kElemBytes<GRAD>);
    static constexpr int kStages = kThread * 3 * kGradResident <= 180 * 1024 ? 3 : 2; // what fits beside the weights and L1

    static __host__ __device__ constexpr int bytes(int threads, int groups)
    {
        return X::bytes(threads, groups) + G::bytes(threads, groups);
    }
};

// FULL: rows have whole warps. RAGGED: rows that are no whole vectors of W, which start anywhere. Each thread then counts its columns
// from the boundary of a vector at or before the row's start; all rows that a thread goes through start alike, and so do those of a
// warp, so that the sums over the rows stay in registers: only the first and the last vector are not whole. (W = 0, pairs of
// elements picked out of the rows' lines, is for rows that start differently in the tensors, and for few: 50030 rows of 2051 float16
// take it 225 us instead of 157, 77821 of 257 66 instead of 44.)
template<int SRC, int GRAD, int E, int W, bool WARP, bool FULL, bool RAGGED>
__global__ void __launch_bounds__(WARP ? 256 : kGradResident, WARP ? 2 : 1) layernorm_grad_kernel(const LayerNormGradKParams p, int span)
{
    namespace cg = cooperative_groups;
    typedef GradRing<SRC, GRAD, E, W> Ring;
    typedef typename Ring::X          X;
    typedef typename Ring::G          G;
    constexpr int           kStages = Ring::kStages;
    __shared__ float2       scratch[2][16]; // two halves, used in turn: one barrier per row
    __shared__ float2       parts[2][8];    // of the CTAs of a cluster
    extern __shared__ uint4 ring[];         // the stages, then the weights; in the end the sums, [groups][2][columns]
    cudaTriggerProgrammaticLaunchCompletion();
    const int       threads = WARP && FULL ? 32 : blockDim.x, groups = blockDim.y;
    const RowThread k    = row_thread<E, W, FULL>(threadIdx.x, threads, threadIdx.y, groups);
    const int       tid  = k.g * threads + k.t, warp = tid >> 5;
    const int       xBytes = X::bytes(threads, groups), stageBytes = Ring::bytes(threads, groups);
    cg::cluster_group cluster = cg::this_cluster();
    const int       ctas = WARP ? 1 : cluster.num_blocks(), rank = WARP ? 0 : cluster.block_rank();
    if (ctas > 1)
        cluster.barrier_arrive(); // waited for in front of the rows, when the copies of the first ones are under way
    // RAGGED: the rows of a warp are as many apart as there are warps, so that they start alike
    const unsigned  step = gridDim.x / ctas * groups, base = blockIdx.x / ctas * groups;
    unsigned        r    = base + (WARP && RAGGED ? warp + k.g % (32 / threads) * (threads * groups / 32) : k.g);
    // columns count from the boundary of a vector before the row's start: this CTA's begin with `from` and hold begin..end of the row
    const int       before = RAGGED ? (p.shift0 + static_cast<int>(r % 8u) * p.shift) & (W - 1) : 0;
    const int       from = rank * span, begin = rank ? 0 : before, end = WARP ? p.cols + before : min(p.cols + before - from, span);
    const unsigned  ring0 = static_cast<unsigned>(__cvta_generic_to_shared(ring));
    f32x2           dw[E / 2], db[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) dw[i] = db[i] = both(0.0f);
    int            half = 0, stage = 0;
    uint8_t       *ring8 = reinterpret_cast<uint8_t *>(ring);
    auto xRow = [&](unsigned n) { return p.src.at(n) + static_cast<long long>(from - before) * kElemBytes<SRC>; };
    auto gRow = [&](unsigned n) { return p.grad.at(n) + static_cast<long long>(from - before) * kElemBytes<GRAD>; };
    auto fetch = [&](int s, unsigned n) {
        if (n < p.rows)
        {
            X::template fetch<RAGGED>(ring0 + s * stageBytes, k, xRow(n), end);
            G::template fetch<RAGGED>(ring0 + s * stageBytes + xBytes, k, gRow(n), end);
        }
        copies_commit();
    };
    auto meet = [&]() { // the threads of a row, where they read each other's copies
        if constexpr (W == 0)
        {
            if constexpr (WARP)
                __syncwarp();
            else
                __syncthreads();
        }
    };
#pragma unroll
    for (int s = 0; s < kStages; ++s)
    {
        X::clear(ring8 + s * stageBytes, k, end);
        G::clear(ring8 + s * stageBytes + xBytes, k, end);
    }
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fetch(s, r + s * step);
    // the weights as float32, one copy for the row groups: thread t's vectors of four are `threads` apart, which no two lanes clash on.
    // Registers would have to be shared with the sums (E = 24 has 48 of those), and from L1 they cost the conversion for each row.
    f32x2    *weights = reinterpret_cast<f32x2 *>(ring8 + kStages * stageBytes);
    const int copies = RAGGED && p.ownWeights ? threads * groups : threads, copy = RAGGED && p.ownWeights ? tid : k.t;
    if (p.weight && p.dsrc.base)
    {
        if (k.g == 0 || (RAGGED && p.ownWeights))
        {
            float f[RAGGED ? E : 8];
            if constexpr (RAGGED)
                load_scattered<E>(p.weight, p.weightType, p.cols, f, [&](int i) { return from - before + k.c + i / W * k.step + i % W; });
#pragma unroll
            for (int j = 0; j < E / 8; ++j)
            {
                f32x2 w[4];
                if constexpr (RAGGED)
                    pairs<8>(f + 8 * j, w);
                else
                    load_param<W>(p.weight, p.weightType, from + k.c + j * (8 / kStep<W>) * k.step, k.step, from + end, w);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    *reinterpret_cast<ulonglong2 *>(weights + ((2 * j + i) * copies + copy) * 2) = make_ulonglong2(w[2 * i], w[2 * i + 1]);
            }
        }
        __syncthreads();
    }
    float nextMean = r < p.rows ? p.mean[r] : 0.0f, nextRstd = r < p.rows ? p.rstd[r] : 0.0f;
    if (ctas > 1)
        cluster.barrier_wait(); // every CTA of the cluster has started, so that its shared memory may be written to
    // every thread of the CTA takes the same number of turns
    for (unsigned first = base; first < p.rows; first += step, r += step)
    {
        const bool  live = r < p.rows;
        const float mean = nextMean, rstd = nextRstd;
        f32x2       h[E / 2], gv[E / 2];
        fetch(stage == 0 ? kStages - 1 : stage - 1, r + (kStages - 1) * step);
        const bool more = r + step < p.rows;
        nextMean        = more ? p.mean[r + step] : 0.0f;
        nextRstd        = more ? p.rstd[r + step] : 0.0f;
        copies_wait<kStages - 1>();
        meet();
        {
            const uint8_t *at = ring8 + stage * stageBytes;
            const unsigned n  = live ? r : 0;
            X::take(at, k, W == 0 ? xRow(n) : nullptr, h, RAGGED ? begin : 0);
            G::take(at + xBytes, k, W == 0 ? gRow(n) : nullptr, gv, RAGGED ? begin : 0);
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) h[i] = mul2(add2(h[i], both(-mean)), both(rstd));
        if (live) // otherwise there are values of an earlier row in the stage
        {
#pragma unroll
            for (int i = 0; i < E / 2; ++i)
            {
                db[i] = add2(db[i], gv[i]);
                dw[i] = fma2(gv[i], h[i], dw[i]);
            }
        }
        if (!p.dsrc.base)
        {
            meet();
            continue;
        }
        if (p.weight)
        {
#pragma unroll
            for (int i = 0; i < E / 4; ++i)
            {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(weights + (i * copies + copy) * 2);
                gv[2 * i]     = mul2(gv[2 * i], w.x);
                gv[2 * i + 1] = mul2(gv[2 * i + 1], w.y);
            }
        }
        f32x2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
        for (int i = 0; i < E / 2; ++i)
        {
            s1 = add2(s1, gv[i]);
            s2 = fma2(gv[i], h[i], s2);
        }
        float t1 = lo2(s1) + hi2(s1), t2 = lo2(s2) + hi2(s2);
        if constexpr (WARP)
        {
            t1 = row_sum<false>(t1, threads, nullptr);
            t2 = row_sum<false>(t2, threads, nullptr);
            meet();
        }
        else
        {
            t1 = warp_sum(t1);
            t2 = warp_sum(t2);
            if ((k.t & 31) == 0)
                scratch[half][warp] = make_float2(t1, t2);
            __syncthreads();
            t1 = t2 = 0.0f;
            for (int i = 0; i < threads >> 5; ++i)
            {
                const float2 o = scratch[half][k.g * (threads >> 5) + i];
                t1 += o.x;
                t2 += o.y;
            }
            if (ctas > 1) // then there is one row at a time
            {
                if (k.t < ctas)
                    *cluster.map_shared_rank(&parts[half][rank], k.t) = make_float2(t1, t2);
                cluster.sync();
                t1 = t2 = 0.0f;
                for (int i = 0; i < ctas; ++i)
                {
                    t1 += parts[half][i].x;
                    t2 += parts[half][i].y;
                }
            }
            half ^= 1;
        }
        if (!live)
            continue;
        const float c1 = t1 * p.invCols, c2 = t2 * p.invCols;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) gv[i] = mul2(add2(fma2(h[i], both(-c2), gv[i]), both(-c1)), both(rstd));
        store_row<E, W, RAGGED>(p.dsrc.at(r) + static_cast<long long>(from - before) * (p.dsrcType == B200PP_F32 ? 4 : 2), p.dsrcType, k, end,
                                gv, begin);
    }
    if (ctas > 1)
        cluster.sync(); // no CTA leaves while another may still write to it
    if (!p.partials)
        return;
    // the CTA's sums: over the rows of a warp by shuffles, then over the row groups (WARP: the warps) through shared memory
    copies_wait<0>();
    float fw[E], fb[E];
    singles<E>(dw, fw);
    singles<E>(db, fb);
    if constexpr (WARP)
        for (int o = threads; o < 32; o <<= 1)
#pragma unroll
            for (int e = 0; e < E; ++e)
            {
                fw[e] += __shfl_xor_sync(0xffffffffu, fw[e], o);
                fb[e] += __shfl_xor_sync(0xffffffffu, fb[e], o);
            }
    const int  slot = WARP ? warp : k.g, slots = WARP ? (threads * groups) >> 5 : groups;
    const bool holds = !WARP || (tid & 31) < threads;
    float     *part = p.partials + static_cast<long long>(blockIdx.x / ctas) * 2 * p.cols + from + begin - before;
    // vectors of up to four, wherever they go: single values, a vector apart, took 8 us of 28 for 300 rows of 5001 float16
    constexpr int P = kStep<W> == 8 ? 4 : kStep<W>;
    if (!RAGGED && slots == 1)
    {
        if (holds)
#pragma unroll
            for (int e = 0; e < E; e += P)
            {
                const int c = k.c + e / kStep<W> * k.step + e % kStep<W>;
                if constexpr (W > 0)
                {
                    if (c < end)
                    {
                        store_vec<B200PP_F32, P>(reinterpret_cast<uint8_t *>(part), c, fw + e);
                        store_vec<B200PP_F32, P>(reinterpret_cast<uint8_t *>(part + p.cols), c, fb + e);
                    }
                }
                else
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        if (c + i < end)
                        {
                            part[c + i]          = fw[e + i];
                            part[p.cols + c + i] = fb[e + i];
                        }
            }
        return;
    }
    float *sums = reinterpret_cast<float *>(ring); // [slots][2][span]
    __syncthreads(); // the ring is not needed any more
    if (holds)
    {
        uint8_t *to = reinterpret_cast<uint8_t *>(sums + slot * 2 * span);
#pragma unroll
        for (int e = 0; e < E; e += P)
        {
            const int c = k.c + e / kStep<W> * k.step + e % kStep<W>;
            store_vec<B200PP_F32, P>(to, c, fw + e);
            store_vec<B200PP_F32, P>(to, span + c, fb + e);
        }
    }
    __syncthreads();
    // (in a cluster there is one row at a time, and one slot)
#pragma unroll 1
    for (int which = 0; which < 2; ++which)
#pragma unroll 4
        for (int c = tid; c < end - begin; c += threads * groups)
        {
            float s = 0.0f;
            for (int i = 0; i < slots; ++i)
            {
                const int first = RAGGED && !rank ? (p.shift0 + static_cast<int>((base + i) % 8u) * p.shift) & (W - 1) : 0;
                s += sums[(2 * i + which) * span + first + c];
            }
            part[which * p.cols + c] = s;
        }
}

// Few rows, where only latency counts: the first `rowCtas` CTAs take a row each for dx, the others 32 columns each for the sums over the
// rows, which reads everything twice (from L2). One launch without a workspace instead of two with one (17 rows of 1000 floats: 5.1 ->
// 2.9 us, and 4.4 of 20 us on the host; 256 of 2048 float16: 8.0 -> 6.4; at 512 rows there is nothing left of it).
constexpr int kFewRows = 256, kFewCols = 4096, kFewThreads = 256;

// Sums over the rows from, from + step ... of column c, eight rows under way at once.
template<int SRC, int GRAD>
__device__ __forceinline__ void layernorm_grad_few_columns(const LayerNormGradKParams &p, int c, unsigned from, unsigned step, float &dw, float &db)
{
    constexpr int N = 8;
    for (unsigned r0 = from; r0 < p.rows; r0 += N * step)
    {
        Vec<SRC, 1>  x[N];
        Vec<GRAD, 1> g[N];
        float        mean[N], rstd[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
        {
            const unsigned r = min(r0 + k * step, p.rows - 1);
            x[k]             = load_raw<kElemBytes<SRC>>(p.src.at(r) + static_cast<long long>(c) * kElemBytes<SRC>);
            g[k]             = load_raw<kElemBytes<GRAD>>(p.grad.at(r) + static_cast<long long>(c) * kElemBytes<GRAD>);
            mean[k]          = p.mean[r];
            rstd[k]          = p.rstd[r];
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
        {
            float xv, gv;
            unpack<SRC, 1>(x[k], &xv);
            unpack<GRAD, 1>(g[k], &gv);
            if (r0 + k * step < p.rows)
            {
                db += gv;
                dw = fmaf(gv, (xv - mean[k]) * rstd[k], dw);
            }
        }
    }
}

template<int SRC>
__global__ void __launch_bounds__(kFewThreads) layernorm_grad_few_kernel(const LayerNormGradKParams p, unsigned rowCtas)
{
    constexpr int    kWarps = kFewThreads / 32, kEach = kFewCols / kFewThreads;
    __shared__ float scratch[2][32], sum[2][kWarps][32];
    const int        lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x < rowCtas)
    {
        const unsigned r = blockIdx.x;
        float          x[kEach], g[kEach], w[kEach], s1 = 0.0f, s2 = 0.0f;
        auto           at = [&](int i) { return static_cast<int>(threadIdx.x) + i * kFewThreads; };
        load_scattered<SRC, kEach>(p.src.at(r), p.cols, x, at);
        load_scattered<kEach>(p.grad.at(r), p.gradType, p.cols, g, at);
        if (p.weight)
            load_scattered<kEach>(p.weight, p.weightType, p.cols, w, at);
        const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
        {
            if (p.weight)
                g[i] *= w[i];
            x[i] = (x[i] - mean) * rstd;
            if (at(i) < p.cols)
            {
                s1 += g[i];
                s2 = fmaf(g[i], x[i], s2);
            }
        }
        const float c1 = block_sum(s1, scratch[0]) * p.invCols, c2 = block_sum(s2, scratch[1]) * p.invCols;
        uint8_t    *dx = p.dsrc.at(r);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (at(i) < p.cols)
                store_elem_as(dx, at(i), p.dsrcType, rstd * (fmaf(x[i], -c2, g[i]) - c1));
        return;
    }
    const int c = static_cast<int>(blockIdx.x - rowCtas) * 32 + lane;
    float     dw = 0.0f, db = 0.0f;
    if (c < p.cols && p.gradType == B200PP_F32)
        layernorm_grad_few_columns<SRC, B200PP_F32>(p, c, warp, kWarps, dw, db);
    else if (c < p.cols && p.gradType == B200PP_BF16)
        layernorm_grad_few_columns<SRC, B200PP_BF16>(p, c, warp, kWarps, dw, db);
    else if (c < p.cols)
        layernorm_grad_few_columns<SRC, B200PP_F16>(p, c, warp, kWarps, dw, db);
    sum[0][warp][lane] = dw;
    sum[1][warp][lane] = db;
    __syncthreads();
    if (warp > 1 || c >= p.cols)
        return;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) s += sum[warp][k][lane];
    if (warp == 0 && p.dweight)
        store_elem_as(p.dweight, c, p.dweightType, s);
    if (warp == 1 && p.dbias)
        store_elem_as(p.dbias, c, p.dbiasType, s);
}

// dx, one CTA per row, any row length: for rows above 65536 values, and for float16 rows with bfloat16 gradients or the other way round.
// Element by element (256 float16 rows of 150528 with all gradients: 1261 us; one such row, on one SM: 525 us; 50176 rows of 768 of mixed
// types: 314 us, where the one-pass kernel takes 44).
template<int SRC>
__global__ void __launch_bounds__(256) layernorm_grad_row_kernel(const LayerNormGradKParams p)
{
    __shared__ float scratch[32];
    for (unsigned r = blockIdx.x; r < p.rows; r += gridDim.x)
    {
        const uint8_t *x = p.src.at(r), *dy = p.grad.at(r);
        uint8_t       *dx   = p.dsrc.at(r);
        const float    mean = p.mean[r], rstd = p.rstd[r];
        float          s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        {
            const float w = p.weight ? load_elem(p.weight, c, p.weightType) : 1.0f;
            const float g = load_elem(dy, c, p.gradType) * w;
            s1 += g;
            s2 = fmaf(g, (load_elem<SRC>(x, c) - mean) * rstd, s2);
        }
        const float c1 = block_sum(s1, scratch) / p.fcols;
        const float c2 = block_sum(s2, scratch) / p.fcols;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        {
            const float w = p.weight ? load_elem(p.weight, c, p.weightType) : 1.0f;
            const float g = load_elem(dy, c, p.gradType) * w;
            const float h = (load_elem<SRC>(x, c) - mean) * rstd;
            store_elem_as(dx, c, p.dsrcType, rstd * (g - c1 - h * c2));
        }
    }
}

// dw and db: a CTA sums one part of the rows for 32 columns; layernorm_grad_join_kernel adds the parts up.
template<int SRC>
__global__ void __launch_bounds__(256) layernorm_grad_columns_kernel(const LayerNormGradKParams p)
{
    __shared__ float sw[8][32], sb[8][32];
    const int        lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long  c    = static_cast<long long>(blockIdx.x) * 32 + lane;
    const unsigned   per  = (p.rows + p.parts - 1) / p.parts;
    const unsigned   r0   = min(p.rows, static_cast<unsigned>(blockIdx.y) * per), r1 = min(p.rows, r0 + per);
    float            dw = 0.0f, db = 0.0f;
    if (c < p.cols)
        for (unsigned r = r0 + warp; r < r1; r += 8)
        {
            const float g = load_elem(p.grad.at(r), c, p.gradType);
            db += g;
            dw = fmaf(g, (load_elem<SRC>(p.src.at(r), c) - p.mean[r]) * p.rstd[r], dw);
        }
    sw[warp][lane] = dw;
    sb[warp][lane] = db;
    __syncthreads();
    if (warp == 0 && c < p.cols)
    {
        for (int k = 1; k < 8; ++k)
        {
            dw += sw[k][lane];
            db += sb[k][lane];
        }
        float *part       = p.partials + static_cast<long long>(blockIdx.y) * 2 * p.cols;
        part[c]           = dw;
        part[p.cols + c]  = db;
    }
}

// Adds up the parts: blockDim.y threads share a column, each takes every blockDim.y-th part, and the first joins them in order.
static __global__ void __launch_bounds__(1024) layernorm_grad_join_kernel(const LayerNormGradKParams p)
{
    __shared__ float sum[32][33];
    const long long  c = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x, n = 2LL * p.cols; // column of dw, db
    float            s = 0.0f;
    cudaGridDependencySynchronize(); // launched early
    if (c < n)
    {
#pragma unroll 4
        for (int k = threadIdx.y; k < p.parts; k += blockDim.y) s += p.partials[k * n + c];
    }
    if (blockDim.y > 1)
    {
        sum[threadIdx.y][threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.y > 0)
            return;
        float t[4] = {};
        for (int k = 0; k < static_cast<int>(blockDim.y); k += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] += sum[k + i][threadIdx.x];
        s = (t[0] + t[1]) + (t[2] + t[3]);
    }
    if (c >= n)
        return;
    if (c < p.cols)
    {
        if (p.dweight)
            store_elem_as(p.dweight, c, p.dweightType, s);
    }
    else if (p.dbias)
        store_elem_as(p.dbias, c - p.cols, p.dbiasType, s);
}

} // namespace b200pp

#endif
